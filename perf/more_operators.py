"""Workloads of the 8-bit row operators and of the drafts' verdict, for timing and comparison.

Five kinds of case, one for each operator of ramforge_b200:

  norm    norm_i8: residual add, RMS norm and 8-bit rows with a scale each, then dequantize_i8 of the rows
  swiglu  swiglu_i8: silu(gate) * up as 8-bit rows, then dequantize_i8 of the rows
  matmul  i8_matmul: 8-bit rows times an 8-bit matrix, a scale for each token and channel; with "acts" the rows are
          quantised by quantize_i8 first
  verify  verify_drafts: which drafted tokens stand, from the target's probabilities and given random numbers, and
          the token behind them
  greedy  verify_greedy: the same where the target always takes its best token

The plain form of each is written here in elementary torch operations in 32 bits (64 for sums of squares, sums of
probabilities and what is compared with them).  Cases are dicts of plain values; `dtype` is the activations' type.
A row of 8-bit codes stands for code * scale, scale = max|y| / 127 in 32 bits; codes are y * (1 / scale) rounded.
"""
import math

import numpy as np
import torch

own = False

_DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_ES = {"f32": 4, "f16": 2, "bf16": 2}
_LEAST = 2.0 ** -126  # a smaller scale counts as 0


# ---- the cases -------------------------------------------------------------------------------------------
def _norm(name, rows, cols, dtype, add):
    return {"name": name, "kind": "norm", "rows": rows, "cols": cols, "dtype": dtype, "add": add}


def _swiglu(name, rows, cols, dtype):
    return {"name": name, "kind": "swiglu", "rows": rows, "cols": cols, "dtype": dtype}


def _matmul(name, t, n, k, dtype, acts, bias):
    return {"name": name, "kind": "matmul", "t": t, "n": n, "k": k, "dtype": dtype, "acts": acts, "bias": bias}


def _verify(name, seqs, t, vocab, dtype, tree, draft, ragged):
    return {"name": name, "kind": "verify", "seqs": seqs, "t": t, "vocab": vocab, "dtype": dtype, "tree": tree,
            "draft": draft, "ragged": ragged}


def _greedy(name, seqs, t, vocab, dtype, tree, ragged):
    return {"name": name, "kind": "greedy", "seqs": seqs, "t": t, "vocab": vocab, "dtype": dtype, "tree": tree,
            "ragged": ragged}


def listed():
    return [
        # one token's hidden state between two halves of a 4096-wide layer: latency
        _norm("norm_one_row", 1, 4096, "f32", True),
        # a long prompt (odd length) between two halves of the layer: HBM bandwidth
        _norm("norm_prompt", 4001, 4096, "bf16", True),
        # a 16-token tree's gate and up rows of a 14336-wide feed-forward: latency
        _swiglu("swiglu_drafts", 16, 14336, "f16"),
        # a prompt's gate and up rows: HBM bandwidth
        _swiglu("swiglu_prompt", 2048, 14336, "bf16"),
        # plain decoding: one token through the fused [q;k;v] projection, with biases
        _matmul("matmul_one_token", 1, 6144, 4096, "f32", False, True),
        # nine nodes of a drafted chain through a 128256-row LM head, logits in 32 bits: HBM bandwidth
        _matmul("matmul_drafts_head", 9, 128256, 4096, "f32", False, False),
        # attention outputs of an odd-length prompt through the output projection, quantised on the way
        _matmul("matmul_ragged_prompt", 333, 4096, 4096, "f16", True, False),
        # a whole prompt through the fused gate/up projection: tensor cores
        _matmul("matmul_prompt", 4096, 28672, 4096, "bf16", False, False),
        # one sequence's drafted tree: latency
        _verify("verify_tree", 1, 24, 128256, "f32", True, True, False),
        # a batch of drafted chains of unequal length: HBM bandwidth
        _verify("verify_chains", 64, 8, 128256, "f32", False, True, True),
        # one short chain over a small vocabulary: latency
        _greedy("greedy_one", 1, 4, 32000, "f32", False, False),
        # a batch of drafted chains over a large vocabulary: HBM bandwidth
        _greedy("greedy_batch", 16, 8, 128256, "bf16", False, False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = rng.choice(["f32", "f16", "bf16"])
    kind = rng.choice(["norm", "swiglu", "matmul", "matmul", "verify", "greedy"])
    if kind in ("norm", "swiglu"):
        cols = _log(rng, 64, 16384)
        if rng.random() < 0.6:  # widths of real layers are multiples of 64
            cols = -(-cols // 64) * 64
        rows = max(1, min(_log(rng, 1, 8192), 4001 * 4096 // cols))
        c = _norm("", rows, cols, dtype, rng.random() < 0.7) if kind == "norm" else _swiglu("", rows, cols, dtype)
    elif kind == "matmul":
        t = _log(rng, 1, 4096)
        n, k = _log(rng, 64, 131072 if t <= 64 else 32768), _log(rng, 64, 16384)
        if rng.random() < 0.6:
            n, k = -(-n // 64) * 64, -(-k // 64) * 64
        k = max(1, min(k, 128256 * 4096 // n, 4096 * 28672 * 4096 // (t * n)))
        c = _matmul("", t, n, k, dtype, rng.random() < 0.4, rng.random() < 0.4)
    else:
        vocab, t = _log(rng, 1000, 151936), _log(rng, 1, 32)
        seqs = max(1, min(_log(rng, 1, 64), 64 * 9 * 128256 // (vocab * (t + 1))))
        tree, ragged = rng.random() < 0.5, rng.random() < 0.5
        if kind == "verify":
            c = _verify("", seqs, t, vocab, dtype, tree, rng.random() < 0.7, ragged)
        else:
            c = _greedy("", seqs, t, vocab, dtype, tree, ragged)
    del c["name"]
    return c


# ---- inputs ----------------------------------------------------------------------------------------------
def _pitch(n):
    """Elements between rows of 8-bit codes: whole 16-byte pieces."""
    return -(-n // 16) * 16


def _acts(gen, rows, cols, dt):
    """Activations as layers see them: a few channels are much larger than the others."""
    x = torch.randn(rows, cols, device="cuda", generator=gen)
    big = torch.rand(cols, device="cuda", generator=gen) < 0.01
    return (x * torch.where(big, 12.0, 1.0)).to(dt)


def _codes(gen, rows, cols, size):
    """8-bit rows with their scales: values of about `size`."""
    q = torch.zeros(rows, _pitch(cols), device="cuda", dtype=torch.int8)
    q[:, :cols] = (torch.randn(rows, cols, device="cuda", generator=gen, dtype=torch.float16) * 32).round_().clamp_(-127, 127)
    return q, (0.5 + torch.rand(rows, device="cuda", generator=gen)) * (size / 32)


def _parents(rs, seqs, t, tree):
    """[seqs][t]: the drafted token that each one follows, -1: the history's last."""
    if not tree:
        return np.tile(np.arange(-1, t - 1), (seqs, 1))
    out = np.empty((seqs, t), np.int64)
    for j in range(t):  # mostly one of the latest few, now and then another first token
        out[:, j] = np.where(rs.rand(seqs) < 0.1, -1, rs.randint(max(-1, j - 4), max(j, 0), size=seqs) if j else -1)
    return out


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rs = np.random.RandomState(seed % (1 << 32))
    dt = _DT[case["dtype"]]
    s = dict(case)
    if case["kind"] in ("norm", "swiglu"):
        rows, cols = case["rows"], case["cols"]
        if case["kind"] == "norm":
            s["x"] = _acts(gen, rows, cols, dt)
            s["res"] = _acts(gen, rows, cols, dt) if case["add"] else None
            s["w"] = 1 + 0.2 * torch.randn(cols, device="cuda", generator=gen)
            s["eps"] = 1e-5
            s["sum"] = torch.empty(rows, cols, device="cuda", dtype=dt) if case["add"] else None
            s["values"] = torch.empty(rows, cols, device="cuda", dtype=dt)
        else:  # rows of the fused projection: gate, then up
            s["gu"] = torch.randn(rows, 2 * cols, device="cuda", generator=gen).to(dt)
            # codes stand for 8 bits; exponentials in 32 bits may tip one over, which 16 bits hold
            s["values"] = torch.empty(rows, cols, device="cuda", dtype=torch.float16 if case["dtype"] == "f32" else dt)
        s["q"] = torch.empty(rows, _pitch(cols), device="cuda", dtype=torch.int8)
        s["scale"] = torch.empty(rows, device="cuda")
        return s
    if case["kind"] == "matmul":
        t, n, k = case["t"], case["n"], case["k"]
        s["w"], s["w_scale"] = _codes(gen, n, k, 0.02)
        if case["acts"]:
            s["x"] = _acts(gen, t, k, dt)
            s["xq"] = torch.empty(t, _pitch(k), device="cuda", dtype=torch.int8)
            s["x_scale"] = torch.empty(t, device="cuda")
        else:
            s["x"] = None
            s["xq"], s["x_scale"] = _codes(gen, t, k, 1.0)
        s["b"] = torch.randn(n, device="cuda", generator=gen) if case["bias"] else None
        s["y"] = torch.empty(t, n, device="cuda", dtype=dt)
        return s
    seqs, t, vocab = case["seqs"], case["t"], case["vocab"]
    parent = _parents(rs, seqs, t, case["tree"])
    s["parent"] = torch.from_numpy(parent.astype(np.int32)).cuda() if case["tree"] else None
    nd = rs.randint(0, t + 1, size=seqs) if case["ragged"] else np.full(seqs, t)
    nd[rs.randint(seqs)] = t
    s["n_draft"] = torch.from_numpy(nd.astype(np.int32)).cuda()
    s["hist"] = torch.from_numpy(rs.randint(0, 30000, size=seqs).astype(np.int32)).cuda()
    logits = 3 * torch.randn(seqs, t + 1, vocab, device="cuda", generator=gen)
    rows = torch.from_numpy(parent + 1).cuda()  # the row that each drafted token was chosen from
    at = torch.arange(seqs, device="cuda")[:, None]
    if case["kind"] == "greedy":
        s["logits"] = logits.to(dt)
        best = s["logits"].float().argmax(-1)
        other = torch.randint(0, vocab, (seqs, t), device="cuda", generator=gen)
        hit = torch.rand(seqs, t, device="cuda", generator=gen) < 0.75
        s["tokens"] = torch.where(hit, best[at, rows], other).int()
        s["best"] = torch.empty(seqs, t + 1, device="cuda", dtype=torch.int32)
    else:
        s["p"] = torch.softmax(logits, -1).to(dt)
        near = logits[:, :t].add_(0.7 * torch.randn(seqs, t, vocab, device="cuda", generator=gen))
        q = torch.softmax(near, -1).to(dt)
        # each drafted token drawn from its row of the draft's probabilities
        u = torch.rand(seqs, t, 1, device="cuda", generator=gen, dtype=torch.float64)
        cum = q.double().cumsum(-1)
        pick = torch.searchsorted(cum[at, rows], u * cum[at, rows, -1:]).clamp_(max=vocab - 1)
        del cum
        s["tokens"] = pick[..., 0].int()
        s["q"] = q if case["draft"] else None
        s["u"] = torch.rand(seqs, t, device="cuda", generator=gen)
        s["u_next"] = torch.rand(seqs, device="cuda", generator=gen)
    s["out"] = torch.empty(seqs, t + 1, device="cuda", dtype=torch.int32)
    s["count"] = torch.empty(seqs, device="cuda", dtype=torch.int32)
    s["pos"] = torch.empty(seqs, t, device="cuda", dtype=torch.int32)
    return s


# ---- one pass --------------------------------------------------------------------------------------------
def run(s):
    if own:
        return _RUN_OWN[s["kind"]](s)
    return _RUN_PLAIN[s["kind"]](s)


def _plain_rows(y):
    """Codes (as numbers) and scales [rows][1] of rows y."""
    scale = y.abs().amax(-1, keepdim=True) / torch.full((), 127.0, device=y.device)
    scale = torch.where(scale < _LEAST, 0.0, scale)
    inv = torch.where(scale > 0, 1 / scale, 0.0)
    return (y * inv).round().clamp(-127, 127), scale


def _plain_norm(s):
    x = s["x"].float()
    if s["res"] is not None:
        x = x + s["res"].float()
    r = (1 / torch.sqrt(x.double().square().mean(-1, keepdim=True) + s["eps"])).float()
    code, scale = _plain_rows(x * s["w"] * r)
    value = (code * scale).to(s["x"].dtype)
    return [value] if s["res"] is None else [x.to(s["x"].dtype), value]


def _plain_swiglu(s):
    g, u = s["gu"].float().split(s["cols"], -1)
    code, scale = _plain_rows(g / (1 + torch.exp(-g)) * u)
    return (code * scale).to(s["values"].dtype)


def _plain_matmul(s):
    k = s["k"]
    if s["x"] is None:
        x, scale = s["xq"][:, :k].float(), s["x_scale"][:, None]
    else:
        x, scale = _plain_rows(s["x"].float())
    y = (x @ s["w"][:, :k].float().T) * scale * s["w_scale"]
    if s["b"] is not None:
        y = y + s["b"]
    return y.to(s["y"].dtype)


def _plain_path(s, took):
    """Outputs of a walk: took [seqs][t] says which drafted tokens stand (they are one path)."""
    t = s["t"]
    depth = took.cumsum(-1)
    pos = torch.where(took, s["hist"][:, None] + depth - 1, -1)
    count = depth[:, -1]
    out = torch.full((s["seqs"], t + 2), -1, device=took.device, dtype=torch.int64)
    out.scatter_(1, torch.where(took, depth - 1, t + 1), s["tokens"].long())  # column t + 1 takes what is left out
    return out[:, :t + 1], count, pos


def _plain_end(out, count, pos, token):
    out = out.scatter(1, count[:, None], token[:, None])
    return {"tokens": out.int(), "count": count.int(), "positions": pos.int()}


def _plain_parents(s):
    """Parents [seqs][t], -2 behind a sequence's last draft."""
    t = s["t"]
    j = torch.arange(t, device=s["tokens"].device)
    parent = (j - 1).expand(s["seqs"], t) if s["parent"] is None else s["parent"].long()
    return torch.where(j < s["n_draft"][:, None], parent, -2)


def _plain_greedy(s):
    best = s["logits"].float().argmax(-1)  # the lowest index of equal ones
    parent = _plain_parents(s)
    at = torch.arange(s["seqs"], device=best.device)
    hit = (parent > -2) & (s["tokens"] == best.gather(1, (parent + 1).clamp(min=0)))
    cur = torch.full((s["seqs"],), -1, device=best.device)
    took = []
    for j in range(s["t"]):  # tokens stand in front of those that follow them
        took.append(hit[:, j] & (parent[:, j] == cur))
        cur = torch.where(took[-1], j, cur)
    return _plain_end(*_plain_path(s, torch.stack(took, 1)), best[at, cur + 1])


def _plain_chains(s):
    t, tokens = s["t"], s["tokens"].long()
    at = torch.arange(s["seqs"], device=tokens.device)
    left = s["p"][:, :t].gather(2, tokens[..., None])[..., 0].double()
    ask = s["u"].double()
    if s["q"] is not None:
        ask = ask * s["q"].gather(2, tokens[..., None])[..., 0].double()
    live = torch.arange(t, device=tokens.device) < s["n_draft"][:, None]
    took = ((ask < left) & live).cumprod(-1).bool()
    count = took.sum(-1)
    no = (count < s["n_draft"])[:, None]  # one was refused there
    p, last = s["p"][at, count].double(), count.clamp(max=t - 1)
    if s["q"] is None:
        rest = p.scatter(1, tokens[at, last][:, None], 0.0)
    else:
        rest = (p - s["q"][at, last].double()).clamp(min=0)
    return _plain_sample(s, torch.where(no, rest, p), p, took)


def _plain_sample(s, r, p, took):
    r = torch.where(r.sum(-1, keepdim=True) > 0, r, p)
    cum = r.cumsum(-1)
    token = (cum <= s["u_next"][:, None].double() * cum[:, -1:]).sum(-1)
    return _plain_end(*_plain_path(s, took), token)


def _plain_verify(s):
    if s["parent"] is None:
        return _plain_chains(s)
    seqs, t = s["seqs"], s["t"]
    parent, tokens = _plain_parents(s), s["tokens"].long()
    at = torch.arange(seqs, device=tokens.device)
    cur = torch.full((seqs,), -1, device=tokens.device)
    a = torch.zeros(seqs, 1, device=tokens.device, dtype=torch.float64)  # share of q that is taken off
    mass = torch.ones_like(a)
    r = s["p"][:, 0].double()  # what is left of the current node's probabilities
    took = []
    for j in range(t):  # siblings are tried in turn, each after the ones before it were refused
        here = parent[:, j] == cur
        c = tokens[:, j:j + 1]
        left = r.gather(1, c)
        if s["q"] is None:
            q, ask = None, s["u"][:, j:j + 1].double() * mass
        else:
            q = s["q"][at, (cur + 1).clamp(max=t - 1)].double()
            ask = s["u"][:, j:j + 1].double() * mass * q.gather(1, c)
        yes = here & (ask < left)[:, 0]
        no = (here & ~yes)[:, None]
        a = torch.where(no, a + mass, torch.where(yes[:, None], 0.0, a))
        cur = torch.where(yes, j, cur)
        p = s["p"][at, cur + 1].double()
        rest = r.scatter(1, c, 0.0) if q is None else (p - a * q).clamp(min=0)
        r = torch.where(no, rest, torch.where(yes[:, None], p, r))
        mass = torch.where(no, r.sum(-1, keepdim=True), torch.where(yes[:, None], 1.0, mass))
        took.append(yes)
    return _plain_sample(s, r, s["p"][at, cur + 1].double(), torch.stack(took, 1))


_RUN_PLAIN = {"norm": _plain_norm, "swiglu": _plain_swiglu, "matmul": _plain_matmul, "verify": _plain_verify,
              "greedy": _plain_greedy}


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _ptr(x):
    return 0 if x is None else x.data_ptr()


def _code(dtype):
    from ramforge_b200 import _lib
    return {torch.float32: _lib.ACT_F32, torch.float16: _lib.ACT_F16, torch.bfloat16: _lib.ACT_BF16}[dtype]


def _own_values(s):
    from ramforge_b200 import dequantize_i8
    dequantize_i8(s["q"].data_ptr(), s["scale"].data_ptr(), s["values"].data_ptr(), _code(s["values"].dtype), s["rows"],
                  s["cols"], q_stride=s["q"].stride(0), stream=_stream())
    return s["values"]


def _own_norm(s):
    from ramforge_b200 import norm_i8
    norm_i8(s["x"].data_ptr(), s["w"].data_ptr(), s["eps"], s["q"].data_ptr(), s["scale"].data_ptr(),
            _code(s["x"].dtype), s["rows"], s["cols"], add_ptr=_ptr(s["res"]), sum_ptr=_ptr(s["sum"]),
            q_stride=s["q"].stride(0), stream=_stream())
    return [_own_values(s)] if s["res"] is None else [s["sum"], _own_values(s)]


def _own_swiglu(s):
    from ramforge_b200 import swiglu_i8
    gu, cols = s["gu"], s["cols"]
    swiglu_i8(gu.data_ptr(), gu.data_ptr() + cols * gu.element_size(), s["q"].data_ptr(), s["scale"].data_ptr(),
              _code(gu.dtype), s["rows"], cols, gate_stride=2 * cols, up_stride=2 * cols, q_stride=s["q"].stride(0),
              stream=_stream())
    return _own_values(s)


def _own_matmul(s):
    from ramforge_b200 import i8_matmul, quantize_i8
    if s["x"] is not None:
        quantize_i8(s["x"].data_ptr(), s["xq"].data_ptr(), s["x_scale"].data_ptr(), _code(s["x"].dtype), s["t"], s["k"],
                    q_stride=s["xq"].stride(0), stream=_stream())
    i8_matmul(s["xq"].data_ptr(), s["x_scale"].data_ptr(), s["w"].data_ptr(), s["w_scale"].data_ptr(),
              s["y"].data_ptr(), _code(s["y"].dtype), s["t"], s["n"], s["k"], x_stride=s["xq"].stride(0),
              w_stride=s["w"].stride(0), bias_ptr=_ptr(s["b"]), stream=_stream())
    return s["y"]


def _own_verify(s):
    from ramforge_b200 import verify_drafts
    verify_drafts(s["p"].data_ptr(), _ptr(s["q"]), _code(s["p"].dtype), s["vocab"], s["seqs"], s["t"],
                  s["tokens"].data_ptr(), s["u"].data_ptr(), s["u_next"].data_ptr(), s["out"].data_ptr(),
                  s["count"].data_ptr(), parent_ptr=_ptr(s["parent"]), n_draft_ptr=s["n_draft"].data_ptr(),
                  hist_len_ptr=s["hist"].data_ptr(), positions_ptr=s["pos"].data_ptr(), stream=_stream())
    return {"tokens": s["out"], "count": s["count"], "positions": s["pos"]}


def _own_greedy(s):
    from ramforge_b200 import verify_greedy
    verify_greedy(s["logits"].data_ptr(), _code(s["logits"].dtype), s["vocab"], s["seqs"], s["t"],
                  s["tokens"].data_ptr(), s["best"].data_ptr(), s["out"].data_ptr(), s["count"].data_ptr(),
                  parent_ptr=_ptr(s["parent"]), n_draft_ptr=s["n_draft"].data_ptr(),
                  hist_len_ptr=s["hist"].data_ptr(), positions_ptr=s["pos"].data_ptr(), stream=_stream())
    return {"tokens": s["out"], "count": s["count"], "positions": s["pos"]}


_RUN_OWN = {"norm": _own_norm, "swiglu": _own_swiglu, "matmul": _own_matmul, "verify": _own_verify,
            "greedy": _own_greedy}


# ---- what a pass cannot do without -----------------------------------------------------------------------
def work(case):
    es = _ES[case["dtype"]]
    if case["kind"] in ("norm", "swiglu"):
        rows, n = case["rows"], case["rows"] * case["cols"]
        if case["kind"] == "norm":  # rows, sums, codes; then codes and values
            return {"bytes": n * ((3 if case["add"] else 1) * es + 1) + n * (1 + es) + 4 * case["cols"] + 8 * rows,
                    "flops": 7 * n}
        return {"bytes": n * (2 * es + 1) + n * (1 + min(es, 2)) + 8 * rows, "flops": 10 * n}
    if case["kind"] == "matmul":
        t, n, k = case["t"], case["n"], case["k"]
        first = t * k * (es + 1) + 4 * t if case["acts"] else 0
        return {"bytes": first + t * k + n * k + 4 * (t + n) + (4 * n if case["bias"] else 0) + t * n * es,
                "flops": 2 * t * n * k}
    seqs, t, vocab = case["seqs"], case["t"], case["vocab"]
    small = seqs * (16 * t + 12)
    if case["kind"] == "greedy":  # the rows of the tokens that stand (three in four do, while they last) and one more
        mean = sum(0.75 ** i for i in range(t + 1)) if not case["ragged"] else sum(
            sum(0.75 ** i for i in range(m + 1)) for m in range(t + 1)) / (t + 1)
        return {"bytes": int(seqs * mean * vocab * es) + small, "flops": int(seqs * mean * vocab)}
    # the last node's row of both (of the target's alone where the draft has none)
    rows = 2 if case["draft"] else 1
    return {"bytes": seqs * rows * vocab * es + small, "flops": 3 * seqs * vocab}


# ---- the same from the definition in 64 bits ---------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "swiglu": _exact_swiglu, "matmul": _exact_matmul, "verify": _exact_walk,
            "greedy": _exact_walk}[case["kind"]](s)


def _np(x):
    return x.double().cpu().numpy()


def _exact_rows(y):
    """Values of rows y (64 bits, or the format's own 32) after their codes: the scale is a 32-bit number."""
    scale = np.abs(y).max(-1, keepdims=True).astype(np.float32) / np.float32(127)
    scale[scale < np.float32(_LEAST)] = 0
    with np.errstate(divide="ignore"):
        inv = np.where(scale > 0, np.float32(1) / scale, np.float32(0))
    code = np.clip(np.rint(y * inv), -127, 127).astype(np.float64)
    return code, scale.astype(np.float64)


def _exact_norm(s):
    # the format's own roundings: the sum, the two products and the reciprocal root are 32-bit numbers
    x = _np(s["x"]).astype(np.float32)
    if s["res"] is not None:
        x = x + _np(s["res"]).astype(np.float32)
    wide = x.astype(np.float64)
    root = np.sqrt((wide * wide).sum(-1, keepdims=True) / x.shape[-1] + s["eps"])
    code, scale = _exact_rows(x * _np(s["w"]).astype(np.float32) * (1 / root).astype(np.float32))
    return [code * scale] if s["res"] is None else [wide, code * scale]


def _exact_swiglu(s):
    gu = _np(s["gu"])
    g, u = gu[:, :s["cols"]], gu[:, s["cols"]:]
    code, scale = _exact_rows(g * u / (1 + np.exp(-g)))
    return code * scale


def _exact_matmul(s):
    k = s["k"]
    if s["x"] is None:
        x, scale = s["xq"][:, :k].double(), s["x_scale"].double()
    else:
        code, scale = _exact_rows(_np(s["x"]).astype(np.float32))
        x, scale = torch.from_numpy(code).cuda(), torch.from_numpy(scale[:, 0]).cuda()
    y = torch.mm(x, s["w"][:, :k].double().t())  # whole numbers below 2^53: exact
    y.mul_(scale[:, None]).mul_(s["w_scale"].double())
    if s["b"] is not None:
        y.add_(s["b"].double())
    return y


def _exact_walk(s):
    seqs, t = s["seqs"], s["t"]
    tokens, nd, hist = s["tokens"].tolist(), s["n_draft"].tolist(), s["hist"].tolist()
    parent = [[j - 1 for j in range(t)]] * seqs if s["parent"] is None else s["parent"].tolist()
    out = np.full((seqs, t + 1), -1, np.int32)
    count, pos = np.zeros(seqs, np.int32), np.full((seqs, t), -1, np.int32)
    for b in range(seqs):
        node, n = -1, 0
        while True:
            kids = [j for j in range(nd[b]) if parent[b][j] == node]
            if s["kind"] == "greedy":
                row = _np(s["logits"][b, node + 1])
                best = int(np.flatnonzero(row == row.max())[0])
                stands = [j for j in kids if tokens[b][j] == best][:1]
            else:
                p = _np(s["p"][b, node + 1])
                left, mass, off, stands = p, 1.0, 0.0, []
                for j in kids:
                    c = tokens[b][j]
                    if s["q"] is None:
                        q = np.zeros(p.size)
                        q[c] = 1
                    else:
                        q = _np(s["q"][b, node + 1])
                    if float(s["u"][b, j]) * mass * q[c] < left[c]:
                        stands = [j]
                        break
                    off += mass
                    left = np.where(q > 0, 0, left) if s["q"] is None else np.maximum(p - off * q, 0)
                    mass = math.fsum(left)
            if not stands:
                break
            node = stands[0]
            out[b, n], pos[b, node] = tokens[b][node], hist[b] + n
            n += 1
        if s["kind"] == "verify":
            if mass <= 0 or not left.any():
                left = p
            run_sum = np.cumsum(left.astype(np.longdouble))
            best = int(np.searchsorted(run_sum, float(s["u_next"][b]) * run_sum[-1], side="right"))
        out[b, n], count[b] = best, n
    return {"tokens": out, "count": count, "positions": pos}
