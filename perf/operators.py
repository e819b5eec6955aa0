"""Workloads of the drafted-token verification operators, for timing and comparison.

Three kinds of case, one for each operator group of ramforge_b200:

  norm_rope   qk_norm_rope: per-head RMS norm of queries and keys and the position rotation, one pass
  kv_write    kv_cache_write of new rows into a cache, then kv_cache_read of the same rows
  kv_read     kv_cache_read of rows that a cache already holds
  tree        tree_attention: drafted tokens (a tree or a chain) over a cached history

The plain form of each is written here in elementary torch operations in 32 bits.  Cases are dicts of plain
values; `dtype` is the activations' type, `cache` the cache's ("f16" or "q8_0": 32-element blocks of 8-bit
codes with one f16 scale, codes and scales in two planes [sequence][kv head][position][...]).
"""
import math

import numpy as np
import torch

own = False

_DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_ES = {"f32": 4, "f16": 2, "bf16": 2}
_CLAMP = 65472.0  # magnitudes above this saturate in a q8_0 cache: 127 * f16(65472 / 127) still rounds to a finite f16


# ---- the cases -------------------------------------------------------------------------------------------
def _norm_rope(name, t, hq, hk, d, dtype, fused):
    return {"name": name, "kind": "norm_rope", "t": t, "hq": hq, "hk": hk, "d": d, "dtype": dtype, "fused": fused}


def _kv(name, kind, rows, seqs, hk, d, dtype, cache, cap, skip):
    return {"name": name, "kind": kind, "rows": rows, "seqs": seqs, "hk": hk, "d": d, "dtype": dtype, "cache": cache,
            "cap": cap, "skip": skip}


def _tree(name, b, t, hq, hk, d, hist, dtype, cache, mask, ragged):
    return {"name": name, "kind": "tree", "b": b, "t": t, "hq": hq, "hk": hk, "d": d, "hist": hist, "dtype": dtype,
            "cache": cache, "mask": mask, "ragged": ragged}


def listed():
    return [
        # one token of a 32-query, 8-KV-head layer, read out of the fused [q;k;v] row of the projection: latency
        _norm_rope("norm_rope_one_token", 1, 32, 8, 128, "f32", True),
        # a long prompt's queries and keys (odd length): HBM bandwidth
        _norm_rope("norm_rope_prompt", 4001, 32, 8, 128, "bf16", False),
        # the accepted third of a 16-token tree goes into an 8-bit cache, then is read back: latency
        _kv("kv_write_accepted", "kv_write", 16, 1, 8, 128, "f32", "q8_0", 2048, 3),
        # a batch of prompts quantised on the way into the cache and read back
        _kv("kv_write_prompts", "kv_write", 8200, 4, 8, 128, "bf16", "q8_0", 4096, 0),
        # a short f16 history with 64-wide heads read back as f32
        _kv("kv_read_short", "kv_read", 600, 2, 2, 64, "f32", "f16", 640, 0),
        # a long 8-bit history read back (a prefix handed to another layer of software)
        _kv("kv_read_long", "kv_read", 32768, 1, 8, 128, "f16", "q8_0", 32768, 0),
        # plain decoding as a tree of one token, 32/4 heads, at the end of a 32 + 128 token run: latency
        _tree("tree_one_token", 1, 1, 32, 4, 128, 160, "f32", "f16", "chain", False),
        # a 16-token tree in a chat-length context over an 8-bit cache
        _tree("tree_16", 1, 16, 32, 8, 128, 4095, "f16", "q8_0", "tree", False),
        # eight sequences of unequal history and unequal drafts, 7 query heads a KV head
        _tree("tree_batch_ragged", 8, 12, 28, 4, 128, 8192, "f32", "f16", "tree", True),
        # one token over a very long 8-bit cache: HBM bandwidth
        _tree("tree_one_token_long", 1, 1, 32, 8, 128, 131072, "f16", "q8_0", "chain", False),
        # a 64-token tree over a long 8-bit cache: tensor cores
        _tree("tree_64_long", 1, 64, 32, 8, 128, 32768, "bf16", "q8_0", "tree", False),
        # the widest: a 256-token chain (a draft run or a prompt's tail) in a 64/8-head layer
        _tree("chain_256_long", 1, 256, 64, 8, 128, 32768, "f16", "f16", "chain", False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_HEADS = [(32, 8, 128), (32, 4, 128), (64, 8, 128), (28, 4, 128), (14, 2, 64), (32, 8, 64), (8, 8, 64), (16, 2, 128)]


def draw(rng):
    hq, hk, d = rng.choice(_HEADS)
    dtype = rng.choice(["f32", "f16", "bf16"])
    cache = rng.choice(["q8_0", "f16"])
    kind = rng.choice(["norm_rope", "kv_write", "kv_read", "tree", "tree", "tree"])
    if kind == "norm_rope":
        c = _norm_rope("", _log(rng, 1, 4001), hq, hk, d, dtype, rng.random() < 0.5)
    elif kind == "tree":
        b = _log(rng, 1, 12)
        t = _log(rng, 1, 256)
        most = 256 * 64 * 32768 * 128 // (b * t * hq * d)  # no more work than the widest listed case
        hist = _log(rng, 1, max(2, min(131072 // b, most)))
        c = _tree("", b, t, hq, hk, d, hist, dtype, cache, rng.choice(["tree", "chain"]), b > 1 and rng.random() < 0.7)
    else:
        seqs = _log(rng, 1, 8)
        rows = max(seqs, _log(rng, 1, 32768 if kind == "kv_read" else 8200))
        c = _kv("", kind, rows, seqs, hk, d, dtype, cache, -(-rows // seqs) + rng.randrange(0, 200),
                rng.choice([0, 0, 3]) if kind == "kv_write" else 0)
    del c["name"]
    return c


# ---- inputs ----------------------------------------------------------------------------------------------
def _cache(gen, cache, seqs, hk, cap, d):
    """A cache as a program holds it: K and V planes (and Q8_0 scales) with values of unit scale."""
    out = {}
    for n in ("k", "v"):
        if cache == "f16":
            out[n] = torch.randn(seqs, hk, cap, d, device="cuda", generator=gen, dtype=torch.float16)
            out[n + "_scale"] = None
        else:
            x = torch.randn(seqs, hk, cap, d, device="cuda", generator=gen, dtype=torch.float16)
            out[n] = (x * 42).round_().clamp_(-127, 127).to(torch.int8)
            out[n + "_scale"] = (torch.rand(seqs, hk, cap, d // 32, device="cuda", generator=gen) * 0.012
                                 + 0.018).half()
    return out


def _ancestors(rs, t):
    """Visibility words [t][ceil(t / 32)] of one tree: each token sees its ancestors and itself."""
    vis = np.zeros((t, t), bool)
    for j in range(t):
        parent = rs.randint(max(0, j - 8), j) if j and rs.rand() > 0.05 else -1
        if parent >= 0:
            vis[j] = vis[parent]
        vis[j, j] = True
    w = -(-t // 32)
    pad = np.zeros((t, w * 32), bool)
    pad[:, :t] = vis
    return np.packbits(pad.reshape(t, w, 32), axis=-1, bitorder="little").view(np.uint32).reshape(t, w).view(np.int32)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rs = np.random.RandomState(seed % (1 << 32))
    dt = _DT[case["dtype"]]
    s = dict(case)
    hk, d = case["hk"], case["d"]
    if case["kind"] == "norm_rope":
        t, hq = case["t"], case["hq"]
        span = 8192
        if case["fused"]:  # q and k are slices of the projection's [q;k;v] rows
            qkv = torch.randn(t, (hq + 2 * hk) * d, device="cuda", generator=gen).to(dt)
            s["q"], s["k"] = qkv[:, :hq * d], qkv[:, hq * d:(hq + hk) * d]
        else:
            s["q"] = torch.randn(t, hq * d, device="cuda", generator=gen).to(dt)
            s["k"] = torch.randn(t, hk * d, device="cuda", generator=gen).to(dt)
        s["q_norm"] = 1 + 0.2 * torch.randn(d, device="cuda", generator=gen)
        s["k_norm"] = 1 + 0.2 * torch.randn(d, device="cuda", generator=gen)
        inv = 10000.0 ** (-2.0 * torch.arange(d // 2, device="cuda", dtype=torch.float64) / d)
        ang = torch.arange(span, device="cuda", dtype=torch.float64)[:, None] * inv
        s["rope"] = torch.stack([ang.cos(), ang.sin()], -1).float().contiguous()  # [position][pair][cos, sin]
        start = int(rs.randint(0, span - t + 1))
        s["pos"] = torch.arange(start, start + t, device="cuda", dtype=torch.int32)
        s["eps"] = 1e-6
        s["q_out"] = torch.empty(t, hq * d, device="cuda", dtype=dt)
        s["k_out"] = torch.empty(t, hk * d, device="cuda", dtype=dt)
        return s
    if case["kind"] in ("kv_write", "kv_read"):
        rows, seqs, cap = case["rows"], case["seqs"], case["cap"]
        s["cache_planes"] = _cache(gen, case["cache"], seqs, hk, cap, d)
        per = -(-rows // seqs)
        seq = np.arange(rows) // per
        base = rs.randint(0, cap - per + 1, size=seqs)
        pos = base[seq] + np.arange(rows) % per
        if case["skip"]:  # one row in `skip` is kept, the kept ones at consecutive positions
            keep = rs.randint(0, case["skip"], size=rows) == 0
            keep[0] = True
            for q in range(seqs):
                at = np.flatnonzero((seq == q) & keep)
                pos[at] = base[q] + np.arange(at.size)
            pos[~keep] = -1
        s["seq"] = torch.from_numpy(seq.astype(np.int32)).cuda()
        s["pos"] = torch.from_numpy(pos.astype(np.int32)).cuda()
        if case["kind"] == "kv_write":
            s["k"] = torch.randn(rows, hk * d, device="cuda", generator=gen).to(dt)
            s["v"] = torch.randn(rows, hk * d, device="cuda", generator=gen).to(dt)
            dt = torch.float16
        s["k_out"] = torch.empty(rows, hk * d, device="cuda", dtype=dt)
        s["v_out"] = torch.empty(rows, hk * d, device="cuda", dtype=dt)
        return s
    b, t, hq, hist = case["b"], case["t"], case["hq"], case["hist"]
    cap = -(-(hist + t) // 64) * 64 + 64
    s["cap"] = cap
    s["cache_planes"] = _cache(gen, case["cache"], b, hk, cap, d)
    hl, nd = np.full(b, hist), np.full(b, t)
    if case["ragged"]:
        hl = rs.randint(0, hist + 1, size=b)
        hl[rs.randint(b)] = hist
        nd = rs.randint(0, t + 1, size=b)
        nd[rs.randint(b)] = t
    for q in range(b):  # what lies past a sequence's end was never written
        end = int(hl[q] + nd[q])
        for n in ("k", "v"):
            (s["cache_planes"][n + "_scale"] if case["cache"] == "q8_0" else s["cache_planes"][n])[q, :, end:] = math.nan
    s["hist_len"] = torch.from_numpy(hl.astype(np.int32)).cuda()
    s["n_draft"] = torch.from_numpy(nd.astype(np.int32)).cuda()
    s["mask"] = (torch.from_numpy(np.stack([_ancestors(rs, t) for _ in range(b)])).cuda()
                 if case["mask"] == "tree" else None)
    s["q"] = (2 * torch.randn(b * t, hq * d, device="cuda", generator=gen)).to(dt)
    s["out"] = torch.empty(b * t, hq * d, device="cuda", dtype=dt)
    return s


# ---- one pass --------------------------------------------------------------------------------------------
def run(s):
    if own:
        return _RUN_OWN[s["kind"]](s)
    return _RUN_PLAIN[s["kind"]](s)


def _plain_norm_rope(s):
    d, pos = s["d"], s["pos"].long()
    cs = s["rope"][pos]  # [t][d/2][2]
    c, sn = cs[:, None, :, 0], cs[:, None, :, 1]

    def one(x, w):
        t = x.shape[0]
        x = x.float().reshape(t, -1, d)
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + s["eps"]) * w
        a, b = x[..., :d // 2], x[..., d // 2:]
        return torch.cat([a * c - b * sn, a * sn + b * c], -1).reshape(t, -1)

    return [one(s["q"], s["q_norm"]).to(s["q"].dtype), one(s["k"], s["k_norm"]).to(s["k"].dtype)]


def _values(planes, n, seq=None, pos=None):
    """The numbers a cache stands for, f32: all of a plane, or rows [i][kv head][d] at (seq[i], pos[i])."""
    at = (slice(None),) if seq is None else (seq, slice(None), pos)
    x = planes[n][at].float()
    sc = planes[n + "_scale"]
    if sc is None:
        return x
    sc = sc[at].float()
    return (x.unflatten(-1, (-1, 32)) * sc[..., None]).half().float().flatten(-2)


def _plain_kv_read(s):
    pos, seq = s["pos"].long(), s["seq"].long()
    here = (pos >= 0)[:, None, None]
    out = []
    for n in ("k", "v"):
        x = _values(s["cache_planes"], n, seq, pos.clamp(min=0))
        out.append(torch.where(here, x, 0.0).reshape(x.shape[0], -1).to(s[n + "_out"].dtype))
    return out


def _plain_kv_write(s):
    planes, d = s["cache_planes"], s["d"]
    kept = (s["pos"] >= 0).nonzero()[:, 0]
    seq, pos = s["seq"].long()[kept], s["pos"].long()[kept]
    for n in ("k", "v"):
        x = s[n][kept].reshape(kept.numel(), -1, d)
        if planes[n + "_scale"] is None:
            planes[n][seq, :, pos] = x.half()
            continue
        x = x.float().clamp(-_CLAMP, _CLAMP).unflatten(-1, (-1, 32))
        scale = (x.abs().amax(-1, keepdim=True) / 127).half()
        inv = torch.where(scale > 0, 1 / scale.float(), 0.0)
        planes[n][seq, :, pos] = (x * inv).round().clamp(-127, 127).to(torch.int8).flatten(-2)
        planes[n + "_scale"][seq, :, pos] = scale[..., 0]
    return _plain_kv_read(s)


def _visible(s, m):
    """[b][t][m] truth values: does drafted token t of sequence b see position p."""
    t, dev = s["t"], s["hist_len"].device
    p = torch.arange(m, device=dev)
    hl, nd = s["hist_len"].long()[:, None, None], s["n_draft"].long()[:, None, None]
    j = p - hl  # index among the drafts, negative in the history
    row = torch.arange(t, device=dev)[None, :, None]
    if s["mask"] is None:
        seen = j <= row
    else:
        bits = ((s["mask"][..., None] >> torch.arange(32, device=dev)) & 1).flatten(-2)  # [b][t][32 w]
        at = j.clamp(0, bits.shape[-1] - 1).expand(-1, t, -1)
        seen = torch.gather(bits, 2, at).bool()
    return (row < nd) & (j < nd) & ((j < 0) | seen)


def _plain_tree(s):
    b, t, hq, hk, d = s["b"], s["t"], s["hq"], s["hk"], s["d"]
    m = s["hist"] + t
    planes = {n: None if x is None else x[:, :, :m] for n, x in s["cache_planes"].items()}
    vis = _visible(s, m)
    real = vis.any(1)[:, None, :, None]  # positions nobody sees may hold anything
    k = torch.where(real, _values(planes, "k"), 0.0)
    v = torch.where(real, _values(planes, "v"), 0.0)
    g = hq // hk
    q = s["q"].float().reshape(b, t, hk, g, d).permute(0, 2, 3, 1, 4).reshape(b, hk, g * t, d)
    sc = (q @ k.transpose(-1, -2) * (1 / math.sqrt(d))).reshape(b, hk, g, t, m)
    see = vis[:, None, None]
    sc = torch.where(see, sc, -math.inf)
    top = sc.amax(-1, keepdim=True)
    e = torch.exp(sc - torch.where(top == -math.inf, 0.0, top))
    l = e.sum(-1, keepdim=True)
    o = (e.reshape(b, hk, g * t, m) @ v).reshape(b, hk, g, t, d) / torch.where(l > 0, l, 1.0)
    return o.permute(0, 3, 1, 2, 4).reshape(b * t, hq * d).to(s["q"].dtype)


_RUN_PLAIN = {"norm_rope": _plain_norm_rope, "kv_write": _plain_kv_write, "kv_read": _plain_kv_read,
              "tree": _plain_tree}


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _ptr(x):
    return 0 if x is None else x.data_ptr()


def _code(name):
    from ramforge_b200 import _lib
    return {"f32": _lib.ACT_F32, "f16": _lib.ACT_F16, "bf16": _lib.ACT_BF16}[name]


def _view(s, cap):
    from ramforge_b200 import KvView, _lib
    p = s["cache_planes"]
    seqs = s["b"] if s["kind"] == "tree" else s["seqs"]
    return KvView(_lib.TYPE_F16 if s["cache"] == "f16" else _lib.TYPE_Q8_0, _ptr(p["k"]), _ptr(p["v"]),
                  _ptr(p["k_scale"]), _ptr(p["v_scale"]), seqs, s["hk"], s["d"], cap)


def _own_norm_rope(s):
    from ramforge_b200 import qk_norm_rope
    qk_norm_rope(s["q"].data_ptr(), s["k"].data_ptr(), s["q_out"].data_ptr(), s["k_out"].data_ptr(),
                 _code(s["dtype"]), s["t"], s["hq"], s["hk"], s["d"], s["rope"].data_ptr(), s["rope"].shape[0],
                 s["pos"].data_ptr(), q_norm_ptr=s["q_norm"].data_ptr(), k_norm_ptr=s["k_norm"].data_ptr(),
                 eps=s["eps"], q_stride=s["q"].stride(0), k_stride=s["k"].stride(0), stream=_stream())
    return [s["q_out"], s["k_out"]]


def _own_kv_read(s):
    from ramforge_b200 import kv_cache_read
    kv_cache_read(_view(s, s["cap"]), s["k_out"].data_ptr(), s["v_out"].data_ptr(),
                  _code("f16" if s["kind"] == "kv_write" else s["dtype"]), s["rows"], s["pos"].data_ptr(),
                  seq_ptr=s["seq"].data_ptr(), stream=_stream())
    return [s["k_out"], s["v_out"]]


def _own_kv_write(s):
    from ramforge_b200 import kv_cache_write
    kv_cache_write(_view(s, s["cap"]), s["k"].data_ptr(), s["v"].data_ptr(), _code(s["dtype"]), s["rows"],
                   s["pos"].data_ptr(), seq_ptr=s["seq"].data_ptr(), stream=_stream())
    return _own_kv_read(s)


def _own_tree(s):
    from ramforge_b200 import tree_attention
    tree_attention(_view(s, s["cap"]), s["q"].data_ptr(), s["out"].data_ptr(), _code(s["dtype"]), s["b"], s["t"],
                   s["hq"], s["hist_len"].data_ptr(), n_draft_ptr=s["n_draft"].data_ptr(), mask_ptr=_ptr(s["mask"]),
                   stream=_stream())
    return s["out"]


_RUN_OWN = {"norm_rope": _own_norm_rope, "kv_write": _own_kv_write, "kv_read": _own_kv_read, "tree": _own_tree}


# ---- what a pass cannot do without -----------------------------------------------------------------------
def _row_bytes(cache, d):
    """Bytes of one head's K or V row in the cache."""
    return 2 * d if cache == "f16" else d + 2 * (d // 32)


def work(case):
    hk, d, es = case["hk"], case["d"], _ES[case["dtype"]]
    if case["kind"] == "norm_rope":
        t, n = case["t"], case["t"] * (case["hq"] + hk) * d
        return {"bytes": 2 * n * es + t * (4 * d + 4) + 8 * d, "flops": 7 * n}
    if case["kind"] == "kv_read":
        n = case["rows"] * hk
        return {"bytes": 2 * n * (_row_bytes(case["cache"], d) + d * es) + 8 * case["rows"], "flops": 2 * n * d}
    if case["kind"] == "kv_write":  # rows that are not kept are neither read nor written, and read back as zeros
        n = case["rows"] * hk
        kept = n / case["skip"] if case["skip"] else n
        return {"bytes": 2 * kept * (d * es + 2 * _row_bytes(case["cache"], d)) + 2 * n * d * 2 + 16 * case["rows"],
                "flops": 6 * kept * d}
    b, t, hq = case["b"], case["t"], case["hq"]
    # ragged: uniform histories and drafts, half of the largest on average
    mean = 0.5 if case["ragged"] else 1.0
    m, rows = b * mean * (case["hist"] + t), b * t
    return {"bytes": 2 * m * hk * _row_bytes(case["cache"], d) + 2 * rows * hq * d * es + 8 * b
            + (4 * rows * -(-t // 32) if case["mask"] == "tree" else 0),
            "flops": 4 * m * mean * t * hq * d}


# ---- the same from the definition in 64 bits ---------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"norm_rope": _exact_norm_rope, "kv_write": _exact_kv_write, "kv_read": _exact_kv_read,
            "tree": _exact_tree}[case["kind"]](s)


def _exact_norm_rope(s):
    out = []
    d, half = s["d"], s["d"] // 2
    table = s["rope"].double().cpu().numpy()[s["pos"].cpu().numpy()]
    turn = (table[..., 0] + 1j * table[..., 1])[:, None, :]
    for n in ("q", "k"):
        x = s[n].double().cpu().numpy().reshape(s["t"], -1, d)
        w = s[n + "_norm"].double().cpu().numpy()
        y = x * w / np.sqrt((x ** 2).sum(-1, keepdims=True) / d + s["eps"])
        z = (y[..., :half] + 1j * y[..., half:]) * turn  # each pair as a complex number, turned by its angle
        out.append(np.concatenate([z.real, z.imag], -1).reshape(s["t"], -1))
    return out


def _numbers(codes, scale):
    """f16-rounded products of codes [..., d] and scales [..., d / 32], as 64-bit numbers."""
    x = codes.astype(np.float64) * np.repeat(scale.astype(np.float64), 32, axis=-1)
    return x.astype(np.float16).astype(np.float64)


def _exact_kv_read(s):
    pos, seq = s["pos"].cpu().numpy(), s["seq"].cpu().numpy()
    out = []
    for n in ("k", "v"):
        x, sc = s["cache_planes"][n].cpu().numpy(), s["cache_planes"][n + "_scale"]
        x = x[seq, :, pos]
        x = x.astype(np.float64) if sc is None else _numbers(x, sc.cpu().numpy()[seq, :, pos])
        out.append(x.reshape(x.shape[0], -1))
    return out


def _exact_kv_write(s):
    kept = s["pos"].cpu().numpy() >= 0
    out = []
    for n in ("k", "v"):
        x = s[n].float().cpu().numpy()
        if s["cache"] == "f16":
            y = x.astype(np.float16).astype(np.float64)
        else:  # the format's own roundings: the scale's quotient in 32 bits, then f16; the code's product in 32 bits
            blk = np.clip(x, -_CLAMP, _CLAMP).reshape(x.shape[0], -1, 32)
            scale = (np.abs(blk).max(-1) / np.float32(127)).astype(np.float16)
            with np.errstate(divide="ignore"):
                inv = np.where(scale > 0, np.float32(1) / scale.astype(np.float32), np.float32(0))
            y = _numbers(np.clip(np.rint(blk * inv[..., None]), -127, 127).reshape(x.shape), scale)
        out.append(np.where(kept[:, None], y, 0.0))
    return out


def _exact_tree(s):
    b, t, hq, hk, d = s["b"], s["t"], s["hq"], s["hk"], s["d"]
    g = hq // hk
    hl, nd = s["hist_len"].tolist(), s["n_draft"].tolist()
    out = torch.zeros(b, t, hq, d, dtype=torch.float64, device="cuda")
    q = s["q"].double().reshape(b, t, hq, d)
    words = None if s["mask"] is None else s["mask"].cpu().numpy().view(np.uint32)
    for i in range(b):
        n, end = nd[i], hl[i] + nd[i]
        if n == 0:
            continue
        if words is None:
            see = np.tril(np.ones((n, n), bool))
        else:
            see = np.array([[(int(words[i, r, j // 32]) >> (j % 32)) & 1 for j in range(n)] for r in range(n)], bool)
        hide = torch.from_numpy(~see).cuda()
        for h in range(hk):
            kv = []
            for x in ("k", "v"):
                y, sc = s["cache_planes"][x][i, h, :end].double(), s["cache_planes"][x + "_scale"]
                if sc is not None:
                    y = (y * sc[i, h, :end].double().repeat_interleave(32, -1)).half().double()
                kv.append(y)
            for e in range(g):
                a = q[i, :n, h * g + e] @ kv[0].T / math.sqrt(d)
                a[:, hl[i]:].masked_fill_(hide, -math.inf)
                out[i, :n, h * g + e] = torch.softmax(a, -1) @ kv[1]
    return out.reshape(b * t, hq * d).cpu().numpy()
