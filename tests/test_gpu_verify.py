"""The drafted-token verification operators (rf_qk_norm_rope, rf_kv_cache_write/read,
rf_tree_attention) against plain restatements in 64 bits.

Tolerances, each from the kernels' arithmetic:
  norm and rotation   at most 16 f32 roundings between an input and an output (13 in the sum of
                      squares, halved by the root, then root, quotient, product and the
                      rotation's three), each 2^-24 of |y_i| + |y_partner|, then one rounding to
                      the output type (half a unit of its last place; 2^-25 f16 subnormal)
  cache               exact: the format fixes every rounding
  attention           see attention_tolerance
"""
import numpy as np
import pytest

from ramforge_b200 import (KvView, _lib, kv_cache_read, kv_cache_write, qk_norm_rope, tree_attention,
                           verify_error_word)

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

ACT = {"f32": (_lib.ACT_F32, torch.float32), "f16": (_lib.ACT_F16, torch.float16),
       "bf16": (_lib.ACT_BF16, torch.bfloat16)}
ROUND = {n: torch.finfo(dt).eps / 2 for n, (_, dt) in ACT.items()}  # one rounding to nearest: half a unit


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ---- norm and rotation ------------------------------------------------------------------------
def rope_table(n, rot):
    inv = 10000.0 ** (-2.0 * torch.arange(rot // 2, device="cuda", dtype=torch.float64) / max(rot, 1))
    a = torch.arange(n, device="cuda", dtype=torch.float64)[:, None] * inv
    return torch.stack([a.cos(), a.sin()], -1).float().contiguous()


def norm_rope_ref(x, heads, D, w, eps, table, pos, rot):
    """64-bit result and the magnitude its f32 error is measured against."""
    y = x.double().reshape(x.shape[0], heads, D)
    if w is not None:
        y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    out, mag = y.clone(), y.abs()
    h = rot // 2
    if h:
        cs = table.double()[pos.long()][:, None]
        a, b = y[..., :h], y[..., h:rot]
        out[..., :h] = a * cs[..., 0] - b * cs[..., 1]
        out[..., h:rot] = a * cs[..., 1] + b * cs[..., 0]
        mag = mag.clone()
        mag[..., :h] = mag[..., h:rot] = a.abs() + b.abs()
    return out.reshape(x.shape[0], -1), mag.reshape(x.shape[0], -1)


def close_norm_rope(got, ref, mag, dtype):
    tol = 16 * 2.0 ** -24 * mag + ROUND[dtype] * ref.abs() * 1.001 + (2.0 ** -25 if dtype == "f16" else 1e-30)
    err = (got.double() - ref).abs()
    assert (err <= tol).all(), (err - tol).max().item()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("T,HQ,HK,D,rot", [
    (1, 32, 8, 128, 128), (3, 28, 4, 128, 128), (17, 14, 2, 64, 64), (70, 7, 1, 64, 64), (5, 3, 3, 256, 256),
    (9, 32, 4, 128, 64), (2, 5, 1, 96, 96), (33, 4, 2, 80, 80), (4, 2, 1, 2, 2), (6, 9, 2, 6, 4), (257, 32, 8, 128, 0),
    (11, 4, 2, 32, 32), (3, 6, 5, 16, 16), (1000, 8, 8, 128, 128)])
def test_norm_rope_shapes(T, HQ, HK, D, rot, dtype):
    code, dt = ACT[dtype]
    g = gen(T * 7 + HQ + D + rot)
    q = (3 * torch.randn(T, HQ * D, device="cuda", generator=g)).to(dt)
    k = torch.randn(T, HK * D, device="cuda", generator=g).to(dt)
    wq, wk = (1 + torch.randn(D, device="cuda", generator=g) for _ in range(2))
    table = rope_table(500, rot) if rot else None
    pos = torch.randint(0, 500, (T,), device="cuda", generator=g, dtype=torch.int32)
    qo, ko = torch.full_like(q, float("nan")), torch.full_like(k, float("nan"))
    qk_norm_rope(q.data_ptr(), k.data_ptr(), qo.data_ptr(), ko.data_ptr(), code, T, HQ, HK, D,
                 table.data_ptr() if rot else 0, 500 if rot else 0, pos.data_ptr() if rot else 0, wq.data_ptr(),
                 wk.data_ptr(), 1e-5, rot_dim=rot)
    for x, o, h, w in ((q, qo, HQ, wq), (k, ko, HK, wk)):
        close_norm_rope(o, *norm_rope_ref(x, h, D, w, 1e-5, table, pos, rot), dtype)
    assert verify_error_word() == 0


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("offset,pad", [(0, 0), (0, 1), (1, 0), (4, 8), (8, 64)])
def test_norm_rope_strides_and_alignment(dtype, offset, pad):
    """q and k as slices of fused rows that start at any element, with any row pitch; only one has a norm."""
    code, dt = ACT[dtype]
    T, HQ, HK, D = 13, 6, 2, 128
    row = (HQ + 2 * HK) * D + pad
    g = gen(offset * 100 + pad)
    buf = torch.randn(T * row + offset, device="cuda", generator=g).to(dt)
    fused = buf[offset:].view(T, row)
    q, k = fused[:, :HQ * D], fused[:, HQ * D:(HQ + HK) * D]
    w = 1 + torch.randn(D, device="cuda", generator=g)
    table, pos = rope_table(64, D), torch.arange(T, device="cuda", dtype=torch.int32)
    qo = torch.full((T, HQ * D + pad), 7.0, device="cuda", dtype=dt)
    ko = torch.full((T, HK * D), 7.0, device="cuda", dtype=dt)
    qk_norm_rope(q.data_ptr(), k.data_ptr(), qo.data_ptr(), ko.data_ptr(), code, T, HQ, HK, D, table.data_ptr(), 64,
                 pos.data_ptr(), k_norm_ptr=w.data_ptr(), q_stride=row, k_stride=row, q_out_stride=HQ * D + pad)
    close_norm_rope(qo[:, :HQ * D], *norm_rope_ref(q, HQ, D, None, 0, table, pos, D), dtype)
    close_norm_rope(ko, *norm_rope_ref(k, HK, D, w, 1e-6, table, pos, D), dtype)
    assert (qo[:, HQ * D:] == 7).all()
    # in place, on a stream of its own
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    keep = fused.clone()
    qk_norm_rope(q.data_ptr(), k.data_ptr(), q.data_ptr(), k.data_ptr(), code, T, HQ, HK, D, table.data_ptr(), 64,
                 pos.data_ptr(), k_norm_ptr=w.data_ptr(), q_stride=row, k_stride=row, q_out_stride=row,
                 k_out_stride=row, stream=s.cuda_stream)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(q, qo[:, :HQ * D]) and torch.equal(k, ko)
    assert torch.equal(fused[:, (HQ + HK) * D:], keep[:, (HQ + HK) * D:])


@pytest.mark.parametrize("D", [128, 80])
def test_norm_rope_positions_out_of_range_and_extreme_rows(D):
    T, HQ = 6, 4
    q = torch.randn(T, HQ * D, device="cuda", generator=gen(1))
    q[1] = 0.0                    # a row of zeros stays zeros: eps keeps the quotient finite
    q[2, :D] = float("nan")
    q[3] *= 1e-18
    table = rope_table(10, D)
    w = torch.ones(D, device="cuda")
    pos = torch.tensor([9, 0, 3, 5, -1, 10], device="cuda", dtype=torch.int32)
    out = torch.full_like(q, 5.0)
    qk_norm_rope(q.data_ptr(), 0, out.data_ptr(), 0, _lib.ACT_F32, T, HQ, 0, D, table.data_ptr(), 10, pos.data_ptr(),
                 q_norm_ptr=w.data_ptr(), eps=1e-6)
    assert verify_error_word() == 2 and verify_error_word() == 0
    assert (out[4:] == 5).all() and (out[1] == 0).all()
    assert out[2, :D].isnan().all() and not out[2, D:].isnan().any()
    ref, mag = norm_rope_ref(q[[0, 3]], HQ, D, w, 1e-6, table, pos[[0, 3]], D)
    close_norm_rope(out[[0, 3]], ref, mag, "f32")
    qk_norm_rope(q.data_ptr(), 0, out.data_ptr(), 0, _lib.ACT_F32, 0, HQ, 0, D, table.data_ptr(), 10, pos.data_ptr())


# ---- the cache ---------------------------------------------------------------------------------
class Cache:
    def __init__(self, kind, seqs, hk, cap, D, fill=0):
        self.kind, self.shape = kind, (seqs, hk, cap, D)
        if kind == "q8_0":
            self.k, self.v = (torch.full((seqs, hk, cap, D), fill, device="cuda", dtype=torch.int8) for _ in range(2))
            self.ks, self.vs = (torch.full((seqs, hk, cap, D // 32), 1.0, device="cuda", dtype=torch.float16)
                                for _ in range(2))
        else:
            self.k, self.v = (torch.full((seqs, hk, cap, D), fill, device="cuda", dtype=torch.float16)
                              for _ in range(2))
            self.ks = self.vs = None
        p = lambda x: 0 if x is None else x.data_ptr()  # noqa: E731
        self.view = KvView(_lib.TYPE_Q8_0 if kind == "q8_0" else _lib.TYPE_F16, p(self.k), p(self.v), p(self.ks),
                           p(self.vs), seqs, hk, D, cap)

    def values(self, which):
        x, s = (self.k, self.ks) if which == "k" else (self.v, self.vs)
        if s is None:
            return x.double()
        return (x.double() * s.double().repeat_interleave(32, -1)).half().double()


def q8_ref(x):
    """Codes and scales of f32 rows [..., D], the format's own arithmetic in numpy."""
    b = x.reshape(x.shape[:-1] + (-1, 32)).astype(np.float32)
    nan = np.isnan(b).any(-1)
    b = np.clip(b, np.float32(-65472), np.float32(65472))
    with np.errstate(all="ignore"):
        scale = (np.abs(b).max(-1) / np.float32(127)).astype(np.float16)
        inv = np.where(scale > 0, np.float32(1) / scale.astype(np.float32), np.float32(0)).astype(np.float32)
        codes = np.clip(np.rint(b * inv[..., None]), -127, 127)
    codes[nan] = 0
    scale[nan] = np.nan
    return codes.astype(np.int8).reshape(x.shape), scale


def write_read(kind, dtype, rows, seqs, hk, D, cap, seed, k=None, v=None, skip=False):
    code, dt = ACT[dtype]
    rs = np.random.RandomState(seed)
    places = rs.permutation(seqs * cap)[:rows]
    seq, pos = (places // cap).astype(np.int32), (places % cap).astype(np.int32)
    if skip:
        pos[rs.rand(rows) < 0.4] = -1 - rs.randint(0, 5)
    g = gen(seed)
    k = torch.randn(rows, hk * D, device="cuda", generator=g) * 3 if k is None else k
    v = torch.randn(rows, hk * D, device="cuda", generator=g) if v is None else v
    k, v = k.to(dt), v.to(dt)
    c = Cache(kind, seqs, hk, cap, D, fill=3)
    ds, dp = torch.from_numpy(seq).cuda(), torch.from_numpy(pos).cuda()
    kv_cache_write(c.view, k.data_ptr(), v.data_ptr(), code, rows, dp.data_ptr(), ds.data_ptr())
    for which, src in (("k", k), ("v", v)):
        x = src.float().cpu().numpy().reshape(rows, hk, D)
        plane, sc = (c.k, c.ks) if which == "k" else (c.v, c.vs)
        want = np.full((seqs, hk, cap, D), 3, np.int8 if kind == "q8_0" else np.float16)
        kept = pos >= 0
        if kind == "q8_0":
            codes, scale = q8_ref(x)
            ws = np.ones((seqs, hk, cap, D // 32), np.float16)
            want[seq[kept], :, pos[kept]] = codes[kept]
            ws[seq[kept], :, pos[kept]] = scale[kept]
            assert np.array_equal(sc.cpu().numpy(), ws, equal_nan=True)
        else:
            with np.errstate(over="ignore"):
                want[seq[kept], :, pos[kept]] = x[kept].astype(np.float16)
        assert np.array_equal(plane.cpu().numpy(), want, equal_nan=kind != "q8_0")
    for od in ("f32", "f16", "bf16"):
        ko, vo = (torch.full((rows, hk * D), 9.0, device="cuda", dtype=ACT[od][1]) for _ in range(2))
        kv_cache_read(c.view, ko.data_ptr(), vo.data_ptr(), ACT[od][0], rows, dp.data_ptr(), ds.data_ptr())
        for which, o in (("k", ko), ("v", vo)):
            val = c.values(which)[ds.long(), :, dp.long().clamp(min=0)].reshape(rows, -1)
            val = torch.where((dp >= 0)[:, None], val, 0.0).to(ACT[od][1])
            assert torch.equal(torch.nan_to_num(o, nan=1e4), torch.nan_to_num(val, nan=1e4))
    assert verify_error_word() == 0
    return c


@pytest.mark.parametrize("kind", ["q8_0", "f16"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,seqs,hk,D,cap,skip", [
    (1, 1, 1, 32, 1, False), (1, 1, 8, 128, 5, False), (16, 1, 8, 128, 40, True), (37, 3, 2, 64, 20, True),
    (5, 2, 3, 96, 4, False), (130, 4, 1, 256, 50, False), (300, 2, 4, 128, 171, True), (4, 1, 5, 160, 7, False)])
def test_cache_write_read(kind, dtype, rows, seqs, hk, D, cap, skip):
    write_read(kind, dtype, rows, seqs, hk, D, cap, rows + D, skip=skip)


@pytest.mark.parametrize("kind", ["q8_0", "f16"])
def test_cache_extreme_values(kind):
    """Zeros, subnormal scales, the largest f16, values beyond it, infinities and NaN, one block each."""
    D = 128
    k = torch.randn(8, D, device="cuda", generator=gen(2))
    k[0] = 0.0
    k[1, :32] = 1e-6 * torch.randn(32, device="cuda", generator=gen(3))
    k[1, 32:64] = 1e-9
    k[2, 5], k[2, 40] = 65504.0, -65472.0
    k[3, 5], k[3, 70] = 3e38, -1e10
    k[4, 33], k[4, 100] = float("inf"), -float("inf")
    k[5, 64] = float("nan")
    k[6] = torch.arange(D, device="cuda") - 64.0  # codes on rounding ties
    k[7, 1] = 5e-5
    c = write_read(kind, "f32", 8, 1, 1, D, 9, 4, k=k, v=k.flip(0).contiguous())
    if kind == "q8_0":
        x = c.values("k")
        assert torch.isfinite(x[~x.isnan()]).all() and x.abs().nan_to_num().max() <= 65504


def test_cache_rows_out_of_range_are_left_out():
    c = Cache("q8_0", 2, 1, 4, 32)
    k = torch.ones(5, 32, device="cuda")
    pos = torch.tensor([4, 0, 0, 3, 2], device="cuda", dtype=torch.int32)
    seq = torch.tensor([0, 2, -1, 1, 0], device="cuda", dtype=torch.int32)
    kv_cache_write(c.view, k.data_ptr(), k.data_ptr(), _lib.ACT_F32, 5, pos.data_ptr(), seq.data_ptr())
    assert verify_error_word() == 2 and verify_error_word() == 0
    want = torch.zeros(2, 1, 4, 32, dtype=torch.int8, device="cuda")
    want[1, 0, 3] = want[0, 0, 2] = 127
    assert torch.equal(c.k, want)
    o = torch.full((5, 32), 9.0, device="cuda")
    kv_cache_read(c.view, o.data_ptr(), 0, _lib.ACT_F32, 5, pos.data_ptr(), seq.data_ptr())
    assert verify_error_word() == 2
    assert (o[:3] == 0).all() and ((o[3:] - 1).abs() < 1e-3).all()


def test_cache_row_strides():
    T, HK, D = 9, 2, 64
    row = 4 * HK * D + 16
    fused = torch.randn(T, row, device="cuda", generator=gen(5)).half()
    k, v = fused[:, 2 * HK * D:3 * HK * D], fused[:, 3 * HK * D:4 * HK * D]
    pos = torch.arange(T, device="cuda", dtype=torch.int32)
    a, b = Cache("q8_0", 1, HK, T, D), Cache("q8_0", 1, HK, T, D)
    kv_cache_write(a.view, k.data_ptr(), v.data_ptr(), _lib.ACT_F16, T, pos.data_ptr(), k_stride=row, v_stride=row)
    kc, vc = k.contiguous(), v.contiguous()
    kv_cache_write(b.view, kc.data_ptr(), vc.data_ptr(), _lib.ACT_F16, T, pos.data_ptr())
    assert torch.equal(a.k, b.k) and torch.equal(a.vs, b.vs)
    o = torch.zeros(T, row, device="cuda", dtype=torch.float16)
    kv_cache_read(a.view, o[:, HK * D:].data_ptr(), o[:, 3 * HK * D:].data_ptr(), _lib.ACT_F16, T, pos.data_ptr(),
                  k_stride=row, v_stride=row)
    assert torch.equal(o[:, HK * D:2 * HK * D].double(), a.values("k")[0].transpose(0, 1).reshape(T, -1))
    assert torch.equal(o[:, 3 * HK * D:4 * HK * D].double(), a.values("v")[0].transpose(0, 1).reshape(T, -1))
    assert (o[:, :HK * D] == 0).all() and (o[:, 2 * HK * D:3 * HK * D] == 0).all() and (o[:, 4 * HK * D:] == 0).all()


# ---- attention ----------------------------------------------------------------------------------
def words_of(vis):
    """Truth values [B][T][T] -> visibility words."""
    B, T, _ = vis.shape
    w = -(-T // 32)
    pad = np.zeros((B, T, w * 32), bool)
    pad[:, :, :T] = vis
    return torch.from_numpy(np.packbits(pad.reshape(B, T, w, 32), -1, "little").view(np.int32).reshape(B, T, w)).cuda()


def tree(rs, T):
    vis = np.zeros((T, T), bool)
    for j in range(T):
        p = rs.randint(max(0, j - 6), j) if j and rs.rand() > 0.15 else -1
        if p >= 0:
            vis[j] = vis[p]
        vis[j, j] = True
    return vis


def random_cache(kind, B, hk, cap, D, seed):
    c = Cache(kind, B, hk, cap, D)
    g = gen(seed)
    for x, s in ((c.k, c.ks), (c.v, c.vs)):
        r = torch.randn(x.shape, device="cuda", generator=g)
        if kind == "q8_0":
            x.copy_((r * 42).round().clamp(-127, 127))
            s.copy_(torch.rand(s.shape, device="cuda", generator=g) * 0.012 + 0.018)
        else:
            x.copy_(r)
    return c


def attention_ref(c, q, B, T, HQ, hist, drafts, vis, scale):
    """64-bit outputs [B*T][HQ*D], the largest scale * sum|q k| met and the largest |v|."""
    _, hk, _, D = c.shape
    G = HQ // hk
    out = torch.zeros(B, T, HQ, D, dtype=torch.float64, device="cuda")
    qq = q.double().reshape(B, T, HQ, D)
    K, V = c.values("k"), c.values("v")
    sabs = vmax = 0.0
    for b in range(B):
        L, n = hist[b], drafts[b]
        if n == 0 or L + n == 0:
            continue
        see = np.ones((n, L + n), bool)
        see[:, L:] = np.tril(np.ones((n, n), bool)) if vis is None else vis[b][:n, :n]
        see_t = torch.from_numpy(see).cuda()
        some = see_t.any(-1)
        for h in range(HQ):
            k, v = K[b, h // G, :L + n], V[b, h // G, :L + n]
            x = qq[b, :n, h]
            s = (x @ k.T * scale).masked_fill(~see_t, -np.inf)
            p = torch.softmax(s, -1)
            p = torch.where(see_t, p, 0.0)
            vv = torch.where(see_t.any(0)[:, None], v, 0.0)
            o = torch.stack([p[r][see_t[r]] @ vv[see_t[r]] for r in range(n)]) if not torch.isfinite(vv).all() \
                else p @ vv
            out[b, :n, h] = torch.where(some[:, None], o, 0.0)
            sabs = max(sabs, (x.abs() @ k.abs().T * scale).nan_to_num().max().item())
            vmax = max(vmax, v.abs().nan_to_num().max().item())
    return out.reshape(B * T, -1), sabs, vmax


def attention_tolerance(dtype, ref, sabs, vmax, n, D):
    """Bound of |out - ref|.  A softmax average moves by at most 2 max|ds| max|v| when scores move by ds, and by
    the relative error of the weights times max|v|.
      ds       the split query keeps 22 bits (2^-22), the products' sums run in D/16 steps of 2^-23 (a tensor
               core's sum truncates) and two more; each of scale * sum|q k|
      weights  2^-20 for exp and its argument's rounding; f32 sums over n keys in steps of 16 or more keys,
               2^-23 each; 16-bit activations: weights rounded to f16 (2^-11, at most 2^-25 absolute below 2^-14)
    and the output's own rounding."""
    t = vmax * (2 * sabs * (2.0 ** -22 + (D / 16 + 2) * 2.0 ** -23) + 2.0 ** -20 + (n / 16 + 8) * 2.0 ** -23)
    if dtype != "f32":
        t += vmax * (2.0 ** -11 + n * 2.0 ** -25)
    return t + ROUND[dtype] * ref.abs() + 2.0 ** -25


def run_tree(c, dtype, B, T, HQ, hist, drafts, vis, seed, scale=0.0, q=None, stream=0):
    code, dt = ACT[dtype]
    D = c.shape[3]
    if q is None:
        q = 2 * torch.randn(B * T, HQ * D, device="cuda", generator=gen(seed))
    q = q.to(dt)
    out = torch.full((B * T, HQ * D), float("nan"), device="cuda", dtype=dt)
    hl = torch.tensor(hist, device="cuda", dtype=torch.int32)
    nd = None if drafts is None else torch.tensor(drafts, device="cuda", dtype=torch.int32)
    mask = None if vis is None else words_of(vis)
    tree_attention(c.view, q.data_ptr(), out.data_ptr(), code, B, T, HQ, hl.data_ptr(),
                   0 if nd is None else nd.data_ptr(), 0 if mask is None else mask.data_ptr(), scale, stream=stream)
    torch.cuda.synchronize()
    return q, out


def check_tree(kind, dtype, B, T, HQ, hk, D, hist, drafts, masked, seed=0, scale=0.0):
    rs = np.random.RandomState(seed + T)
    hist = [hist] * B if isinstance(hist, int) else hist
    dr = [T] * B if drafts is None else drafts
    cap = max(h + n for h, n in zip(hist, dr)) + 3
    c = random_cache(kind, B, hk, cap, D, seed + 11)
    for b in range(B):  # never written: anything may be there
        for x in ((c.ks, c.vs) if kind == "q8_0" else (c.k, c.v)):
            x[b, :, hist[b] + dr[b]:] = float("nan")
    vis = np.stack([tree(rs, T) for _ in range(B)]) if masked else None
    q, out = run_tree(c, dtype, B, T, HQ, hist, drafts, vis, seed, scale)
    ref, sabs, vmax = attention_ref(c, q, B, T, HQ, hist, dr, vis, scale or D ** -0.5)
    err = (out.double() - ref).abs()
    tol = attention_tolerance(dtype, ref, sabs, vmax, cap, D)
    assert not out.isnan().any()
    assert (err <= tol).all(), ((err / tol).max().item(), err.max().item())
    assert verify_error_word() == 0


@pytest.mark.parametrize("kind", ["q8_0", "f16"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("B,T,HQ,hk,D,hist,masked", [
    (1, 1, 32, 4, 128, 160, False),      # plain decoding
    (1, 1, 1, 1, 64, 0, False),          # one token, no history: out = v
    (1, 2, 2, 2, 128, 1, True),
    (1, 3, 28, 4, 128, 127, True),       # 7 query heads a KV head
    (1, 5, 14, 2, 64, 128, True),
    (2, 16, 32, 8, 128, 129, True),
    (1, 33, 8, 2, 64, 255, True),        # mask rows of two words, drafts across a 32-word edge
    (3, 40, 8, 8, 128, 77, False),
    (1, 64, 16, 2, 128, 700, True),      # 512 rows a KV head
    (1, 130, 7, 7, 64, 31, True),        # drafts longer than a key tile
    (2, 7, 12, 4, 128, 2000, True),
    (1, 1, 64, 1, 128, 900, False)])     # one KV head, 64 query heads
def test_tree_shapes(kind, dtype, B, T, HQ, hk, D, hist, masked):
    check_tree(kind, dtype, B, T, HQ, hk, D, hist, None, masked, seed=T + hist)


@pytest.mark.parametrize("kind", ["q8_0", "f16"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_tree_ragged_batches(kind, dtype):
    """Histories and draft counts of zero, one and many side by side."""
    check_tree(kind, dtype, 6, 9, 8, 2, 128, [0, 1, 513, 0, 130, 64], [9, 0, 5, 0, 1, 9], True, seed=3)
    check_tree(kind, dtype, 9, 4, 4, 4, 64, [3, 2500, 0, 0, 255, 256, 257, 1, 90], [4, 4, 0, 3, 2, 1, 4, 0, 4], False,
               seed=4)


@pytest.mark.parametrize("kind", ["q8_0", "f16"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_tree_ctas_that_change_units(kind, dtype):
    """More work units than SMs: a CTA ends one unit and begins another, with runs of a single key tile and row
    tiles that are half empty or less among them."""
    check_tree(kind, dtype, 5, 40, 32, 8, 128, 1100, None, True, seed=40)
    rs = np.random.RandomState(1)
    hist = rs.randint(0, 900, 24).tolist()
    drafts = rs.choice([3, 20, 32, 33, 64], 24, p=[.3, .2, .2, .1, .2]).tolist()
    check_tree(kind, dtype, 24, 64, 32, 8, 128, hist, drafts, True, seed=41)
    check_tree(kind, dtype, 24, 64, 32, 8, 64, hist, drafts, False, seed=42)
    check_tree(kind, dtype, 24, 4, 32, 8, 128, hist, [min(n, 4) for n in drafts], True, seed=43)


@pytest.mark.parametrize("kind", ["q8_0", "f16"])
def test_tree_one_key_tile_then_many(kind):
    """200 tokens over 20000 positions: a CTA whose first unit has one tile left, and the next ones 46."""
    check_tree(kind, "f32", 1, 200, 28, 4, 128, 20000, None, True, seed=44)


@pytest.mark.parametrize("T", [1, 2, 4, 8, 15, 17, 31, 32, 48, 65, 100])
def test_tree_lengths(T):
    """Row counts around every tile edge (4 query heads a KV head), odd histories."""
    for hist in (0, 63, 64, 65, 1023):
        check_tree("q8_0", "f16", 1, T, 8, 2, 128, hist, None, True, seed=hist)
    check_tree("f16", "f32", 1, T, 8, 2, 64, 321, None, True, seed=5)


def test_tree_scale_and_sharp_scores():
    """Scores far apart (one key takes nearly all the weight), and a scale of the caller's."""
    check_tree("f16", "f32", 1, 6, 8, 2, 128, 500, None, True, seed=6, scale=0.9)
    check_tree("q8_0", "f16", 1, 20, 8, 2, 128, 500, None, True, seed=7, scale=1.3)
    check_tree("q8_0", "bf16", 1, 20, 8, 2, 64, 500, None, True, seed=8, scale=1e-6)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("T,HQ", [(4, 4), (40, 8)])
def test_tree_rows_that_see_nothing_and_hidden_nan(dtype, T, HQ):
    """No history: a token whose mask row is empty gets zeros.  A draft whose K or V is NaN or infinite
    reaches only the tokens that see it."""
    hk, D = 2, 128
    for kind in ("q8_0", "f16"):
        c = random_cache(kind, 1, hk, 300, D, 9)
        vis = np.tril(np.ones((1, T, T), bool))
        vis[0, 2] = False            # sees nothing
        vis[0, :, 1] = False         # draft 1 is seen by token 1 alone
        vis[0, 1, 1] = True
        vis[0, :, 3] = False         # nobody sees draft 3
        plane_k, plane_v = (c.ks, c.vs) if kind == "q8_0" else (c.k, c.v)
        for hist in (0, 200):
            for bad in (float("nan"), float("inf")):
                plane_v[0, :, hist + 1] = bad
                plane_k[0, :, hist + 3] = bad
                plane_v[0, :, hist + 3] = bad
                q, out = run_tree(c, dtype, 1, T, HQ, [hist], None, vis, 10)
                rest = [t for t in range(T) if t not in (1,)]
                ref, sabs, vmax = attention_ref(c, q, 1, T, HQ, [hist], [T], vis, D ** -0.5)
                o = out.reshape(T, -1)
                vmax = min(vmax, 6.0)
                tol = attention_tolerance(dtype, ref[rest], min(sabs, 1e3), vmax, hist + T, D)
                assert ((o[rest].double() - ref[rest]).abs() <= tol).all(), (kind, hist, bad)
                assert not torch.isfinite(o[1]).any()
                if hist == 0:
                    assert (o[2] == 0).all()
                plane_v[0, :, hist + 1] = 0.5
                plane_k[0, :, hist + 3] = 0.5
                plane_v[0, :, hist + 3] = 0.5


def test_tree_nan_query_stays_in_its_row():
    for T, HQ in ((3, 4), (48, 8)):
        c = random_cache("q8_0", 1, 2, 400, 128, 12)
        q = torch.randn(T, HQ * 128, device="cuda", generator=gen(13))
        _, clean = run_tree(c, "f16", 1, T, HQ, [300], None, None, 0, q=q)
        q2 = q.clone()
        q2[1, 128:256] = float("nan")
        _, out = run_tree(c, "f16", 1, T, HQ, [300], None, None, 0, q=q2)
        assert out[1, 128:256].isnan().all()
        out[1, 128:256] = clean[1, 128:256]
        assert torch.equal(out, clean)


def test_tree_large_and_small_queries():
    """Magnitudes that leave f16: queries near 1e6 against keys near 1e-5, and the reverse."""
    for dtype in ("f32", "bf16"):
        for qs, ks in ((1e6, 2e-6), (1e-7, 1e4)):
            for T in (2, 40):
                c = random_cache("f16", 1, 2, 300, 128, 14)
                c.k.mul_(ks)
                q = torch.randn(T, 8 * 128, device="cuda", generator=gen(15)) * qs
                q, out = run_tree(c, dtype, 1, T, 8, [200], None, None, 0, q=q)
                ref, sabs, vmax = attention_ref(c, q, 1, T, 8, [200], [T], None, 128 ** -0.5)
                err = (out.double() - ref).abs()
                assert (err <= attention_tolerance(dtype, ref, sabs, vmax, 300, 128)).all(), (dtype, qs, T)


def test_tree_lengths_that_do_not_fit_are_reported():
    c = random_cache("q8_0", 4, 2, 50, 64, 16)
    q, out = run_tree(c, "f32", 4, 3, 4, [10, 48, -1, 5], [3, 3, 2, 4], None, 17)
    assert verify_error_word() == 2 and verify_error_word() == 0
    assert (out[3:] == 0).all() and out[:3].abs().sum() > 0
    ref, sabs, vmax = attention_ref(c, q, 4, 3, 4, [10, 0, 0, 0], [3, 0, 0, 0], None, 0.125)
    assert ((out.double() - ref).abs() <= attention_tolerance("f32", ref, sabs, vmax, 50, 64)).all()


@pytest.mark.parametrize("T,dtype", [(1, "f16"), (6, "f32"), (64, "bf16")])
def test_tree_offsets_past_32_bits(T, dtype):
    """The second sequence's planes start past 2^31 elements."""
    hk, D, cap = 8, 128, 2_200_000
    c = Cache("q8_0", 2, hk, cap, D)
    hist = 400
    small = random_cache("q8_0", 2, hk, hist + T, D, 18)
    for big, x in ((c.k, small.k), (c.v, small.v), (c.ks, small.ks), (c.vs, small.vs)):
        big[:, :, :hist + T] = x
    q, out = run_tree(c, dtype, 2, T, 16, [hist, hist], None, None, 19)
    _, want = run_tree(small, dtype, 2, T, 16, [hist, hist], None, None, 19, q=q.float())
    assert torch.equal(out, want)
    pos = torch.tensor([cap - 1], device="cuda", dtype=torch.int32)
    seq = torch.tensor([1], device="cuda", dtype=torch.int32)
    k = torch.randn(1, hk * D, device="cuda", generator=gen(20))
    kv_cache_write(c.view, k.data_ptr(), k.data_ptr(), _lib.ACT_F32, 1, pos.data_ptr(), seq.data_ptr())
    codes, _ = q8_ref(k.cpu().numpy().reshape(hk, D))
    assert np.array_equal(c.k[1, :, cap - 1].cpu().numpy(), codes)
    o = torch.empty(1, hk * D, device="cuda")
    kv_cache_read(c.view, o.data_ptr(), 0, _lib.ACT_F32, 1, pos.data_ptr(), seq.data_ptr())
    assert ((o - k).abs() <= k.abs().max() / 127).all()


def test_tree_strided_rows_repeat_and_streams():
    """q inside fused rows, out with a pitch; the same call gives the same bits, on any stream, side by side."""
    hk, HQ, D, T, B = 2, 8, 128, 12, 2
    c = random_cache("q8_0", B, hk, 1500, D, 21)
    row = (HQ + 2 * hk) * D
    fused = torch.randn(B * T, row, device="cuda", generator=gen(22)).half()
    hl = torch.tensor([1400, 333], device="cuda", dtype=torch.int32)
    out = torch.full((B * T, HQ * D + 8), 3.0, device="cuda", dtype=torch.float16)
    call = lambda o, st: tree_attention(c.view, fused.data_ptr(), o.data_ptr(), _lib.ACT_F16, B, T, HQ,  # noqa: E731
                                        hl.data_ptr(), q_stride=row, out_stride=HQ * D + 8, stream=st)
    call(out, 0)
    q = fused[:, :HQ * D].contiguous()
    _, want = run_tree(c, "f16", B, T, HQ, [1400, 333], None, None, 0, q=q)
    assert torch.equal(out[:, :HQ * D], want) and (out[:, HQ * D:] == 3).all()
    streams = [torch.cuda.Stream() for _ in range(4)]
    outs = [[torch.empty_like(out).fill_(3.0) for _ in range(5)] for _ in streams]
    torch.cuda.synchronize()
    for i in range(5):
        for s, o in zip(streams, outs):
            call(o[i], s.cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(x, out) for o in outs for x in o)


def test_verify_step_in_a_cuda_graph():
    """Norm and rotation, cache write and attention captured once and replayed with new device lengths."""
    T, HQ, hk, D, cap = 8, 8, 2, 128, 600
    c = random_cache("q8_0", 1, hk, cap, D, 23)
    qkv = torch.randn(T, (HQ + 2 * hk) * D, device="cuda", generator=gen(24))
    row = qkv.shape[1]
    q, k, v = qkv[:, :HQ * D], qkv[:, HQ * D:(HQ + hk) * D], qkv[:, (HQ + hk) * D:]
    w, table = torch.ones(D, device="cuda"), rope_table(cap, D)
    qo, ko, out = torch.empty(T, HQ * D, device="cuda"), torch.empty(T, hk * D, device="cuda"), \
        torch.empty(T, HQ * D, device="cuda")
    hl, pos = torch.zeros(1, device="cuda", dtype=torch.int32), torch.zeros(T, device="cuda", dtype=torch.int32)

    def step():
        st = torch.cuda.current_stream().cuda_stream
        qk_norm_rope(q.data_ptr(), k.data_ptr(), qo.data_ptr(), ko.data_ptr(), _lib.ACT_F32, T, HQ, hk, D,
                     table.data_ptr(), cap, pos.data_ptr(), w.data_ptr(), w.data_ptr(), q_stride=row, k_stride=row,
                     stream=st)
        kv_cache_write(c.view, ko.data_ptr(), v.data_ptr(), _lib.ACT_F32, T, pos.data_ptr(), v_stride=row, stream=st)
        tree_attention(c.view, qo.data_ptr(), out.data_ptr(), _lib.ACT_F32, 1, T, HQ, hl.data_ptr(), stream=st)

    def at(n):
        hl.fill_(n)
        pos.copy_(torch.arange(n, n + T, device="cuda", dtype=torch.int32))

    at(100)
    step()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for n in (0, 37, 590):
        at(n)
        g.replay()
        torch.cuda.synchronize()
        got = out.clone()
        ref, sabs, vmax = attention_ref(c, qo, 1, T, HQ, [n], [T], None, D ** -0.5)
        assert ((got.double() - ref).abs() <= attention_tolerance("f32", ref, sabs, vmax, cap, D)).all()
        step()
        assert torch.equal(out, got)
    assert verify_error_word() == 0


@pytest.mark.parametrize("T,HQ", [(1, 4), (3, 4), (40, 8)])
def test_tree_lengths_written_just_before(T, HQ):
    """Lengths, queries and cache rows that the kernels right before in the stream write: call after call with no
    wait between them, each with its own history."""
    hk, D, cap = 2, 128, 2000
    c = random_cache("q8_0", 1, hk, cap, D, 30)
    q = torch.randn(T, HQ * D, device="cuda", generator=gen(31)).half()
    hists = [int(x) for x in np.random.RandomState(32).randint(0, cap - T + 1, size=40)]
    want = [run_tree(c, "f16", 1, T, HQ, [h], None, None, 0, q=q)[1] for h in hists]
    hl = torch.zeros(1, device="cuda", dtype=torch.int32)
    q2, outs = torch.zeros_like(q), [torch.empty_like(q) for _ in hists]
    st = torch.cuda.current_stream().cuda_stream
    for h, o in zip(hists, outs):
        q2.copy_(q)
        hl.fill_(h)
        tree_attention(c.view, q2.data_ptr(), o.data_ptr(), _lib.ACT_F16, 1, T, HQ, hl.data_ptr(), stream=st)
        q2.zero_()
        hl.fill_(-1)
    torch.cuda.synchronize()
    for h, o, w in zip(hists, outs, want):
        assert torch.equal(o, w), h
    assert verify_error_word() == 0


def test_example_verifies_drafts():
    """examples/verify_drafts.py: projection, norm and rotation, cache and attention as they are used together."""
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "verify_drafts.py")
    spec = importlib.util.spec_from_file_location("verify_drafts", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    # the same values in another order: f32 sums of some 60 terms, far below the 1e-5 the example allows itself
    assert m.main() <= 1e-5
