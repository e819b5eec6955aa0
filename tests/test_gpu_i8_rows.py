"""8-bit rows (rf_norm_i8, rf_swiglu_i8, rf_quantize_i8, rf_dequantize_i8) against the format's definition.

The format fixes every rounding of the norm's and the plain rows' codes and scales, so those are compared for
equality (the mean of squares is taken in 64 bits on both sides: the reciprocal root's 32 bits do not show its
order).  SwiGLU's exponential and quotient are exact to a few units: with g of up to 2^5 the kernel's y is off by at
most (|g| + 12) 2^-24 |y| (the exponent's rounding |g| 2^-24, two units of ex2, the sum, two of the quotient, the
product), its scale by one rounding more, and a code lies within half a step and 127 * 2^-23 steps of y / scale.
"""
import numpy as np
import pytest

from ramforge_b200 import _lib, dequantize_i8, norm_i8, quantize_i8, swiglu_i8

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

ACT = {"f32": (_lib.ACT_F32, torch.float32), "f16": (_lib.ACT_F16, torch.float16),
       "bf16": (_lib.ACT_BF16, torch.bfloat16)}
F = np.float32


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rows_of(y):
    """(codes, scales) of f32 rows by the definition."""
    with np.errstate(all="ignore"):
        y = y.astype(F)
        top = np.abs(y).max(-1)
        scale = top / F(127)
        scale[scale < F(2.0 ** -126)] = 0
        inv = np.where(scale > 0, F(1) / scale, F(0))
        code = np.clip(np.rint(y * inv[:, None]), -127, 127)
        wild = ~np.isfinite(y).all(-1)
        code[wild], scale[wild] = 0, np.nan
        return code.astype(np.int8), scale.astype(F)


def norm_rows(x, add, w, eps):
    with np.errstate(all="ignore"):
        s = x if add is None else x + add
        wide = s.astype(np.float64)
        r = (1 / np.sqrt((wide * wide).sum(-1, keepdims=True) / s.shape[-1] + np.float64(F(eps)))).astype(F)
        return s, (s if w is None else s * w) * r


def f32(x):
    return x.float().cpu().numpy()


class Codes:
    def __init__(self, rows, cols, pad=0, offset=0):
        self.buf = torch.full((offset + rows * (cols + pad),), 99, device="cuda", dtype=torch.int8)
        self.q = self.buf[offset:].view(rows, cols + pad)
        self.scale = torch.full((rows,), 7.0, device="cuda")
        self.cols = cols

    def same(self, code, scale):
        np.testing.assert_array_equal(self.scale.cpu().numpy(), scale)
        np.testing.assert_array_equal(self.q[:, :self.cols].cpu().numpy(), code)
        assert (self.q[:, self.cols:] == 99).all()


SHAPES = [(1, 1), (1, 7), (3, 8), (2, 33), (5, 64), (17, 255), (4, 256), (1, 4096), (33, 4096), (1000, 4096), (1500, 4095), (700, 1001), (1300, 129), (900, 500), (800, 14336), (9, 4097), (2, 5000),
          (3, 14336), (2, 16384), (2, 16385), (1, 32768), (1, 40001), (2, 65536), (700, 1024), (300, 96)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_norm(rows, cols, dtype):
    code, dt = ACT[dtype]
    g = gen(rows * 31 + cols)
    x = torch.randn(rows, cols, device="cuda", generator=g).to(dt)
    add = (3 * torch.randn(rows, cols, device="cuda", generator=g)).to(dt)
    w = 1 + 0.5 * torch.randn(cols, device="cuda", generator=g)
    total = torch.full_like(x, float("nan"))
    out = Codes(rows, cols, pad=(-cols) % 16)
    norm_i8(x.data_ptr(), w.data_ptr(), 1e-5, out.q.data_ptr(), out.scale.data_ptr(), code, rows, cols,
            add_ptr=add.data_ptr(), sum_ptr=total.data_ptr(), q_stride=out.q.stride(0))
    s, y = norm_rows(f32(x), f32(add), f32(w), 1e-5)
    out.same(*rows_of(y))
    assert torch.equal(total.cpu(), torch.from_numpy(s).to(dt))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_quantize_and_back(rows, cols, dtype):
    code, dt = ACT[dtype]
    x = torch.randn(rows, cols, device="cuda", generator=gen(rows + cols)).to(dt)
    out = Codes(rows, cols)
    quantize_i8(x.data_ptr(), out.q.data_ptr(), out.scale.data_ptr(), code, rows, cols)
    c, s = rows_of(f32(x))
    out.same(c, s)
    for to in ACT:
        values = torch.full((rows, cols), float("nan"), device="cuda", dtype=ACT[to][1])
        dequantize_i8(out.q.data_ptr(), out.scale.data_ptr(), values.data_ptr(), ACT[to][0], rows, cols)
        want = torch.from_numpy(c.astype(F) * s[:, None]).to(ACT[to][1])
        assert torch.equal(values.cpu(), want)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_swiglu(rows, cols, dtype):
    code, dt = ACT[dtype]
    gu = (4 * torch.randn(rows, 2 * cols, device="cuda", generator=gen(rows * 5 + cols))).clamp_(-32, 32).to(dt)
    out = Codes(rows, cols, pad=(-cols) % 16)
    swiglu_i8(gu.data_ptr(), gu.data_ptr() + cols * gu.element_size(), out.q.data_ptr(), out.scale.data_ptr(), code,
              rows, cols, gate_stride=2 * cols, up_stride=2 * cols, q_stride=out.q.stride(0))
    g, u = f32(gu).astype(np.float64)[:, :cols], f32(gu).astype(np.float64)[:, cols:]
    y = g * u / (1 + np.exp(-g))
    slack = (np.abs(g) + 12) * 2.0 ** -24 * np.abs(y) + 1e-37
    scale = out.scale.cpu().numpy().astype(np.float64)[:, None]
    top = np.abs(y).max(-1, keepdims=True)
    assert (np.abs(scale - top / 127) <= (slack.max(-1, keepdims=True) + 2.0 ** -24 * top) / 127 * 1.01).all()
    got = out.q[:, :cols].cpu().numpy() * scale
    assert (np.abs(got - y) <= scale * (0.5 + 127 * 2.0 ** -22) + slack).all()
    assert (out.q[:, cols:] == 99).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("cols", [64, 96, 100])
@pytest.mark.parametrize("offset,pad", [(0, 0), (1, 0), (0, 3), (8, 8), (4, 12)])
def test_strides_and_alignment(offset, pad, cols, dtype):
    """Rows that begin anywhere, sums written over the residual, codes at any byte; what lies between rows stays."""
    code, dt = ACT[dtype]
    rows = 5
    g = gen(offset * 50 + pad * 7 + cols)
    buf = torch.randn(offset + rows * (cols + pad), device="cuda", generator=g).to(dt)
    x = buf[offset:].view(rows, cols + pad)
    res = torch.randn(offset + rows * (cols + pad), device="cuda", generator=g).to(dt)
    add = res[offset:].view(rows, cols + pad)
    before = add.clone()
    wbuf = torch.randn(cols + 1, device="cuda", generator=g)
    w = wbuf[offset % 2:][:cols]
    out = Codes(rows, cols, pad=pad, offset=offset)
    norm_i8(x.data_ptr(), w.data_ptr(), 1e-6, out.q.data_ptr(), out.scale.data_ptr(), code, rows, cols,
            add_ptr=add.data_ptr(), sum_ptr=add.data_ptr(), x_stride=x.stride(0), add_stride=add.stride(0),
            sum_stride=add.stride(0), q_stride=out.q.stride(0))
    s, y = norm_rows(f32(x)[:, :cols], f32(before)[:, :cols], f32(w), 1e-6)
    out.same(*rows_of(y))
    assert torch.equal(add[:, :cols].cpu(), torch.from_numpy(s).to(dt)) and torch.equal(add[:, cols:], before[:, cols:])
    values = torch.full((rows, cols + pad), 5.0, device="cuda", dtype=dt)
    dequantize_i8(out.q.data_ptr(), out.scale.data_ptr(), values.data_ptr(), code, rows, cols,
                  q_stride=out.q.stride(0), out_stride=values.stride(0))
    assert torch.equal(values[:, :cols].cpu(), torch.from_numpy(rows_of(y)[0].astype(F) * rows_of(y)[1][:, None]).to(dt))
    assert (values[:, cols:] == 5).all()
    quantize_i8(x.data_ptr(), out.q.data_ptr(), out.scale.data_ptr(), code, rows, cols, x_stride=x.stride(0),
                q_stride=out.q.stride(0))
    out.same(*rows_of(f32(x)[:, :cols]))


def test_extreme_rows():
    """Zeros, numbers below the least scale, the largest ones, infinities and NaN, each in a row of its own."""
    cols = 200
    x = torch.randn(9, cols, device="cuda", generator=gen(3))
    x[0] = 0
    x[1] *= 1e-40        # subnormal numbers: the scale would be below 2^-126
    x[2] *= 1e-36
    x[3] = 3.0e38
    x[4, 17] = float("inf")
    x[5, 199] = float("nan")
    x[6, 0] = -float("inf")
    x[7] = -3.4e38
    out = Codes(9, cols)
    quantize_i8(x.data_ptr(), out.q.data_ptr(), out.scale.data_ptr(), _lib.ACT_F32, 9, cols)
    out.same(*rows_of(f32(x)))
    assert out.scale[4:7].isnan().all() and (out.scale[:2] == 0).all()
    values = torch.empty(9, cols, device="cuda")
    dequantize_i8(out.q.data_ptr(), out.scale.data_ptr(), values.data_ptr(), _lib.ACT_F32, 9, cols)
    assert values[4:7].isnan().all() and (values[:2] == 0).all()
    for w, eps in ((None, 1e-6), (None, 0.0), (float("inf"), 1e-6), (float("nan"), 1e-6)):
        weight = None if w is None else torch.ones(cols, device="cuda")
        if w is not None:
            weight[5] = w
        norm_i8(x.data_ptr(), 0 if weight is None else weight.data_ptr(), eps, out.q.data_ptr(), out.scale.data_ptr(),
                _lib.ACT_F32, 9, cols)
        out.same(*rows_of(norm_rows(f32(x), None, None if weight is None else f32(weight), eps)[1]))
    g = torch.tensor([[-200.0, 1, 2, 3], [float("inf"), 0, 0, 0], [-float("inf"), 1, 1, 1], [float("nan"), 1, 1, 1],
                      [1, 1, 1, 1]], device="cuda")
    u = torch.ones_like(g)
    u[4, 2] = float("inf")
    small = Codes(5, 4)
    swiglu_i8(g.data_ptr(), u.data_ptr(), small.q.data_ptr(), small.scale.data_ptr(), _lib.ACT_F32, 5, 4)
    assert small.scale[1:].isnan().all() and (small.q[1:] == 0).all()
    assert small.q[0].tolist()[0] == 0 and small.q[0].tolist()[3] == 127


def test_rows_do_not_depend_on_their_place_and_graphs_replay():
    """A row alone, in a batch, and in a captured graph replayed on new data has the same codes."""
    rows, cols = 37, 4096
    g = gen(11)
    x = torch.randn(rows, cols, device="cuda", generator=g).bfloat16()
    w = torch.randn(cols, device="cuda", generator=g)
    a, b = Codes(rows, cols), Codes(rows, cols)
    norm_i8(x.data_ptr(), w.data_ptr(), 1e-5, a.q.data_ptr(), a.scale.data_ptr(), _lib.ACT_BF16, rows, cols)
    for r in range(rows):
        norm_i8(x[r].data_ptr(), w.data_ptr(), 1e-5, b.q[r].data_ptr(), b.scale[r:].data_ptr(), _lib.ACT_BF16, 1, cols)
    assert torch.equal(a.q, b.q) and torch.equal(a.scale, b.scale)
    held = torch.zeros_like(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        st = torch.cuda.current_stream().cuda_stream
        norm_i8(held.data_ptr(), w.data_ptr(), 1e-5, b.q.data_ptr(), b.scale.data_ptr(), _lib.ACT_BF16, rows, cols,
                stream=st)
    held.copy_(x)
    graph.replay()
    assert torch.equal(a.q, b.q) and torch.equal(a.scale, b.scale)


@pytest.mark.parametrize("rows,cols", [(2000, 4096), (3000, 512), (100, 4096), (1400, 4095)])
def test_rows_that_the_call_before_writes(rows, cols):
    """Values written by dequantize_i8 and read by norm_i8 and quantize_i8 at once, call after call with no wait
    between them: each call begins while the one before it ends."""
    g = gen(rows)
    w = torch.randn(cols, device="cuda", generator=g)
    seen = [(torch.randint(-127, 128, (rows, cols), device="cuda", generator=g, dtype=torch.int8),
             0.001 + torch.rand(rows, device="cuda", generator=g)) for _ in range(4)]
    values, total = torch.empty(rows, cols, device="cuda"), torch.empty(rows, cols, device="cuda")

    def calls(q, scale, out, wait):
        for fn in (lambda: dequantize_i8(q.data_ptr(), scale.data_ptr(), values.data_ptr(), _lib.ACT_F32, rows, cols),
                   lambda: norm_i8(values.data_ptr(), w.data_ptr(), 1e-5, out[0].q.data_ptr(), out[0].scale.data_ptr(),
                                   _lib.ACT_F32, rows, cols, add_ptr=values.data_ptr(), sum_ptr=total.data_ptr()),
                   lambda: quantize_i8(total.data_ptr(), out[1].q.data_ptr(), out[1].scale.data_ptr(), _lib.ACT_F32,
                                       rows, cols)):
            fn()
            if wait:
                torch.cuda.synchronize()

    want = [(Codes(rows, cols), Codes(rows, cols)) for _ in seen]
    for (q, scale), out in zip(seen, want):
        calls(q, scale, out, True)
    got = [(Codes(rows, cols), Codes(rows, cols)) for _ in range(20)]
    torch.cuda.synchronize()
    for i, out in enumerate(got):
        calls(*seen[i % 4], out, False)
    torch.cuda.synchronize()
    for i, out in enumerate(got):
        for a, b in zip(out, want[i % 4]):
            assert torch.equal(a.q, b.q) and torch.equal(a.scale, b.scale), i


def placed(rows, cols, gap, lead, dt, seed):
    """A [rows, cols] view `lead` elements into a buffer, `gap` apart; everything beside the rows is NaN."""
    buf = torch.full((lead + rows * (cols + gap),), float("nan"), device="cuda", dtype=dt)
    view = buf[lead:].view(rows, cols + gap)[:, :cols]
    view.copy_(torch.randn(rows, cols, device="cuda", generator=gen(seed)))
    return buf, view


def beside_is_nan(buf, view):
    mask = torch.ones_like(buf, dtype=torch.bool)
    lead = view.storage_offset()
    mask[lead:].view(view.shape[0], view.stride(0))[:, :view.shape[1]] = False
    return bool(buf[mask].isnan().all())


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("rows,cols,gap,leads", [
    (2500, 601, 0, (0, 0)), (2500, 601, 0, (3, 6)), (1000, 4095, 0, (1, 0)), (1000, 4093, 2, (5, 2)),
    (2600, 522, 1, (2, 7)), (1000, 4096, 4, (4, 0)), (4000, 515, 6, (7, 3)), (950, 4094, 1, (6, 1)), (320, 14335, 0, (1, 2))])
def test_many_rows_at_any_place(rows, cols, gap, leads, in_place, dtype):
    """Rows that begin anywhere within 16 bytes, the two inputs at different places, NaN in all that lies beside them."""
    code, dt = ACT[dtype]
    xb, x = placed(rows, cols, gap, leads[0], dt, rows + cols)
    ab, add = placed(rows, cols, gap, leads[1], dt, rows + cols + 1)
    if in_place:
        tb, total = xb, x
    else:
        tb, total = placed(rows, cols, gap, leads[0], dt, 1)
    w = 1 + 0.5 * torch.randn(cols, device="cuda", generator=gen(cols))
    s, y = norm_rows(f32(x), f32(add), f32(w), 1e-5)
    out = Codes(rows, cols, pad=-cols % 8 + 8)
    norm_i8(x.data_ptr(), w.data_ptr(), 1e-5, out.q.data_ptr(), out.scale.data_ptr(), code, rows, cols,
            add_ptr=add.data_ptr(), sum_ptr=total.data_ptr(), x_stride=x.stride(0), add_stride=add.stride(0),
            sum_stride=total.stride(0), q_stride=out.q.stride(0))
    c, scale = rows_of(y)
    out.same(c, scale)
    assert torch.equal(total.cpu(), torch.from_numpy(s).to(dt))
    assert beside_is_nan(tb, total) and beside_is_nan(ab, add) and beside_is_nan(xb, x)
    for to in ACT:
        vb, values = placed(rows, cols, gap, leads[1], ACT[to][1], 2)
        dequantize_i8(out.q.data_ptr(), out.scale.data_ptr(), values.data_ptr(), ACT[to][0], rows, cols,
                      q_stride=out.q.stride(0), out_stride=values.stride(0))
        assert torch.equal(values.cpu(), torch.from_numpy(c.astype(F) * scale[:, None]).to(ACT[to][1]))
        assert beside_is_nan(vb, values)
    # no second input, no weights
    norm_i8(add.data_ptr(), 0, 1e-6, out.q.data_ptr(), out.scale.data_ptr(), code, rows, cols, x_stride=add.stride(0),
            q_stride=out.q.stride(0))
    out.same(*rows_of(norm_rows(f32(add), None, None, 1e-6)[1]))
    quantize_i8(add.data_ptr(), out.q.data_ptr(), out.scale.data_ptr(), code, rows, cols, x_stride=add.stride(0),
                q_stride=out.q.stride(0))
    out.same(*rows_of(f32(add)))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols", [(2500, 601), (1000, 4095), (330, 14335), (4000, 515)])
def test_many_rows_are_as_alone(rows, cols, dtype):
    """A row's codes are the same in a call of many rows and in one of its own, wild rows among them."""
    code, dt = ACT[dtype]
    gu = torch.randn(rows, 2 * cols, device="cuda", generator=gen(rows)).to(dt)
    gu[7, 3], gu[rows - 1, cols - 1], gu[11, 2 * cols - 1] = float("nan"), float("inf"), float("-inf")
    gu[12] = 0
    es, wide = gu.element_size(), -(-cols // 8) * 8
    many, one = Codes(rows, cols, pad=wide - cols), Codes(rows, cols, pad=wide - cols)
    swiglu_i8(gu.data_ptr(), gu.data_ptr() + cols * es, many.q.data_ptr(), many.scale.data_ptr(), code, rows, cols,
              gate_stride=2 * cols, up_stride=2 * cols, q_stride=wide)
    looked = [0, 1, 7, 11, 12, rows // 2, rows - 2, rows - 1]
    for r in looked:
        at = gu.data_ptr() + 2 * r * cols * es
        swiglu_i8(at, at + cols * es, one.q[r].data_ptr(), one.scale[r:].data_ptr(), code, 1, cols)
    assert torch.equal(many.q[looked], one.q[looked]) and (many.q[:, cols:] == 99).all()
    assert torch.equal(many.scale[looked].view(torch.int32), one.scale[looked].view(torch.int32))
    assert many.scale[[7, 11, rows - 1]].isnan().all() and not many.q[[7, 11, 12, rows - 1], :cols].any()


@pytest.mark.parametrize("rows,cols", [(1400, 4095), (2500, 601), (700, 1999), (400, 7001)])
def test_rows_at_any_place_that_the_call_before_writes(rows, cols):
    """The same chain with codes in whole eights and rows of values at any place, and SwiGLU of neighbours."""
    g = gen(rows)
    wide = -(-cols // 8) * 8
    w = torch.randn(cols, device="cuda", generator=g)
    seen = [(torch.randint(-127, 128, (rows, wide), device="cuda", generator=g, dtype=torch.int8),
             0.001 + torch.rand(rows, device="cuda", generator=g)) for _ in range(4)]
    values, total = torch.empty(rows, cols, device="cuda"), torch.empty(rows, cols, device="cuda")

    def calls(q, scale, out, wait):
        for fn in (lambda: dequantize_i8(q.data_ptr(), scale.data_ptr(), values.data_ptr(), _lib.ACT_F32, rows, cols,
                                         q_stride=wide),
                   lambda: norm_i8(values.data_ptr(), w.data_ptr(), 1e-5, out[0].q.data_ptr(), out[0].scale.data_ptr(),
                                   _lib.ACT_F32, rows, cols, add_ptr=values.data_ptr(), sum_ptr=total.data_ptr(),
                                   q_stride=wide),
                   lambda: swiglu_i8(total.data_ptr(), values.data_ptr(), out[1].q.data_ptr(),
                                     out[1].scale.data_ptr(), _lib.ACT_F32, rows, cols, q_stride=wide)):
            fn()
            if wait:
                torch.cuda.synchronize()

    def outputs():
        return Codes(rows, cols, pad=wide - cols), Codes(rows, cols, pad=wide - cols)

    want = [outputs() for _ in seen]
    for (q, scale), out in zip(seen, want):
        calls(q, scale, out, True)
    got = [outputs() for _ in range(20)]
    torch.cuda.synchronize()
    for i, out in enumerate(got):
        calls(*seen[i % 4], out, False)
    torch.cuda.synchronize()
    for i, out in enumerate(got):
        for a, b in zip(out, want[i % 4]):
            assert torch.equal(a.q, b.q) and torch.equal(a.scale, b.scale), i


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols", [(700, 8200), (900, 11008), (620, 14336), (640, 16384), (597, 9216)])
def test_many_long_rows_are_as_alone(rows, cols, dtype):
    """Long rows, of which an SM has few at a time: codes and scales as in calls of one row, for SwiGLU and plain rows."""
    code, dt = ACT[dtype]
    x = torch.randn(rows, cols, device="cuda", generator=gen(rows)).to(dt)
    up = torch.randn(rows, cols, device="cuda", generator=gen(cols)).to(dt)
    up[5, cols - 1], x[rows - 3, 0], x[9] = float("inf"), float("nan"), 0
    gated, plain, one = Codes(rows, cols), Codes(rows, cols), Codes(rows, cols)
    swiglu_i8(x.data_ptr(), up.data_ptr(), gated.q.data_ptr(), gated.scale.data_ptr(), code, rows, cols)
    quantize_i8(x.data_ptr(), plain.q.data_ptr(), plain.scale.data_ptr(), code, rows, cols)
    plain.same(*rows_of(f32(x)))
    for r in range(rows):
        swiglu_i8(x[r].data_ptr(), up[r].data_ptr(), one.q[r].data_ptr(), one.scale[r:].data_ptr(), code, 1, cols)
    assert torch.equal(gated.q, one.q)
    assert torch.equal(gated.scale.view(torch.int32), one.scale.view(torch.int32))
    assert gated.scale[[5, rows - 3]].isnan().all() and not gated.q[[5, 9, rows - 3]].any()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [295, 296, 591, 592, 593])
@pytest.mark.parametrize("cols,lead", [(64, 3), (65, 0), (100, 1), (301, 5), (513, 2), (1023, 7), (1025, 1), (2801, 3)])
def test_counts_at_which_the_kernel_changes(rows, cols, lead, dtype):
    code, dt = ACT[dtype]
    xb, x = placed(rows, cols, 0, lead, dt, rows + cols)
    ab, add = placed(rows, cols, 1, 0, dt, rows + cols + 1)
    out, out2 = Codes(rows, cols, pad=-cols % 8 + 8), Codes(rows, cols, pad=-cols % 8 + 8)
    norm_i8(x.data_ptr(), 0, 1e-5, out.q.data_ptr(), out.scale.data_ptr(), code, rows, cols, add_ptr=add.data_ptr(),
            x_stride=x.stride(0), add_stride=add.stride(0), q_stride=out.q.stride(0))
    quantize_i8(add.data_ptr(), out2.q.data_ptr(), out2.scale.data_ptr(), code, rows, cols, x_stride=add.stride(0),
                q_stride=out2.q.stride(0))
    out.same(*rows_of(norm_rows(f32(x), f32(add), None, 1e-5)[1]))
    out2.same(*rows_of(f32(add)))
    assert beside_is_nan(xb, x) and beside_is_nan(ab, add)
