"""rf_i8_matmul against the exact product in 64 bits.

The sum is exact; then y goes through the sum's conversion to f32 and two products (three roundings, each half a
unit: 2^-24 of the value), the bias's addition (2^-24 of the result), and one rounding to the output's type.
"""
import pytest

from ramforge_b200 import _lib, i8_matmul, quantize_i8, verify_error_word

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

ACT = {"f32": (_lib.ACT_F32, torch.float32), "f16": (_lib.ACT_F16, torch.float16),
       "bf16": (_lib.ACT_BF16, torch.bfloat16)}


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def codes(g, rows, k, pad=None, low=-128):
    """int8 rows at a pitch of whole 16-byte pieces; what lies between the rows is not zero."""
    pitch = k + (-k) % 16 + (0 if pad is None else pad)
    return torch.randint(low, 128, (rows, pitch), device="cuda", generator=g, dtype=torch.int8)[:, :k]


def close(y, x, sx, w, sw, bias, dtype):
    acc = x.double() @ w.double().T
    part = acc * sx.double()[:, None] * sw.double()
    ref = part if bias is None else part + bias.double()
    tol = 3.01 * 2.0 ** -24 * part.abs() + 2.0 ** -24 * ref.abs() + torch.finfo(y.dtype).eps / 2 * 1.001 * ref.abs()
    tol = tol + {"f32": 1e-44, "f16": 2.0 ** -25, "bf16": 1e-40}[dtype]
    err = (y.double() - ref).abs()
    assert (err <= tol).all(), ((err - tol).max().item(), (err > tol).nonzero()[:3].tolist())


def product(x, sx, w, sw, dtype, bias=None, y=None, stream=0):
    t, n = x.shape[0], w.shape[0]
    if y is None:
        y = torch.full((t, n), float("nan"), device="cuda", dtype=ACT[dtype][1])
    i8_matmul(x.data_ptr(), sx.data_ptr(), w.data_ptr(), sw.data_ptr(), y.data_ptr(), ACT[dtype][0], t, n, x.shape[1],
              x_stride=x.stride(0), w_stride=w.stride(0), y_stride=y.stride(0),
              bias_ptr=0 if bias is None else bias.data_ptr(), stream=stream)
    return y


SHAPES = [(1, 1, 1), (1, 6144, 4096), (2, 130, 16), (3, 127, 17), (7, 1000, 4096), (8, 128, 128), (9, 129, 127),
          (15, 4096, 4096), (16, 256, 129), (17, 4096, 14336), (31, 300, 1000), (32, 512, 512), (33, 65, 2048),
          (48, 1000, 640), (64, 4096, 4096), (65, 28672, 512), (100, 333, 333), (128, 4096, 4096), (129, 384, 4096),
          (200, 5000, 96), (255, 130, 4096), (256, 2048, 2048), (257, 4097, 1023), (333, 4096, 4096), (400, 1, 100),
          (513, 700, 65536), (600, 6144, 4096), (1000, 5555, 777), (2048, 4096, 1024), (2049, 14336, 272),
          (4096, 4096, 64), (3, 128256, 512), (1, 64, 65536), (16, 40, 65536),
          (130, 20000, 300), (257, 10001, 333), (384, 12800, 128), (145, 37900, 1000), (4000, 300, 64), (9000, 200, 50)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("t,n,k", SHAPES)
def test_shapes(t, n, k, dtype):
    g = gen(t * 7 + n * 3 + k)
    x, w = codes(g, t, k), codes(g, n, k)
    sx = 0.001 + 0.001 * torch.rand(t, device="cuda", generator=g)
    sw = 0.01 / k + 0.01 / k * torch.rand(n, device="cuda", generator=g)
    bias = torch.randn(n, device="cuda", generator=g) if (t + n) % 2 else None
    close(product(x, sx, w, sw, dtype, bias), x, sx, w, sw, bias, dtype)
    assert verify_error_word() == 0


@pytest.mark.parametrize("t,n,k", [(1, 300, 500), (12, 300, 500), (300, 300, 500), (700, 9000, 500)])
@pytest.mark.parametrize("pad", [0, 16, 48])
def test_strides(t, n, k, pad):
    """Slices of wider buffers: rows of y between others' columns stay as they are, one element off alignment too."""
    g = gen(t + n + pad)
    x, w = codes(g, t, k, pad), codes(g, n, k, pad)
    sx, sw = torch.rand(t, device="cuda", generator=g), torch.rand(n, device="cuda", generator=g)
    for dtype, skip in (("f32", 0), ("f32", 3), ("bf16", 8), ("f16", 1)):
        wide = torch.full((t, n + 2 * pad + skip), 3.0, device="cuda", dtype=ACT[dtype][1])
        y = wide[:, skip:skip + n]
        sy = sw / k
        product(x, sx, w, sy, dtype, y=y)
        close(y, x, sx, w, sy, None, dtype)
        assert (wide[:, :skip] == 3).all() and (wide[:, skip + n:] == 3).all()


@pytest.mark.parametrize("t", [1, 5, 40, 300])
def test_largest_sums(t):
    """All codes -128 over the longest rows: 2^30, and every partial sum exact."""
    k, n = 65536, 150
    x = torch.full((t, k), -128, device="cuda", dtype=torch.int8)
    w = x.new_full((n, k), -128)
    w[1] = 127
    one_t, one_n = torch.ones(t, device="cuda"), torch.ones(n, device="cuda")
    y = product(x, one_t, w, one_n, "f32")
    assert (y[:, 0] == 2.0 ** 30).all() and (y[:, 1] == -float(128 * 127 * k)).all() and (y[:, 2:] == 2.0 ** 30).all()


@pytest.mark.parametrize("t", [1, 3, 20, 300])
def test_rows_that_are_not_finite(t):
    """A NaN scale makes its token's or channel's results NaN, and no others."""
    g = gen(t)
    x, w = codes(g, t, 256), codes(g, 200, 256)
    sx, sw = torch.rand(t, device="cuda", generator=g), torch.rand(200, device="cuda", generator=g)
    sx[t // 2] = float("nan")
    sw[77] = float("nan")
    y = product(x, sx, w, sw, "bf16")
    bad = torch.zeros(t, 200, device="cuda", dtype=torch.bool)
    bad[t // 2], bad[:, 77] = True, True
    assert torch.equal(y.isnan(), bad)


def test_a_token_does_not_depend_on_the_batch():
    """Whole-number sums: a token alone, among few and among many has the same bits."""
    g = gen(8)
    x, w = codes(g, 700, 4096, low=-127), codes(g, 4096, 4096, low=-127)
    sx, sw = torch.rand(700, device="cuda", generator=g), torch.rand(4096, device="cuda", generator=g) / 4096
    bias = torch.randn(4096, device="cuda", generator=g)
    for dtype, b in (("bf16", None), ("f32", None), ("f32", bias)):
        y = product(x, sx, w, sw, dtype, b)
        for at, m in ((0, 1), (5, 12), (3, 64), (100, 100), (0, 300), (690, 10)):
            assert torch.equal(product(x[at:at + m], sx[at:], w, sw, dtype, b), y[at:at + m]), (dtype, m)
        few = product(x[:3, :1024], sx, w[:, :1024], sw, dtype, b)  # small enough for the kernel of few tokens
        assert torch.equal(few, product(x[:200, :1024], sx, w[:, :1024], sw, dtype, b)[:3])


def test_quantised_on_the_stream_and_replayed():
    """quantize_i8 of both operands and the product in one captured graph: new data at each replay; then the same
    calls on two streams at once."""
    t, n, k = 40, 4096, 4096
    g = gen(4)
    x, w = torch.zeros(t, k, device="cuda"), torch.zeros(n, k, device="cuda")
    xq, wq = torch.empty(t, k, device="cuda", dtype=torch.int8), torch.empty(n, k, device="cuda", dtype=torch.int8)
    sx, sw = torch.empty(t, device="cuda"), torch.empty(n, device="cuda")
    y = torch.empty(t, n, device="cuda")

    def calls(st):
        quantize_i8(w.data_ptr(), wq.data_ptr(), sw.data_ptr(), _lib.ACT_F32, n, k, stream=st)
        quantize_i8(x.data_ptr(), xq.data_ptr(), sx.data_ptr(), _lib.ACT_F32, t, k, stream=st)
        product(xq, sx, wq, sw, "f32", y=y, stream=st)

    calls(torch.cuda.current_stream().cuda_stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        calls(torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        x.copy_(torch.randn(t, k, device="cuda", generator=g))
        w.copy_(torch.randn(n, k, device="cuda", generator=g))
        y.fill_(float("nan"))
        graph.replay()
        close(y, xq, sx, wq, sw, None, "f32")
        ref = x.double() @ w.double().T
        # a code is off by at most half a step of max / 127: for normal numbers about 2 % of the result's size
        assert (y.double() - ref).norm() < 0.03 * ref.norm()
    outs, streams = [torch.full((t, n), float("nan"), device="cuda") for _ in range(4)], [torch.cuda.Stream() for _ in range(4)]
    torch.cuda.synchronize()
    for _ in range(5):
        for o, s in zip(outs, streams):
            product(xq, sx, wq, sw, "f32", y=o, stream=s.cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(o, y) for o in outs)
    assert verify_error_word() == 0


@pytest.mark.parametrize("t", [3, 30, 200])
def test_products_of_rows_that_the_call_before_writes(t):
    """Each product's rows are the quantised results of the one before, with no wait between the calls."""
    n = 2048
    g = gen(t + 50)
    w = codes(g, n, n, low=-127)
    sw = torch.full((n,), 1.0 / (73 * n ** 0.5), device="cuda")
    x = torch.randn(t, n, device="cuda", generator=g)

    def chain(wait):
        y, outs = x.clone(), []
        for _ in range(12):
            q, s = torch.empty(t, n, device="cuda", dtype=torch.int8), torch.empty(t, device="cuda")
            new = torch.empty(t, n, device="cuda")
            quantize_i8(y.data_ptr(), q.data_ptr(), s.data_ptr(), _lib.ACT_F32, t, n)
            if wait:
                torch.cuda.synchronize()
            product(q, s, w, sw, "f32", y=new)
            if wait:
                torch.cuda.synchronize()
            outs.append(new)
            y = new
        torch.cuda.synchronize()
        return outs

    want = chain(True)
    for _ in range(5):
        for a, b in zip(chain(False), want):
            assert torch.equal(a, b)
