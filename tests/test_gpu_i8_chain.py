"""Norm weights that the call before writes: dequantize_i8 gives f32 rows, and one of them may be the next norm's weights."""
import pytest

from ramforge_b200 import _lib, dequantize_i8, norm_i8

from .test_gpu_i8_rows import Codes, gen, torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,cols,pad", [(600, 4096, 0), (1200, 512, 0), (1200, 1001, 7), (600, 2049, 7), (1200, 333, 0),
                                           (40, 4096, 0)])
def test_weights_that_the_call_before_writes(rows, cols, pad):
    """A norm reads the weights, the next call writes them anew, another norm reads them; no wait between."""
    g = gen(rows + cols)
    x = torch.randn(rows, cols, device="cuda", generator=g)
    few = torch.randn(100, cols, device="cuda", generator=g)
    w, one = torch.ones(cols, device="cuda"), torch.full((1,), 0.01, device="cuda")
    seen = [torch.randint(-127, 128, (1, cols), device="cuda", generator=g, dtype=torch.int8) for _ in range(4)]
    before, scratch = Codes(100, cols, pad=3), torch.randn(1 << 24, device="cuda")

    def calls(i, out, wait):
        for fn in (lambda: norm_i8(few.data_ptr(), w.data_ptr(), 1e-5, before.q.data_ptr(), before.scale.data_ptr(),
                                   _lib.ACT_F32, 100, cols, q_stride=before.q.stride(0)),
                   lambda: dequantize_i8(seen[i % 4].data_ptr(), one.data_ptr(), w.data_ptr(), _lib.ACT_F32, 1, cols),
                   lambda: norm_i8(x.data_ptr(), w.data_ptr(), 1e-5, out.q.data_ptr(), out.scale.data_ptr(),
                                   _lib.ACT_F32, rows, cols, q_stride=out.q.stride(0))):
            fn()
            if wait:
                torch.cuda.synchronize()

    want, got = [Codes(rows, cols, pad=pad) for _ in seen], [Codes(rows, cols, pad=pad) for _ in range(24)]
    for i, out in enumerate(want):
        calls(i, out, True)
    assert not torch.equal(want[0].q, want[1].q)
    torch.cuda.synchronize()
    for i, out in enumerate(got):
        scratch.mul_(1.0)  # the calls behind it are queued up when it ends
        calls(i, out, False)
    torch.cuda.synchronize()
    for i, out in enumerate(got):
        assert torch.equal(out.q, want[i % 4].q) and torch.equal(out.scale, want[i % 4].scale), i
