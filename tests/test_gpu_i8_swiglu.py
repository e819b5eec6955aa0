"""SwiGLU over the whole range of its gate, and at the counts and widths at which one kernel takes over from another.

A row of one column has y itself in its scale: |y| / 127 rounded.  y's bound, in units of 2^-24 of its size: the
exponent's argument g log2(e) is a rounded product with a rounded constant, |g| (1 + 0.22); two units of ex2's last place
are 4, the sum 1, a unit of the quotient's 2, two products 2, the scale's division 1: 1.22 |g| + 10."""
import numpy as np
import pytest

from ramforge_b200 import _lib, swiglu_i8, verify_error_word

from .test_gpu_i8_rows import ACT, Codes, beside_is_nan, f32, gen, placed, torch

pytestmark = pytest.mark.gpu


def one_column(gate, up):
    n = gate.numel()
    q, scale = torch.full((n,), 99, device="cuda", dtype=torch.int8), torch.empty(n, device="cuda")
    swiglu_i8(gate.data_ptr(), up.data_ptr(), q.data_ptr(), scale.data_ptr(), _lib.ACT_F32, n, 1)
    return q.cpu().numpy(), scale.double().cpu().numpy()


@pytest.mark.parametrize("lo,hi", [(1e-4, 1), (1, 8), (8, 32), (32, 60), (60, 87.3)])
@pytest.mark.parametrize("sign", [-1.0, 1.0])
def test_the_whole_range_of_the_gate(sign, lo, hi):
    n = 400000
    g = gen(int(hi))
    gate = sign * torch.exp(torch.empty(n, device="cuda").uniform_(float(np.log(lo)), float(np.log(hi)), generator=g))
    up = (1 + torch.rand(n, device="cuda", generator=g)) * (1e30 if sign < 0 else 1.0)  # y stays a normal number
    q, scale = one_column(gate, up)
    gd, ud = gate.double().cpu().numpy(), up.double().cpu().numpy()
    y = gd * ud / (1 + np.exp(-gd))
    assert (q == np.where(y > 0, 127, -127)).all()
    assert (np.abs(scale * 127 - np.abs(y)) <= (1.25 * np.abs(gd) + 12) * 2.0 ** -24 * np.abs(y)).all()


def test_gates_below_the_range():
    gate = -torch.logspace(np.log10(87.34), 38, 5000, device="cuda")
    q, scale = one_column(gate, torch.full_like(gate, 1e30))
    assert not q.any() and not scale.any()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [295, 296, 591, 592, 593])
@pytest.mark.parametrize("cols,leads", [(256, (0, 0)), (512, (0, 0)), (511, (3, 6)), (513, (1, 2)), (1024, (0, 0)), (1023, (7, 1)),
                                        (2799, (2, 5)), (2801, (5, 0)), (4097, (1, 3)), (4104, (0, 0))])
def test_counts_at_which_the_kernel_changes(rows, cols, leads, dtype):
    """Rows anywhere, gate and up at places of their own, NaN in all that lies beside them: as each row by itself."""
    code, dt = ACT[dtype]
    gb, gate = placed(rows, cols, 0, leads[0], dt, rows + cols)
    ub, up = placed(rows, cols, leads[1], leads[1], dt, rows + cols + 1)
    out, one = Codes(rows, cols, pad=-cols % 8 + 8), Codes(rows, cols, pad=-cols % 8 + 8)
    es = gate.element_size()
    swiglu_i8(gate.data_ptr(), up.data_ptr(), out.q.data_ptr(), out.scale.data_ptr(), code, rows, cols,
              gate_stride=gate.stride(0), up_stride=up.stride(0), q_stride=out.q.stride(0))
    for r in range(rows):
        swiglu_i8(gate.data_ptr() + r * gate.stride(0) * es, up.data_ptr() + r * up.stride(0) * es, one.q[r].data_ptr(),
                  one.scale[r:].data_ptr(), code, 1, cols)
    assert torch.equal(out.q, one.q) and torch.equal(out.scale, one.scale)
    g, u = f32(gate).astype(np.float64), f32(up).astype(np.float64)
    y = g * u / (1 + np.exp(-g))
    top = np.abs(y).max(-1)
    slack = (1.25 * np.abs(g) + 12) * 2.0 ** -24 * np.abs(y)
    scale = out.scale.double().cpu().numpy()
    assert (np.abs(scale * 127 - top) <= slack.max(-1) + 2.0 ** -23 * top).all()
    got = out.q[:, :cols].cpu().numpy() * scale[:, None]
    assert (np.abs(got - y) <= scale[:, None] * (0.5 + 127 * 2.0 ** -22) + slack).all()
    assert beside_is_nan(gb, gate) and beside_is_nan(ub, up) and verify_error_word() == 0
