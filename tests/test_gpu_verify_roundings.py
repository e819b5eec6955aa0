"""rf_tree_attention with 16-bit activations rounds each weight to f16 once (attention_tolerance: 2^-11 of the weights,
times the largest |v|), also where the softmax's reference is raised between two pieces of a tile."""
import math

import pytest

from ramforge_b200 import verify_error_word

from .test_gpu_verify import Cache, attention_ref, attention_tolerance, run_tree, torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T,G", [(5, 4), (4, 4), (40, 4)])
def test_weights_are_rounded_once(T, G, D, dtype):
    """One row's scores jump by 20 (in base 2) after 32 keys, so that all rows next to it are rescaled there; in those,
    the first keys' weights and the factor are just below the middle of two f16, and so would be their product's
    roundings: 31 keys of v = 1 weigh nearly the same as two of v = -1, and the difference shows what was lost."""
    hist = 128
    c = Cache("f16", 1, 1, hist + T, D)
    low = 1 - math.log2(1 + 16.47 / 1024)   # weights of 64 (1 + 16.47 / 1024) under the reference of key 0
    rise = 3 - math.log2(1 + 32.47 / 1024)  # a factor of (1 + 32.47 / 1024) / 8
    s = torch.full((hist + T,), -30.0, dtype=torch.float64)
    s[0], s[1:32], s[32:34] = 0.0, -low, rise
    coarse = s.half()
    c.k[0, 0, :, 0] = coarse.cuda()
    c.k[0, 0, :, 1] = (s - coarse.double()).half().cuda()
    c.k[0, 0, 32:hist, 2] = 20.0
    c.v[0, 0, 1:32] = 1.0
    c.v[0, 0, 32:34] = -1.0
    q = torch.zeros(T, G, D, device="cuda")
    q[..., 0] = q[..., 1] = 1.0
    q[0, 0] = 0.0
    q[0, 0, 2] = 1.0
    q, out = run_tree(c, dtype, 1, T, G, [hist], None, None, 0, scale=math.log(2), q=q.reshape(T, G * D))
    ref, sabs, vmax = attention_ref(c, q, 1, T, G, [hist], [T], None, math.log(2))
    err = (out.double() - ref).abs()
    tol = attention_tolerance(dtype, ref, sabs, vmax, hist + T, D)
    assert (err <= tol).all(), (err / tol).max().item()
    assert verify_error_word() == 0
