"""rf_tree_attention over caches that hold values which are not finite, on every kernel shape: up to 8 and up to 16
query rows a KV head, and the tcgen05 kernel with one and two row tiles, at both head dimensions.

What a token sees makes its output not finite in the dimensions concerned; what it does not see leaves it as if the
value were another.  Outputs that stay finite are held to the bounds of attention_tolerance with the largest finite
|v| that they can meet.
"""
import numpy as np
import pytest

from ramforge_b200 import verify_error_word

from .test_gpu_verify import attention_ref, attention_tolerance, random_cache, run_tree, torch

pytestmark = pytest.mark.gpu

# tokens, query heads a KV head: 1, 4, 8, 12, 16, 20, 160 and 40 * 7 query rows a KV head
SHAPES = [(1, 1), (4, 1), (2, 4), (3, 4), (4, 4), (5, 4), (40, 4), (40, 7)]


def bad_block(c, which, h, p, d, value):
    """Element (head h, position p, dimension d) of the first sequence becomes `value` (infinite or NaN): the element
    itself, or its block's scale.  Returns the dimensions concerned."""
    x, s = (c.k, c.ks) if which == "k" else (c.v, c.vs)
    if s is None:
        x[0, h, p, d] = value
        return [d]
    s[0, h, p, d // 32] = value
    codes = x[0, h, p, d // 32 * 32:d // 32 * 32 + 32]
    codes[codes == 0] = 1  # 0 * infinity
    return list(range(d // 32 * 32, d // 32 * 32 + 32))


def check(out, ref, dtype, sabs, vmax, cap, D, spoilt):
    """Outputs that `spoilt` [tokens][heads][D] marks are not finite, the others are finite and near."""
    o, r = out.reshape(spoilt.shape), ref.reshape(spoilt.shape)
    assert not torch.isfinite(o[spoilt]).any()
    tol = attention_tolerance(dtype, r, sabs, vmax, cap, D)
    assert ((o.double() - r).abs() <= tol)[~spoilt].all()


@pytest.mark.parametrize("kind", ["q8_0", "f16"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T,G", SHAPES)
def test_history_values_reach_every_token(T, G, D, dtype, kind):
    """A V value of the history that is not finite, at the first and the last position and around the edges of the
    steps and tiles in which drafts lie, too."""
    hk = 2
    for hist in (1, 5, 37, 300):
        c = random_cache(kind, 1, hk, hist + T + 2, D, hist)
        vis = np.tril(np.ones((1, T, T), bool))
        v0, s0 = c.v.clone(), None if c.vs is None else c.vs.clone()
        q, _ = run_tree(c, dtype, 1, T, hk * G, [hist], None, vis, 5)
        ref, sabs, vmax = attention_ref(c, q, 1, T, hk * G, [hist], [T], vis, D ** -0.5)
        for p in sorted({0, hist // 2, max(hist - 17, 0), max(hist - 4, 0), hist - 1}):
            for value in (float("inf"), float("nan")):
                dims = bad_block(c, "v", 1, p, D - 7, value)
                _, out = run_tree(c, dtype, 1, T, hk * G, [hist], None, vis, 5)
                spoilt = torch.zeros(T, hk * G, D, dtype=torch.bool, device="cuda")
                spoilt[:, G:, dims] = True
                check(out, ref, dtype, sabs, vmax, hist + T, D, spoilt)
                if value != value:
                    assert out.reshape(spoilt.shape)[spoilt].isnan().all()
                c.v.copy_(v0)
                if s0 is not None:
                    c.vs.copy_(s0)
    assert verify_error_word() == 0


@pytest.mark.parametrize("kind", ["q8_0", "f16"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T,G", [s for s in SHAPES if s[0] > 1])
def test_draft_values_reach_those_that_see_them(T, G, D, dtype, kind):
    """One element (f16) or one block (Q8_0) of a draft's V row, seen by its own token alone."""
    hk, j = 2, 1
    for hist in (0, 3, 131):
        for value in (float("inf"), -float("inf"), float("nan")):
            c = random_cache(kind, 1, hk, hist + T + 2, D, hist + 1)
            vis = np.tril(np.ones((1, T, T), bool))
            vis[0, :, j] = False
            vis[0, j, j] = True
            q, _ = run_tree(c, dtype, 1, T, hk * G, [hist], None, vis, 6)
            ref, sabs, vmax = attention_ref(c, q, 1, T, hk * G, [hist], [T], vis, D ** -0.5)
            dims = bad_block(c, "v", 0, hist + j, 40, value)
            _, out = run_tree(c, dtype, 1, T, hk * G, [hist], None, vis, 6)
            spoilt = torch.zeros(T, hk * G, D, dtype=torch.bool, device="cuda")
            spoilt[j, :G, dims] = True
            check(out, ref, dtype, sabs, vmax, hist + T, D, spoilt)
    assert verify_error_word() == 0


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T,G", [s for s in SHAPES if s[0] > 1])
@pytest.mark.parametrize("code,scale", [(127, 600.0), (-127, 600.0), (-128, 512.0), (-128, 515.5), (126, -521.0)])
def test_finite_scales_whose_products_overflow(code, scale, D, dtype, T, G):
    """A finite Q8_0 scale whose product with one code leaves f16: that element alone is infinite, and reaches only
    the token that sees it.  The codes go down to -128, which a caller's planes may hold."""
    hk, j, d = 2, 1, 37
    sign = 1.0 if code * scale > 0 else -1.0
    assert abs(code * scale) >= 65520  # rounds to infinity
    for hist in (0, 3, 131):
        c = random_cache("q8_0", 1, hk, hist + T + 2, D, hist + 2)
        vis = np.tril(np.ones((1, T, T), bool))
        vis[0, :, j] = False
        vis[0, j, j] = True
        c.v[0, :, hist + j].clamp_(-5, 5)
        c.v[0, 0, hist + j, d] = 0
        c.vs[0, 0, hist + j, d // 32] = scale
        q, _ = run_tree(c, dtype, 1, T, hk * G, [hist], None, vis, 7)
        ref, sabs, vmax = attention_ref(c, q, 1, T, hk * G, [hist], [T], vis, D ** -0.5)
        c.v[0, 0, hist + j, d] = code
        _, out = run_tree(c, dtype, 1, T, hk * G, [hist], None, vis, 7)
        spoilt = torch.zeros(T, hk * G, D, dtype=torch.bool, device="cuda")
        spoilt[j, :G, d] = True
        rest = torch.arange(T, device="cuda") != j  # they never meet the large values
        tol = torch.where(rest[:, None, None], 0.0, 1.0).expand(T, hk * G, D)
        r, o = ref.reshape(T, hk * G, D), out.reshape(T, hk * G, D)
        low = attention_tolerance(dtype, r, sabs, 6.0, hist + T, D)
        high = attention_tolerance(dtype, r, sabs, vmax, hist + T, D)
        tol = torch.where(tol > 0, high, low)
        assert ((o.double() - r).abs() <= tol)[~spoilt].all()
        assert (o[spoilt] == sign * float("inf")).all()
    assert verify_error_word() == 0
