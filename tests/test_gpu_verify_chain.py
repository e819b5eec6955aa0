"""Verification calls one behind the other with nothing else in the stream, layer after layer through the same
buffers, as a model's layers use them: each kernel begins while the one before it ends, and must see what that wrote
and not what its own buffers held a layer ago.  The same bits as with a wait after every call."""
import pytest

from ramforge_b200 import kv_cache_read, kv_cache_write, qk_norm_rope, tree_attention, verify_error_word

from .test_gpu_verify import ACT, gen, random_cache, rope_table, torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("kind", ["q8_0", "f16"])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("T,HQ,hk,D,hist", [(1, 8, 2, 128, 5), (4, 8, 2, 128, 60), (3, 4, 4, 64, 0), (12, 8, 2, 128, 100),
                                            (40, 16, 2, 128, 30), (7, 32, 8, 128, 3000)])
def test_layers_through_the_same_buffers(T, HQ, hk, D, hist, dtype, kind, graph):
    layers = 24
    code, dt = ACT[dtype]
    g = gen(T + D + hist)
    row = (HQ + 2 * hk) * D
    x = torch.randn(layers, T, row, device="cuda", generator=g).to(dt)
    c = random_cache(kind, 1, hk, hist + T + 1, D, 70)
    w, table = 1 + 0.1 * torch.randn(D, device="cuda", generator=g), rope_table(hist + T + 1, D)
    at = torch.arange(hist, hist + T, device="cuda", dtype=torch.int32)
    hl = torch.tensor([hist], device="cuda", dtype=torch.int32)
    q, k = (torch.zeros(T, n * D, device="cuda", dtype=dt) for n in (HQ, hk))
    kb, vb = (torch.zeros(T, hk * D, device="cuda", dtype=dt) for _ in range(2))
    bufs = (q, k, kb, vb, c.k, c.v) + (() if c.ks is None else (c.ks, c.vs))
    start = [b.clone() for b in bufs]

    def layer(i, out, back, st, wait):
        src = x[i]
        calls = [
            lambda: qk_norm_rope(src.data_ptr(), src[:, HQ * D:].data_ptr(), q.data_ptr(), k.data_ptr(), code, T, HQ, hk,
                                 D, table.data_ptr(), hist + T + 1, at.data_ptr(), w.data_ptr(), w.data_ptr(),
                                 q_stride=row, k_stride=row, stream=st),
            lambda: kv_cache_write(c.view, k.data_ptr(), src[:, (HQ + hk) * D:].data_ptr(), code, T, at.data_ptr(),
                                   v_stride=row, stream=st),
            lambda: tree_attention(c.view, q.data_ptr(), out.data_ptr(), code, 1, T, HQ, hl.data_ptr(), stream=st),
            lambda: kv_cache_read(c.view, kb.data_ptr(), vb.data_ptr(), code, T, at.data_ptr(), stream=st),
            # what was read goes back a place on, and the attention sees the drafts as they then are
            lambda: kv_cache_write(c.view, vb.data_ptr(), kb.data_ptr(), code, T, at.data_ptr(), stream=st),
            lambda: tree_attention(c.view, q.data_ptr(), back.data_ptr(), code, 1, T, HQ, hl.data_ptr(), stream=st)]
        for f in calls:
            f()
            if wait:
                torch.cuda.synchronize()

    def run(wait):
        for b, s in zip(bufs, start):
            b.copy_(s)
        outs = torch.zeros(2, layers, T, HQ * D, device="cuda", dtype=dt)
        torch.cuda.synchronize()
        if wait or not graph:
            st = torch.cuda.current_stream().cuda_stream
            for i in range(layers):
                layer(i, outs[0, i], outs[1, i], st, wait)
        else:
            cg = torch.cuda.CUDAGraph()
            with torch.cuda.graph(cg):
                st = torch.cuda.current_stream().cuda_stream
                for i in range(layers):
                    layer(i, outs[0, i], outs[1, i], st, False)
            cg.replay()
        torch.cuda.synchronize()
        return outs

    want = run(True)
    assert torch.isfinite(want).all() and not torch.equal(want[0, 0], want[0, 1])
    for _ in range(3):
        assert torch.equal(run(False), want)
    assert verify_error_word() == 0


# ---- index words that the kernel right before writes --------------------------------------------
class LateWord:
    """An int32 in the last row of a long cache read: that call begins, lets its successor begin early, and writes zeros
    over the word at its end."""

    def __init__(self, hk=8, D=128, rows=20000):
        self.src = random_cache("f16", 1, hk, 64, D, 80)
        self.rows = rows
        self.pos = torch.full((rows,), 5, device="cuda", dtype=torch.int32)
        self.pos[-1] = -1
        self.buf = torch.zeros(rows, hk * D, device="cuda")
        self.word = self.buf[-1].view(torch.int32)

    def set(self, value):
        self.word.fill_(value)
        torch.cuda.synchronize()

    def clear_late(self):
        kv_cache_read(self.src.view, self.buf.data_ptr(), 0, ACT["f32"][0], self.rows, self.pos.data_ptr())


@pytest.mark.parametrize("kind", ["q8_0", "f16"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("T,HQ", [(1, 8), (2, 16), (8, 16), (1, 64), (40, 32)])
def test_lengths_that_the_kernel_before_writes_at_its_end(T, HQ, dtype, kind):
    late = LateWord()
    code, dt = ACT[dtype]
    c = random_cache(kind, 1, 8, 400, 128, 3)
    q = torch.randn(T, HQ * 128, device="cuda", generator=gen(1)).to(dt)
    want, out = torch.empty_like(q), torch.empty_like(q)
    call = lambda o: tree_attention(c.view, q.data_ptr(), o.data_ptr(), code, 1, T, HQ,  # noqa: E731
                                    late.word.data_ptr())
    late.set(0)
    call(want)
    torch.cuda.synchronize()
    for _ in range(5):
        late.set(300)
        late.clear_late()
        call(out)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    assert verify_error_word() == 0


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_positions_that_the_kernel_before_writes_at_its_end(dtype):
    late = LateWord()
    code, dt = ACT[dtype]
    for D in (128, 80):
        q = torch.randn(1, 8 * D, device="cuda", generator=gen(2)).to(dt)
        out, want = torch.empty_like(q), torch.empty_like(q)
        table = rope_table(500, D)
        for o in (want, out):
            late.set(0 if o is want else 77)
            if o is out:
                late.clear_late()
            qk_norm_rope(q.data_ptr(), 0, o.data_ptr(), 0, code, 1, 8, 0, D, table.data_ptr(), 500, late.word.data_ptr())
            torch.cuda.synchronize()
        assert torch.equal(out, want)
    for kind in ("q8_0", "f16"):
        c = random_cache(kind, 1, 1, 90, 128, 9)
        first, at77 = c.values("k")[0, 0, 0], c.values("k")[0, 0, 77]
        late.set(77)
        late.clear_late()
        o = torch.zeros(128, device="cuda")
        kv_cache_read(c.view, o.data_ptr(), 0, ACT["f32"][0], 1, late.word.data_ptr())
        torch.cuda.synchronize()
        assert torch.equal(o.double(), first)
        late.set(77)
        late.clear_late()
        k = torch.randn(128, device="cuda", generator=gen(3)).to(dt)
        kv_cache_write(c.view, k.data_ptr(), k.data_ptr(), code, 1, late.word.data_ptr())
        torch.cuda.synchronize()
        assert torch.equal(c.values("k")[0, 0, 77], at77) and not torch.equal(c.values("k")[0, 0, 0], first)
    assert verify_error_word() == 0
