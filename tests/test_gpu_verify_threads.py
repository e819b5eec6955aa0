"""The verification calls from several host threads at once, each on a stream of its own: the same bits as alone."""
import threading

import pytest

from ramforge_b200 import kv_cache_write, tree_attention, verify_error_word

from .test_gpu_verify import ACT, Cache, gen, random_cache, torch

pytestmark = pytest.mark.gpu


def test_calls_from_several_threads():
    hk, HQ, D, cap, threads, rounds = 2, 8, 128, 700, 6, 20
    work = []
    for i in range(threads):
        kind, dtype, T = ("f16", "q8_0")[i % 2], ("f16", "f32", "bf16")[i % 3], (3, 12, 40)[i // 2]
        c = random_cache(kind, 1, hk, cap, D, i)
        own = Cache(kind, 1, hk, cap, D)
        q = torch.randn(T, HQ * D, device="cuda", generator=gen(50 + i)).to(ACT[dtype][1])
        hl = torch.tensor([600 + i], device="cuda", dtype=torch.int32)
        k = torch.randn(T, hk * D, device="cuda", generator=gen(60 + i)).to(ACT[dtype][1])
        pos = torch.arange(T, device="cuda", dtype=torch.int32)
        work.append((c, own, q, hl, k, pos, ACT[dtype][0], T, torch.cuda.Stream()))

    def step(w, out, stream):
        c, own, q, hl, k, pos, code, T, _ = w
        tree_attention(c.view, q.data_ptr(), out.data_ptr(), code, 1, T, HQ, hl.data_ptr(), stream=stream)
        kv_cache_write(own.view, k.data_ptr(), k.data_ptr(), code, T, pos.data_ptr(), stream=stream)

    outs = [[torch.empty_like(w[2]) for _ in range(rounds)] for w in work]
    torch.cuda.synchronize()
    errors, gate = [], threading.Barrier(threads)

    def run(i):
        try:
            gate.wait(30)
            for o in outs[i]:
                step(work[i], o, work[i][-1].cuda_stream)
            work[i][-1].synchronize()
        except Exception as e:  # noqa: BLE001 - reported by the main thread
            errors.append(e)

    ts = [threading.Thread(target=run, args=(i,)) for i in range(threads)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    assert not errors, errors
    for w, os_ in zip(work, outs):
        want = torch.empty_like(w[2])
        step(w, want, 0)
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for o in os_)
        assert torch.equal(w[1].k, w[1].v) and w[1].k.any()
    assert verify_error_word() == 0
