"""The calls on 8-bit rows, their product and the verdict from several host threads at once, each on a stream of its own:
the same bits as alone."""
import threading

import pytest

from ramforge_b200 import (_lib, dequantize_i8, i8_matmul, norm_i8, quantize_i8, swiglu_i8, verify_drafts,
                           verify_error_word, verify_greedy)

from .test_gpu_i8_rows import gen, torch

pytestmark = pytest.mark.gpu


class Work:
    """One pass of a small layer with 8-bit weights, then the verdict on its logits, both ways."""

    def __init__(self, i):
        g = gen(300 + i)
        self.t, self.n, self.k = (1, 6, 40, 90, 200, 333)[i], (600, 1000, 384, 2048, 777, 1024)[i], (512, 257, 1024, 640, 2048, 96)[i]
        self.pitch = -(-self.k // 16) * 16
        self.x = torch.randn(self.t, self.k, device="cuda", generator=g)
        self.w = torch.ones(self.k, device="cuda")
        self.m = torch.randn(self.n, self.k, device="cuda", generator=g)
        self.tokens = torch.randint(0, self.n // 5, (1, 4), device="cuda", generator=g, dtype=torch.int32)
        self.u = torch.rand(5, device="cuda", generator=g)
        self.stream = torch.cuda.Stream()

    def outputs(self):
        t, n, k, p = self.t, self.n, self.k, self.pitch
        new = lambda *s, d=torch.float32: torch.zeros(*s, device="cuda", dtype=d)  # noqa: E731
        return dict(q=new(t, p, d=torch.int8), s=new(t), wq=new(n, p, d=torch.int8), ws=new(n), y=new(t, n),
                    gq=new(t, n // 2, d=torch.int8), gs=new(t), back=new(t, n // 2), best=new(1, 1, d=torch.int32),
                    out=new(1, 1, d=torch.int32), count=new(1, d=torch.int32), out2=new(1, 5, d=torch.int32),
                    count2=new(1, d=torch.int32))

    def calls(self, o, st):
        t, n, k, p, F = self.t, self.n, self.k, self.pitch, _lib.ACT_F32
        quantize_i8(self.m.data_ptr(), o["wq"].data_ptr(), o["ws"].data_ptr(), F, n, k, q_stride=p, stream=st)
        norm_i8(self.x.data_ptr(), self.w.data_ptr(), 1e-5, o["q"].data_ptr(), o["s"].data_ptr(), F, t, k, q_stride=p, stream=st)
        i8_matmul(o["q"].data_ptr(), o["s"].data_ptr(), o["wq"].data_ptr(), o["ws"].data_ptr(), o["y"].data_ptr(), F, t, n, k,
                  x_stride=p, w_stride=p, stream=st)
        swiglu_i8(o["y"].data_ptr(), o["y"].data_ptr() + 4 * (n // 2), o["gq"].data_ptr(), o["gs"].data_ptr(), F, t, n // 2,
                  gate_stride=n, up_stride=n, stream=st)
        dequantize_i8(o["gq"].data_ptr(), o["gs"].data_ptr(), o["back"].data_ptr(), F, t, n // 2, stream=st)
        verify_greedy(o["y"].data_ptr(), F, n, 1, 0, 0, o["best"].data_ptr(), o["out"].data_ptr(), o["count"].data_ptr(),
                      stream=st)
        # weights' scales are numbers above 0: the rows that the tokens follow
        verify_drafts(o["ws"].data_ptr(), 0, F, n // 5, 1, 4, self.tokens.data_ptr(), self.u.data_ptr(),
                      self.u[4:].data_ptr(), o["out2"].data_ptr(), o["count2"].data_ptr(), stream=st)


def test_calls_from_several_threads():
    works, rounds = [Work(i) for i in range(6)], 15
    outs = [[w.outputs() for _ in range(rounds)] for w in works]
    torch.cuda.synchronize()
    errors, gate = [], threading.Barrier(len(works))

    def run(w, mine):
        try:
            gate.wait(30)
            for o in mine:
                w.calls(o, w.stream.cuda_stream)
            w.stream.synchronize()
        except Exception as e:  # noqa: BLE001 - reported by the main thread
            errors.append(e)

    threads = [threading.Thread(target=run, args=x) for x in zip(works, outs)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for w, mine in zip(works, outs):
        want = w.outputs()
        w.calls(want, 0)
        torch.cuda.synchronize()
        assert want["y"].abs().max() > 0 and want["out2"][0, 0] >= 0
        for o in mine:
            assert all(torch.equal(o[n], want[n]) for n in want)
    assert verify_error_word() == 0
