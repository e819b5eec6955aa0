"""The verdict on drafted tokens where a shorter way through it would go wrong, or take long."""
import numpy as np
import pytest

from ramforge_b200 import _lib, verify_drafts, verify_error_word, verify_greedy

from .test_gpu_accept import Case, same, torch

pytestmark = pytest.mark.gpu


def test_little_left_behind_certain_drafts():
    """Certain drafts that have nearly all of what is left, each refused by a random number just below 1: the sum of
    the rest is 1e-21 of the first one's, and the last draft's share of it a hundredth."""
    seqs, vocab, below = 16, 200, 1 - 2.0 ** -24
    c = Case(seqs, 4, vocab, draft=False)
    c.given_parents = True
    c.parent[:], c.tokens[:] = -1, [3, 50, 120, 199]
    c.p.zero_()
    c.p[:, 0] = 1e-21 / vocab
    c.p[:, 0, 3], c.p[:, 0, 50], c.p[:, 0, 199] = below, 2.0 ** -24, 1e-23
    c.p[:, 0, 120] = 4e-15 * (1 + 0.01 * torch.arange(seqs, device="cuda"))
    c.u[:], c.u[:, 3] = below, 0.9
    w = c.want()
    assert (w[1] == 0).all() and not np.isin(w[0][:, 0], c.tokens).any()
    same(c.run(), w)
    assert verify_error_word() == 0


def graph_us(fn, calls=20):
    """Microseconds of a call among others, the least of fifteen."""
    fn(torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(calls):
            fn(torch.cuda.current_stream().cuda_stream)
    times = []
    for _ in range(15):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        graph.replay()
        b.record()
        torch.cuda.synchronize()
        times.append(a.elapsed_time(b) * 1e3 / calls)
    return min(times)


def greedy_rows(logits, vocab, stride):
    code = {torch.float32: _lib.ACT_F32, torch.float16: _lib.ACT_F16, torch.bfloat16: _lib.ACT_BF16}[logits.dtype]
    n = logits.shape[0]
    best, out, count = (torch.full((n,), -7, device="cuda", dtype=torch.int32) for _ in range(3))

    def call(stream=0):
        verify_greedy(logits.data_ptr(), code, vocab, n, 0, 0, best.data_ptr(), out.data_ptr(), count.data_ptr(),
                      logits_stride=stride, stream=stream)
    call()
    assert torch.equal(best, out) and not count.any()
    return best, call


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab,gap", [(9, 128256, 0), (9, 50257, 0), (300, 50257, 3), (1, 131, 0), (12, 4097, 2),
                                            (400, 9, 1)])
def test_greedy_rows_of_nan_and_infinities(rows, vocab, gap, dtype):
    """Rows with nothing above -infinity: the first -infinity wherever it lies, 0 where there is none; largest numbers
    more than once, in front of every place that a thread or a 16-byte piece may begin at."""
    rs = np.random.RandomState(rows + vocab)
    logits = torch.full((rows, vocab + gap), float("nan"), device="cuda", dtype=dtype)
    want = np.zeros(rows, np.int64)
    for r in range(rows):
        kind, at = r % 3, rs.randint(vocab)
        if kind == 0:      # NaN, and one -infinity or more behind it
            want[r] = at
            logits[r, at] = logits[r, rs.randint(at, vocab)] = -float("inf")
            if r % 2:
                logits[r, at:vocab] = -float("inf")
        elif kind == 1:    # NaN alone
            want[r] = 0
        else:              # two equal numbers between them
            want[r] = at
            logits[r, at] = logits[r, rs.randint(at, vocab)] = -3.0
            logits[r, rs.randint(vocab)] = -float("inf") if rs.rand() < 0.5 else float("nan")
            held = logits[r, :vocab].float().cpu().numpy()
            want[r] = np.where(np.isnan(held), -np.inf, held).argmax() if (held == -3).any() else (
                np.flatnonzero(held == -np.inf)[0] if (held == -np.inf).any() else 0)
    best, _ = greedy_rows(logits, vocab, vocab + gap)
    np.testing.assert_array_equal(best.cpu().numpy(), want)
    assert verify_error_word() == 0


@pytest.mark.parametrize("rows", [9, 300])
def test_greedy_rows_of_nan_take_no_longer(rows):
    """What is in a row does not show in the time: NaN alone, or one -infinity at its end, as numbers."""
    vocab = 128256
    logits = torch.randn(rows, vocab, device="cuda", dtype=torch.bfloat16)
    usual = graph_us(greedy_rows(logits, vocab, vocab)[1])
    logits.fill_(float("nan"))
    empty = graph_us(greedy_rows(logits, vocab, vocab)[1])
    logits[:, -1] = -float("inf")
    late = graph_us(greedy_rows(logits, vocab, vocab)[1])
    assert max(empty, late) < 3 * usual, (usual, empty, late)


def test_a_leaf_behind_refused_drafts_takes_one_pass():
    """Certain drafts behind the history: the last one stands after one or after two were refused, and nothing follows
    it.  Either way the row of the history is summed up once and the last draft's once, so the times are alike."""
    vocab = 4000000  # passes of 40 us each, beside which nothing else shows
    p = torch.softmax(torch.randn(1, 4, vocab, device="cuda", generator=torch.Generator(device="cuda").manual_seed(4)), -1)
    out, count = torch.full((4,), -7, device="cuda", dtype=torch.int32), torch.zeros(1, device="cuda", dtype=torch.int32)
    tokens, parent = torch.tensor([5, 6, 7], device="cuda", dtype=torch.int32), torch.full((3,), -1, device="cuda", dtype=torch.int32)
    u_next = torch.full((1,), 0.5, device="cuda")
    times = []
    for refused in (1, 2):
        u = torch.where(torch.arange(3, device="cuda") < refused, 0.99, 0.0)
        times.append(graph_us(lambda st: verify_drafts(
            p.data_ptr(), 0, _lib.ACT_F32, vocab, 1, 3, tokens.data_ptr(), u.data_ptr(), u_next.data_ptr(), out.data_ptr(),
            count.data_ptr(), parent_ptr=parent.data_ptr(), stream=st)))
        assert count.item() == 1 and out[0].item() == 5 + refused and out[2:].tolist() == [-1, -1]
    assert times[1] < 1.2 * times[0], times


@pytest.mark.parametrize("seqs,t", [(64, 4), (50, 0)])
def test_rows_at_a_padded_stride_without_a_draft(seqs, t):
    """Rows of an odd vocabulary at 16-byte places take no longer than rows of an even one, where no draft has rows."""
    stride, times = 50264, []
    p = torch.softmax(torch.randn(seqs, t + 1, stride, device="cuda", generator=torch.Generator(device="cuda").manual_seed(t)), -1)
    out = torch.empty(seqs, t + 1, device="cuda", dtype=torch.int32)
    count, tokens = torch.empty(seqs, device="cuda", dtype=torch.int32), torch.full((seqs, t), 9, device="cuda", dtype=torch.int32)
    u, u_next = torch.full((seqs, t), 0.5, device="cuda"), torch.full((seqs,), 0.5, device="cuda")
    for vocab in (50264, 50257):
        times.append(graph_us(lambda st: verify_drafts(
            p.data_ptr(), 0, _lib.ACT_F32, vocab, seqs, t, tokens.data_ptr(), u.data_ptr(), u_next.data_ptr(),
            out.data_ptr(), count.data_ptr(), target_stride=stride, stream=st)))
        row = p[:, 0, :vocab].double()
        row[:, 9] = 0 if t else row[:, 9]
        cum = row.cumsum(-1)
        want = torch.searchsorted(cum, 0.5 * cum[:, -1:], right=True)[:, 0]
        assert not count.any() and torch.equal(out[:, 0].long(), want)
    assert times[1] < 1.15 * times[0], times
