"""The verdict on drafted tokens (rf_verify_drafts, rf_verify_greedy) against the definition in 64 bits, walked on
the host.  All results are whole numbers and compared for equality: random numbers are inputs, and a border is
missed only where a 64-bit sum's last bits decide."""
import math

import numpy as np
import pytest

from ramforge_b200 import _lib, verify_drafts, verify_error_word, verify_greedy

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

ACT = {"f32": (_lib.ACT_F32, torch.float32), "f16": (_lib.ACT_F16, torch.float16),
       "bf16": (_lib.ACT_BF16, torch.bfloat16)}


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def wide(x):
    return None if x is None else x.double().cpu().numpy()


def path_out(b, t, path, token, tokens, hist):
    out, pos = np.full(t + 1, -1), np.full(t, -1)
    for i, j in enumerate(path):
        out[i], pos[j] = tokens[b][j], hist[b] + i
    out[len(path)] = token
    return out, len(path), pos


def walk(p, q, tokens, parent, n_draft, u, u_next, hist):
    """The definition, one sequence at a time: (out_tokens, n_accepted, positions)."""
    res = []
    for b in range(p.shape[0]):
        t, node, path = len(tokens[b]), -1, []
        while True:
            row = np.where(p[b, node + 1] > 0, p[b, node + 1], 0.0)
            r, mass, off, go = row, 1.0, 0.0, False
            for j in range(n_draft[b]):
                c = tokens[b][j]
                if parent[b][j] != node or j <= node or not 0 <= c < row.size:
                    continue
                qc = 1.0 if q is None else q[b, node + 1, c]
                if float(u[b][j]) * qc * mass < r[c]:
                    node, go = j, True
                    path.append(j)
                    break
                off += mass
                if q is None:
                    r = r.copy()
                    r[c] = 0
                else:
                    r = np.fmax(row - off * q[b, node + 1], 0)
                mass = math.fsum(r)
            if not go:
                break
        if not r.any():
            r = row
        token = -1
        if r.any():
            cum = np.cumsum(r.astype(np.longdouble))
            token = int(np.searchsorted(cum, max(float(u_next[b]), 0.0) * cum[-1], side="right"))
            token = min(token, int(np.flatnonzero(r)[-1]))
        res.append(path_out(b, t, path, token, tokens, hist))
    return [np.array(x) for x in zip(*res)]


def parents(rs, seqs, t, tree):
    if not tree:
        return np.tile(np.arange(-1, t - 1), (seqs, 1))
    out = np.full((seqs, t), -1)
    for j in range(1, t):
        out[:, j] = rs.randint(max(-1, j - 5), j, size=seqs)
    return out


class Case:
    def __init__(self, seqs, t, vocab, dtype="f32", tree=False, draft=True, ragged=False, seed=0, spread=2.0, pad=0):
        g, rs = gen(seed + 17 * vocab + t), np.random.RandomState(seed)
        code, dt = ACT[dtype]
        self.code, self.seqs, self.t, self.vocab = code, seqs, t, vocab
        logits = spread * torch.randn(seqs, t + 1, vocab + pad, device="cuda", generator=g)
        self.p = torch.softmax(logits, -1).to(dt)[..., :vocab]
        near = logits[:, :max(t, 1)] + 0.8 * torch.randn(seqs, max(t, 1), vocab + pad, device="cuda", generator=g)
        q = torch.softmax(near, -1).to(dt)[..., :vocab]
        self.q = q if draft and t else None
        self.parent = parents(rs, seqs, t, tree)
        rows = q.double().cpu().numpy()
        self.tokens = np.zeros((seqs, t), np.int64)
        for b in range(seqs):
            for j in range(t):
                cum = np.cumsum(rows[b, self.parent[b, j] + 1])
                self.tokens[b, j] = min(np.searchsorted(cum, rs.rand() * cum[-1], side="right"), vocab - 1)
        self.n_draft = rs.randint(0, t + 1, size=seqs) if ragged else np.full(seqs, t)
        self.u, self.u_next = rs.rand(seqs, t).astype(np.float32), rs.rand(seqs).astype(np.float32)
        self.hist = rs.randint(0, 1000, size=seqs)
        self.given_parents = tree

    def run(self, stream=0, dev=None):
        d = dev or self.device()
        out = [torch.full(s, -7, device="cuda", dtype=torch.int32) for s in ((self.seqs, self.t + 1), (self.seqs,),
                                                                             (self.seqs, self.t))]
        verify_drafts(self.p.data_ptr(), 0 if self.q is None else self.q.data_ptr(), self.code, self.vocab, self.seqs,
                      self.t, d["tokens"].data_ptr(), d["u"].data_ptr(), d["u_next"].data_ptr(), out[0].data_ptr(),
                      out[1].data_ptr(), parent_ptr=d["parent"].data_ptr() if self.given_parents else 0,
                      n_draft_ptr=d["n_draft"].data_ptr(), hist_len_ptr=d["hist"].data_ptr(),
                      positions_ptr=out[2].data_ptr(), target_stride=self.p.stride(1),
                      draft_stride=0 if self.q is None else self.q.stride(1), stream=stream)
        return out

    def device(self):
        d = {n: torch.from_numpy(np.ascontiguousarray(getattr(self, n)).astype(np.int32)).cuda()
             for n in ("tokens", "parent", "n_draft", "hist")}
        d["u"], d["u_next"] = torch.from_numpy(self.u).cuda(), torch.from_numpy(self.u_next).cuda()
        return d

    def want(self):
        return walk(wide(self.p), wide(self.q), self.tokens, self.parent, np.clip(self.n_draft, 0, self.t), self.u,
                    self.u_next, self.hist)


def same(got, want):
    for g, w in zip(got, want):
        np.testing.assert_array_equal(g.cpu().numpy(), w)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("draft", [True, False])
@pytest.mark.parametrize("seqs,t,vocab,tree,ragged", [
    (1, 1, 1, False, False), (1, 4, 7, False, False), (40, 5, 33, False, True), (40, 12, 50, True, True),
    (3, 1, 1000, False, False), (60, 9, 257, True, False), (7, 40, 4000, True, True), (2, 8, 32000, False, True),
    (5, 3, 50257, True, False), (2, 16, 128256, True, False), (1, 8, 128256, False, False),
    (7, 4, 70001, True, True), (8, 4, 70001, True, True), (130, 2, 3001, False, False), (300, 2, 101, True, True), (150, 3, 600, False, True),
    (2, 300, 31, True, False), (1, 1024, 20, False, False), (1, 1024, 20, True, False)])
def test_walks(seqs, t, vocab, tree, ragged, draft, dtype):
    for seed in range(3 if vocab < 5000 else 1):
        c = Case(seqs, t, vocab, dtype, tree, draft, ragged, seed, pad=-vocab % 8 if seed else 0)
        same(c.run(), c.want())
    assert verify_error_word() == 0


def test_plain_sampling_without_drafts():
    c = Case(50, 0, 777)
    same(c.run(), c.want())


@pytest.mark.parametrize("draft", [True, False])
def test_many_siblings(draft):
    """All drafts follow the history and most are refused: what is left shrinks with each."""
    c = Case(30, 24, 12, "f32", True, draft, False, 5, spread=1.0)
    c.parent[:] = -1
    c.u[:] = 0.6 + 0.399 * c.u
    if c.q is not None:  # siblings are drawn from one row, and here from one unlike the target's
        c.q[:, 0] = torch.softmax(2 * torch.randn(30, 12, device="cuda", generator=gen(1)), -1)
    same(c.run(), c.want())


def test_borders():
    """Random numbers of 0 and just below 1, equal rows, rows of one token, a token that neither side can draw."""
    c = Case(8, 3, 40, seed=2)
    c.u[0], c.u_next[0] = 0.0, 0.0
    c.u[1], c.u_next[1] = 1 - 2.0 ** -24, 1 - 2.0 ** -24
    c.q[2] = c.p[2, :3]                      # equal: all stand, whatever the numbers
    c.u[2] = 1 - 2.0 ** -24
    c.p[3] = 0
    c.p[3, :, 11] = 1                        # the target is certain
    c.tokens[3] = [11, 11, 5]
    c.p[4, 0, c.tokens[4, 0]] = 0            # the target never says this one
    c.u[4] = 0.0
    c.p[5, 0], c.q[5, 0] = c.q[5, 0] * 0.5, c.q[5, 0]   # nothing is left once the draft's share is taken off
    c.u[5] = 0.9
    c.u_next[6], c.u_next[7] = 1.0, -1.0
    c.q[6], c.q[7, 0, :20] = 0, float("nan")
    c.p[7, 0, 30:] = float("nan")
    w = c.want()
    assert w[1][2] == 3 and w[1][4] == 0 and w[1][5] == 0 and w[0][5][0] >= 0
    same(c.run(), w)
    assert verify_error_word() == 0


def test_indices_out_of_range():
    c = Case(6, 4, 30, tree=True, seed=3)
    c.tokens[0, 0], c.tokens[1, 1] = 30, -5
    c.parent[2, 1], c.parent[3, 0] = 1, 0
    c.n_draft[4], c.n_draft[5] = 5, -1
    got = c.run()
    assert verify_error_word() == 2 and verify_error_word() == 0
    want = c.want()
    for b in (4, 5):
        want[0][b], want[1][b], want[2][b] = -1, 0, -1
    same(got, want)
    c = Case(2, 2, 30)
    c.p[1] = 0  # a row without a number above 0
    got = c.run()
    assert got[0][1].tolist() == [-1, -1, -1] and got[1].tolist()[1] == 0 and verify_error_word() == 2
    same([g[:1] for g in got], [w[:1] for w in c.want()])


@pytest.mark.parametrize("draft", [True, False])
def test_tokens_follow_the_target(draft):
    """The first token of 60000 sequences with the same rows: each share within 5 standard deviations of the
    target's probability, for a chain and for siblings drawn from the same row."""
    n, vocab = 60000, 6
    g = gen(9)
    p = torch.tensor([0.35, 0.05, 0.2, 0.25, 0.15, 0.0], device="cuda")
    q = torch.tensor([0.1, 0.3, 0.2, 0.05, 0.05, 0.3], device="cuda")
    for tree in (False, True):
        t = 3
        c = Case(1, t, vocab)
        c.seqs, c.given_parents = n, tree
        c.p, c.q = p.expand(n, t + 1, vocab).contiguous(), q.expand(n, t, vocab).contiguous()
        c.parent = np.tile([-1, -1, -1] if tree else [-1, 0, 1], (n, 1))
        c.tokens = torch.multinomial(q, n * t, replacement=True, generator=g).view(n, t).cpu().numpy()
        if not draft:  # certain drafts, the same of each sequence
            c.q, c.tokens = None, np.tile([1, 0, 2], (n, 1))
        c.n_draft, c.hist = np.full(n, t), np.zeros(n, np.int64)
        c.u = torch.rand(n, t, device="cuda", generator=g).cpu().numpy()
        c.u_next = torch.rand(n, device="cuda", generator=g).cpu().numpy()
        first = c.run()[0][:, 0]
        share = torch.bincount(first, minlength=vocab).double().cpu() / n
        pd = p.double().cpu()
        assert ((share - pd).abs() <= 5 * (pd * (1 - pd) / n).sqrt()).all(), share
    assert verify_error_word() == 0


def best_of(logits):
    x = np.where(np.isnan(logits), -np.inf, logits)
    return x.argmax(-1)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("seqs,t,vocab,tree,ragged", [
    (1, 0, 5, False, False), (1, 1, 1, False, False), (9, 6, 33, True, True), (1, 4, 32000, False, False),
    (16, 8, 50257, False, True), (3, 24, 128256, True, False), (200, 3, 300, True, False), (1, 1024, 9, True, False),
    (1, 1024, 9, False, False), (2, 5, 128257, False, False)])
def test_greedy(seqs, t, vocab, tree, ragged, dtype):
    code, dt = ACT[dtype]
    rs = np.random.RandomState(vocab + t)
    logits = torch.randn(seqs, t + 1, vocab, device="cuda", generator=gen(t)).to(dt)
    if dtype != "f32" or vocab > 3000:  # coarse numbers: many equal largest ones
        logits = (logits * 4).round() / 4
    logits[rs.randint(seqs), 0, :vocab // 2] = float("nan")
    best = best_of(wide(logits))
    parent = parents(rs, seqs, t, tree)
    at = np.arange(seqs)[:, None]
    tokens = np.where(rs.rand(seqs, t) < 0.8, best[at, parent + 1], rs.randint(0, vocab, (seqs, t)))
    n_draft = rs.randint(0, t + 1, size=seqs) if ragged else np.full(seqs, t)
    hist = rs.randint(0, 500, seqs)
    dev = [torch.from_numpy(np.ascontiguousarray(x).astype(np.int32)).cuda() for x in (tokens, parent, n_draft, hist)]
    out = [torch.full(s, -7, device="cuda", dtype=torch.int32) for s in ((seqs, t + 1), (seqs, t + 1), (seqs,), (seqs, t))]
    verify_greedy(logits.data_ptr(), code, vocab, seqs, t, dev[0].data_ptr(), out[0].data_ptr(), out[1].data_ptr(),
                  out[2].data_ptr(), parent_ptr=dev[1].data_ptr() if tree else 0, n_draft_ptr=dev[2].data_ptr(),
                  hist_len_ptr=dev[3].data_ptr(), positions_ptr=out[3].data_ptr())
    res = []
    for b in range(seqs):
        node, path = -1, []
        while True:
            kids = [j for j in range(node + 1, n_draft[b]) if parent[b, j] == node and tokens[b, j] == best[b, node + 1]]
            if not kids:
                break
            node = kids[0]
            path.append(node)
        res.append(path_out(b, t, path, best[b, node + 1], tokens, hist))
        assert out[0][b, :n_draft[b] + 1].tolist() == best[b, :n_draft[b] + 1].tolist()
        assert (out[0][b, n_draft[b] + 1:] == -7).all()
    same(out[1:], [np.array(x) for x in zip(*res)])
    assert verify_error_word() == 0


def test_greedy_special_rows():
    """Infinities, zeros of both signs, rows of NaN alone; indices out of range; rows at a stride and off alignment."""
    vocab, inf, nan = 10, float("inf"), float("nan")
    rows = torch.tensor([[-inf] * 10, [nan] * 10, [-0.0, 0.0] * 5, [0.0, -0.0] * 5, [1.0, inf, inf, 2, 3, 4, 5, 6, 7, nan],
                         [-3.0, -2, -1, -1, -5, -6, -7, -8, -9, -inf]], device="cuda")
    buf = torch.full((6 * 13 + 1,), 9e9, device="cuda")
    held = buf[1:].view(6, 13)
    held[:, :vocab] = rows
    best = torch.full((6,), -7, device="cuda", dtype=torch.int32)
    out, count = best.clone(), best.clone()
    verify_greedy(held.data_ptr(), _lib.ACT_F32, vocab, 6, 0, 0, best.data_ptr(), out.data_ptr(), count.data_ptr(),
                  logits_stride=13)
    assert best.tolist() == [0, 0, 0, 0, 1, 2] and out.tolist() == best.tolist() and count.tolist() == [0] * 6
    assert verify_error_word() == 0
    # sequences of 2 drafts: a token out of range, a parent that is not before its draft, a count out of range
    logits = torch.zeros(3, 3, vocab, device="cuda")
    logits[:, :, 4] = 1
    tokens = torch.tensor([[10, 4], [4, 4], [4, 4]], device="cuda", dtype=torch.int32)
    parent = torch.tensor([[-1, -1], [-1, 1], [-1, 0]], device="cuda", dtype=torch.int32)
    nd = torch.tensor([2, 2, 3], device="cuda", dtype=torch.int32)
    best, out = (torch.full((3, 3), -7, device="cuda", dtype=torch.int32) for _ in range(2))
    count = torch.full((3,), -7, device="cuda", dtype=torch.int32)
    verify_greedy(logits.data_ptr(), _lib.ACT_F32, vocab, 3, 2, tokens.data_ptr(), best.data_ptr(), out.data_ptr(),
                  count.data_ptr(), parent_ptr=parent.data_ptr(), n_draft_ptr=nd.data_ptr())
    assert verify_error_word() == 2
    assert out.tolist() == [[4, 4, -1], [4, 4, -1], [-1, -1, -1]] and count.tolist() == [1, 1, 0]


def test_replayed_and_on_several_streams():
    """A captured verdict replayed on new rows and numbers; then eight calls on four streams at once."""
    c = Case(4, 6, 5000, tree=True, ragged=True, seed=8)
    dev = c.device()
    c.run(dev=dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = c.run(stream=torch.cuda.current_stream().cuda_stream, dev=dev)
    for seed in (9, 10):
        n = Case(4, 6, 5000, tree=True, ragged=True, seed=seed)
        c.p.copy_(n.p), c.q.copy_(n.q)
        for name, x in n.device().items():
            dev[name].copy_(x)
        graph.replay()
        same(out, n.want())
    cases = [Case(3, 5, 9000, tree=i % 2 == 0, draft=i % 3 > 0, seed=20 + i) for i in range(8)]
    devs, streams = [k.device() for k in cases], [torch.cuda.Stream() for _ in range(4)]
    torch.cuda.synchronize()
    outs = []
    for i, (k, d) in enumerate(zip(cases, devs)):
        with torch.cuda.stream(streams[i % 4]):
            outs.append(k.run(stream=streams[i % 4].cuda_stream, dev=d))
    torch.cuda.synchronize()
    for k, o in zip(cases, outs):
        same(o, k.want())
    assert verify_error_word() == 0
