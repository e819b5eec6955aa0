"""Rounds of speculative decoding on a small decoder with 8-bit weights, every step of a round on the device.

A round feeds the last token and a tree of drafted ones through all layers at once (norms and SwiGLU as 8-bit rows,
products in whole numbers, attention over an 8-bit cache), takes the verdict on the drafts, and writes the cache rows
of those that stand at their positions.  The host reads one number a round: how many stand.  A round is captured in a
CUDA graph once and replayed.  The tokens have to be those of plain decoding, one at a time.

    python examples/draft_rounds.py
"""
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from ramforge_b200 import (KvView, _lib, i8_matmul, kv_cache_write, norm_i8, qk_norm_rope, quantize_i8,  # noqa: E402
                           swiglu_i8, tree_attention, verify_drafts, verify_error_word, verify_greedy)

VOCAB, EMBD, HEADS, KV_HEADS, HEAD_DIM, FFN, LAYERS, CAPACITY = 1000, 512, 8, 2, 64, 1408, 2, 512
EPS = 1e-5
# the tree of a round: parent of each draft (-1: the last token)
PARENTS = [-1, 0, 1, 2, -1, 4, 0]


def stream():
    return torch.cuda.current_stream().cuda_stream


def int32(values):
    return torch.tensor(values, device="cuda", dtype=torch.int32)


class Linear8:
    """A weight matrix as 8-bit rows, one scale a channel."""

    def __init__(self, g, n_out, n_in):
        w = torch.randn(n_out, n_in, device="cuda", generator=g) * n_in ** -0.5
        self.n_out, self.n_in = n_out, n_in
        self.q = torch.empty(n_out, n_in, device="cuda", dtype=torch.int8)
        self.scale = torch.empty(n_out, device="cuda")
        quantize_i8(w.data_ptr(), self.q.data_ptr(), self.scale.data_ptr(), _lib.ACT_F32, n_out, n_in, stream=stream())

    def __call__(self, rows):
        q, scale = rows
        y = torch.empty(q.shape[0], self.n_out, device="cuda")
        i8_matmul(q.data_ptr(), scale.data_ptr(), self.q.data_ptr(), self.scale.data_ptr(), y.data_ptr(), _lib.ACT_F32,
                  q.shape[0], self.n_out, self.n_in, stream=stream())
        return y


def rows8(t, n):
    return torch.empty(t, n, device="cuda", dtype=torch.int8), torch.empty(t, device="cuda")


def norm8(x, delta, weight):
    """x += delta (where there is one); the norm of it as 8-bit rows."""
    out = rows8(*x.shape)
    norm_i8(x.data_ptr(), weight.data_ptr(), EPS, out[0].data_ptr(), out[1].data_ptr(), _lib.ACT_F32, *x.shape,
            add_ptr=0 if delta is None else delta.data_ptr(), sum_ptr=0 if delta is None else x.data_ptr(), stream=stream())
    return out


class Layer:
    def __init__(self, g):
        self.qkv = Linear8(g, (HEADS + 2 * KV_HEADS) * HEAD_DIM, EMBD)
        self.o = Linear8(g, EMBD, HEADS * HEAD_DIM)
        self.gate_up, self.down = Linear8(g, 2 * FFN, EMBD), Linear8(g, EMBD, FFN)
        self.norms = [1 + 0.1 * torch.randn(n, device="cuda", generator=g) for n in (EMBD, EMBD, HEAD_DIM, HEAD_DIM)]
        shape = (1, KV_HEADS, CAPACITY, HEAD_DIM)
        self.k, self.v = (torch.zeros(shape, device="cuda", dtype=torch.int8) for _ in range(2))
        self.ks, self.vs = (torch.zeros(*shape[:3], HEAD_DIM // 32, device="cuda", dtype=torch.float16) for _ in range(2))
        self.cache = KvView(_lib.TYPE_Q8_0, self.k.data_ptr(), self.v.data_ptr(), self.ks.data_ptr(), self.vs.data_ptr(),
                            1, KV_HEADS, HEAD_DIM, CAPACITY)
        self.rows = None  # keys and values of the latest pass, for those that stand

    def write(self, slots, first=0):
        k, v = self.rows
        kv_cache_write(self.cache, k[first:].data_ptr(), v[first:].data_ptr(), _lib.ACT_F32, k.shape[0] - first,
                       slots.data_ptr(), v_stride=v.stride(0), stream=stream())

    def __call__(self, x, delta, rope, positions, slots, hist, mask):
        t = x.shape[0]
        qkv = self.qkv(norm8(x, delta, self.norms[0]))
        q, k, v = qkv.split([HEADS * HEAD_DIM, KV_HEADS * HEAD_DIM, KV_HEADS * HEAD_DIM], dim=1)
        qo, ko = torch.empty(t, q.shape[1], device="cuda"), torch.empty(t, k.shape[1], device="cuda")
        qk_norm_rope(q.data_ptr(), k.data_ptr(), qo.data_ptr(), ko.data_ptr(), _lib.ACT_F32, t, HEADS, KV_HEADS, HEAD_DIM,
                     rope.data_ptr(), CAPACITY, positions.data_ptr(), self.norms[2].data_ptr(), self.norms[3].data_ptr(),
                     q_stride=qkv.shape[1], k_stride=qkv.shape[1], stream=stream())
        self.rows = ko, v
        self.write(slots)
        out = torch.empty_like(qo)
        tree_attention(self.cache, qo.data_ptr(), out.data_ptr(), _lib.ACT_F32, 1, t, HEADS, hist.data_ptr(),
                       mask_ptr=0 if mask is None else mask.data_ptr(), stream=stream())
        o = rows8(*out.shape)
        quantize_i8(out.data_ptr(), o[0].data_ptr(), o[1].data_ptr(), _lib.ACT_F32, *out.shape, stream=stream())
        gu = self.gate_up(norm8(x, self.o(o), self.norms[1]))
        h = rows8(t, FFN)
        swiglu_i8(gu.data_ptr(), gu.data_ptr() + 4 * FFN, h[0].data_ptr(), h[1].data_ptr(), _lib.ACT_F32, t, FFN,
                  gate_stride=2 * FFN, up_stride=2 * FFN, stream=stream())
        return self.down(h)


class Model:
    def __init__(self, seed=1):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.embd = torch.randn(VOCAB, EMBD, device="cuda", generator=g)
        self.layers = [Layer(g) for _ in range(LAYERS)]
        self.norm = 1 + 0.1 * torch.randn(EMBD, device="cuda", generator=g)
        self.head = Linear8(g, VOCAB, EMBD)
        inv = 10000.0 ** (-2.0 * torch.arange(HEAD_DIM // 2, device="cuda") / HEAD_DIM)
        angle = torch.arange(CAPACITY, device="cuda")[:, None] * inv
        self.rope = torch.stack([angle.cos(), angle.sin()], -1).contiguous()

    def __call__(self, tokens, positions, slots, hist, mask=None):
        """Logits of a pass: tokens at rotary positions, cached at slots, over `hist` positions and one another."""
        x, delta = self.embd[tokens.long()], None
        for layer in self.layers:
            delta = layer(x, delta, self.rope, positions, slots, hist, mask)
        return self.head(norm8(x, delta, self.norm))

    def prompt(self, tokens):
        at = int32(range(len(tokens)))
        return self(int32(tokens), at, at, int32([0]))[-1:].clone()


class Round:
    """A round's buffers, and its calls: a tree of drafts behind the last token."""

    def __init__(self, model, parents):
        t = len(parents)
        self.model, self.t = model, t
        self.fed = torch.zeros(t + 1, device="cuda", dtype=torch.int32)  # the last token, then the drafts
        self.hist = int32([0])                                           # cached positions before the last token
        self.parents = int32(parents)
        depth, sees = [0], np.zeros((t + 1, -(-(t + 1) // 32)), np.uint32)
        sees[0, 0] = 1
        for j, parent in enumerate(parents):  # row 1 + j: draft j, behind row 1 + parent
            depth.append(depth[parent + 1] + 1)
            sees[j + 1] = sees[parent + 1]
            sees[j + 1, (j + 1) // 32] |= np.uint32(1 << ((j + 1) % 32))
        self.depth, self.mask = int32(depth), torch.from_numpy(sees.view(np.int32)).cuda()
        self.index = int32(range(t + 1))
        self.best, self.out = (torch.zeros(t + 1, device="cuda", dtype=torch.int32) for _ in range(2))
        self.count, self.keep = int32([0]), torch.zeros(max(t, 1), device="cuda", dtype=torch.int32)
        self.graph = None

    def calls(self):
        logits = self.model(self.fed, self.hist + self.depth, self.hist + self.index, self.hist, self.mask)
        after = self.hist + 1  # the drafts that stand go behind the last token
        verify_greedy(logits.data_ptr(), _lib.ACT_F32, VOCAB, 1, self.t, self.fed[1:].data_ptr(), self.best.data_ptr(),
                      self.out.data_ptr(), self.count.data_ptr(), parent_ptr=self.parents.data_ptr(),
                      hist_len_ptr=after.data_ptr(), positions_ptr=self.keep.data_ptr(), stream=stream())
        for layer in self.model.layers:
            layer.write(self.keep, first=1)
        return logits

    def __call__(self, last, drafts, hist):
        """The tokens that a round gives: the drafts that stand, and the one behind them."""
        self.fed.copy_(int32([last] + list(drafts)))
        self.hist.fill_(hist)
        if self.graph is None:
            self.calls()  # once outside: the first calls load code
            self.graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(self.graph):
                self.logits = self.calls()
        self.graph.replay()
        return self.out[:int(self.count) + 1].tolist()


def plain(model, prompt, n):
    """Greedy decoding, one token a pass."""
    tokens, hist = [int(model.prompt(prompt).argmax())], len(prompt)
    while len(tokens) < n:
        at = int32([hist])
        tokens.append(int(model(int32([tokens[-1]]), at, at, int32([hist])).argmax()))
        hist += 1
    return tokens


def drafted(model, prompt, n, guess):
    """The same by rounds; guess(tokens so far) gives a round's drafts."""
    step = Round(model, PARENTS)
    tokens, hist, rounds = [int(model.prompt(prompt).argmax())], len(prompt), 0
    while len(tokens) < n:
        new = step(tokens[-1], guess(tokens), hist)
        tokens += new
        hist += len(new)
        rounds += 1
    return tokens[:n], rounds, step


def sampled(step, seed=5):
    """The verdict on the last round's tree by random numbers: target probabilities of its logits, a draft that is
    near them.  Returns the calls' inputs and results."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = step.t
    p = torch.softmax(step.logits, -1)
    q = torch.softmax(step.logits[:t] + torch.randn(t, VOCAB, device="cuda", generator=g), -1)
    tokens = torch.multinomial(q[(step.parents + 1).long()], 1, generator=g)[:, 0].int()
    u, u_next = torch.rand(t, device="cuda", generator=g), torch.rand(1, device="cuda", generator=g)
    out, count, keep = (torch.zeros(m, device="cuda", dtype=torch.int32) for m in (t + 1, 1, t))
    verify_drafts(p.data_ptr(), q.data_ptr(), _lib.ACT_F32, VOCAB, 1, t, tokens.data_ptr(), u.data_ptr(),
                  u_next.data_ptr(), out.data_ptr(), count.data_ptr(), parent_ptr=step.parents.data_ptr(),
                  hist_len_ptr=step.hist.data_ptr(), positions_ptr=keep.data_ptr(), stream=stream())
    return (p, q, tokens, u, u_next), (out, count, keep)


def main(n=60):
    model = Model()
    rng = np.random.RandomState(2)
    prompt = rng.randint(0, VOCAB, 20).tolist()
    want = plain(model, prompt, n)

    def guess(tokens):  # what a draft model would give: mostly right, here made from the answer
        ahead = (want + [0] * 8)[len(tokens):]
        wrong = rng.randint(0, VOCAB, len(PARENTS)).tolist()
        chain = [ahead[i] if rng.rand() < 0.8 else wrong[i] for i in range(4)]
        return chain + [ahead[0], ahead[1], ahead[1]]

    got, rounds, step = drafted(model, prompt, n, guess)
    _, (out, count, _) = sampled(step)
    print("%d tokens in %d rounds; sampled verdict: %d drafts stand, tokens %s" % (
        n, rounds, int(count), [x for x in out.tolist() if x >= 0]))
    if got != want or verify_error_word():
        raise SystemExit("rounds of drafts and plain decoding disagree")
    return rounds


if __name__ == "__main__":
    main()
