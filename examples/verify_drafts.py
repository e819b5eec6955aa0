"""Drafted tokens verified in one pass, as speculative decoding does it, on one attention layer.

A prompt's keys and values go into an 8-bit cache.  Then a tree of drafted tokens is projected,
normalised and rotated, cached behind the history and attended in one call each; one path of the
tree is accepted, its rows are written again at consecutive positions, and the last accepted token
is checked against plain decoding over the cache that is left.

    python examples/verify_drafts.py
"""
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from ramforge_b200 import (KvView, QMatrix, _lib, kv_cache_write, qk_norm_rope, synth,  # noqa: E402
                           tree_attention, verify_error_word)

EMBD, HEADS, KV_HEADS, HEAD_DIM, CAPACITY = 1024, 8, 2, 128, 256
PROMPT = 50
# parent of each drafted token (-1: follows the prompt); three branches, up to four deep
PARENTS = [-1, 0, 1, 1, 3, -1, 5, 6, 0, 8, -1]


class Layer:
    """The attention half of a decoder layer: Q8_0 projection, per-head norms, rotation, Q8_0 cache."""

    def __init__(self, seed=1):
        rows = (HEADS + 2 * KV_HEADS) * HEAD_DIM
        w = synth.normal(seed, 100, rows * EMBD, std=0.02).reshape(rows, EMBD)
        self.qkv = QMatrix(synth.Q8_0, synth.quantize(synth.Q8_0, w), rows, EMBD)
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.q_norm, self.k_norm = (1 + 0.1 * torch.randn(HEAD_DIM, device="cuda", generator=g) for _ in range(2))
        inv = 10000.0 ** (-2.0 * torch.arange(HEAD_DIM // 2, device="cuda") / HEAD_DIM)
        angle = torch.arange(CAPACITY, device="cuda")[:, None] * inv
        self.rope = torch.stack([angle.cos(), angle.sin()], -1).contiguous()
        shape = (1, KV_HEADS, CAPACITY, HEAD_DIM)
        self.k, self.v = (torch.zeros(shape, device="cuda", dtype=torch.int8) for _ in range(2))
        scales = (1, KV_HEADS, CAPACITY, HEAD_DIM // 32)
        self.ks, self.vs = (torch.zeros(scales, device="cuda", dtype=torch.float16) for _ in range(2))
        self.cache = KvView(_lib.TYPE_Q8_0, self.k.data_ptr(), self.v.data_ptr(), self.ks.data_ptr(),
                            self.vs.data_ptr(), 1, KV_HEADS, HEAD_DIM, CAPACITY)

    def project(self, x, positions):
        """q [T][H * hd], k and v [T][KV * hd] of hidden rows x, normalised and rotated."""
        T, q_row, kv_row = x.shape[0], HEADS * HEAD_DIM, KV_HEADS * HEAD_DIM
        qkv = torch.empty(T, q_row + 2 * kv_row, device="cuda")
        self.qkv.gemm(x.data_ptr(), qkv.data_ptr(), T, stream=torch.cuda.current_stream().cuda_stream)
        q, k, v = qkv.split([q_row, kv_row, kv_row], dim=1)
        qo, ko = torch.empty(T, q_row, device="cuda"), torch.empty(T, kv_row, device="cuda")
        qk_norm_rope(q.data_ptr(), k.data_ptr(), qo.data_ptr(), ko.data_ptr(), _lib.ACT_F32, T, HEADS, KV_HEADS,
                     HEAD_DIM, self.rope.data_ptr(), CAPACITY, positions.data_ptr(), self.q_norm.data_ptr(),
                     self.k_norm.data_ptr(), q_stride=qkv.shape[1], k_stride=qkv.shape[1],
                     stream=torch.cuda.current_stream().cuda_stream)
        return qo, ko, v.contiguous()

    def write(self, k, v, slots):
        kv_cache_write(self.cache, k.data_ptr(), v.data_ptr(), _lib.ACT_F32, k.shape[0], slots.data_ptr(),
                       stream=torch.cuda.current_stream().cuda_stream)

    def attend(self, q, history, mask=None):
        out = torch.empty_like(q)
        hist = torch.tensor([history], device="cuda", dtype=torch.int32)
        tree_attention(self.cache, q.data_ptr(), out.data_ptr(), _lib.ACT_F32, 1, q.shape[0], HEADS, hist.data_ptr(),
                       mask_ptr=0 if mask is None else mask.data_ptr(),
                       stream=torch.cuda.current_stream().cuda_stream)
        return out


def int32(values):
    return torch.tensor(values, device="cuda", dtype=torch.int32)


def main():
    layer = Layer()
    g = torch.Generator(device="cuda").manual_seed(2)
    prompt = torch.randn(PROMPT, EMBD, device="cuda", generator=g)
    drafts = torch.randn(len(PARENTS), EMBD, device="cuda", generator=g)

    # the prompt fills the cache
    at = int32(range(PROMPT))
    _, k, v = layer.project(prompt, at)
    layer.write(k, v, at)

    # the tree: a token's position follows its depth, its cache place its number; it sees its ancestors and itself
    depth, sees = [], np.zeros((len(PARENTS), -(-len(PARENTS) // 32)), np.uint32)
    for j, parent in enumerate(PARENTS):
        depth.append(0 if parent < 0 else depth[parent] + 1)
        if parent >= 0:
            sees[j] = sees[parent]
        sees[j, j // 32] |= np.uint32(1 << (j % 32))
    mask = torch.from_numpy(sees.view(np.int32)).cuda()
    q, k, v = layer.project(drafts, int32([PROMPT + d for d in depth]))
    layer.write(k, v, int32(range(PROMPT, PROMPT + len(PARENTS))))
    out = layer.attend(q, PROMPT, mask)

    # the model agreed with one path (here: the deepest); its rows move up, the others are dropped
    path = [max(range(len(PARENTS)), key=lambda j: depth[j])]
    while PARENTS[path[0]] >= 0:
        path.insert(0, PARENTS[path[0]])
    slots = [-1] * len(PARENTS)
    for i, j in enumerate(path):
        slots[j] = PROMPT + i
    layer.write(k, v, int32(slots))

    # plain decoding of the last accepted token over the cache as it now is
    last = path[-1]
    again = layer.attend(q[last:last + 1], PROMPT + len(path) - 1)
    difference = (again[0] - out[last]).abs().max().item() / out[last].abs().max().item()
    print("accepted tokens", path, "difference from plain decoding %.1e" % difference)
    if difference > 1e-5 or verify_error_word():
        raise SystemExit("verification and decoding disagree")
    return difference


if __name__ == "__main__":
    main()
