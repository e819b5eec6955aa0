"""The verdict on drafted tokens where a shorter way through it would go wrong, or take long."""
import numpy as np
import pytest

from ramforge_b200 import verify_error_word

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
