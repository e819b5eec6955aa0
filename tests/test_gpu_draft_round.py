"""A round of drafting as a user runs it (examples/draft_rounds.py): 8-bit projections, attention, verdict and cache
rows in one captured graph, against plain decoding and, call by call, against the calls' definitions."""
import importlib.util
import os

import numpy as np
import pytest

from ramforge_b200 import verify_error_word
from tests.test_gpu_accept import walk

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def rounds():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "draft_rounds.py")
    spec = importlib.util.spec_from_file_location("draft_rounds", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def test_example_gives_the_tokens_of_plain_decoding(rounds):
    n = rounds.main()
    assert n < 60  # some drafts stood in some rounds


def test_a_replayed_round_is_the_round_called_directly(rounds):
    """Same bits from the graph and from the calls, and a cache that holds the rows of what stands."""
    model = rounds.Model(seed=3)
    prompt = list(range(7, 27))
    model.prompt(prompt)
    step = rounds.Round(model, rounds.PARENTS)
    for drafts in ([5, 6, 7, 8, 9, 10, 11], [1, 2, 3, 4, 5, 6, 7]):
        step(4, drafts, len(prompt))
        got = [x.clone() for x in (step.logits, step.best, step.out, step.count, step.keep)]
        caches = [layer.k.clone() for layer in model.layers]
        logits = step.calls()
        for a, b in zip(got, (logits, step.best, step.out, step.count, step.keep)):
            assert torch.equal(a, b)
        for a, layer in zip(caches, model.layers):
            assert torch.equal(a, layer.k)
    assert verify_error_word() == 0


def test_a_drafted_token_has_the_hidden_state_of_plain_decoding(rounds):
    """A chain of drafts gives the logits of the same tokens fed one at a time.  The two differ in the order of the
    attention's sums, about 1e-6, which tips over one code in some 10^4; a code that tips moves its row by one step, 3 %
    of the size of one of 512 numbers, 0.14 % of the row.  2e-2 is 14 of them in the same row."""
    model = rounds.Model(seed=4)
    prompt, chain = list(range(30, 60)), [11, 500, 3, 77]
    model.prompt(prompt)
    step = rounds.Round(model, [-1, 0, 1, 2])
    step(9, chain, len(prompt))
    many = step.logits.clone()
    one = []
    for i, token in enumerate([9] + chain):
        at = rounds.int32([len(prompt) + i])
        one.append(model(rounds.int32([token]), at, at, rounds.int32([len(prompt) + i])))
    one = torch.cat(one)
    assert (many - one).norm() <= 2e-2 * one.norm()
    assert torch.equal(many.argmax(-1), one.argmax(-1))


def test_sampled_verdict_of_a_round(rounds):
    model = rounds.Model(seed=5)
    model.prompt(list(range(20)))
    step = rounds.Round(model, rounds.PARENTS)
    step(3, [1, 2, 3, 4, 5, 6, 7], 20)
    for seed in range(20):
        (p, q, tokens, u, u_next), got = rounds.sampled(step, seed)
        want = walk(p[None].double().cpu().numpy(), q[None].double().cpu().numpy(), [tokens.tolist()], [rounds.PARENTS],
                    [step.t], u[None].cpu().numpy(), u_next.cpu().numpy(), [20])
        for a, b in zip(got, want):
            np.testing.assert_array_equal(a.cpu().numpy(), np.ravel(b))
    assert verify_error_word() == 0
