"""A device wait that ran out is looked at before its results are: the engine's
serving paths raise and stay where they were.  (The wait itself does not run
out here: the status word is set as a kernel would set it.)"""

import numpy as np
import pytest
import torch

from tests.test_gpu_serving_engine import SMALL, engine, ragged
from torch2iron_b200 import _lib, synth

pytestmark = pytest.mark.gpu

TIMEOUT = 4      # T2B_ERR_TIMEOUT


def chain(eng, nodes=5):
    tok = np.repeat(eng.tokens.cpu().numpy()[:, None], nodes, 1)
    return tok, np.tile(np.arange(-1, nodes - 1), (tok.shape[0], 1))


def test_decode_tree_can_be_repeated_after_a_timeout():
    model, prompts = synth.random_model(SMALL, seed=111), ragged(SMALL, [9, 30], 112)
    a, b = engine(SMALL, model, 2), engine(SMALL, model, 2)
    for e in (a, b):
        e.prefill_packed(prompts)
    tree = chain(a)
    before = [t.clone() for t in (a.pos, a.tokens, a.next_tokens)]
    a.err.fill_(TIMEOUT)
    with pytest.raises(_lib.T2BError):
        a.decode_tree(*tree)
    assert all(torch.equal(x, y) for x, y in zip(before, (a.pos, a.tokens, a.next_tokens)))
    assert int(a.err) == 0
    for x, y in zip(a.decode_tree(*tree), b.decode_tree(*tree)):
        assert torch.equal(x, y)
    for name in ("pos", "tokens", "next_tokens"):
        assert torch.equal(getattr(a, name), getattr(b, name))
    for r, n in enumerate(a.pos.tolist()):
        assert all(torch.equal(x[r, :, :n], y[r, :, :n]) for x, y in zip(a.k_cache + a.v_cache, b.k_cache + b.v_cache))


def test_scores_of_a_timed_out_prefill_are_not_returned():
    model, prompts = synth.random_model(SMALL, seed=113), ragged(SMALL, [9, 30], 114)
    eng = engine(SMALL, model, 2)
    eng.tokens.fill_(3)
    eng.pos.fill_(1)
    eng.err.fill_(TIMEOUT)
    with pytest.raises(_lib.T2BError):
        eng.prefill_packed(prompts, score=True)
    assert eng.tokens.tolist() == [3, 3] and eng.pos.tolist() == [1, 1]
    assert eng.prefill_packed(prompts, score=True).logprob.shape == (39,)
    assert eng.pos.tolist() == [9, 30]
