"""The engine's serving paths over a quantised lm_head, and draft trees on models
whose greedy picks are sure for many steps."""

import numpy as np
import pytest
import torch

from tests.gpu_util import max_abs
from tests.test_gpu_serving_engine import SMALL, SURE, WIDE, drafts, engine, greedy, padded, ragged
from torch2iron_b200 import synth

pytestmark = pytest.mark.gpu


def quantised_head(cfg, seed):
    model = synth.random_model(cfg, seed=seed)
    model["lm_head"] = synth.quantize_rtn_autogptq(model["embed"].float())
    return model


@pytest.mark.parametrize("cfg,seed,head,T,take", [(WIDE, 211, False, 20, 4), (WIDE, 211, False, 130, 6), (SMALL, 208, False, 40, 5),
                                                  (SMALL, 208, True, 12, 3)])
def test_decode_tree_follows_sure_greedy_picks(cfg, seed, head, T, take):
    """Prompts whose first ten greedy picks each lead by more than two paths'
    difference: the trees emit exactly those tokens, ``take`` at least at a time."""
    model = quantised_head(cfg, seed) if head else synth.random_model(cfg, seed=seed)
    prompts, rng, steps = ragged(cfg, [30, 30], seed + 1000), np.random.default_rng(seed), 16
    want, sure, _ = greedy(cfg, model, prompts, steps)
    rows = [b for b in range(2) if sure[b] >= 10]
    assert rows == [0, 1] or (head and rows)
    eng = engine(cfg, model, 2)
    eng.prefill_packed(prompts)
    emitted = [[int(t)] for t in eng.next_tokens.cpu()]
    taken = 0
    while max(len(e) for e in emitted) + take <= 10:
        n = [len(e) for e in emitted]
        chain = [[emitted[b][-1], *want[b, n[b]:n[b] - 1 + take].tolist()] for b in range(2)]
        tok, par = drafts(rng, chain, T, cfg.vocab_size)
        path, count, following = eng.decode_tree(tok, par)
        for b in range(2):
            emitted[b] += [int(tok[b, i]) for i in path[b, 1:int(count[b])]] + [int(following[b])]
        for b in rows:
            assert int(count[b]) >= take
            assert emitted[b][:10] == want[b, :min(10, len(emitted[b]))].tolist()
        taken += 1
    assert taken >= 1


def test_prompt_scores_over_a_quantised_head():
    """As over a dense head: logits of the packed and the one-token path agree within 2e-2."""
    cfg, lens, K = SMALL, [300, 21, 1], 5
    model, prompts = quantised_head(cfg, 61), ragged(SMALL, lens, 62)
    steps = engine(cfg, model, len(lens), max_ctx=320)
    pad, logits = padded(prompts), []
    for t in range(pad.shape[1]):
        steps.tokens.copy_(pad[:, t].int().cuda())
        steps.pos.fill_(t)
        steps.run_step()
        logits.append(steps.logits.double().cpu())
    logits = torch.stack(logits, 1)
    eng = engine(cfg, model, len(lens), max_ctx=320)
    got = eng.prefill_packed(prompts, score=True, num_top=K)
    for b, n in enumerate(lens):
        s, logp = got.of(b), torch.log_softmax(logits[b, :n], -1)
        if n > 1:
            assert max_abs(s["logprob"], logp[:-1].gather(1, prompts[b][1:, None])[:, 0]) <= 4e-2
        assert max_abs(s["entropy"], -(logp.exp() * logp).sum(-1)) <= 4e-2 * (1 + np.log(cfg.vocab_size))
        assert max_abs(s["top_logprob"], logp.topk(K, -1).values) <= 4e-2
        top = logits[b, n - 1].topk(2).values
        if top[0] - top[1] > SURE:
            assert int(eng.next_tokens[b]) == int(logits[b, n - 1].argmax()) == int(s["top_index"][-1, 0])
