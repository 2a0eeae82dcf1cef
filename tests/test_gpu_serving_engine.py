"""The engine's serving paths on the GPU: packed prefill against the padded one,
prompt scores against the logits of one-token steps, draft trees against plain
greedy decoding, and all of it in one loop."""

import numpy as np
import pytest
import torch

from tests.gpu_util import max_abs, oracle_decoder
from torch2iron_b200 import synth
from torch2iron_b200.config import QuantizedQwenConfig
from torch2iron_b200.engine import DecodeEngine

pytestmark = pytest.mark.gpu

SMALL = QuantizedQwenConfig(vocab_size=512, emb_dim=256, n_layers=2, n_heads=4, n_kv_groups=2, head_dim=64,
                            hidden_dim=512, rms_norm_eps=1e-6, rope_base=1e6)
WIDE = QuantizedQwenConfig(vocab_size=640, emb_dim=512, n_layers=2, n_heads=8, n_kv_groups=2, head_dim=128,
                           hidden_dim=768, rms_norm_eps=1e-6, rope_base=1e6, tie_word_embeddings=False)
SURE = 4e-2          # top-2 margin above which two paths within the 2e-2 logit bar pick the same token


def ragged(cfg, lens, seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, cfg.vocab_size, (n,), generator=g) for n in lens]


def padded(prompts):
    out = torch.zeros(len(prompts), max(len(t) for t in prompts), dtype=torch.int64)
    for b, t in enumerate(prompts):
        out[b, :len(t)] = t
    return out


def engine(cfg, model, batch, max_ctx=128, **kw):
    return DecodeEngine(cfg, model, batch=batch, max_ctx=max_ctx, use_graph=False, **kw)


@pytest.mark.parametrize("cfg,lens,chunk", [(SMALL, [5, 37, 1, 64], None), (SMALL, [5, 37, 1, 64], 16),
                                            (SMALL, [90, 2, 33], 7), (WIDE, [100, 3, 128, 60, 77], None),
                                            (WIDE, [1], None), (SMALL, [128] * 4, 300)])
def test_prefill_packed_matches_the_padded_prefill(cfg, lens, chunk):
    model = synth.random_model(cfg, seed=51)
    prompts = ragged(cfg, lens, 52)
    a = engine(cfg, model, len(lens))
    a.prefill(padded(prompts), lengths=lens)
    b = engine(cfg, model, len(lens))
    assert b.prefill_packed(prompts, chunk_rows=chunk) is None
    torch.cuda.synchronize()
    assert int(b.err.item()) == 0
    for li in range(cfg.n_layers):
        for r, n in enumerate(lens):
            assert max_abs(a.k_cache[li][r, :, :n], b.k_cache[li][r, :, :n]) <= 5e-2
            assert max_abs(a.v_cache[li][r, :, :n], b.v_cache[li][r, :, :n]) <= 5e-2
            assert (b.k_cache[li][r, :, n:] == 0).all() and (b.v_cache[li][r, :, n:] == 0).all()
    assert max_abs(a.logits, b.logits) <= 2e-2
    assert b.pos.tolist() == lens
    top = a.logits.topk(2, dim=-1).values
    sure = (top[:, 0] - top[:, 1]) > SURE
    assert torch.equal(a.next_tokens[sure], b.next_tokens[sure]) and torch.equal(b.tokens, b.next_tokens)
    if max(lens) < 128:
        b.tokens.copy_(a.tokens)
        a.advance()
        b.advance()
        assert max_abs(a.logits, b.logits) <= 2e-2


@pytest.mark.parametrize("cfg,lens,chunk,K", [(SMALL, [9, 30, 1], None, 4), (WIDE, [70, 2, 21], 40, 0),
                                              (SMALL, [128, 128, 127], None, 32)])
def test_prompt_scores_match_stepwise_logits(cfg, lens, chunk, K):
    """Logits of the two paths agree within 2e-2, so a log probability (a logit
    and a log-sum of logits) and a top value within 4e-2; the entropy moves by
    at most sum p |dlog p| (1 + |log p|) <= 4e-2 (1 + log V)."""
    model = synth.random_model(cfg, seed=61)
    prompts = ragged(cfg, lens, 62)
    steps = engine(cfg, model, len(lens))
    pad = padded(prompts)
    logits = []
    for t in range(pad.shape[1]):
        steps.tokens.copy_(pad[:, t].int().cuda())
        steps.pos.fill_(t)
        steps.run_step()
        logits.append(steps.logits.double().cpu())
    logits = torch.stack(logits, 1)                                     # [B, P, V]
    eng = engine(cfg, model, len(lens), keep_logits=False)
    got = eng.prefill_packed(prompts, score=True, num_top=K, chunk_rows=chunk)
    assert got.lengths == lens
    for b, n in enumerate(lens):
        s = got.of(b)
        logp = torch.log_softmax(logits[b, :n], -1)
        assert s["logprob"].shape == (n - 1,) and s["entropy"].shape == (n,)
        if n > 1:
            want = logp[:-1].gather(1, prompts[b][1:, None])[:, 0]
            assert max_abs(s["logprob"], want) <= 4e-2
        ent = -(logp.exp() * logp).sum(-1)
        assert max_abs(s["entropy"], ent) <= 4e-2 * (1 + np.log(cfg.vocab_size))
        if K:
            ref = logp.topk(K, -1)
            assert max_abs(s["top_logprob"], ref.values) <= 4e-2
            picked = logp.gather(1, s["top_index"].long().cpu())
            assert max_abs(picked, ref.values) <= 8e-2               # what it picked is as likely as the best
        else:
            assert s["top_logprob"] is None and s["top_index"] is None
    at = np.cumsum(lens) - 1
    assert torch.isnan(got.logprob[at]).all()                           # a prompt's last token has no successor in it


def greedy(cfg, model, prompts, steps, max_ctx=128):
    """Plain greedy tokens [B, steps], and per row the steps whose margin is sure up to the first that is not."""
    eng = engine(cfg, model, len(prompts), max_ctx)
    eng.prefill(padded(prompts), lengths=[len(t) for t in prompts])
    toks, sure = [], []
    for i in range(steps):
        if i:
            eng.advance()
        top = eng.logits.topk(2, -1).values
        toks.append(eng.next_tokens.cpu().clone())
        sure.append(((top[:, 0] - top[:, 1]) > SURE).cpu())
    return torch.stack(toks, 1), torch.stack(sure, 1).int().cumprod(1).sum(1).tolist(), eng


def drafts(rng, chain, T, vocab):
    """A tree per row that holds ``chain[b]`` (the pending token first) as one branch among random nodes."""
    B = len(chain)
    tok = rng.integers(0, vocab, (B, T))
    par = np.array([[-1] + [rng.integers(0, i) for i in range(1, T)] for _ in range(B)])
    for b, c in enumerate(chain):
        at = np.concatenate([[0], 1 + np.sort(rng.choice(T - 1, len(c) - 1, replace=False))]) if len(c) > 1 else np.array([0])
        tok[b, at], par[b, at[1:]] = c, at[:-1]
    return tok, par


@pytest.mark.parametrize("cfg,lens,T,take", [(SMALL, [5, 37, 1], 6, 3), (WIDE, [30, 2, 17, 60], 20, 5),
                                             (SMALL, [9], 1, 1), (SMALL, [3, 11], 100, 8), (WIDE, [40] * 3, 130, 2)])
def test_decode_tree_emits_the_greedy_tokens(cfg, lens, T, take):
    """Trees that hold the true continuation among wrong drafts: every accepted
    token is the plain decoder's, and the true branch is accepted as far as the
    plain decoder's picks are sure."""
    model, rng, steps = synth.random_model(cfg, seed=71), np.random.default_rng(72), 24
    prompts = ragged(cfg, lens, 73)
    want, sure, plain = greedy(cfg, model, prompts, steps)
    eng = engine(cfg, model, len(lens))
    eng.prefill_packed(prompts)
    B = len(lens)
    emitted = [[int(t)] for t in eng.next_tokens.cpu()]
    good = [sure[b] > 0 and emitted[b][0] == int(want[b, 0]) for b in range(B)]
    assert all(good[b] or sure[b] == 0 for b in range(B))
    for _ in range(4):
        n = [len(e) for e in emitted]
        if max(n) + take >= steps:
            break
        chain = [want[b, n[b] - 1:n[b] - 1 + take].tolist() for b in range(B)]
        for b in range(B):
            chain[b][0] = emitted[b][-1]
        tok, par = drafts(rng, chain, T, cfg.vocab_size)
        path, count, following = eng.decode_tree(tok, par)
        for b in range(B):
            k = int(count[b])
            walk = path[b, :k].tolist()
            assert k >= 1 and walk[0] == 0 and path[b, k:].eq(-1).all()
            assert all(par[b, y] == x for x, y in zip(walk, walk[1:]))
            emitted[b] += [int(tok[b, i]) for i in walk[1:]] + [int(following[b])]
            m = min(len(emitted[b]), sure[b])
            assert emitted[b][:m] == want[b, :m].tolist()
            if n[b] - 1 + take < sure[b]:
                assert k >= take                        # the whole true branch (or a longer lucky one)
        assert eng.pos.tolist() == [lens[b] + len(emitted[b]) - 1 for b in range(B)]
        assert eng.tokens.tolist() == [e[-1] for e in emitted]
    # the caches hold what plain decoding of the same tokens writes
    for b in range(B):
        m = lens[b] + min(len(emitted[b]) - 1, sure[b] - 1)
        for li in range(cfg.n_layers):
            if m > lens[b]:
                assert max_abs(eng.k_cache[li][b, :, :m], plain.k_cache[li][b, :, :m]) <= 5e-2
                assert max_abs(eng.v_cache[li][b, :, :m], plain.v_cache[li][b, :, :m]) <= 5e-2


def test_decode_tree_of_one_node_is_a_decode_step():
    cfg, lens = SMALL, [7, 20]
    model, prompts = synth.random_model(cfg, seed=81), ragged(SMALL, [7, 20], 82)
    a, b = engine(cfg, model, 2), engine(cfg, model, 2)
    for e in (a, b):
        e.prefill_packed(prompts)
    b.tokens.copy_(a.tokens)
    tok = a.tokens.cpu()[:, None]
    path, count, following = a.decode_tree(tok, torch.full((2, 1), -1))
    b.advance()
    top = b.logits.topk(2, -1).values.cpu()
    sure = (top[:, 0] - top[:, 1]) > SURE
    assert count.tolist() == [1, 1] and torch.equal(following[sure], b.next_tokens.cpu()[sure])
    for li in range(cfg.n_layers):
        for r, n in enumerate(lens):
            assert max_abs(a.k_cache[li][r, :, :n + 1], b.k_cache[li][r, :, :n + 1]) <= 5e-2


def test_serving_paths_between_captured_steps():
    """Packed prefill, captured one-token steps and draft trees share the engine's state in any order."""
    cfg, model = SMALL, synth.random_model(SMALL, seed=101)
    prompts = ragged(cfg, [6, 25, 40], 102)
    states = []
    for graph in (False, True):
        eng = DecodeEngine(cfg, model, batch=3, max_ctx=128, use_graph=graph)
        eng.prefill_packed(prompts)
        log = [eng.next_tokens.tolist()]
        for _ in range(2):
            eng.advance()
            log.append(eng.next_tokens.tolist())
            tok = np.stack([eng.tokens.cpu().numpy(), np.full(3, 7), np.full(3, 9)], 1)
            log += [t.tolist() for t in eng.decode_tree(tok, np.tile([-1, 0, 0], (3, 1)))]
        eng.prefill_packed(prompts, score=True)               # and again over the same caches
        log.append(eng.next_tokens.tolist())
        eng.advance()
        log.append(eng.pos.tolist())
        states.append(log)
        eng.release()
    assert states[0] == states[1] and states[0][0] == states[0][-2]


def test_decode_tree_dead_and_full_rows_stay():
    cfg, model = SMALL, synth.random_model(SMALL, seed=91)
    eng = engine(cfg, model, 3, max_ctx=64)
    eng.prefill_packed(ragged(cfg, [10, 64, 63], 92))
    before = [t.clone() for t in (eng.tokens, eng.pos)]
    caches = [t.clone() for t in eng.k_cache]
    tok = np.repeat(eng.tokens.cpu().numpy()[:, None], 4, 1)
    path, count, following = eng.decode_tree(tok, np.tile([-1, 0, 1, 2], (3, 1)), num_nodes=[0, 4, 4])
    assert count.tolist()[:2] == [0, 0] and int(count[2]) == 1          # dead, full, room for the root alone
    assert eng.tokens[:2].equal(before[0][:2]) and eng.pos.tolist() == [10, 64, 64]
    assert following[:2].tolist() == [-1, -1] and path[:2].eq(-1).all()
    for a, b in zip(eng.k_cache, caches):
        assert torch.equal(a[:2], b[:2]) and torch.equal(a[2, :, :63], b[2, :, :63])


def test_decode_tree_takes_padded_trees():
    """Nodes behind num_nodes may hold any token and parent; a row's result does not depend on them."""
    cfg, model = SMALL, synth.random_model(SMALL, seed=93)
    prompts = ragged(cfg, [12, 30], 94)
    got = []
    for fill, T in ((-1, 6), (10 ** 6, 9)):
        eng = engine(cfg, model, 2)
        eng.prefill_packed(prompts)
        tok, par = np.full((2, T), fill), np.full((2, T), fill)
        tok[:, 0], par[:, 0] = eng.tokens.cpu().numpy(), -1
        tok[0, 1:3], par[0, 1:3] = [3, 4], [0, 1]
        path, count, following = eng.decode_tree(tok, par, num_nodes=torch.tensor([3, 1]))
        assert (path[0] < 3).all() and (path[1] < 1).all()
        got.append((count.tolist(), following.tolist(), eng.pos.tolist()))
    assert got[0] == got[1]


def test_packed_prefill_and_tree_refusals():
    eng = engine(SMALL, synth.random_model(SMALL, seed=95), 2, max_ctx=64)
    ok = [[1, 2, 3], [4]]
    for bad in ([[1]], [[1], []], [[1], [2] * 65], [[1], [512]], [[1], [-1]], [[1], [0.5]]):
        with pytest.raises(ValueError):
            eng.prefill_packed(bad)
    with pytest.raises(ValueError):
        eng.prefill_packed(ok, num_top=3)
    with pytest.raises(ValueError):
        eng.prefill_packed(ok, score=True, num_top=33)
    with pytest.raises(ValueError):
        eng.prefill_packed(ok, chunk_rows=-1)
    eng.prefill_packed(ok)
    for tok, par, live in (([[1, 2]], [[-1, 0]], None), ([[1, 2]] * 2, [[-1, 1]] * 2, None), ([[1, 512]] * 2, [[-1, 0]] * 2, None),
                           ([[1, 2]] * 2, [[-1, 0]] * 2, [1, 3]), ([[1]] * 2, [[-1, 0]] * 2, None),
                           ([[1] * 257] * 2, [[-1] + [0] * 256] * 2, None)):
        with pytest.raises(ValueError):
            eng.decode_tree(tok, par, live)


def test_scored_packed_prompt_agrees_with_the_oracle():
    """Last-position logits of the packed path against the fp32 oracle decoder."""
    cfg, model, lens = SMALL, synth.random_model(SMALL, seed=97), [21, 21]
    prompts = ragged(cfg, lens, 98)
    eng = engine(cfg, model, 2, max_ctx=64)
    got = eng.prefill_packed(prompts, score=True, num_top=1)
    ref = oracle_decoder(cfg, model, 2, 64).prefill(torch.stack(prompts))
    assert max_abs(eng.logits, ref) <= 2e-2
    logp = torch.log_softmax(ref.double(), -1)
    last = torch.stack([got.of(b)["top_logprob"][-1, 0] for b in range(2)])
    assert max_abs(last, logp.max(-1).values) <= 4e-2
