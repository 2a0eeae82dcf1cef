"""The serving operators at sizes, values and calls that their first tests do not reach."""

import math

import numpy as np
import pytest
import torch

from tests.serving_ref import assert_attention, attention_rows
from tests.test_gpu_serving import check_packed, gen, ints, randn
from torch2iron_b200.operators import DraftTreeAttention, DraftTreeCommit, PackedAttention, draft_tree

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


# ---------------------------------------------------------------------------
# scores so large that neighbouring fp32 values are units apart
# ---------------------------------------------------------------------------
def run_packed(q, k, v, scale):
    n, nh, hd = q.shape
    nkv = k.shape[1]
    out, lse = torch.empty_like(q), torch.empty(n, nh, device="cuda")
    PackedAttention(tokens=n, num_seqs=1, num_kv_groups=nkv, q_heads_per_group=nh // nkv, head_dim=hd, dtype=q.dtype,
                    scale=scale)(q, k, v, ints([0, n]), out, lse=lse)
    return out, lse


@pytest.mark.parametrize("size", [2.0 ** 20, 2.0 ** 24, 3e7, 6e7, 1.1e8, 2.0 ** 28, 7e8, 3e9])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_equal_scores_of_any_size_give_the_mean(size, dtype):
    """Equal keys: every weight is the same, whatever the scores' rounding, so row
    i is the mean of v[0..i]: a weight is at most half a step of its type off (u),
    the sum and the result's rounding as in ``assert_attention``."""
    n, hd = 300, 64
    a = math.sqrt(size * math.log(2.0))                       # scores of about size in powers of two
    q = torch.zeros(n, 2, hd, device="cuda", dtype=dtype)
    q[:, :, :3] = torch.tensor([a, a / 700, -a / 900])
    q[::2] *= -1
    k = torch.zeros(n, 1, hd, device="cuda", dtype=dtype)
    k[:, :, :3] = torch.tensor([a, a / 3, a / 7])
    v = randn(gen(1), n, 1, hd, dtype=dtype)
    out, lse = run_packed(q, k, v, 1.0)
    u = torch.finfo(dtype).eps / 2
    i = torch.arange(1, n + 1, dtype=torch.float64)[:, None, None]
    mean = v.double().cpu().cumsum(0) / i
    off = v.double().cpu().abs().cumsum(0) / i * (u + (300 + 4) * 2.0 ** -24)
    got = out.double().cpu()
    assert torch.isfinite(got).all() and torch.isfinite(lse).all()
    assert ((got - mean).abs() <= off + u * (mean.abs() + off).clamp(min=torch.finfo(dtype).tiny) + 2.0 ** -30).all()


@pytest.mark.parametrize("base,step", [(2.0 ** 24, 2.0), (2.0 ** 25, 4.0), (2.0 ** 26, 8.0), (2.0 ** 27, 16.0),
                                       (-(2.0 ** 27), 16.0), (2.0 ** 28, 32.0)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_scores_that_rise_by_their_own_spacing(base, step, dtype):
    """Scores base + step * (block of 128 keys), exact in fp32, in powers of two:
    the reference of the exponents has to follow a rise that its own rounding
    nearly hides.  The weights are powers of two, so only sums and the result round."""
    n, hd = 700, 64
    scale = float(np.float32(math.log(2.0)))
    assert np.float32(scale) * np.float32(1.4426950408889634) == 1.0
    q = torch.zeros(n, 1, hd)
    k = torch.zeros(n, 1, hd)
    q[:, 0, 0], k[:, 0, 0] = 2.0 ** 14, base / 2.0 ** 14
    q[:, 0, 1] = step
    block = torch.arange(n) // 128
    k[:, 0, 1] = block.float()
    q, k, v = q.to(dtype).cuda(), k.to(dtype).cuda(), randn(gen(2), n, 1, hd, dtype=dtype)
    out, _ = run_packed(q, k, v, scale)
    w = torch.exp2(step * (block[None] - block[:, None]).double()).tril()
    want = (w @ v[:, 0].double().cpu()) / w.sum(1, keepdim=True)
    size = (w @ v[:, 0].double().cpu().abs()) / w.sum(1, keepdim=True)
    u = torch.finfo(dtype).eps / 2
    off = size * (700 + 8) * 2.0 ** -24 + (2.0 ** -32 * 700 if dtype == HF else 0.0) * 8
    got = out[:, 0].double().cpu()
    assert torch.isfinite(got).all()
    assert ((got - want).abs() <= off + u * (want.abs() + off).clamp(min=torch.finfo(dtype).tiny) + 2.0 ** -30).all()


@pytest.mark.parametrize("dtype,q_scale", [(HF, 3000.0), (BF, 1e4), (BF, 1e6)])
def test_huge_random_scores_stay_inside_the_values(dtype, q_scale):
    """Scores whose own rounding exceeds a power of two: which key wins is open, the result is finite and between
    the least and the largest value seen."""
    n, hd = 500, 128
    q, k = randn(gen(3), n, 4, hd, dtype=dtype, scale=q_scale), randn(gen(4), n, 2, hd, dtype=dtype, scale=q_scale)
    v = randn(gen(5), n, 2, hd, dtype=dtype)
    out, lse = run_packed(q, k, v, 1.0)
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()
    low, high = (f(v.float(), 0).values.repeat_interleave(2, 1) for f in (torch.cummin, torch.cummax))
    slack = 2 * torch.finfo(dtype).eps * v.float().abs().max()
    assert (out.float() >= low - slack).all() and (out.float() <= high + slack).all()


@pytest.mark.parametrize("size", [2.0 ** 20, 1.1e8, 3e9])
@pytest.mark.parametrize("ctx", [100, 5000])
def test_equal_scores_of_any_size_over_a_cache(size, ctx):
    """The same for a tree whose items have one tile and are cut between CTAs: bounds as above."""
    T, hd, a = 20, 64, math.sqrt(size * math.log(2.0))
    one = torch.tensor([a, a / 3, a / 7])
    q, k, v = torch.zeros(1, T, 2, hd), torch.zeros(1, 1, 5056, hd), randn(gen(6), 1, 1, 5056, hd, dtype=HF)
    q[..., :3], k[..., :3] = one, one
    q[:, ::3] *= -1
    q, k = q.half().cuda(), k.half().cuda()
    kd, vd = k[:, :, :T].transpose(1, 2).contiguous(), randn(gen(7), 1, T, 1, hd, dtype=HF)
    mask, _ = draft_tree(np.arange(-1, T - 1)[None])
    out, lse = torch.empty_like(q), torch.empty(1, T, 2, device="cuda")
    DraftTreeAttention(batch=1, nodes=T, max_ctx=5056, num_kv_groups=1, q_heads_per_group=2, dtype=HF, scale=1.0)(
        q, k, v, kd, vd, ints([ctx]), mask.cuda(), out, lse=lse)
    seen = torch.cat([v[0, 0, :ctx], vd[0, :, 0]]).double().cpu()
    n = torch.arange(ctx + 1, ctx + T + 1, dtype=torch.float64)[:, None]
    mean, size_of = seen.cumsum(0)[ctx:] / n, seen.abs().cumsum(0)[ctx:] / n
    u = 2.0 ** -11
    off = size_of * (u + (ctx + 40) * 2.0 ** -24)
    got = out[0].double().cpu()
    assert torch.isfinite(lse).all()
    assert ((got - mean[:, None]).abs() <= (off + u * (mean.abs() + off).clamp(min=2.0 ** -14) + 2.0 ** -30)[:, None]).all()


# ---------------------------------------------------------------------------
# many sequences
# ---------------------------------------------------------------------------
def test_packed_half_a_million_tokens_of_short_prompts():
    """32768 prompts of 16 tokens over 8 key heads: some of them against the reference, each row finite."""
    S, n, nh, hd = 32768, 16, 8, 64
    g = torch.Generator(device="cuda").manual_seed(8)
    q, k, v = (torch.randn(S * n, nh, hd, generator=g, device="cuda").to(BF) for _ in range(3))
    out, lse = torch.full_like(q, math.nan), torch.full((S * n, nh), math.nan, device="cuda")
    op = PackedAttention(tokens=S * n, num_seqs=S, num_kv_groups=nh, q_heads_per_group=1, head_dim=hd)
    op(q, k, v, torch.arange(0, S * n + 1, n, dtype=torch.int32, device="cuda"), out, lse=lse)
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()
    seen = torch.arange(n)[None] <= torch.arange(n)[:, None]
    for s in (0, 1, 639, 640, 641, 10007, S - 1):
        r = slice(s * n, (s + 1) * n)
        assert_attention(out[r], lse[r], attention_rows(q[r], k[r], v[r], seen, op.scale))


# ---------------------------------------------------------------------------
# results over inputs
# ---------------------------------------------------------------------------
def test_attention_in_place_of_q_gives_the_same_bits():
    g, n, nh, nkv, hd = gen(60), [700, 1, 90, 1500], 8, 2, 64
    total, start = sum(n), np.concatenate([[0], np.cumsum(n)])
    fused = randn(g, total, nh + 2 * nkv, hd)
    q, k, v = fused[:, :nh], fused[:, nh:nh + nkv], fused[:, nh + nkv:]
    op = PackedAttention(tokens=total, num_seqs=4, num_kv_groups=nkv, q_heads_per_group=4, head_dim=hd)
    out, keys = torch.empty(total, nh, hd, dtype=BF, device="cuda"), fused[:, nh:].clone()
    op(q, k, v, ints(start), out)
    op(q, k, v, ints(start), q)
    assert torch.equal(q, out) and torch.equal(fused[:, nh:], keys)
    B, T = 2, 40
    q, kd, vd = randn(g, B, T, nh, hd), randn(g, B, T, nkv, hd), randn(g, B, T, nkv, hd)
    kc, vc = randn(g, B, nkv, 4096, hd), randn(g, B, nkv, 4096, hd)
    mask, _ = draft_tree(np.tile(np.arange(-1, T - 1), (B, 1)))
    op = DraftTreeAttention(batch=B, nodes=T, max_ctx=4096, num_kv_groups=nkv, q_heads_per_group=4, head_dim=hd)
    out = torch.empty_like(q)
    op(q, kc, vc, kd, vd, ints([4000, 10]), mask.cuda(), out)
    op(q, kc, vc, kd, vd, ints([4000, 10]), mask.cuda(), q)
    assert torch.equal(q, out)


def test_results_over_inputs_are_refused():
    g, n, nkv, hd = gen(61), 6, 2, 64
    buf = randn(g, n, 4 + nkv + 1, hd)
    op = PackedAttention(tokens=n, num_seqs=1, num_kv_groups=nkv, q_heads_per_group=2, head_dim=hd)
    q, v = randn(g, n, 4, hd), randn(g, n, nkv, hd)
    with pytest.raises(RuntimeError, match="argument"):
        op(q, buf[:, :nkv], v, ints([0, n]), buf[:, 1:5])
    op(q, buf[:, :nkv], v, ints([0, n]), buf[:, nkv:nkv + 4])
    cache, draft = randn(g, 2, 1, nkv, 64, hd), randn(g, 1, 1, 3, nkv, hd)
    commit = DraftTreeCommit(layers=1, batch=1, nodes=3, max_ctx=64, num_kv_groups=nkv, head_dim=hd)
    tree, row = [ints([[0, 0, 0]]) for _ in range(4)], [ints([0]) for _ in range(4)]
    inside = cache[0:1, :, :, 10:13].transpose(2, 3)
    for kd, kc in ((inside, cache[0:1]), (draft, cache[1:2])):
        with pytest.raises(RuntimeError, match="argument"):
            commit(*tree[:3], row[0], kd, draft, kc, cache[1:2], tree[3], *row[1:])
    commit(*tree[:3], row[0], draft, draft, cache[0:1], cache[1:2], tree[3], *row[1:])


@pytest.mark.parametrize("S,long", [(640, ()), (641, (0, 640)), (1500, (639, 640, 1281)), (1500, (1499,))])
def test_packed_more_sequences_than_threads(S, long):
    """The list's start is counted 640 sequences at a time: empty ones beside that
    border, and some long enough to be cut between CTAs."""
    n = [(i * 7) % 4 for i in range(S)]
    for i in (638, 639, 640, 641, 1279, 1280):
        if i < S:
            n[i] = 0
    for i in long:
        n[i] = 3000
    check_packed(n, (2, 1, 64), extra_rows=5)


def test_packed_one_prompt_of_more_pairs_than_half_the_threads():
    """128 query heads on one key head make a pair of two tokens: each thread looks for a cut in several pairs."""
    check_packed([3, 1500, 0, 700], (128, 1, 64), extra_rows=1)


def test_packed_one_prompt_of_more_than_20480_tokens():
    """The same with 4 query heads per key head (64 tokens a pair); the reference of some rows."""
    n, nh, nkv, hd = 22001, 4, 1, 64
    g = gen(70)
    q, k, v = randn(g, n, nh, hd, scale=1.5), randn(g, n, nkv, hd), randn(g, n, nkv, hd)
    out, lse = torch.full_like(q, math.nan), torch.full((n, nh), math.nan, device="cuda")
    op = PackedAttention(tokens=n, num_seqs=1, num_kv_groups=nkv, q_heads_per_group=nh, head_dim=hd)
    op(q, k, v, ints([0, n]), out, lse=lse)
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()
    rows = torch.tensor([0, 63, 64, 127, 128, 5000, 10239, 10240, 20479, 20480, 20543, 20544, 21951, 21952, 22000])
    seen = torch.arange(n)[None] <= rows[:, None]
    assert_attention(out[rows], lse[rows], attention_rows(q[rows], k, v, seen, op.scale))


def test_calls_without_any_row_write_nothing():
    g, nkv, hd = gen(71), 2, 64
    q, kv = randn(g, 9, 4, hd), randn(g, 9, nkv, hd)
    for S in (1, 5, 700):
        op = PackedAttention(tokens=9, num_seqs=S, num_kv_groups=nkv, q_heads_per_group=2, head_dim=hd)
        for start in (0, 4, 9):
            out, lse = torch.full_like(q, 7.0), torch.full((9, 4), 7.0, device="cuda")
            op(q, kv, kv, ints([start] * (S + 1)), out, lse=lse)
            assert (out == 7).all() and (lse == 7).all()
    B, T = 3, 5
    q, kd, cache = randn(g, B, T, 4, hd), randn(g, B, T, nkv, hd), randn(g, B, nkv, 64, hd)
    out, lse = torch.full_like(q, 7.0), torch.full((B, T, 4), 7.0, device="cuda")
    mask = torch.ones(B, T, 1, dtype=torch.int64, device="cuda")
    op = DraftTreeAttention(batch=B, nodes=T, max_ctx=64, num_kv_groups=nkv, q_heads_per_group=2, head_dim=hd)
    for live in ([0, 0, 0], [-3, 0, -1]):
        op(q, cache, cache, kd, kd, ints([64, 0, 9]), mask, out, num_nodes=ints(live), lse=lse)
        assert (out == 7).all() and (lse == 7).all()


def test_packed_starts_outside_the_tensors_are_clamped_to_their_rows():
    """The rows that the clamped starts leave have their values, the others are not written."""
    g, nkv, hd = gen(72), 2, 64
    q, k, v = randn(g, 10, 4, hd), randn(g, 40, nkv, hd), randn(g, 40, nkv, hd)
    op = PackedAttention(tokens=10, num_seqs=3, num_kv_groups=nkv, q_heads_per_group=2, head_dim=hd, kv_tokens=40)
    out, lse = torch.full_like(q, math.nan), torch.full((10, 4), math.nan, device="cuda")
    op(q, k, v, ints([-5, 2, 2, 2000000000]), out, k_start=ints([0, 3, 5]), k_len=ints([7, 1, 9]), lse=lse)
    for rows, n, first, k_len in ((slice(0, 2), 2, 0, 7), (slice(2, 10), 8, 5, 9)):
        seen = torch.arange(k_len)[None] <= k_len - n + torch.arange(n)[:, None]
        keys = slice(first, first + k_len)
        assert_attention(out[rows], lse[rows], attention_rows(q[rows], k[keys], v[keys], seen, op.scale))
    out.fill_(7.0)
    op(q, k, v, ints([4, 4, 6, 6]), out, k_start=ints([0, 30, 0]), k_len=ints([7, 2000000000, 9]), lse=lse)
    assert (out[:4] == 7).all() and (out[6:] == 7).all()
    assert_attention(out[4:6], None, attention_rows(q[4:6], k[30:], v[30:], torch.ones(2, 10, dtype=torch.bool), op.scale))


def test_commit_of_fp16_caches():
    g, L, B, T, nkv, hd, ctx = gen(73), 3, 2, 6, 2, 128, 64
    kd, vd = randn(g, L, B, T, nkv, hd, dtype=HF), randn(g, L, B, T, nkv, hd, dtype=HF)
    kc, vc = randn(g, L, B, nkv, ctx, hd, dtype=HF), randn(g, L, B, nkv, ctx, hd, dtype=HF)
    want = [kc.clone(), vc.clone()]
    parents, tokens, predicted = [[-1, 0, 1, 1, 3, 4]] * 2, [[9, 1, 2, 3, 4, 5]] * 2, [[1, 3, 0, 4, 5, 8], [7] * 6]
    out = [ints([[0] * T] * B)] + [ints([0] * B) for _ in range(3)]
    DraftTreeCommit(layers=L, batch=B, nodes=T, max_ctx=ctx, num_kv_groups=nkv, head_dim=hd, dtype=HF)(
        ints(tokens), ints(parents), ints(predicted), ints([20, 63]), kd, vd, kc, vc, *out)
    paths = [[0, 1, 3, 4, 5], [0]]
    for b, at in ((0, 20), (1, 63)):
        for i, n in enumerate(paths[b]):
            want[0][:, b, :, at + i], want[1][:, b, :, at + i] = kd[:, b, n], vd[:, b, n]
        assert out[0][b].tolist() == paths[b] + [-1] * (T - len(paths[b]))
    assert out[2].tolist() == [8, 7] and out[3].tolist() == [25, 64]
    assert torch.equal(kc, want[0]) and torch.equal(vc, want[1])
    with pytest.raises(ValueError):
        DraftTreeCommit(layers=L, batch=B, nodes=T, max_ctx=ctx, num_kv_groups=nkv, head_dim=hd)(
            ints(tokens), ints(parents), ints(predicted), ints([20, 63]), kd, vd, kc, vc, *out)
