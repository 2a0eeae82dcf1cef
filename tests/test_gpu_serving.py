"""The serving operators on the GPU against plain 64-bit implementations:
ragged and empty sequences, head layouts, strides, garbage in unseen places,
masks that leave a row empty, graph replay, other streams, and a run of all
four as a speculative serving loop uses them."""

import math

import numpy as np
import pytest
import torch

from tests.serving_ref import assert_attention, attention_rows, commit_walk, logprob_rows
from torch2iron_b200.operators import (DraftTreeAttention, DraftTreeCommit, PackedAttention, TokenLogProbs,
                                       draft_tree)

pytestmark = pytest.mark.gpu

BF, HF, F32, I32 = torch.bfloat16, torch.float16, torch.float32, torch.int32


def ints(v):
    return torch.tensor(v, dtype=I32, device="cuda")


def randn(g, *shape, dtype=BF, scale=1.0):
    return (torch.randn(*shape, generator=g) * scale).to(dtype).cuda()


def gen(seed):
    return torch.Generator().manual_seed(seed)


# ---------------------------------------------------------------------------
# packed attention
# ---------------------------------------------------------------------------
def packed_ref(q, keys, n, k_len, scale):
    """keys(s) -> (k, v) [k_len, nkv, hd] of sequence s; concatenated references."""
    parts, at = [], 0
    for s, (a, m) in enumerate(zip(n, k_len)):
        k, v = keys(s)
        seen = torch.arange(max(m, 1))[None] <= m - a + torch.arange(a)[:, None]
        if m <= 0:
            seen[:] = False
            k = v = torch.zeros(1, *k.shape[1:], dtype=k.dtype)
        parts.append(attention_rows(q[at:at + a], k, v, seen, scale))
        at += a
    return tuple(torch.cat([p[i] for p in parts]) for i in range(4))


def check_packed(n, heads, dtype=BF, out_dtype=None, scale=None, q_scale=1.5, seed=0, extra_rows=3):
    nh, nkv, hd = heads
    g = gen(seed + sum(n))
    total = sum(n) + extra_rows
    q = randn(g, total, nh, hd, dtype=dtype, scale=q_scale)
    k, v = randn(g, total, nkv, hd, dtype=dtype), randn(g, total, nkv, hd, dtype=dtype)
    if extra_rows:                               # rows behind the last sequence: anything
        q[-extra_rows:], k[-extra_rows:], v[-extra_rows:] = math.nan, math.inf, math.nan
    start = np.concatenate([[0], np.cumsum(n)])
    op = PackedAttention(tokens=total, num_seqs=len(n), num_kv_groups=nkv, q_heads_per_group=nh // nkv, head_dim=hd,
                         dtype=dtype, out_dtype=out_dtype, scale=scale)
    out = torch.full((total, nh, hd), 7.0, dtype=out_dtype or dtype, device="cuda")
    lse = torch.full((total, nh), 7.0, device="cuda")
    op(q, k, v, ints(start), out, lse=lse)
    torch.cuda.synchronize()
    live = sum(n)
    assert (out[live:] == 7).all() and (lse[live:] == 7).all()
    ref = packed_ref(q, lambda s: (k[start[s]:start[s + 1]], v[start[s]:start[s + 1]]), n, n, op.scale)
    assert_attention(out[:live], lse[:live], ref)
    again = torch.full_like(out, 7.0)
    op(q, k, v, ints(start), again)
    assert torch.equal(out, again)               # the same bits every time, with and without lse


@pytest.mark.parametrize("n", [[1], [2], [1, 1, 1], [5, 130, 1, 64], [127, 128, 129], [300], [3, 0, 7, 0], [0, 0, 5],
                               [63, 64, 65, 66], [257, 2, 511]])
def test_packed_lengths(n):
    check_packed(n, (4, 2, 64))


@pytest.mark.parametrize("heads", [(1, 1, 64), (4, 4, 128), (3, 1, 128), (14, 2, 64), (16, 8, 128), (32, 8, 64),
                                   (32, 8, 128), (40, 1, 64), (128, 1, 128), (100, 1, 128), (5, 5, 64)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_packed_heads_and_types(heads, dtype):
    check_packed([37, 1, 150], heads, dtype)


@pytest.mark.parametrize("dtype,out_dtype", [(BF, HF), (HF, BF)])
def test_packed_out_types(dtype, out_dtype):
    check_packed([70, 3], (8, 2, 128), dtype, out_dtype)


@pytest.mark.parametrize("q_scale,scale", [(1.5, 1.0), (40.0, None), (1e-3, 0.01), (10.0, 1.0)])
def test_packed_scales(q_scale, scale):
    check_packed([190, 20], (4, 2, 128), scale=scale, q_scale=q_scale)


def test_packed_many_short_sequences():
    check_packed([1 + (i * 7) % 5 for i in range(300)], (4, 2, 64), extra_rows=0)


def test_packed_rising_and_falling_scores():
    """Scores that grow (or fall) along the keys, so that the running maximum moves at every step (or never)."""
    n, hd = 900, 64
    for sign in (1.0, -1.0):
        q = torch.zeros(n, 2, hd)
        q[:, :, 0] = 8.0
        k = torch.zeros(n, 1, hd)
        k[:, 0, 0] = sign * torch.linspace(0, 60, n)
        k = (k + 0.1 * torch.randn(n, 1, hd, generator=gen(3))).to(BF).cuda()
        q, v = q.to(BF).cuda(), randn(gen(4), n, 1, hd)
        out, lse = torch.empty_like(q), torch.empty(n, 2, device="cuda")
        op = PackedAttention(tokens=n, num_seqs=1, num_kv_groups=1, q_heads_per_group=2, head_dim=hd)
        op(q, k, v, ints([0, n]), out, lse=lse)
        assert_attention(out, lse, packed_ref(q, lambda s: (k, v), [n], [n], op.scale))


@pytest.mark.parametrize("n,k_len,heads", [([1, 1, 1], [1, 700, 64], (8, 2, 128)), ([3, 40, 1], [300, 40, 129], (4, 2, 64)),
                                           ([5, 2], [0, 1], (4, 2, 64)), ([6, 1, 4], [2, 0, 256], (4, 4, 128)),
                                           ([200, 1], [1000, 2049], (32, 8, 128)), ([1], [5000], (16, 8, 128))])
def test_packed_over_cache_rows(n, k_len, heads):
    """Suffixes, single tokens, rows without any key; everything behind k_len is NaN."""
    nh, nkv, hd = heads
    g = gen(sum(k_len))
    total, S, ctx = sum(n), len(n), -(-max(k_len) // 64) * 64 + 64
    q = randn(g, total, nh, hd, scale=1.5)
    k, v = randn(g, S, nkv, ctx, hd), randn(g, S, nkv, ctx, hd)
    for s, m in enumerate(k_len):
        k[s, :, m:], v[s, :, m:] = math.nan, math.nan
    out, lse = torch.full_like(q, 7.0), torch.full((total, nh), 7.0, device="cuda")
    op = PackedAttention(tokens=total, num_seqs=S, num_kv_groups=nkv, q_heads_per_group=nh // nkv, head_dim=hd,
                         max_ctx=ctx)
    op(q, k, v, ints(np.concatenate([[0], np.cumsum(n)])), out, k_len=ints(k_len), lse=lse)
    ref = packed_ref(q, lambda s: (k[s, :, :k_len[s]].transpose(0, 1), v[s, :, :k_len[s]].transpose(0, 1)), n, k_len,
                     op.scale)
    assert_attention(out, lse, ref)


def test_packed_keys_at_given_starts_shared_and_out_of_order():
    n, k_start, k_len = [4, 1, 30, 2], [50, 50, 0, 211], [90, 90, 30, 45]
    g, nkv, hd, nh = gen(9), 2, 128, 6
    q = randn(g, sum(n), nh, hd, scale=1.5)
    k, v = randn(g, 256, nkv, hd), randn(g, 256, nkv, hd)
    out, lse = torch.empty_like(q), torch.empty(sum(n), nh, device="cuda")
    op = PackedAttention(tokens=sum(n), num_seqs=4, num_kv_groups=nkv, q_heads_per_group=3, head_dim=hd, kv_tokens=256)
    op(q, k, v, ints(np.concatenate([[0], np.cumsum(n)])), out, k_start=ints(k_start), k_len=ints(k_len), lse=lse)
    ref = packed_ref(q, lambda s: (k[k_start[s]:k_start[s] + k_len[s]], v[k_start[s]:k_start[s] + k_len[s]]), n, k_len,
                     op.scale)
    assert_attention(out, lse, ref)


def test_packed_strided_views():
    """q, k and v as views of one fused tensor, k/v head-major, out inside a wider tensor."""
    n, nh, nkv, hd = [33, 100], 8, 2, 64
    total, g = sum(n), gen(21)
    fused = randn(g, total, nh + 2 * nkv, hd, scale=1.2)
    q, k, v = fused[:, :nh], fused[:, nh:nh + nkv], fused[:, nh + nkv:]
    start = np.concatenate([[0], np.cumsum(n)])
    wide = torch.full((total, nh + 3, 2 * hd), 7.0, dtype=BF, device="cuda")
    op = PackedAttention(tokens=total, num_seqs=2, num_kv_groups=nkv, q_heads_per_group=nh // nkv, head_dim=hd)
    out = wide[:, 1:1 + nh, hd:]
    op(q, k, v, ints(start), out)
    ref = packed_ref(q, lambda s: (k[start[s]:start[s + 1]], v[start[s]:start[s + 1]]), n, n, op.scale)
    assert_attention(out, None, ref)
    assert (wide[:, 0] == 7).all() and (wide[:, nh + 1:] == 7).all() and (wide[:, :, :hd] == 7).all()
    heads_first = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
    other = torch.empty_like(heads_first[0])
    op(*heads_first, ints(start), other)
    assert torch.equal(other, out)


@pytest.mark.parametrize("heads", [(4, 2, 64), (6, 2, 128), (5, 1, 64)])
def test_packed_results_do_not_depend_on_rows_outside(heads):
    """The same bits whatever lies in the rows before, between and behind the sequences' own."""
    nh, nkv, hd = heads
    g, n = gen(50), [700, 30, 260]
    total = sum(n) + 40
    q, k, v = randn(g, total, nh, hd, scale=4.0), randn(g, total, nkv, hd), randn(g, total, nkv, hd)
    op = PackedAttention(tokens=total, num_seqs=3, num_kv_groups=nkv, q_heads_per_group=nh // nkv, head_dim=hd)
    start, got = ints([0, 700, 730, 990]), []
    for fill in (0.0, 300.0, -math.inf, math.nan):
        q[990:] = fill
        out, lse = torch.empty_like(q), torch.empty(total, nh, device="cuda")
        op(q, k, v, start, out, lse=lse)
        got.append((out[:990].clone(), lse[:990].clone()))
    for out, lse in got[1:]:
        assert torch.equal(out, got[0][0]) and torch.equal(lse, got[0][1])


def test_packed_refusals_on_the_device():
    op = PackedAttention(tokens=4, num_seqs=1, num_kv_groups=2, q_heads_per_group=2, head_dim=64)
    q, kv, start = torch.zeros(4, 4, 64, dtype=BF, device="cuda"), torch.zeros(4, 2, 64, dtype=BF, device="cuda"), ints([0, 4])
    odd = torch.zeros(4 * 4 * 64 + 8, dtype=BF, device="cuda")
    for bad in (dict(q=odd[4:4 + 1024].view(4, 4, 64)), dict(k=kv[:1].expand(4, 2, 64)), dict(q_start=start.long()),
                dict(q=torch.zeros(4, 4, 128, dtype=BF, device="cuda")[:, :, ::2]), dict(out=q.float()),
                dict(k=torch.zeros(4, 2 * 64 + 4, dtype=BF, device="cuda")[:, :128].view(4, 2, 64)),
                dict(lse=torch.zeros(4, 4, dtype=BF, device="cuda")), dict(k_start=ints([0])), dict(k_len=ints([4])),
                dict(k_start=ints([0, 0]), k_len=ints([4, 4]))):
        args = dict(q=q, k=kv, v=kv, q_start=start, out=torch.zeros_like(q))
        args.update(bad)
        with pytest.raises(ValueError):
            op(**args)
    with pytest.raises(ValueError):
        PackedAttention(tokens=4, num_seqs=1, num_kv_groups=2, q_heads_per_group=2, head_dim=64, max_ctx=64)(
            q, torch.zeros(1, 2, 64, 64, dtype=BF, device="cuda"), torch.zeros(1, 2, 64, 64, dtype=BF, device="cuda"),
            start, torch.zeros_like(q))


def test_packed_lengths_outside_the_tensors_are_clamped():
    """Starts and lengths past the extents read nothing outside: the sequence ends with the tensor."""
    g, nkv, hd = gen(5), 2, 64
    q, k, v = randn(g, 10, 4, hd), randn(g, 40, nkv, hd), randn(g, 40, nkv, hd)
    op = PackedAttention(tokens=10, num_seqs=3, num_kv_groups=nkv, q_heads_per_group=2, head_dim=hd, kv_tokens=40)
    out, lse = torch.full_like(q, 7.0), torch.full((10, 4), 7.0, device="cuda")
    op(q, k, v, ints([0, 2, 4, 6]), out, k_start=ints([30, 50, -9]), k_len=ints([2000000000, 10, 5]), lse=lse)
    assert (out[6:] == 7).all()
    # sequence 0: queries 0 and 1 see keys up to 2e9 - 2 + i, of which the 10 from row 30 on exist
    ref = attention_rows(q[:2], k[30:], v[30:], torch.ones(2, 10, dtype=torch.bool), op.scale)
    assert_attention(out[:2], lse[:2], ref)
    assert (out[2:6] == 0).all() and torch.isneginf(lse[2:6]).all()      # starts outside: no keys
    out.fill_(7.0)
    op(q, k, v, ints([-5, 2, 1, 2000000000]), out, k_start=ints([0, 0, 0]), k_len=ints([7, 1, 9]))
    assert torch.isfinite(out.float()).all()


def test_packed_graph_replay_with_other_lengths_and_another_stream():
    g, nh, nkv, hd, total = gen(13), 8, 2, 128, 600
    q, k, v = randn(g, total, nh, hd, scale=1.5), randn(g, total, nkv, hd), randn(g, total, nkv, hd)
    start = ints([0, 10, 300, 600])
    op = PackedAttention(tokens=total, num_seqs=3, num_kv_groups=nkv, q_heads_per_group=4, head_dim=hd)
    out = torch.full_like(q, 7.0)
    op(q, k, v, start, out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        op(q, k, v, start, out)
    for n in ([10, 290, 300], [600, 0, 0], [1, 1, 500]):
        start.copy_(ints(np.concatenate([[0], np.cumsum(n)])))
        out.fill_(7.0)
        graph.replay()
        eager = torch.full_like(q, 7.0)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            op(q, k, v, start, eager)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        at = np.concatenate([[0], np.cumsum(n)])
        ref = packed_ref(q, lambda s: (k[at[s]:at[s + 1]], v[at[s]:at[s + 1]]), n, n, op.scale)
        assert_attention(out[:sum(n)], None, ref)
        assert (out[sum(n):] == 7).all()


def test_packed_two_streams_at_once():
    g, nh, nkv, hd = gen(31), 8, 2, 64
    jobs = []
    for n in ([400, 3], [77, 800]):
        total = sum(n)
        q, k, v = randn(g, total, nh, hd), randn(g, total, nkv, hd), randn(g, total, nkv, hd)
        op = PackedAttention(tokens=total, num_seqs=2, num_kv_groups=nkv, q_heads_per_group=4, head_dim=hd)
        start = ints([0, n[0], total])
        alone = torch.empty_like(q)
        op(q, k, v, start, alone)
        jobs.append((op, q, k, v, start, torch.empty_like(q), alone, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(20):
        for op, q, k, v, start, out, _, st in jobs:
            with torch.cuda.stream(st):
                op(q, k, v, start, out)
    torch.cuda.synchronize()
    for *_, out, alone, _ in jobs:
        assert torch.equal(out, alone)


# ---------------------------------------------------------------------------
# tree attention
# ---------------------------------------------------------------------------
def random_mask(rng, B, T, live, empty_row=False):
    bits = np.tril(rng.random((B, T, T)) < 0.4)
    for b in range(B):
        np.fill_diagonal(bits[b], True)
    if empty_row:
        bits[:, min(1, T - 1)] = False
    words = (T + 63) // 64
    wide = np.ones((B, T, words * 64), np.uint8)            # bits of nodes that do not exist are set as well
    wide[:, :, :T] = bits
    packed = np.packbits(wide, axis=2, bitorder="little").view("<i8").reshape(B, T, words).copy()
    return torch.from_numpy(bits), torch.from_numpy(packed).cuda()


def check_tree(B, T, ctx, heads, live=None, dtype=BF, max_ctx=None, empty_row=False, head_major=False, seed=0):
    nh, nkv, hd = heads
    g, rng = gen(seed + T), np.random.default_rng(seed + T)
    max_ctx = max_ctx or -(-max(max(ctx), 1) // 64) * 64
    q = randn(g, B, T, nh, hd, dtype=dtype, scale=1.5)
    kc, vc = randn(g, B, nkv, max_ctx, hd, dtype=dtype), randn(g, B, nkv, max_ctx, hd, dtype=dtype)
    kd, vd = randn(g, B, T, nkv, hd, dtype=dtype), randn(g, B, T, nkv, hd, dtype=dtype)
    if head_major:
        kd, vd = (t.permute(2, 0, 1, 3).contiguous().permute(1, 2, 0, 3) for t in (kd, vd))
    nodes = live or [T] * B
    for b in range(B):
        kc[b, :, ctx[b]:], vc[b, :, ctx[b]:] = math.nan, math.nan
        kd[b, nodes[b]:], vd[b, nodes[b]:] = math.inf, math.nan
    bits, mask = random_mask(rng, B, T, live, empty_row)
    op = DraftTreeAttention(batch=B, nodes=T, max_ctx=max_ctx, num_kv_groups=nkv, q_heads_per_group=nh // nkv,
                            head_dim=hd, dtype=dtype)
    out, lse = torch.full_like(q, 7.0), torch.full((B, T, nh), 7.0, device="cuda")
    op(q, kc, vc, kd, vd, ints(ctx), mask, out, num_nodes=None if live is None else ints(live), lse=lse)
    torch.cuda.synchronize()
    for b in range(B):
        m = nodes[b]
        assert (out[b, m:] == 7).all() and (lse[b, m:] == 7).all()
        if m == 0:
            continue
        k, v = (torch.cat([c[b, :, :ctx[b]].transpose(0, 1), d[b, :m]]) for c, d in ((kc, kd), (vc, vd)))
        seen = torch.cat([torch.ones(m, ctx[b], dtype=torch.bool), bits[b, :m, :m]], 1)
        assert_attention(out[b, :m], lse[b, :m], attention_rows(q[b, :m], k, v, seen, op.scale))
    again = torch.full_like(out, 7.0)
    op(q, kc, vc, kd, vd, ints(ctx), mask, again, num_nodes=None if live is None else ints(live))
    assert torch.equal(out, again)


@pytest.mark.parametrize("T", [1, 2, 5, 33, 64, 65, 128, 130, 256])
def test_tree_sizes(T):
    check_tree(2, T, [77, 129], (4, 2, 64))


@pytest.mark.parametrize("ctx", [[0], [1], [63], [127, 128, 129], [0, 1000, 3], [256, 0]])
def test_tree_contexts(ctx):
    check_tree(len(ctx), 9, ctx, (4, 2, 128))


@pytest.mark.parametrize("heads", [(1, 1, 64), (6, 2, 128), (14, 2, 64), (16, 8, 128), (32, 8, 64), (32, 8, 128),
                                   (128, 1, 64)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_tree_heads_and_types(heads, dtype):
    check_tree(2, 12, [200, 31], heads, dtype=dtype)


def test_tree_ragged_batch_with_dead_rows():
    check_tree(6, 20, [300, 0, 64, 5, 1, 130], (8, 2, 128), live=[20, 3, 0, 1, 19, 7])


def test_tree_with_rows_left_over_in_a_tile_repeats_its_bits():
    """3 q heads per kv head leave 2 of a tile's 128 rows unused: what lies there decides nothing."""
    for seed in range(3):
        check_tree(3, 129, [2602, 256, 256], (24, 8, 128), live=[118, 82, 124], seed=seed)
    check_tree(2, 40, [1500, 900], (5, 1, 64))


def test_tree_rows_that_see_nothing():
    check_tree(2, 6, [0, 40], (4, 2, 64), empty_row=True)


def test_tree_nodes_that_no_mask_names_may_hold_anything():
    """A padded batch without num_nodes: unused nodes have empty masks and uninitialised K/V."""
    g, B, T, nh, nkv, hd, ctx = gen(40), 2, 70, 4, 2, 128, 100
    used = [[0, 1, 5, 69], [0, 40, 66]]
    q, kc, vc = randn(g, B, T, nh, hd), randn(g, B, nkv, 128, hd), randn(g, B, nkv, 128, hd)
    kd, vd = randn(g, B, T, nkv, hd), randn(g, B, T, nkv, hd)
    bits = torch.zeros(B, T, T, dtype=torch.bool)
    for b in range(B):
        for i in used[b]:
            for j in used[b]:
                bits[b, i, j] = j <= i
        idle = [j for j in range(T) if j not in used[b]]
        kd[b, idle], vd[b, idle] = math.nan, math.inf
    packed = np.packbits(np.pad(bits.numpy(), ((0, 0), (0, 0), (0, 128 - T))), axis=2, bitorder="little").view("<i8")
    op = DraftTreeAttention(batch=B, nodes=T, max_ctx=128, num_kv_groups=nkv, q_heads_per_group=2, head_dim=hd)
    out, lse = torch.empty_like(q), torch.empty(B, T, nh, device="cuda")
    op(q, kc, vc, kd, vd, ints([ctx, 0]), torch.from_numpy(packed.copy()).cuda(), out, lse=lse)
    for b, c in enumerate((ctx, 0)):
        k, v = (torch.cat([x[b, :, :c].transpose(0, 1), d[b]]) for x, d in ((kc, kd), (vc, vd)))
        seen = torch.cat([torch.ones(T, c, dtype=torch.bool), bits[b]], 1)
        assert_attention(out[b], lse[b], attention_rows(q[b], k, v, seen, op.scale))


def test_packed_infinite_and_nan_keys_stay_with_the_rows_that_see_them():
    g, n, hd = gen(41), 200, 64
    q, k, v = randn(g, n, 2, hd), randn(g, n, 1, hd), randn(g, n, 1, hd)
    k[150] = math.nan
    out = torch.empty_like(q)
    op = PackedAttention(tokens=n, num_seqs=1, num_kv_groups=1, q_heads_per_group=2, head_dim=hd)
    op(q, k, v, ints([0, n]), out)
    seen = torch.arange(150)[None] <= torch.arange(150)[:, None]
    assert_attention(out[:150], None, attention_rows(q[:150], k[:150], v[:150], seen, op.scale))
    assert torch.isnan(out[150:]).all()


def test_tensors_of_another_device_than_the_current_one_are_refused(monkeypatch):
    from torch2iron_b200 import operators
    op = TokenLogProbs(rows=1, vocab=4)
    args = (torch.zeros(1, 4, device="cuda"), ints([0]), torch.zeros(1, device="cuda"))
    op(*args)
    monkeypatch.setattr(operators, "_current_device", lambda t: 1)
    with pytest.raises(ValueError, match="current CUDA device"):
        op(*args)


def test_tree_head_major_drafts_and_full_cache():
    check_tree(3, 17, [128, 64, 128], (8, 2, 64), max_ctx=128, head_major=True)


def test_tree_long_context():
    check_tree(1, 40, [9001], (32, 8, 128))
    check_tree(2, 3, [4097, 20], (8, 2, 64))


def test_tree_equals_a_causal_suffix():
    """A chain is a prompt's suffix: the same keys through PackedAttention give the same values within the bounds."""
    g, B, T, nh, nkv, hd, ctx = gen(77), 2, 19, 8, 2, 128, 200
    q = randn(g, B, T, nh, hd, scale=1.5)
    kc, vc = randn(g, B, nkv, 256, hd), randn(g, B, nkv, 256, hd)
    kd, vd = (c[:, :, ctx:ctx + T].transpose(1, 2).contiguous() for c in (kc, vc))
    mask, _ = draft_tree(np.tile(np.arange(-1, T - 1), (B, 1)))
    out, other = torch.empty_like(q), torch.empty_like(q)
    DraftTreeAttention(batch=B, nodes=T, max_ctx=256, num_kv_groups=nkv, q_heads_per_group=4, head_dim=hd)(
        q, kc, vc, kd, vd, ints([ctx] * B), mask.cuda(), out)
    PackedAttention(tokens=B * T, num_seqs=B, num_kv_groups=nkv, q_heads_per_group=4, head_dim=hd, max_ctx=256)(
        q.view(B * T, nh, hd), kc, vc, ints([0, T, 2 * T]), other.view(B * T, nh, hd), k_len=ints([ctx + T] * B))
    for b in range(B):
        k, v = (c[b, :, :ctx + T].transpose(0, 1) for c in (kc, vc))
        seen = torch.arange(ctx + T)[None] <= ctx + torch.arange(T)[:, None]
        ref = attention_rows(q[b], k, v, seen, hd ** -0.5)
        assert_attention(out[b], None, ref)
        assert_attention(other[b], None, ref)


def test_tree_graph_replay_with_growing_context():
    g, B, T, nh, nkv, hd = gen(8), 2, 7, 8, 2, 64
    q, kd, vd = randn(g, B, T, nh, hd), randn(g, B, T, nkv, hd), randn(g, B, T, nkv, hd)
    kc, vc = randn(g, B, nkv, 4096, hd), randn(g, B, nkv, 4096, hd)
    bits, mask = random_mask(np.random.default_rng(1), B, T, None)
    ctx = ints([10, 20])
    op = DraftTreeAttention(batch=B, nodes=T, max_ctx=4096, num_kv_groups=nkv, q_heads_per_group=4, head_dim=hd)
    out = torch.empty_like(q)
    op(q, kc, vc, kd, vd, ctx, mask, out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        op(q, kc, vc, kd, vd, ctx, mask, out)
    for c in ([0, 500], [4096, 1], [2000, 3000]):
        ctx.copy_(ints(c))
        graph.replay()
        for b in range(B):
            k, v = (torch.cat([x[b, :, :c[b]].transpose(0, 1), d[b]]) for x, d in ((kc, kd), (vc, vd)))
            seen = torch.cat([torch.ones(T, c[b], dtype=torch.bool), bits[b]], 1)
            assert_attention(out[b], None, attention_rows(q[b], k, v, seen, op.scale))


def test_tree_refusals_on_the_device():
    op = DraftTreeAttention(batch=2, nodes=3, max_ctx=64, num_kv_groups=2, q_heads_per_group=2, head_dim=64)
    z = lambda *s, dtype=BF: torch.zeros(*s, dtype=dtype, device="cuda")  # noqa: E731
    good = dict(q=z(2, 3, 4, 64), k_cache=z(2, 2, 64, 64), v_cache=z(2, 2, 64, 64), k_draft=z(2, 3, 2, 64),
                v_draft=z(2, 3, 2, 64), ctx_len=ints([1, 2]), mask=z(2, 3, 1, dtype=torch.int64), out=z(2, 3, 4, 64))
    for bad in (dict(q=z(2, 4, 4, 64)[:, :3]), dict(k_cache=z(2, 2, 65, 64)[:, :, :64]), dict(mask=z(2, 3, 1, dtype=I32)),
                dict(mask=z(2, 3, 2, dtype=torch.int64)), dict(k_draft=z(2, 1, 2, 64).expand(2, 3, 2, 64)),
                dict(num_nodes=ints([3])), dict(ctx_len=ints([1])), dict(lse=z(2, 3, 4))):
        with pytest.raises(ValueError):
            op(**{**good, **bad})


# ---------------------------------------------------------------------------
# commit
# ---------------------------------------------------------------------------
def random_trees(rng, B, T, live, kinds=3):
    """Few token values, so that walks are long and siblings often equal."""
    parents = np.array([[-1] + [rng.integers(max(0, i - 3), i) for i in range(1, T)] for _ in range(B)])
    return parents, rng.integers(0, kinds, (B, T)), rng.integers(0, kinds, (B, T))


@pytest.mark.parametrize("L,B,T,nkv,hd,kinds", [(1, 1, 1, 1, 64, 1), (2, 3, 7, 2, 64, 2), (70, 2, 33, 2, 128, 1),
                                                (3, 5, 130, 4, 64, 2), (1, 2, 256, 8, 128, 1), (2, 4, 64, 3, 8, 1)])
@pytest.mark.parametrize("form", ["stacked", "lists", "head_major"])
def test_commit(L, B, T, nkv, hd, kinds, form):
    rng, g, max_ctx = np.random.default_rng(L + T), gen(T), 192
    parents, tokens, predicted = random_trees(rng, B, T, None, kinds)
    live = [T - (i * 2) % max(1, T // 2) for i in range(B)]
    ctx = [(max_ctx - 4, 0, 100, max_ctx, -3)[i % 5] for i in range(B)]
    if B > 3:
        live[1] = 0
    kd, vd = randn(g, L, B, T, nkv, hd), randn(g, L, B, T, nkv, hd)
    kc, vc = randn(g, L, B, nkv, max_ctx, hd), randn(g, L, B, nkv, max_ctx, hd)
    want_k, want_v = kc.clone(), vc.clone()
    if form == "head_major":
        kd, vd = (t.permute(0, 3, 1, 2, 4).contiguous().permute(0, 2, 3, 1, 4) for t in (kd, vd))
    args = [list(t.unbind(0)) if form == "lists" else t for t in (kd, vd, kc, vc)]
    out = [ints(np.full((B, T), 9))] + [ints([9] * B) for _ in range(3)]
    op = DraftTreeCommit(layers=L, batch=B, nodes=T, max_ctx=max_ctx, num_kv_groups=nkv, head_dim=hd)
    op(ints(tokens), ints(parents), ints(predicted), ints(ctx), *args, *out, num_nodes=ints(live))
    torch.cuda.synchronize()
    for b in range(B):
        path = commit_walk(tokens[b], parents[b], predicted[b], ctx[b], live[b], max_ctx)
        for i, n in enumerate(path):
            want_k[:, b, :, ctx[b] + i] = kd[:, b, n]
            want_v[:, b, :, ctx[b] + i] = vd[:, b, n]
        assert out[0][b].tolist() == path + [-1] * (T - len(path))
        assert [int(t[b]) for t in out[1:]] == [len(path), predicted[b][path[-1]] if path else -1, ctx[b] + len(path)]
    assert torch.equal(kc, want_k) and torch.equal(vc, want_v)


def test_commit_ignores_malformed_parents():
    """Parents that point forward, at themselves or outside end a walk; nothing loops and nothing is read outside."""
    parents = [[3, 0, 2, 2, 900, -7], [0, 1, 2, 3, 4, 5]]
    tokens, predicted = [[1] * 6] * 2, [[1] * 6] * 2
    g = gen(2)
    kd, kc = randn(g, 1, 2, 6, 2, 64), randn(g, 1, 2, 2, 64, 64)
    out = [ints(np.zeros((2, 6)))] + [ints([0, 0]) for _ in range(3)]
    DraftTreeCommit(layers=1, batch=2, nodes=6, max_ctx=64, num_kv_groups=2)(
        ints(tokens), ints(parents), ints(predicted), ints([0, 0]), kd, kd, kc, kc.clone(), *out)
    for b in range(2):
        path = commit_walk(tokens[b], parents[b], predicted[b], 0, 6, 64)
        assert out[0][b].tolist() == path + [-1] * (6 - len(path))


def test_commit_graph_replay():
    rng, g, L, B, T = np.random.default_rng(5), gen(6), 2, 2, 8
    kd, kc = randn(g, L, B, T, 2, 64), randn(g, L, B, 2, 64, 64)
    tok, par, pred = (ints(np.zeros((B, T))) for _ in range(3))
    out = [ints(np.zeros((B, T)))] + [ints([0] * B) for _ in range(3)]
    ctx, vc = ints([3, 60]), kc.clone()
    op = DraftTreeCommit(layers=L, batch=B, nodes=T, max_ctx=64, num_kv_groups=2)
    op(tok, par, pred, ctx, kd, kd, kc, vc, *out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        op(tok, par, pred, ctx, kd, kd, kc, vc, *out)
    for _ in range(4):
        parents, tokens, predicted = random_trees(rng, B, T, None, 2)
        for dst, src in ((tok, tokens), (par, parents), (pred, predicted)):
            dst.copy_(ints(src))
        graph.replay()
        for b, c in enumerate((3, 60)):
            path = commit_walk(tokens[b], parents[b], predicted[b], c, T, 64)
            assert out[0][b].tolist() == path + [-1] * (T - len(path))
            for i, n in enumerate(path):
                assert torch.equal(kc[:, b, :, c + i], kd[:, b, n]) and torch.equal(vc[:, b, :, c + i], kd[:, b, n])


def test_commit_in_place_is_refused():
    z = lambda *s, dtype=BF: torch.zeros(*s, dtype=dtype, device="cuda")  # noqa: E731
    ctx, row = z(2, dtype=I32), lambda: z(2, dtype=I32)  # noqa: E731
    op = DraftTreeCommit(layers=1, batch=2, nodes=3, max_ctx=64, num_kv_groups=2)
    tree = [z(2, 3, dtype=I32) for _ in range(4)]
    with pytest.raises(RuntimeError, match="argument"):
        op(*tree[:3], ctx, z(1, 2, 3, 2, 64), z(1, 2, 3, 2, 64), z(1, 2, 2, 64, 64), z(1, 2, 2, 64, 64), tree[3], row(), row(), ctx)


def test_commit_refusals_on_the_device():
    z = lambda *s, dtype=BF: torch.zeros(*s, dtype=dtype, device="cuda")  # noqa: E731
    op = DraftTreeCommit(layers=2, batch=2, nodes=3, max_ctx=64, num_kv_groups=2)
    tree, row = lambda: z(2, 3, dtype=I32), lambda: z(2, dtype=I32)  # noqa: E731
    good = dict(tokens=tree(), parents=tree(), predicted=tree(), ctx_len=row(), k_drafts=z(2, 2, 3, 2, 64),
                v_drafts=z(2, 2, 3, 2, 64), k_caches=z(2, 2, 2, 64, 64), v_caches=z(2, 2, 2, 64, 64), path=tree(),
                num_accepted=row(), next_token=row(), new_len=row())
    for bad in (dict(tokens=tree().long()), dict(k_drafts=[z(2, 3, 2, 64)]), dict(k_caches=z(2, 2, 2, 65, 64)[..., :64, :]),
                dict(v_caches=[z(2, 2, 64, 64), z(2, 2, 64, 64).half()]), dict(path=z(2, 4, dtype=I32)[:, :3]),
                dict(k_drafts=[z(2, 3, 2, 64), z(2, 2, 3, 64).transpose(1, 2)]), dict(num_nodes=z(3, dtype=I32))):
        with pytest.raises(ValueError):
            op(**{**good, **bad})


# ---------------------------------------------------------------------------
# log probabilities
# ---------------------------------------------------------------------------
def check_logprobs(x, tokens, K):
    """fp32 bounds: the sum of V positive terms through a tree of partial sums
    (32 per thread and chunk, then 8 levels) is off by at most (32 + chunks +
    16) 2^-24 relative, each exponential by 2^-21; the entropy's terms by
    twice that, relative to the sum of their magnitudes."""
    M, V = x.shape
    op = TokenLogProbs(rows=M, vocab=V, num_top=K, dtype=x.dtype)
    got = {k: torch.full((M,), 7.0, device="cuda") for k in ("logprob", "entropy", "lse")}
    tops = {"top_logprob": torch.full((M, K), 7.0, device="cuda"), "top_index": torch.full((M, K), 7, dtype=I32, device="cuda")} \
        if K else {}
    op(x, tokens, got["logprob"], entropy=got["entropy"], lse=got["lse"], **tops)
    torch.cuda.synchronize()
    want = logprob_rows(x, tokens, K)
    rel = (48 + V / 8192 + 16) * 2.0 ** -24 + 2.0 ** -21
    for name in ("lse", "logprob", "entropy", *(["top_logprob"] if K else [])):
        y = (got | tops)[name].double().cpu().numpy()
        ref = want[name]
        assert np.array_equal(np.isnan(y), np.isnan(ref)), name
        assert np.array_equal(np.isinf(y), np.isinf(ref)) and (y[np.isinf(y)] == ref[np.isinf(ref)]).all(), name
        fin = np.isfinite(ref)
        tol = 2 * rel * (1 + np.abs(ref[fin])) + np.abs(ref[fin]) * 2.0 ** -22
        assert (np.abs(y[fin] - ref[fin]) <= tol).all(), (name, np.abs(y[fin] - ref[fin]).max())
    if K:
        assert np.array_equal(tops["top_index"].cpu().numpy(), want["top_index"])
    return got


@pytest.mark.parametrize("M,V,K", [(1, 1, 0), (1, 1, 1), (3, 2, 2), (2, 31, 31), (5, 33, 32), (1, 4095, 20), (1, 4096, 1),
                                   (3, 8191, 5), (2, 8193, 32), (70, 1000, 7), (1, 151936, 20), (4, 128256, 0),
                                   (449, 2500, 3), (7, 40001, 32)])
@pytest.mark.parametrize("dtype", [F32, BF, HF])
def test_logprobs_sizes(M, V, K, dtype):
    g = gen(V + K)
    x = (torch.randn(M, V, generator=g) * 3).to(dtype).cuda()
    tokens = torch.randint(0, V, (M,), generator=g).int().cuda()
    check_logprobs(x, tokens, K)


@pytest.mark.parametrize("pad,off", [(1, 0), (3, 1), (5, 3), (8, 2)])
@pytest.mark.parametrize("dtype", [F32, BF])
def test_logprobs_row_strides_and_alignment(pad, off, dtype):
    g = gen(pad)
    wide = torch.full((6, 9001 + pad + off), math.nan, dtype=dtype, device="cuda")
    x = wide[:, off:off + 9001]
    x.copy_(torch.randn(6, 9001, generator=g))
    check_logprobs(x, torch.randint(0, 9001, (6,), generator=g).int().cuda(), 9)


def order_cases(V):
    up = torch.arange(V).float() / V * 20
    ties = torch.zeros(V)
    few = torch.full((V,), -math.inf)
    few[V // 3::7777] = 2.0
    steps = (torch.arange(V) // 8192).float()
    signed = torch.zeros(V)
    signed[::2] = -0.0
    return torch.stack([up, -up, ties, few, steps, -steps, signed, torch.full((V,), -math.inf)])


@pytest.mark.parametrize("V", [20000, 151936])
def test_logprobs_orders_and_ties(V):
    """Sorted, constant, nearly all masked and stepped rows: candidate lists at their fullest."""
    x = order_cases(V).cuda()
    check_logprobs(x, ints([0, V - 1, 5, V // 3, V - 1, 0, 1, 2]), 32)
    check_logprobs(x.repeat(60, 1), ints([0, V - 1, 5, V // 3, V - 1, 0, 1, 2] * 60), 20)     # a CTA per row


@pytest.mark.parametrize("dtype", [F32, BF, HF])
def test_logprobs_extreme_values(dtype):
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    V = 10000
    x = torch.randn(6, V, generator=gen(1))
    x[0, 1:] = low
    x[1] = low
    x[2, ::3] = low
    x[3, 77] = high
    x[4, 5], x[4, 6] = high, low
    x[5, :-1] = -math.inf
    x = x.to(dtype).cuda()
    check_logprobs(x, ints([0, 3, 1, 77, 9, V - 1]), 4)


def test_logprobs_bad_tokens_nan_and_infinity():
    x = torch.randn(5, 5000, generator=gen(2))
    x[2, 17], x[3, 4000], x[4, 30] = math.nan, math.inf, math.nan
    x[4, :30] = -math.inf
    x = x.cuda()
    op = TokenLogProbs(rows=5, vocab=5000, num_top=2)
    lp, ent, tl, ti = (torch.zeros(5, device="cuda"), torch.zeros(5, device="cuda"), torch.zeros(5, 2, device="cuda"),
                       torch.zeros(5, 2, dtype=I32, device="cuda"))
    op(x, ints([-1, 5000, 3, 4, 100]), lp, entropy=ent, top_logprob=tl, top_index=ti)
    assert torch.isnan(lp).all()                        # two bad tokens, a NaN, an infinity, a NaN
    assert torch.isfinite(ent[:2]).all() and torch.isnan(ent[2:]).all() and torch.isnan(tl[2:]).all()
    assert int(ti[3, 0]) == 4000
    for r in (2, 4):                                    # NaN ranks as -inf
        y = torch.where(torch.isnan(x[r]), -math.inf, x[r])
        assert ti[r].tolist() == torch.sort(y, descending=True, stable=True).indices[:2].tolist()


def test_logprobs_repeat_and_graph():
    x = torch.randn(3, 151936, generator=gen(4)).cuda()
    op = TokenLogProbs(rows=3, vocab=151936, num_top=5)
    bufs = [torch.zeros(3, device="cuda"), torch.zeros(3, device="cuda"), torch.zeros(3, 5, device="cuda"),
            torch.zeros(3, 5, dtype=I32, device="cuda")]
    tok = ints([1, 2, 3])
    run = lambda: op(x, tok, bufs[0], entropy=bufs[1], top_logprob=bufs[2], top_index=bufs[3])  # noqa: E731
    run()
    first = [b.clone() for b in bufs]
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        run()
    for b in bufs:
        b.zero_()
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(first, bufs))
    x.copy_(x.flip(1))
    graph.replay()
    assert torch.equal(bufs[3], 151935 - first[3])       # no ties in these rows
    check_logprobs(x, tok, 5)


def test_logprobs_refusals_on_the_device():
    op = TokenLogProbs(rows=2, vocab=10, num_top=2)
    x, t, lp = torch.zeros(2, 10, device="cuda"), ints([0, 1]), torch.zeros(2, device="cuda")
    tl, ti = torch.zeros(2, 2, device="cuda"), torch.zeros(2, 2, dtype=I32, device="cuda")
    for bad in (dict(logits=torch.zeros(10, 2, device="cuda").t()), dict(logits=x[:1].expand(2, 10)), dict(tokens=t.long()),
                dict(top_index=None), dict(top_logprob=None), dict(logprob=lp.half()), dict(top_index=ti.long()),
                dict(logits=x.half())):
        with pytest.raises(ValueError):
            op(**{**dict(logits=x, tokens=t, logprob=lp, top_logprob=tl, top_index=ti), **bad})
