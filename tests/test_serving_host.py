"""CPU checks of the serving operators: the plain references against hand
values, the draft-tree helper, and every refusal that happens on the host."""

import ctypes as C
import math

import pytest
import torch

from tests.serving_ref import attention_rows, commit_walk, logprob_rows
from torch2iron_b200 import _lib
from torch2iron_b200.operators import (DraftTreeAttention, DraftTreeCommit, PackedAttention, TokenLogProbs,
                                       draft_tree)

ERR_SHAPE, ERR_ALIGN, ERR_ARG, ERR_WORKSPACE = 1, 2, 6, 5


def test_reference_attention_on_two_keys():
    q = torch.zeros(2, 1, 64)
    q[:, 0, 0] = 1.0
    k = torch.zeros(2, 1, 64)
    k[1, 0, 0] = math.log(3.0)
    v = torch.zeros(2, 1, 64)
    v[0, 0, 0], v[1, 0, 0] = 4.0, 8.0
    seen = torch.tensor([[True, False], [True, True]])
    out, lse, *_ = attention_rows(q.bfloat16().double().float(), k, v, seen, 1.0)
    assert out[0, 0, 0] == 4.0 and abs(out[1, 0, 0] - 7.0) < 1e-6
    assert lse[0, 0] == 0.0 and abs(lse[1, 0] - math.log(4.0)) < 1e-6


def test_reference_logprobs_ties_and_masks():
    x = torch.tensor([[0.0, 1.0, 1.0, -math.inf], [-math.inf] * 4])
    got = logprob_rows(x, torch.tensor([1, 2]), 4)
    assert got["top_index"].tolist() == [[1, 2, 0, 3], [0, 1, 2, 3]]
    assert got["entropy"][1] == 0 and math.isinf(got["logprob"][1])


def test_reference_walk_takes_the_lowest_of_equal_children():
    #        node 0 -> 1 (tok 5), 2 (tok 5); 2 -> 3
    assert commit_walk([9, 5, 5, 6], [-1, 0, 0, 2], [5, 6, 6, 0], 3, 4, 100) == [0, 1]
    assert commit_walk([9, 5, 5, 6], [-1, 0, 0, 1], [5, 6, 6, 0], 3, 4, 100) == [0, 1, 3]
    assert commit_walk([9, 5, 5, 6], [-1, 0, 0, 1], [5, 6, 6, 0], 3, 4, 5) == [0, 1]      # the cache is full
    assert commit_walk([9, 5], [-1, 0], [5, 0], 5, 2, 5) == [] and commit_walk([9], [-1], [0], 0, 0, 5) == []


def test_draft_tree_mask_and_depth():
    parents = [[-1, 0, 0, 1, 3, 2], [7, 0, 1, 2, 3, 4]]
    mask, depth = draft_tree(parents, [6, 4])
    assert mask.shape == (2, 6, 1) and mask.dtype == torch.int64
    assert mask[0, :, 0].tolist() == [1, 3, 5, 11, 27, 37]
    assert mask[1, :, 0].tolist() == [1, 3, 7, 15, 0, 0]
    assert depth.tolist() == [[0, 1, 1, 2, 3, 2], [0, 1, 2, 3, 0, 0]]
    chain = torch.arange(-1, 129)[None]
    mask, depth = draft_tree(chain)
    assert mask.shape == (1, 130, 3)
    assert mask[0, 129].tolist() == [-1, -1, 3] and mask[0, 63].tolist() == [-1, 0, 0]
    assert int(depth[0, 129]) == 129
    assert draft_tree([[-1]], [0])[0].tolist() == [[[0]]]


@pytest.mark.parametrize("parents,live", [([[-1, 1]], None), ([[-1, -1]], None), ([[-1, 2, 0]], None),
                                          ([[-1, 0]], [3]), ([[-1, 0]], [-1]), ([[-1, 0]], [1, 1]), ([-1, 0], None),
                                          ([[-1.0, 0.0]], None)])
def test_draft_tree_refusals(parents, live):
    with pytest.raises(ValueError):
        draft_tree(parents, live)


@pytest.mark.parametrize("kw", [dict(tokens=0), dict(num_seqs=0), dict(head_dim=96), dict(q_heads_per_group=0),
                                dict(q_heads_per_group=129), dict(num_kv_groups=0), dict(dtype=torch.float32),
                                dict(out_dtype=torch.float32), dict(scale=0.0), dict(scale=-1.0),
                                dict(scale=math.nan), dict(scale=math.inf), dict(kv_tokens=0), dict(max_ctx=0),
                                dict(max_ctx=64, kv_tokens=64)])
def test_packed_attention_constructor_refusals(kw):
    with pytest.raises(ValueError):
        PackedAttention(**{**dict(tokens=4, num_seqs=2), **kw})


@pytest.mark.parametrize("kw", [dict(batch=0), dict(nodes=0), dict(nodes=257), dict(max_ctx=0), dict(head_dim=32),
                                dict(dtype=torch.float32), dict(scale=0.0)])
def test_tree_attention_constructor_refusals(kw):
    with pytest.raises(ValueError):
        DraftTreeAttention(**{**dict(batch=1, nodes=4, max_ctx=64), **kw})


@pytest.mark.parametrize("kw", [dict(layers=0), dict(batch=0), dict(nodes=257), dict(max_ctx=0), dict(head_dim=12),
                                dict(head_dim=2048), dict(num_kv_groups=0), dict(dtype=torch.float32)])
def test_tree_commit_constructor_refusals(kw):
    with pytest.raises(ValueError):
        DraftTreeCommit(**{**dict(layers=1, batch=1, nodes=4, max_ctx=64), **kw})


@pytest.mark.parametrize("kw", [dict(rows=0), dict(vocab=0), dict(num_top=33), dict(num_top=-1),
                                dict(vocab=5, num_top=6), dict(dtype=torch.float64)])
def test_token_logprobs_constructor_refusals(kw):
    with pytest.raises(ValueError):
        TokenLogProbs(**{**dict(rows=1, vocab=100), **kw})


def test_operators_refuse_host_tensors():
    q = torch.zeros(4, 32, 64, dtype=torch.bfloat16)
    kv = torch.zeros(4, 8, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA device"):
        PackedAttention(tokens=4, num_seqs=1)(q, kv, kv, torch.zeros(2, dtype=torch.int32), q.clone())
    with pytest.raises(ValueError, match="CUDA device"):
        TokenLogProbs(rows=1, vocab=4)(torch.zeros(1, 4), torch.zeros(1, dtype=torch.int32), torch.zeros(1))


def test_operators_refuse_wrong_shapes_and_types():
    op = PackedAttention(tokens=4, num_seqs=1)
    q = torch.zeros(4, 32, 64, dtype=torch.bfloat16)
    kv = torch.zeros(4, 8, 64, dtype=torch.bfloat16)
    start = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="q: expected shape"):
        op(q[:3], kv, kv, start, q)
    with pytest.raises(ValueError, match="q: expected torch.bfloat16"):
        op(q.half(), kv, kv, start, q)


def test_arg_specs():
    spec = PackedAttention(tokens=9, num_seqs=3, num_kv_groups=2, q_heads_per_group=3, head_dim=128).get_arg_spec()
    assert [s.shape for s in spec] == [(9, 6, 128), (9, 2, 128), (9, 2, 128), (4,), (9, 6, 128)]
    spec = PackedAttention(tokens=9, num_seqs=3, num_kv_groups=2, max_ctx=64).get_arg_spec()
    assert spec[1].shape == (3, 2, 64, 64)
    spec = DraftTreeAttention(batch=2, nodes=65, max_ctx=64, num_kv_groups=2).get_arg_spec()
    assert spec[1].shape == (2, 2, 64, 64) and spec[3].shape == (2, 65, 2, 64) and spec[6].shape == (2, 65, 2)
    spec = DraftTreeCommit(layers=3, batch=2, nodes=5, max_ctx=64, num_kv_groups=2).get_arg_spec()
    assert spec[4].shape == (3, 2, 5, 2, 64) and spec[6].shape == (3, 2, 2, 64, 64)
    assert len(TokenLogProbs(rows=2, vocab=7).get_arg_spec()) == 4
    assert TokenLogProbs(rows=2, vocab=7, num_top=3).get_arg_spec()[4].shape == (2, 3)


@pytest.fixture
def base():
    buf = (C.c_uint8 * 16384)()
    at = (C.addressof(buf) + 255) & ~255           # aligned host stand-ins (never dereferenced)
    yield at
    del buf


def test_packed_attention_rejects_bad_arguments_on_the_host(base):
    f = _lib.load().t2b_packed_attention

    def call(q=base, k=base + 256, v=base + 512, out=base + 768, dtype=0, out_dtype=0, q_start=base + 1024, k_start=None,
             k_len=None, n_seqs=1, total_q=4, kv_seqs=0, kv_tokens=4, nh=4, nkv=2, hd=64, q_row=256, q_head=64,
             k_tok=128, k_head=64, k_seq=8, scale=0.125, ws=base + 2048, ws_bytes=1 << 40):
        return f(q, k, v, out, None, dtype, out_dtype, q_start, k_start, k_len, n_seqs, total_q, kv_seqs, kv_tokens, nh,
                 nkv, hd, q_row, q_head, 256, 64, k_tok, k_head, k_seq, k_tok, k_head, k_seq, scale, ws, ws_bytes, None)

    assert call(q=None) == ERR_ARG and call(k=None) == ERR_ARG and call(out=None) == ERR_ARG
    assert call(q_start=None) == ERR_ARG
    assert call(dtype=2) == ERR_ARG and call(out_dtype=2) == ERR_ARG
    assert call(scale=0.0) == ERR_ARG and call(scale=math.nan) == ERR_ARG and call(scale=math.inf) == ERR_ARG
    assert call(hd=96) == ERR_SHAPE and call(nh=5) == ERR_SHAPE and call(nh=2 * 129) == ERR_SHAPE
    assert call(total_q=0) == ERR_SHAPE and call(n_seqs=0) == ERR_SHAPE and call(kv_tokens=0) == ERR_SHAPE
    assert call(q=base + 8) == ERR_ALIGN and call(v=base + 514) == ERR_ALIGN
    assert call(q_row=260) == ERR_ALIGN and call(k_tok=0) == ERR_ALIGN and call(k_head=4) == ERR_ALIGN
    assert call(k_start=base + 1280) == ERR_ARG and call(k_len=base + 1280) == ERR_ARG      # they go together
    assert call(kv_seqs=1) == ERR_ARG                                                       # cache rows need k_len
    assert call(kv_seqs=1, k_len=base + 1280, k_start=base + 1536) == ERR_ARG
    assert call(kv_seqs=1, n_seqs=2, k_len=base + 1280) == ERR_ARG                          # fewer rows than sequences


def test_tree_attention_rejects_bad_arguments_on_the_host(base):
    f = _lib.load().t2b_tree_attention

    def call(q=base, kc=base + 256, kd=base + 512, ctx=base + 768, mask=base + 1024, dtype=0, B=1, T=4, nh=4, nkv=2,
             hd=64, max_ctx=64, kd_node=128, scale=0.125):
        return f(q, kc, kc, kd, kd, base + 1536, None, dtype, 0, ctx, None, mask, B, T, nh, nkv, hd, max_ctx, 256, 64,
                 256, 64, 512, kd_node, 64, 512, kd_node, 64, scale, base + 2048, 1 << 40, None)

    assert call(q=None) == ERR_ARG and call(kc=None) == ERR_ARG and call(kd=None) == ERR_ARG
    assert call(ctx=None) == ERR_ARG and call(mask=None) == ERR_ARG and call(dtype=2) == ERR_ARG
    assert call(B=0) == ERR_SHAPE and call(T=0) == ERR_SHAPE and call(T=257) == ERR_SHAPE
    assert call(max_ctx=0) == ERR_SHAPE and call(hd=80) == ERR_SHAPE and call(B=1 << 24, T=256) == ERR_SHAPE
    assert call(kd=base + 520) == ERR_ALIGN and call(mask=base + 1028) == ERR_ALIGN and call(kd_node=100) == ERR_ALIGN
    assert call(scale=-1.0) == ERR_ARG


def test_tree_commit_rejects_bad_arguments_on_the_host(base):
    f = _lib.load().t2b_tree_commit
    good = (C.c_void_p * 2)(base + 4096, base + 8192)

    def call(tokens=base, layers=good, n_layers=2, B=1, T=4, nkv=2, hd=64, max_ctx=64, kd_row=512, path=base + 256):
        return f(tokens, base, base, base, None, layers, good, good, good, n_layers, path, base, base, base, B, T, nkv,
                 hd, max_ctx, kd_row, 128, 64, 512, 128, 64, None)

    assert call(tokens=None) == ERR_ARG and call(path=None) == ERR_ARG and call(layers=None) == ERR_ARG
    assert call(layers=(C.c_void_p * 2)(base, None)) == ERR_ARG
    assert call(layers=(C.c_void_p * 2)(base, base + 4)) == ERR_ALIGN
    assert call(n_layers=0) == ERR_SHAPE and call(B=0) == ERR_SHAPE and call(T=257) == ERR_SHAPE
    assert call(hd=12) == ERR_SHAPE and call(max_ctx=0) == ERR_SHAPE and call(nkv=0) == ERR_SHAPE
    assert call(kd_row=4) == ERR_ALIGN


def test_tree_commit_refuses_results_over_inputs(base):
    """Every CTA reads a row's inputs while one writes its results: an update in place would race."""
    f = _lib.load().t2b_tree_commit
    good = (C.c_void_p * 1)(base + 8192)

    def call(ctx=base + 512, path=base + 1024, count=base + 1536, nxt=base + 2048, length=base + 2560, live=None):
        return f(base, base + 128, base + 256, ctx, live, good, good, good, good, 1, path, count, nxt, length, 2, 4, 2, 64,
                 64, 512, 128, 64, 512, 128, 64, None)

    assert call(length=base + 512) == ERR_ARG                  # new_len over ctx_len
    assert call(path=base + 124) == ERR_ARG                    # path over tokens and parents
    assert call(nxt=base + 1540) == ERR_ARG                    # next_token over num_accepted
    assert call(live=base + 2560) == ERR_ARG                   # new_len over num_nodes
    assert call(count=base + 256) == ERR_ARG


def test_token_logprobs_rejects_bad_arguments_on_the_host(base):
    f = _lib.load().t2b_token_logprobs

    def call(x=base, dtype=2, M=2, V=100, ld=100, tokens=base + 1024, logprob=base + 1280, top=0, tl=None, ti=None):
        return f(x, dtype, M, V, ld, tokens, logprob, None, None, top, tl, ti, None)

    assert call(x=None) == ERR_ARG and call(dtype=3) == ERR_ARG
    assert call(tokens=None) == ERR_ARG and call(logprob=None) == ERR_ARG
    assert call(tokens=None, logprob=None) == ERR_ARG                      # nothing asked for
    assert call(top=3) == ERR_ARG and call(ti=base + 2048) == ERR_ARG
    assert call(M=0) == ERR_SHAPE and call(V=0) == ERR_SHAPE and call(ld=99) == ERR_SHAPE
    assert call(top=33, ti=base + 2048) == ERR_SHAPE and call(V=2, ld=2, top=3, ti=base + 2048) == ERR_SHAPE
    assert call(x=base + 2) == ERR_ALIGN
