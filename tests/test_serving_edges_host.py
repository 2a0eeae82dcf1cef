"""Host checks of the serving operators beyond their first tests."""

import ctypes as C
import math

import pytest

from torch2iron_b200 import _lib
from torch2iron_b200.operators import DraftTreeAttention, PackedAttention, draft_tree

ERR_SHAPE, ERR_ALIGN, ERR_ARG, ERR_WORKSPACE = 1, 2, 6, 5


@pytest.fixture
def base():
    buf = (C.c_uint8 * 16384)()
    yield (C.addressof(buf) + 255) & ~255          # aligned host stand-ins (never dereferenced)
    del buf


# A call that passes the size checks ends at the missing workspace: nothing is launched.
@pytest.mark.parametrize("seqs,tokens,heads,want", [
    (32768, 524288, (32, 8), ERR_WORKSPACE),       # many short prompts
    (1, 1 << 20, (32, 8), ERR_WORKSPACE), (1000, 1 << 20, (32, 8), ERR_WORKSPACE), (1 << 20, 1 << 20, (8, 8), ERR_WORKSPACE),
    (1, 1 << 23, (32, 8), ERR_SHAPE), (1, 0x7fffffff, (128, 1), ERR_SHAPE), (0x7fffffff, 0x7fffffff, (64, 64), ERR_SHAPE),
])
def test_packed_attention_counts_each_prompts_own_keys(base, seqs, tokens, heads, want):
    nh, nkv = heads
    got = _lib.load().t2b_packed_attention(
        base, base + (1 << 40), base + (2 << 40), base + (3 << 40), None, 0, 0, base + 1024, None, None, seqs, tokens, 0,
        tokens, nh, nkv, 64,
        nh * 64, 64, nh * 64, 64, nkv * 64, 64, 8, nkv * 64, 64, 8, 0.125, None, 0, None)
    assert got == want


def test_a_prompt_of_tokens_one_by_one_counts_no_more_sequences_than_rows(base):
    """A decode batch in a table of many more sequences: those without rows have no work."""
    args = lambda seqs: (base, base + (1 << 48), base + (2 << 48), base + (1 << 40), None, 0, 0, base + 1024, None,  # noqa: E731
                         base + 1536, seqs, 64, seqs, 65536, 32, 8, 64, 2048, 64, 2048, 64, 64, 64 * 65536, 512 * 65536, 64, 64 * 65536,
                         512 * 65536, 0.125, None, 0, None)
    assert _lib.load().t2b_packed_attention(*args(1 << 18)) == ERR_WORKSPACE


# ---------------------------------------------------------------------------
# results over inputs (every call below that is not refused ends at its missing workspace)
# ---------------------------------------------------------------------------
def packed(base, out, q=None, k=None, v=None, lse=None, rows=8, nh=4, nkv=2, hd=64, q_strides=None, o_strides=None,
           k_strides=None, v_strides=None):
    q_strides, o_strides = (s or (nh * hd, hd) for s in (q_strides, o_strides))
    k_strides, v_strides = (s or (nkv * hd, hd) for s in (k_strides, v_strides))
    return _lib.load().t2b_packed_attention(
        q or base, k or base + (1 << 20), v or base + (2 << 20), out, lse, 0, 0, base + (3 << 20), None, None, 1, rows, 0,
        rows, nh, nkv, hd, *q_strides, *o_strides, *k_strides, 8, *v_strides, 8, 0.125, None, 0, None)


def test_packed_attention_refuses_results_over_its_inputs(base):
    base <<= 8                                       # (addresses alone count)
    ok, far = ERR_WORKSPACE, base + (4 << 20)
    assert packed(base, far) == ok
    assert packed(base, base) == ok                                                   # in place of q, row by row
    assert packed(base, base, q_strides=(512, 64)) == ERR_ARG                         # over q in another layout
    assert packed(base, base + 128) == ERR_ARG and packed(base, base + 512) == ERR_ARG
    for at in (1 << 20, 2 << 20):                                                     # over k, over v
        assert packed(base, base + at) == ERR_ARG
        assert packed(base, base + at + 8 * 2 * 64 * 2 - 128) == ERR_ARG              # its last head
        assert packed(base, base + at + 8 * 2 * 64 * 2) == ok
        assert packed(base, base + at - 8 * 4 * 64 * 2) == ok
        assert packed(base, far, lse=base + at + 64) == ERR_ARG                       # the log-sums
    assert packed(base, far, lse=far + 256) == ERR_ARG
    assert packed(base, far, lse=base + 16) == ERR_ARG


def test_packed_attention_takes_views_of_one_fused_tensor(base):
    """Rows of [q | k | v | out] in one allocation interleave without a common element."""
    base <<= 8
    ok, row = ERR_WORKSPACE, (4 + 2 + 2 + 4) * 64
    s = (row, 64)
    views = dict(k=base + 4 * 128, v=base + 6 * 128, q_strides=s, k_strides=s, v_strides=s)
    assert packed(base, base + 8 * 128, o_strides=s, **views) == ok
    assert packed(base, base, o_strides=s, **views) == ok                             # out in place of q
    assert packed(base, base + 7 * 128, o_strides=s, **views) == ERR_ARG              # its first head is v's last
    assert packed(base, base + 9 * 128, o_strides=s, **views) == ERR_ARG              # its last head is the next row's q
    half = (2 * 4 * 128, 128)                                                         # heads of 128: k in the first half
    assert packed(base + (8 << 20), base + 128, k=base, k_strides=half, o_strides=half) == ok
    assert packed(base + (8 << 20), base + 112, k=base, k_strides=half, o_strides=half) == ERR_ARG
    flip = (64, 8 * 64)                                                               # head-major
    assert packed(base, base + (8 << 20), o_strides=flip, k_strides=flip) == ok
    assert packed(base, base + 4 * 8 * 128 + (1 << 20) - 8 * 128, o_strides=flip, k_strides=flip) == ok
    assert packed(base, base + (1 << 20) + 8 * 128, o_strides=flip, k_strides=flip) == ERR_ARG


@pytest.mark.parametrize("rows,nh", [(1, 4), (1, 1), (5, 1), (3, 4)])
def test_packed_attention_takes_the_last_rows_of_a_fused_tensor_in_place(base, rows, nh):
    """The last tokens of [q | k | v] rows over all keys there, out in place of q: one row, or one head, has no stride
    in common with the keys' rows."""
    base <<= 8
    nkv, keys, row = 1, 100, (nh + 2) * 64

    def call(out_at):
        q = base + (keys - rows) * row * 2
        return _lib.load().t2b_packed_attention(
            q, base + nh * 128, base + (nh + 1) * 128, q + out_at, None, 0, 0, base + (3 << 20), base + (4 << 20),
            base + (5 << 20), 1, rows, 0, keys, nh, nkv, 64, row, 64, row, 64, row, 64, 8, row, 64, 8, 0.125, None, 0, None)

    assert call(0) == ERR_WORKSPACE
    assert call(128) == ERR_ARG and call(-128) == ERR_ARG        # over k, over the v of the row before


def tree(base, out, lse=None, kd=None, B=2, T=4, nh=4, nkv=2, hd=64, ctx=64):
    return _lib.load().t2b_tree_attention(
        base, base + (1 << 20), base + (2 << 20), kd or base + (3 << 20), base + (4 << 20), out, lse, 0, 0, base + (5 << 20),
        None, base + (6 << 20), B, T, nh, nkv, hd, ctx, nh * hd, hd, nh * hd, hd, T * nkv * hd, nkv * hd, hd, T * nkv * hd,
        nkv * hd, hd, 0.125, None, 0, None)


def test_tree_attention_refuses_results_over_its_inputs(base):
    base <<= 8
    assert tree(base, base + (7 << 20)) == ERR_WORKSPACE and tree(base, base) == ERR_WORKSPACE
    assert tree(base, base + (7 << 20), kd=base + (1 << 20)) == ERR_WORKSPACE          # drafts inside the cache are only read
    for at in (1, 2, 3, 4):
        assert tree(base, base + (at << 20) + 256) == ERR_ARG
        assert tree(base, base + (7 << 20), lse=base + (at << 20) + 256) == ERR_ARG


def test_tree_commit_refuses_caches_over_drafts_and_over_one_another(base):
    base <<= 8
    B, T, nkv, hd, ctx, L = 2, 4, 2, 64, 64, 3
    draft, cache = B * T * nkv * hd * 2, B * nkv * ctx * hd * 2
    stack = lambda at, size: [base + at + i * size for i in range(L)]  # noqa: E731
    kd, vd, kc, vc = stack(1 << 20, draft), stack(2 << 20, draft), stack(3 << 20, cache), stack(4 << 20, cache)

    def call(kd=kd, vd=vd, kc=kc, vc=vc, path=base + (5 << 20), B=B):
        arrays = [(C.c_void_p * L)(*a) for a in (kd, vd, kc, vc)]
        i32 = [base + (6 << 20) + i * 4096 for i in range(8)]
        return _lib.load().t2b_tree_commit(*i32[:4], None, *arrays, L, path, *i32[4:7], B, T, nkv, hd, ctx, T * nkv * hd,
                                           nkv * hd, hd, T * nkv * hd, nkv * hd, hd, None)

    for bad in (dict(kd=[kc[0], *kd[1:]]), dict(vd=[*vd[:2], kc[2] + cache - 16]), dict(kd=[*kd[:2], vc[0] - 16]),
                dict(kc=[kc[0], kc[0], kc[2]]), dict(vc=kc), dict(kc=[kc[2], kc[1], kc[0] + cache // 2]), dict(vc=[*vc[:2], vd[1]]),
                dict(path=kc[1] + 32), dict(path=vd[2] + 32)):
        assert call(**bad) == ERR_ARG, bad


@pytest.mark.parametrize("live", [[1.5, 2.0], [math.nan, 2.0], ["1", "2"]])
def test_draft_tree_takes_whole_numbers_of_nodes(live):
    with pytest.raises(ValueError):
        draft_tree([[-1, 0], [-1, 0]], live)
    assert draft_tree([[-1, 0], [-1, 0]], [1.0, 2.0])[0].tolist() == [[[1], [0]], [[1], [3]]]


@pytest.mark.parametrize("scale", [3e38, 1e39, 1e-60])
def test_a_scale_has_to_fit_the_kernels_fp32(base, scale):
    """The kernels multiply by scale * log2(e) in 32 bits."""
    with pytest.raises(ValueError):
        PackedAttention(tokens=4, num_seqs=1, scale=scale)
    with pytest.raises(ValueError):
        DraftTreeAttention(batch=1, nodes=4, max_ctx=64, scale=scale)
    far = [base + (i << 20) for i in range(5)]
    got = _lib.load().t2b_packed_attention(*far[:4], None, 0, 0, far[4], None, None, 1, 4, 0, 4, 4, 2, 64, 256, 64, 256, 64, 128,
                                           64, 8, 128, 64, 8, scale, None, 0, None)
    assert got == ERR_ARG
