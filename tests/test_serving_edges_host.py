"""Host checks of the serving operators beyond their first tests."""

import ctypes as C

import pytest

from torch2iron_b200 import _lib

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
        base, base + 256, base + 512, base + 768, None, 0, 0, base + 1024, None, None, seqs, tokens, 0, tokens, nh, nkv, 64,
        nh * 64, 64, nh * 64, 64, nkv * 64, 64, 8, nkv * 64, 64, 8, 0.125, None, 0, None)
    assert got == want


def test_a_prompt_of_tokens_one_by_one_counts_no_more_sequences_than_rows(base):
    """A decode batch in a table of many more sequences: those without rows have no work."""
    args = lambda seqs: (base, base + 256, base + 512, base + 768, None, 0, 0, base + 1024, None, base + 1536, seqs, 64,  # noqa: E731
                         seqs, 65536, 32, 8, 64, 2048, 64, 2048, 64, 64, 64 * 65536, 512 * 65536, 64, 64 * 65536,
                         512 * 65536, 0.125, None, 0, None)
    assert _lib.load().t2b_packed_attention(*args(1 << 18)) == ERR_WORKSPACE
