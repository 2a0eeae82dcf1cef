"""Workspace sizes of the linears, on the host."""

import pytest

from torch2iron_b200 import _lib


@pytest.mark.parametrize("K", [256, 2048, 4096, 8192, 9728, 12288, 13824, 18944])
@pytest.mark.parametrize("N", [128, 256, 512, 640, 1024, 2560, 4096, 19456])
def test_a_workspace_sized_for_some_rows_serves_fewer(N, K):
    """An engine keeps the buffers of its longest pass and runs shorter ones in them."""
    L = _lib.load()
    need = [L.t2b_w4a16_gemm_workspace_bytes(M, N, K) for M in (*range(1, 300), 1000, 1025, 8192)]
    assert need == sorted(need)
    assert [L.t2b_down_residual_workspace_bytes(M, N, K) for M in (1, 24, 32)] == [need[0], need[23], need[31]]
