"""One split-K workspace under calls of different sizes: prompt passes, short last
chunks and draft trees run any number of rows through an engine's buffers."""

import numpy as np
import pytest
import torch

from torch2iron_b200 import _lib, synth
from torch2iron_b200 import weights as W
from torch2iron_b200.config import QuantizedQwenConfig
from torch2iron_b200.engine import DecodeEngine

pytestmark = pytest.mark.gpu


def gemm(w, x, ws):
    M, K = x.shape
    y = torch.full((M, w.out_features), 7.0, device="cuda")
    _lib.call("t2b_w4a16_gemm", _lib.ptr(w.qw), _lib.ptr(w.meta), w.fmt, _lib.ptr(x), _lib.DTYPE[x.dtype], _lib.ptr(y),
              _lib.DTYPE[torch.float32], M, w.out_features, K, 128, _lib.ptr(ws), ws.numel(), _lib.stream())
    return y


@pytest.mark.parametrize("rows", [[43, 18, 6, 43, 1, 2, 43], [1, 43, 3, 64, 5, 200, 18], [256, 1, 255]])
def test_calls_of_other_sizes_leave_the_counters_alone(rows):
    """9728 inputs split into more k-slices than a cluster holds; the calls that
    share a workspace give the bits that each gives alone."""
    K, g = 9728, torch.Generator().manual_seed(11)
    ws_of = lambda N, M: _lib.load().t2b_w4a16_gemm_workspace_bytes(M, N, K)  # noqa: E731
    weights = {N: W.from_autogptq(synth.random_linear(N, K, g)) for N in (256, 2560)}
    torch.cuda.synchronize()
    shared = torch.zeros(max(ws_of(N, M) for N in weights for M in rows), dtype=torch.uint8, device="cuda")
    for M in rows:
        for N, w in weights.items():
            assert ws_of(N, M) > 0
            x = torch.randn(M, K, generator=g).half().cuda()
            alone = gemm(w, x, torch.zeros(ws_of(N, M), dtype=torch.uint8, device="cuda"))
            assert torch.equal(gemm(w, x, shared), alone), (M, N)


def test_more_tiles_than_the_counters_header_holds():
    """821 x 20 tiles in fp32 activations (the CUDA-core path at any row count), before and behind a small call.
    Products and sums in 32 bits, in any order: off by at most (K + 1) 2^-24 of the sum of magnitudes."""
    M, N, K, g = 6561, 2560, 9728, torch.Generator().manual_seed(12)
    w = W.from_autogptq(synth.random_linear(N, K, g))
    torch.cuda.synchronize()
    big, small = torch.randn(M, K, generator=g).cuda(), torch.randn(3, K, generator=g).cuda()
    n = _lib.load().t2b_w4a16_gemm_workspace_bytes(M, N, K)
    shared = torch.zeros(n, dtype=torch.uint8, device="cuda")
    alone = gemm(w, small, torch.zeros_like(shared))
    first = gemm(w, big, shared)
    assert torch.equal(gemm(w, small, shared), alone)
    assert torch.equal(gemm(w, big, shared), first)
    assert torch.equal(gemm(w, small, shared), alone)
    dense = W.dequantize(w).double()
    for x, y in ((big, first), (small, alone)):
        want, size = x.double() @ dense.t(), x.double().abs() @ dense.abs().t()
        assert ((y - want).abs() <= (K + 1) * 2.0 ** -24 * size).all()


CFG = QuantizedQwenConfig(vocab_size=512, emb_dim=256, n_layers=2, n_heads=4, n_kv_groups=2, head_dim=64,
                          hidden_dim=9728, rms_norm_eps=1e-6, rope_base=1e6)


@pytest.mark.parametrize("nodes", [[9, 3, 9], [2, 20]])
def test_draft_trees_behind_a_packed_prompt(nodes):
    """A packed prompt of 43 rows, then trees of fewer rows over the same buffers: as over fresh ones."""
    model, g = synth.random_model(CFG, seed=21), torch.Generator().manual_seed(22)
    prompts = [torch.randint(0, CFG.vocab_size, (n,), generator=g) for n in (30, 13)]
    states = []
    for fresh in (True, False):
        eng = DecodeEngine(CFG, model, batch=2, max_ctx=128, use_graph=False)
        eng.prefill_packed(prompts)
        log = []
        for T in nodes:
            if fresh:
                eng._pf = None                     # new activations and zeroed workspaces
            tok = np.random.default_rng(T).integers(0, CFG.vocab_size, (2, T))
            tok[:, 0] = eng.tokens.cpu().numpy()
            path, count, following = eng.decode_tree(tok, np.tile(np.arange(-1, T - 1), (2, 1)))
            log += [path.tolist(), count.tolist(), following.tolist()]
        states.append((log, [t.clone() for t in eng.k_cache + eng.v_cache]))
    assert states[0][0] == states[1][0]
    assert all(torch.equal(a, b) for a, b in zip(states[0][1], states[1][1]))


def test_a_tree_of_fewer_rows_than_the_prompt_needs_more_partials():
    """64 rows run in k-slices twice as large as 48 do: the smaller call's workspace is the larger."""
    model, g = synth.random_model(CFG, seed=31), torch.Generator().manual_seed(32)
    eng = DecodeEngine(CFG, model, batch=2, max_ctx=128, use_graph=False)
    eng.prefill_packed([torch.randint(0, CFG.vocab_size, (n,), generator=g) for n in (40, 24)])
    tok = np.repeat(eng.tokens.cpu().numpy()[:, None], 24, 1)
    _, count, _ = eng.decode_tree(tok, np.tile(np.arange(-1, 23), (2, 1)))
    assert (count >= 1).all()
