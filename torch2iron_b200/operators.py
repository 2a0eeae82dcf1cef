"""The reference's decode operators, by name, backed by the sm_100a kernels.

Each class keeps the constructor fields of the torch2iron operator it
replaces (NPU-only tiling fields are accepted and validated the same way, so
existing call sites construct them unchanged), raises ``ValueError`` from
``__post_init__`` on bad shapes as the reference does, reports an
``get_arg_spec()`` list of ``ArgSpec(direction, shape, dtype)``, and runs on
``__call__(*buffers)`` with CUDA tensors in arg-spec order.

Replaced operators (reference file:line):

* ``W4A16GEMV``        src/models/quantized_qwen3/operators/w4a16_gemv/op.py:21-126
* ``W4A16GEMM``, ``W4A16KGroupGEMM``, ``W4A16PairedKGroupGEMM``, ``W4A16NShardGEMM``
                       src/models/quantized_qwen3/operators/w4a16_gemm/op.py:22-399
* ``RMSNormRoPE``      src/torch2iron/operators/rms_norm_rope/op.py:19-90
* ``LlamaChunkedAttention``  src/torch2iron/operators/llama_chunked_attention/op.py:20-165
* ``ResidualAddRMSNorm``     src/torch2iron/operators/residual_add_rms_norm/op.py:19-85
* ``SiLUMul``          src/torch2iron/operators/silu_mul/op.py:20-80
* ``CopyPresentPacketKV``    src/torch2iron/operators/copy_present_packet_kv/op.py:18-80

Operators of a serving loop that the reference has no counterpart for (its
runner decodes one greedy token per row and step, ``qwen_npu.py:166-236``):
``PackedAttention`` (causal attention over prompts of different lengths,
without padding), ``DraftTreeAttention`` and ``DraftTreeCommit`` (verifying a
tree of drafted tokens over the KV cache and moving the accepted branch into
it) and ``TokenLogProbs``.

The GEMM family's weight argument is the T2B layout (``W4Weight``) instead
of the AIE ``aie::mmul<4,8,8>`` tile stream, which has no meaning off the
NPU; ``W4A16GEMV`` consumes the reference's own ``qparam`` rows unchanged.
"""

from __future__ import annotations

import math
from array import array
from dataclasses import dataclass, field
from typing import NamedTuple

import numpy as np
import torch

from . import _lib
from .weights import W4Weight

_HALF = (torch.bfloat16, torch.float16)


class ArgSpec(NamedTuple):
    direction: str
    shape: tuple
    dtype: torch.dtype


def _ws(nbytes: int, device) -> tuple[torch.Tensor, int]:
    n = max(int(nbytes), 256)
    t = torch.zeros(n, dtype=torch.uint8, device=device)
    return t, n


def _check_shape(t: torch.Tensor, shape, name: str):
    if tuple(t.shape) != tuple(shape) and t.numel() != int(torch.tensor(shape).prod()):
        raise ValueError(f"{name}: expected shape {tuple(shape)}, got {tuple(t.shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{name}: must be contiguous")


@dataclass
class W4A16GEMV:
    """``y = x . W^T`` over the reference ``qparam`` rows: a batch-1 GEMV, or
    ``num_batches`` rows, sharing one ``qparam`` (``shared_qparam``, one
    launch over all rows) or each with its own (one launch per row, as the
    reference's per-batch arg spec lays them out).  ``M`` not a multiple of
    the kernel's 128-row tile runs on a zero-padded copy of the rows."""

    M: int
    K: int
    num_aie_columns: int = 1
    tile_size_input: int = 2
    tile_size_output: int | None = None
    num_batches: int = 1
    shared_qparam: bool = False
    group_size: int = 128
    kernel_vector_size: int = field(default=32, repr=False)
    context: object = field(default=None, repr=False)

    def __post_init__(self):
        if self.tile_size_output is None:
            self.tile_size_output = self.tile_size_input
        if self.K % 2 != 0:
            raise ValueError("K must be even for packed int4 weights")
        if self.K % self.group_size != 0:
            raise ValueError("K must be a multiple of group_size")
        if self.kernel_vector_size != 32:
            raise ValueError("W4A16GEMV currently supports kernel_vector_size=32 only")
        if self.group_size % self.kernel_vector_size != 0:
            raise ValueError("group_size must be a multiple of kernel_vector_size")
        if not (self.tile_size_output % self.tile_size_input == 0 and self.tile_size_output >= self.tile_size_input):
            raise ValueError("tile_size_output must be a multiple of tile_size_input")
        # B200 kernel constraints
        if self.group_size != 128:
            raise ValueError("the B200 kernel supports group_size=128")
        if self.K % 256:
            raise ValueError("the B200 kernel needs K % 256 == 0")

    @property
    def num_groups(self) -> int:
        return self.K // self.group_size

    @property
    def qparam_row_bytes(self) -> int:
        return self.K // 2 + self.num_groups * 2

    def get_arg_spec(self):
        batch_dim = (self.num_batches,) if self.num_batches > 1 else ()
        qparam_dim = () if self.shared_qparam else batch_dim
        return [ArgSpec("in", qparam_dim + (self.M, self.qparam_row_bytes), torch.uint8),
                ArgSpec("in", batch_dim + (self.K,), torch.bfloat16),
                ArgSpec("out", batch_dim + (self.M,), torch.bfloat16)]

    def __call__(self, qparam: torch.Tensor, x: torch.Tensor, y: torch.Tensor) -> torch.Tensor:
        for t, spec, nm in zip((qparam, x, y), self.get_arg_spec(), ("qparam", "x", "y")):
            _check_shape(t, spec.shape, nm)
        L = _lib.lib()
        rows = self.num_batches
        n_pad = -(-self.M // 128) * 128
        per_batch = rows > 1 and not self.shared_qparam
        qp = qparam.reshape(rows if per_batch else 1, self.M, self.qparam_row_bytes)
        if n_pad != self.M:                                   # rows past M: zero weights and scales
            padded = torch.zeros(qp.shape[0], n_pad, self.qparam_row_bytes, dtype=torch.uint8, device=qp.device)
            padded[:, :self.M].copy_(qp)
            qp = padded
            out = torch.empty(rows, n_pad, dtype=y.dtype, device=y.device)
        else:
            out = y.reshape(rows, self.M)
        xr = x.reshape(rows, self.K)
        ws, n = _ws(L.t2b_w4a16_gemm_workspace_bytes(1 if per_batch else rows, n_pad, self.K), qparam.device)
        calls = [(qp[b], xr[b:b + 1], out[b:b + 1], 1) for b in range(rows)] if per_batch else \
            [(qp[0], xr, out, rows)]
        for w, xb, yb, m in calls:
            _lib.call("t2b_w4a16_gemm", _lib.ptr(w), None, _lib.WFMT_QPARAM, _lib.ptr(xb), _lib.DTYPE[x.dtype],
                      _lib.ptr(yb), _lib.DTYPE[y.dtype], m, n_pad, self.K, self.group_size, _lib.ptr(ws), n,
                      _lib.stream())
        if n_pad != self.M:
            y.reshape(rows, self.M).copy_(out[:, :self.M])
        return y


@dataclass
class W4A16GEMM:
    """``C[M,N] = A[M,K] . W^T`` with ``W`` a T2B ``W4Weight`` ``[N, K]``."""

    M: int
    K: int
    N: int
    num_aie_columns: int = 8
    num_aie_rows: int = 4
    tile_m: int = 8
    tile_k: int = 128
    tile_n: int = 64
    group_size: int = 128
    context: object = field(default=None, repr=False)

    def __post_init__(self):
        self._reference_checks()
        if self.group_size != 128 or self.K % 256 or self.N % 128:
            raise ValueError("the B200 kernel needs group_size=128, K % 256 == 0, N % 128 == 0")

    def _reference_checks(self):
        if self.tile_k != self.group_size:
            raise ValueError("W4A16GEMM currently requires tile_k == group_size")
        if self.K % self.tile_k != 0:
            raise ValueError("K must be a multiple of tile_k")

    def get_arg_spec(self):
        return [ArgSpec("in", (self.M, self.K), torch.bfloat16),
                ArgSpec("in", (self.N, self.K // 2), torch.uint8),
                ArgSpec("out", (self.M, self.N), torch.bfloat16)]

    def __call__(self, a: torch.Tensor, w: W4Weight, c: torch.Tensor) -> torch.Tensor:
        if (w.out_features, w.in_features) != (self.N, self.K):
            raise ValueError("weight shape does not match the operator")
        _check_shape(a, (self.M, self.K), "A")
        _check_shape(c, (self.M, self.N), "C")
        L = _lib.lib()
        ws, n = _ws(L.t2b_w4a16_gemm_workspace_bytes(self.M, self.N, self.K), a.device)
        _lib.call("t2b_w4a16_gemm", _lib.ptr(w.qw), _lib.ptr(w.meta), _lib.WFMT_T2B, _lib.ptr(a), _lib.DTYPE[a.dtype],
                  _lib.ptr(c), _lib.DTYPE[c.dtype], self.M, self.N, self.K, self.group_size, _lib.ptr(ws), n,
                  _lib.stream())
        return c


@dataclass
class W4A16KGroupGEMM(W4A16GEMM):
    """Same contraction; ``k_group`` (K tiles per AIE call) is a scheduling hint with no B200 meaning."""

    k_group: int = 2

    def _reference_checks(self):
        super()._reference_checks()
        if (self.K // self.tile_k) % self.k_group != 0:
            raise ValueError("k_tiles must be divisible by k_group")


@dataclass
class W4A16NShardGEMM(W4A16GEMM):
    pass


@dataclass
class W4A16PairedKGroupGEMM(W4A16KGroupGEMM):
    """One activation stream, two weights (K/V or gate/up), two outputs."""

    def get_arg_spec(self):
        return [ArgSpec("in", (self.M, self.K), torch.bfloat16),
                ArgSpec("in", (2, self.N, self.K // 2), torch.uint8),
                ArgSpec("out", (self.M, self.N), torch.bfloat16),
                ArgSpec("out", (self.M, self.N), torch.bfloat16)]

    def __call__(self, a: torch.Tensor, w_pair: W4Weight, c0: torch.Tensor, c1: torch.Tensor):
        """``w_pair`` holds the two weights row-concatenated (``weights.concat_rows``)."""
        if (w_pair.out_features, w_pair.in_features) != (2 * self.N, self.K):
            raise ValueError("paired weight must be [2N, K]")
        tmp = torch.empty(self.M, 2 * self.N, dtype=c0.dtype, device=a.device)
        W4A16GEMM(self.M, self.K, 2 * self.N)(a, w_pair, tmp)
        c0.copy_(tmp[:, :self.N])
        c1.copy_(tmp[:, self.N:])
        return c0, c1


@dataclass
class RMSNormRoPE:
    """Weighted RMSNorm then RoPE per row; ``rope_mode`` "interleaved" follows
    ``model.py:184-196`` (the CPU reference), "two_halves" follows the NPU
    kernel ``rms_norm_rope/kernel.cc:39-67``."""

    rows: int
    cols: int
    angle_rows: int
    num_aie_columns: int = 8
    epsilon: float = 1e-5
    rope_mode: str = "interleaved"
    context: object = field(default=None, repr=False)

    def __post_init__(self):
        if self.cols % 32 != 0:
            raise ValueError("cols must be divisible by 32")
        if self.rows % self.num_aie_columns != 0:
            raise ValueError("rows must be divisible by num_aie_columns")
        if self.angle_rows > self.rows or self.rows % self.angle_rows != 0:
            raise ValueError("angle_rows must divide rows")
        if self.angle_rows < self.num_aie_columns or self.angle_rows % self.num_aie_columns != 0:
            raise ValueError("angle_rows must be divisible by num_aie_columns")
        if self.epsilon <= 0:
            raise ValueError("epsilon must be positive")
        if self.rope_mode not in ("interleaved", "two_halves"):
            raise ValueError("rope_mode must be 'interleaved' or 'two_halves'")

    def get_arg_spec(self):
        bf = torch.bfloat16
        return [ArgSpec("in", (self.rows, self.cols), bf), ArgSpec("in", (self.cols,), bf),
                ArgSpec("in", (self.angle_rows, self.cols), bf), ArgSpec("out", (self.rows, self.cols), bf)]

    def __call__(self, inp, w, angles, out):
        for t, spec, nm in zip((inp, w, angles, out), self.get_arg_spec(), ("in", "w", "angles", "out")):
            _check_shape(t, spec.shape, nm)
        _lib.call("t2b_rms_norm_rope", _lib.ptr(inp), _lib.ptr(w), _lib.ptr(angles), _lib.ptr(out), self.rows,
                  self.cols, self.angle_rows, self.epsilon, 0 if self.rope_mode == "interleaved" else 1,
                  _lib.stream())
        return out


@dataclass
class LlamaChunkedAttention:
    """GQA decode attention over the packet cache (mask-skipped slots)."""

    max_seq_len: int
    num_kv_groups: int = 8
    q_heads_per_group: int = 4
    head_dim: int = 64
    chunk_size: int = 64
    packed_fifo_depth: int | None = None
    kernel_vector_size: int = field(default=32, repr=False)
    context: object = field(default=None, repr=False)

    def __post_init__(self):
        if self.max_seq_len <= 0:
            raise ValueError("max_seq_len must be positive")
        if self.chunk_size <= 0:
            raise ValueError("chunk_size must be positive")
        if self.max_seq_len % self.chunk_size != 0:
            raise ValueError("max_seq_len must be divisible by chunk_size")
        if self.num_kv_groups <= 0:
            raise ValueError("num_kv_groups must be positive")
        if self.q_heads_per_group <= 0:
            raise ValueError("q_heads_per_group must be positive")
        if self.head_dim <= 0:
            raise ValueError("head_dim must be positive")
        if self.head_dim % self.kernel_vector_size != 0:
            raise ValueError("head_dim must be divisible by kernel_vector_size")
        if self.chunk_size != 64 or self.head_dim not in (64, 128) or self.q_heads_per_group not in (1, 2, 4, 8):
            raise ValueError("the B200 kernel needs chunk_size=64, head_dim in (64,128), q_heads_per_group in 1/2/4/8")

    @property
    def packed_chunk_elements(self):
        return 2 * self.chunk_size * self.head_dim + self.chunk_size

    @property
    def packed_elements(self):
        return self.num_kv_groups * (self.max_seq_len // self.chunk_size) * self.packed_chunk_elements

    def get_arg_spec(self):
        bf = torch.bfloat16
        q = (self.num_kv_groups, self.q_heads_per_group, self.head_dim)
        return [ArgSpec("in", q, bf), ArgSpec("in", (self.packed_elements,), bf), ArgSpec("out", q, bf)]

    def __call__(self, q, packet, out):
        for t, spec, nm in zip((q, packet, out), self.get_arg_spec(), ("Q", "packet", "out")):
            _check_shape(t, spec.shape, nm)
        L = _lib.lib()
        ws, n = _ws(L.t2b_decode_attention_workspace_bytes(1, self.num_kv_groups * self.q_heads_per_group,
                                                           self.num_kv_groups, self.head_dim, self.max_seq_len),
                    q.device)
        _lib.call("t2b_packet_attention", _lib.ptr(q), _lib.ptr(packet), _lib.ptr(out), self.num_kv_groups,
                  self.q_heads_per_group, self.head_dim, self.max_seq_len, self.chunk_size, _lib.ptr(ws), n,
                  _lib.stream())
        return out


@dataclass
class ResidualAddRMSNorm:
    size: int
    num_aie_columns: int
    tile_size: int
    epsilon: float = 1e-5
    context: object = field(default=None, repr=False)

    def __post_init__(self):
        if self.epsilon <= 0:
            raise ValueError("epsilon must be positive")
        if self.size % (self.num_aie_columns * self.tile_size) != 0:
            raise ValueError("size must be divisible by num_aie_columns * tile_size")

    def get_arg_spec(self):
        bf = torch.bfloat16
        return [ArgSpec("in", (self.size,), bf), ArgSpec("in", (self.size,), bf), ArgSpec("in", (self.tile_size,), bf),
                ArgSpec("out", (self.size,), bf), ArgSpec("out", (self.size,), bf)]

    def __call__(self, x, update, w, x_out, norm_out):
        for t, spec, nm in zip((x, update, w, x_out, norm_out), self.get_arg_spec(),
                               ("x", "update", "w", "x_out", "norm_out")):
            _check_shape(t, spec.shape, nm)
        _lib.call("t2b_residual_add_rms_norm", _lib.ptr(x), _lib.ptr(update), _lib.ptr(w), _lib.ptr(x_out),
                  _lib.ptr(norm_out), self.size, self.tile_size, self.epsilon, _lib.stream())
        return x_out, norm_out


@dataclass
class SiLUMul:
    size: int
    tile_size: int
    num_aie_columns: int = 8
    context: object = field(default=None, repr=False)

    def __post_init__(self):
        if self.size % (self.num_aie_columns * self.tile_size) != 0:
            raise ValueError(f"size ({self.size}) must be a multiple of "
                             f"num_aie_columns * tile_size ({self.num_aie_columns * self.tile_size})")

    def get_arg_spec(self):
        bf = torch.bfloat16
        return [ArgSpec("in", (self.size,), bf), ArgSpec("in", (self.size,), bf), ArgSpec("out", (self.size,), bf)]

    def __call__(self, a, b, out):
        for t, spec, nm in zip((a, b, out), self.get_arg_spec(), ("left", "right", "out")):
            _check_shape(t, spec.shape, nm)
        _lib.call("t2b_silu_mul", _lib.ptr(a), _lib.ptr(b), _lib.ptr(out), self.size, _lib.stream())
        return out


@dataclass
class CopyPresentPacketKV:
    kv_dim: int
    num_kv_groups: int
    head_dim: int
    packet_elements: int
    packet_elements_per_group: int
    key_packet_offset: int
    value_packet_offset: int
    dtype: object = field(default=torch.bfloat16, repr=False)
    transfer_size: int | None = None
    mask_packet_offset: int | None = None
    context: object = field(default=None, repr=False)

    def __post_init__(self):
        if self.kv_dim != self.num_kv_groups * self.head_dim:
            raise ValueError("kv_dim must equal num_kv_groups * head_dim")

    def get_arg_spec(self):
        bf = torch.bfloat16
        return [ArgSpec("in", (self.kv_dim,), bf), ArgSpec("in", (self.kv_dim,), bf),
                ArgSpec("out", (self.kv_dim,), bf), ArgSpec("out", (self.kv_dim,), bf),
                ArgSpec("out", (self.packet_elements,), bf)]

    def __call__(self, k, v, present_k, present_v, packet):
        for t, spec, nm in zip((k, v, present_k, present_v, packet), self.get_arg_spec(),
                               ("key", "value", "present_key", "present_value", "packet")):
            _check_shape(t, spec.shape, nm)
        moff = -1 if self.mask_packet_offset is None else self.mask_packet_offset
        _lib.call("t2b_copy_present_packet_kv", _lib.ptr(k), _lib.ptr(v), _lib.ptr(present_k), _lib.ptr(present_v),
                  _lib.ptr(packet), self.num_kv_groups, self.head_dim, self.packet_elements_per_group,
                  self.key_packet_offset, self.value_packet_offset, moff, _lib.stream())
        return present_k, present_v, packet


# ---------------------------------------------------------------------------
# serving operators
# ---------------------------------------------------------------------------
def _check_arg(name: str, t: torch.Tensor, shape: tuple, dtype: torch.dtype, dev: int, contiguous: bool = True) -> None:
    """Shape, type, device (the current one, ``dev``) and layout of one argument."""
    if t.shape == shape and t.dtype is dtype and t.get_device() == dev and (not contiguous or t.is_contiguous()):
        return
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name}: expected shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.dtype != dtype:
        raise ValueError(f"{name}: expected {dtype}, got {t.dtype}")
    if not t.is_cuda or t.get_device() != dev:
        raise ValueError(f"{name}: expected a tensor on the current CUDA device, got {t.device}")
    raise ValueError(f"{name}: must be contiguous")


def _current_device(t: torch.Tensor) -> int:
    """The current device's index (-2, which no tensor has, where there is none)."""
    return torch._C._cuda_getDevice() if t.is_cuda else -2


def _strides(name: str, t: torch.Tensor) -> list[int]:
    """Element strides of every axis but the last (contiguous) one, as the
    kernels take them: nonzero multiples of 8 on a 16-byte aligned base."""
    *out, inner = t.stride()
    low = 0
    for s in out:
        low |= s
    if inner == 1 and low % 8 == 0 and t.data_ptr() % 16 == 0 and 0 not in out:
        return out
    shape = t.shape
    if inner != 1 and shape[-1] > 1:
        raise ValueError(f"{name}: the last axis must be contiguous")
    if t.data_ptr() % 16:
        raise ValueError(f"{name}: must start on a 16-byte boundary")
    for i, s in enumerate(out):
        if shape[i] == 1:
            out[i] = 8                                 # an axis of one has no stride
        elif s % 8 or s == 0:
            raise ValueError(f"{name}: strides {t.stride()} must be nonzero multiples of 8 elements")
    return out


def _addr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _check_heads(op) -> None:
    if op.num_kv_groups <= 0:
        raise ValueError("num_kv_groups must be positive")
    if not 0 < op.q_heads_per_group <= 128:
        raise ValueError("q_heads_per_group must be in 1..128")
    if op.head_dim not in (64, 128):
        raise ValueError("the B200 kernel needs head_dim in (64, 128)")
    if op.dtype not in _HALF:
        raise ValueError("dtype must be torch.bfloat16 or torch.float16")
    if op.out_dtype is None:
        op.out_dtype = op.dtype
    if op.out_dtype not in _HALF:
        raise ValueError("out_dtype must be torch.bfloat16 or torch.float16")
    if op.scale is None:
        op.scale = 1.0 / math.sqrt(op.head_dim)
    if not 2.0 ** -149 <= op.scale < 2.0 ** 127:      # the kernels' fp32 scale * log2(e)
        raise ValueError("scale must be positive and finite in 32 bits")


@dataclass
class PackedAttention:
    """Causal GQA attention over ``num_seqs`` packed sequences of different lengths.

    ``q`` and ``out`` hold the queries of all sequences one after the other,
    sequence s in rows ``q_start[s]`` to ``q_start[s + 1] - 1``; query i of its
    n queries sees keys 0 .. k_len - n + i.  Without ``max_ctx`` the keys are
    packed ``[kv_tokens, num_kv_groups, head_dim]``, as the queries are or, with
    ``k_start`` and ``k_len``, from row ``k_start[s]`` on.  With ``max_ctx`` they
    are cache rows ``[num_seqs, num_kv_groups, max_ctx, head_dim]`` and ``k_len``
    says how many of each row count, the sequence's own queries among them.
    A query without keys gets zeros (and ``lse`` -inf); rows of ``out`` and
    ``lse`` outside every sequence keep what they held.  ``out`` may be ``q``
    itself, and otherwise shares no memory with the inputs.  A call that could have
    more than 2^31 - 1 units of work (``t2b_packed_attention``; one prompt of 1.4
    million tokens at 32 over 8 heads) is refused.  A device wait that ran out is
    seen in the status word bound to the stream (``_lib.status_word``), and there
    alone; its rows are not to be used."""

    tokens: int
    num_seqs: int
    num_kv_groups: int = 8
    q_heads_per_group: int = 4
    head_dim: int = 64
    kv_tokens: int | None = None
    max_ctx: int | None = None
    dtype: torch.dtype = torch.bfloat16
    out_dtype: torch.dtype | None = None
    scale: float | None = None

    def __post_init__(self):
        if self.tokens <= 0:
            raise ValueError("tokens must be positive")
        if self.num_seqs <= 0:
            raise ValueError("num_seqs must be positive")
        if self.max_ctx is not None and (self.max_ctx <= 0 or self.kv_tokens is not None):
            raise ValueError("max_ctx (cache rows) must be positive and excludes kv_tokens (packed keys)")
        if self.max_ctx is None and self.kv_tokens is None:
            self.kv_tokens = self.tokens
        if self.kv_tokens is not None and self.kv_tokens <= 0:
            raise ValueError("kv_tokens must be positive")
        _check_heads(self)

    @property
    def num_heads(self) -> int:
        return self.num_kv_groups * self.q_heads_per_group

    def _kv_shape(self) -> tuple:
        if self.max_ctx is None:
            return (self.kv_tokens, self.num_kv_groups, self.head_dim)
        return (self.num_seqs, self.num_kv_groups, self.max_ctx, self.head_dim)

    def get_arg_spec(self):
        q = (self.tokens, self.num_heads, self.head_dim)
        return [ArgSpec("in", q, self.dtype), ArgSpec("in", self._kv_shape(), self.dtype),
                ArgSpec("in", self._kv_shape(), self.dtype), ArgSpec("in", (self.num_seqs + 1,), torch.int32),
                ArgSpec("out", q, self.out_dtype)]

    def __call__(self, q, k, v, q_start, out, k_start=None, k_len=None, lse=None):
        dev, cached, i32 = _current_device(q), self.max_ctx is not None, torch.int32
        rows, kv = (self.tokens, self.num_heads, self.head_dim), self._kv_shape()
        _check_arg("q", q, rows, self.dtype, dev, False)
        _check_arg("k", k, kv, self.dtype, dev, False)
        _check_arg("v", v, kv, self.dtype, dev, False)
        _check_arg("q_start", q_start, (self.num_seqs + 1,), i32, dev)
        _check_arg("out", out, rows, self.out_dtype, dev, False)
        if cached and (k_start is not None or k_len is None):
            raise ValueError("cache rows take k_len and no k_start")
        if not cached and (k_start is None) != (k_len is None):
            raise ValueError("packed keys take k_start and k_len together")
        if not cached and k_start is None and self.kv_tokens != self.tokens:
            raise ValueError("keys without k_start are packed as the queries are: kv_tokens must equal tokens")
        if k_start is not None:
            _check_arg("k_start", k_start, (self.num_seqs,), i32, dev)
        if k_len is not None:
            _check_arg("k_len", k_len, (self.num_seqs,), i32, dev)
        if lse is not None:
            _check_arg("lse", lse, rows[:2], torch.float32, dev)
        qs, os, ks, vs = _strides("q", q), _strides("out", out), _strides("k", k), _strides("v", v)
        if cached:       # (row, head, token) -> (token, head, row)
            ks.reverse()
            vs.reverse()
        else:
            ks.append(8)
            vs.append(8)
        L = _lib.load()
        n = L.t2b_varlen_attention_workspace_bytes(self.head_dim)
        ws = torch.empty(n, dtype=torch.uint8, device=q.device)
        _lib.check("t2b_packed_attention", L.t2b_packed_attention(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), _addr(lse), _lib.DTYPE[self.dtype],
            _lib.DTYPE[self.out_dtype], q_start.data_ptr(), _addr(k_start), _addr(k_len), self.num_seqs, self.tokens,
            self.num_seqs if cached else 0, kv[2] if cached else kv[0], rows[1], self.num_kv_groups, self.head_dim, *qs,
            *os, *ks, *vs, self.scale, ws.data_ptr(), n, _lib.raw_stream(dev)))
        return out


def draft_tree(parents, num_nodes=None) -> tuple[torch.Tensor, torch.Tensor]:
    """Host helper: ``(mask, depth)`` of drafted trees ``parents [batch, nodes]``.

    Node 0 is the root (its parent entry is not read); every other node's
    parent precedes it.  ``mask`` int64 ``[batch, nodes, (nodes + 63) // 64]``
    has the bits of each node's ancestors and of the node itself, ``depth``
    int32 ``[batch, nodes]`` its distance from the root.  Nodes from
    ``num_nodes[b]`` on get an empty mask and depth 0."""
    par = np.asarray(parents.cpu() if isinstance(parents, torch.Tensor) else parents)
    if par.ndim != 2 or par.shape[1] < 1 or not np.issubdtype(par.dtype, np.integer):
        raise ValueError("parents must be integers [batch, nodes]")
    B, T = par.shape
    live = np.full(B, T) if num_nodes is None else \
        np.asarray(num_nodes.cpu() if isinstance(num_nodes, torch.Tensor) else num_nodes).reshape(-1)
    if live.shape != (B,) or live.dtype.kind not in "biuf" or not ((live >= 0) & (live <= T) & (live == np.trunc(live))).all():
        raise ValueError(f"num_nodes must be {B} whole numbers in 0..{T}")
    node = np.arange(T)
    used = node[None] < live[:, None]
    if (used & (node[None] > 0) & ((par < 0) | (par >= node[None]))).any():
        raise ValueError("a node's parent must precede it")
    sees = np.zeros((B, T, T), bool)
    depth = np.zeros((B, T), np.int32)
    rows = np.arange(B)
    for i in range(T):
        if i:
            up = np.where(used[:, i], par[:, i], 0)
            sees[:, i] = sees[rows, up]
            depth[:, i] = depth[rows, up] + 1
        sees[:, i, i] = True
        sees[~used[:, i], i] = False
        depth[~used[:, i], i] = 0
    words = (T + 63) // 64
    bits = np.zeros((B, T, words * 64), np.uint8)
    bits[:, :, :T] = sees
    packed = np.packbits(bits, axis=2, bitorder="little")
    return torch.from_numpy(packed.view("<i8").reshape(B, T, words).copy()), torch.from_numpy(depth)


@dataclass
class DraftTreeAttention:
    """GQA attention of ``nodes`` drafted tokens per batch row over the KV cache.

    Node i of row b sees the ``ctx_len[b]`` cached keys of its row and the
    drafted nodes whose bit is set in ``mask[b, i]`` (``draft_tree``); the
    drafted K/V stay outside the cache until ``DraftTreeCommit`` moves the
    accepted ones.  Nodes from ``num_nodes[b]`` on are not computed: their rows
    of ``out`` and ``lse`` keep what they held.  ``out`` may be ``q`` itself, and
    otherwise shares no memory with the inputs.  A device wait that ran out is
    seen in the stream's status word, as for ``PackedAttention``."""

    batch: int
    nodes: int
    max_ctx: int
    num_kv_groups: int = 8
    q_heads_per_group: int = 4
    head_dim: int = 64
    dtype: torch.dtype = torch.bfloat16
    out_dtype: torch.dtype | None = None
    scale: float | None = None

    def __post_init__(self):
        if self.batch <= 0:
            raise ValueError("batch must be positive")
        if not 0 < self.nodes <= 256:
            raise ValueError("the B200 kernel needs nodes in 1..256")
        if self.max_ctx <= 0:
            raise ValueError("max_ctx must be positive")
        _check_heads(self)

    @property
    def num_heads(self) -> int:
        return self.num_kv_groups * self.q_heads_per_group

    @property
    def mask_words(self) -> int:
        return (self.nodes + 63) // 64

    def get_arg_spec(self):
        q = (self.batch, self.nodes, self.num_heads, self.head_dim)
        cache = (self.batch, self.num_kv_groups, self.max_ctx, self.head_dim)
        draft = (self.batch, self.nodes, self.num_kv_groups, self.head_dim)
        return [ArgSpec("in", q, self.dtype), ArgSpec("in", cache, self.dtype), ArgSpec("in", cache, self.dtype),
                ArgSpec("in", draft, self.dtype), ArgSpec("in", draft, self.dtype),
                ArgSpec("in", (self.batch,), torch.int32),
                ArgSpec("in", (self.batch, self.nodes, self.mask_words), torch.int64), ArgSpec("out", q, self.out_dtype)]

    def __call__(self, q, k_cache, v_cache, k_draft, v_draft, ctx_len, mask, out, num_nodes=None, lse=None):
        dev, B, T, hd = _current_device(q), self.batch, self.nodes, self.head_dim
        rows, draft = (B, T, self.num_heads, hd), (B, T, self.num_kv_groups, hd)
        cache = (B, self.num_kv_groups, self.max_ctx, hd)
        _check_arg("q", q, rows, self.dtype, dev, False)
        _check_arg("k_cache", k_cache, cache, self.dtype, dev)
        _check_arg("v_cache", v_cache, cache, self.dtype, dev)
        _check_arg("k_draft", k_draft, draft, self.dtype, dev, False)
        _check_arg("v_draft", v_draft, draft, self.dtype, dev, False)
        _check_arg("ctx_len", ctx_len, (B,), torch.int32, dev)
        _check_arg("mask", mask, (B, T, self.mask_words), torch.int64, dev)
        _check_arg("out", out, rows, self.out_dtype, dev, False)
        if num_nodes is not None:
            _check_arg("num_nodes", num_nodes, (B,), torch.int32, dev)
        if lse is not None:
            _check_arg("lse", lse, rows[:3], torch.float32, dev)
        if k_cache.data_ptr() % 16 or v_cache.data_ptr() % 16:
            raise ValueError("the caches must start on a 16-byte boundary")
        qs, os = self._rows("q", q), self._rows("out", out)
        kd, vd = _strides("k_draft", k_draft), _strides("v_draft", v_draft)
        L = _lib.load()
        n = L.t2b_varlen_attention_workspace_bytes(hd)
        ws = torch.empty(n, dtype=torch.uint8, device=q.device)
        _lib.check("t2b_tree_attention", L.t2b_tree_attention(
            q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), k_draft.data_ptr(), v_draft.data_ptr(), out.data_ptr(),
            _addr(lse), _lib.DTYPE[self.dtype], _lib.DTYPE[self.out_dtype], ctx_len.data_ptr(), _addr(num_nodes),
            mask.data_ptr(), B, T, rows[2], self.num_kv_groups, hd, self.max_ctx, *qs, *os, *kd, *vd, self.scale,
            ws.data_ptr(), n, _lib.raw_stream(dev)))
        return out

    def _rows(self, name, t) -> list[int]:
        """(row, head) strides of ``[batch, nodes, ..]`` seen as ``[batch * nodes, ..]``."""
        b, node, head = _strides(name, t)
        if self.nodes == 1:
            return [b, head]
        if self.batch > 1 and b != self.nodes * node:
            raise ValueError(f"{name}: the nodes of consecutive batch rows must follow one another")
        return [node, head]


@dataclass
class DraftTreeCommit:
    """Greedy walk through each row's verified tree, and the move of the
    accepted nodes' K/V rows of every layer into the caches.

    From node c the walk goes to the lowest later node n with ``parents[n] ==
    c`` and ``tokens[n] == predicted[c]`` (``predicted``: the model's token
    after each node), while the cache has room.  ``k_drafts`` / ``v_drafts``
    are ``[layers, batch, nodes, kv, head_dim]`` or a sequence of one tensor per
    layer, ``k_caches`` / ``v_caches`` likewise ``[layers, batch, kv, max_ctx,
    head_dim]``.  Writes ``path`` (-1 behind the walk's end), ``num_accepted``,
    ``next_token`` and ``new_len = ctx_len + num_accepted``; they and the caches
    share no memory with the drafts, the other inputs or one another.  A row with
    no live node or no room accepts nothing (next token -1)."""

    layers: int
    batch: int
    nodes: int
    max_ctx: int
    num_kv_groups: int = 8
    head_dim: int = 64
    dtype: torch.dtype = torch.bfloat16

    def __post_init__(self):
        if self.layers <= 0 or self.batch <= 0:
            raise ValueError("layers and batch must be positive")
        if not 0 < self.nodes <= 256:
            raise ValueError("the B200 kernel needs nodes in 1..256")
        if self.max_ctx <= 0:
            raise ValueError("max_ctx must be positive")
        if not 0 < self.num_kv_groups <= 1024:
            raise ValueError("num_kv_groups must be in 1..1024")
        if self.head_dim <= 0 or self.head_dim % 8 or self.head_dim > 1024:
            raise ValueError("head_dim must be a multiple of 8, at most 1024")
        if self.dtype not in _HALF:
            raise ValueError("dtype must be torch.bfloat16 or torch.float16")

    def get_arg_spec(self):
        i32, tree = torch.int32, (self.batch, self.nodes)
        draft = (self.layers, self.batch, self.nodes, self.num_kv_groups, self.head_dim)
        cache = (self.layers, self.batch, self.num_kv_groups, self.max_ctx, self.head_dim)
        return [ArgSpec("in", tree, i32), ArgSpec("in", tree, i32), ArgSpec("in", tree, i32),
                ArgSpec("in", (self.batch,), i32), ArgSpec("in", draft, self.dtype), ArgSpec("in", draft, self.dtype),
                ArgSpec("inout", cache, self.dtype), ArgSpec("inout", cache, self.dtype), ArgSpec("out", tree, i32),
                ArgSpec("out", (self.batch,), i32), ArgSpec("out", (self.batch,), i32),
                ArgSpec("out", (self.batch,), i32)]

    def _layers(self, name: str, ts, shape: tuple, dev: int, contiguous: bool):
        """Host array of the layers' device pointers (64 bits each), and the strides they share."""
        if isinstance(ts, torch.Tensor):
            _check_arg(name, ts, (self.layers, *shape), self.dtype, dev, False)
            step, *strides = _strides(name, ts)
            if contiguous and not ts.is_contiguous() and not ts[0].is_contiguous():
                raise ValueError(f"{name}: must be contiguous")
            base, step = ts.data_ptr(), step * 2
            at = array("Q", range(base, base + step * self.layers, step))
        else:
            if len(ts) != self.layers:
                raise ValueError(f"{name}: expected {self.layers} layers, got {len(ts)}")
            layout = ts[0].stride()
            for t in ts:
                _check_arg(name, t, shape, self.dtype, dev, contiguous)
                if t.stride() != layout:
                    raise ValueError(f"{name}: the layers' strides differ")
            strides = _strides(name, ts[0])
            at = array("Q", [t.data_ptr() for t in ts])
            if any(a % 16 for a in at):
                raise ValueError(f"{name}: must start on a 16-byte boundary")
        return at, strides

    def __call__(self, tokens, parents, predicted, ctx_len, k_drafts, v_drafts, k_caches, v_caches, path, num_accepted,
                 next_token, new_len, num_nodes=None):
        dev, i32, tree, row = _current_device(tokens), torch.int32, (self.batch, self.nodes), (self.batch,)
        _check_arg("tokens", tokens, tree, i32, dev)
        _check_arg("parents", parents, tree, i32, dev)
        _check_arg("predicted", predicted, tree, i32, dev)
        _check_arg("ctx_len", ctx_len, row, i32, dev)
        _check_arg("path", path, tree, i32, dev)
        _check_arg("num_accepted", num_accepted, row, i32, dev)
        _check_arg("next_token", next_token, row, i32, dev)
        _check_arg("new_len", new_len, row, i32, dev)
        if num_nodes is not None:
            _check_arg("num_nodes", num_nodes, row, i32, dev)
        draft = (self.batch, self.nodes, self.num_kv_groups, self.head_dim)
        cache = (self.batch, self.num_kv_groups, self.max_ctx, self.head_dim)
        kd, kds = self._layers("k_drafts", k_drafts, draft, dev, False)
        vd, vds = self._layers("v_drafts", v_drafts, draft, dev, False)
        kc, _ = self._layers("k_caches", k_caches, cache, dev, True)
        vc, _ = self._layers("v_caches", v_caches, cache, dev, True)
        _lib.check("t2b_tree_commit", _lib.load().t2b_tree_commit(
            tokens.data_ptr(), parents.data_ptr(), predicted.data_ptr(), ctx_len.data_ptr(), _addr(num_nodes),
            *(a.buffer_info()[0] for a in (kd, vd, kc, vc)), self.layers, path.data_ptr(), num_accepted.data_ptr(),
            next_token.data_ptr(), new_len.data_ptr(), self.batch, self.nodes, self.num_kv_groups, self.head_dim,
            self.max_ctx, *kds, *vds, _lib.raw_stream(dev)))
        return path, num_accepted, next_token, new_len


@dataclass
class TokenLogProbs:
    """Log probabilities of given tokens over logits rows, with the entropy and
    the ``num_top`` most likely tokens of each row (largest first, ties to the
    lowest index), in fp32.

    ``logits [rows, vocab]`` may have a row stride above ``vocab``.  A token
    outside the vocabulary gets NaN; a value of -inf is masked out, and a row of
    nothing else gets log probabilities -inf and entropy 0."""

    rows: int
    vocab: int
    num_top: int = 0
    dtype: torch.dtype = torch.float32

    def __post_init__(self):
        if self.rows <= 0 or self.vocab <= 0:
            raise ValueError("rows and vocab must be positive")
        if not 0 <= self.num_top <= min(32, self.vocab):
            raise ValueError("num_top must be in 0..min(32, vocab)")
        if self.dtype not in _lib.DTYPE:
            raise ValueError("dtype must be torch.float32, torch.bfloat16 or torch.float16")

    def get_arg_spec(self):
        f32, row = torch.float32, (self.rows,)
        spec = [ArgSpec("in", (self.rows, self.vocab), self.dtype), ArgSpec("in", row, torch.int32),
                ArgSpec("out", row, f32), ArgSpec("out", row, f32)]
        if self.num_top:
            spec += [ArgSpec("out", (self.rows, self.num_top), f32),
                     ArgSpec("out", (self.rows, self.num_top), torch.int32)]
        return spec

    def __call__(self, logits, tokens, logprob, entropy=None, top_logprob=None, top_index=None, lse=None):
        dev, f32, row, top = _current_device(logits), torch.float32, (self.rows,), (self.rows, self.num_top)
        _check_arg("logits", logits, (self.rows, self.vocab), self.dtype, dev, False)
        ld = logits.stride(0) if self.rows > 1 else self.vocab
        if self.vocab > 1 and logits.stride(1) != 1 or ld < self.vocab:
            raise ValueError("logits: rows must be contiguous and must not overlap")
        _check_arg("tokens", tokens, row, torch.int32, dev)
        _check_arg("logprob", logprob, row, f32, dev)
        if entropy is not None:
            _check_arg("entropy", entropy, row, f32, dev)
        if lse is not None:
            _check_arg("lse", lse, row, f32, dev)
        if (self.num_top > 0) != (top_logprob is not None) or (self.num_top > 0) != (top_index is not None):
            raise ValueError("top_logprob and top_index go with num_top > 0")
        if self.num_top:
            _check_arg("top_logprob", top_logprob, top, f32, dev)
            _check_arg("top_index", top_index, top, torch.int32, dev)
        _lib.check("t2b_token_logprobs", _lib.load().t2b_token_logprobs(
            logits.data_ptr(), _lib.DTYPE[self.dtype], self.rows, self.vocab, ld, tokens.data_ptr(), logprob.data_ptr(),
            _addr(entropy), _addr(lse), self.num_top, _addr(top_logprob), _addr(top_index), _lib.raw_stream(dev)))
        return logprob
