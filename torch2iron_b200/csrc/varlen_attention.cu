// Attention over sequences of different lengths: packed prompts (causal) and
// trees of drafted tokens over the KV cache.
//
//   out[r, h] = sum_j softmax_j(scale * q[r, h] . k[j, h / qpg]) v[j, h / qpg]
//
// over the keys row r sees.  Packed: row r is query i of the n queries of its
// sequence and sees keys 0 .. k_len - n + i (model.py:266-279 without
// padding).  Tree: row r is node i of batch row b and sees the ctx_len[b]
// cached keys and the drafted nodes whose bit is set in mask[b][i].
//
// One warp per (row, head): the lanes hold head_dim / 32 components each, the
// dot product is a warp sum, and the running maximum, sum and output of the
// softmax stay in fp32 registers.

#include <math.h>

#include "t2b_common.cuh"
#include "launch.cuh"

namespace t2b {

constexpr int VA_MAX_NODES = 256;

struct VaParams {
  const void *q, *k, *v, *kd, *vd;   // kd, vd: drafted nodes (tree)
  void* out;
  float* lse;                         // [rows][n_heads] (nullable)
  int f16, out_f16;
  int rows, n_heads, qpg, n_seqs;
  size_t q_row, q_head, o_row, o_head;
  size_t k_tok, k_head, k_seq, v_tok, v_head, v_seq;
  size_t kd_row, kd_node, kd_head, vd_row, vd_node, vd_head;
  int kv_tokens;                      // token extent of k and v
  int cached;                         // keys of sequence s live in cache row s
  const int *q_start, *k_start, *k_len;          // packed
  const int *ctx_len, *n_nodes;                  // tree
  const unsigned long long* mask;                // [B][T][words]
  int T, words;                                  // T > 0: tree
  float scale_log2;
};

template <int E>
T2B_DEV void va_load(const void* p, size_t off, int f16, int lane, float (&x)[E]) {
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const size_t i = off + lane * E + e;
    x[e] = f16 ? __half2float(static_cast<const __half*>(p)[i]) : __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  }
}

template <int HD>
__global__ void __launch_bounds__(128) varlen_attention_kernel(const VaParams P) {
  constexpr int E = HD / 32;
  grid_dep_wait();
  grid_dep_launch();
  const int lane = threadIdx.x & 31;
  const long long w = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (w >= (long long)P.rows * P.n_heads) return;
  const int r = (int)(w / P.n_heads), h = (int)(w % P.n_heads), g = h / P.qpg;
  int s, n_pre, first = 0, n_draft = 0;
  const unsigned long long* mrow = nullptr;
  if (P.T) {
    s = r / P.T;
    const int node = r - s * P.T;
    n_draft = P.n_nodes ? min(P.n_nodes[s], P.T) : P.T;
    if (node >= n_draft) return;
    n_pre = max(0, min(P.ctx_len[s], P.kv_tokens));
    mrow = P.mask + (size_t)r * P.words;
  } else {
    int lo = 0, hi = P.n_seqs;   // the last sequence that starts at or before r
    while (lo + 1 < hi) {
      const int mid = (lo + hi) / 2;
      if (P.q_start[mid] <= r) lo = mid;
      else hi = mid;
    }
    s = lo;
    const int q0 = P.q_start[s], q1 = P.q_start[s + 1];
    if (r < q0 || r >= q1) return;
    first = P.cached ? 0 : (P.k_start ? P.k_start[s] : q0);
    const int len = P.k_len ? P.k_len[s] : q1 - q0;
    n_pre = max(0, min(len - (q1 - q0) + (r - q0) + 1, P.kv_tokens - first));
    if (first < 0) n_pre = 0;
  }
  float q[E], o[E], m = -INFINITY, l = 0.f;
  va_load<E>(P.q, r * P.q_row + h * P.q_head, P.f16, lane, q);
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.f;
  auto step = [&](const void* kp, size_t ko, const void* vp, size_t vo) {
    float k[E], v[E], d = 0.f;
    va_load<E>(kp, ko, P.f16, lane, k);
    va_load<E>(vp, vo, P.f16, lane, v);
#pragma unroll
    for (int e = 0; e < E; ++e) d += q[e] * k[e];
    d = warp_sum(d) * P.scale_log2;
    const float mn = fmaxf(m, d), c = exp2f(m - mn), p = exp2f(d - mn);
    m = mn;
    l = l * c + p;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = o[e] * c + p * v[e];
  };
  const size_t seq = P.cached ? s : 0;
  for (int j = 0; j < n_pre; ++j)
    step(P.k, seq * P.k_seq + (size_t)(first + j) * P.k_tok + g * P.k_head, P.v,
         seq * P.v_seq + (size_t)(first + j) * P.v_tok + g * P.v_head);
  for (int j = 0; j < n_draft; ++j)
    if (mrow[j >> 6] >> (j & 63) & 1)
      step(P.kd, s * P.kd_row + j * P.kd_node + g * P.kd_head, P.vd, s * P.vd_row + j * P.vd_node + g * P.vd_head);
  const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e)
    store_act(P.out, P.out_f16 ? X_F16 : X_BF16, r * P.o_row + h * P.o_head + lane * E + e, o[e] * inv);
  if (P.lse && lane == 0)
    P.lse[(size_t)r * P.n_heads + h] = l > 0.f ? (m + log2f(l)) * 0.6931471805599453f : -INFINITY;
}

static bool va_misaligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }

static int va_launch(VaParams& P, int head_dim, cudaStream_t st) {
  const long long warps = (long long)P.rows * P.n_heads;
  const dim3 grid((unsigned)((warps + 3) / 4));
  if (head_dim == 128) return launch_pdl(varlen_attention_kernel<128>, grid, dim3(128), 0, st, P);
  return launch_pdl(varlen_attention_kernel<64>, grid, dim3(128), 0, st, P);
}

}  // namespace t2b

using namespace t2b;

extern "C" size_t t2b_varlen_attention_workspace_bytes(int rows, int n_heads, int n_kv, int head_dim) {
  return 0;
}

static int va_check(const void* q, const void* k, const void* v, const void* out, int dtype, int out_dtype, int rows,
                    int n_heads, int n_kv, int head_dim, float scale, std::initializer_list<size_t> strides) {
  if (!q || !k || !v || !out) return T2B_ERR_ARG;
  if ((dtype != T2B_DTYPE_BF16 && dtype != T2B_DTYPE_F16) || (out_dtype != T2B_DTYPE_BF16 && out_dtype != T2B_DTYPE_F16))
    return T2B_ERR_ARG;
  if (!(scale > 0.f) || !isfinite(scale)) return T2B_ERR_ARG;
  if (head_dim != 64 && head_dim != 128) return T2B_ERR_SHAPE;
  if (rows < 1 || n_kv < 1 || n_heads < 1 || n_heads % n_kv || n_heads / n_kv > 128) return T2B_ERR_SHAPE;
  if (va_misaligned(q) || va_misaligned(k) || va_misaligned(v) || va_misaligned(out)) return T2B_ERR_ALIGN;
  for (size_t s : strides)
    if (s % 8 || s == 0) return T2B_ERR_ALIGN;
  return T2B_OK;
}

extern "C" int t2b_packed_attention(const void* q, const void* k, const void* v, void* out, float* lse, int dtype,
                                    int out_dtype, const int32_t* q_start, const int32_t* k_start,
                                    const int32_t* k_len, int n_seqs, int total_q, int kv_seqs, int kv_tokens,
                                    int n_heads, int n_kv, int head_dim, size_t q_row, size_t q_head, size_t o_row,
                                    size_t o_head, size_t k_tok, size_t k_head, size_t k_seq, size_t v_tok,
                                    size_t v_head, size_t v_seq, float scale, void* workspace,
                                    size_t workspace_bytes, void* stream) {
  const int rc = va_check(q, k, v, out, dtype, out_dtype, total_q, n_heads, n_kv, head_dim, scale,
                          {q_row, q_head, o_row, o_head, k_tok, k_head, k_seq, v_tok, v_head, v_seq});
  if (rc != T2B_OK) return rc;
  if (!q_start) return T2B_ERR_ARG;
  if (n_seqs < 1 || kv_tokens < 1 || kv_seqs < 0) return T2B_ERR_SHAPE;
  if (kv_seqs ? (kv_seqs < n_seqs || !k_len || k_start) : (k_start == nullptr) != (k_len == nullptr)) return T2B_ERR_ARG;
  VaParams P{};
  P.q = q, P.k = k, P.v = v, P.out = out, P.lse = lse;
  P.f16 = dtype == T2B_DTYPE_F16, P.out_f16 = out_dtype == T2B_DTYPE_F16;
  P.rows = total_q, P.n_heads = n_heads, P.qpg = n_heads / n_kv, P.n_seqs = n_seqs;
  P.q_row = q_row, P.q_head = q_head, P.o_row = o_row, P.o_head = o_head;
  P.k_tok = k_tok, P.k_head = k_head, P.k_seq = k_seq, P.v_tok = v_tok, P.v_head = v_head, P.v_seq = v_seq;
  P.kv_tokens = kv_tokens, P.cached = kv_seqs > 0;
  P.q_start = q_start, P.k_start = k_start, P.k_len = k_len;
  P.scale_log2 = scale * 1.4426950408889634f;
  return va_launch(P, head_dim, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int t2b_tree_attention(const void* q, const void* k_cache, const void* v_cache, const void* k_draft,
                                  const void* v_draft, void* out, float* lse, int dtype, int out_dtype,
                                  const int32_t* ctx_len, const int32_t* n_nodes, const uint64_t* mask, int B, int T,
                                  int n_heads, int n_kv, int head_dim, int max_ctx, size_t q_row, size_t q_head,
                                  size_t o_row, size_t o_head, size_t kd_row, size_t kd_node, size_t kd_head,
                                  size_t vd_row, size_t vd_node, size_t vd_head, float scale, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  if (B < 1 || T < 1 || T > VA_MAX_NODES || max_ctx < 1 || (long long)B * T > 0x7fffffffll) return T2B_ERR_SHAPE;
  const int rc = va_check(q, k_cache, v_cache, out, dtype, out_dtype, B * T, n_heads, n_kv, head_dim, scale,
                          {q_row, q_head, o_row, o_head, kd_row, kd_node, kd_head, vd_row, vd_node, vd_head});
  if (rc != T2B_OK) return rc;
  if (!k_draft || !v_draft || !ctx_len || !mask) return T2B_ERR_ARG;
  if (va_misaligned(k_draft) || va_misaligned(v_draft) || (reinterpret_cast<uintptr_t>(mask) & 7)) return T2B_ERR_ALIGN;
  VaParams P{};
  P.q = q, P.k = k_cache, P.v = v_cache, P.kd = k_draft, P.vd = v_draft, P.out = out, P.lse = lse;
  P.f16 = dtype == T2B_DTYPE_F16, P.out_f16 = out_dtype == T2B_DTYPE_F16;
  P.rows = B * T, P.n_heads = n_heads, P.qpg = n_heads / n_kv, P.n_seqs = B;
  P.q_row = q_row, P.q_head = q_head, P.o_row = o_row, P.o_head = o_head;
  P.k_tok = P.v_tok = head_dim, P.k_head = P.v_head = (size_t)max_ctx * head_dim;
  P.k_seq = P.v_seq = (size_t)n_kv * max_ctx * head_dim;
  P.kd_row = kd_row, P.kd_node = kd_node, P.kd_head = kd_head;
  P.vd_row = vd_row, P.vd_node = vd_node, P.vd_head = vd_head;
  P.kv_tokens = max_ctx, P.cached = 1;
  P.ctx_len = ctx_len, P.n_nodes = n_nodes;
  P.mask = reinterpret_cast<const unsigned long long*>(mask);
  P.T = T, P.words = (T + 63) / 64;
  P.scale_log2 = scale * 1.4426950408889634f;
  return va_launch(P, head_dim, reinterpret_cast<cudaStream_t>(stream));
}
