// Log probabilities of given tokens over logits rows, with the entropy of
// each row and its most likely alternatives, in one pass over the logits:
//
//   m = max x, s = sum exp(x - m), z = sum (x - m) exp(x - m)
//   lse = m + log s, logprob(t) = (x[t] - m) - log s, entropy = log s - z / s
//
// The reference reads whole logits rows on the host (qwen_npu.py:321); a row
// of 151936 fp32 values is 608 KB, so the pass is bound by HBM.
//
// A CTA owns one row, or one of up to 8 equal ranges of it where there are few
// rows: the CTAs of a row are one thread-block cluster, and the first joins
// the others' (m, s, z) and best keys from their shared memory in range order,
// so there is no workspace and the result is the same every time.  A thread
// holds 32 values of a chunk in registers, so the maximum is known before the
// exponentials and the running sums are rescaled once per chunk.  All sums are
// fp32.  Measured: 1500 rows of 151936 fp32 188 us a call = 4.85 TB/s (0.74 of
// the measured copy; three CTAs per SM wait for their loads, at 80 registers
// with 28 to 32 bytes of spill stores a thread, and the rows are 3.4 waves of
// CTAs); one row with 20 alternatives 12 us a call, of which the alternatives'
// barriers and rankings are about half.
//
// Alternatives: a value and its index form one 64-bit key (order-preserving
// value bits << 32 | ~index: larger value first, ties to the lower index).
// A thread whose chunk maximum passes the K-th best value so far appends its
// candidates to a shared list, which is cut back to K when it has grown.  The
// first chunk is bounded by the K-th largest of 64 group maxima instead: at
// least K values reach it.  Where ties or an unlucky order would overflow the
// list, the chunk is bounded by whole keys: those are distinct, so at most K
// groups of 128 values hold a candidate and the list suffices for any order.

#include <math.h>

#include <algorithm>

#include "t2b_common.cuh"
#include "launch.cuh"

namespace t2b {

constexpr int LP_THREADS = 256;
constexpr int LP_PER = 32;                            // values per thread and chunk
constexpr int LP_CHUNK = LP_THREADS * LP_PER;
constexpr int LP_MAX_TOP = 32;
constexpr int LP_GROUPS = LP_THREADS / 4;             // a quad of threads: 128 values of a chunk
constexpr int LP_CAP = LP_MAX_TOP * 4 * LP_PER + LP_MAX_TOP;
constexpr int LP_CUT = 256;                           // list length that triggers a cut back to K
constexpr int LP_MAX_SPLITS = 8;                      // CTAs of a cluster; a thread fetches one key of the others
static_assert(LP_MAX_SPLITS * LP_MAX_TOP <= LP_THREADS, "one key per thread");
constexpr float LP_LOG2E = 1.4426950408889634f;

typedef unsigned long long u64;

struct LpParams {
  const void* x;
  size_t ld;
  int M, V, splits, per_split;
  const int* tokens;
  float *logprob, *entropy, *lse, *top_logprob;
  int* top_index;
  int K;
};

T2B_DEV u64 lp_key(float v, int i) {
  if (v != v) v = -INFINITY;
  const uint32_t u = __float_as_uint(v + 0.f);   // -0 and +0 are one value
  const uint32_t ord = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return ((u64)ord << 32) | (0xFFFFFFFFu - (uint32_t)i);
}
T2B_DEV float lp_value(u64 k) {
  const uint32_t ord = (uint32_t)(k >> 32);
  return __uint_as_float((ord & 0x80000000u) ? (ord & 0x7FFFFFFFu) : ~ord);
}
T2B_DEV u64 lp_quad_max(u64 k) {
#pragma unroll
  for (int o = 1; o <= 2; o <<= 1) {
    const u64 other = __shfl_xor_sync(0xffffffffu, k, o);
    k = other > k ? other : k;
  }
  return k;
}

T2B_DEV float lp_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Running (m, s, z) of a set of values; z is relative to m.
struct LpSum {
  float m, s, z;
};
T2B_DEV LpSum lp_rescale(LpSum a, float m) {
  if (a.m == m || a.m == -INFINITY) return {m, a.s, a.z};   // nothing but -inf so far: s = z = 0
  const float d = fmaxf(a.m - m, -1e30f);                     // (a difference that overflows has c = 0)
  const float c = lp_ex2(d * LP_LOG2E);
  return {m, a.s * c, (a.z + a.s * d) * c};
}
// The lanes' sums joined in lane order's butterfly: the maximum first, then
// each lane's sums are rescaled once and added.
T2B_DEV LpSum lp_warp_join(LpSum a) {
  a = lp_rescale(a, warp_max(a.m));
  return {a.m, warp_sum(a.s), warp_sum(a.z)};
}

template <typename T>
T2B_DEV float lp_float(T v);
template <>
T2B_DEV float lp_float<float>(float v) { return v; }
template <>
T2B_DEV float lp_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
T2B_DEV float lp_float<__half>(__half v) { return __half2float(v); }

struct LpShared {
  u64 list[LP_CAP];
  u64 top[LP_MAX_TOP];
  u64 group[LP_GROUPS];
  u64 bound;
  float value_bound;
  LpSum sum[LP_THREADS / 32];
  int n;
};

// The K-th largest of the group maxima (0 with fewer than K non-empty groups)
// into S.bound.  Every thread calls it.
T2B_DEV void lp_group_bound(LpShared& S, u64 mine, int K) {
  const int tid = threadIdx.x;
  mine = lp_quad_max(mine);
  if ((tid & 3) == 0) S.group[tid >> 2] = mine;
  if (tid == 0) S.bound = 0;
  __syncthreads();
  if (tid < LP_GROUPS) {
    const u64 k = S.group[tid];
    int rank = 0;
#pragma unroll 8
    for (int i = 0; i < LP_GROUPS; ++i) rank += S.group[i] > k;
    if (rank == K - 1 && k) S.bound = k;   // keys are distinct: one group at most
  }
  __syncthreads();
}

// The same on values: at least K values of the chunk reach it (-inf where
// fewer than K groups have one).
T2B_DEV float lp_group_value(LpShared& S, float mine, int K) {
  const int tid = threadIdx.x;
  float* group = reinterpret_cast<float*>(S.group);
#pragma unroll
  for (int o = 1; o <= 2; o <<= 1) mine = fmaxf(mine, __shfl_xor_sync(0xffffffffu, mine, o));
  if ((tid & 3) == 0) group[tid >> 2] = mine;
  if (tid == 0) S.value_bound = -INFINITY;
  __syncthreads();
  if (tid < LP_GROUPS) {
    const float v = group[tid];
    int above = 0, from = 0;
#pragma unroll 16
    for (int i = 0; i < LP_GROUPS; ++i) {
      above += group[i] > v;
      from += group[i] >= v;
    }
    if (above < K && from >= K) S.value_bound = v;   // (every thread that writes holds the same value)
  }
  __syncthreads();
  return S.value_bound;
}

// Cut the list of S.n keys to its K largest, in order, at list[0..K); empty
// places hold 0.  Every thread calls it, after a barrier.
T2B_DEV void lp_cut(LpShared& S, int K) {
  const int tid = threadIdx.x;
  int n = S.n;
  if (n > LP_CUT) {   // first drop what is under the group bound
    constexpr int R = (LP_CAP + LP_THREADS - 1) / LP_THREADS;
    u64 mine = 0;
    for (int i = tid; i < n; i += LP_THREADS) mine = S.list[i] > mine ? S.list[i] : mine;
    lp_group_bound(S, mine, K);
    u64 keep[R];
#pragma unroll
    for (int r = 0; r < R; ++r) keep[r] = tid + r * LP_THREADS < n ? S.list[tid + r * LP_THREADS] : 0;
    const u64 bound = S.bound;
    __syncthreads();
    if (tid == 0) S.n = 0;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (keep[r] && keep[r] >= bound) S.list[atomicAdd(&S.n, 1)] = keep[r];
    __syncthreads();
    n = S.n;
  }
  if (tid < K) S.top[tid] = 0;
  __syncthreads();
  for (int i = tid; i < n; i += LP_THREADS) {
    const u64 k = S.list[i];
    int rank = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) rank += S.list[j] > k;
    if (rank < K && k) S.top[rank] = k;
  }
  __syncthreads();
  if (tid < K) S.list[tid] = S.top[tid];
  if (tid == 0) S.n = min(n, K);
  __syncthreads();
}

// The same shared-memory location in cluster CTA `rank`.
T2B_DEV u64 lp_peer_u64(const u64* p, uint32_t rank) {
  u64 v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(map_peer(smem_u32(p), rank)) : "memory");
  return v;
}
T2B_DEV float lp_peer_f32(const float* p, uint32_t rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(map_peer(smem_u32(p), rank)) : "memory");
  return v;
}

template <typename T>
__global__ void __launch_bounds__(LP_THREADS, 3) token_logprobs_kernel(const LpParams P) {
  constexpr int VEC = 16 / sizeof(T), NV = LP_PER / VEC;
  __shared__ LpShared S;
  grid_dep_wait();
  grid_dep_launch();
  const int tid = threadIdx.x, K = P.K;
  const int row = blockIdx.x, split = blockIdx.y;   // a cluster holds the ranges of one row
  const T* x = static_cast<const T*>(P.x) + (size_t)row * P.ld;
  const int v0 = split * P.per_split, v1 = min(P.V, v0 + P.per_split);   // v0 < V: splits = ceil(V / per_split)
  // 16-byte loads fall on the row's own alignment: group g covers values
  // base + g * VEC .., base the last aligned index at or before v0 (may be
  // before the range: such edge groups are read value by value)
  const int shift = (int)((reinterpret_cast<uintptr_t>(x + v0) % 16) / sizeof(T));
  const int base = v0 - shift;
  LpSum a = {-INFINITY, 0.f, 0.f};
  float floor = -INFINITY;   // the K-th best value at the last cut: only larger ones are candidates
  if (tid == 0) S.n = 0;
  __syncthreads();
  for (int c0 = base; c0 < v1; c0 += LP_CHUNK) {
    float v[LP_PER];
    if (c0 >= v0 && c0 + LP_CHUNK <= v1) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const uint4 w = __ldcs(reinterpret_cast<const uint4*>(x + c0 + (i * LP_THREADS + tid) * VEC));
        const T* t = reinterpret_cast<const T*>(&w);
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[i * VEC + e] = lp_float<T>(t[e]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int g = c0 + (i * LP_THREADS + tid) * VEC;
        if (g >= v0 && g + VEC <= v1) {
          const uint4 w = __ldcs(reinterpret_cast<const uint4*>(x + g));
          const T* t = reinterpret_cast<const T*>(&w);
#pragma unroll
          for (int e = 0; e < VEC; ++e) v[i * VEC + e] = lp_float<T>(t[e]);
        } else {
#pragma unroll
          for (int e = 0; e < VEC; ++e) v[i * VEC + e] = g + e >= v0 && g + e < v1 ? lp_float<T>(x[g + e]) : -INFINITY;
        }
      }
    }
    float hi[2] = {v[0], v[1]}, lo[2] = {v[0], v[1]};
#pragma unroll
    for (int e = 2; e < LP_PER; ++e) {
      hi[e & 1] = fmaxf(hi[e & 1], v[e]);
      lo[e & 1] = fminf(lo[e & 1], v[e]);
    }
    const float cm = fmaxf(hi[0], hi[1]);
    if (cm > a.m) a = lp_rescale(a, cm);
    const float ms = a.m == -INFINITY ? 0.f : a.m;
    float s[4] = {0.f, 0.f, 0.f, 0.f}, z[4] = {0.f, 0.f, 0.f, 0.f};
    if (fminf(lo[0], lo[1]) > -1e30f) {
#pragma unroll
      for (int e = 0; e < LP_PER; ++e) {
        const float d = v[e] - ms, p = lp_ex2(d * LP_LOG2E);
        s[e & 3] += p;
        z[e & 3] = fmaf(p, d, z[e & 3]);
      }
    } else {   // masked values (-inf) add nothing
#pragma unroll
      for (int e = 0; e < LP_PER; ++e) {
        const float d = v[e] - ms, p = lp_ex2(d * LP_LOG2E);
        s[e & 3] += p;
        z[e & 3] = fmaf(p, fmaxf(d, -1e30f), z[e & 3]);
      }
    }
    a.s += (s[0] + s[1]) + (s[2] + s[3]);
    a.z += (z[0] + z[1]) + (z[2] + z[3]);
    if (K) {
      auto index = [&](int e) { return c0 + ((e / VEC) * LP_THREADS + tid) * VEC + e % VEC; };
      auto inside = [&](int e) { return index(e) >= v0 && index(e) < v1; };
      const bool first = c0 == base;
      if (first) floor = lp_group_value(S, cm, K);
      int at = 0;
      // (later values tied with the K-th best so far have a higher index and lose)
      if (first ? !(cm < floor) : cm > floor) {
        uint32_t hits = 0;
#pragma unroll
        for (int e = 0; e < LP_PER; ++e) hits |= (uint32_t)(first ? !(v[e] < floor) : v[e] > floor) << e;
        while (hits) {   // a lane has one candidate or two; taking its value by selects keeps v in registers
          const int h = __ffs(hits) - 1;
          hits &= hits - 1;
          float value = v[0];
#pragma unroll
          for (int e = 1; e < LP_PER; ++e) value = e == h ? v[e] : value;
          if (!inside(h)) continue;
          at = atomicAdd(&S.n, 1);
          if (at < LP_CAP) S.list[at] = lp_key(value, index(h));
        }
      }
      if (__syncthreads_or(first || at >= LP_CUT)) {
        if (S.n > LP_CAP) {   // this chunk's candidates again, bounded by whole keys
          const int n = LP_CAP;
          constexpr int R = (LP_CAP + LP_THREADS - 1) / LP_THREADS;
          u64 keep[R];
#pragma unroll
          for (int r = 0; r < R; ++r) {
            const u64 k = tid + r * LP_THREADS < n ? S.list[tid + r * LP_THREADS] : 0;
            keep[r] = (int)(0xFFFFFFFFu - (uint32_t)k) < c0 ? k : 0;   // of earlier chunks
          }
          __syncthreads();
          if (tid == 0) S.n = 0;
          __syncthreads();
#pragma unroll
          for (int r = 0; r < R; ++r)
            if (keep[r]) S.list[atomicAdd(&S.n, 1)] = keep[r];
          __syncthreads();
          lp_cut(S, K);
          u64 mine = 0;
#pragma unroll
          for (int e = 0; e < LP_PER; ++e)
            if (inside(e)) {
              const u64 k = lp_key(v[e], index(e));
              mine = k > mine ? k : mine;
            }
          lp_group_bound(S, mine, K);
          const u64 bound = S.bound;
#pragma unroll
          for (int e = 0; e < LP_PER; ++e)
            if (inside(e)) {
              const u64 k = lp_key(v[e], index(e));
              if (k >= bound) S.list[atomicAdd(&S.n, 1)] = k;
            }
          __syncthreads();
        }
        lp_cut(S, K);
        floor = S.n < K ? -INFINITY : lp_value(S.list[K - 1]);
      }
    }
  }
  // ---- the CTA's sums, in a fixed order ----
  a = lp_warp_join(a);
  if ((tid & 31) == 0) S.sum[tid >> 5] = a;
  __syncthreads();
  const int lane = tid & 31;
  a = lane < LP_THREADS / 32 ? S.sum[lane] : LpSum{-INFINITY, 0.f, 0.f};
  a = lp_warp_join(a);
  __syncthreads();
  if (K) lp_cut(S, K);

  if (P.splits > 1) {
    // ---- the ranges of a row meet in the first CTA's shared memory ----
    if (tid == 0) S.sum[0] = a;
    if (K && tid < K && tid >= S.n) S.list[tid] = 0;
    cluster_sync();
    if (split == 0) {
      const int from = K ? tid / K : P.splits;   // thread: place tid % K of range `from`
      u64 key = 0;
      if (from < P.splits) key = from ? lp_peer_u64(&S.list[tid - from * K], from) : S.list[tid];
      LpSum b = {-INFINITY, 0.f, 0.f};
      if (lane < P.splits)
        b = {lp_peer_f32(&S.sum[0].m, lane), lp_peer_f32(&S.sum[0].s, lane), lp_peer_f32(&S.sum[0].z, lane)};
      a = lp_warp_join(b);
      if (K) {
        // the ranges' keys are in order: at least K of all reach the least of
        // their ceil(K / splits)-th ones, and only those are ranked
        const int deep = (K + P.splits - 1) / P.splits - 1;
        if (from < P.splits && tid - from * K == deep) S.group[from] = key;
        if (tid == 0) S.n = 0;
        __syncthreads();
        u64 bound = S.group[0];
        for (int i = 1; i < P.splits; ++i) bound = S.group[i] < bound ? S.group[i] : bound;
        if (key && key >= bound) S.list[atomicAdd(&S.n, 1)] = key;
        __syncthreads();
        lp_cut(S, K);
      }
    }
    cluster_sync();   // the other CTAs' shared memory has been read
    if (split) return;
  }
  const float ls = logf(a.s);
  const bool none = a.m == -INFINITY && a.s == 0.f;   // nothing but -inf: no distribution
  if (tid == 0) {
    if (P.logprob) {
      const int t = P.tokens[row];
      P.logprob[row] = t < 0 || t >= P.V ? NAN : none ? -INFINITY : (lp_float<T>(x[t]) - a.m) - ls;
    }
    if (P.entropy) P.entropy[row] = none ? 0.f : ls - a.z / a.s;
    if (P.lse) P.lse[row] = none ? -INFINITY : a.m + ls;
  }
  if (tid < K) {
    const u64 k = S.list[tid];
    if (P.top_logprob) P.top_logprob[(size_t)row * K + tid] = none ? -INFINITY : (lp_value(k) - a.m) - ls;
    if (P.top_index) P.top_index[(size_t)row * K + tid] = (int)(0xFFFFFFFFu - (uint32_t)k);
  }
}

// Ranges a row is cut into (a power of two): as many as keep all CTAs resident
// at once (three per SM), each range at least 2048 values.  (65 rows of 128256
// in 8 ranges ran in two waves: 26.6 us.)
static int lp_splits(int M, int V) {
  int n = 1;
  while (n < LP_MAX_SPLITS && 2ll * M * n <= 444 && V / (2 * n) >= 2048) n *= 2;
  return n;
}

static int lp_launch(void (*kern)(LpParams), LpParams& P, cudaStream_t st) {
  const dim3 grid(P.M, P.splits);
  if (P.splits == 1) return launch_pdl(kern, grid, dim3(LP_THREADS), 0, st, P);
  return launch_pdl_cluster(kern, grid, dim3(LP_THREADS), 0, st, P.splits, P);
}

}  // namespace t2b

using namespace t2b;

extern "C" int t2b_token_logprobs(const void* logits, int dtype, int M, int V, size_t ld, const int32_t* tokens,
                                  float* logprob, float* entropy, float* lse, int num_top, float* top_logprob,
                                  int32_t* top_index, void* stream) {
  if (!logits || (dtype != T2B_DTYPE_BF16 && dtype != T2B_DTYPE_F16 && dtype != T2B_DTYPE_F32)) return T2B_ERR_ARG;
  if ((tokens == nullptr) != (logprob == nullptr)) return T2B_ERR_ARG;
  if (num_top ? !top_logprob && !top_index : top_logprob || top_index) return T2B_ERR_ARG;
  if (!logprob && !entropy && !lse && !num_top) return T2B_ERR_ARG;
  if (M < 1 || V < 1 || V > 0x7fff0000 || ld < (size_t)V || num_top < 0 || num_top > LP_MAX_TOP || num_top > V)
    return T2B_ERR_SHAPE;
  if (reinterpret_cast<uintptr_t>(logits) % (dtype == T2B_DTYPE_F32 ? 4 : 2)) return T2B_ERR_ALIGN;
  LpParams P{};
  P.x = logits, P.ld = ld, P.M = M, P.V = V;
  P.splits = lp_splits(M, V);
  P.per_split = (V + P.splits - 1) / P.splits;
  P.splits = (V + P.per_split - 1) / P.per_split;
  P.tokens = tokens, P.logprob = logprob, P.entropy = entropy, P.lse = lse;
  P.K = num_top, P.top_logprob = top_logprob, P.top_index = top_index;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == T2B_DTYPE_F32) return lp_launch(token_logprobs_kernel<float>, P, st);
  if (dtype == T2B_DTYPE_F16) return lp_launch(token_logprobs_kernel<__half>, P, st);
  return lp_launch(token_logprobs_kernel<__nv_bfloat16>, P, st);
}
