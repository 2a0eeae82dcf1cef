// Attention over sequences of different lengths on tcgen05: packed prompts
// (causal) and trees of drafted tokens over the KV cache.
//
//   out[r, h] = sum_j softmax_j(scale * q[r, h] . k[j, h / qpg]) v[j, h / qpg]
//
// over the keys row r sees.  Packed: row r is query i of the n queries of its
// sequence and sees keys 0 .. k_len - n + i (model.py:266-279 without
// padding).  Tree: row r is node i of batch row b and sees the ctx_len[b]
// cached keys and the drafted nodes whose bit is set in mask[b][i].
//
// Work.  The qpg query heads of a kv head share its keys, so a tile is 128
// MMA rows = 128 / qpg tokens x qpg heads, and an item two neighbouring tiles
// of one (sequence, kv head).  An item's keys are blocks of 128, and one
// (item, block) is a unit.  All units of the call form one list, which the
// CTAs (one per SM) cut into equal ranges: prompts of any lengths, long
// contexts with few rows and single tokens balance alike without the host
// knowing a length.  An item cut between CTAs leaves fp32 partials (output,
// maximum, sum) that a second kernel joins in a fixed order; items of up to
// VA_SNAP blocks are not cut.
//
// CTA: two softmax groups of four warps, a TMA warp and an MMA warp.
//   S_t = Q_t K^T     A, B from shared memory (128-byte swizzled TMA tiles)
//   P_t = 2^(S_t c - m)    TMEM -> registers -> TMEM, 16 bits, over S_t
//   O_t += P_t V      A from TMEM, B = V as loaded (MN-major)
// A thread owns one row: no shuffles.  While a group is busy with the
// exponentials of its block the tensor core runs the other group's two
// products.  With both tiles live the groups take one tile each and share
// the K/V blocks; an item of one tile (small trees, single tokens, ends of
// prompts) alternates its blocks between the groups, and group 0 joins the
// two results at the end straight from TMEM.
//
// Numerics.  Scores, maxima, sums and O are fp32; the weights are rounded
// once, to the operands' 16-bit type, as A of the second product (the sum
// uses them before rounding).  The exponent's reference m is moved, and O
// rescaled, only when a row's maximum outgrows it: it starts VA_HEAD below the
// first block's maximum and moves when a score passes m + VA_ROOM, so a weight
// is at most 2^15 (in fp16 range) and the largest is at least 2^VA_HEAD of the
// time it was set, which keeps small fp16 weights 2^7 further from underflow.
//
// Every mbarrier wait is time-bounded (T2B_ERR_TIMEOUT in the status word,
// then every role stops at its next wait).

#include <math.h>

#include <algorithm>
#include <initializer_list>

#include "t2b_common.cuh"
#include "launch.cuh"
#include "tmap.cuh"
#include "tcgen05.cuh"

namespace t2b {

constexpr int VA_MAX_NODES = 256;
constexpr int VA_ROWS = 128;            // rows per tile (MMA M), keys per block (MMA N)
constexpr int VA_THREADS = 384;         // 8 softmax warps, TMA, MMA, 2 that only fill the warpgroup
// Registers: 384 threads are launched with 168 each (64512); the softmax
// warpgroups take 208 and the third gives down to 80: 2 * 128 * 208 + 128 * 80
// = 63488.
constexpr int VA_REGS_SOFTMAX = 208, VA_REGS_OTHER = 80;
constexpr int VA_SNAP = 4;              // items of up to this many blocks stay in one CTA
constexpr int VA_MIN_UNITS = 2;         // units per CTA, at least
constexpr float VA_HEAD = 7.f, VA_ROOM = 15.f;

struct VaParams {
  CUtensorMap qmap;                     // (hd, heads, rows), box (64, qpg, tokens per tile)
  CUtensorMap kmap, vmap;               // (hd, tokens, heads, sequences), box (64, 128, 1, 1)
  CUtensorMap kdmap, vdmap;             // drafted nodes (tree)
  void* out;
  float* lse;                           // [rows][n_heads] (nullable)
  int out_f16;
  int rows, n_heads, n_kv, qpg, n_seqs;
  int tpt;                              // tokens per tile
  size_t o_row, o_head;
  int kv_tokens, cached;                // token extent of K and V; keys of sequence s in cache row s
  const int *q_start, *k_start, *k_len; // packed
  const int *ctx_len, *n_nodes;         // tree
  const uint32_t* mask;                 // [B][T][2 * words]
  int T, words;
  float scale_log2;
  float* part_o;                        // [2 * grid][256][hd]
  float2* part_ml;                      // [2 * grid][256]
  int4* head;                           // [2 * grid]: (tail item s, p, g, tail flag), (first continues, ends, -, -)
  int* err;
};

template <int HD>
struct VaGeom {
  static constexpr int TILE = VA_ROWS * HD * 2;        // one Q tile, K block or V block
  static constexpr int STAGES = HD == 128 ? 5 : 8;     // K and V blocks in flight
  static constexpr int OFF_KV = 2 * TILE;
  static constexpr int OFF_ML = OFF_KV + STAGES * TILE;   // float2 [128]: group 1's (m, l)
  static constexpr int OFF_BAR = OFF_ML + VA_ROWS * 8;
  static constexpr int N_BARS = 2 + 2 * STAGES + 9;
  static constexpr int OFF_MISC = OFF_BAR + N_BARS * 8;
  static constexpr int BYTES = OFF_MISC + 256 + 1024;      // + slack to 1024-align the base
  static constexpr uint32_t S0 = 0, O0 = 256;              // TMEM columns: S_t at S0 + 128 t, O_t at O0 + HD t
  static_assert(BYTES <= 232448, "shared memory of one CTA");
};

// One sequence: rows q0 .. q0 + n - 1.  Packed: key j at token first + j, row
// i sees min(off + i + 1, avail) keys.  Tree: avail cached keys, n nodes.
struct VaSeq {
  int q0, n, first, avail, off;
};

template <bool TREE>
T2B_DEV VaSeq va_seq(const VaParams& P, int s) {
  VaSeq q;
  if (TREE) {
    q.q0 = s * P.T;
    q.n = P.n_nodes ? max(0, min(P.n_nodes[s], P.T)) : P.T;
    q.first = 0;
    q.avail = max(0, min(P.ctx_len[s], P.kv_tokens));
    q.off = 0;
  } else {
    q.q0 = max(0, min(P.q_start[s], P.rows));
    q.n = max(q.q0, min(P.q_start[s + 1], P.rows)) - q.q0;
    q.first = P.cached ? 0 : (P.k_start ? P.k_start[s] : q.q0);
    const int len = P.k_len ? max(0, P.k_len[s]) : q.n;
    q.off = len - q.n;
    q.avail = q.first < 0 || q.first >= P.kv_tokens ? 0 : min(len, P.kv_tokens - q.first);
    if (q.avail == 0) q.first = 0;
  }
  return q;
}
T2B_DEV int va_blocks(int keys) { return (keys + VA_ROWS - 1) / VA_ROWS; }
// keys that query i of a packed sequence sees
T2B_DEV int va_limit(const VaSeq& q, int i) { return max(0, min(q.off + i + 1, q.avail)); }
// blocks of tile t (0, 1) of pair p; the pair's blocks are those of its last live tile
template <bool TREE>
T2B_DEV int va_tile_blocks(const VaSeq& q, int tpt, int p, int t) {
  if (TREE) return va_blocks(q.avail) + va_blocks(q.n);
  return max(1, va_blocks(va_limit(q, min(q.n, (2 * p + t + 1) * tpt) - 1)));
}
T2B_DEV int va_pairs(const VaSeq& q, int tpt) { return (q.n + 2 * tpt - 1) / (2 * tpt); }

// A position in the list of units: block b of item (s, p, g).
struct VaCursor {
  int s, p, g, b;
};
struct VaSegment {
  VaSeq q;
  int s, p, g;
  int b0, n;          // first block, blocks of this CTA
  int nb, n0;         // the item's blocks; blocks of tile 0 in this segment (two tiles)
  bool dual;          // both tiles live
};

template <bool TREE>
struct VaWalk {
  VaCursor c;
  int left;
  VaSeq q;
  T2B_DEV VaWalk(const VaParams& P, VaCursor at, int units) : c(at), left(units) {
    if (left > 0) q = va_seq<TREE>(P, c.s);
  }
  T2B_DEV bool next(const VaParams& P, VaSegment& seg) {
    if (left <= 0) return false;
    seg.q = q;
    seg.s = c.s;
    seg.p = c.p;
    seg.g = c.g;
    seg.dual = q.n > (2 * c.p + 1) * P.tpt;
    seg.nb = va_tile_blocks<TREE>(q, P.tpt, c.p, seg.dual ? 1 : 0);
    seg.b0 = c.b;
    seg.n = min(left, seg.nb - c.b);
    seg.n0 = seg.dual ? min(seg.n, va_tile_blocks<TREE>(q, P.tpt, c.p, 0) - c.b) : seg.n;
    left -= seg.n;
    c.b = 0;
    if (left > 0 && ++c.g == P.n_kv) {
      c.g = 0;
      if (++c.p == va_pairs(q, P.tpt)) {
        c.p = 0;
        do {
          ++c.s;
          q = va_seq<TREE>(P, c.s);
        } while (q.n == 0 && c.s + 1 < P.n_seqs);
      }
    }
    return true;
  }
};

T2B_DEV void tma_load_4d(void* dst, const void* tmap, int x, int y, int z, int w, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(tmap)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
      : "memory");
}
// UMMA descriptor of an MN-major operand, 128-byte swizzle: 64 contiguous
// elements per 128-byte row, 8-row groups 1024 B apart along k, the next 64
// elements `mn_stride` bytes on.
T2B_DEV uint64_t sdesc_mn_sw128(uint32_t saddr, uint32_t mn_stride) {
  uint64_t d = 0;
  d |= (uint64_t)((saddr >> 4) & 0x3FFFu);
  d |= (uint64_t)(mn_stride >> 4) << 16;
  d |= (uint64_t)(1024u >> 4) << 32;
  d |= (uint64_t)1u << 46;
  d |= (uint64_t)2u << 61;
  return d;
}
T2B_DEV void tmem_st32(uint32_t taddr, const uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
      "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]),
      "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]),
      "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}
T2B_DEV float va_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <bool F16>
T2B_DEV uint32_t va_pack(float lo, float hi) {
  uint32_t r;
  if (F16) asm("cvt.rn.f16x2.f32 %0, %2, %1;" : "=r"(r) : "f"(lo), "f"(hi));
  else asm("cvt.rn.bf16x2.f32 %0, %2, %1;" : "=r"(r) : "f"(lo), "f"(hi));
  return r;
}
T2B_DEV uint32_t va_pack_out(float lo, float hi, int f16) { return f16 ? f16x2_sat(lo, hi) : va_pack<false>(lo, hi); }

// Keys 32 w .. 32 w + 31 below `n` of a block, as bits.
T2B_DEV uint32_t va_bits_below(int n, int w) {
  const int k = n - 32 * w;
  return k >= 32 ? 0xffffffffu : k <= 0 ? 0u : (1u << k) - 1u;
}

template <int HD, bool F16, bool TREE>
__global__ void __launch_bounds__(VA_THREADS, 1) varlen_attention_kernel(const __grid_constant__ VaParams P) {
  using G = VaGeom<HD>;
  constexpr int NS = G::STAGES, HALVES = HD / 64;
  extern __shared__ __align__(1024) uint8_t smem_dyn[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~uintptr_t(1023));
  float2* s_ml = reinterpret_cast<float2*>(sm + G::OFF_ML);
  uint64_t* q_full = reinterpret_cast<uint64_t*>(sm + G::OFF_BAR);
  uint64_t* q_empty = q_full + 1;
  uint64_t* kv_full = q_full + 2;
  uint64_t* kv_empty = kv_full + NS;
  uint64_t* s_full = kv_empty + NS;      // [2]
  uint64_t* p_full = s_full + 2;         // [2]
  uint64_t* o_full = p_full + 2;         // [2]
  uint64_t* g1_full = o_full + 2;
  uint64_t* g1_empty = g1_full + 1;
  uint64_t* done = g1_full + 2;
  long long* s_scan = reinterpret_cast<long long*>(sm + G::OFF_MISC);          // [11]
  VaCursor* s_at = reinterpret_cast<VaCursor*>(sm + G::OFF_MISC + 96);
  int* s_flag = reinterpret_cast<int*>(sm + G::OFF_MISC + 128);
  long long* s_range = reinterpret_cast<long long*>(sm + G::OFF_MISC + 144);   // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sm + G::OFF_MISC + 160);
  volatile int* abort_flag = s_flag;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int i = 0; i < NS; ++i) {
      mbar_init(&kv_full[i], 1);
      mbar_init(&kv_empty[i], 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&s_full[t], 1);
      mbar_init(&p_full[t], 4);   // one arrival per softmax warp
      mbar_init(&o_full[t], 1);
    }
    mbar_init(g1_full, 4);
    mbar_init(g1_empty, 4);
    mbar_init(done, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 9) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  grid_dep_wait();

  // ---- this CTA's range of the list of units ----
  const int c = blockIdx.x;
  auto seq_units = [&](int s) -> long long {
    if (s >= P.n_seqs) return 0;
    const VaSeq q = va_seq<TREE>(P, s);
    const int pairs = va_pairs(q, P.tpt);
    long long u = 0;
    if (TREE) {
      u = (long long)pairs * va_tile_blocks<TREE>(q, P.tpt, 0, 0);
    } else {
      for (int p = 0; p < pairs; ++p) u += va_tile_blocks<TREE>(q, P.tpt, p, 1);
    }
    return u * P.n_kv;
  };
  // inclusive sum of one value per thread over the block (and the block's total)
  auto block_scan = [&](long long v, long long& total) -> long long {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long w = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += w;
    }
    __syncthreads();
    if (lane == 31) s_scan[warp] = v;
    __syncthreads();
    long long before = 0;
    total = 0;
    for (int w = 0; w < VA_THREADS / 32; ++w) {
      if (w < warp) before += s_scan[w];
      total += s_scan[w];
    }
    return before + v;
  };
  long long total = 0;
  for (int s0 = 0; s0 < P.n_seqs; s0 += VA_THREADS) {
    long long t;
    block_scan(seq_units(s0 + tid), t);
    total += t;
  }
  const int parts = (int)min((long long)gridDim.x, max(1ll, total / VA_MIN_UNITS));
  const bool busy = total > 0 && c < parts;
  if (tid == 0) {
    s_range[0] = 0;
    s_range[1] = busy ? total : 0;   // (kept where the range's end is the end of the list)
  }
  if (busy) {
    const long long cut[2] = {total * c / parts, total * (c + 1) / parts};
    long long base = 0;
    for (int s0 = 0; s0 < P.n_seqs; s0 += VA_THREADS) {
      long long t;
      const long long mine = seq_units(s0 + tid);
      const long long end = base + block_scan(mine, t), begin = end - mine;
      base += t;
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (cut[i] >= begin && cut[i] < end) {   // the cut falls into sequence s0 + tid
          const int s = s0 + tid;
          const VaSeq q = va_seq<TREE>(P, s);
          const int pairs = va_pairs(q, P.tpt);
          long long u = begin;
          int p = 0, nb;
          for (;; ++p) {
            nb = va_tile_blocks<TREE>(q, P.tpt, p, 1);
            if (cut[i] < u + (long long)nb * P.n_kv) break;
            u += (long long)nb * P.n_kv;
          }
          int g = (int)((cut[i] - u) / nb), b = (int)((cut[i] - u) % nb);
          long long at = cut[i];
          if (nb <= VA_SNAP && b) {
            if (2 * b < nb) {
              at -= b;
            } else {   // up to the next item
              at += nb - b;
              if (++g == P.n_kv) {
                g = 0;
                ++p;
              }
            }
            b = 0;
          }
          s_range[i] = at;
          if (i == 0) {
            int ns = s;
            if (p == pairs) {   // (behind the sequence: the next one that has rows; unused at the list's end)
              p = 0;
              do ++ns;
              while (ns < P.n_seqs && va_seq<TREE>(P, ns).n == 0);
            }
            *s_at = {ns, p, g, b};
          }
        }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tbase = *tmem_slot;
  const int units = (int)(s_range[1] - s_range[0]);
  const VaCursor start = units > 0 ? *s_at : VaCursor{0, 0, 0, 0};
  grid_dep_launch();   // this CTA holds its TMEM: dependents may start

  const int tpt = P.tpt, qpg = P.qpg;
  if (warp >= 8) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(VA_REGS_OTHER));
  VaWalk<TREE> walk(P, start, units);
  VaSegment seg;
  if (warp == 8) {
    // ---- TMA: per segment K0, (Q), K1, V0, K2, V1, ..: the order the MMAs take them ----
    if (lane == 0) {
      int pos = 0, nseg = 0, q_loads = 0;
      bool ok = true;
      for (; ok && walk.next(P, seg); ++nseg) {
        auto load_q = [&] {
          if (nseg > 0) ok = mbar_wait_bounded(q_empty, (nseg - 1) & 1, P.err);
          if (!ok) return;
          const int tiles = seg.dual ? 2 : 1, row = seg.q.q0 + 2 * seg.p * tpt;
          mbar_arrive_expect_tx(q_full, (uint32_t)(tiles * HALVES * tpt * qpg * 128));
          for (int t = 0; t < tiles; ++t)
            for (int hf = 0; hf < HALVES; ++hf)
              tma_load_3d(sm + t * G::TILE + hf * (VA_ROWS * 128), &P.qmap, hf * 64, seg.g * qpg, row + t * tpt, q_full);
          q_loads = nseg + 1;
        };
        if (nseg == 0) load_q();
        const int nbp = TREE ? va_blocks(seg.q.avail) : 0;
        const int seq = TREE || P.cached ? seg.s : 0;
        for (int i = 0; ok && i < 2 * seg.n; ++i, ++pos) {
          const bool is_k = i == 0 || ((i & 1) && i < 2 * seg.n - 1);
          const int b = seg.b0 + (is_k ? (i + 1) / 2 : i == 2 * seg.n - 1 ? seg.n - 1 : i / 2 - 1);
          const int st = pos % NS;
          if (pos >= NS) ok = mbar_wait_bounded(&kv_empty[st], ((pos / NS) - 1) & 1, P.err);
          if (!ok || *abort_flag) {
            ok = false;
            break;
          }
          const bool draft = TREE && b >= nbp;
          const void* map = draft ? (is_k ? &P.kdmap : &P.vdmap) : (is_k ? &P.kmap : &P.vmap);
          const int tok = draft ? (b - nbp) * VA_ROWS : seg.q.first + b * VA_ROWS;
          uint8_t* dst = sm + G::OFF_KV + st * G::TILE;
          mbar_arrive_expect_tx(&kv_full[st], (uint32_t)G::TILE);
          for (int hf = 0; hf < HALVES; ++hf)
            tma_load_4d(dst + hf * (VA_ROWS * 128), map, hf * 64, tok, seg.g, seq, &kv_full[st]);
          if (i == 1 && nseg > 0) load_q();
        }
      }
      if (!ok) *abort_flag = 1;
      // every load has landed before the CTA may exit
      for (int i = max(0, pos - NS); i < pos; ++i) mbar_wait_bounded(&kv_full[i % NS], (i / NS) & 1, P.err);
      if (q_loads) mbar_wait_bounded(q_full, (q_loads - 1) & 1, P.err);
    }
  } else if (warp == 9) {
    // ---- MMA issuer (lane 0; the warp's other lanes help to clear V rows) ----
    constexpr uint32_t FMT = F16 ? 0u : (1u << 7) | (1u << 10);
    constexpr uint32_t ID_S = (1u << 4) | FMT | ((uint32_t)(VA_ROWS >> 3) << 17) | ((uint32_t)(VA_ROWS >> 4) << 24);
    constexpr uint32_t ID_O = (1u << 4) | FMT | (1u << 16) | ((uint32_t)(HD >> 3) << 17) | ((uint32_t)(VA_ROWS >> 4) << 24);
    int ring = 0, nseg = 0, np[2] = {0, 0};
    bool ok = true;
    for (; ok && walk.next(P, seg); ++nseg) {
      const int n = seg.n, nbp = TREE ? va_blocks(seg.q.avail) : 0;
      auto at_k = [&](int i) { return ring + (i ? 2 * i - 1 : 0); };
      auto at_v = [&](int i) { return ring + (i < n - 1 ? 2 * i + 2 : 2 * n - 1); };
      auto wait = [&](uint64_t* bar, uint32_t ph) {
        ok = __all_sync(0xffffffffu, ok && *abort_flag == 0 && mbar_wait_bounded(bar, ph, P.err));
        tc_fence_after();
      };
      auto kv_wait = [&](int at) { wait(&kv_full[at % NS], (at / NS) & 1); };
      auto kv_done = [&](int at) {
        if (ok && lane == 0) mma_commit(&kv_empty[at % NS]);
      };
      auto mma_s = [&](int t, int i) {   // S_t = Q K(i)^T
        kv_wait(at_k(i));
        if (ok && lane == 0) {
          const uint32_t qa = smem_u32(sm) + (seg.dual ? t : 0) * G::TILE;
          const uint32_t ka = smem_u32(sm) + G::OFF_KV + (at_k(i) % NS) * G::TILE;
#pragma unroll
          for (int ks = 0; ks < HD / 16; ++ks) {
            const uint32_t o = (ks >> 2) * (VA_ROWS * 128) + (ks & 3) * 32;
            mma_ss(tbase + G::S0 + t * 128, sdesc_sw128(qa + o), sdesc_sw128(ka + o), ID_S, ks > 0);
          }
          mma_commit(&s_full[t]);
        }
      };
      auto v_ready = [&](int i) {   // V(i) is there, and its rows past the sequence's keys are zero
        kv_wait(at_v(i));
        const int b = seg.b0 + i;
        const int valid = TREE && b >= nbp ? seg.q.n - (b - nbp) * VA_ROWS : seg.q.avail - b * VA_ROWS;
        if (ok && valid < VA_ROWS) {   // their weights are 0, but 0 * (whatever lies there) may be NaN
          uint8_t* v = sm + G::OFF_KV + (at_v(i) % NS) * G::TILE;
          for (int hf = 0; hf < HALVES; ++hf)
            for (int o = max(0, valid) * 128 + lane * 16; o < VA_ROWS * 128; o += 512)
              *reinterpret_cast<uint4*>(v + hf * (VA_ROWS * 128) + o) = make_uint4(0u, 0u, 0u, 0u);
          fence_proxy_async();
          __syncwarp();
        }
      };
      auto mma_o = [&](int t, int i, bool first) {   // O_t += P_t V(i)
        wait(&p_full[t], np[t]++ & 1);
        if (ok && lane == 0) {
          const uint32_t va = smem_u32(sm) + G::OFF_KV + (at_v(i) % NS) * G::TILE;
#pragma unroll
          for (int ks = 0; ks < VA_ROWS / 16; ++ks)
            mma_ts(tbase + G::O0 + t * HD, tbase + G::S0 + t * 128 + ks * 8, sdesc_mn_sw128(va + ks * 2048, VA_ROWS * 128),
                   ID_O, !(first && ks == 0));
        }
      };
      auto o_done = [&](int t) {
        if (ok && lane == 0) mma_commit(&o_full[t]);
      };
      auto q_done = [&] {
        if (ok && lane == 0) mma_commit(q_empty);
      };
      wait(q_full, nseg & 1);
      if (seg.dual) {
        if (seg.n0 > 0) mma_s(0, 0);
        mma_s(1, 0);
        kv_done(at_k(0));
        if (n == 1) q_done();
        for (int i = 0; i < n && ok; ++i) {
          v_ready(i);
          if (i < seg.n0) {
            mma_o(0, i, i == 0);
            if (i + 1 < seg.n0) mma_s(0, i + 1);
            else o_done(0);
          }
          mma_o(1, i, i == 0);
          kv_done(at_v(i));
          if (i + 1 < n) {
            mma_s(1, i + 1);
            kv_done(at_k(i + 1));
            if (i + 1 == n - 1) q_done();
          } else {
            o_done(1);
          }
        }
      } else {
        for (int i = 0; i < 2 && i < n; ++i) {
          mma_s(i, i);
          kv_done(at_k(i));
        }
        if (n <= 2) q_done();
        for (int i = 0; i < n && ok; ++i) {
          v_ready(i);
          mma_o(i & 1, i, i < 2);
          kv_done(at_v(i));
          if (i + 2 < n) {
            mma_s(i & 1, i + 2);
            kv_done(at_k(i + 2));
            if (i + 2 == n - 1) q_done();
          } else {
            o_done(i & 1);
          }
        }
      }
      ring += 2 * n;
    }
    if (!ok) *abort_flag = 1;
    // every MMA issued here has retired before TMEM is released
    if (lane == 0) {
      mma_commit(done);
      mbar_wait_bounded(done, 0, P.err);
    }
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(VA_REGS_SOFTMAX));
    VaWalk<TREE> walk(P, start, units);
    VaSegment seg;
    // ---- softmax group t: thread = row ----
    const int t = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lanes = tbase + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t s_col = lanes + G::S0 + t * 128, o_col = lanes + G::O0 + t * HD;
    const int tok_in_tile = row / qpg, head_in_group = row - tok_in_tile * qpg;
    const float scale = P.scale_log2;
    int ns = 0, nseg_o = 0, ng1 = 0;
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t ph) {
      ok = __all_sync(0xffffffffu, ok && *abort_flag == 0 && mbar_wait_bounded(bar, ph, P.err));
      tc_fence_after();
    };
    int4 tail = make_int4(0, 0, 0, 0), first = make_int4(-1, 0, 0, 0);   // this CTA's ends, for the joining kernel
    while (ok && walk.next(P, seg)) {
      if (first.x < 0) first = make_int4(seg.b0 > 0, seg.b0 + seg.n == seg.nb, 0, 0);
      if (seg.b0 == 0 && seg.n < seg.nb) tail = make_int4(seg.s, seg.p, seg.g, 1);
      const int tile = seg.dual ? t : 0;
      const int i_row = (2 * seg.p + tile) * tpt + tok_in_tile;      // query or node of this row
      const bool live = tok_in_tile < tpt && i_row < seg.q.n;
      const int nbp = TREE ? va_blocks(seg.q.avail) : 0;
      // packed: this row's keys, and the fewest any row of the tile sees
      const int limit = TREE ? 0 : live ? va_limit(seg.q, i_row) : 0;
      const int tile_limit = TREE ? seg.q.avail : va_limit(seg.q, (2 * seg.p + tile) * tpt);
      const int step = seg.dual ? 1 : 2, n = seg.dual ? (t ? seg.n : seg.n0) : seg.n;
      float m = -INFINITY, l = 0.f;
      bool any = false;
      for (int i = seg.dual ? 0 : t; i < n && ok; i += step) {
        const int b = seg.b0 + i, kb = b * VA_ROWS;
        const bool draft = TREE && b >= nbp;
        uint4 bits = make_uint4(0u, 0u, 0u, 0u);
        if (draft && live) {   // (before the wait: the load overlaps it)
          const uint32_t* mrow = P.mask + ((size_t)seg.s * P.T + i_row) * P.words * 2;
          const int w = (b - nbp) * 4;
          const uint2 lo = *reinterpret_cast<const uint2*>(mrow + w);
          const uint2 hi = w + 2 < 2 * P.words ? *reinterpret_cast<const uint2*>(mrow + w + 2) : make_uint2(0u, 0u);
          const int valid = seg.q.n - (b - nbp) * VA_ROWS;
          bits = make_uint4(lo.x & va_bits_below(valid, 0), lo.y & va_bits_below(valid, 1), hi.x & va_bits_below(valid, 2),
                            hi.y & va_bits_below(valid, 3));
        }
        wait(&s_full[t], ns++ & 1);
        if (!ok) break;
        uint32_t s[128];
#pragma unroll
        for (int k = 0; k < 4; ++k) tmem_ld32(s_col + k * 32, *reinterpret_cast<uint32_t(*)[32]>(&s[k * 32]));
        tmem_ld_wait();
        if (draft || kb + VA_ROWS > tile_limit) {
          if (!draft) {
            const int seen = (TREE ? seg.q.avail : limit) - kb;
            bits = make_uint4(va_bits_below(seen, 0), va_bits_below(seen, 1), va_bits_below(seen, 2), va_bits_below(seen, 3));
          }
#pragma unroll
          for (int e = 0; e < 128; ++e) {
            const uint32_t w = e < 32 ? bits.x : e < 64 ? bits.y : e < 96 ? bits.z : bits.w;
            if (!(w >> (e & 31) & 1u)) s[e] = 0xff800000u;   // -inf
          }
        }
        float mx[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) mx[k] = __uint_as_float(s[k]);
#pragma unroll
        for (int e = 4; e < 128; ++e) mx[e & 3] = fmaxf(mx[e & 3], __uint_as_float(s[e]));
        const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * scale;
        if (__any_sync(0xffffffffu, top > m + VA_ROOM)) {
          const float mn = fmaxf(m, top - VA_HEAD);
          if (any) {   // the rows of O so far follow the new reference
            const float f = mn == -INFINITY ? 1.f : va_ex2(m - mn);
            l *= f;
#pragma unroll 1
            for (int k = 0; k < HD / 32; ++k) {
              uint32_t o[32];
              tmem_ld32(o_col + k * 32, o);
              tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              tmem_st32(o_col + k * 32, o);
            }
          }
          m = mn;
        }
        any = true;
        const float ref = m == -INFINITY ? 0.f : m;
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          uint32_t w[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            const float p0 = va_ex2(fmaf(__uint_as_float(s[k * 64 + 2 * e]), scale, -ref));
            const float p1 = va_ex2(fmaf(__uint_as_float(s[k * 64 + 2 * e + 1]), scale, -ref));
            sum[(2 * e) & 3] += p0;
            sum[(2 * e + 1) & 3] += p1;
            w[e] = va_pack<F16>(p0, p1);
          }
          tmem_st32(s_col + k * 32, w);
        }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[t]);
      }
      if (ok && any) wait(&o_full[t], nseg_o++ & 1);
      if (!ok) break;
      float f0 = 1.f, f1 = 0.f;
      const bool merge = !seg.dual && seg.n > 1;
      if (!seg.dual) {
        if (t == 1) {   // hand (m, l) and O_1 to group 0, and wait until it has read them
          if (!merge) continue;
          s_ml[row] = make_float2(m, l);
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(g1_full);
          wait(g1_empty, ng1++ & 1);
          continue;
        }
        if (merge) {
          wait(g1_full, ng1 & 1);
          if (!ok) break;
          const float2 other = s_ml[row];
          const float mn = fmaxf(m, other.x), ref = mn == -INFINITY ? 0.f : mn;
          f0 = va_ex2(m - ref);
          f1 = va_ex2(other.x - ref);
          l = l * f0 + other.y * f1;
          m = mn;
        }
      }
      const bool whole = seg.n == seg.nb;
      const int slot = 2 * c + (seg.b0 == 0);
      const size_t r = (size_t)(seg.q.q0 + i_row);
      const int h = seg.g * qpg + head_in_group;
      if (whole) {
        const float inv = l > 0.f ? 1.f / l : l;   // (a NaN stays one)
        f0 *= inv;
        f1 *= inv;
        if (live && P.lse) P.lse[r * P.n_heads + h] = (m + __log2f(l)) * 0.6931471805599453f;
      } else if (live) {
        P.part_ml[(size_t)slot * 256 + tile * VA_ROWS + row] = make_float2(m, l);
      }
#pragma unroll 1
      for (int k = 0; k < HD / 32 && any; ++k) {
        uint32_t o[32];
        tmem_ld32(o_col + k * 32, o);
        tmem_ld_wait();
        if (merge) {
          uint32_t o1[32];
          tmem_ld32(o_col + HD + k * 32, o1);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 32; ++e)
            o[e] = __float_as_uint(__uint_as_float(o[e]) * f0 + __uint_as_float(o1[e]) * f1);
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f0);
        }
        if (!live) continue;
        if (whole) {
          uint4* dst = reinterpret_cast<uint4*>(static_cast<uint16_t*>(P.out) + r * P.o_row + h * P.o_head + k * 32);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float* f = reinterpret_cast<const float*>(&o[e * 8]);
            dst[e] = make_uint4(va_pack_out(f[0], f[1], P.out_f16), va_pack_out(f[2], f[3], P.out_f16),
                                va_pack_out(f[4], f[5], P.out_f16), va_pack_out(f[6], f[7], P.out_f16));
          }
        } else {
          uint4* dst = reinterpret_cast<uint4*>(P.part_o + ((size_t)slot * 256 + tile * VA_ROWS + row) * HD + k * 32);
#pragma unroll
          for (int e = 0; e < 8; ++e) dst[e] = make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
        }
      }
      tc_fence_before();
      if (merge) {
        ++ng1;
        __syncwarp();
        if (lane == 0) mbar_arrive(g1_empty);
      }
    }
    if (!ok) *abort_flag = 1;
    if (tid == 0) {
      P.head[2 * c] = tail;
      P.head[2 * c + 1] = make_int4(ok && first.x > 0, first.y, 0, 0);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tbase, 512);
  }
}

// Joins the partials of the items that were cut: block (c, y) takes rows 32 y
// .. 32 y + 31 of the item that begins in CTA c and ends in a later one.  The
// pieces are CTA c's last and the first of the CTAs after it, in that order.
template <int HD, bool TREE>
__global__ void __launch_bounds__(256) varlen_join_kernel(const __grid_constant__ VaParams P, int grid) {
  grid_dep_wait();
  grid_dep_launch();
  const int c = blockIdx.x;
  const int4 tail = P.head[2 * c];
  if (!tail.w) return;
  int last = c;
  for (;;) {
    ++last;
    if (last >= grid) return;   // (a CTA gave up: its word says so)
    const int4 f = P.head[2 * last + 1];
    if (!f.x) return;
    if (f.y) break;
  }
  const VaSeq q = va_seq<TREE>(P, tail.x);
  constexpr int LPR = HD / 4, RPB = 256 / LPR;   // threads per row, rows at once
  const int col = (threadIdx.x % LPR) * 4;
  for (int rr = threadIdx.x / LPR; rr < 32; rr += RPB) {
    const int row = blockIdx.y * 32 + rr, tile = row / VA_ROWS, in_tile = row % VA_ROWS;
    const int tok = in_tile / P.qpg, i_row = (2 * tail.y + tile) * P.tpt + tok;
    if (tok >= P.tpt || i_row >= q.n) continue;
    const size_t at0 = (size_t)(2 * c + 1) * 256 + row;
    float m = P.part_ml[at0].x;
    for (int j = c + 1; j <= last; ++j) m = fmaxf(m, P.part_ml[(size_t)(2 * j) * 256 + row].x);
    const float ref = m == -INFINITY ? 0.f : m;
    float l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int j = c; j <= last; ++j) {
      const size_t at = j == c ? at0 : (size_t)(2 * j) * 256 + row;
      const float2 ml = P.part_ml[at];
      if (ml.x == -INFINITY) continue;   // no key of this row in the piece (its O may not be written)
      const float f = va_ex2(ml.x - ref);
      const float4 x = *reinterpret_cast<const float4*>(P.part_o + at * HD + col);
      l += ml.y * f;
      o.x += x.x * f;
      o.y += x.y * f;
      o.z += x.z * f;
      o.w += x.w * f;
    }
    const float inv = l > 0.f ? 1.f / l : l;
    const int h = tail.z * P.qpg + in_tile - tok * P.qpg;
    const size_t r = (size_t)(q.q0 + i_row);
    uint2* dst = reinterpret_cast<uint2*>(static_cast<uint16_t*>(P.out) + r * P.o_row + h * P.o_head + col);
    *dst = make_uint2(va_pack_out(o.x * inv, o.y * inv, P.out_f16), va_pack_out(o.z * inv, o.w * inv, P.out_f16));
    if (P.lse && col == 0) P.lse[r * P.n_heads + h] = (m + __log2f(l)) * 0.6931471805599453f;
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
static bool va_misaligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }

constexpr int VA_MAX_CTAS = 148;

static int va_host_blocks(int keys) { return (keys + VA_ROWS - 1) / VA_ROWS; }

static size_t va_ws_bytes(int hd) {
  return (size_t)2 * VA_MAX_CTAS * (sizeof(int4) + 256 * (sizeof(float2) + (size_t)hd * sizeof(float)));
}

// 16-bit tensor map with 128-byte swizzle; an axis of extent 1 has no stride.
static bool va_map(CUtensorMap* m, bool f16, const void* base, int rank, const size_t* dim, const size_t* stride,
                   const int* box) {
  const EncodeTiledFn encode = encode_tiled();
  if (encode == nullptr) return false;
  cuuint64_t d[4], st[3];
  cuuint32_t bx[4], es[4];
  for (int i = 0; i < rank; ++i) {
    d[i] = dim[i];
    bx[i] = (cuuint32_t)box[i];
    es[i] = 1;
    if (i) st[i - 1] = (dim[i] == 1 ? dim[0] : stride[i - 1]) * 2;
  }
  return encode(m, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank,
                const_cast<void*>(base), d, st, bx, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
static bool va_kv_map(CUtensorMap* m, bool f16, const void* base, int hd, size_t tokens, size_t heads, size_t seqs,
                      size_t tok, size_t head, size_t seq) {
  const size_t dim[4] = {(size_t)hd, tokens, heads, seqs}, stride[3] = {tok, head, seq};
  const int box[4] = {64, VA_ROWS, 1, 1};
  return va_map(m, f16, base, 4, dim, stride, box);
}

template <int HD, bool F16, bool TREE>
static int va_launch_t(VaParams& P, int grid, bool join, cudaStream_t st) {
  auto kern = varlen_attention_kernel<HD, F16, TREE>;
  if (allow_smem(kern, VaGeom<HD>::BYTES) != T2B_OK) return T2B_ERR_LAUNCH;
  const int rc = launch_pdl(kern, dim3(grid), dim3(VA_THREADS), (size_t)VaGeom<HD>::BYTES, st, P);
  if (rc != T2B_OK || !join) return rc;
  return launch_pdl(varlen_join_kernel<HD, TREE>, dim3(grid, 8), dim3(256), 0, st, P, grid);
}

// max_blocks: no item has more blocks of keys; pairs: no more (sequence, pair of tiles).
static int va_launch(VaParams& P, int hd, bool f16, const void* q, size_t q_row, size_t q_head, long long pairs,
                     long long max_blocks, void* ws, size_t ws_bytes, cudaStream_t st) {
  if (!ws || ws_bytes < va_ws_bytes(hd)) return T2B_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(ws) & 255) return T2B_ERR_ALIGN;
  P.head = static_cast<int4*>(ws);
  P.part_ml = reinterpret_cast<float2*>(P.head + 2 * VA_MAX_CTAS);
  P.part_o = reinterpret_cast<float*>(P.part_ml + 2 * VA_MAX_CTAS * 256);
  P.err = error_word(st);
  const size_t dim[3] = {(size_t)hd, (size_t)P.n_heads, (size_t)P.rows}, stride[2] = {q_head, q_row};
  const int box[3] = {64, P.qpg, P.tpt};
  if (!va_map(&P.qmap, f16, q, 3, dim, stride, box)) return T2B_ERR_ARG;
  int dev = 0, sms = VA_MAX_CTAS;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return T2B_ERR_LAUNCH;
  const long long units = pairs * max_blocks * P.n_kv;
  const int grid = (int)std::max(1ll, std::min<long long>({units / VA_MIN_UNITS, sms, VA_MAX_CTAS}));
  const bool join = grid > 1 && max_blocks > VA_SNAP;
  const bool tree = P.T > 0;
  if (hd == 128) {
    if (f16) return tree ? va_launch_t<128, true, true>(P, grid, join, st) : va_launch_t<128, true, false>(P, grid, join, st);
    return tree ? va_launch_t<128, false, true>(P, grid, join, st) : va_launch_t<128, false, false>(P, grid, join, st);
  }
  if (f16) return tree ? va_launch_t<64, true, true>(P, grid, join, st) : va_launch_t<64, true, false>(P, grid, join, st);
  return tree ? va_launch_t<64, false, true>(P, grid, join, st) : va_launch_t<64, false, false>(P, grid, join, st);
}

}  // namespace t2b

using namespace t2b;

extern "C" size_t t2b_varlen_attention_workspace_bytes(int head_dim) {
  return head_dim == 64 || head_dim == 128 ? va_ws_bytes(head_dim) : 0;
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
  const bool f16 = dtype == T2B_DTYPE_F16;
  P.out = out, P.lse = lse, P.out_f16 = out_dtype == T2B_DTYPE_F16;
  P.rows = total_q, P.n_heads = n_heads, P.n_kv = n_kv, P.qpg = n_heads / n_kv, P.n_seqs = n_seqs;
  P.tpt = VA_ROWS / P.qpg;
  P.o_row = o_row, P.o_head = o_head;
  P.kv_tokens = kv_tokens, P.cached = kv_seqs > 0;
  const size_t seqs = kv_seqs ? kv_seqs : 1;
  if (!va_kv_map(&P.kmap, f16, k, head_dim, kv_tokens, n_kv, seqs, k_tok, k_head, k_seq) ||
      !va_kv_map(&P.vmap, f16, v, head_dim, kv_tokens, n_kv, seqs, v_tok, v_head, v_seq))
    return T2B_ERR_ARG;
  P.q_start = q_start, P.k_start = k_start, P.k_len = k_len;
  P.scale_log2 = scale * 1.4426950408889634f;
  return va_launch(P, head_dim, f16, q, q_row, q_head, total_q / (2 * P.tpt) + (long long)n_seqs,
                   std::max(1, va_host_blocks(kv_tokens)), workspace, workspace_bytes, reinterpret_cast<cudaStream_t>(stream));
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
  const bool f16 = dtype == T2B_DTYPE_F16;
  P.out = out, P.lse = lse, P.out_f16 = out_dtype == T2B_DTYPE_F16;
  P.rows = B * T, P.n_heads = n_heads, P.n_kv = n_kv, P.qpg = n_heads / n_kv, P.n_seqs = B;
  P.tpt = VA_ROWS / P.qpg;
  P.o_row = o_row, P.o_head = o_head;
  P.kv_tokens = max_ctx, P.cached = 1;
  P.ctx_len = ctx_len, P.n_nodes = n_nodes;
  P.mask = reinterpret_cast<const uint32_t*>(mask);
  P.T = T, P.words = (T + 63) / 64;
  P.scale_log2 = scale * 1.4426950408889634f;
  const size_t head = (size_t)max_ctx * head_dim;
  if (!va_kv_map(&P.kmap, f16, k_cache, head_dim, max_ctx, n_kv, B, head_dim, head, n_kv * head) ||
      !va_kv_map(&P.vmap, f16, v_cache, head_dim, max_ctx, n_kv, B, head_dim, head, n_kv * head) ||
      !va_kv_map(&P.kdmap, f16, k_draft, head_dim, T, n_kv, B, kd_node, kd_head, kd_row) ||
      !va_kv_map(&P.vdmap, f16, v_draft, head_dim, T, n_kv, B, vd_node, vd_head, vd_row))
    return T2B_ERR_ARG;
  return va_launch(P, head_dim, f16, q, q_row, q_head, (long long)B * ((T + 2 * P.tpt - 1) / (2 * P.tpt)),
                   va_host_blocks(max_ctx) + va_host_blocks(T), workspace, workspace_bytes,
                   reinterpret_cast<cudaStream_t>(stream));
}
