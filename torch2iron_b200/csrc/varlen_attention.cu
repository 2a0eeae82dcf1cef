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
// of one (sequence, kv head), or its last one.  An item's keys are blocks of
// 128; a block counts one unit for one tile and two for two, an item VA_ITEM
// units more (about what its start and end cost).  The units of the call form
// one list, which the CTAs (one per SM) cut into equal ranges: prompts of any
// lengths, long contexts with few rows and single tokens balance alike without
// the host knowing a length.  An item cut between CTAs leaves fp32 partials
// (output, maximum, sum) that a second kernel joins in a fixed order; items of
// up to VA_SNAP blocks are not cut.  (24 ragged prompts, replays of a graph: 276
// us with blocks alone counted, 180 us with the items' own cost.)  The cut, and
// with it the order of a row's sums, follows from the whole call: the same call
// repeats its bits, the same row in another call need not.
//
// CTA: two softmax groups of eight warps, a TMA warp and an MMA warp.
//   S_t = Q_t K^T     A, B from shared memory (128-byte swizzled TMA tiles)
//   P_t = 2^(S_t c - m)    TMEM -> registers -> TMEM, 16 bits, over S_t
//   O_t += P_t V      A from TMEM, B = V as loaded (MN-major)
// A thread has 64 of a block's keys for one row: no shuffles, and one barrier
// of two warps a block.  While a group is busy with the exponentials of its
// block the tensor core runs the other group's two products.  With both tiles
// live the groups take one tile each and share the K/V blocks; an item of one
// tile (small trees, single tokens, ends of prompts) alternates its blocks
// between the groups, and group 0 joins the two results at the end straight
// from TMEM.
//
// Bound.  A block of two tiles of head_dim 128 is 2048 clocks of MMAs and 2048
// of exponentials (16 a clock) for 64 KB of K and V, which HBM brings in 2700:
// the floor is the products for long prompts and HBM for few rows over a long
// context.  No unit is full: a block takes 3100 clocks, since a tile's two
// products and its softmax wait for one another and two tiles do not hide that
// wholly.  Measured (head_dim 128, 32 over 8 heads): prompts of 3600, 6830 and
// 12001 tokens 1.65 ms a call in a loop = 1.01 PFLOP/s (one launch on a cool
// GPU 1.38 ms = 1.21), the MMA pipe and the special-function unit each busy 62 %
// of the cycles; trees of 63 nodes over 60001 and 45001 keys 142 us a call = 3.05
// TB/s, both at 54 %; trees of 21 nodes at head_dim 64 64 us = 3.3 TB/s, the
// special-function unit at 50 % and the MMA pipe at 25 %.  Tried and not kept:
// one softmax warpgroup per tile (1600 against 1414 us on the prompts), part of
// the exponentials as polynomials on the FMA pipes (no gain: packed FMAs take
// two slots), scores kept in registers instead of read twice (1.60 against 1.44
// ms, more spills; ptxas reports 72 to 88 bytes of spill stores a thread as it
// is, at the 96 registers that 640 threads leave).
//
// Numerics.  Scores, maxima, sums and O are fp32; the weights are rounded
// once, to the operands' 16-bit type, as A of the second product (the sum
// uses them before rounding).  The exponent's reference m is moved, and O
// rescaled, only when a row's maximum outgrows it: it starts VA_HEAD below the
// first block's maximum and moves when a score is more than VA_ROOM above it,
// and the largest weight is at least 2^VA_HEAD of the time it was set, which
// keeps small fp16 weights 2^7 further from underflow.  An exponent is one FMA
// of the score, so it can exceed the rounded difference that was compared by
// half the spacing of fp32 values there: below 2^23 a weight is at most 2^15.5,
// in fp16 range.  A row whose m lies further out takes the branch that moves m
// at every block, and there its scores are scaled and rounded as the maximum
// was, and written back less m (over the scale, which the FMA multiplies by): a
// weight is at most 2^15 and the largest of a block that moved m at least 1.
//
// Every mbarrier wait is time-bounded (T2B_ERR_TIMEOUT in the status word,
// then every role stops at its next wait).

#include <math.h>

#include <algorithm>
#include <initializer_list>
#include <type_traits>
#include <utility>

#include "t2b_common.cuh"
#include "launch.cuh"
#include "tmap.cuh"
#include "tcgen05.cuh"

namespace t2b {

constexpr int VA_MAX_NODES = 256;
constexpr int VA_ROWS = 128;            // rows per tile (MMA M), keys per block (MMA N)
constexpr int VA_THREADS = 640;         // 16 softmax warps, TMA, MMA, 2 that only fill the warpgroup
// Registers: 640 threads are launched with 96 each (61440); the four softmax
// warpgroups take 104 and the fifth gives down to 64: 512 * 104 + 128 * 64 = 61440.
constexpr int VA_REGS_SOFTMAX = 104, VA_REGS_OTHER = 64;
constexpr int VA_WARP_TMA = 16, VA_WARP_MMA = 17;
constexpr int VA_ITEM = 4;              // units an item costs beside its blocks (see Work)
constexpr int VA_SNAP = 8;              // items of up to this many blocks stay in one CTA
constexpr int VA_MIN_UNITS = 5;         // units per CTA, at least
constexpr float VA_HEAD = 7.f, VA_ROOM = 15.f;
constexpr float VA_FAR = 8388608.f;     // 2^23: from here on fp32 values are 1 and more apart

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
  static constexpr int OFF_X = OFF_ML + VA_ROWS * 8;      // float [2][128]: what the halves of a row tell each other
  static constexpr int OFF_BAR = OFF_X + 2 * VA_ROWS * 4;
  static constexpr int N_BARS = 2 + 2 * STAGES + 11;
  static constexpr int OFF_MISC = OFF_BAR + N_BARS * 8;
  static constexpr int BYTES = OFF_MISC + 192;
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
// x / t for x >= 0; a shift where t is a power of two (as the q heads per kv head mostly are)
T2B_DEV int va_div(int x, int t) { return (t & (t - 1)) == 0 ? x >> (__ffs(t) - 1) : x / t; }
T2B_DEV int va_pairs(const VaSeq& q, int tpt) { return va_div(q.n + 2 * tpt - 1, 2 * tpt); }
// sum of floor((a i + b) / 128), i < n, by the Euclidean recursion on the
// lattice points under a line (its divisions are by 128, by a, ..).
T2B_DEV uint32_t va_floor_sum(uint32_t n, uint32_t a, uint32_t b) {
  uint32_t sum = 0, m = VA_ROWS;
  while (n) {
    const uint32_t qa = va_div(a, m), qb = va_div(b, m);
    sum += n * (n - 1) / 2 * qa + n * qb;
    a -= qa * m;
    b -= qb * m;
    const uint32_t y = a * n + b;
    n = va_div(y, m);
    b = y - n * m;
    const uint32_t t = m;
    m = a;
    a = t;
  }
  return sum;
}
// Units of pair p of a sequence, for one kv head.
template <bool TREE>
T2B_DEV uint32_t va_units(const VaSeq& q, int tpt, int p) {
  return va_tile_blocks<TREE>(q, tpt, p, 1) * (q.n > (2 * p + 1) * tpt ? 2 : 1) + VA_ITEM;
}
// Units of pairs 0 .. k - 1, in closed form: pairs that see at most one block,
// then a line's blocks, then pairs that see every key.  (The sequences of a
// long prompt have hundreds of pairs; a loop over them cost 14 us at the start
// of a call.)
template <bool TREE>
T2B_DEV uint32_t va_units_before(const VaSeq& q, int tpt, int pairs, int k) {
  uint32_t last = 0;
  if (k == pairs && k > 0) last = va_units<TREE>(q, tpt, --k);   // only the last pair may be short or alone
  if (TREE) return last + (k ? (uint32_t)k * va_units<TREE>(q, tpt, 0) : 0u);
  const int t = 2 * tpt;                                // pair p sees min(off + (p + 1) t, avail) keys
  const int one = VA_ROWS - q.off < t ? 0 : min(k, va_div(VA_ROWS - q.off, t));
  const int rise = q.avail - q.off <= 0 ? one : max(one, min(k, va_div(q.avail - q.off + t - 1, t) - 1));
  uint32_t blocks = one + (k - rise) * max(1, va_blocks(q.avail));
  if (rise > one) blocks += va_floor_sum(rise - one, t, q.off + (one + 1) * t + VA_ROWS - 1);
  return last + 2 * blocks + k * VA_ITEM;
}

// A position in the list of units: block b of item (s, p, g).
struct VaCursor {
  int s, p, g, b;
};
// Walks a range of the list, one item's blocks at a time.
template <bool TREE>
struct VaWalk {
  VaSeq q;            // the item's sequence
  int s, p, g;        // the item
  int b0, n;          // first block, blocks of this CTA
  int nb, n0;         // the item's blocks; blocks of tile 0 among the n (two tiles)
  bool dual;          // both tiles live
  int left;           // units behind this item's

  T2B_DEV VaWalk(VaCursor at, int units) : s(at.s), p(at.p), g(at.g - 1), b0(at.b), n(-1), left(units) {}
  T2B_DEV bool next(const VaParams& P) {
    if (left <= 0) return false;
    if (n < 0) {
      q = va_seq<TREE>(P, s);
    } else {
      b0 = 0;
    }
    if (++g == P.n_kv) {
      g = 0;
      if (++p == va_pairs(q, P.tpt)) {
        p = 0;
        do {
          s = min(s + 1, P.n_seqs - 1);   // (the bound acts only where the lengths changed under the call)
          q = va_seq<TREE>(P, s);
        } while (q.n == 0 && s + 1 < P.n_seqs);
      }
    }
    dual = q.n > (2 * p + 1) * P.tpt;
    nb = va_tile_blocks<TREE>(q, P.tpt, p, dual ? 1 : 0);
    const int w = dual ? 2 : 1;
    n = min(left / w, nb - b0);
    n0 = dual ? min(n, va_tile_blocks<TREE>(q, P.tpt, p, 0) - b0) : n;
    left -= n * w + (b0 + n == nb ? VA_ITEM : 0);
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
T2B_DEV void va_prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
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
// One lane of the (converged) warp.  The MMAs are issued under this predicate
// and not under lane == 0: ptxas then knows that one lane runs the block and
// keeps the descriptors in uniform registers (64 clocks per 128x128x16 MMA,
// the pipe's rate, against 134 to issue one under a lane test).
T2B_DEV bool va_elect() {
  uint32_t p;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(p));
  return p != 0;
}
// two fp32 values in one 64-bit register: the packed forms issue both lanes at once
typedef unsigned long long f32x2;
T2B_DEV f32x2 va_pair(float a, float b) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
T2B_DEV void va_split(f32x2 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
T2B_DEV f32x2 va_fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
T2B_DEV f32x2 va_add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
T2B_DEV float va_max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
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

// The whole warp waits for a phase of `bar`, at most 0.5 s: true once it is
// complete, false (the same in every lane) when the time is up or another role
// of the CTA has given up.
T2B_DEV bool va_wait(uint64_t* bar, uint32_t phase, volatile int* abort_flag, int* err) {
  if (__all_sync(0xffffffffu, mbar_try_wait(bar, phase))) return true;
  const uint64_t t0 = globaltimer_ns();
  for (;;) {
#pragma unroll 1
    for (int i = 0; i < 16; ++i)
      if (__all_sync(0xffffffffu, mbar_try_wait(bar, phase))) return true;
    const bool late = globaltimer_ns() - t0 > 500000000ull;
    if (__any_sync(0xffffffffu, late || *abort_flag != 0)) {
      if (late && err) atomicCAS(err, 0, T2B_ERR_TIMEOUT);
      return false;
    }
  }
}

// The two warps that hold the halves of 32 rows: a barrier, and one that
// returns whether any of their 64 lanes says so.
T2B_DEV void va_pair_sync(int id) { asm volatile("bar.sync %0, 64;" ::"r"(id) : "memory"); }
T2B_DEV bool va_pair_any(int id, bool v) {
  uint32_t r;
  asm volatile("{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n bar.red.or.pred q, %2, 64, p;\n selp.u32 %0, 1, 0, q;\n}\n"
               : "=r"(r)
               : "r"((uint32_t)v), "r"(id)
               : "memory");
  return r != 0;
}

// 4x4 transpose of 16-byte pieces over a quad of lanes.
T2B_DEV void va_transpose(uint4 (&x)[4], int lane) {
#pragma unroll
  for (int m = 1; m <= 2; m <<= 1) {
    const bool up = (lane & m) != 0;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      if (c & m) continue;
      const uint4 send = up ? x[c] : x[c + m];
      uint4 got;
      got.x = __shfl_xor_sync(0xffffffffu, send.x, m);
      got.y = __shfl_xor_sync(0xffffffffu, send.y, m);
      got.z = __shfl_xor_sync(0xffffffffu, send.z, m);
      got.w = __shfl_xor_sync(0xffffffffu, send.w, m);
      if (up) x[c] = got;
      else x[c + m] = got;
    }
  }
}

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
  uint8_t* sm = smem_dyn;
  if (smem_u32(sm) & 1023) {   // (the swizzled tiles need it; the kernel has no other shared memory)
    if (threadIdx.x == 0) {
      P.head[2 * blockIdx.x] = P.head[2 * blockIdx.x + 1] = make_int4(0, 0, 0, 0);
      if (P.err) atomicCAS(P.err, 0, T2B_ERR_ALIGN);
    }
    return;
  }
  float* s_x = reinterpret_cast<float*>(sm + G::OFF_X);
  float2* s_ml = reinterpret_cast<float2*>(sm + G::OFF_ML);
  uint64_t* q_full = reinterpret_cast<uint64_t*>(sm + G::OFF_BAR);
  uint64_t* q_empty = q_full + 1;
  uint64_t* kv_full = q_full + 2;
  uint64_t* kv_empty = kv_full + NS;
  uint64_t* s_full = kv_empty + NS;      // [2]
  uint64_t* p_full = s_full + 2;         // [2][halves of a block]
  uint64_t* o_full = p_full + 4;         // [2]
  uint64_t* g1_full = o_full + 2;
  uint64_t* g1_empty = g1_full + 1;
  uint64_t* done = g1_full + 2;
  uint32_t* s_scan = reinterpret_cast<uint32_t*>(sm + G::OFF_MISC);            // [warps]
  VaCursor* s_at = reinterpret_cast<VaCursor*>(sm + G::OFF_MISC + 80);
  uint2* s_cut = reinterpret_cast<uint2*>(sm + G::OFF_MISC + 96);              // [2]: sequence, unit inside it
  uint32_t* s_range = reinterpret_cast<uint32_t*>(sm + G::OFF_MISC + 112);     // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sm + G::OFF_MISC + 120);
  int* s_flag = reinterpret_cast<int*>(sm + G::OFF_MISC + 124);
  volatile int* s_bad = reinterpret_cast<volatile int*>(sm + G::OFF_MISC + 128);   // [8]: a warp of the pair gave up
  volatile int* abort_flag = s_flag;

  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);   // (uniform, and known to be)
  if (tid == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int i = 0; i < NS; ++i) {
      mbar_init(&kv_full[i], 1);
      mbar_init(&kv_empty[i], 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&s_full[t], 1);
      mbar_init(&p_full[2 * t], 4);   // one arrival per softmax warp
      mbar_init(&p_full[2 * t + 1], 4);
      mbar_init(&o_full[t], 1);
    }
    mbar_init(g1_full, 8);    // one arrival per warp of the group
    mbar_init(g1_empty, 8);
    mbar_init(done, 1);
    *abort_flag = 0;
    for (int i = 0; i < 8; ++i) s_bad[i] = 0;
    fence_mbar_init();
  }
  if (tid == 32) {   // the descriptors are kernel parameters: their fetch need not wait for the predecessor
    va_prefetch_map(&P.qmap);
    va_prefetch_map(&P.kmap);
    va_prefetch_map(&P.vmap);
    if (TREE) {
      va_prefetch_map(&P.kdmap);
      va_prefetch_map(&P.vdmap);
    }
  }
  if (warp == VA_WARP_MMA) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  grid_dep_wait();

  // ---- this CTA's range of the list of units (at most 2^31 - 1: checked on the host) ----
  const int c = blockIdx.x;
  VaSeq mine;
  auto seq_units = [&](int s) -> uint32_t {
    if (s >= P.n_seqs) return 0;
    mine = va_seq<TREE>(P, s);
    const int pairs = va_pairs(mine, P.tpt);
    return va_units_before<TREE>(mine, P.tpt, pairs, pairs) * P.n_kv;
  };
  // inclusive sum of one value per thread over the block, and the block's total
  auto block_scan = [&](uint32_t v, uint32_t& sum) -> uint32_t {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t w = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += w;
    }
    __syncthreads();
    if (lane == 31) s_scan[warp] = v;
    __syncthreads();
    uint32_t before = 0;
    sum = 0;
#pragma unroll
    for (int w = 0; w < VA_THREADS / 32; ++w) {
      const uint32_t x = s_scan[w];
      before += w < warp ? x : 0u;
      sum += x;
    }
    return before + v;
  };
  uint32_t total = 0, units0 = 0, end0 = 0;   // the first VA_THREADS sequences' are kept
  for (int s0 = 0; s0 < P.n_seqs; s0 += VA_THREADS) {
    uint32_t sum;
    const uint32_t u = seq_units(s0 + tid), e = block_scan(u, sum);
    if (s0 == 0) units0 = u, end0 = e;
    total += sum;
  }
  const uint32_t parts = min((uint32_t)gridDim.x, max(1u, total / VA_MIN_UNITS));
  const bool busy = total > 0 && c < (int)parts;
  const uint32_t each = total / parts, more = total - each * parts;   // the first `more` ranges have one unit more
  const uint32_t cut[2] = {each * c + min((uint32_t)c, more), each * (c + 1) + min((uint32_t)c + 1, more)};
  if (tid == 0) {
    s_range[0] = 0;
    s_range[1] = busy ? total : 0;   // (kept where the range's end is the end of the list)
    s_cut[0] = s_cut[1] = make_uint2(0xffffffffu, 0u);
  }
  if (busy) {
    uint32_t base = 0;
    for (int s0 = 0; s0 < P.n_seqs; s0 += VA_THREADS) {
      uint32_t u = units0, e = end0, sum;
      if (P.n_seqs > VA_THREADS) {
        u = seq_units(s0 + tid);
        e = block_scan(u, sum) + base;
        base += sum;
      } else {
        __syncthreads();
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (cut[i] < e && cut[i] >= e - u) s_cut[i] = make_uint2(s0 + tid, cut[i] - (e - u));
    }
    __syncthreads();
    // half of the threads look for each cut inside its sequence
    const int i = tid / (VA_THREADS / 2), t = tid - i * (VA_THREADS / 2);
    const int s = (int)s_cut[i].x;
    if (s >= 0) {
      const uint32_t u = s_cut[i].y;
      const VaSeq q = va_seq<TREE>(P, s);
      const int pairs = va_pairs(q, P.tpt), step = (pairs + VA_THREADS / 2 - 1) / (VA_THREADS / 2);
      int p = t * step;
      uint32_t at = p < pairs ? va_units_before<TREE>(q, P.tpt, pairs, p) * P.n_kv : 0u;
      for (const int last = min(pairs, p + step); p < last; ++p) {
        const uint32_t w = va_units<TREE>(q, P.tpt, p);
        if (u >= at && u - at < w * P.n_kv) {   // one thread's
          const int bw = q.n > (2 * p + 1) * P.tpt ? 2 : 1, nb = (int)(w - VA_ITEM) / bw;
          int g = (u - at) / w, rest = (u - at) - g * w, b = rest / bw, np = p;
          uint32_t place = cut[i] - rest;       // the item's start
          if (b >= nb || (nb <= VA_SNAP && rest)) {
            if (2 * rest >= (int)w) {           // up to the next item
              place += w;
              if (++g == P.n_kv) {
                g = 0;
                ++np;
              }
            }
            b = 0;
          }
          place += b * bw;
          s_range[i] = place;
          if (i == 0) {
            int ns = s;
            if (np == pairs) {   // (behind the sequence: the next one that has rows; unused at the list's end)
              np = 0;
              do ++ns;
              while (ns < P.n_seqs && va_seq<TREE>(P, ns).n == 0);
            }
            *s_at = {ns, np, g, b};
          }
        }
        at += w * P.n_kv;
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
  if (warp >= VA_WARP_TMA) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(VA_REGS_OTHER));
    VaWalk<TREE> seg(start, units);
    if (warp == VA_WARP_TMA) {
      // ---- TMA: per segment K0, (Q), K1, V0, K2, V1, ..: the order the MMAs take them ----
      if (lane == 0) {
        int pos = 0, nseg = 0, q_loads = 0;
        bool ok = true;
        int4 tail = make_int4(0, 0, 0, 0), first = make_int4(0, 0, 0, 0);   // this CTA's ends, for the joining kernel
        for (; ok && seg.next(P); ++nseg) {
          if (nseg == 0) first = make_int4(seg.b0 > 0, seg.b0 + seg.n == seg.nb, 0, 0);
          if (seg.b0 == 0 && seg.n < seg.nb) tail = make_int4(seg.s, seg.p, seg.g, 1);
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
        if (!ok) tail.w = first.x = 0;
        P.head[2 * c] = tail;
        P.head[2 * c + 1] = first;
      }
    } else if (warp == VA_WARP_MMA) {
      // ---- MMA issuer (one lane; the others help to clear V rows).  It shares its
      //      scheduler with four softmax warps, so every instruction here delays
      //      the tensor pipe: descriptors are a base plus an offset, the waits for
      //      K and V come before those for P, and a block's MMAs and commits are
      //      issued in one go.  (A second issuer for the other tile was slower:
      //      the pipe then interleaves the two tiles' products and finishes both
      //      late; packed prompts of 12k tokens 1.48 -> 2.46 ms.) ----
      constexpr uint32_t FMT = F16 ? 0u : (1u << 7) | (1u << 10);
      constexpr uint32_t ID_S = (1u << 4) | FMT | ((uint32_t)(VA_ROWS >> 3) << 17) | ((uint32_t)(VA_ROWS >> 4) << 24);
      constexpr uint32_t ID_O = (1u << 4) | FMT | (1u << 16) | ((uint32_t)(HD >> 3) << 17) | ((uint32_t)(VA_ROWS >> 4) << 24);
      // descriptors of Q tile 0 and of K and V in stage 0 (the offsets stay inside the address field)
      const uint64_t q_desc = sdesc_sw128(smem_u32(sm)), k_desc = sdesc_sw128(smem_u32(sm) + G::OFF_KV);
      const uint64_t v_desc = sdesc_mn_sw128(smem_u32(sm) + G::OFF_KV, VA_ROWS * 128);
      int ring = 0, nseg = 0;
      uint32_t np[2] = {0u, 0u};
      bool ok = true;
      auto wait = [&](uint64_t* bar, uint32_t ph) {
        ok = ok && va_wait(bar, ph, abort_flag, P.err);
        tc_fence_after();
      };
      for (; ok && seg.next(P); ++nseg) {
        const int n = seg.n;
        const uint64_t q1_desc = q_desc + (seg.dual ? (G::TILE >> 4) : 0);
        auto at_k = [&](int i) { return ring + (i ? 2 * i - 1 : 0); };
        auto at_v = [&](int i) { return ring + (i < n - 1 ? 2 * i + 2 : 2 * n - 1); };
        auto kv_wait = [&](int at) { wait(&kv_full[at % NS], (at / NS) & 1); };
        auto issue_s = [&](auto tile, int st) {   // S_t = Q K^T, K in stage st
          constexpr int t = decltype(tile)::value;
          const uint64_t qd = t ? q1_desc : q_desc, kd = k_desc + st * (G::TILE >> 4);
#pragma unroll
          for (int ks = 0; ks < HD / 16; ++ks) {
            const uint32_t o = ((ks >> 2) * (VA_ROWS * 128) + (ks & 3) * 32) >> 4;
            mma_ss(tbase + G::S0 + t * 128, qd + o, kd + o, ID_S, ks > 0);
          }
          mma_commit(&s_full[t]);
        };
        // O_t += P_t V(i), then S_t of block j (-1: none, O_t is complete).  `free`:
        // V(i) and K(j) have no other reader.
        auto advance = [&](auto tile, int i, bool first, int j, bool free) {
          constexpr int t = decltype(tile)::value;
          const int sv = at_v(i) % NS, sk = j >= 0 ? at_k(j) % NS : 0;
          const uint64_t vd = v_desc + sv * (G::TILE >> 4);
          const uint32_t ph = np[t]++ & 1;
          wait(&p_full[2 * t], ph);
          if (ok && va_elect()) {
#pragma unroll
            for (int ks = 0; ks < 4; ++ks)
              mma_ts(tbase + G::O0 + t * HD, tbase + G::S0 + t * 128 + ks * 8, vd + ks * (2048 >> 4), ID_O, !(first && ks == 0));
          }
          wait(&p_full[2 * t + 1], ph);
          if (ok && va_elect()) {
#pragma unroll
            for (int ks = 4; ks < 8; ++ks)
              mma_ts(tbase + G::O0 + t * HD, tbase + G::S0 + t * 128 + 64 + (ks & 3) * 8, vd + ks * (2048 >> 4), ID_O, 1u);
            if (free) mma_commit(&kv_empty[sv]);
            if (j >= 0) {
              issue_s(tile, sk);
              if (free) mma_commit(&kv_empty[sk]);
              if (free && j == n - 1) mma_commit(q_empty);
            } else {
              mma_commit(&o_full[t]);
            }
          }
        };
        // Drafted nodes that any node's mask names, blocks 0 and 1 of the drafts
        // (read while the first block's softmax runs).
        const int nbp = TREE ? va_blocks(seg.q.avail) : 0;
        uint32_t named[8];
        auto read_named = [&] {
          if (!TREE || seg.b0 + n <= nbp) return;
          const int words = 2 * P.words;
          const uint32_t* rows = P.mask + (size_t)seg.s * P.T * words;
#pragma unroll
          for (int w = 0; w < 8; ++w) named[w] = 0u;
          for (int r = lane; r < seg.q.n; r += 32) {
#pragma unroll
            for (int w = 0; w < 8; ++w)
              if (w < words) named[w] |= rows[(size_t)r * words + w];
          }
#pragma unroll
          for (int w = 0; w < 8; ++w) named[w] = __reduce_or_sync(0xffffffffu, named[w]);
        };
        // Rows of V(i) that no row of the item sees are cleared: their weights are
        // 0, but 0 * (whatever lies there) may be NaN.
        auto clear = [&](int i) {
          const int b = seg.b0 + i;
          const bool draft = TREE && b >= nbp;
          const int valid = draft ? seg.q.n - (b - nbp) * VA_ROWS : seg.q.avail - b * VA_ROWS;
          uint8_t* v = sm + G::OFF_KV + (at_v(i) % NS) * G::TILE + (lane & 7) * 16;
          bool any = false;
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            uint32_t seen = va_bits_below(valid, w);
            if (draft) seen &= b > nbp ? named[4 + w] : named[w];
            if (seen == 0xffffffffu) continue;
            any = true;
            for (int r = lane >> 3; r < 32; r += 4)   // 8 lanes clear one row's 128 bytes
              if (!(seen >> r & 1u))
                for (int hf = 0; hf < HALVES; ++hf)
                  *reinterpret_cast<uint4*>(v + hf * (VA_ROWS * 128) + (w * 32 + r) * 128) = make_uint4(0u, 0u, 0u, 0u);
          }
          if (any) {
            fence_proxy_async();
            __syncwarp();
          }
        };
        // the first block that is not whole: a prefix's or prompt's end, then the drafts
        const int ragged = seg.q.avail / VA_ROWS - seg.b0;
        constexpr std::integral_constant<int, 0> T0{};
        constexpr std::integral_constant<int, 1> T1{};
        wait(q_full, nseg & 1);
        kv_wait(at_k(0));
        if (seg.dual) {
          if (ok && va_elect()) {
            const int st = at_k(0) % NS;
            if (seg.n0 > 0) issue_s(T0, st);
            issue_s(T1, st);
            mma_commit(&kv_empty[st]);
            if (n == 1) mma_commit(q_empty);
          }
          read_named();
          for (int i = 0; i < n && ok; ++i) {
            kv_wait(at_v(i));
            if (i >= ragged && ok) clear(i);
            const int j = i + 1 < n ? i + 1 : -1;
            if (j >= 0) kv_wait(at_k(j));
            if (i < seg.n0) advance(T0, i, i == 0, j < seg.n0 ? j : -1, false);
            advance(T1, i, i == 0, j, true);
          }
        } else {
          if (n > 1) kv_wait(at_k(1));
          if (ok && va_elect()) {
            issue_s(T0, at_k(0) % NS);
            mma_commit(&kv_empty[at_k(0) % NS]);
            if (n > 1) {
              issue_s(T1, at_k(1) % NS);
              mma_commit(&kv_empty[at_k(1) % NS]);
            }
            if (n <= 2) mma_commit(q_empty);
          }
          read_named();
          for (int i = 0; i < n && ok; ++i) {
            kv_wait(at_v(i));
            if (i >= ragged && ok) clear(i);
            const int j = i + 2 < n ? i + 2 : -1;
            if (j >= 0) kv_wait(at_k(j));
            if (i & 1) advance(T1, i, i < 2, j, true);
            else advance(T0, i, i < 2, j, true);
          }
        }
        ring += 2 * n;
      }
      if (!ok) *abort_flag = 1;
      // every MMA issued here has retired before TMEM is released
      __syncwarp();
      if (va_elect()) mma_commit(done);
      mbar_wait_bounded(done, 0, P.err);
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(VA_REGS_SOFTMAX));
    VaWalk<TREE> seg(start, units);
    // ---- softmax group t, half u: a thread has 64 of the 128 keys of a block for
    //      one row, and half of the row's output columns.  Two warps make a pair
    //      for 32 rows; every decision that a pair's barriers depend on is taken
    //      by both (va_pair_any), so that none is left at one. ----
    const int t = warp >> 3, u = (warp >> 2) & 1, row = (warp & 3) * 32 + lane;
    const int pair = t * 4 + (warp & 3), bar = 1 + pair;
    const uint32_t lanes = tbase + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t s_col = lanes + G::S0 + t * 128 + u * 64, p_col = s_col;
    const uint32_t o_col = lanes + G::O0 + t * HD + u * (HD / 2);
    float* x_slot = s_x + t * VA_ROWS + row;
    const int tok_in_tile = row / qpg, head_in_group = row - tok_in_tile * qpg;
    const float scale = P.scale_log2;
    int ns = 0, nseg_o = 0, ng1 = 0;
    bool ok = true;
    auto wait = [&](uint64_t* b, uint32_t ph) {
      ok = ok && va_wait(b, ph, abort_flag, P.err);
      tc_fence_after();
    };
    auto agree = [&] { ok = !va_pair_any(bar, !ok); };
    while (ok && seg.next(P)) {
      const int tile = seg.dual ? t : 0;
      const int i_row = (2 * seg.p + tile) * tpt + tok_in_tile;      // query or node of this row
      const bool live = tok_in_tile < tpt && i_row < seg.q.n;
      const int nbp = TREE ? va_blocks(seg.q.avail) : 0;
      // packed: this row's keys, and the fewest any row of the tile sees
      const int limit = TREE ? seg.q.avail : live ? va_limit(seg.q, i_row) : 0;
      const int tile_limit = TREE ? seg.q.avail : va_limit(seg.q, (2 * seg.p + tile) * tpt);
      const int step = seg.dual ? 1 : 2, n = seg.dual ? (t ? seg.n : seg.n0) : seg.n;
      float m = -INFINITY, l = 0.f;
      float limit_m = -INFINITY, ref = 0.f;   // a greater score moves m; what the exponents subtract
      bool any = false;
      for (int i = seg.dual ? 0 : t; i < n && ok; i += step) {
        const int b = seg.b0 + i, kb = b * VA_ROWS;
        const bool draft = TREE && b >= nbp;
        const bool masked = draft || kb + VA_ROWS > tile_limit;
        uint2 bits = make_uint2(0u, 0u);
        if (draft) {
          const int word = (b - nbp) * 4 + u * 2, valid = seg.q.n - (b - nbp) * VA_ROWS;
          if (live && word < 2 * P.words) {   // (before the wait: the load overlaps it)
            bits = *reinterpret_cast<const uint2*>(P.mask + ((size_t)seg.s * P.T + i_row) * P.words * 2 + word);
            bits = make_uint2(bits.x & va_bits_below(valid, 2 * u), bits.y & va_bits_below(valid, 2 * u + 1));
          }
        } else if (masked) {
          bits = make_uint2(va_bits_below(limit - kb, 2 * u), va_bits_below(limit - kb, 2 * u + 1));
        }
        wait(&s_full[t], ns++ & 1);
        float mx[4];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          uint32_t s[32];
          tmem_ld32(s_col + k * 32, s);
          tmem_ld_wait();
          if (masked) {
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (!((k == 0 ? bits.x : bits.y) >> e & 1u)) s[e] = 0xff800000u;   // -inf
          }
          if (k == 0) {
#pragma unroll
            for (int e = 0; e < 4; ++e) mx[e] = __uint_as_float(s[e]);
          }
#pragma unroll
          for (int e = k == 0 ? 4 : 0; e < 32; e += 2)
            mx[(e >> 1) & 3] = va_max3(mx[(e >> 1) & 3], __uint_as_float(s[e]), __uint_as_float(s[e + 1]));
        }
        const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * scale;
        if (!ok) s_bad[pair] = 1;
        // (behind this barrier both halves hold their scores; a row that is not live
        // holds whatever was there, and must not decide when its neighbours rescale)
        if (va_pair_any(bar, (live && top > limit_m) || !ok)) {
          if (u) *x_slot = top;
          va_pair_sync(bar);
          if (s_bad[pair]) {
            ok = false;
            break;
          }
          if (!u) *x_slot = fmaxf(m, fmaxf(top, *x_slot) - VA_HEAD);
          va_pair_sync(bar);
          const float mn = *x_slot;
          if (any) {   // the rows of O so far follow the new reference
            const float f = mn == -INFINITY ? 1.f : va_ex2(m - mn);
            l *= f;
#pragma unroll 1
            for (int k = 0; k < HD / 64; ++k) {
              uint32_t o[32];
              tmem_ld32(o_col + k * 32, o);
              tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              tmem_st32(o_col + k * 32, o);
            }
            tmem_st_wait();
          }
          m = mn;
          const bool far = live && fabsf(m) >= VA_FAR && m != -INFINITY;
          limit_m = far ? -INFINITY : __fadd_rd(m, VA_ROOM);   // (rounded down: the comparison is exact)
          ref = far || m == -INFINITY ? 0.f : m;
          if (__any_sync(0xffffffffu, far)) {   // a far row's scores become differences from m (see Numerics)
            const float per = 1.f / scale;
#pragma unroll 1
            for (int k = 0; k < 4; ++k) {
              uint32_t s[16];
              tmem_ld16(s_col + k * 16, s);
              tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 16; ++e)
                if (far) s[e] = __float_as_uint(__fsub_rn(__fmul_rn(__uint_as_float(s[e]), scale), m) * per);
              tmem_st16(s_col + k * 16, s);
            }
            tmem_st_wait();
          }
          tc_fence_before();
          va_pair_sync(bar);   // both halves of O are ready before either half of P is announced
        }
        any = true;
        const f32x2 scale2 = va_pair(scale, scale), ref2 = va_pair(-ref, -ref);
        f32x2 sum[2] = {0ull, 0ull};
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          uint32_t w[16], s[32];
          tmem_ld32(s_col + j * 32, s);
          tmem_ld_wait();
          if (masked) {
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (!((j == 0 ? bits.x : bits.y) >> e & 1u)) s[e] = 0xff800000u;   // -inf
          }
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int i0 = 2 * e;
            float p0, p1;
            va_split(va_fma2(va_pair(__uint_as_float(s[i0]), __uint_as_float(s[i0 + 1])), scale2, ref2), p0, p1);
            p0 = va_ex2(p0);
            p1 = va_ex2(p1);
            sum[e & 1] = va_add2(sum[e & 1], va_pair(p0, p1));
            w[e] = va_pack<F16>(p0, p1);
          }
          tmem_st16(p_col + j * 16, w);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[2 * t + u]);
        float l0, l1;
        va_split(va_add2(sum[0], sum[1]), l0, l1);
        l += l0 + l1;
      }
      if (!ok) break;
      if (any) wait(&o_full[t], nseg_o++ & 1);
      agree();
      if (!ok) break;
      if (u) *x_slot = l;   // the row's sum
      va_pair_sync(bar);
      if (!u) *x_slot = l += *x_slot;
      va_pair_sync(bar);
      l = *x_slot;
      float f0 = 1.f, f1 = 0.f;
      const bool merge = !seg.dual && seg.n > 1;
      if (!seg.dual) {
        if (t == 1) {   // hand (m, l) and O_1 to group 0, and wait until it has read them
          if (!merge) continue;
          if (!u) s_ml[row] = make_float2(m, l);
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(g1_full);
          wait(g1_empty, ng1++ & 1);
          agree();
          continue;
        }
        if (merge) {
          wait(g1_full, ng1++ & 1);
          agree();
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
        if (live && !u && P.lse) P.lse[r * P.n_heads + h] = (m + __log2f(l)) * 0.6931471805599453f;
      } else if (live && !u) {
        P.part_ml[(size_t)slot * 256 + tile * VA_ROWS + row] = make_float2(m, l);
      }
      // Rows leave in 16-byte pieces that a quad of lanes has transposed, so that
      // a store covers 64 contiguous bytes of 8 rows and not 16 of 32.
      uint8_t* start = nullptr;
      if (live && any)
        start = whole ? static_cast<uint8_t*>(P.out) + (r * P.o_row + h * P.o_head) * 2 + u * HD
                     : reinterpret_cast<uint8_t*>(P.part_o + ((size_t)slot * 256 + tile * VA_ROWS + row) * HD + u * (HD / 2));
      uint8_t* dst[4];   // this lane's piece of the quad's rows
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        dst[j] = reinterpret_cast<uint8_t*>(
            __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(start), (lane & ~3) + j));
        if (dst[j]) dst[j] += (lane & 3) * 16;
      }
      auto store = [&](uint4 (&x)[4], int off) {
        va_transpose(x, lane);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (dst[j]) *reinterpret_cast<uint4*>(dst[j] + off) = x[j];
      };
#pragma unroll 1
      for (int k = 0; k < HD / 64 && any; ++k) {
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
        uint4 x[4];
        if (whole) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float* f = reinterpret_cast<const float*>(&o[e * 8]);
            x[e] = make_uint4(va_pack_out(f[0], f[1], P.out_f16), va_pack_out(f[2], f[3], P.out_f16),
                              va_pack_out(f[4], f[5], P.out_f16), va_pack_out(f[6], f[7], P.out_f16));
          }
          store(x, k * 64);
        } else {
#pragma unroll
          for (int half = 0; half < 2; ++half) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int i = half * 16 + e * 4;
              x[e] = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
            }
            store(x, k * 128 + half * 64);
          }
        }
      }
      tc_fence_before();
      if (merge) {
        __syncwarp();
        if (lane == 0) mbar_arrive(g1_empty);
      }
    }
    if (!ok) *abort_flag = 1;
  }
  tc_fence_before();
  __syncthreads();
  if (warp == VA_WARP_MMA) {
    tc_fence_after();
    tmem_dealloc(tbase, 512);
  }
}

constexpr int VA_JOIN_Y = 8;            // blocks per item that was cut

// Joins the partials of the items that were cut: block (c, y) takes a few rows
// of the item that begins in CTA c and ends in a later one.  The pieces are
// CTA c's last and the first of the CTAs after it, joined in that order.  The
// loads of eight pieces are in flight at once.
template <int HD, bool TREE>
__global__ void __launch_bounds__(256) varlen_join_kernel(const __grid_constant__ VaParams P, int grid) {
  constexpr int LPR = HD / 4, ROWS = 256 / LPR, BATCH = 8;   // threads per row, rows per block
  grid_dep_wait();
  grid_dep_launch();
  const int c = blockIdx.x;
  const int4 tail = P.head[2 * c];
  if (!tail.w) return;
  const VaSeq q = va_seq<TREE>(P, tail.x);
  const int col = (threadIdx.x % LPR) * 4;
  int last = c;
  for (;;) {
    if (++last >= grid) return;   // (a CTA gave up: the status word says so)
    const int4 f = P.head[2 * last + 1];
    if (!f.x) return;
    if (f.y) break;
  }
  for (int row = blockIdx.y * ROWS + threadIdx.x / LPR; row < 2 * VA_ROWS; row += ROWS * VA_JOIN_Y) {
    const int tile = row / VA_ROWS, in_tile = row % VA_ROWS;
    const int tok = in_tile / P.qpg, i_row = (2 * tail.y + tile) * P.tpt + tok;
    if (tok >= P.tpt || i_row >= q.n) continue;
    float m = -INFINITY, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int j0 = c; j0 <= last; j0 += BATCH) {
      float2 ml[BATCH];
      float4 x[BATCH];
#pragma unroll
      for (int k = 0; k < BATCH; ++k) {
        const int j = j0 + k;
        const size_t at = (size_t)(2 * j + (j == c)) * 256 + row;
        ml[k] = j <= last ? P.part_ml[at] : make_float2(-INFINITY, 0.f);
        x[k] = j <= last ? *reinterpret_cast<const float4*>(P.part_o + at * HD + col) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
      float mn = m;
#pragma unroll
      for (int k = 0; k < BATCH; ++k) mn = fmaxf(mn, ml[k].x);
      const float ref = mn == -INFINITY ? 0.f : mn;
      const float f = va_ex2(m - ref);
      l *= f;
      o = make_float4(o.x * f, o.y * f, o.z * f, o.w * f);
#pragma unroll
      for (int k = 0; k < BATCH; ++k) {
        if (ml[k].x == -INFINITY) continue;   // no key of this row in the piece (its O may not be written)
        const float w = va_ex2(ml[k].x - ref);
        l += ml[k].y * w;
        o.x += x[k].x * w;
        o.y += x[k].y * w;
        o.z += x[k].z * w;
        o.w += x[k].w * w;
      }
      m = mn;
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
constexpr int VA_MAX_KEYS = 0x7fff0000;   // (positions plus a block stay in an int)

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
  return launch_pdl(varlen_join_kernel<HD, TREE>, dim3(grid, VA_JOIN_Y), dim3(256), 0, st, P, grid);
}

// Upper bounds of a call's units, which the kernel counts in 32 bits.  The host
// knows no length: `pairs` bounds the pairs of tiles of all sequences, and each
// may see all keys there are.
static double va_most_units(double pairs, int max_blocks, int n_kv) {
  return pairs * (2.0 * max_blocks + VA_ITEM) * n_kv;
}
// Prompts over their own packed keys: pair p of a prompt sees 2 tpt (p + 1) keys
// at most, so a prompt of x pairs has tpt / 64 x (x + 1) units of keys and
// (2 + VA_ITEM) x more, and all prompts together no more than one of all rows
// has beside the short ones' first pairs.
static double va_most_units_own(int rows, double seqs, int tpt, int n_kv) {
  const double x = rows / (2 * tpt) + 1;
  return (tpt / 64.0 * (x * x + 3 * x + 2 * seqs) + (2 + VA_ITEM) * (x + seqs)) * n_kv;
}

// units: no more of them; max_blocks: no item has more blocks of keys.
static int va_check_sizes(int hd, double units, const void* ws, size_t ws_bytes) {
  if (units > 2147483647.0) return T2B_ERR_SHAPE;
  if (!ws || ws_bytes < va_ws_bytes(hd)) return T2B_ERR_WORKSPACE;
  return reinterpret_cast<uintptr_t>(ws) & 255 ? T2B_ERR_ALIGN : T2B_OK;
}
static int va_launch(VaParams& P, int hd, bool f16, const void* q, size_t q_row, size_t q_head, double units,
                     int max_blocks, void* ws, cudaStream_t st) {
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
  const int grid = std::max(1, std::min({(int)(units / VA_MIN_UNITS), sms, VA_MAX_CTAS}));
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

// Memory of a tensor: `inner` bytes at every combination of the axes (the
// greatest stride first, axes of one left out).
struct VaBox {
  uintptr_t at;
  long long inner;
  int n;
  long long dim[3], stride[3];
  VaBox(const void* p, long long bytes, std::initializer_list<std::pair<size_t, size_t>> axes = {})   // (extent, 16-bit stride)
      : at(reinterpret_cast<uintptr_t>(p)), inner(bytes), n(0) {
    for (const auto& x : axes) {
      if (x.first == 1) continue;
      int i = n++;
      for (; i > 0 && stride[i - 1] < (long long)x.second * 2; --i) dim[i] = dim[i - 1], stride[i] = stride[i - 1];
      dim[i] = (long long)x.first, stride[i] = (long long)x.second * 2;
    }
  }
  long long span(int level) const {
    long long s = inner;
    for (int i = level; i < n; ++i) s += (dim[i] - 1) * stride[i];
    return s;
  }
};
// No byte in common: the spans are apart, or what lies in one period of the
// greater stride is (both repeat with it, as rows or heads of one wider tensor
// do, or one does and the other lies between).  `d`: from a's start to b's.
static bool va_apart(const VaBox& a, const VaBox& b, int i, int j, long long d) {
  if (d >= a.span(i) || d + b.span(j) <= 0) return true;
  const long long sa = i < a.n ? a.stride[i] : 0, sb = j < b.n ? b.stride[j] : 0, s = std::max(sa, sb);
  if (s == 0) return false;
  i += sa == s, j += sb == s;
  if (a.span(i) > s || b.span(j) > s) return false;
  const long long r = ((d % s) + s) % s;
  return va_apart(a, b, i, j, r) && va_apart(a, b, i, j, r - s);
}
static bool va_apart(const VaBox& a, const VaBox& b) { return va_apart(a, b, 0, 0, (long long)(b.at - a.at)); }
// The results overlap neither the inputs nor one another; out may lie on q, row by row.
static bool va_results_apart(const VaBox& out, const float* lse, size_t lse_values, const VaBox& q, bool same_layout,
                             std::initializer_list<VaBox> inputs) {
  if (!(out.at == q.at && same_layout) && !va_apart(out, q)) return false;
  for (const VaBox& x : inputs)
    if (!va_apart(out, x)) return false;
  if (!lse) return true;
  const VaBox sums(lse, (long long)lse_values * 4);
  for (const VaBox& x : inputs)
    if (!va_apart(sums, x)) return false;
  return va_apart(sums, out) && va_apart(sums, q);
}

static int va_check(const void* q, const void* k, const void* v, const void* out, int dtype, int out_dtype, int rows,
                    int n_heads, int n_kv, int head_dim, float scale, std::initializer_list<size_t> strides) {
  if (!q || !k || !v || !out) return T2B_ERR_ARG;
  if ((dtype != T2B_DTYPE_BF16 && dtype != T2B_DTYPE_F16) || (out_dtype != T2B_DTYPE_BF16 && out_dtype != T2B_DTYPE_F16))
    return T2B_ERR_ARG;
  if (!(scale > 0.f) || !isfinite(scale * 1.4426950408889634f)) return T2B_ERR_ARG;
  if (head_dim != 64 && head_dim != 128) return T2B_ERR_SHAPE;
  if (rows < 1 || rows > VA_MAX_KEYS || n_kv < 1 || n_heads < 1 || n_heads % n_kv || n_heads / n_kv > 128) return T2B_ERR_SHAPE;
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
  if (n_seqs < 1 || n_seqs > VA_MAX_KEYS || kv_tokens < 1 || kv_tokens > VA_MAX_KEYS || kv_seqs < 0) return T2B_ERR_SHAPE;
  if (kv_seqs ? (kv_seqs < n_seqs || !k_len || k_start) : (k_start == nullptr) != (k_len == nullptr)) return T2B_ERR_ARG;
  const size_t heads = n_heads, kv_heads = n_kv, rows = total_q, keys = kv_tokens, bytes = 2 * (size_t)head_dim;
  const size_t cache_rows = kv_seqs ? kv_seqs : 1;
  if (!va_results_apart(VaBox(out, bytes, {{rows, o_row}, {heads, o_head}}), lse, rows * heads,
                        VaBox(q, bytes, {{rows, q_row}, {heads, q_head}}),
                        (rows == 1 || q_row == o_row) && (heads == 1 || q_head == o_head),
                        {VaBox(k, bytes, {{cache_rows, k_seq}, {keys, k_tok}, {kv_heads, k_head}}),
                         VaBox(v, bytes, {{cache_rows, v_seq}, {keys, v_tok}, {kv_heads, v_head}})}))
    return T2B_ERR_ARG;
  VaParams P{};
  const bool f16 = dtype == T2B_DTYPE_F16;
  P.out = out, P.lse = lse, P.out_f16 = out_dtype == T2B_DTYPE_F16;
  P.rows = total_q, P.n_heads = n_heads, P.n_kv = n_kv, P.qpg = n_heads / n_kv, P.n_seqs = n_seqs;
  P.tpt = VA_ROWS / P.qpg;
  P.o_row = o_row, P.o_head = o_head;
  P.kv_tokens = kv_tokens, P.cached = kv_seqs > 0;
  const int max_blocks = va_host_blocks(kv_tokens);
  const double live = std::min(n_seqs, total_q);   // sequences with rows
  double units = va_most_units(total_q / (2 * P.tpt) + live, max_blocks, n_kv);
  if (!k_len) units = std::min(units, va_most_units_own(total_q, live, P.tpt, n_kv));
  const int sized = va_check_sizes(head_dim, units, workspace, workspace_bytes);
  if (sized != T2B_OK) return sized;
  if (!va_kv_map(&P.kmap, f16, k, head_dim, kv_tokens, n_kv, cache_rows, k_tok, k_head, k_seq) ||
      !va_kv_map(&P.vmap, f16, v, head_dim, kv_tokens, n_kv, cache_rows, v_tok, v_head, v_seq))
    return T2B_ERR_ARG;
  P.q_start = q_start, P.k_start = k_start, P.k_len = k_len;
  P.scale_log2 = scale * 1.4426950408889634f;
  return va_launch(P, head_dim, f16, q, q_row, q_head, units, max_blocks, workspace, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int t2b_tree_attention(const void* q, const void* k_cache, const void* v_cache, const void* k_draft,
                                  const void* v_draft, void* out, float* lse, int dtype, int out_dtype,
                                  const int32_t* ctx_len, const int32_t* n_nodes, const uint64_t* mask, int B, int T,
                                  int n_heads, int n_kv, int head_dim, int max_ctx, size_t q_row, size_t q_head,
                                  size_t o_row, size_t o_head, size_t kd_row, size_t kd_node, size_t kd_head,
                                  size_t vd_row, size_t vd_node, size_t vd_head, float scale, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  if (B < 1 || T < 1 || T > VA_MAX_NODES || max_ctx < 1 || max_ctx > VA_MAX_KEYS || (long long)B * T > VA_MAX_KEYS)
    return T2B_ERR_SHAPE;
  const int rc = va_check(q, k_cache, v_cache, out, dtype, out_dtype, B * T, n_heads, n_kv, head_dim, scale,
                          {q_row, q_head, o_row, o_head, kd_row, kd_node, kd_head, vd_row, vd_node, vd_head});
  if (rc != T2B_OK) return rc;
  if (!k_draft || !v_draft || !ctx_len || !mask) return T2B_ERR_ARG;
  if (va_misaligned(k_draft) || va_misaligned(v_draft) || (reinterpret_cast<uintptr_t>(mask) & 7)) return T2B_ERR_ALIGN;
  const size_t rows = (size_t)B * T, nodes = T, heads = n_heads, kv_heads = n_kv, batch = B, bytes = 2 * (size_t)head_dim;
  const long long cache = (long long)batch * kv_heads * max_ctx * bytes;
  if (!va_results_apart(VaBox(out, bytes, {{rows, o_row}, {heads, o_head}}), lse, rows * heads,
                        VaBox(q, bytes, {{rows, q_row}, {heads, q_head}}),
                        (rows == 1 || q_row == o_row) && (heads == 1 || q_head == o_head),
                        {VaBox(k_cache, cache), VaBox(v_cache, cache),
                         VaBox(k_draft, bytes, {{batch, kd_row}, {nodes, kd_node}, {kv_heads, kd_head}}),
                         VaBox(v_draft, bytes, {{batch, vd_row}, {nodes, vd_node}, {kv_heads, vd_head}})}))
    return T2B_ERR_ARG;
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
  const int max_blocks = va_host_blocks(max_ctx) + va_host_blocks(T);
  const double units = va_most_units((double)B * ((T + 2 * P.tpt - 1) / (2 * P.tpt)), max_blocks, n_kv);
  const int sized = va_check_sizes(head_dim, units, workspace, workspace_bytes);
  if (sized != T2B_OK) return sized;
  const size_t head = (size_t)max_ctx * head_dim;
  if (!va_kv_map(&P.kmap, f16, k_cache, head_dim, max_ctx, n_kv, B, head_dim, head, n_kv * head) ||
      !va_kv_map(&P.vmap, f16, v_cache, head_dim, max_ctx, n_kv, B, head_dim, head, n_kv * head) ||
      !va_kv_map(&P.kdmap, f16, k_draft, head_dim, T, n_kv, B, kd_node, kd_head, kd_row) ||
      !va_kv_map(&P.vdmap, f16, v_draft, head_dim, T, n_kv, B, vd_node, vd_head, vd_row))
    return T2B_ERR_ARG;
  return va_launch(P, head_dim, f16, q, q_row, q_head, units, max_blocks, workspace, reinterpret_cast<cudaStream_t>(stream));
}
