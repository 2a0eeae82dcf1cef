// Commit of a verified draft tree: the greedy walk through each row's tree and
// the move of the accepted nodes' K/V rows into the cache, all layers at once.
//
// Walk of row b: cur = 0 (the root, the last emitted token); the next node is
// the lowest n > cur with parents[n] == cur and tokens[n] == predicted[cur],
// predicted being the model's greedy token after each node; it ends where no
// such node exists, or where the cache is full.  The i-th accepted node's K/V
// row goes to cache position ctx_len[b] + i.
//
// Grid (row b, layer): every CTA repeats its row's walk (one warp, a ballot
// per 32 nodes of a level) and copies the accepted rows of its layer, so no
// CTA waits for another; the CTA of layer 0 writes the walk's results.  The
// copies are 16 bytes a thread, bounded by latency at the sizes of a decode
// step: replays of a graph take 4.0 us for 28 layers of one row and 7.5 us for 16
// layers of 64 rows of 48 nodes (19 MB moved, 2.5 TB/s), a call 21 to 25 us on
// the host.

#include <algorithm>
#include <new>
#include <utility>

#include "t2b_common.cuh"
#include "launch.cuh"

namespace t2b {

constexpr int TC_MAX_NODES = 256;
constexpr int TC_LAYERS = 64;    // layers per launch (their pointers are kernel parameters)
constexpr int TC_THREADS = 256;

struct TcParams {
  const int *tokens, *parents, *predicted, *ctx_len, *n_nodes;
  int *path, *n_accepted, *next_token, *new_len;
  int B, T, n_kv, max_ctx, row16;       // row16: 16-byte pieces of one head's row
  size_t kd_row, kd_node, kd_head, vd_row, vd_node, vd_head;   // 16-byte units
  int first;                            // this launch holds layer 0
  const uint4 *kd[TC_LAYERS], *vd[TC_LAYERS];
  uint4 *kc[TC_LAYERS], *vc[TC_LAYERS];
};

__global__ void __launch_bounds__(TC_THREADS) tree_commit_kernel(const __grid_constant__ TcParams P) {
  __shared__ int s_tok[TC_MAX_NODES], s_par[TC_MAX_NODES], s_pred[TC_MAX_NODES], s_path[TC_MAX_NODES];
  __shared__ int s_count;
  grid_dep_wait();
  grid_dep_launch();
  const int b = blockIdx.x, layer = blockIdx.y, tid = threadIdx.x;
  const int T = P.T, ctx = P.ctx_len[b];
  const int live = P.n_nodes ? min(P.n_nodes[b], T) : T;
  for (int i = tid; i < T; i += TC_THREADS) {
    s_tok[i] = P.tokens[(size_t)b * T + i];
    s_par[i] = P.parents[(size_t)b * T + i];
    s_pred[i] = P.predicted[(size_t)b * T + i];
  }
  __syncthreads();
  if (tid < 32) {
    int count = 0;
    if (live > 0 && ctx >= 0 && ctx < P.max_ctx) {
      int cur = 0;
      for (;;) {
        if (tid == 0) s_path[count] = cur;
        ++count;
        if (ctx + count >= P.max_ctx) break;
        const int want = s_pred[cur];
        int next = -1;
        for (int n0 = (cur + 1) & ~31; n0 < live && next < 0; n0 += 32) {
          const int n = n0 + tid;
          const bool fits = n > cur && n < live && s_par[n] == cur && s_tok[n] == want;
          const unsigned hit = __ballot_sync(0xffffffffu, fits);
          if (hit) next = n0 + __ffs(hit) - 1;
        }
        if (next < 0) break;
        cur = next;
      }
    }
    if (tid == 0) s_count = count;
  }
  __syncthreads();
  const int count = s_count;
  if (P.first && layer == 0) {
    for (int i = tid; i < T; i += TC_THREADS) P.path[(size_t)b * T + i] = i < count ? s_path[i] : -1;
    if (tid == 0) {
      P.n_accepted[b] = count;
      P.next_token[b] = count ? s_pred[s_path[count - 1]] : -1;
      P.new_len[b] = ctx + count;
    }
  }
  const uint4 *kd = P.kd[layer] + b * P.kd_row, *vd = P.vd[layer] + b * P.vd_row;
  const size_t c0 = (size_t)b * P.n_kv * P.max_ctx;
  const int row16 = P.row16, per_head = count * row16, total = per_head * P.n_kv;
  for (int e = tid; e < total; e += TC_THREADS) {
    const int h = e / per_head, rest = e - h * per_head, i = rest / row16, c = rest - i * row16;
    const size_t dst = (c0 + (size_t)h * P.max_ctx + ctx + i) * row16 + c;
    const int n = s_path[i];
    const uint4 kv = kd[n * P.kd_node + h * P.kd_head + c];
    const uint4 vv = vd[n * P.vd_node + h * P.vd_head + c];
    P.kc[layer][dst] = kv;
    P.vc[layer][dst] = vv;
  }
}

// Memory that a call reads or writes.
struct TcSpan {
  uintptr_t lo, hi;
  bool write;
};
// No write meets another span.  Tensors of all layers mostly lie in order, so
// sorting them costs little (28 layers: 120 spans).
static bool tc_apart(TcSpan* s, size_t n) {
  std::sort(s, s + n, [](const TcSpan& a, const TcSpan& b) { return a.lo < b.lo; });
  uintptr_t read = 0, written = 0;   // ends so far
  for (size_t i = 0; i < n; ++i) {
    if (s[i].lo < written || (s[i].write && s[i].lo < read)) return false;
    uintptr_t& end = s[i].write ? written : read;
    end = std::max(end, s[i].hi);
  }
  return true;
}

}  // namespace t2b

using namespace t2b;

extern "C" int t2b_tree_commit(const int32_t* tokens, const int32_t* parents, const int32_t* predicted,
                               const int32_t* ctx_len, const int32_t* n_nodes, const void* const* k_draft,
                               const void* const* v_draft, void* const* k_cache, void* const* v_cache, int n_layers,
                               int32_t* path, int32_t* n_accepted, int32_t* next_token, int32_t* new_len, int B,
                               int T, int n_kv, int head_dim, int max_ctx, size_t kd_row, size_t kd_node,
                               size_t kd_head, size_t vd_row, size_t vd_node, size_t vd_head, void* stream) {
  if (!tokens || !parents || !predicted || !ctx_len || !path || !n_accepted || !next_token || !new_len) return T2B_ERR_ARG;
  if (!k_draft || !v_draft || !k_cache || !v_cache) return T2B_ERR_ARG;
  if (B < 1 || T < 1 || T > TC_MAX_NODES || n_layers < 1 || n_kv < 1 || max_ctx < 1) return T2B_ERR_SHAPE;
  if (head_dim < 8 || head_dim % 8 || head_dim > 1024 || n_kv > 1024) return T2B_ERR_SHAPE;
  for (size_t s : {kd_row, kd_node, kd_head, vd_row, vd_node, vd_head})
    if (s % 8) return T2B_ERR_ALIGN;
  for (int l = 0; l < n_layers; ++l)
    for (const void* p : {k_draft[l], v_draft[l], (const void*)k_cache[l], (const void*)v_cache[l]}) {
      if (!p) return T2B_ERR_ARG;
      if (reinterpret_cast<uintptr_t>(p) & 15) return T2B_ERR_ALIGN;
    }
  // Every CTA reads a row's inputs while one writes its results, and the layers
  // are copied at once: what is written must be apart from all the rest.
  const size_t tree = (size_t)B * T, rows = B;
  const std::pair<const int32_t*, size_t> words[] = {{tokens, tree}, {parents, tree}, {predicted, tree}, {ctx_len, rows},
                                                     {n_nodes, n_nodes ? rows : 0}, {path, tree}, {n_accepted, rows},
                                                     {next_token, rows}, {new_len, rows}};
  const size_t cache = 2 * rows * n_kv * max_ctx * head_dim;
  const size_t kd = 2 * ((B - 1) * kd_row + (T - 1) * kd_node + (n_kv - 1) * kd_head + head_dim);
  const size_t vd = 2 * ((B - 1) * vd_row + (T - 1) * vd_node + (n_kv - 1) * vd_head + head_dim);
  TcSpan* span = new (std::nothrow) TcSpan[9 + 4 * (size_t)n_layers];
  if (!span) return T2B_ERR_LAUNCH;
  size_t n_spans = 0;
  auto add = [&](const void* p, size_t bytes, bool write) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(p);
    if (bytes) span[n_spans++] = {at, at + bytes, write};
  };
  for (int i = 0; i < 9; ++i) add(words[i].first, words[i].second * sizeof(int32_t), i >= 5);
  for (int l = 0; l < n_layers; ++l) add(k_draft[l], kd, false);
  for (int l = 0; l < n_layers; ++l) add(v_draft[l], vd, false);
  for (int l = 0; l < n_layers; ++l) add(k_cache[l], cache, true);
  for (int l = 0; l < n_layers; ++l) add(v_cache[l], cache, true);
  const bool apart = tc_apart(span, n_spans);
  delete[] span;
  if (!apart) return T2B_ERR_ARG;
  TcParams P{};
  P.tokens = tokens, P.parents = parents, P.predicted = predicted, P.ctx_len = ctx_len, P.n_nodes = n_nodes;
  P.path = path, P.n_accepted = n_accepted, P.next_token = next_token, P.new_len = new_len;
  P.B = B, P.T = T, P.n_kv = n_kv, P.max_ctx = max_ctx, P.row16 = head_dim / 8;
  P.kd_row = kd_row / 8, P.kd_node = kd_node / 8, P.kd_head = kd_head / 8;
  P.vd_row = vd_row / 8, P.vd_node = vd_node / 8, P.vd_head = vd_head / 8;
  for (int l0 = 0; l0 < n_layers; l0 += TC_LAYERS) {
    const int n = n_layers - l0 < TC_LAYERS ? n_layers - l0 : TC_LAYERS;
    for (int l = 0; l < n; ++l) {
      P.kd[l] = static_cast<const uint4*>(k_draft[l0 + l]);
      P.vd[l] = static_cast<const uint4*>(v_draft[l0 + l]);
      P.kc[l] = static_cast<uint4*>(k_cache[l0 + l]);
      P.vc[l] = static_cast<uint4*>(v_cache[l0 + l]);
    }
    P.first = l0 == 0;
    const int rc = launch_pdl(tree_commit_kernel, dim3(B, n), dim3(TC_THREADS), 0, reinterpret_cast<cudaStream_t>(stream), P);
    if (rc != T2B_OK) return rc;
  }
  return T2B_OK;
}
