// k_tree.hip - drafted trees: what every row may attend to, and what the chosen tokens
// confirm (qllama_tree_plan, qllama_tree_accept; semantics in qserve.h).  No counterpart
// in the reference, which decodes one token at a time (llama.c:528-600).
#include <hip/hip_runtime.h>

#include "qserve_host.h"

namespace {

constexpr int kMaxNodes = 1024;

// First row of a request, and its number of rows.
__device__ inline int tree_rows(const int *starts, int r, int max_rows, int *first) {
  const int a = min(max(starts[r], 0), max_rows), b = min(max(starts[r + 1], 0), max_rows);
  *first = a;
  return max(b - a, 0);
}

// A block a request, a thread a row: each row starts with its own bit and its parent, and in
// round k takes over the bits of the row 2^k above it and that row's own way up, so that a
// tree of depth d takes log2 d rounds.  A launch and a chain of trips to memory, not bytes: 2.7
// us for 4 requests of 8 rows, 3.5 for 200 of 64.
__global__ void k_tree_plan(QTreePlan p) {
  __shared__ uint64_t bits[2][4][256];
  __shared__ int up[2][256];
  const int r = blockIdx.x, t = threadIdx.x, W = p.words, N = 64 * W;
  int first;
  const int m = tree_rows(p.starts, r, p.max_rows, &first);
  const int ctx = p.lens[r] - m;
  int above = -1;
  if (t < m && t < p.nodes) {
    above = p.parents[r * p.parent_stride + t];
    if (above >= t) above = -1;
  }
  uint64_t mine[4];
  for (int w = 0; w < W; w++) mine[w] = w == t >> 6 ? 1ull << (t & 63) : 0;
  int at = 0;
  while (__syncthreads_or(above >= 0)) {
    for (int w = 0; w < W; w++) bits[at][w][t] = mine[w];
    up[at][t] = above;
    __syncthreads();
    if (above >= 0) {
      for (int w = 0; w < W; w++) mine[w] |= bits[at][w][above];
      above = up[at][above];
    }
    at ^= 1;
  }
  if (t < m) {
    int depth = -1;
    for (int w = 0; w < W; w++) {
      p.mask[(int64_t)(first + t) * W + w] = mine[w];
      depth += __popcll(mine[w]);
    }
    p.positions[first + t] = ctx + depth;
  }
  for (int j = N + t; j < m; j += N) {
    for (int w = 0; w < W; w++) p.mask[(int64_t)(first + j) * W + w] = 0;
    p.positions[first + j] = ctx + j;
  }
}

// A wave a request.  Its rows' parents, tokens and choices lie in LDS; a step down looks at
// 64 rows at a time: 2.8 us for 4 requests of 8 rows, 3.9 for 200 of 64.
__global__ __launch_bounds__(64) void k_tree_accept(QTreeAccept p) {
  __shared__ int parent[kMaxNodes], token[kMaxNodes], choice[kMaxNodes], path[kMaxNodes];
  const int r = blockIdx.x, lane = threadIdx.x;
  int first;
  const int m = tree_rows(p.starts, r, p.max_rows, &first);
  const int n = min(m, p.nodes);                      // rows that can have a parent
  for (int j = lane; j < n; j += 64) {
    parent[j] = p.parents[r * p.parent_stride + j];
    token[j] = p.tokens[first + j];
    choice[j] = p.chosen[first + j];
  }
  __syncthreads();
  int count = 0, last = -1;
  for (int at = m > 0 ? 0 : -1; at >= 0;) {
    if (lane == 0) path[count] = at;
    count++;
    last = choice[at];
    int next = -1;
    for (int c0 = at + 1; c0 < n && next < 0 && last >= 0; c0 += 64) {
      const int c = c0 + lane;
      const uint64_t fits = __ballot(c < n && parent[c] == at && token[c] == last);
      if (fits) next = c0 + __builtin_ctzll(fits);
    }
    at = next;
  }
  __syncthreads();
  if (lane == 0) {
    p.accepted[r] = count;
    p.last[r] = last;
    p.lens_out[r] = p.lens[r] - m + count;
  }
  for (int k = lane; k < m; k += 64) {
    const int row = k < count ? path[k] : -1;
    const bool moved = row >= 0 && row != k;
    p.path[first + k] = row >= 0 ? first + row : -1;
    p.src[first + k] = moved ? p.slots[first + row] : -1;
    p.dst[first + k] = moved ? p.slots[first + k] : -1;
  }
}

}  // namespace

extern "C" int qllama_tree_plan(const QTreePlan *p, void *stream) {
  static const char fn[] = "qllama_tree_plan";
  if (!p) return qs::refuse(fn, "null argument");
  if (p->n_req < 0 || p->n_req > 8192) return qs::refuse(fn, "n_req must be 0 .. 8192");
  if (p->nodes < 1 || p->nodes > kMaxNodes || p->parent_stride < p->nodes) return qs::refuse(fn, "nodes must be 1 .. 1024, parent_stride at least nodes");
  if (p->words < 1 || p->words > 4 || p->max_rows < 0 || p->max_rows > (1 << 30)) return qs::refuse(fn, "words must be 1 .. 4, max_rows 0 .. 2^30");
  if (p->n_req == 0) return 0;
  if (!p->starts || !p->lens || !p->parents || (p->max_rows && (!p->positions || !p->mask))) return qs::refuse(fn, "null buffer");
  if (qs::misaligned(p->starts, 4) || qs::misaligned(p->lens, 4) || qs::misaligned(p->parents, 4) || qs::misaligned(p->positions, 4) ||
      qs::misaligned(p->mask, 8))
    return qs::refuse(fn, "a buffer is not aligned to its elements");
  qs::OnDevice on(p->starts, (hipStream_t)stream);
  if (on.why) return qs::refuse(fn, on.why);
  QS_LAUNCH(fn, k_tree_plan, dim3(p->n_req), dim3(64 * p->words), 0, (hipStream_t)stream, *p);
  return 0;
}

extern "C" int qllama_tree_accept(const QTreeAccept *p, void *stream) {
  static const char fn[] = "qllama_tree_accept";
  if (!p) return qs::refuse(fn, "null argument");
  if (p->n_req < 0 || p->n_req > 8192) return qs::refuse(fn, "n_req must be 0 .. 8192");
  if (p->nodes < 1 || p->nodes > kMaxNodes || p->parent_stride < p->nodes) return qs::refuse(fn, "nodes must be 1 .. 1024, parent_stride at least nodes");
  if (p->max_rows < 0 || p->max_rows > (1 << 30)) return qs::refuse(fn, "max_rows must be 0 .. 2^30");
  if (p->n_req == 0) return 0;
  const void *all[] = {p->starts, p->lens, p->parents, p->accepted, p->last, p->lens_out};
  const void *rows[] = {p->tokens, p->chosen, p->slots, p->path, p->src, p->dst};
  for (const void *x : all)
    if (!x) return qs::refuse(fn, "null buffer");
  for (const void *x : rows)
    if (p->max_rows && !x) return qs::refuse(fn, "null buffer");
  for (const void *x : all)
    if (qs::misaligned(x, 4)) return qs::refuse(fn, "a buffer is not aligned to its elements");
  for (const void *x : rows)
    if (qs::misaligned(x, 4)) return qs::refuse(fn, "a buffer is not aligned to its elements");
  const int32_t *out[] = {p->path, p->src, p->dst}, *in[] = {p->tokens, p->chosen, p->slots};
  for (const int32_t *x : out)
    for (const int32_t *y : in)
      if (p->max_rows && x == y) return qs::refuse(fn, "an output is one of the inputs");
  qs::OnDevice on(p->starts, (hipStream_t)stream);
  if (on.why) return qs::refuse(fn, on.why);
  QS_LAUNCH(fn, k_tree_accept, dim3(p->n_req), dim3(64), 0, (hipStream_t)stream, *p);
  return 0;
}
