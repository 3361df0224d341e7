// k_tattn.hip - attention of several new tokens a request over a paged key-value cache, with
// a mask among the new ones (qllama_tree_attention; semantics in qserve.h).  No
// counterpart in the reference, whose decode attention (llama.c:554-576) serves one token.
#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include "qserve_host.h"

namespace {

constexpr float kNegInf = -__builtin_inff();

template <int T>
__device__ inline float element(const void *p, long long at) {
  if constexpr (T == QLLAMA_KV_F32) return static_cast<const float *>(p)[at];
  else if constexpr (T == QLLAMA_KV_F16) return __half2float(static_cast<const __half *>(p)[at]);
  else if constexpr (T == QLLAMA_KV_BF16) return __uint_as_float((uint32_t)static_cast<const unsigned short *>(p)[at] << 16);
  else return (float)static_cast<const signed char *>(p)[at];
}

// A block of four waves a (request, query head), row by row; a wave every fourth token, a
// lane every 64th dim, with the running maximum and sum of a softmax.
template <int T>
__global__ __launch_bounds__(256) void k_tree_attn(QPagedKV c, QTreeQuery a, float scale) {
  __shared__ float part[4][258];
  const int h = blockIdx.x, r = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int kvh = h / (a.n_heads / c.n_kv);
  const int first = min(max(a.starts[r], 0), a.rows), m = max(min(max(a.starts[r + 1], 0), a.rows) - first, 0);
  const int len = min(max(a.lens[r], 0), a.width * c.page_size), ctx = max(len - m, 0);
  for (int j = 0; j < m; j++) {
    const int i = first + j;
    float q[4], o[4] = {0, 0, 0, 0}, top = kNegInf, sum = 0.0f;
    for (int x = 0; x < 4; x++) q[x] = lane + 64 * x < c.head_dim ? a.q[i * a.q_stride + (long long)h * c.head_dim + lane + 64 * x] * scale : 0.0f;
    for (int t = wave; t < len; t += 4) {
      const int b = t - ctx;
      if (b >= 0 && !(a.mask ? b < 64 * a.words && (a.mask[(long long)i * a.words + (b >> 6)] >> (b & 63) & 1) : b <= j)) continue;
      const int page = a.table[r * a.table_stride + t / c.page_size], place = t % c.page_size;
      if (page < 0 || page >= c.n_pages) continue;
      const long long at = page * c.page_stride + kvh * c.head_stride + place * c.slot_stride;
      const long long sat = T == QLLAMA_KV_I8 ? page * c.scale_page_stride + kvh * c.scale_head_stride + place * c.scale_slot_stride : 0;
      float s = 0.0f;
      for (int x = 0; x < 4; x++)
        if (lane + 64 * x < c.head_dim) s += q[x] * element<T>(c.k, at + lane + 64 * x);
      for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d);
      if constexpr (T == QLLAMA_KV_I8) s *= c.k_scale[sat];
      const float up = fmaxf(top, s), by = top == kNegInf ? 0.0f : __expf(top - up), w = s == kNegInf ? 0.0f : __expf(s - up);
      sum = sum * by + w;
      const float v = T == QLLAMA_KV_I8 ? w * c.v_scale[sat] : w;
      for (int x = 0; x < 4; x++)
        if (lane + 64 * x < c.head_dim) o[x] = o[x] * by + v * element<T>(c.v, at + lane + 64 * x);
      top = up;
    }
    __syncthreads();
    for (int x = 0; x < 4; x++) part[wave][lane + 64 * x] = o[x];
    if (lane == 0) { part[wave][256] = top; part[wave][257] = sum; }
    __syncthreads();
    float most = kNegInf, all = 0.0f, y = 0.0f;
    for (int w = 0; w < 4; w++) most = fmaxf(most, part[w][256]);
    for (int w = 0; w < 4; w++) {
      const float by = part[w][256] == kNegInf ? 0.0f : __expf(part[w][256] - most);
      all += part[w][257] * by;
      y += part[w][threadIdx.x] * by;
    }
    if ((int)threadIdx.x < c.head_dim) a.o[i * a.o_stride + (long long)h * c.head_dim + threadIdx.x] = all == 0.0f ? 0.0f : y / all;
    if (threadIdx.x == 0 && a.lse) a.lse[i * a.lse_stride + h] = all == 0.0f ? kNegInf : most + __logf(all);
    __syncthreads();
  }
}

}  // namespace

extern "C" size_t qllama_tree_attention_work(const QPagedKV *c, int rows, int n_req, int n_heads, int nodes) {
  if (qs::bad_cache(c) || rows < 0 || n_req < 0 || n_heads < 1 || n_heads > 65535 || n_heads % c->n_kv || nodes < 0) return 0;
  return 16;
}

extern "C" int qllama_tree_attention(const QPagedKV *c, const QTreeQuery *a, void *stream) {
  static const char fn[] = "qllama_tree_attention";
  if (const char *why = qs::bad_cache(c)) return qs::refuse(fn, why);
  if (!a || a->n_req < 0 || a->rows < 0 || a->rows > (1 << 23) || a->nodes < 0) return qs::refuse(fn, "null argument, n_req or nodes < 0, or rows not 0 .. 2^23");
  if (a->n_heads < 1 || a->n_heads > 65535 || a->n_heads % c->n_kv) return qs::refuse(fn, "n_heads must be a multiple of the cache's KV heads");
  if (a->n_req == 0 || a->rows == 0) return 0;
  if (!a->q || !a->o || !a->table || !a->lens || !a->starts) return qs::refuse(fn, "null q, o, table, lens or starts");
  if (a->mask ? a->words < 1 || a->words > 4 : a->words != 0) return qs::refuse(fn, "a mask has 1 .. 4 words a row, no mask has 0");
  const int64_t qd = (int64_t)a->n_heads * c->head_dim;
  if (a->q_stride < qd || a->o_stride < qd || (a->lse && a->lse_stride < a->n_heads)) return qs::refuse(fn, "a row stride below the row's length");
  if (a->width < 1 || a->table_stride < a->width || (int64_t)a->width * c->page_size > INT_MAX - 1024)   // a step past it still fits
    return qs::refuse(fn, "bad table width (width * page_size must be below 2^31 - 1024) or stride");
  if (!(a->scale >= 0.0f) || a->scale > 2.35e38f)      // times log2 e within a float's range
    return qs::refuse(fn, "scale must be 0 .. 2.35e38");
  if (a->q == a->o) return qs::refuse(fn, "o must not be q");
  if (qs::misaligned(a->q, 4) || qs::misaligned(a->o, 4) || qs::misaligned(a->lse, 4) || qs::misaligned(a->table, 4) || qs::misaligned(a->lens, 4) ||
      qs::misaligned(a->starts, 4) || qs::misaligned(a->mask, 8))
    return qs::refuse(fn, "a buffer is not aligned to its elements");
  if (!a->work || qs::misaligned(a->work, 16) || a->work_bytes < qllama_tree_attention_work(c, a->rows, a->n_req, a->n_heads, a->nodes))
    return qs::refuse(fn, "work is missing, misaligned or smaller than qllama_tree_attention_work");
  qs::OnDevice on(c->k, (hipStream_t)stream);
  if (on.why) return qs::refuse(fn, on.why);
  const float scale = a->scale > 0.0f ? a->scale : 1.0f / __builtin_sqrtf((float)c->head_dim);
  const dim3 grid(a->n_heads, a->n_req);
  void (*f)(QPagedKV, QTreeQuery, float) = c->type == QLLAMA_KV_F32 ? k_tree_attn<QLLAMA_KV_F32> : c->type == QLLAMA_KV_F16 ? k_tree_attn<QLLAMA_KV_F16>
                                         : c->type == QLLAMA_KV_BF16 ? k_tree_attn<QLLAMA_KV_BF16> : k_tree_attn<QLLAMA_KV_I8>;
  QS_LAUNCH(fn, f, grid, dim3(256), 0, (hipStream_t)stream, *c, *a, scale);
  return 0;
}
