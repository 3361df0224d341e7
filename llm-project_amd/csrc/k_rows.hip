// k_rows.hip - a token from every row of logits (qllama_sample_rows; semantics in
// qserve.h): sample_token (sampler.c:54-143) for many rows with settings and random
// numbers of their own, and min-p.
//
// No row is sorted.  A token's weight e = exp((l - max) / T) is held as a whole number
// of 2^-43 in 64 bits, so sums are exact in any order and LDS atomics give the same
// bits every time; a histogram over log2 e with the number and the weight of the tokens
// in each bin tells in which bin the kept set ends, and in which the drawn token lies;
// only that bin's tokens are put in order.  A bin that holds too many of them (equal or
// nearly equal logits) is divided by the bits of (logit, index) until few are left.
#include <hip/hip_runtime.h>

#include "qserve_host.h"

namespace {

constexpr int kThreads = 1024;
constexpr int kBins = 2048;
constexpr int kList = 2048;           // tokens of a bin that are put in order at once
constexpr double kUnit = 8796093022208.0;   // 2^43
constexpr double kLog2e = 1.4426950408889634074;

typedef unsigned long long u64;

// A logit and its index as one number, larger for earlier in the order; 0: masked.
__device__ inline u64 token_key(float l, int i) {
  if (!(l > -__builtin_inff())) return 0;               // -inf and NaN
  const uint32_t b = __float_as_uint(l + 0.0f);         // -0 as 0
  const uint32_t o = b & 0x80000000u ? ~b : b | 0x80000000u;
  return (u64)o << 32 | (0xffffffffu - (uint32_t)i);
}
__device__ inline float key_logit(u64 k) {
  const uint32_t o = (uint32_t)(k >> 32);
  return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ inline int key_index(u64 k) { return (int)(0xffffffffu - (uint32_t)k); }

// -log2 of a token's weight
__device__ inline double depth(float l, float top, double per) { return l == top ? 0.0 : ((double)top - (double)l) * per; }

// 2^-t, 0 <= t: the nearest power of two times the Taylor series of the rest (|r| <=
// 0.35, its 13th term 2e-16); 0 past t = 64
__device__ inline double weight(double t) {
  if (!(t <= 64.0)) return 0.0;
  const double k = rint(t), r = (k - t) * 0.69314718055994530942;
  double s = 1.0 / 479001600.0;
  s = fma(s, r, 1.0 / 39916800.0);
  s = fma(s, r, 1.0 / 3628800.0);
  s = fma(s, r, 1.0 / 362880.0);
  s = fma(s, r, 1.0 / 40320.0);
  s = fma(s, r, 1.0 / 5040.0);
  s = fma(s, r, 1.0 / 720.0);
  s = fma(s, r, 1.0 / 120.0);
  s = fma(s, r, 1.0 / 24.0);
  s = fma(s, r, 1.0 / 6.0);
  s = fma(s, r, 0.5);
  s = fma(s, r, 1.0);
  s = fma(s, r, 1.0);
  return ldexp(s, -(int)k);
}
__device__ inline u64 units(double t) { return (u64)(weight(t) * kUnit + 0.5); }

// bins of equal width in log2; tokens without weight in the last
__device__ inline int bin_of(double t) { return t < 44.5 ? (int)(t * 46.0) : kBins - 1; }

struct Mass { u64 w; uint32_t n; };

struct Shared {
  u64 w[kBins];
  uint32_t n[kBins];
  u64 list[kList];
  u64 part_w[kThreads / 64];
  uint32_t part_n[kThreads / 64];
  uint32_t fill;
  int found;
};

// Inclusive sums over the block's threads.
__device__ Mass scan(Mass v, Shared &s) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int d = 1; d < 64; d <<= 1) {
    const u64 w = __shfl_up(v.w, d);
    const uint32_t n = __shfl_up(v.n, d);
    if (lane >= d) { v.w += w; v.n += n; }
  }
  __syncthreads();
  if (lane == 63) { s.part_w[wave] = v.w; s.part_n[wave] = v.n; }
  __syncthreads();
  for (int i = 0; i < wave; i++) { v.w += s.part_w[i]; v.n += s.part_n[i]; }
  return v;
}

__device__ void clear(Shared &s) {
  __syncthreads();
  for (int b = threadIdx.x; b < kBins; b += kThreads) { s.w[b] = 0; s.n[b] = 0; }
  __syncthreads();
}

// w and n become inclusive sums from bin 0 on.
__device__ void accumulate(Shared &s) {
  __syncthreads();
  const int b = 2 * threadIdx.x;
  const u64 w0 = s.w[b], w1 = s.w[b + 1];
  const uint32_t n0 = s.n[b], n1 = s.n[b + 1];
  const Mass v = scan({w0 + w1, n0 + n1}, s);
  s.w[b] = v.w - w1; s.w[b + 1] = v.w;
  s.n[b] = v.n - n1; s.n[b + 1] = v.n;
  __syncthreads();
}

// The first bin (sums accumulated, on top of `before`) where n tokens or the weight are
// reached; the last one that holds a token where they never are.
__device__ int find_bin(Shared &s, Mass before, uint32_t n, double w) {
  if (threadIdx.x == 0) s.found = kBins;
  __syncthreads();
  const uint32_t all = s.n[kBins - 1];
  int at = kBins;
  for (int b = 2 * threadIdx.x + 1; b >= 2 * (int)threadIdx.x; b--)
    if (s.n[b] && (before.n + s.n[b] >= n || (double)(before.w + s.w[b]) >= w || s.n[b] == all)) at = b;
  if (at < kBins) atomicMin(&s.found, at);
  __syncthreads();
  return s.found;
}

struct Row {
  const float *l;
  int V;
  float top;
  double per;                   // log2(e) / T
};

struct Found { Mass upto; u64 key; };   // number and weight up to and with a token, and the token

// The token at which, in order, n tokens or the weight are reached first.  s.w and s.n
// hold the accumulated first histogram; they are changed.
__device__ Found locate(const Row &row, Shared &s, uint32_t n, double w) {
  Mass before = {0, 0};
  const int bin = find_bin(s, before, n, w);
  uint32_t inside = s.n[bin] - (bin ? s.n[bin - 1] : 0);
  if (bin) before = {s.w[bin - 1], s.n[bin - 1]};
  u64 prefix = 0;
  int shift = 64;               // of the bits that are settled
  while (inside > kList) {
    const int next = shift > 11 ? shift - 11 : 0;
    clear(s);
    for (int i = threadIdx.x; i < row.V; i += kThreads) {
      const float l = row.l[i];
      const u64 k = token_key(l, i);
      if (!k) continue;
      const double t = depth(l, row.top, row.per);
      if (bin_of(t) != bin || (shift < 64 && k >> shift != prefix)) continue;
      const int d = kBins - 1 - (int)((k >> next) & (kBins - 1));
      atomicAdd(&s.w[d], units(t));
      atomicAdd(&s.n[d], 1u);
    }
    accumulate(s);
    const int d = find_bin(s, before, n, w);
    inside = s.n[d] - (d ? s.n[d - 1] : 0);
    if (d) { before.w += s.w[d - 1]; before.n += s.n[d - 1]; }
    prefix = (shift < 64 ? prefix << (shift - next) : 0) | (u64)(kBins - 1 - d);   // the last digit repeats settled bits
    shift = next;
  }

  __syncthreads();
  if (threadIdx.x == 0) s.fill = 0;
  int pow2 = 64;
  while (pow2 < (int)inside) pow2 <<= 1;
  for (int i = threadIdx.x; i < pow2; i += kThreads) s.list[i] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < row.V; i += kThreads) {
    const float l = row.l[i];
    const u64 k = token_key(l, i);
    if (!k || bin_of(depth(l, row.top, row.per)) != bin || (shift < 64 && k >> shift != prefix)) continue;
    s.list[atomicAdd(&s.fill, 1u)] = k;
  }
  for (int size = 2; size <= pow2; size <<= 1)
    for (int d = size >> 1; d; d >>= 1) {
      __syncthreads();
      for (int i = threadIdx.x; i < pow2 / 2; i += kThreads) {
        const int a = 2 * i - (i & (d - 1)), b = a + d;
        const u64 x = s.list[a], y = s.list[b];
        if ((x < y) == ((a & size) == 0)) { s.list[a] = y; s.list[b] = x; }
      }
    }
  __syncthreads();

  const int i0 = 2 * threadIdx.x;
  u64 k[2], m[2];
  for (int i = 0; i < 2; i++) {
    k[i] = i0 + i < pow2 ? s.list[i0 + i] : 0;
    m[i] = k[i] ? units(depth(key_logit(k[i]), row.top, row.per)) : 0;
  }
  const Mass v = scan({m[0] + m[1], (uint32_t)(k[0] != 0) + (k[1] != 0)}, s);
  if (threadIdx.x == 0) s.found = kList;
  __syncthreads();
  for (int i = 1; i >= 0; i--) {
    const Mass u = {before.w + v.w - (i ? 0 : m[1]), before.n + v.n - (i ? 0 : k[1] != 0)};
    if (k[i] && (u.n >= n || (double)u.w >= w || u.n == before.n + inside)) atomicMin(&s.found, i0 + i);
  }
  __syncthreads();
  const int at = s.found;
  if (i0 <= at && at < i0 + 2) {                  // its thread tells the others
    const int i = at - i0;
    s.part_w[0] = before.w + v.w - (i ? 0 : m[1]);
    s.part_n[0] = before.n + v.n - (i ? 0 : k[1] != 0);
  }
  __syncthreads();
  const Found f = {{s.part_w[0], s.part_n[0]}, s.list[at]};
  __syncthreads();
  return f;
}

__global__ __launch_bounds__(kThreads) void k_sample_rows(QSampleRows a) {
  __shared__ Shared s;
  const int r = blockIdx.x;
  Row row = {a.logits + r * a.stride, a.vocab, 0.0f, 0.0};
  const float T = a.temperature ? a.temperature[r] : 1.0f;
  const bool greedy = !(T > 0.0f);

  u64 best = 0;
  for (int i = threadIdx.x; i < row.V; i += kThreads) {
    const u64 k = token_key(row.l[i], i);
    best = k > best ? k : best;
  }
  for (int d = 32; d; d >>= 1) {
    const u64 o = __shfl_xor(best, d);
    best = o > best ? o : best;
  }
  if ((threadIdx.x & 63) == 0) s.part_w[threadIdx.x >> 6] = best;
  __syncthreads();
  for (int i = 0; i < kThreads / 64; i++) best = s.part_w[i] > best ? s.part_w[i] : best;
  if (!best || greedy) {
    if (threadIdx.x == 0) {
      a.token[r] = best ? key_index(best) : -1;
      if (a.prob) a.prob[r] = best ? 1.0f : 0.0f;
      if (a.kept) a.kept[r] = best ? 1 : 0;
    }
    return;
  }
  row.top = key_logit(best);
  row.per = kLog2e / (double)T;

  // min-p limits the number of tokens: e >= min_p, that is depth <= -log2(min_p)
  float mp = a.min_p ? a.min_p[r] : 0.0f;
  const bool by_min = mp > 0.0f;
  if (mp > 1.0f) mp = 1.0f;
  clear(s);
  uint32_t passing = 0;
  for (int i = threadIdx.x; i < row.V; i += kThreads) {
    const float l = row.l[i];
    if (!(l > -__builtin_inff())) continue;
    const double t = depth(l, row.top, row.per), e = weight(t);
    const int b = bin_of(t);
    const u64 w = (u64)(e * kUnit + 0.5);
    if (w) atomicAdd(&s.w[b], w);
    atomicAdd(&s.n[b], 1u);
    passing += by_min && e >= (double)mp;
  }
  accumulate(s);
  const u64 all_w = s.w[kBins - 1];
  const uint32_t all_n = s.n[kBins - 1];
  if (by_min) {
    for (int d = 32; d; d >>= 1) passing += __shfl_xor(passing, d);
    if ((threadIdx.x & 63) == 0) s.part_n[threadIdx.x >> 6] = passing;
    __syncthreads();
    passing = 0;
    for (int i = 0; i < kThreads / 64; i++) passing += s.part_n[i];
  }
  const int k = a.top_k ? a.top_k[r] : 0;
  const float p = a.top_p ? a.top_p[r] : 0.0f;
  uint32_t n = all_n;
  if (k > 0 && (uint32_t)k < n) n = k;
  if (by_min && passing < n) n = passing;
  if (n < 1) n = 1;
  const bool by_mass = p > 0.0f && p < 1.0f;

  // the histogram is used twice: kept aside in registers while the first search changes it
  const u64 w0 = s.w[2 * threadIdx.x], w1 = s.w[2 * threadIdx.x + 1];
  const uint32_t n0 = s.n[2 * threadIdx.x], n1 = s.n[2 * threadIdx.x + 1];
  Mass kept = {all_w, all_n};
  if (n < all_n || by_mass) {
    kept = locate(row, s, n, by_mass ? (double)p * (double)all_w : __builtin_inf()).upto;
    s.w[2 * threadIdx.x] = w0; s.w[2 * threadIdx.x + 1] = w1;
    s.n[2 * threadIdx.x] = n0; s.n[2 * threadIdx.x + 1] = n1;
    __syncthreads();
  }
  float u = a.u[r];
  u = u > 0.0f ? (u < 1.0f ? u : 0x1.fffffep-1f) : 0.0f;
  const Found f = locate(row, s, kept.n, (double)u * (double)kept.w);
  if (threadIdx.x == 0) {
    a.token[r] = key_index(f.key);
    if (a.prob) a.prob[r] = (float)(weight(depth(key_logit(f.key), row.top, row.per)) * kUnit / (double)kept.w);
    if (a.kept) a.kept[r] = (int)kept.n;
  }
}

}  // namespace

extern "C" size_t qllama_sample_rows_work(int rows, int vocab) {
  if (rows < 0 || vocab < 1 || vocab > (1 << 20)) return 0;
  return 16;
}

extern "C" int qllama_sample_rows(const QSampleRows *s, void *stream) {
  static const char fn[] = "qllama_sample_rows";
  if (!s || s->rows < 0) return qs::refuse(fn, "null argument or rows < 0");
  if (s->vocab < 1 || s->vocab > (1 << 20) || s->stride < s->vocab) return qs::refuse(fn, "vocab must be 1 .. 1048576, stride at least vocab");
  if (s->rows == 0) return 0;
  if (!s->logits || !s->u || !s->token) return qs::refuse(fn, "null logits, u or token");
  if (qs::misaligned(s->logits, 4) || qs::misaligned(s->u, 4) || qs::misaligned(s->token, 4) || qs::misaligned(s->kept, 4) || qs::misaligned(s->prob, 4) ||
      qs::misaligned(s->temperature, 4) || qs::misaligned(s->top_k, 4) || qs::misaligned(s->top_p, 4) || qs::misaligned(s->min_p, 4))
    return qs::refuse(fn, "a buffer is not aligned to its elements");
  if (!s->work || qs::misaligned(s->work, 16) || s->work_bytes < qllama_sample_rows_work(s->rows, s->vocab))
    return qs::refuse(fn, "work is missing, misaligned or smaller than qllama_sample_rows_work");
  qs::OnDevice on(s->logits, (hipStream_t)stream);
  if (on.why) return qs::refuse(fn, on.why);
  QS_LAUNCH(fn, k_sample_rows, dim3(s->rows), dim3(kThreads), 0, (hipStream_t)stream, *s);
  return 0;
}
