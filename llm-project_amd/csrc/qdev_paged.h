// qdev_paged.h - what the attention kernels over a paged cache share: where a token lies,
// 16-bit parts of float operands and their matrix products, maxima and sums over lanes.
#ifndef QDEV_PAGED_H
#define QDEV_PAGED_H

#include <hip/hip_runtime.h>

#include "qserve.h"

namespace qpaged {

typedef float f2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr float kNegInf = -__builtin_inff();

__host__ __device__ inline int clamp_len(int len, int width, int page_size) {
  const int most = width * page_size;   // fits: checked by the host
  return len < 0 ? 0 : len > most ? most : len;
}

// Where a token lies: its table entry (of the last token for one behind it, so that the
// entry can always be read; len > 0) and its place there; then the entry's page, -1 for
// no page of the cache or no token.
__host__ __device__ inline int entry_of(long long key, int len, int page_size, int *place) {
  const int k = key < len ? (int)key : len - 1, e = k / page_size;
  *place = k - e * page_size;
  return e;
}
__host__ __device__ inline int page_of(int entry, long long key, int len, int n_pages) {
  return key < len && entry >= 0 && entry < n_pages ? entry : -1;
}

// What a part with maximum m counts against the maximum of all.  A part without one holds
// zeros, or the NaN of its scores, which has to stay.
__device__ inline float part_weight(float m, float top) { return m == kNegInf ? 1.0f : __builtin_amdgcn_exp2f(m - top); }

// max of a lane's value with those of lanes l ^ 16, l ^ 32 and l ^ 48
__device__ inline float max_groups(float x) {
  const uint32_t u = __float_as_uint(x);
  u2 r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const uint32_t y = __float_as_uint(fmaxf(__uint_as_float(r.x), __uint_as_float(r.y)));
  r = __builtin_amdgcn_permlane16_swap(y, y, false, false);
  return fmaxf(__uint_as_float(r.x), __uint_as_float(r.y));
}
__device__ inline float sum_groups(float x) {
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

__device__ inline uint32_t hi16s(uint32_t b, uint32_t a) { return __builtin_amdgcn_perm(b, a, 0x07060302); }
__device__ inline uint32_t lo16s(uint32_t b, uint32_t a) { return __builtin_amdgcn_perm(b, a, 0x05040100); }

// Parts of a float operand of 8 values: sums of the parts are the values (bf16: all 24
// bits by cutting; f16: to nearest twice, off by 2^-23 at most and without a bias, where
// cutting twice takes up to 3 x 2^-23).
struct Parts3 { u4 p[3]; };
__device__ inline Parts3 cut3(const float (&x)[8]) {
  Parts3 r;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    float a = x[2 * i], b = x[2 * i + 1];
#pragma unroll
    for (int k = 0; k < 3; k++) {
      r.p[k][i] = hi16s(__float_as_uint(b), __float_as_uint(a));
      if (k < 2) {
        a -= __uint_as_float(__float_as_uint(a) & 0xffff0000u);
        b -= __uint_as_float(__float_as_uint(b) & 0xffff0000u);
      }
    }
  }
  return r;
}
struct Parts2 { u4 p[2]; };
__device__ inline Parts2 cut2(const float (&x)[8]) {
  Parts2 r;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const h2 hi = __builtin_convertvector(f2{x[2 * i], x[2 * i + 1]}, h2);
    const h2 lo = __builtin_convertvector(f2{x[2 * i] - (float)hi.x, x[2 * i + 1] - (float)hi.y}, h2);
    r.p[0][i] = __builtin_bit_cast(uint32_t, hi);
    r.p[1][i] = __builtin_bit_cast(uint32_t, lo);
  }
  return r;
}

template <int T>
__device__ inline f4 mfma16(u4 a, u4 b, f4 c) {
  if constexpr (T != QLLAMA_KV_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, a), __builtin_bit_cast(bf8, b), c, 0, 0, 0);
}

}  // namespace qpaged

#endif
