// k_rows.hip - a token from every row of logits (qllama_sample_rows; semantics in
// qserve.h): sample_token (sampler.c:54-143) for many rows with settings and random
// numbers of their own, and min-p.
//
// No row is sorted.  With u = 16 log2(e) l / T, a token's weight 2^(u / 16) is that of
// its cell floor(u) of a grid that all rows of one temperature share, times 2^(f / 16), f
// = u - floor(u) in [0, 1).  Only the second factor, between 1 and 1.045, needs a token's
// own arithmetic (six terms), and in a histogram over the cells it adds up as a whole
// number of 2^-38 beside the number of tokens in one 64-bit word: sums are exact in any
// order, so LDS atomics give the same bits every time, and slices of a row add up without
// knowing its maximum.  k_sample_slices reads a row once, a slice a block, and leaves
// each slice's histogram of 768 cells (48 powers of two) and the largest logit of every 256
// tokens.  k_sample_pick puts a row's histograms together and finds in which cell the
// kept set ends.  With up to 64 tokens to the end of that cell it reads all of them again,
// from the groups of 256 that may hold some, and a wave puts them in order and finds the
// end and the drawn token (that instead of two searches: 21 -> 16 us at 4 rows of
// 128256 tokens).  Otherwise it searches first in the cell where the set ends, then in the
// one in which the drawn token lies: the cell's range of (logit, index) is divided into up
// to 512 parts until the one where the search ends holds 64 tokens at most.
#include <hip/hip_runtime.h>

#include "qserve_host.h"

namespace {

typedef unsigned long long u64;

// A slice of a row is a block's.  4 rows of 128256 tokens took 15.3 us with slices of 8192,
// 16.6 with 4096 (more histograms to put together), 18.1 with 16384; 192 rows 61, 78 (an
// earlier form: 75 with 8192) and 62 to 66.
constexpr int kSliceThreads = 512, kQuads = 4, kSlice = 4 * kSliceThreads * kQuads, kSliceGroups = kSlice / 256;
constexpr int kBins = 768;            // cells of a histogram: the tokens past it weigh less than 2^-47 of the largest
constexpr double kGrid = 16.0;        // cells a power of two
constexpr int kPickThreads = kBins;   // one a cell
constexpr int kParts = 512;           // parts of a divided range
constexpr int kList = 2048;           // tokens of a cell that are kept in LDS
constexpr int kUnitBits = 43;         // a row's weights are whole numbers of 2^-43
constexpr int kFractionBits = 38;
constexpr double kLog2e = 1.4426950408889634074;
constexpr int kCountShift = 48;       // a histogram word: number of tokens, sum of 2^38 (2^(f / 16) - 1)

// A slice of a row in the workspace, behind all histograms and before the largest logits
// of all groups of 256 tokens.
struct Slice {
  u64 best;                           // token_key of the first largest logit, 0: all masked
  uint32_t n;                         // tokens that are not masked
  uint32_t pad;
};

// A logit and its index (20 bits) as one number, larger for earlier in the order; 0: masked.
__device__ inline u64 token_key(float l, int i) {
  if (!(l > -__builtin_inff())) return 0;               // -inf and NaN
  const uint32_t b = __float_as_uint(l + 0.0f);         // -0 as 0
  const uint32_t o = b & 0x80000000u ? ~b : b | 0x80000000u;
  return (u64)o << 20 | (0xfffffu - (uint32_t)i);
}
__device__ inline float key_logit(u64 k) {
  const uint32_t o = (uint32_t)(k >> 20);
  return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ inline int key_index(u64 k) { return (int)(0xfffffu - (uint32_t)(k & 0xfffffu)); }
__device__ inline u64 smallest_key(float l) { return token_key(l, 0xfffff); }   // of all tokens with this logit

// 2^38 (2^(f / 16) - 1), 0 <= f <= 1, rounded to whole: six terms of the exponential's
// series (the seventh is 2^-6 at most), and 2^52 whose addition rounds
struct Series {
  double a[6];
  __host__ __device__ inline Series() {
    constexpr double x = 0.69314718055994530942 / kGrid, s = (double)(1ull << kFractionBits);
    a[0] = s * x; a[1] = a[0] * x / 2; a[2] = a[1] * x / 3; a[3] = a[2] * x / 4; a[4] = a[3] * x / 5; a[5] = a[4] * x / 6;
  }
  __host__ __device__ inline u64 operator()(double f) const {
    double s = a[5];
#pragma unroll
    for (int i = 4; i >= 0; i--) s = fma(s, f, a[i]);
    return __builtin_bit_cast(u64, fma(s, f, 4503599627370496.0)) & 0xfffffffffffffull;
  }
};

// A token below `top`: its cell's distance from top's (kBins: past the last) and f.  per: 16
// log2(e) / T.  Tokens equal to top share its cell whatever it is, infinity too.
struct Place { int bin; double f; };
__host__ __device__ inline Place place_of(float l, float top, double cell_top, double per) {
  const double u = (double)l * per, cell = floor(u), d = cell_top - cell;
  if (l == top && !(u - cell >= 0.0)) return {0, 0.0};
  return {d < kBins ? (int)d : kBins, u - cell};
}
__host__ __device__ inline double cell_of(float l, double per) { return floor((double)l * per); }

// 2^(5 - bin / 16): a histogram's 2^-38 as units of 2^-43, and the cell's weight.  The
// sixteenths by the exponential's series (0.65^16 / 16! is 5e-17).
__host__ __device__ inline double scale_of(int bin) {
  const double x = (bin & 15) * (-0.69314718055994530942 / kGrid);
  double s = 1.0 / 1307674368000.0;
  s = fma(s, x, 1.0 / 87178291200.0);
  s = fma(s, x, 1.0 / 6227020800.0);
  s = fma(s, x, 1.0 / 479001600.0);
  s = fma(s, x, 1.0 / 39916800.0);
  s = fma(s, x, 1.0 / 3628800.0);
  s = fma(s, x, 1.0 / 362880.0);
  s = fma(s, x, 1.0 / 40320.0);
  s = fma(s, x, 1.0 / 5040.0);
  s = fma(s, x, 1.0 / 720.0);
  s = fma(s, x, 1.0 / 120.0);
  s = fma(s, x, 1.0 / 24.0);
  s = fma(s, x, 1.0 / 6.0);
  s = fma(s, x, 0.5);
  s = fma(s, x, 1.0);
  s = fma(s, x, 1.0);
  return ldexp(s, kUnitBits - kFractionBits - (bin >> 4));
}
// n tokens of a cell, x of whose fractions: their weight in units.  In bin 0 exact, so
// equal largest logits weigh alike, alone and together; elsewhere rounded.
__host__ __device__ inline u64 units(int bin, double scale, u64 n, u64 x) {
  const u64 raw = (n << kFractionBits) + x;
  return bin == 0 ? raw << (kUnitBits - kFractionBits) : (u64)((double)raw * scale + 0.5);
}
// A token's weight unrounded, in units
__device__ inline double weight(Place p) { return exp2(kUnitBits + (p.f - p.bin) * (1.0 / kGrid)); }

__host__ __device__ inline double per_of(float temperature) { return kGrid * kLog2e / (double)temperature; }

// What one row asks for.
struct Ask {
  double per;                         // 16 log2(e) / T
  bool greedy;
};
__device__ inline Ask ask_of(const QSampleRows &a, int r) {
  const float T = a.temperature ? a.temperature[r] : 1.0f;
  return {per_of(T), !(T > 0.0f)};
}

struct Mass { u64 w; uint32_t n; };

template <int CTRL, int ROWS>
__device__ inline uint32_t from_lane(uint32_t x) { return __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xf, false); }
template <int CTRL, int ROWS = 0xf>
__device__ inline void add_from(Mass &v) {
  const uint32_t lo = from_lane<CTRL, ROWS>((uint32_t)v.w), hi = from_lane<CTRL, ROWS>((uint32_t)(v.w >> 32));
  v.n += from_lane<CTRL, ROWS>(v.n);
  v.w += (u64)hi << 32 | lo;
}
// Inclusive sums over a wave: within rows of 16 lanes, then from row to row.
__device__ inline Mass wave_scan(Mass v) {
  add_from<0x111>(v);           // row_shr 1, 2, 4, 8
  add_from<0x112>(v);
  add_from<0x114>(v);
  add_from<0x118>(v);
  add_from<0x142, 0xa>(v);      // row_bcast 15 to rows 1 and 3, 31 to rows 2 and 3
  add_from<0x143, 0xc>(v);
  return v;
}

template <int CTRL, int ROWS = 0xf>
__device__ inline float max_from(float x) {
  const int u = __float_as_int(x);
  return fmaxf(x, __int_as_float(__builtin_amdgcn_update_dpp(u, u, CTRL, ROWS, 0xf, false)));
}
// The largest value of a wave, in every lane.
__device__ inline float wave_max(float x) {
  x = max_from<0x111>(x);
  x = max_from<0x112>(x);
  x = max_from<0x114>(x);
  x = max_from<0x118>(x);
  x = max_from<0x142, 0xa>(x);
  x = max_from<0x143, 0xc>(x);
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 63));
}

// The largest of each of four values over a wave: of x[i] in lanes 16 i .. 16 i + 15.
__device__ inline float wave_max4(const float (&x)[4]) {
  typedef uint32_t u2 __attribute__((ext_vector_type(2)));
  float y[2];
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const u2 h = __builtin_amdgcn_permlane32_swap(__float_as_uint(x[i]), __float_as_uint(x[i + 2]), false, false);
    y[i] = fmaxf(__uint_as_float(h.x), __uint_as_float(h.y));
  }
  const u2 h = __builtin_amdgcn_permlane16_swap(__float_as_uint(y[0]), __float_as_uint(y[1]), false, false);
  float z = fmaxf(__uint_as_float(h.x), __uint_as_float(h.y));
  z = max_from<0x128>(z);       // row_ror 8, 4, 2, 1
  z = max_from<0x124>(z);
  z = max_from<0x122>(z);
  return max_from<0x121>(z);
}

// A slice of kSlice tokens in registers: the only reading of most of a row.  Near the
// memory's rate for many rows: 192 rows of 128256 tokens 27.4 us, 98 MB read and 16 MB
// of histograms written (greedy rows leave none), beside 16 tokens' arithmetic and atomics a thread; 4 rows
// 5.3 us.
__global__ __launch_bounds__(kSliceThreads) void k_sample_slices(QSampleRows a, Slice *slices, u64 *hist, float *groups) {
  __shared__ u64 h[kBins], bests[kSliceThreads / 64];
  __shared__ uint32_t counts[kSliceThreads / 64];
  const int r = blockIdx.y, t = threadIdx.x;
  const size_t at = (size_t)r * gridDim.x + blockIdx.x;
  const float *row = a.logits + r * a.stride;
  const int i0 = blockIdx.x * kSlice;
  float l[kQuads][4];
#pragma unroll
  for (int j = 0; j < kQuads; j++) {
    const int i = i0 + (j * kSliceThreads + t) * 4;
    if (i + 4 <= a.vocab) {
      __builtin_memcpy(l[j], row + i, sizeof l[j]);      // any 4-byte boundary
    } else {
#pragma unroll
      for (int c = 0; c < 4; c++) l[j][c] = i + c < a.vocab ? row[i + c] : -__builtin_inff();
    }
  }
  const Ask ask = ask_of(a, r);
  for (int b = t; b < kBins; b += kSliceThreads) h[b] = 0;
  float most = -__builtin_inff();
  uint32_t count = 0;
#pragma unroll
  for (int j = 0; j < kQuads; j += 4) {
    float x[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      x[i] = fmaxf(fmaxf(l[j + i][0], l[j + i][1]), fmaxf(l[j + i][2], l[j + i][3]));      // of a NaN and a number the number
#pragma unroll
      for (int c = 0; c < 4; c++) count += __builtin_popcountll(__ballot(l[j + i][c] >= -3.4028234663852886e38f));    // in scalar registers
    }
    const float group = wave_max4(x);
    if ((t & 15) == 0) groups[at * kSliceGroups + (j + (t >> 4 & 3)) * (kSliceThreads / 64) + (t >> 6)] = group;
    most = fmaxf(most, group);
  }
  most = wave_max(most);
  u64 best = token_key(most, 0);
  if (ask.greedy) {                                      // its index counts
    best = 0;
#pragma unroll
    for (int j = kQuads - 1; j >= 0; j--)
#pragma unroll
      for (int c = 3; c >= 0; c--)
        if (l[j][c] == most) best = token_key(most, i0 + (j * kSliceThreads + t) * 4 + c);
    for (int d = 32; d; d >>= 1) {
      const u64 o = __shfl_xor(best, d);
      best = o > best ? o : best;
    }
  }
  if ((t & 63) == 0) { bests[t >> 6] = best; counts[t >> 6] = count; }
  __syncthreads();
  count = 0;
#pragma unroll
  for (int i = 0; i < kSliceThreads / 64; i++) {
    best = bests[i] > best ? bests[i] : best;
    count += counts[i];
  }
  if (t == 0) slices[at] = {best, count, 0};
  if (ask.greedy || !best) return;                       // no histogram is read

  const float top = key_logit(best);
  const double cell_top = cell_of(top, ask.per);
  Series whole;
#pragma unroll
  for (int i = 0; i < 6; i++) asm volatile("" : "+v"(whole.a[i]));     // kept in registers, not moved there for every token
  if (fabs(cell_top) < 1e15) {
#pragma unroll
    for (int j = 0; j < kQuads; j++)
#pragma unroll
      for (int c = 0; c < 4; c++) {
        const double u = (double)l[j][c] * ask.per, cell = floor(u), d = cell_top - cell;
        if (d < kBins) atomicAdd(&h[(int)d], whole(u - cell) | 1ull << kCountShift);      // NaN and -inf are not
      }
  } else {                                               // infinite or enormous logits
    for (int i = i0 + t; i < min(i0 + kSlice, a.vocab); i += kSliceThreads) {
      const float x = row[i];
      const Place p = place_of(x, top, cell_top, ask.per);
      if (x > -__builtin_inff() && p.bin < kBins) atomicAdd(&h[p.bin], whole(p.f) | 1ull << kCountShift);
    }
  }
  __syncthreads();
  for (int b = t; b < kBins; b += kSliceThreads) hist[at * kBins + b] = h[b];
}

constexpr int kPickWaves = kPickThreads / 64;
constexpr int kAhead = 4;             // loads of a thread under way; 8 took 18.9 us against 16.6 (more registers than there are)

// Where a search stands: a place (a bin, a part), what lies before it, the tokens inside,
// the scale of the bin.
struct Hit { int at; Mass before; uint32_t inside; double scale; };

// Sets of what waves tell each other, used in turn: a set is written again only after the
// barrier behind the next one's writing, when all have read it.
struct Shared {
  u64 w[kParts], list[kList];
  uint32_t n[kParts];
  u64 few[64], order[64];
  double scale[kBins];
  u64 scan_w[2][kPickWaves];
  uint32_t scan_n[2][kPickWaves];
  Hit hit[2][kPickWaves];
  int hit_at[2][kPickWaves];
  u64 found_w[2], found_key[2];
  uint32_t found_n[2], n_some[2], n_list[2], n_few;          // of the first search and the second
};

// Inclusive sums over the block's threads.
__device__ Mass scan(Mass v, Shared &s, int &turn) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  turn ^= 1;
  v = wave_scan(v);
  if (lane == 63) { s.scan_w[turn][wave] = v.w; s.scan_n[turn][wave] = v.n; }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kPickWaves - 1; i++) {
    v.w += i < wave ? s.scan_w[turn][i] : 0;
    v.n += i < wave ? s.scan_n[turn][i] : 0;
  }
  return v;
}

// What the first thread has that says so.
__device__ Hit first_of(bool here, const Hit &mine, Shared &s, int &turn) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  turn ^= 1;
  const uint64_t b = __ballot(here);
  if (lane == (b ? __builtin_ctzll(b) : 0)) {
    s.hit_at[turn][wave] = b ? mine.at : -1;
    s.hit[turn][wave] = mine;
  }
  __syncthreads();
  int w = 0;
#pragma unroll
  for (int i = kPickWaves - 1; i >= 0; i--) w = s.hit_at[turn][i] >= 0 ? i : w;
  return s.hit[turn][w];
}

// Where a search ends: at the first token at which n tokens or the weight w are reached,
// before the first one whose key is below `floor`, or at the last.
struct Goal { uint32_t n; double w; u64 floor; };
__device__ inline bool reached(Mass m, Goal g) { return m.n >= g.n || (double)m.w >= g.w; }

struct Row {
  const float *l;
  int V, groups;                // tokens; groups of 256
  const float *most;            // LDS: their largest logits
  uint16_t *some;               // LDS: the groups that a search reads
  float top;
  double cell_top, per, inverse;   // 1 / per
};

struct Found { Mass upto; u64 key; };   // number and weight up to and with a token, and the token (0: none below `before`)

constexpr uint32_t kOrdLowest = 0x00800000u, kOrdInf = 0xff800000u;    // of the lowest finite float, and infinity
__device__ inline uint32_t ord_of(float l) {
  const uint32_t b = __float_as_uint(l);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ inline float of_ord(uint32_t o) { return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o); }

// The smallest float that passes a test which a larger one passes too, near c: a wave
// tries 64 (half: 32, in each half of the wave) neighbours at once.  0: it is not among them.
__device__ inline uint32_t neighbour(float c, int n) {
  const long long o = (long long)ord_of(c) + (int)(threadIdx.x & (n - 1)) - n / 2;
  return o < kOrdLowest ? kOrdLowest : o > kOrdInf ? kOrdInf : (uint32_t)o;
}
__device__ inline float finite(double x) { return (float)fmin(fmax(x, -3.4028234663852886e38), 3.4028234663852886e38); }

// Range of the keys of a cell's tokens.  Its ends are near where the arithmetic puts them;
// where that has no room for them (infinite or enormous logits or temperatures) they are
// searched among all floats.
__device__ void range_of(const Row &row, int bin, u64 &lo, u64 &hi) {
  const int half = threadIdx.x >> 5 & 1, i = threadIdx.x & 31;        // its low end, and the next cell's
  const double want = row.cell_top - bin + half;
  if (row.per > 0.0 && fabs(row.cell_top) < 1e15) {
    const uint32_t o = neighbour(finite(want * row.inverse), 32);
    const uint64_t pass = __ballot(cell_of(of_ord(o), row.per) >= want);
    const uint32_t below = (uint32_t)pass, above = (uint32_t)(pass >> 32);
    if (below && !(below & 1) && above && !(above & 1)) {
      lo = (u64)__shfl(o, __builtin_ctz(below)) << 20;
      hi = (u64)__shfl(o, 32 + __builtin_ctz(above)) << 20;
      return;
    }
  }
  uint32_t from = kOrdLowest, n = kOrdInf - kOrdLowest + 1;          // the first in the cell or above is from .. from + n
  while (__ballot(n > 0)) {
    const uint32_t part = n / 32 + (n % 32 != 0), at = part * (i + 1) - 1;
    const bool pass = at >= n || place_of(of_ord(from + at), row.top, row.cell_top, row.per).bin <= bin - half;
    const uint32_t f = __builtin_ctz((uint32_t)(__ballot(pass) >> (32 * half)));
    const uint32_t last = part * (f + 1) - 1 < n ? part * (f + 1) - 1 : n;
    from += n ? part * f : 0;
    n = n ? last - part * f : 0;
  }
  lo = (u64)__shfl(from, 0) << 20;
  hi = (u64)__shfl(from, 32) << 20;
}

// The key below which tokens weigh less than m (0 < m <= 1) of the largest.
__device__ u64 floor_of(float m, const Row &row) {
  if (!(fabsf(row.top) < __builtin_inff()) || m >= 1.0f) return smallest_key(row.top);
  if (!(row.per > 0.0)) return 1;                         // all weigh alike
  const uint32_t o = neighbour(finite((double)row.top + log2((double)m) * kGrid * row.inverse), 64);
  const float l = of_ord(o);
  const uint64_t pass = __ballot(l >= row.top || exp2(((double)l - (double)row.top) * row.per / kGrid) >= (double)m);
  return (u64)__shfl(o, pass ? __builtin_ctzll(pass) : 63) << 20;
}

// Every token with a key in [lo, hi), as f(key, place), among the first n_some groups in
// row.some, a group a wave's load.
template <typename F>
__device__ void for_tokens(const Row &row, int n_some, u64 lo, u64 hi, F f) {
  // keys below -inf's and above inf's are no logits
  const float least = lo >> 20 >= kOrdLowest ? of_ord((uint32_t)(lo >> 20)) : -__builtin_inff(),
              most = hi >> 20 < kOrdInf ? of_ord((uint32_t)(hi >> 20)) : __builtin_inff();
  const int all = n_some * 64;
  const auto first = [&](int q) { return q < all ? (row.some[q >> 6] << 8) + (q & 63) * 4 : row.V; };
  for (int q0 = threadIdx.x; q0 < all; q0 += 8 * kPickThreads) {
    float l[8][4];
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const int at = first(q0 + j * kPickThreads);
      if (at + 4 <= row.V) {
        __builtin_memcpy(l[j], row.l + at, sizeof l[j]);
      } else {
#pragma unroll
        for (int c = 0; c < 4; c++) l[j][c] = at + c < row.V ? row.l[at + c] : -__builtin_inff();
      }
    }
    uint32_t in_range = 0;      // few: read again one by one, which keeps the code short (it runs once, from a cold cache)
#pragma unroll
    for (int j = 0; j < 8; j++)
#pragma unroll
      for (int c = 0; c < 4; c++) in_range |= (uint32_t)(l[j][c] >= least && l[j][c] <= most) << (4 * j + c);
    for (; in_range; in_range &= in_range - 1) {
      const int b = __builtin_ctz(in_range), at = first(q0 + (b >> 2) * kPickThreads) + (b & 3);
      const float x = at < row.V ? row.l[at] : -__builtin_inff();
      const u64 k = token_key(x, at);
      if (k >= lo && k < hi && k) f(k, place_of(x, row.top, row.cell_top, row.per));
    }
  }
  __syncthreads();
}

// l[b / 4][b % 4], from registers.
__device__ inline float pick_of(const float (&l)[kAhead][4], int b) {
  float x[kAhead * 4];
#pragma unroll
  for (int i = 0; i < kAhead * 4; i++) x[i] = l[i >> 2][i & 3];
#pragma unroll
  for (int h = 1; h < kAhead * 4; h *= 2) {
    const bool odd = b & h;
#pragma unroll
    for (int i = 0; i < kAhead * 4; i += 2 * h) x[i] = odd ? x[i + h] : x[i];
  }
  return x[0];
}

// The keys in [lo, hi) of the tokens of those groups into s.list.
__device__ void list_tokens(const Row &row, Shared &s, int n_some, u64 lo, u64 hi, uint32_t &fill) {
  const float least = lo >> 20 >= kOrdLowest ? of_ord((uint32_t)(lo >> 20)) : -3.4028234663852886e38f,
              most = hi >> 20 < kOrdInf ? of_ord((uint32_t)(hi >> 20)) : __builtin_inff();
  const int all = n_some * 64;
  const auto first = [&](int q) { return q < all ? (row.some[q >> 6] << 8) + (q & 63) * 4 : row.V; };
  for (int q0 = threadIdx.x; q0 - (int)threadIdx.x < all; q0 += kAhead * kPickThreads) {
    float l[kAhead][4];
#pragma unroll
    for (int j = 0; j < kAhead; j++) {
      const int at = first(q0 + j * kPickThreads);
      if (at + 4 <= row.V) {
        __builtin_memcpy(l[j], row.l + at, sizeof l[j]);
      } else {
#pragma unroll
        for (int c = 0; c < 4; c++) l[j][c] = at + c < row.V ? row.l[at + c] : -__builtin_inff();
      }
    }
    uint32_t in_range = 0;
#pragma unroll
    for (int j = 0; j < kAhead; j++)
#pragma unroll
      for (int c = 0; c < 4; c++) in_range |= (uint32_t)(l[j][c] >= least && l[j][c] <= most) << (4 * j + c);
    for (; in_range; in_range &= in_range - 1) {
      const int b = __builtin_ctz(in_range);
      const u64 k = token_key(pick_of(l, b), first(q0 + (b >> 2) * kPickThreads) + (b & 3));
      if (k >= lo && k < hi) s.list[min(atomicAdd(&fill, 1u), kList - 1u)] = k;    // never more, by the histogram
    }
  }
  __syncthreads();
}

// Divide the range [lo, hi) of keys, in which `inside` tokens lie and before which
// `before` is, and go to the part where the search ends.  each(f) calls f(key, place) for
// the range's tokens, and synchronizes.
template <typename E>
__device__ void divide(Shared &s, int &turn, Goal goal, const Hit &bin, u64 &lo, u64 &hi, Mass &before, uint32_t &inside, E each) {
  const int span = 64 - __builtin_clzll((hi - lo - 1) | 1), shift = span > 9 ? span - 9 : 0;
  const int t = threadIdx.x;
  if (t < kParts) { s.w[t] = 0; s.n[t] = 0; }
  __syncthreads();
  each([&](u64 k, Place p) {
    const int d = (int)((hi - 1 - k) >> shift);
    atomicAdd(&s.w[d], units(bin.at, bin.scale, 1, Series()(p.f)));
    atomicAdd(&s.n[d], 1u);
  });
  const Mass own = t < kParts ? Mass{s.w[t], s.n[t]} : Mass{0, 0};
  const Mass upto = scan(own, s, turn);
  const bool ends = own.n && (reached({before.w + upto.w, before.n + upto.n}, goal) || upto.n == inside);
  const bool floor_here = goal.floor && t < kParts && (goal.floor >= hi ? t == 0 : goal.floor >= lo && (int)((hi - 1 - goal.floor) >> shift) == t);
  const Hit h = first_of(ends || floor_here, {t, {upto.w - own.w, upto.n - own.n}, own.n, 0.0}, s, turn);
  before.w += h.before.w;
  before.n += h.before.n;
  inside = h.inside;
  const u64 top = hi - ((u64)h.at << shift), bottom = hi - lo > (u64)(h.at + 1) << shift ? hi - ((u64)(h.at + 1) << shift) : lo;
  lo = bottom;
  hi = top;
}

// The token at which a search ends that lies in bin h.at.  list_bin: the bin all of
// whose tokens s.list holds, or -1.  `both`: with no more than 64 tokens up to the end
// of the bin they are all put in order, and the one that u times the kept weight falls on
// is found on the way; `both` is cleared where that was not done.
__device__ Found locate(const Row &row, Shared &s, int &turn, int search, Goal goal, const Hit &h, int &list_bin, bool &both, double u) {
  const int t = threadIdx.x, bin = h.at;
  Mass before = h.before;
  uint32_t inside = h.inside;
  both = both && before.n + inside <= 64;
  if (!inside && !both) return {before, 0};
  u64 lo, hi;
  range_of(row, bin, lo, hi);
  if (both) {
    inside += before.n;
    before = {0, 0};
    hi = 1ull << 52;
  }
  if (list_bin != bin) {
    const float least = lo >> 20 >= kOrdLowest ? of_ord((uint32_t)(lo >> 20)) : -3.4028234663852886e38f;
    for (int g0 = t & ~63; g0 < row.groups; g0 += kPickThreads) {      // the groups that may hold some
      const bool has = g0 + (t & 63) < row.groups && row.most[g0 + (t & 63)] >= least;
      const uint64_t all = __ballot(has);
      uint32_t at = 0;
      if ((t & 63) == 0 && all) at = atomicAdd(&s.n_some[search], (uint32_t)__builtin_popcountll(all));
      at = __builtin_amdgcn_readfirstlane(at);
      if (has) row.some[at + __builtin_popcountll(all & ((1ull << (t & 63)) - 1))] = (uint16_t)(g0 + (t & 63));
    }
    __syncthreads();
    const int n_some = s.n_some[search];
    list_bin = bin;
    while (inside > kList) {
      divide(s, turn, goal, h, lo, hi, before, inside, [&](auto f) { for_tokens(row, n_some, lo, hi, f); });
      list_bin = -1;
    }
    if (!inside) return {before, 0};
    list_tokens(row, s, n_some, lo, hi, s.n_list[search]);
  }
  const uint32_t listed = inside;
  const auto in_list = [&](auto f) {
    for (uint32_t i = t; i < listed; i += kPickThreads) {
      const u64 k = s.list[i];
      if (k >= lo && k < hi) f(k, place_of(key_logit(k), row.top, row.cell_top, row.per));
    }
    __syncthreads();
  };
  const u64 *few = s.list;
  if (listed > 64) {
    while (inside > 64) divide(s, turn, goal, h, lo, hi, before, inside, in_list);
    if (!inside) return {before, 0};
    if (t == 0) s.n_few = 0;
    __syncthreads();
    in_list([&](u64 k, Place) { s.few[min(atomicAdd(&s.n_few, 1u), 63u)] = k; });
    few = s.few;
  }
  turn ^= 1;
  if (t < 64) {                 // a wave puts them in order: every lane counts the keys before its own
    const u64 mine = t < (int)inside ? few[t] : 0;
    const auto of_lane = [&](u64 x, int i) { return (u64)__builtin_amdgcn_readlane((int)(x >> 32), i) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)x, i); };
    int rank = 0;
    for (int i = 0; i < (int)inside; i++) rank += of_lane(mine, i) > mine;
    if (mine) s.order[rank] = mine;
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    const u64 k = mine ? s.order[t] : 0;
    const Place p = place_of(key_logit(k), row.top, row.cell_top, row.per);
    Mass m = {k ? units(p.bin, s.scale[min(p.bin, kBins - 1)], 1, Series()(p.f)) : 0, k != 0};
    m = wave_scan(m);
    const u64 next = __shfl_down(k, 1);
    m = {before.w + m.w, before.n + m.n};
    const uint64_t stops = __ballot(k && (reached(m, goal) || t + 1 == (int)inside || next < goal.floor));
    const bool none = __shfl(k, 0) < goal.floor;          // not even the first of them
    const int end = __builtin_ctzll(stops);
    if (none ? t == 0 : t == end) {
      s.found_w[turn] = none ? before.w : m.w;
      s.found_n[turn] = none ? before.n : m.n;
      if (!both) s.found_key[turn] = none ? 0 : k;
    }
    if (both) {
      const uint64_t there = __ballot(t >= end || (double)m.w >= u * (double)of_lane(m.w, end));
      if (t == __builtin_ctzll(there)) s.found_key[turn] = k;
    }
  }
  __syncthreads();
  return {{s.found_w[turn], s.found_n[turn]}, s.found_key[turn]};
}

// A row's settings, read before they are needed.
struct Limits {
  float u, p, m;
  int k;
  __device__ inline Limits(const QSampleRows &a, int r)
      : u(a.u[r]), p(a.top_p ? a.top_p[r] : 0.0f), m(a.min_p ? a.min_p[r] : 0.0f), k(a.top_k ? a.top_k[r] : 0) {}
};

__device__ inline void write_first(const QSampleRows &a, int r, u64 best) {
  a.token[r] = best ? key_index(best) : -1;
  if (a.prob) a.prob[r] = best ? 1.0f : 0.0f;
  if (a.kept) a.kept[r] = best ? 1 : 0;
}

// A row's token, from thread t's cell t: n tokens, x of whose fractions.  A chain of short
// steps, each a barrier or a trip to memory behind the one before: 10.8 us for 4 rows
// with top-k 40 and top-p 0.95.  Of 192 rows with settings of their own (35 us) a few keep
// thousands of tokens and end in cells that every group may hold some of: their CU reads
// most of the row again, at some 16 bytes a cycle, which takes 15 us.  (768 threads with four
// loads of 16 bytes each under way, and 1.5 us a trip, come to as much: whether the CU or
// what is under way sets that rate has not been told apart.)
__device__ void pick(const QSampleRows &a, int r, const Row &row, Shared &s, const Limits &limits, uint32_t n, u64 x, uint32_t all_n) {
  const int t = threadIdx.x;
  int turn = 0;
  if (t < 2) { s.n_some[t] = 0; s.n_list[t] = 0; }
  const double scale = scale_of(t);
  const Mass own = {units(t, scale, n, x), n};
  s.scale[t] = scale;
  const Mass upto = scan(own, s, turn);
  const Mass before = {upto.w - own.w, upto.n - own.n};
  if (t == kPickThreads - 1) { s.found_w[0] = upto.w; s.found_n[0] = upto.n; }
  __syncthreads();
  const Mass held = {s.found_w[0], s.found_n[0]};          // tokens behind the last bin weigh nothing

  const bool by_min = limits.m > 0x1p-43f;
  const bool by_mass = limits.p > 0.0f && limits.p < 1.0f, by_count = limits.k > 0 && (uint32_t)limits.k < all_n;
  const float u = limits.u > 0.0f ? (limits.u < 1.0f ? limits.u : 0x1.fffffep-1f) : 0.0f;
  Mass kept = {held.w, by_count ? (uint32_t)limits.k : all_n};   // a limit among the tokens that weigh nothing needs no search
  Found f = {{0, 0}, 0};
  int list_bin = -1;
  // first where the kept set ends, then the token; one code for both, as it runs from a cold cache
  const u64 floor = by_min ? floor_of(limits.m, row) : 0;
  const int floor_bin = by_min ? place_of(key_logit(floor), row.top, row.cell_top, row.per).bin : kBins;
#pragma unroll 1
  for (int search = (by_count && kept.n < held.n) || by_mass || by_min ? 0 : 1; search < 2; search++) {
    Goal goal = {kept.n, (double)u * (double)kept.w, 0};
    if (search == 0) {
      goal.w = by_mass ? (double)limits.p * (double)held.w : __builtin_inf();
      goal.floor = floor;
    }
    const bool ends = own.n && (reached(upto, goal) || upto.n == held.n);
    bool both = search == 0;
    f = locate(row, s, turn, search, goal, first_of(ends || (search == 0 && t == floor_bin), {t, before, own.n, scale}, s, turn), list_bin, both, (double)u);
    if (search == 0) kept = f.upto;
    if (both) break;
  }
  if (t == 0) {
    a.token[r] = key_index(f.key);
    if (a.prob) a.prob[r] = (float)(weight(place_of(key_logit(f.key), row.top, row.cell_top, row.per)) / (double)kept.w);
    if (a.kept) a.kept[r] = (int)kept.n;
  }
}

// A row's token from its slices' histograms.
__global__ __launch_bounds__(kPickThreads) void k_sample_pick(QSampleRows a, int slices, int groups, const Slice *recs, const u64 *hist, const float *most) {
  extern __shared__ float dyn[];
  __shared__ Shared s;
  int *offs = reinterpret_cast<int *>(dyn + groups);       // the row's bin that is a slice's first; kBins: none is
  const int r = blockIdx.x, t = threadIdx.x;
  const Ask ask = ask_of(a, r);
  const Limits limits(a, r);
  recs += (size_t)r * slices;
  hist += (size_t)r * slices * kBins;
  for (int i = t; i < groups; i += kPickThreads) dyn[i] = most[(size_t)r * slices * kSliceGroups + i];

  // every wave reduces the slices' records
  u64 best = 0;
  uint32_t all_n = 0;
  for (int i = t & 63; i < slices; i += 64) {
    const Slice x = recs[i];
    if (t < 64) offs[i] = __float_as_int(x.best ? key_logit(x.best) : -__builtin_inff());    // for now its largest logit
    best = x.best > best ? x.best : best;
    all_n += x.n;
  }
  for (int d = 32; d; d >>= 1) {
    const u64 o = __shfl_xor(best, d);
    best = o > best ? o : best;
    all_n += __shfl_xor(all_n, d);
  }
  if (!best || ask.greedy) {
    if (t == 0) write_first(a, r, best);
    return;
  }
  Row row = {a.logits + r * a.stride, a.vocab, groups, dyn, reinterpret_cast<uint16_t *>(offs + slices), key_logit(best), 0.0, ask.per, 1.0 / ask.per};
  row.cell_top = cell_of(row.top, row.per);
  if (t < 64)
    for (int i = t; i < slices; i += 64) {
      const float top = __int_as_float(offs[i]);
      offs[i] = top > -__builtin_inff() ? place_of(top, row.top, row.cell_top, row.per).bin : kBins;
    }
  __syncthreads();

  u64 x = 0;
  uint32_t n = 0;
#pragma unroll 16
  for (int i = 0; i < slices; i++) {
    const int b = t - offs[i];
    u64 y = hist[(size_t)i * kBins + (b < 0 ? 0 : b)];
    y = b < 0 ? 0 : y;
    n += (uint32_t)(y >> kCountShift);
    x += y & ((1ull << kCountShift) - 1);
  }
  pick(a, r, row, s, limits, n, x, all_n);
}

}  // namespace

extern "C" size_t qllama_sample_rows_work(int rows, int vocab) {
  if (rows < 0 || rows > 65535 || vocab < 1 || vocab > (1 << 20)) return 0;
  return 16 + (size_t)rows * ((vocab + kSlice - 1) / kSlice) * (kBins * sizeof(u64) + sizeof(Slice) + kSliceGroups * sizeof(float));
}

extern "C" unsigned long long qllama_test_sample_weight(float logit, float top, float temperature) {
  const double per = per_of(temperature);
  const Place p = place_of(logit, top, cell_of(top, per), per);
  return p.bin < kBins ? units(p.bin, scale_of(p.bin), 1, Series()(p.f)) : 0;
}

extern "C" int qllama_sample_rows(const QSampleRows *s, void *stream) {
  static const char fn[] = "qllama_sample_rows";
  if (!s || s->rows < 0 || s->rows > 65535) return qs::refuse(fn, "null argument, or rows not 0 .. 65535");
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
  const int slices = (s->vocab + kSlice - 1) / kSlice, groups = (s->vocab + 255) / 256;
  u64 *hist = static_cast<u64 *>(s->work);
  Slice *recs = reinterpret_cast<Slice *>(hist + (size_t)s->rows * slices * kBins);
  float *most = reinterpret_cast<float *>(recs + (size_t)s->rows * slices);
  QS_LAUNCH(fn, k_sample_slices, dim3(slices, s->rows), dim3(kSliceThreads), 0, (hipStream_t)stream, *s, recs, hist, most);
  const size_t lds = groups * (sizeof(float) + sizeof(uint16_t)) + slices * sizeof(int);
  QS_LAUNCH(fn, k_sample_pick, dim3(s->rows), dim3(kPickThreads), lds, (hipStream_t)stream, *s, slices, groups, recs, hist, most);
  return 0;
}
