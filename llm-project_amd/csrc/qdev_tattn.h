// qdev_tattn.h - attention of several new tokens a request over a paged key-value cache, with
// a mask among the new ones (qllama_tree_attention; semantics in qserve.h): the kernels, of
// which k_tattn_f32.hip, k_tattn_f16.hip, k_tattn_bf16.hip and k_tattn_i8.hip each compile a
// cache type's.  No counterpart in the reference, whose decode attention
// (llama.c:554-576) serves one token.
//
// The columns of a (request, KV head) are its rows times the query heads that share the KV
// head; a tile is 16 CG of them, and takes every key and value of the request once: CG waves
// side by side, 16 columns each, share what they stage in LDS.  S^T = K q^T on the matrix
// cores puts a column in a lane's column and 4 keys of each 16 in its rows; the same lane's
// weights are then the operand of O^T += V^T P^T, whose contraction slots are matched to the
// keys that the lane holds, so weights never move between lanes; values come out of LDS by
// transposing reads.
//
// The work of a call is the key steps of all tiles, laid one behind another, and for each tile
// some steps more for its beginning and end; every group of CG waves takes an equal share,
// whatever the lengths are, without the host knowing one.  A share that ends inside a tile
// leaves its maxima, sums and weighted values in the workspace, and k_tree_join puts a tile's
// parts together.  Where the tables are short a block takes whole tiles, its waves also parts
// of the keys that meet at the end, and there is no second launch (launch() has the rule).
//
// Precision as in k_pattn.hip: float queries and weights meet 16-bit keys and values as three
// (bf16, int8 codes) or two (f16) 16-bit parts; f32 rows go through the fp32 MFMA, or,
// from 33 columns on with heads of up to 128, as three parts themselves, as close as 32-bit
// products.
//
// What bounds it: up to 32 columns memory (int8: the codes' conversion too); from 64 on the
// matrix products of the parts and the softmax beside them:
// of a step's 6700 cycles (64 keys, 128 bf16 columns, heads of 128) 4500 are products and
// weights, 1500 of them on the matrix cores' own count for each of a SIMD's two waves, the
// rest is staging, places and the barrier.  Measured (both kernels; 32 query and 8 KV heads
// of 128 if not said; a 1 GiB copy moves 5.1 TB/s, a large bf16 product 1190 TFLOP/s):
//   64 ragged requests of up to 2560 tokens, bf16, 4 rows      84-89 us   4.5 TB/s
//   the same, 8 rows                                           88-91 us   4.3 TB/s
//   32 of them, up to 16 rows                                  72 us      3.0 TB/s
//   32 of them, up to 32 rows                                  89 us      2.0 TB/s, 570 TFLOP/s in parts
//   32 of them, up to 64 rows                                  162 us     700 TFLOP/s in parts
//   2 requests of up to 60000 tokens, f16, 48 rows             117-127 us 2.8 TB/s, 410 TFLOP/s in parts
//   64 requests of up to 4100 tokens, int8, 7 rows             101-114 us 2.6 TB/s
//   6 requests of up to 2048 tokens, f32, heads of 64, 200 rows in a chain  114-128 us  620 TFLOP/s in parts
//   the same, heads of 128, bf16 117 us, f16 106, int8 119      640, 480, 630 TFLOP/s in parts
//   1 request of 2060 tokens, bf16, 8 rows                     22 us
// Measured and not kept: 32 columns a wave (queries and sums of both spill: 225 us against 144 at
// 32 rows); blocks of eight waves whatever the columns, on other parts of a step's keys, that
// begin and end tiles together (113 against 99 at 16 rows); scores a step ahead of the weights,
// so that products run beside the exponentials (107 against 102 at 8 rows, 192 against 201 at
// 64; with registers that the queries need); a raised priority while
// products run (95 against 89 at 32 rows); blocks of one XCD on shares beside each other (132
// against 127 for the two long requests).
#ifndef QDEV_TATTN_H
#define QDEV_TATTN_H

#include <hip/hip_runtime.h>

#include "qdev_paged.h"
#include "qserve_host.h"

namespace qtree {

constexpr int kShares = 2048;         // eight waves a CU; a share takes as many as lie side by side

struct TaArgs {
  const char *k, *v;
  const float *ks, *vs;
  const float *q;
  float *o, *lse;
  const uint64_t *mask;
  const int *starts, *table, *lens;
  float *part;
  int4 *split;
  long long pst, hst, sst;            // bytes
  long long scp, sch, scs;            // floats
  long long q_stride, o_stride, lse_stride, table_stride;
  int rows, n_req, n_kv, G, hd, n_pages, page_size, width, words;
  int wide;                           // rows and strides are multiples of 16 bytes
  float qscale;                       // scale * log2(e)
};

// Launches a call on its cache's type; tile: as pick() in k_tattn.hip numbers them.
int launch_f32(const char *fn, const TaArgs &a, int tile, hipStream_t stream);
int launch_f16(const char *fn, const TaArgs &a, int tile, hipStream_t stream);
int launch_bf16(const char *fn, const TaArgs &a, int tile, hipStream_t stream);
int launch_i8(const char *fn, const TaArgs &a, int tile, hipStream_t stream);

}  // namespace qtree

#ifdef QTREE_TYPE
namespace {

using namespace qpaged;
using namespace qtree;

// What a type, a padded head size, the waves side by side and the parts of a step's keys fix.
template <int T, int HDP, int CG_, int KP_>
struct Cfg {
  static constexpr int CG = CG_, KP = KP_, THREADS = 64 * CG * KP, COLS = 16 * CG;
  static constexpr int SHARES = kShares / CG;
  // f32 rows: as they are, or (many columns) in three bf16 parts, queries and weights too, which the matrix cores take 16 times
  // as fast: the six products of parts that count make it 2.7 times.  Dropped ones, of a second with a third part or two
  // thirds, add up to 2^-24 of a product, what rounding it to 32 bits takes (with cut queries and weights it was 2^-21.6, always
  // toward 0)
  static constexpr bool SPLIT = T == QLLAMA_KV_F32 && (HDP == 64 ? CG >= 4 : HDP == 128 && CG == 8), F32 = T == QLLAMA_KV_F32 && !SPLIT;
  static constexpr bool HALF = T == QLLAMA_KV_F16;
  static constexpr int PLANES = SPLIT ? 3 : 1;
  static constexpr int ES = T == QLLAMA_KV_F32 ? 4 : T == QLLAMA_KV_I8 ? 1 : 2;         // of an element in the cache
  static constexpr int LES = F32 ? 4 : 2;                               // in LDS, of a part (int8: bf16, which holds the codes)
  static constexpr int LT = T == QLLAMA_KV_I8 || SPLIT ? QLLAMA_KV_BF16 : T;            // the products' type
  static constexpr int SUB = F32 ? 1 : 2, KEYS = 16 * SUB;              // keys that a wave takes at a time
  // times that it does between two barriers, as far as registers and LDS allow
  static constexpr int TIMES = SPLIT ? (HDP == 64 && CG == 8 ? 2 : 1) : CG >= 4 && HDP <= 128 ? 2 : 1, KS = KEYS * TIMES, STEP = KS * KP;
  // keys, and steps, whose time a tile's beginning and end take
  static constexpr int OVERKEYS = CG == 8 ? 256 : CG == 4 && HDP > 64 ? 128 : 64, OVER = OVERKEYS / STEP < 1 ? 1 : OVERKEYS / STEP;
  static constexpr int ROWB = HDP * LES, CH = ROWB / 16, SWZ = (CH < 16 ? CH : 16) - 1, EPC = 16 / LES;
  static constexpr int PLANEB = KS * ROWB, SIDEB = PLANES * PLANEB, PARTB = 2 * SIDEB;  // a part's keys, then values
  static constexpr int NBUF = CG == 1 ? 1 : 2;                          // a wave alone with its part needs no second buffer
  static constexpr bool ONCE = CG <= 2;                                 // a tile has a request's columns, all or nearly: loads past the caches' retention
  // threads that stage a part, and units of each: 16 bytes of the cache (split: 32), CPU chunks of 16 bytes in LDS (split: one a part)
  static constexpr int LOADS = SPLIT ? 2 : 1, CPU = T == QLLAMA_KV_I8 ? 2 : 1, TP = 64 * CG, U = 2 * KS * CH / CPU / TP;
  static constexpr int DPL = HDP / 16, QC = F32 ? HDP / 16 : HDP / 32;
  static constexpr int PARTS = F32 ? 1 : HALF ? 2 : 3;
  // weights are held times this in f16 products: two parts then keep 23 bits down to 2^-17 of the largest and the rest to 2^-40
  static constexpr float RAISED = HALF ? 32768.0f : 1.0f;
  // LDS: staged parts (and what waves hand over at a tile's end), places of the keys, absent keys, scales
  static constexpr int HANDB = (KP / 2) * CG * (DPL * 1024 + 512);
  static constexpr int STAGEB = NBUF * KP * PARTB > HANDB ? NBUF * KP * PARTB : HANDB;
  static constexpr int OFFB = 4 * KP * KS * 8, GONEB = 4 * KP * 8, SCALEB = T == QLLAMA_KV_I8 ? 2 * 2 * KP * KS * 4 : 0;
  static constexpr int LDSB = STAGEB + OFFB + GONEB + SCALEB;
  static constexpr int PARTF = CG * (DPL * 256 + 32);                   // floats of a tile's part in the workspace
};

typedef short s4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s4 s4_lds;

// Rows of request r, and the first of them.
__device__ inline int rows_of(const TaArgs &a, int r, int *first) {
  const int x = min(max(a.starts[r], 0), a.rows), y = min(max(a.starts[r + 1], 0), a.rows);
  *first = x;
  return max(y - x, 0);
}

// Inclusive sums over a wave.
__device__ inline long long scan64(long long x) {
  const int lane = threadIdx.x & 63;
  for (int d = 1; d < 64; d <<= 1) {
    const long long y = __shfl_up(x, d);
    if (lane >= d) x += y;
  }
  return x;
}

__device__ inline long long uniform(long long x) {
  return (long long)((unsigned long long)(unsigned)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32 | (unsigned)__builtin_amdgcn_readfirstlane((int)x));
}

// Which of 32 consecutive new rows from b0 on (before 0: earlier tokens) row i, the j-th of its request, attends to.
__device__ inline uint32_t seen_of(const TaArgs &a, int i, int j, int b0) {
  if (b0 <= -32) return ~0u;
  if (!a.mask) {
    const int n = j + 1 - b0;
    return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1;
  }
  const uint64_t *w = a.mask + (long long)i * a.words;
  if (b0 < 0) return (uint32_t)(w[0] << -b0) | ((1u << -b0) - 1);
  if (b0 >= 64 * a.words) return 0;
  const int at = b0 >> 6, sh = b0 & 63;
  uint64_t x = w[at] >> sh;
  if (sh > 32 && at + 1 < a.words) x |= w[at + 1] << (64 - sh);
  return (uint32_t)x;
}

// Whether a cached float is an infinity or a NaN.
template <int T>
__device__ inline bool odd_value(uint32_t x) {
  constexpr uint32_t E = T == QLLAMA_KV_F32 ? 0x7f800000u : T == QLLAMA_KV_F16 ? 0x7c00u : 0x7f80u;
  return (x & E) == E;
}

// 8 floats as sums of three bf16 numbers, each rounded to nearest: exact, the second at most 2^-8 and the third 2^-17 of the
// first.  ANY: the first has to be kept within bf16's range, which ends 2^-8 below a float's.
typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
template <bool ANY>
__device__ inline Parts3 round3(const float (&x)[8]) {
  Parts3 r;
  constexpr float most = 0x1.fep127f;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    float a = x[2 * i], b = x[2 * i + 1];
#pragma unroll
    for (int k = 0; k < 3; k++) {
      const f2 y = !ANY || k ? f2{a, b} : f2{__builtin_amdgcn_fmed3f(a, -most, most), __builtin_amdgcn_fmed3f(b, -most, most)};
      r.p[k][i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(y, bf2));
      if (k < 2) {
        a -= __uint_as_float(r.p[k][i] << 16);
        b -= __uint_as_float(r.p[k][i] & 0xffff0000u);
      }
    }
  }
  return r;
}

// The dim of a head whose output is element c of an accumulator's row `lane` of 16.
template <typename C>
__device__ inline int dim_of(int c, int lane) { return C::F32 ? 64 * (c / 4) + 4 * lane + c % 4 : 16 * c + lane; }

// A column's outputs from what a lane holds: rows 4 g .. of every accumulator.
template <typename C>
__device__ inline void put(float *o, const f4 (&acc)[C::DPL], int g, int hd, float by) {
  by *= 1.0f / C::RAISED;
#pragma unroll
  for (int i = 0; i < C::DPL; i++) {
    const int k = i % 4, c = i - k;                   // f32: dims beside each other lie in four accumulators
    const float x[4] = {(C::F32 ? acc[c][k] : acc[i][0]) * by, (C::F32 ? acc[c + 1][k] : acc[i][1]) * by,
                        (C::F32 ? acc[c + 2][k] : acc[i][2]) * by, (C::F32 ? acc[c + 3][k] : acc[i][3]) * by};
    const int d = C::F32 ? dim_of<C>(c, 4 * g + k) : dim_of<C>(i, 4 * g);
    if (d < hd) __builtin_memcpy(o + d, x, sizeof x);
  }
}

// WHOLE: a block takes whole tiles of request blockIdx.y.
template <int T, int HDP, int CG, int KP, bool WHOLE>
__global__ __launch_bounds__((Cfg<T, HDP, CG, KP>::THREADS), 2) void k_tree_attn(TaArgs a) {
  using C = Cfg<T, HDP, CG, KP>;
  constexpr int SUB = C::SUB, KS = C::KS, STEP = C::STEP, DPL = C::DPL, U = C::U, CH = C::CH;
  extern __shared__ __align__(16) char lds[];
  long long *offs = reinterpret_cast<long long *>(lds + C::STAGEB);                 // [4][KP][KS]: where a key lies, -1 for nowhere
  uint64_t *gone = reinterpret_cast<uint64_t *>(lds + C::STAGEB + C::OFFB);         // [4][KP]: bits of keys that are nowhere
  float *scales = reinterpret_cast<float *>(lds + C::STAGEB + C::OFFB + C::GONEB);  // [2][k, v][KP][KS]
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int part = wave / CG, cg = wave % CG, tp = cg * 64 + lane;                  // tp: among the threads that stage the part
  const bool looks = cg == 0;                                                       // the wave that finds the part's keys

  const auto sync = [] {
    if constexpr (CG == 1) {            // a wave is alone with its part
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    } else {
      __syncthreads();
    }
  };
  // a request's new rows, tokens, column tiles of a KV head and steps of a tile
  int r = 0, first = 0, m = 0, len = 0, ct = 0, steps = 0;
  const auto request = [&](int x) {     // one for the wave
    m = __builtin_amdgcn_readfirstlane(rows_of(a, x, &first));
    first = __builtin_amdgcn_readfirstlane(first);
    len = __builtin_amdgcn_readfirstlane(clamp_len(a.lens[x], a.width, a.page_size));
    ct = (m * a.G + C::COLS - 1) / C::COLS;
    steps = (len + STEP - 1) / STEP;
  };

  long long u = 0, end = 0, share = 0;  // units from u up to end are this block's
  int tile = 0;                         // fits: the host has checked rows * n_heads
  int at = 0;                           // units of the tile that shares before this one take
  if constexpr (WHOLE) {
    r = blockIdx.y;
    request(r);
    tile = blockIdx.x;
    u = tile;
    end = ct * a.n_kv;
  } else {
    const auto units_of = [&](int x) -> long long {
      if (x >= a.n_req) return 0;
      int i0;
      const int rows = rows_of(a, x, &i0), tokens = clamp_len(a.lens[x], a.width, a.page_size);
      return tokens ? (long long)((rows * a.G + C::COLS - 1) / C::COLS) * a.n_kv * ((tokens + STEP - 1) / STEP + C::OVER) : 0;
    };
    long long upto = scan64(units_of(lane)), units = uniform(__shfl(upto, 63));            // of requests up to the lane's, 64 at a time
    for (int x = 64; x < a.n_req; x += 64) units += uniform(__shfl(scan64(units_of(x + lane)), 63));
    share = max((units + C::SHARES - 1) / C::SHARES, 2LL);      // one request of 2060 tokens: 27 us with 1, 22.5 with 2
    u = blockIdx.x * share;
    end = min(u + share, units);
    if (threadIdx.x == 0) a.split[blockIdx.x] = make_int4(0, 0, 0, 0);
    long long before = 0;               // units before the request
    for (; u < end; r += 64) {
      if (r) upto = scan64(units_of(r + lane));
      const uint64_t past = __ballot(before + upto > u);
      if (past) {
        const int at = __builtin_ctzll(past);
        if (at) before += uniform(__shfl(upto, at - 1));
        r += at;
        break;
      }
      before += uniform(__shfl(upto, 63));
    }
    if (u < end) {
      request(r);
      tile = (int)((u - before) / (steps + C::OVER));
      at = (int)(u - before - (long long)tile * (steps + C::OVER));
    }
  }
  const long long begin = u;
  const int step_e = STEP / a.page_size, step_p = STEP - step_e * a.page_size;

  while (u < end) {
    if constexpr (!WHOLE) {
      if (tile == ct * a.n_kv) {           // the next request that has rows and tokens
        do request(++r); while (ct == 0 || steps == 0);
        tile = 0;
      }
    }
    // a tile's first OVER units stand for what it takes beside its steps
    const int take = WHOLE ? 1 : (int)min(end - u, (long long)(steps + C::OVER - at));
    const int from = WHOLE ? 0 : max(at - C::OVER, 0), to = WHOLE ? steps : max(at + take - C::OVER, 0);
    if (!WHOLE && to == from) break;                  // the share ends before the tile's first step
    const int kvh = tile / ct, c0 = (tile - kvh * ct) * C::COLS;        // its first column
    const int cols = min(C::COLS, m * a.G - c0);
    const int ctx = max(len - m, 0);
    const int *table = a.table + r * a.table_stride;
    const char *kbase = a.k + kvh * a.hst, *vbase = a.v + kvh * a.hst;
    // without a mask nothing behind the tile's last row is seen
    int last = to;
    if (!a.mask) {
      const long long keys = (long long)ctx + (c0 + cols - 1) / a.G + 1;
      last = (int)min((long long)to, (keys + STEP - 1) / STEP);
    }

    // ---- finding and staging keys and values: in step s those of s + 1 are under way, the places of s + 2 are settled
    // and the table entries of s + 3 asked for
    // (every wave asks, so that nothing waits where the paths of the one that writes and the others meet)
    int key = from * STEP + part * KS + lane % KS, entry = key / a.page_size, place = key - entry * a.page_size;       // asked for next
    const int last_entry = len > 0 ? (len - 1) / a.page_size : 0;
    int page_at = 0, key_at = 0, place_at = 0;        // asked for: a table entry, its key and the key's place
    const auto ask = [&] {
      page_at = table[min(entry, last_entry)];        // there is a token
      key_at = key;
      place_at = place;
      key += STEP;
      entry += step_e;
      place += step_p;
      if (place >= a.page_size) { place -= a.page_size; entry++; }
    };
    const auto settle = [&](int s) -> long long {     // where the lane's scales lie
      const bool there = key_at < len && page_at >= 0 && page_at < a.n_pages;
      const long long off = there ? page_at * a.pst + place_at * a.sst : -1;
      const uint64_t no = __ballot(!there);
      if (looks) {
        if (lane < KS) offs[((s & 3) * KP + part) * KS + lane] = off;
        if (lane == 0) gone[(s & 3) * KP + part] = no;
      }
      return T == QLLAMA_KV_I8 ? (there ? page_at : 0) * a.scp + kvh * a.sch + (there ? place_at : 0) * a.scs : 0;
    };
    u4 staged[U * C::LOADS];
    uint32_t dead = 0;                                // units of no key, or of no dim
    constexpr int UNITS = KS * CH / C::CPU, PER = CH / C::CPU;                 // of a part's keys, of a row
    const auto issue = [&](int s) {
      dead = 0;
#pragma unroll
      for (int x = 0; x < U; x++) {
        const int unit = tp + x * C::TP, is_v = unit >= UNITS, at = is_v ? unit - UNITS : unit;
        const int row = at / PER, d = (at % PER) * C::EPC * C::CPU;
        const long long off = offs[((s & 3) * KP + part) * KS + row];
        const bool no = off < 0 || d >= a.hd;
        const char *p = (is_v ? vbase : kbase) + (no ? 0 : off + d * C::ES);
        if (no) dead |= 1u << x;
        if constexpr (T == QLLAMA_KV_I8) {
          const bool half = no || d + 8 >= a.hd;      // the row may end within the 16 codes
          if (half) dead |= 0x10000u << x;
          if (a.wide) {
            staged[x] = C::ONCE ? __builtin_nontemporal_load(reinterpret_cast<const u4 *>(p)) : *reinterpret_cast<const u4 *>(p);
          } else {
            const u2 lo = *reinterpret_cast<const u2 *>(p), hi = *reinterpret_cast<const u2 *>(half ? p : p + 8);
            staged[x] = u4{lo.x, lo.y, hi.x, hi.y};
          }
        } else {
#pragma unroll
          for (int i = 0; i < C::LOADS; i++) {
            const u4 *q = reinterpret_cast<const u4 *>(p) + i;
            staged[x * C::LOADS + i] = C::ONCE ? __builtin_nontemporal_load(q) : *q;
          }
        }
      }
    };
    uint32_t odd = 0;                                 // whether a new token's value was not finite
    const auto write = [&](int s) {
      const bool fresh = s * STEP + (part + 1) * KS > ctx;        // new tokens among the part's keys
      char *to_lds = lds + (C::NBUF == 1 ? part : (s & 1) * KP + part) * C::PARTB;
#pragma unroll
      for (int x = 0; x < U; x++) {
        const int unit = tp + x * C::TP, is_v = unit >= UNITS, at = is_v ? unit - UNITS : unit;
        const int row = at / PER, chunk = at % PER * C::CPU;
        char *to = to_lds + is_v * C::SIDEB + row * C::ROWB;
        if constexpr (T == QLLAMA_KV_I8) {            // bf16 holds a code
#pragma unroll
          for (int h = 0; h < 2; h++) {
            u4 w;
#pragma unroll
            for (int i = 0; i < 4; i++) {
              const uint32_t b = staged[x][2 * h + i / 2] >> (16 * (i % 2));
              w[i] = hi16s(__float_as_uint((float)(signed char)(b >> 8)), __float_as_uint((float)(signed char)b));
            }
            if (dead >> (x + 16 * h) & 1) w = u4{0, 0, 0, 0};
            *reinterpret_cast<u4 *>(to + (((chunk + h) ^ (row & C::SWZ)) << 4)) = w;
          }
        } else {
          u4 w[C::LOADS];
#pragma unroll
          for (int k = 0; k < C::LOADS; k++) {
            w[k] = staged[x * C::LOADS + k];
            if (dead >> x & 1) w[k] = u4{0, 0, 0, 0};
            if (fresh && is_v) {                      // what is not finite must not reach the columns that do not see it
#pragma unroll
              for (int i = 0; i < 4; i++) {
                const uint32_t all = w[k][i];
                if constexpr (C::ES == 4) {
                  w[k][i] = odd_value<T>(all) ? 0 : all;
                } else {
                  w[k][i] = (odd_value<T>(all & 0xffffu) ? 0 : all & 0xffffu) | (odd_value<T>(all >> 16) ? 0 : all & 0xffff0000u);
                }
                odd |= w[k][i] ^ all;
              }
            }
          }
          to += (chunk ^ (row & C::SWZ)) << 4;
          if constexpr (C::SPLIT) {
            float f[8];
#pragma unroll
            for (int i = 0; i < 8; i++) f[i] = __uint_as_float(w[i / 4][i % 4]);
            const Parts3 y = round3<true>(f);
#pragma unroll
            for (int k = 0; k < 3; k++) *reinterpret_cast<u4 *>(to + k * C::PLANEB) = y.p[k];
          } else {
            *reinterpret_cast<u4 *>(to) = w[0];
          }
        }
      }
    };
    const auto write_scales = [&](int s, float k, float v) {
      if (looks && lane < KS) {
        float *to = scales + ((s & 1) * 2 * KP + part) * KS + lane;
        to[0] = k;
        to[KP * KS] = v;
      }
    };

    // table entries, then the queries, then the first keys and values are under way; the queries are cut meanwhile
    const bool any = from < last, live = cg * 16 < cols;
    const int col = c0 + min(cg * 16 + n, cols - 1);  // the lane's column; those past the last repeat it
    const int row = first + col / a.G, head = kvh * a.G + col % a.G;
    constexpr int QE = C::F32 ? 4 : 8;
    float f[C::QC][QE];
    long long scale_at = 0, scale_next = 0;           // of the steps that are settled
    {
      int pages[2], keys[2], places[2];
      if (any) {
#pragma unroll
        for (int i = 0; i < 2; i++) {
          ask();
          pages[i] = page_at; keys[i] = key_at; places[i] = place_at;
        }
        ask();
      }
      const float *q = a.q + row * a.q_stride + (long long)head * a.hd;
#pragma unroll
      for (int c = 0; c < C::QC; c++) {
        const int d = 4 * QE * c + QE * g;
        __builtin_memcpy(f[c], q + (d < a.hd ? d : 0), sizeof f[c]);             // 4-byte aligned
      }
      if (any) {
        const int p2 = page_at, k2 = key_at, x2 = place_at;
        page_at = pages[0]; key_at = keys[0]; place_at = places[0];
        scale_at = settle(from);
        page_at = pages[1]; key_at = keys[1]; place_at = places[1];
        scale_next = settle(from + 1);
        page_at = p2; key_at = k2; place_at = x2;
      }
    }
    sync();
    float ks1 = 0.0f, vs1 = 0.0f;
    if (any) {
      issue(from);
      if constexpr (T == QLLAMA_KV_I8) {
        ks1 = a.ks[scale_at];
        vs1 = a.vs[scale_at];
      }
    }

    // the wave's queries, as parts of 16 bits
    u4 qp[C::QC][C::PARTS];
    float unscale = 1.0f, most = 0.0f;
#pragma unroll
    for (int c = 0; c < C::QC; c++)
#pragma unroll
      for (int e = 0; e < QE; e++) {
        f[c][e] = 4 * QE * c + QE * g < a.hd ? f[c][e] * a.qscale : 0.0f;
        most = fmaxf(most, fabsf(f[c][e]));
      }
    if constexpr (C::HALF) {                          // into f16's range, by a power of two
      most = max_groups(most);
      const int e = most > 0.0f && most < __builtin_inff() ? ilogbf(most) - 13 : 0;
      unscale = ldexpf(1.0f, e);
#pragma unroll
      for (int c = 0; c < C::QC; c++)
#pragma unroll
        for (int i = 0; i < QE; i++) f[c][i] = ldexpf(f[c][i], -e);
    }
#pragma unroll
    for (int c = 0; c < C::QC; c++) {
      if constexpr (C::F32) {
#pragma unroll
        for (int e = 0; e < QE; e++) qp[c][0][e] = __float_as_uint(f[c][e]);
      } else if constexpr (C::HALF) {
        const Parts2 y = cut2(f[c]);
#pragma unroll
        for (int p = 0; p < C::PARTS; p++) qp[c][p] = y.p[p];
      } else {
        const Parts3 y = C::SPLIT ? round3<true>(f[c]) : cut3(f[c]);
#pragma unroll
        for (int p = 0; p < C::PARTS; p++) qp[c][p] = y.p[p];
      }
    }

    float top = kNegInf, sum = 0.0f;                  // of the lane's column; sum over the lane's keys
    f4 acc[DPL];
#pragma unroll
    for (int c = 0; c < DPL; c++) acc[c] = f4{0, 0, 0, 0};

    // keys KEYS t .. of step s's part
    const auto compute = [&](int s, int t) {
      const char *kl = lds + (C::NBUF == 1 ? part : (s & 1) * KP + part) * C::PARTB + t * C::KEYS * C::ROWB, *vl = kl + C::SIDEB;
      const int key0 = s * STEP + part * KS + t * C::KEYS;
      f4 d[SUB];
#pragma unroll
      for (int i = 0; i < SUB; i++) d[i] = f4{0, 0, 0, 0};
#pragma unroll
      for (int y = C::PLANES - 1; y >= 0; y--) {      // the smallest products first: their sums round to less
        u4 kf[C::QC][SUB];
#pragma unroll
        for (int c = 0; c < C::QC; c++)
#pragma unroll
          for (int i = 0; i < SUB; i++)
            kf[c][i] = *reinterpret_cast<const u4 *>(kl + y * C::PLANEB + (16 * i + n) * C::ROWB + (((4 * c + g) ^ (n & C::SWZ)) << 4));
        __builtin_amdgcn_sched_barrier(0);            // all under way before the first product
#pragma unroll
        for (int c = 0; c < C::QC; c++)
#pragma unroll
          for (int i = 0; i < SUB; i++) {
            if constexpr (C::F32) {
#pragma unroll
              for (int e = 0; e < 4; e++)
                d[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kf[c][i][e]), __uint_as_float(qp[c][0][e]), d[i], 0, 0, 0);
            } else {
#pragma unroll
              for (int p = 0; p < C::PARTS - y; p++) d[i] = mfma16<C::LT>(kf[c][i], qp[c][C::SPLIT ? C::PARTS - 1 - y - p : p], d[i]);
            }
          }
      }

      f4 fv[SUB];
      if constexpr (T == QLLAMA_KV_I8) {
        const float *f = scales + ((s & 1) * 2 * KP + part) * KS + t * C::KEYS;
#pragma unroll
        for (int i = 0; i < SUB; i++) {
          d[i] *= *reinterpret_cast<const f4 *>(f + 16 * i + 4 * g);
          fv[i] = *reinterpret_cast<const f4 *>(f + KP * KS + 16 * i + 4 * g);
        }
      }
      if constexpr (C::HALF) {
#pragma unroll
        for (int i = 0; i < SUB; i++) d[i] *= unscale;
      }
      const uint32_t none = __builtin_amdgcn_readfirstlane((uint32_t)(gone[(s & 3) * KP + part] >> (t * C::KEYS)) & (C::KEYS == 32 ? ~0u : 0xffffu));
      uint32_t seen = ~0u;
      if (none != 0 || key0 + C::KEYS > ctx) {        // one for the wave
        seen = seen_of(a, row, row - first, key0 - ctx) & ~none;
#pragma unroll
        for (int i = 0; i < SUB; i++)
#pragma unroll
          for (int j = 0; j < 4; j++)
            if (!(seen >> (16 * i + 4 * g + j) & 1)) {
              d[i][j] = kNegInf;
              if constexpr (T == QLLAMA_KV_I8) fv[i][j] = 0.0f;          // whatever the scale is
            }
      }
      if constexpr (C::SPLIT) {
        // parts of an infinity, or whose products leave a float's range, give a NaN or an infinity for what may be none: such
        // scores one by one, for a column that is not NaN already
        float all = 0.0f;
#pragma unroll
        for (int i = 0; i < SUB; i++)
#pragma unroll
          for (int j = 0; j < 4; j++) all += d[i][j];
        if (__any(all - all != 0.0f && sum == sum)) {
          const float *q = a.q + row * a.q_stride + (long long)head * a.hd;
#pragma unroll
          for (int i = 0; i < SUB; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
              if (d[i][j] - d[i][j] == 0.0f || sum != sum || !(seen >> (16 * i + 4 * g + j) & 1)) continue;
              const float *k = reinterpret_cast<const float *>(kbase + offs[((s & 3) * KP + part) * KS + t * C::KEYS + 16 * i + 4 * g + j]);
              float x = 0.0f;
#pragma unroll 1
              for (int e = 0; e < a.hd; e += 8) {
                float y[8], z[8];
                __builtin_memcpy(y, q + e, sizeof y);
                __builtin_memcpy(z, k + e, sizeof z);
#pragma unroll
                for (int l = 0; l < 8; l++) x = fmaf(y[l] * a.qscale, z[l], x);
              }
              d[i][j] = x;
            }
        }
      }
      float up = d[0][0];
#pragma unroll
      for (int i = 0; i < SUB; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) up = fmaxf(up, d[i][j]);
      up = fmaxf(top, max_groups(up));
      if (__any(up > top)) {                          // rare after the first steps
        const float by = top == kNegInf ? 1.0f : __builtin_amdgcn_exp2f(top - up);     // without a maximum all is 0, or the NaN of its scores
        sum *= by;
#pragma unroll
        for (int c = 0; c < DPL; c++) acc[c] *= by;
        top = up;
      }
      const float ref = top == kNegInf ? 0.0f : top;
      u4 pp[C::PARTS];
      float p[4 * SUB];
#pragma unroll
      for (int i = 0; i < SUB; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
          float w = __builtin_amdgcn_exp2f(d[i][j] - ref);
          sum += w;
          if constexpr (T == QLLAMA_KV_I8) w *= fv[i][j];
          p[4 * i + j] = C::HALF ? w * C::RAISED : w;
        }
      if constexpr (C::HALF) {
        const Parts2 y = cut2(p);
#pragma unroll
        for (int k = 0; k < C::PARTS; k++) pp[k] = y.p[k];
      } else if constexpr (!C::F32) {
        const Parts3 y = C::SPLIT ? round3<false>(p) : cut3(p);
#pragma unroll
        for (int k = 0; k < C::PARTS; k++) pp[k] = y.p[k];
      }

      if constexpr (C::F32) {
#pragma unroll
        for (int y = 0; y < DPL / 4; y++)             // dims 64 y + 4 n .. of the lane's 4 keys
#pragma unroll
          for (int j = 0; j < 4; j++) {
            const f4 v = *reinterpret_cast<const f4 *>(vl + (4 * g + j) * C::ROWB + (((16 * y + n) ^ ((4 * g + j) & C::SWZ)) << 4));
#pragma unroll
            for (int c = 0; c < 4; c++) acc[4 * y + c] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[c], p[j], acc[4 * y + c], 0, 0, 0);
          }
      } else {
        // a transposing read: lane n of a group names row n / 4 and 4 dims of it, and gets dim n of the group's 4 keys
        const int row = 4 * g + n / 4;
        const char *at = vl + row * C::ROWB + n % 2 * 8;
        const int turn = (n % 4 / 2) ^ (row & C::SWZ);
#pragma unroll
        for (int c = 0; c < DPL; c++)
#pragma unroll
          for (int z = 0; z < C::PLANES; z++) {
            u4 vv;                                    // dim 16 c + n, 8 keys
#pragma unroll
            for (int i = 0; i < SUB; i++) {
              const u2 y = __builtin_bit_cast(
                  u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((s4_lds *)(at + z * C::PLANEB + 16 * i * C::ROWB + (((2 * c) ^ turn) << 4))));
              vv[2 * i] = y.x;
              vv[2 * i + 1] = y.y;
            }
#pragma unroll
            for (int k = 0; k < C::PARTS - z; k++) acc[c] = mfma16<C::LT>(vv, pp[k], acc[c]);
          }
      }
    };

    if (any) {
      write(from);
      if constexpr (T == QLLAMA_KV_I8) {
        write_scales(from, ks1, vs1);
      }
    }
    sync();
    for (int s = from; s < last; s++) {
      if (s + 1 < last) {
        // before the loads below: what this waits for is older than they
        if constexpr (T == QLLAMA_KV_I8) { ks1 = a.ks[scale_next]; vs1 = a.vs[scale_next]; }
        scale_next = settle(s + 2);
        ask();
        issue(s + 1);
      }
      if (live) {
#pragma unroll
        for (int t = 0; t < C::TIMES; t++) compute(s, t);
      }
      if (s + 1 < last) {
        write(s + 1);
        if constexpr (T == QLLAMA_KV_I8) {
          write_scales(s + 1, ks1, vs1);
        }
      }
      sync();
    }

    // ---- values of new tokens that are not finite: NaN where they are seen
    bool found = false;
    if constexpr (T != QLLAMA_KV_I8) found = CG == 1 ? __any(odd != 0) : __syncthreads_or(odd != 0);
    if (live && found) {
#pragma unroll 1
      for (int s = from; s < last; s++) {
        const int key0 = s * STEP + part * KS;
        if (key0 + KS <= ctx) continue;               // its values were taken as they are
#pragma unroll 1
        for (int k = key0; k < min(key0 + KS, len); k++) {
          const int page = table[k / a.page_size];
          if (page < 0 || page >= a.n_pages || !(seen_of(a, row, row - first, k - ctx) & 1)) continue;
          const char *v = vbase + page * a.pst + k % a.page_size * a.sst;
#pragma unroll
          for (int j = 0; j < 4; j++)
#pragma unroll
            for (int c = 0; c < DPL; c++) {
              const int d = dim_of<C>(c, 4 * g + j);
              if (d < a.hd && odd_value<T>(C::ES == 4 ? reinterpret_cast<const uint32_t *>(v)[d] : reinterpret_cast<const unsigned short *>(v)[d]))
                acc[c][j] = __builtin_nanf("");
            }
        }
      }
    }

    // ---- parts of the keys meet, two by two; the first part's waves hold the tile then
    sum = sum_groups(sum);
    if constexpr (KP > 1) {
      if constexpr (CG == 1) __syncthreads();
#pragma unroll
      for (int half = KP / 2; half; half /= 2) {
        if (part >= half && part < 2 * half && live) {
          char *at = lds + ((part - half) * CG + cg) * (DPL * 1024 + 512);
#pragma unroll
          for (int c = 0; c < DPL; c++) *reinterpret_cast<f4 *>(at + (c * 64 + lane) * 16) = acc[c];
          *reinterpret_cast<f2 *>(at + DPL * 1024 + lane * 8) = f2{top, sum};
        }
        __syncthreads();
        if (part < half && live) {
          const char *at = lds + (part * CG + cg) * (DPL * 1024 + 512);
          const f2 other = *reinterpret_cast<const f2 *>(at + DPL * 1024 + lane * 8);
          const float up = fmaxf(top, other.x), mine = part_weight(top, up), its = part_weight(other.x, up);
          sum = sum * mine + other.y * its;
          top = up;
#pragma unroll
          for (int c = 0; c < DPL; c++) acc[c] = acc[c] * mine + *reinterpret_cast<const f4 *>(at + (c * 64 + lane) * 16) * its;
        }
        __syncthreads();
      }
    }

    const bool whole = from == 0 && to == steps;
    if (part == 0 && live) {
      if (WHOLE || whole) {
        if (cg * 16 + n < cols) {
          put<C>(a.o + row * a.o_stride + (long long)head * a.hd, acc, g, a.hd, sum == 0.0f ? 0.0f : 1.0f / sum);
          if (g == 0 && a.lse) a.lse[row * a.lse_stride + head] = sum == 0.0f ? kNegInf : (top + __builtin_amdgcn_logf(sum)) * 0.69314718056f;
        }
      } else {
        float *o = a.part + ((long long)blockIdx.x * 2 + (u == begin ? 0 : 1)) * C::PARTF;
#pragma unroll
        for (int c = 0; c < DPL; c++) *reinterpret_cast<f4 *>(o + ((cg * DPL + c) * 64 + lane) * 4) = acc[c];
        if (g == 0) {
          o += CG * DPL * 256 + cg * 32 + n;
          o[0] = top;
          o[16] = sum;
        }
      }
    }
    if constexpr (WHOLE) {
      u += gridDim.x;
      tile = (int)u;
    } else {
      if (from == 0 && !whole && threadIdx.x == 0)    // the tile goes on in the shares behind this one
        a.split[blockIdx.x] = make_int4(1 + (int)((steps - to + share - 1) / share), r, tile, u == begin ? 0 : 1);
      u += take;
      at = 0;
      tile++;
    }
  }

  // requests without a token have no unit: their rows' outputs are set here
  if constexpr (!WHOLE) {
    for (int x = blockIdx.x; x < a.n_req; x += C::SHARES) {
      if (a.lens[x] > 0) continue;
      int i0;
      const int rows = rows_of(a, x, &i0), heads = a.n_kv * a.G;
      for (int i = i0; i < i0 + rows; i++)
        for (int d = threadIdx.x; d < heads * a.hd; d += C::THREADS) {
          a.o[i * a.o_stride + d] = 0.0f;
          if (a.lse && d < heads) a.lse[i * a.lse_stride + d] = kNegInf;
        }
    }
  }
}

// A block a share and 16 columns: where a tile begins in the share and goes on behind it, its
// parts are put together: a wave every fourth part in the order of their keys, then the
// four waves'.  Outputs leave through LDS in whole rows (in 4-byte pieces straight from the
// lanes that hold them the join took 40 us of 99, 32 requests with trees of up to 16 rows).
template <int T, int HDP, int CG>
__global__ __launch_bounds__(256) void k_tree_join(TaArgs a) {
  using C = Cfg<T, HDP, CG, 1>;
  constexpr int DPL = C::DPL, ROW = HDP + 4;
  __shared__ __align__(16) float hand[2][DPL * 256 + 128];
  const int4 s = a.split[blockIdx.x];
  const int parts = s.x, r = s.y, block = blockIdx.y;
  if (!parts) return;
  int first;
  const int m = rows_of(a, r, &first), ct = (m * a.G + C::COLS - 1) / C::COLS;
  const int kvh = s.z / ct, c0 = (s.z - kvh * ct) * C::COLS + block * 16, cols = min(16, m * a.G - c0);
  if (cols <= 0) return;
  const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4, w = threadIdx.x >> 6;
  const int stat = CG * DPL * 256 + block * 32 + n;
  float top = kNegInf, sum = 0.0f;
  f4 acc[DPL];
#pragma unroll
  for (int c = 0; c < DPL; c++) acc[c] = f4{0, 0, 0, 0};
#pragma unroll 4
  for (int i = w; i < parts; i += 4) {
    // the first part may follow another tile's in its share
    const float *p = a.part + (2LL * (blockIdx.x + i) + (i ? 0 : s.w)) * C::PARTF;
    const float its_top = p[stat], its_sum = p[stat + 16];
    f4 x[DPL];
#pragma unroll
    for (int c = 0; c < DPL; c++) x[c] = *reinterpret_cast<const f4 *>(p + ((block * DPL + c) * 64 + lane) * 4);
    const float up = fmaxf(top, its_top), mine = part_weight(top, up), its = part_weight(its_top, up);
    sum = sum * mine + its_sum * its;
    top = up;
#pragma unroll
    for (int c = 0; c < DPL; c++) acc[c] = acc[c] * mine + x[c] * its;
  }
#pragma unroll
  for (int half = 2; half; half /= 2) {
    if (w >= half && w < 2 * half) {
#pragma unroll
      for (int c = 0; c < DPL; c++) *reinterpret_cast<f4 *>(hand[w - half] + (c * 64 + lane) * 4) = acc[c];
      *reinterpret_cast<f2 *>(hand[w - half] + DPL * 256 + lane * 2) = f2{top, sum};
    }
    __syncthreads();
    if (w < half) {
      const f2 other = *reinterpret_cast<const f2 *>(hand[w] + DPL * 256 + lane * 2);
      const float up = fmaxf(top, other.x), mine = part_weight(top, up), its = part_weight(other.x, up);
      sum = sum * mine + other.y * its;
      top = up;
#pragma unroll
      for (int c = 0; c < DPL; c++) acc[c] = acc[c] * mine + *reinterpret_cast<const f4 *>(hand[w] + (c * 64 + lane) * 4) * its;
    }
    __syncthreads();
  }
  float *rows = hand[0];
  static_assert(16 * ROW <= 2 * (DPL * 256 + 128), "rows in LDS");
  if (w == 0) {
    put<C>(rows + n * ROW, acc, g, HDP, sum == 0.0f ? 0.0f : 1.0f / sum);
    if (g == 0 && a.lse && n < cols) {
      const int row = (c0 + n) / a.G;
      a.lse[(first + row) * a.lse_stride + kvh * a.G + c0 + n - row * a.G] = sum == 0.0f ? kNegInf : (top + __builtin_amdgcn_logf(sum)) * 0.69314718056f;
    }
  }
  __syncthreads();
  constexpr int PER = HDP / 4;                        // threads of a row
  const int d = threadIdx.x % PER * 4;
  if (d < a.hd) {
    for (int x = threadIdx.x / PER; x < cols; x += 256 / PER) {
      const int row = (c0 + x) / a.G, head = kvh * a.G + c0 + x - row * a.G;
      __builtin_memcpy(a.o + (first + row) * a.o_stride + (long long)head * a.hd + d, rows + x * ROW + d, 16);
    }
  }
}

template <int T, int HDP, int CG>
int launch(const char *fn, const TaArgs &a, hipStream_t stream) {
  constexpr int KP = CG >= 4 ? 1 : 4 / CG;            // parts of a step's keys where a block takes whole tiles
  using W = Cfg<T, HDP, CG, KP>;
  using C = Cfg<T, HDP, CG, 1>;
  static_assert(W::LDSB <= 160 * 1024 && C::LDSB <= 160 * 1024, "LDS");
  const long long room = ((long long)a.width * a.page_size + W::STEP - 1) / W::STEP;
  const long long tiles = ((long long)a.rows * a.G / W::COLS + a.n_req) * a.n_kv;
  // Whole tiles where their steps are few, more where there are tiles for all CUs.  Against shares, us (8 KV heads, hd 128):
  // 16 bf16 requests of up to 300 tokens and 8 rows 16.6 / 21.3, 32 of 500 and 16 rows 30.7 / 34.9, 2 int8 ones of 100 and
  // 10 rows 10.8 / 14.3; few tiles of more steps the other way: 4 of 450 and 16 rows 27.6 / 19.2, one f32 request of 200
  // tokens, 2 KV heads of 48, 13.8 / 12.2
  const bool whole = room <= (tiles >= 256 ? 16 : tiles >= 128 ? 8 : 4) && a.n_req <= 65535;
  void (*f)(TaArgs) = whole ? k_tree_attn<T, HDP, CG, KP, true> : k_tree_attn<T, HDP, CG, 1, false>;
  const int lds = whole ? W::LDSB : C::LDSB;
  if (lds > 64 * 1024 &&              // past what a launch may take unasked
      hipFuncSetAttribute(reinterpret_cast<const void *>(f), hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess) {
    (void)hipGetLastError();
    return qs::refuse(fn, "hipFuncSetAttribute failed");
  }
  if (whole) {
    const long long each = ((long long)a.rows * a.G / a.n_req + W::COLS - 1) / W::COLS;       // column tiles of a request, about
    const long long x = each < 1 ? a.n_kv : each * a.n_kv;
    QS_LAUNCH(fn, f, dim3((unsigned)(x < 65535 ? x : 65535), a.n_req), dim3(W::THREADS), lds, stream, a);
    return 0;
  }
  QS_LAUNCH(fn, f, dim3(C::SHARES), dim3(C::THREADS), lds, stream, a);
  QS_LAUNCH(fn, (k_tree_join<T, HDP, CG>), dim3(C::SHARES, CG), dim3(256), 0, stream, a);
  return 0;
}

template <int T, int HDP>
int launch_tile(const char *fn, const TaArgs &a, int tile, hipStream_t stream) {
  if constexpr (HDP == 256) return tile == 2 ? launch<T, HDP, 4>(fn, a, stream) : launch<T, HDP, 8>(fn, a, stream);
  else {
    switch (tile) {
      case 0: return launch<T, HDP, 1>(fn, a, stream);
      case 1: return launch<T, HDP, 2>(fn, a, stream);
      case 2:
        if constexpr (T != QLLAMA_KV_F32 || HDP != 128) return launch<T, HDP, 4>(fn, a, stream);       // f32: pick() takes 128 columns
      default: return launch<T, HDP, 8>(fn, a, stream);
    }
  }
}

template <int T>
int launch_hd(const char *fn, const TaArgs &a, int tile, hipStream_t stream) {
  return a.hd <= 64 ? launch_tile<T, 64>(fn, a, tile, stream) : a.hd <= 128 ? launch_tile<T, 128>(fn, a, tile, stream) : launch_tile<T, 256>(fn, a, tile, stream);
}

}  // namespace
#endif

#endif
