// qdev_tattn.h - attention of several new tokens a request over a paged key-value cache, with
// a mask among the new ones (qllama_tree_attention; semantics in qserve.h): the kernels, of
// which k_tattn_f32.hip, k_tattn_f16.hip, k_tattn_bf16.hip and k_tattn_i8.hip each compile a
// cache type's.  No counterpart in the reference, whose decode attention
// (llama.c:554-576) serves one token.
//
// The columns of a (request, KV head) are its rows times the query heads that share the KV
// head; a tile is up to COLS of them, and takes every key and value of the request
// through LDS once.  Eight waves: CG groups of columns, and KP = 8 / CG parts of a step's
// keys, so that few columns leave every wave a part of the keys to itself, and many share
// what was staged.  S^T = K q^T on the matrix cores puts a column in a lane's column and 4
// keys of each 16 in its rows; the same lane's weights are then the operand of
// O^T += V^T P^T, whose contraction slots are matched to the keys that the lane holds, so
// weights never move between lanes.
//
// The work of a call is the key steps of all tiles, laid one behind another; every block
// takes an equal share of them, whatever the lengths are, without the host knowing one.  A
// share that ends inside a tile leaves its maxima, sums and weighted values in the
// workspace, and k_tree_join puts a tile's parts together.  Where the tables are short a
// block takes whole tiles, and there is no second launch.
#ifndef QDEV_TATTN_H
#define QDEV_TATTN_H

#include <hip/hip_runtime.h>

#include "qdev_paged.h"
#include "qserve_host.h"

namespace qtree {

constexpr int kShares = 512;          // two blocks a CU; of eight waves, one

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


// What a type, a padded head size, 16-column groups of a wave and waves side by side fix.
template <int T, int HDP, int NC_, int CG_>
struct Cfg {
  static constexpr int NC = NC_, CG = CG_, WAVES = CG == 8 ? 8 : 4, THREADS = 64 * WAVES, KP = WAVES / CG, COLS = 16 * NC * CG;
  static constexpr int SHARES = kShares * 4 / WAVES;
  static constexpr int OVER = CG >= 4 ? 4 : 2;                          // steps that a tile's beginning and end take the time of
  static constexpr bool F32 = T == QLLAMA_KV_F32, HALF = T == QLLAMA_KV_F16;
  static constexpr int ES = F32 ? 4 : T == QLLAMA_KV_I8 ? 1 : 2;        // of an element in the cache
  static constexpr int LES = F32 ? 4 : 2;                               // in LDS (int8: bf16, which holds the codes)
  static constexpr int LT = T == QLLAMA_KV_I8 ? QLLAMA_KV_BF16 : T;     // the products' type
  static constexpr int SUB = F32 ? 1 : 2, KS = 16 * SUB, STEP = KS * KP;      // keys of a wave's step and of a block's
  static constexpr int ROWB = HDP * LES, CH = ROWB / 16, SWZ = (CH < 16 ? CH : 16) - 1, EPC = 16 / LES;
  static constexpr int PARTB = 2 * KS * ROWB;                           // a part's keys, then values
  static constexpr int NBUF = CG == 1 ? 1 : 2;                          // a wave alone with its part needs no second buffer
  static constexpr int TP = 64 * CG, U = 2 * KS * CH / TP;              // threads that stage a part, 16-byte units of each
  static constexpr int DPL = HDP / 16, QC = F32 ? HDP / 16 : HDP / 32;
  static constexpr int PARTS = F32 ? 1 : HALF ? 2 : 3;
  // a value row in LDS: piece x of lane (n, g) takes dims 16 PD x + PD n .. of key 4 g + j
  static constexpr int PB = 4 * LES, PD = PB / LES, PIECES = HDP / (16 * PD), PW = PB / 4;
  // weights are held times this in f16 products: two parts then keep 23 bits down to 2^-17 of the largest and the rest to 2^-40
  static constexpr float RAISED = HALF ? 32768.0f : 1.0f;
  // LDS: staged parts (and what waves hand over at a tile's end), places of the keys, scales, absent keys
  static constexpr int HANDB = (KP / 2) * CG * NC * (DPL * 1024 + 512);
  static constexpr int STAGEB = NBUF * KP * PARTB > HANDB ? NBUF * KP * PARTB : HANDB;
  static constexpr int OFFB = 4 * KP * KS * 8, SCALEB = T == QLLAMA_KV_I8 ? 2 * 2 * KP * KS * 4 : 0;
  static constexpr int LDSB = STAGEB + OFFB + SCALEB + 4 * KP * 4;
  static constexpr int PARTF = CG * NC * (DPL * 256 + 32);              // floats of a tile's part in the workspace
};

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

// The dim of a head whose output is element c of an accumulator's row `lane` of 16.
template <typename C>
__device__ inline int dim_of(int c, int lane) { return 16 * C::PD * (c / C::PD) + C::PD * lane + c % C::PD; }

// A column's outputs from what a lane holds: dims c mod PD of the piece of lane 4 g + i.
template <typename C>
__device__ inline void put(float *o, const f4 (&acc)[C::DPL], int g, int hd, float by) {
  by *= 1.0f / C::RAISED;
#pragma unroll
  for (int i = 0; i < 4; i++)
#pragma unroll
    for (int c = 0; c < C::DPL; c += 4) {
      const float x[4] = {acc[c][i] * by, acc[c + 1][i] * by, acc[c + 2][i] * by, acc[c + 3][i] * by};
      const int d = dim_of<C>(c, 4 * g + i);
      if (d < hd) __builtin_memcpy(o + d, x, sizeof x);
    }
}

// WHOLE: a block takes whole tiles of request blockIdx.y.
template <int T, int HDP, int NC, int CG, bool WHOLE>
__global__ __launch_bounds__((Cfg<T, HDP, NC, CG>::THREADS), 2) void k_tree_attn(TaArgs a) {
  using C = Cfg<T, HDP, NC, CG>;
  constexpr int SUB = C::SUB, KS = C::KS, STEP = C::STEP, DPL = C::DPL, U = C::U, CH = C::CH, KP = C::KP;
  extern __shared__ __align__(16) char lds[];
  long long *offs = reinterpret_cast<long long *>(lds + C::STAGEB);                 // [4][KP][KS]: where a key lies, -1 for nowhere
  float *scales = reinterpret_cast<float *>(lds + C::STAGEB + C::OFFB);             // [2][k, v][KP][KS]
  uint32_t *gone = reinterpret_cast<uint32_t *>(lds + C::STAGEB + C::OFFB + C::SCALEB);       // [4][KP]: bits of keys that are nowhere
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

  long long u = 0, end = 0, share = 0, tile = 0;
  int at = 0;                           // units of the tile that shares before this one take
  if constexpr (WHOLE) {
    r = blockIdx.y;
    request(r);
    tile = blockIdx.x;
    u = tile;
    end = (long long)ct * a.n_kv;
  } else {
    const auto units_of = [&](int x) -> long long {
      if (x >= a.n_req) return 0;
      int i0;
      const int rows = rows_of(a, x, &i0), tokens = clamp_len(a.lens[x], a.width, a.page_size);
      return tokens ? (long long)((rows * a.G + C::COLS - 1) / C::COLS) * a.n_kv * ((tokens + STEP - 1) / STEP + C::OVER) : 0;
    };
    long long upto = scan64(units_of(lane)), units = __shfl(upto, 63);
    for (int x = 64; x < a.n_req; x += 64) units += __shfl(scan64(units_of(x + lane)), 63);
    units = uniform(units);
    share = (units + C::SHARES - 1) / C::SHARES;
    u = blockIdx.x * share;
    end = u + share < units ? u + share : units;
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
      tile = (u - before) / (steps + C::OVER);
      at = (int)(u - before - tile * (steps + C::OVER));
    }
  }
  const long long begin = u;
  const int step_e = STEP / a.page_size, step_p = STEP - step_e * a.page_size;

  while (u < end) {
    if constexpr (!WHOLE) {
      if (tile == (long long)ct * a.n_kv) {           // the next request that has rows and tokens
        do request(++r); while (ct == 0 || steps == 0);
        tile = 0;
      }
    }
    // a tile's first OVER units stand for what it takes beside its steps
    const int take = WHOLE ? 1 : (int)min(end - u, (long long)(steps + C::OVER - at));
    const int from = WHOLE ? 0 : max(at - C::OVER, 0), to = WHOLE ? steps : max(at + take - C::OVER, 0);
    if (!WHOLE && to == from) break;                  // the share ends before the tile's first step
    const int kvh = (int)(tile / ct), c0 = (int)(tile - (long long)kvh * ct) * C::COLS;        // its first column
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

    // ---- finding and staging keys and values
    int entry = 0, place = 0, key = 0;                // of the lane's key in the step that is looked for next
    if (looks) {
      key = from * STEP + part * KS + (lane & (KS - 1));
      entry = key / a.page_size;
      place = key - entry * a.page_size;
    }
    const int last_entry = len > 0 ? (len - 1) / a.page_size : 0;
    const auto look = [&](int ahead) -> int {         // the table entry of the step that is settled next, or the one behind it
      const int e = ahead ? entry + step_e + (place + step_p >= a.page_size) : entry;
      return len > 0 ? table[min(e, last_entry)] : -1;
    };
    int page1 = 0, place1 = 0, page1_a = 0, place1_a = 0;       // where the scales of the lane's key lie, of the step settled last and the first
    const auto settle = [&](int s, int page) {
      const bool there = key < len && page >= 0 && page < a.n_pages;
      if (lane < KS) offs[((s & 3) * KP + part) * KS + lane] = there ? page * a.pst + place * a.sst : -1;
      const uint64_t no = __ballot(!there);
      if (lane == 0) gone[(s & 3) * KP + part] = (uint32_t)no & (KS == 32 ? ~0u : 0xffffu);
      page1 = there ? page : 0;
      place1 = there ? place : 0;
      key += STEP;
      entry += step_e;
      place += step_p;
      if (place >= a.page_size) { place -= a.page_size; entry++; }
    };
    u4 staged[U];
    uint32_t dead = 0;                                // units of no key, or of no dim
    float ks1 = 0.0f, vs1 = 0.0f;
    const auto issue = [&](int s, int scale_page, int scale_place) {
      dead = 0;
#pragma unroll
      for (int x = 0; x < U; x++) {
        const int unit = tp + x * C::TP, is_v = unit >= KS * CH, at = is_v ? unit - KS * CH : unit;
        const int row = at / CH, d = (at % CH) * C::EPC;
        const long long off = offs[((s & 3) * KP + part) * KS + row];
        const bool no = off < 0 || d >= a.hd;
        const char *p = (is_v ? vbase : kbase) + (no ? 0 : off + d * C::ES);
        if (no) dead |= 1u << x;
        if constexpr (T == QLLAMA_KV_I8) {
          const u2 w = *reinterpret_cast<const u2 *>(p);
          staged[x][0] = w.x;
          staged[x][1] = w.y;
        } else {
          staged[x] = *reinterpret_cast<const u4 *>(p);
        }
      }
      if constexpr (T == QLLAMA_KV_I8) {
        if (looks) {
          const long long at = scale_page * a.scp + kvh * a.sch + scale_place * a.scs;
          ks1 = a.ks[at];
          vs1 = a.vs[at];
        }
      }
    };
    const auto write = [&](int s) {
      char *to_lds = lds + (C::NBUF == 1 ? part : (s & 1) * KP + part) * C::PARTB;
#pragma unroll
      for (int x = 0; x < U; x++) {
        const int unit = tp + x * C::TP, is_v = unit >= KS * CH, at = is_v ? unit - KS * CH : unit;
        const int row = at / CH, chunk = at % CH;
        u4 w = staged[x];
        if constexpr (T == QLLAMA_KV_I8) {            // bf16 holds a code
          const uint32_t b[2] = {w[0], w[1]};
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const int b0 = (int)(b[i / 2] << (24 - 16 * (i % 2))) >> 24, b1 = (int)(b[i / 2] << (16 - 16 * (i % 2))) >> 24;
            w[i] = hi16s(__float_as_uint((float)b1), __float_as_uint((float)b0));
          }
        }
        if (dead >> x & 1) w = u4{0, 0, 0, 0};
        *reinterpret_cast<u4 *>(to_lds + is_v * KS * C::ROWB + row * C::ROWB + ((chunk ^ (row & C::SWZ)) << 4)) = w;
      }
      if constexpr (T == QLLAMA_KV_I8) {
        if (looks && lane < KS) {
          float *to = scales + ((s & 1) * 2 * KP + part) * KS + lane;
          to[0] = ks1;
          to[KP * KS] = vs1;
        }
      }
    };

    // both table entries, then the queries, then the first keys and values are under way; the queries are cut meanwhile
    const bool any = from < last, live = cg * 16 * NC < cols;
    const auto col_of = [&](int x) -> int { return c0 + min(cg * 16 * NC + 16 * x + n, cols - 1); };         // columns past the last repeat it
    const auto row_of = [&](int x) -> int { return col_of(x) / a.G; };
    const auto head_of = [&](int x) -> int { return kvh * a.G + col_of(x) % a.G; };
    int page_a = -1, page_b = -1;
    if (any && looks) {
      page_a = look(0);
      page_b = look(1);
    }
    constexpr int QE = C::F32 ? 4 : 8;
    float f[NC][C::QC][QE];
#pragma unroll
    for (int x = 0; x < NC; x++) {
      const float *q = a.q + (first + row_of(x)) * a.q_stride + (long long)head_of(x) * a.hd;
#pragma unroll
      for (int c = 0; c < C::QC; c++) {
        const int d = 4 * QE * c + QE * g;
        __builtin_memcpy(f[x][c], q + (d < a.hd ? d : 0), sizeof f[x][c]);       // 4-byte aligned
      }
    }
    if (any && looks) {
      settle(from, page_a);
      page1_a = page1; place1_a = place1;
      settle(from + 1, page_b);
    }
    sync();
    if (any) issue(from, page1_a, place1_a);

    // the wave's queries, as parts of 16 bits
    u4 qp[NC][C::QC][C::PARTS];
    float unscale[NC];
#pragma unroll
    for (int x = 0; x < NC; x++) {
      unscale[x] = 1.0f;
      float most = 0.0f;
#pragma unroll
      for (int c = 0; c < C::QC; c++)
#pragma unroll
        for (int e = 0; e < QE; e++) {
          f[x][c][e] = 4 * QE * c + QE * g < a.hd ? f[x][c][e] * a.qscale : 0.0f;
          most = fmaxf(most, fabsf(f[x][c][e]));
        }
      if constexpr (C::HALF) {                        // into f16's range, by a power of two
        most = max_groups(most);
        const int e = most > 0.0f && most < __builtin_inff() ? ilogbf(most) - 13 : 0;
        unscale[x] = ldexpf(1.0f, e);
#pragma unroll
        for (int c = 0; c < C::QC; c++)
#pragma unroll
          for (int i = 0; i < QE; i++) f[x][c][i] = ldexpf(f[x][c][i], -e);
      }
#pragma unroll
      for (int c = 0; c < C::QC; c++) {
        if constexpr (C::F32) {
#pragma unroll
          for (int e = 0; e < QE; e++) qp[x][c][0][e] = __float_as_uint(f[x][c][e]);
        } else if constexpr (C::HALF) {
          const Parts2 y = cut2(f[x][c]);
#pragma unroll
          for (int p = 0; p < C::PARTS; p++) qp[x][c][p] = y.p[p];
        } else {
          const Parts3 y = cut3(f[x][c]);
#pragma unroll
          for (int p = 0; p < C::PARTS; p++) qp[x][c][p] = y.p[p];
        }
      }
    }

    float top[NC], sum[NC];                           // of the lane's columns; sum over the lane's keys
    f4 acc[NC][DPL];
#pragma unroll
    for (int x = 0; x < NC; x++) {
      top[x] = kNegInf;
      sum[x] = 0.0f;
#pragma unroll
      for (int c = 0; c < DPL; c++) acc[x][c] = f4{0, 0, 0, 0};
    }

    bool odd = false;                                 // a new token's value was not finite
    const auto compute = [&](int s) {
      const char *kl = lds + (C::NBUF == 1 ? part : (s & 1) * KP + part) * C::PARTB, *vl = kl + KS * C::ROWB;
      const int key0 = s * STEP + part * KS;
      f4 d[NC][SUB];
#pragma unroll
      for (int x = 0; x < NC; x++)
#pragma unroll
        for (int i = 0; i < SUB; i++) d[x][i] = f4{0, 0, 0, 0};
#pragma unroll
      for (int c = 0; c < C::QC; c++)
#pragma unroll
        for (int i = 0; i < SUB; i++) {
          const u4 kk = *reinterpret_cast<const u4 *>(kl + (16 * i + n) * C::ROWB + (((4 * c + g) ^ (n & C::SWZ)) << 4));
#pragma unroll
          for (int x = 0; x < NC; x++) {
            if constexpr (C::F32) {
#pragma unroll
              for (int e = 0; e < 4; e++)
                d[x][i] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kk[e]), __uint_as_float(qp[x][c][0][e]), d[x][i], 0, 0, 0);
            } else {
#pragma unroll
              for (int p = 0; p < C::PARTS; p++) d[x][i] = mfma16<C::LT>(kk, qp[x][c][p], d[x][i]);
            }
          }
        }

      f4 fk[SUB], fv[SUB];
      if constexpr (T == QLLAMA_KV_I8) {
        const float *f = scales + ((s & 1) * 2 * KP + part) * KS;
#pragma unroll
        for (int i = 0; i < SUB; i++) {
          fk[i] = *reinterpret_cast<const f4 *>(f + 16 * i + 4 * g);
          fv[i] = *reinterpret_cast<const f4 *>(f + KP * KS + 16 * i + 4 * g);
        }
      }
#pragma unroll
      for (int x = 0; x < NC; x++)
#pragma unroll
        for (int i = 0; i < SUB; i++) {
          if constexpr (C::HALF) d[x][i] *= unscale[x];
          if constexpr (T == QLLAMA_KV_I8) d[x][i] *= fk[i];
        }

      const uint32_t none = __builtin_amdgcn_readfirstlane(gone[(s & 3) * KP + part]);
      const bool masked = none != 0 || key0 + KS > ctx;          // one for the wave
      uint32_t seen[NC];
      if (masked) {
#pragma unroll
        for (int x = 0; x < NC; x++) {
          seen[x] = seen_of(a, first + row_of(x), row_of(x), key0 - ctx) & ~none;
#pragma unroll
          for (int i = 0; i < SUB; i++)
#pragma unroll
            for (int j = 0; j < 4; j++)
              if (!(seen[x] >> (16 * i + 4 * g + j) & 1)) d[x][i][j] = kNegInf;
        }
      }

      float up[NC];
      bool more = false;
#pragma unroll
      for (int x = 0; x < NC; x++) {
        up[x] = d[x][0][0];
#pragma unroll
        for (int i = 0; i < SUB; i++)
#pragma unroll
          for (int j = 0; j < 4; j++) up[x] = fmaxf(up[x], d[x][i][j]);
        up[x] = fmaxf(top[x], max_groups(up[x]));
        more |= up[x] > top[x];
      }
      if (__any(more)) {                              // rare after the first steps
#pragma unroll
        for (int x = 0; x < NC; x++) {
          const float by = top[x] == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(top[x] - up[x]);
          sum[x] *= top[x] == kNegInf ? 1.0f : by;    // a sum without a maximum is 0, or the NaN of its scores
#pragma unroll
          for (int c = 0; c < DPL; c++) acc[x][c] *= top[x] == kNegInf ? 1.0f : by;
          top[x] = up[x];
        }
      }
      u4 pp[NC][C::PARTS];
      float p32[NC][4];
#pragma unroll
      for (int x = 0; x < NC; x++) {
        const float ref = top[x] == kNegInf ? 0.0f : top[x];
        float p[8];
#pragma unroll
        for (int i = 0; i < SUB; i++)
#pragma unroll
          for (int j = 0; j < 4; j++) {
            float w = __builtin_amdgcn_exp2f(d[x][i][j] - ref);
            sum[x] += w;
            if constexpr (T == QLLAMA_KV_I8) {
              w *= fv[i][j];
              if (masked && !(seen[x] >> (16 * i + 4 * g + j) & 1)) w = 0.0f;        // whatever the scale is
            }
            if constexpr (C::F32) p32[x][j] = w;
            else p[4 * i + j] = w * C::RAISED;
          }
        if constexpr (C::HALF) {
          const Parts2 y = cut2(p);
#pragma unroll
          for (int k = 0; k < C::PARTS; k++) pp[x][k] = y.p[k];
        } else if constexpr (!C::F32) {
          const Parts3 y = cut3(p);
#pragma unroll
          for (int k = 0; k < C::PARTS; k++) pp[x][k] = y.p[k];
        }
      }

      const bool fresh = T != QLLAMA_KV_I8 && key0 + KS > ctx && key0 < len;        // new tokens among the keys
#pragma unroll
      for (int y = 0; y < C::PIECES; y++) {
        uint32_t v[SUB][4][C::PW];
#pragma unroll
        for (int i = 0; i < SUB; i++)
#pragma unroll
          for (int j = 0; j < 4; j++) {
            const int byte = C::PB * (16 * y + n), row = 16 * i + 4 * g + j;
            __builtin_memcpy(v[i][j], __builtin_assume_aligned(vl + row * C::ROWB + (((byte >> 4) ^ ((4 * g + j) & C::SWZ)) << 4) + (byte & 15), C::PB), C::PB);
          }
        if (fresh) {                                  // what is not finite must not reach the columns that do not see it
#pragma unroll
          for (int i = 0; i < SUB; i++)
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
              for (int w = 0; w < C::PW; w++) {
                uint32_t &x = v[i][j][w];
                if constexpr (C::F32) {
                  if (odd_value<T>(x)) { x = 0; odd = true; }
                } else {
                  if (odd_value<T>(x & 0xffffu)) { x &= 0xffff0000u; odd = true; }
                  if (odd_value<T>(x >> 16)) { x &= 0xffffu; odd = true; }
                }
              }
        }
#pragma unroll
        for (int c = 0; c < C::PD; c++) {
          const int at = y * C::PD + c;
          if constexpr (C::F32) {
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
              for (int x = 0; x < NC; x++)
                acc[x][at] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(v[0][j][c]), p32[x][j], acc[x][at], 0, 0, 0);
          } else {
            u4 vv;                                    // dim c of the lane's piece, 8 keys
#pragma unroll
            for (int i = 0; i < SUB; i++)
#pragma unroll
              for (int j = 0; j < 2; j++) {
                const uint32_t lo = v[i][2 * j][c / 2], hi = v[i][2 * j + 1][c / 2];
                vv[2 * i + j] = c % 2 ? hi16s(hi, lo) : lo16s(hi, lo);
              }
#pragma unroll
            for (int x = 0; x < NC; x++)
#pragma unroll
              for (int k = 0; k < C::PARTS; k++) acc[x][at] = mfma16<C::LT>(vv, pp[x][k], acc[x][at]);
          }
        }
      }
    };

    if (any) write(from);
    sync();
    for (int s = from; s < last; s++) {
      int page = 0;
      if (s + 1 < last) {
        issue(s + 1, page1, place1);
        if (looks) page = look(0);                    // of step s + 2
      }
      if (live) compute(s);
      if (s + 1 < last) {
        if (looks) settle(s + 2, page);
        write(s + 1);
      }
      sync();
    }

    // ---- values of new tokens that are not finite: NaN where they are seen
    if (live && __any(odd)) {
#pragma unroll 1
      for (int s = from; s < last; s++) {
        const int key0 = s * STEP + part * KS;
#pragma unroll 1
        for (int k = max(key0, ctx); k < min(key0 + KS, len); k++) {
          const int page = table[k / a.page_size];
          if (page < 0 || page >= a.n_pages) continue;
          const char *v = vbase + page * a.pst + k % a.page_size * a.sst;
#pragma unroll
          for (int x = 0; x < NC; x++) {
            const int i = row_of(x);
            if (!(seen_of(a, first + i, i, k - ctx) & 1)) continue;
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
              for (int c = 0; c < DPL; c++) {
                const int d = dim_of<C>(c, 4 * g + j);
                if (d < a.hd && odd_value<T>(C::F32 ? reinterpret_cast<const uint32_t *>(v)[d] : reinterpret_cast<const unsigned short *>(v)[d]))
                  acc[x][c][j] = __builtin_nanf("");
              }
          }
        }
      }
    }

    // ---- parts of the keys meet, two by two; the first part's waves hold the tile then
#pragma unroll
    for (int x = 0; x < NC; x++) sum[x] = sum_groups(sum[x]);
    if constexpr (KP > 1) {
      if constexpr (CG == 1) __syncthreads();
#pragma unroll
      for (int half = KP / 2; half; half /= 2) {
        if (part >= half && part < 2 * half && live) {
          char *at = lds + ((part - half) * CG + cg) * (NC * (DPL * 1024 + 512));
#pragma unroll
          for (int x = 0; x < NC; x++) {
#pragma unroll
            for (int c = 0; c < DPL; c++) *reinterpret_cast<f4 *>(at + ((x * DPL + c) * 64 + lane) * 16) = acc[x][c];
            *reinterpret_cast<f2 *>(at + NC * DPL * 1024 + (x * 64 + lane) * 8) = f2{top[x], sum[x]};
          }
        }
        __syncthreads();
        if (part < half && live) {
          const char *at = lds + (part * CG + cg) * (NC * (DPL * 1024 + 512));
#pragma unroll
          for (int x = 0; x < NC; x++) {
            const f2 other = *reinterpret_cast<const f2 *>(at + NC * DPL * 1024 + (x * 64 + lane) * 8);
            const float up = fmaxf(top[x], other.x), mine = part_weight(top[x], up), its = part_weight(other.x, up);
            sum[x] = sum[x] * mine + other.y * its;
            top[x] = up;
#pragma unroll
            for (int c = 0; c < DPL; c++) acc[x][c] = acc[x][c] * mine + *reinterpret_cast<const f4 *>(at + ((x * DPL + c) * 64 + lane) * 16) * its;
          }
        }
        __syncthreads();
      }
    }

    const bool whole = from == 0 && to == steps;
    if (part == 0 && live) {
#pragma unroll
      for (int x = 0; x < NC; x++) {
        if (WHOLE || whole) {
          if (cg * 16 * NC + 16 * x + n < cols) {
            const long long i = first + row_of(x);
            put<C>(a.o + i * a.o_stride + (long long)head_of(x) * a.hd, acc[x], g, a.hd, sum[x] == 0.0f ? 0.0f : 1.0f / sum[x]);
            if (g == 0 && a.lse) a.lse[i * a.lse_stride + head_of(x)] = sum[x] == 0.0f ? kNegInf : (top[x] + __builtin_amdgcn_logf(sum[x])) * 0.69314718056f;
          }
        } else {
          float *o = a.part + ((long long)blockIdx.x * 2 + (u == begin ? 0 : 1)) * C::PARTF;
#pragma unroll
          for (int c = 0; c < DPL; c++) *reinterpret_cast<f4 *>(o + (((cg * NC + x) * DPL + c) * 64 + lane) * 4) = acc[x][c];
          if (g == 0) {
            o += CG * NC * DPL * 256 + (cg * NC + x) * 32 + n;
            o[0] = top[x];
            o[16] = sum[x];
          }
        }
      }
    }
    if constexpr (WHOLE) {
      u += gridDim.x;
      tile = u;
    } else {
      if (from == 0 && !whole && threadIdx.x == 0)    // the tile goes on in the shares behind this one
        a.split[blockIdx.x] = make_int4(1 + (int)((steps - to + share - 1) / share), r, (int)tile, u == begin ? 0 : 1);
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
template <int T, int HDP, int NC, int CG>
__global__ __launch_bounds__(256) void k_tree_join(TaArgs a) {
  using C = Cfg<T, HDP, NC, CG>;
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
  const int stat = CG * NC * DPL * 256 + block * 32 + n;
  float top = kNegInf, sum = 0.0f;
  f4 acc[DPL];
#pragma unroll
  for (int c = 0; c < DPL; c++) acc[c] = f4{0, 0, 0, 0};
#pragma unroll 2
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

template <int T, int HDP, int NC, int CG>
int launch(const char *fn, const TaArgs &a, hipStream_t stream) {
  using C = Cfg<T, HDP, NC, CG>;
  static_assert(C::LDSB <= 160 * 1024, "LDS");
  const long long room = ((long long)a.width * a.page_size + C::STEP - 1) / C::STEP;
  const bool whole = room <= 4 && a.n_req <= 65535;
  void (*f)(TaArgs) = whole ? k_tree_attn<T, HDP, NC, CG, true> : k_tree_attn<T, HDP, NC, CG, false>;
  if (C::LDSB > 64 * 1024 &&          // past what a launch may take unasked
      hipFuncSetAttribute(reinterpret_cast<const void *>(f), hipFuncAttributeMaxDynamicSharedMemorySize, C::LDSB) != hipSuccess) {
    (void)hipGetLastError();
    return qs::refuse(fn, "hipFuncSetAttribute failed");
  }
  if (whole) {
    const long long each = ((long long)a.rows * a.G / a.n_req + C::COLS - 1) / C::COLS;       // column tiles of a request, about
    const long long x = each < 1 ? a.n_kv : each * a.n_kv;
    QS_LAUNCH(fn, f, dim3((unsigned)(x < 65535 ? x : 65535), a.n_req), dim3(C::THREADS), C::LDSB, stream, a);
    return 0;
  }
  QS_LAUNCH(fn, f, dim3(C::SHARES), dim3(C::THREADS), C::LDSB, stream, a);
  QS_LAUNCH(fn, (k_tree_join<T, HDP, NC, CG>), dim3(C::SHARES, CG * NC), dim3(256), 0, stream, a);
  return 0;
}

template <int T, int HDP>
int launch_tile(const char *fn, const TaArgs &a, int tile, hipStream_t stream) {
  if constexpr (HDP == 256) return tile == 2 ? launch<T, HDP, 1, 4>(fn, a, stream) : launch<T, HDP, 1, 8>(fn, a, stream);
  else {
    switch (tile) {
      case 0: return launch<T, HDP, 1, 1>(fn, a, stream);
      case 1: return launch<T, HDP, 1, 2>(fn, a, stream);
      case 2: return launch<T, HDP, 1, 4>(fn, a, stream);
      case 3: return launch<T, HDP, 1, 8>(fn, a, stream);
      default: return launch<T, HDP, 2, 8>(fn, a, stream);
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
