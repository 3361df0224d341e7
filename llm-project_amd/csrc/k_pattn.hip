// k_pattn.hip - attention of one new token per request over a paged key-value cache
// (qllama_paged_attention; semantics in qserve.h).  No counterpart in the reference,
// whose decode attention (llama.c:554-576) serves one sequence and one dense cache.
//
// Memory bound: every key and value row is read once, 2 n_kv hd element bytes a token,
// and each byte takes part in n_heads / n_kv multiply-adds (4 at the shapes below).
//
// The work of a call is the key steps of all (request, KV head, 16 query heads) tiles,
// laid one behind another; every wave takes an equal share of them, whatever the
// lengths are, so ragged batches and one long request fill the chip alike without the
// host knowing a length.  A share that ends inside a tile leaves its maximum, sum and
// weighted values in the workspace, and k_paged_join puts a tile's parts together.
// Waves never meet: with four of them on a tile, meeting in LDS at its end, 512 requests
// of up to 300 f16 tokens (8 KV heads of 128, pages of 16) took 167 us, with shares of
// their own 134 (98 with what follows; 89 again with waves that meet, without a second launch).  Only for short tables a block takes
// a tile, a wave a part of its steps, and they do meet: one launch instead of two (launch()
// has the rule and its figures).
//
// A wave keeps its running maximum, sum and outputs in registers, its queries in LDS, and
// takes a step of 16 or 32 keys at a time straight from the pages into registers.
// S^T = K q^T on the matrix cores puts a query head in a lane's column and 4 keys of
// each 16 in its rows; the same lane's weights are then the operand of O^T += V^T P^T,
// whose contraction slots are matched to the keys the lane holds, so weights never move
// between lanes.  A lane loads whole pieces of a value row (16 lanes a row), and the
// pieces of 8 keys are turned by byte permutes.
//
// What is under way carries the bandwidth: two waves a SIMD, a step's values and the next
// step's keys (int8: and scales, 138 -> 131 us at the third row below) in registers.  Loading
// the values a step ahead too took 82 us against 76 at the first row, 138 against 131 at
// the third; three waves a SIMD (with fewer registers) 110 against 84 at the time, twice
// the blocks 92.
//
// Precision: float queries and weights meet 16-bit keys and values as parts that add up
// to them (bf16: three parts of 8 bits, f16: two of 11), one MFMA a part.  int8 codes
// become f16, with the values' scales in the weights, whose power of two follows the
// largest product so far: three instructions for two codes, where bf16 takes five and a
// third part (139 -> 132 us).  fp32 caches use the fp32 MFMA.  At 8 TB/s the parts take a
// sixth of the bf16 matrix rate.
//
// Measured (both kernels, 32 query and 8 KV heads; a 1 GiB copy moves 5.1 TB/s):
//   64 ragged requests of up to 2560 tokens, bf16, hd 128     73   us   4.8 TB/s
//   2 requests, up to 120000 tokens, f16, hd 128             134   us   5.5 TB/s
//   128 requests of up to 4100 tokens, int8, hd 128          126   us   4.5 TB/s
//   64 ragged requests of up to 2560 tokens, f32, hd 128     125   us   5.6 TB/s
//   the same, hd 64                                           68   us   5.1 TB/s
//   24 requests of up to 768 tokens, f32, hd 64               17.0 us   2.1 TB/s
//   1 request of 2060 tokens, bf16, hd 128                    12.5 us   0.7 TB/s
//   1 request of 200 tokens, f32, 6 + 2 heads of 48             7.2 us
// The short ones are launches and a chain of dependent trips to memory (lengths,
// table, keys, values, parts).  An int8 step has half a 16-bit one's bytes under way and
// the same chain of waits.
#include <hip/hip_runtime.h>

#include "qserve_host.h"

namespace {

typedef float f2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256, kWaves = 4;
constexpr int kBlocks = 512;          // two blocks of four waves a CU
constexpr int kShares = kBlocks * kWaves;
constexpr int kMinShare = 1;          // steps a wave takes at least; one request of 2060 tokens took 12.5 us, with 2 or 4 13.3
constexpr float kNegInf = -__builtin_inff();

struct PaArgs {
  const char *k, *v;
  const float *ks, *vs;
  const float *q;
  float *o, *lse;
  const int *table, *lens;
  float *part;
  int4 *split;
  long long pst, hst, sst;            // bytes
  long long scp, sch, scs;            // floats
  long long q_stride, o_stride, lse_stride, table_stride;
  int n_req, n_heads, n_kv, G, tiles, rows, hd, n_pages, page_size, width;
  float qscale;                       // scale * log2(e)
};

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

// Inclusive sums over a wave: within rows of 16 lanes, then from row to row.
template <int CTRL, int ROWS>
__device__ inline int from_lane(int x) { return __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xf, false); }
__device__ inline int wave_scan(int x) {
  x += from_lane<0x111, 0xf>(x);        // row_shr 1, 2, 4, 8
  x += from_lane<0x112, 0xf>(x);
  x += from_lane<0x114, 0xf>(x);
  x += from_lane<0x118, 0xf>(x);
  x += from_lane<0x142, 0xa>(x);        // row_bcast 15 to rows 1 and 3, 31 to rows 2 and 3
  return x + from_lane<0x143, 0xc>(x);
}

// Steps of a wave's share when all tiles together take `units`.
__device__ inline long long share_of(long long units) {
  const long long s = (units + kShares - 1) / kShares;
  return s < kMinShare ? kMinShare : s;
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

// W words of a row; STREAM: read once by its request (one tile of query heads a KV head), so
// past the caches' retention: 84 -> 77 us at 64 ragged bf16 requests, together with whole
// 64-byte runs a load; more tiles of a KV head find the rows in L2.  Pages that requests
// share are read so too: 64 requests on one request's pages take 72 us, on their own 73
template <bool STREAM, int W>
__device__ inline void load_words(uint32_t (&d)[W], const char *p) {
  typedef uint32_t vec __attribute__((ext_vector_type(W), aligned(W > 2 ? 8 : 4)));
  if constexpr (W == 1) {
    d[0] = *reinterpret_cast<const uint32_t *>(p);
  } else {
    const vec x = STREAM ? __builtin_nontemporal_load(reinterpret_cast<const vec *>(p)) : *reinterpret_cast<const vec *>(p);
#pragma unroll
    for (int i = 0; i < W; i++) d[i] = x[i];
  }
}

__device__ inline uint32_t hi16s(uint32_t b, uint32_t a) { return __builtin_amdgcn_perm(b, a, 0x07060302); }
__device__ inline uint32_t lo16s(uint32_t b, uint32_t a) { return __builtin_amdgcn_perm(b, a, 0x05040100); }
// 2^-9 times two int8 codes as f16: the codes plus 128, the bytes of y : x that SELECT
// names, are subnormal numbers of 2^-24, and one packed multiply-add makes them 2^-9 and takes
// the 128 off, exactly.  x and y have had the top bits of their bytes turned.
constexpr int kCodeBits = 9, kRaise = 120;
template <uint32_t SELECT>
__device__ inline uint32_t codes(uint32_t y, uint32_t x) {
  const h2 u = __builtin_bit_cast(h2, __builtin_amdgcn_perm(y, x, SELECT));
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(u, h2{32768.0f16, 32768.0f16}, h2{-0.25f16, -0.25f16}));
}

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

// Waves that meet at most, as the registers allow.
constexpr int meeting(int hdp) { return hdp > 128 ? 4 : 8; }

// What a type and a padded head size fix.
template <int T, int HDP>
struct Cfg {
  static constexpr int ES = T == QLLAMA_KV_F32 ? 4 : T == QLLAMA_KV_I8 ? 1 : 2;
  static constexpr int SUB = T == QLLAMA_KV_F32 ? 1 : 2;       // 16-key groups of a step
  static constexpr int STEP = 16 * SUB;
  // a key's row: load x takes bytes 64 x + 16 g .. of it in lane (key, g), EL elements
  static constexpr int KL = HDP * ES / 64, EL = 16 / ES;
  // a value row: piece x of lane (n, g) takes dims 16 PD x + PD n .. of key 4 g + j
  static constexpr int PB0 = HDP * ES / 16, PB1 = PB0 < 16 ? PB0 : 16, PB = PB1 < 8 * ES ? PB1 : 8 * ES;
  static constexpr int PD = PB / ES, PIECES = HDP / (16 * PD), PW = PB / 4;
  static constexpr int DPL = HDP / 16;                         // dims of a value row in a lane
  static constexpr int PARTS = T == QLLAMA_KV_F32 ? 1 : T == QLLAMA_KV_BF16 ? 3 : 2;
  static constexpr bool HALF = PARTS == 2;                     // f16 products
  static constexpr int MEETING = meeting(HDP);
  // a query row in LDS: a part's values, and 64 bytes that spread rows over the banks
  static constexpr int QES = T == QLLAMA_KV_F32 ? 4 : 2;
  static constexpr int QROW = HDP * QES + 64;
  // what weights are held times in the products: f16 parts then keep 23 bits down to 2^-17
  // of the largest weight and the rest to 2^-40.  Not in the exponent, where a 15 beside a
  // small score takes 2^-21 of the weight and of lse.
  static constexpr float RAISED = T == QLLAMA_KV_F16 ? 32768.0f : 1.0f;
};

template <int T, int HDP>
struct KTile { uint32_t w[Cfg<T, HDP>::SUB][Cfg<T, HDP>::KL][4]; };
template <int T>
struct Scales { float k[T == QLLAMA_KV_I8 ? 2 : 1][4], v[T == QLLAMA_KV_I8 ? 2 : 1][4]; };
template <int T, int HDP>
struct VTile { uint32_t w[Cfg<T, HDP>::SUB][4][Cfg<T, HDP>::PIECES][Cfg<T, HDP>::PW]; };

// Where the keys of a wave's steps lie.  UNI (page_size a multiple of 16): lane l holds
// the page and place of 16-key group first + l, read from the table 64 groups at a
// time, and a group's address is uniform.  Otherwise lane l holds those of key first +
// l and they go to the lanes that load the key.  A page outside the cache is -1.
template <bool UNI>
struct Window {
  int first, page, place;
  __device__ inline long long key() const { return UNI ? ((long long)first + (threadIdx.x & 63)) * 16 : (long long)first + (threadIdx.x & 63); }
  __device__ inline void request(const PaArgs &a, const int *table, int from, int len) {
    first = from;
    page = table[entry_of(key(), len, a.page_size, &place)];
  }
  __device__ inline void settle(const PaArgs &a, int len) { page = page_of(page, key(), len, a.n_pages); }
};

// MEET: a block's waves share one tile, a request's where blockIdx says, and meet in LDS.
template <int T, int HDP, bool UNI, bool STREAM, bool MEET>
__global__ __launch_bounds__(MEET ? 64 * meeting(HDP) : kThreads, HDP > 128 ? 1 : 2) void k_paged_attn(PaArgs a) {
  using C = Cfg<T, HDP>;
  constexpr int SUB = C::SUB, STEP = C::STEP, CH = HDP / 32, DPL = C::DPL;
  extern __shared__ __align__(16) char dyn[];       // a wave's queries: [part][row]
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4;           // key, query head or value piece; group of 16 lanes
  const int tiles = a.n_kv * a.tiles;
  char *q_lds = dyn + wave * (C::PARTS * a.rows * C::QROW);
  const int waves = blockDim.x >> 6;
  float *parts = reinterpret_cast<float *>(dyn + waves * (C::PARTS * a.rows * C::QROW));          // of waves that meet

  // this wave's share of all steps; shares of one block lie far apart, so that few of
  // them are spread over the CUs
  const auto len_of = [&](int r) { return r < a.n_req ? clamp_len(a.lens[r], a.width, a.page_size) : 0; };
  int len, r = 0, steps = 0, tile = 0, from = 0;    // a request, its steps, where in them this wave begins
  long long u, end, share = 0;                      // units from u up to end are this wave's
  const int id = wave * kBlocks + blockIdx.x;
  if constexpr (MEET) {
    r = blockIdx.y;
    tile = blockIdx.x;
    len = __builtin_amdgcn_readfirstlane(len_of(r));
    steps = (len + STEP - 1) / STEP;
    const int each = (steps + waves - 1) / waves;
    from = wave * each;
    u = from;
    end = from + each < steps ? from + each : steps;
  } else {
    len = len_of(lane);                               // of request `lane` of the 64 in hand, then of the one at work
    int upto = wave_scan((len + STEP - 1) / STEP);    // steps of those up to it
    long long units = (long long)__builtin_amdgcn_readlane(upto, 63) * tiles;
    for (int r = 64; r < a.n_req; r += 64)
      units += (long long)__builtin_amdgcn_readlane(wave_scan((len_of(r + lane) + STEP - 1) / STEP), 63) * tiles;
    share = share_of(units);
    u = id * share;
    end = u + share < units ? u + share : units;
    if (lane == 0) a.split[id] = make_int4(0, 0, 0, 0);
    long long r_begin = 0;                            // the first unit of the request it begins in
    for (; u < end; r += 64) {
      if (r) {
        len = len_of(r + lane);
        upto = wave_scan((len + STEP - 1) / STEP);
      }
      const uint64_t past = __ballot(r_begin + (long long)upto * tiles > u);
      if (past) {
        const int at = __builtin_ctzll(past);
        len = __builtin_amdgcn_readlane(len, at);
        r_begin += (long long)(__builtin_amdgcn_readlane(upto, at) - (len + STEP - 1) / STEP) * tiles;
        r += at;
        break;
      }
      r_begin += (long long)__builtin_amdgcn_readlane(upto, 63) * tiles;
    }

    len = __builtin_amdgcn_readfirstlane(len);        // one for the wave from here on
    if (u < end) {
      const unsigned long long at = u - r_begin;
      steps = (len + STEP - 1) / STEP;
      tile = __builtin_amdgcn_readfirstlane(at >> 32 ? (int)(at / (unsigned)steps) : (int)((unsigned)at / (unsigned)steps));
      from = (int)(at - (unsigned long long)tile * steps);
    }
  }
  const long long begin = u;
  Window<UNI> win;
  win.first = -1;

  while (u < end) {
    if (tile == tiles) {                            // the next request that has tokens
      do len = __builtin_amdgcn_readfirstlane(len_of(++r)); while (len == 0);
      steps = (len + STEP - 1) / STEP;
      tile = 0;
      win.first = -1;
    }
    const int to = (int)(end - u < steps - from ? from + (end - u) : steps);
    const int kvh = a.tiles == 1 ? tile : tile / a.tiles, part = a.tiles == 1 ? 0 : tile - kvh * a.tiles;
    const int h0 = kvh * a.G + part * 16, rows = a.G - part * 16 < 16 ? a.G - part * 16 : 16;
    const int *table = a.table + r * a.table_stride;
    const int row = n % rows;                       // columns past the tile's heads repeat them
    const bool fresh = win.first != (UNI ? from * SUB : from * STEP);    // a request's tiles read the same pages
    if (fresh) win.request(a, table, UNI ? from * SUB : from * STEP, len);

    // queries: head h0 + row, dims 32 c + 8 g ..
    float qf[CH][8];
    const float *q = a.q + r * a.q_stride + (long long)(h0 + row) * a.hd;
#pragma unroll
    for (int c = 0; c < CH; c++) {
      const int d = 32 * c + 8 * g;
      __builtin_memcpy(qf[c], q + (d < a.hd ? d : 0), sizeof qf[c]);       // 4-byte aligned; head_dim is a multiple of 8
    }
    if (fresh) win.settle(a, len);

    const char *kbase = a.k + kvh * a.hst, *vbase = a.v + kvh * a.hst;
    // a lane's place behind a row, UNI: behind the first row of 16; padded dims read dim 0: their
    // products are dropped, or with 0
    unsigned k_off[C::KL], v_off[C::PIECES];
#pragma unroll
    for (int x = 0; x < C::KL; x++) k_off[x] = (64 * x + 16 * g < a.hd * C::ES ? 64 * x + 16 * g : 0) + (UNI ? n * (int)a.sst : 0);
#pragma unroll
    for (int x = 0; x < C::PIECES; x++)
      v_off[x] = (16 * C::PD * x + C::PD * n < a.hd ? (16 * C::PD * x + C::PD * n) * C::ES : 0) + (UNI ? 4 * g * (int)a.sst : 0);

    // page and place of 16-key group i of step s (UNI), or of its key j
    auto lookup = [&](int s, int i, int j, int *place) -> int {
      if constexpr (UNI) {
        const int at = s * SUB + i - win.first;
        *place = __builtin_amdgcn_readlane(win.place, at) + j;
        return __builtin_amdgcn_readlane(win.page, at);
      } else {
        const int at = s * STEP + 16 * i + j - win.first;
        *place = __shfl(win.place, at);
        return __shfl(win.page, at);
      }
    };
    auto advance = [&](int s) {                     // the window holds step s
      const int at = UNI ? s * SUB : s * STEP;
      if (at - win.first >= 64) {
        win.request(a, table, at, len);
        win.settle(a, len);
      }
    };
    auto load_k = [&](int s, KTile<T, HDP> &k) {
#pragma unroll
      for (int i = 0; i < SUB; i++) {
        int place;
        int page = lookup(s, i, UNI ? 0 : n, &place);
        if (page < 0) { page = 0; place = 0; }
        const char *p = kbase + page * a.pst + place * a.sst;
#pragma unroll
        for (int x = 0; x < C::KL; x++) {
          if (T != QLLAMA_KV_I8 || a.hd % 16 == 0) {
            load_words<STREAM>(k.w[i][x], p + k_off[x]);
          } else {                                  // the row may end within the 16 bytes
            uint32_t lo[2], hi[2];
            load_words<STREAM>(lo, p + k_off[x]);
            load_words<STREAM>(hi, p + (64 * x + 16 * g + 8 < a.hd ? k_off[x] + 8 : k_off[x]));
            k.w[i][x][0] = lo[0]; k.w[i][x][1] = lo[1]; k.w[i][x][2] = hi[0]; k.w[i][x][3] = hi[1];
          }
        }
      }
    };
    auto load_v = [&](int s, VTile<T, HDP> &v) {
#pragma unroll
      for (int i = 0; i < SUB; i++) {
        const char *p = vbase;
        if constexpr (UNI) {
          int place;
          int page = lookup(s, i, 0, &place);
          if (page < 0) { page = 0; place = 0; }
          p += page * a.pst + place * a.sst;
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const char *pj = p;
          if constexpr (UNI) {
            pj += j * a.sst;
          } else {
            int place;
            int page = lookup(s, i, 4 * g + j, &place);
            if (page < 0) { page = 0; place = 0; }
            pj += page * a.pst + place * a.sst;
          }
#pragma unroll
          for (int x = 0; x < C::PIECES; x++) load_words<STREAM>(v.w[i][j][x], pj + v_off[x]);
        }
      }
    };

    auto load_scales = [&](int s, Scales<T> &f) {
      if constexpr (T == QLLAMA_KV_I8) {
#pragma unroll
        for (int i = 0; i < SUB; i++) {
          int first = 0;
          const int page = UNI ? lookup(s, i, 0, &first) : 0;
          if (UNI && a.scs == 1) {                  // 4 keys' scales beside each other, on any 4-byte boundary
            const long long at = (page < 0 ? 4 * g : page * a.scp + first + 4 * g) + kvh * a.sch;
            __builtin_memcpy(f.k[i], a.ks + at, sizeof f.k[i]);
            __builtin_memcpy(f.v[i], a.vs + at, sizeof f.v[i]);
          } else {
#pragma unroll
            for (int j = 0; j < 4; j++) {
              int place = first + 4 * g + j;
              const int of = UNI ? page : lookup(s, i, 4 * g + j, &place);
              const long long at = of < 0 ? 0 : of * a.scp + kvh * a.sch + place * a.scs;
              f.k[i][j] = a.ks[at];
              f.v[i][j] = a.vs[at];
            }
          }
        }
      }
    };

    KTile<T, HDP> k0, k1;
    Scales<T> f0, f1;
    load_scales(from, f0);
    load_k(from, k0);

    // into LDS, scaled so that weights are powers of two
    float unscale = 1.0f;
    {
      float qmax = 0.0f;
#pragma unroll
      for (int c = 0; c < CH; c++)
#pragma unroll
        for (int i = 0; i < 8; i++) {
          qf[c][i] = 32 * c + 8 * g < a.hd ? qf[c][i] * a.qscale : 0.0f;
          qmax = fmaxf(qmax, fabsf(qf[c][i]));
        }
      int e = 0;
      if constexpr (C::HALF) {                      // into f16's range, by a power of two
        qmax = max_groups(qmax);
        e = qmax > 0.0f && qmax < __builtin_inff() ? ilogbf(qmax) - 13 : 0;
        unscale = ldexpf(1.0f, T == QLLAMA_KV_I8 ? e + kCodeBits : e);
      }
      __builtin_amdgcn_wave_barrier();              // the last tile's reads come first
#pragma unroll
      for (int c = 0; c < CH; c++) {
        char *to_lds = q_lds + row * C::QROW + (32 * c + 8 * g) * C::QES;
        if constexpr (T == QLLAMA_KV_F32) {
          if (n < rows) __builtin_memcpy(__builtin_assume_aligned(to_lds, 16), qf[c], sizeof qf[c]);
        } else if constexpr (C::HALF) {
#pragma unroll
          for (int i = 0; i < 8; i++) qf[c][i] = ldexpf(qf[c][i], -e);
          const Parts2 x = cut2(qf[c]);
#pragma unroll
          for (int p = 0; p < 2; p++)
            if (n < rows) *reinterpret_cast<u4 *>(to_lds + p * a.rows * C::QROW) = x.p[p];
        } else {
          const Parts3 x = cut3(qf[c]);
#pragma unroll
          for (int p = 0; p < 3; p++)
            if (n < rows) *reinterpret_cast<u4 *>(to_lds + p * a.rows * C::QROW) = x.p[p];
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
    const char *q_mine = q_lds + row * C::QROW;

    float m = kNegInf, l = 0.0f;                    // of the lane's query head; l over the lane's keys
    // int8: weights times scales are held times 2^raise, which keeps the largest magnitude so far below
    // 2^15 and within a factor of 2^16 of it or so, whatever the scales are
    int raise = kRaise;
    float slack = 0.0f;                             // what a larger score has left over of a factor of 2
    f4 acc[DPL];
#pragma unroll
    for (int c = 0; c < DPL; c++) acc[c] = f4{0, 0, 0, 0};

    auto step = [&](int s, KTile<T, HDP> &k, KTile<T, HDP> &k_next, Scales<T> &f, Scales<T> &f_next) {
      VTile<T, HDP> v;
      bool out[SUB][4];                             // a key behind the last, or on no page
      bool absent = (s + 1) * STEP > len;
#pragma unroll
      for (int i = 0; i < SUB; i++) {
        int page[4], place[4], group_place = 0;
        const int group_page = UNI ? lookup(s, i, 0, &group_place) : 0;
#pragma unroll
        for (int j = 0; j < 4; j++) {
          if constexpr (UNI) {
            page[j] = group_page;
            place[j] = group_place + 4 * g + j;
          } else {
            page[j] = lookup(s, i, 4 * g + j, &place[j]);
          }
          out[i][j] = page[j] < 0 || s * STEP + 16 * i + 4 * g + j >= len;
          absent |= page[j] < 0;
        }
      }
      load_v(s, v);
      if (s + 1 < to) {
        advance(s + 1);
        load_scales(s + 1, f_next);
        load_k(s + 1, k_next);
      }

      // scores of 16 SUB keys for the lane's query head
      f4 d[SUB];
#pragma unroll
      for (int i = 0; i < SUB; i++) d[i] = f4{0, 0, 0, 0};
      asm volatile("" ::: "memory");                // the queries are read from LDS in every step, not kept in registers
#pragma unroll
      for (int x = 0; x < C::KL; x++) {
        if constexpr (T == QLLAMA_KV_F32) {
          const f4 q = *reinterpret_cast<const f4 *>(q_mine + 64 * x + 16 * g);
#pragma unroll
          for (int e = 0; e < 4; e++) d[0] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(k.w[0][x][e]), q[e], d[0], 0, 0, 0);
        } else {
#pragma unroll
          for (int h = 0; h < C::EL / 8; h++) {     // 8 dims an MFMA
            u4 qp[C::PARTS];
#pragma unroll
            for (int p = 0; p < C::PARTS; p++)
              qp[p] = *reinterpret_cast<const u4 *>(q_mine + p * a.rows * C::QROW + ((64 * x + 16 * g) / C::ES + 8 * h) * 2);
#pragma unroll
            for (int i = 0; i < SUB; i++) {
              u4 kk;
              if constexpr (T == QLLAMA_KV_I8) {
#pragma unroll
                for (int w = 0; w < 2; w++) {
                  const uint32_t b = k.w[i][x][2 * h + w] ^ 0x80808080u;
                  kk[2 * w] = codes<0x0c010c00>(b, b);
                  kk[2 * w + 1] = codes<0x0c030c02>(b, b);
                }
              } else {
                kk = u4{k.w[i][x][0], k.w[i][x][1], k.w[i][x][2], k.w[i][x][3]};
              }
#pragma unroll
              for (int p = 0; p < C::PARTS; p++) d[i] = mfma16<T>(kk, qp[p], d[i]);
            }
          }
        }
      }
      float sc[SUB][4];
#pragma unroll
      for (int i = 0; i < SUB; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
          sc[i][j] = d[i][j];
          if constexpr (C::HALF) sc[i][j] *= unscale;
          if constexpr (T == QLLAMA_KV_I8) sc[i][j] *= f.k[i][j];
        }
      if (__any(absent)) {
#pragma unroll
        for (int i = 0; i < SUB; i++)
#pragma unroll
          for (int j = 0; j < 4; j++) {
            if (out[i][j]) {                        // whatever the slot holds, NaN too, counts nothing
              sc[i][j] = kNegInf;
              if constexpr (T == QLLAMA_KV_I8) f.v[i][j] = 0.0f;
#pragma unroll
              for (int x = 0; x < C::PIECES; x++)
#pragma unroll
                for (int w = 0; w < C::PW; w++) v.w[i][j][x][w] = 0;
            }
          }
      }

      float top = sc[0][0];
#pragma unroll
      for (int i = 0; i < SUB; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) top = fmaxf(top, sc[i][j]);
      top = fmaxf(m, max_groups(top));
      if (__any(top > m)) {                         // rare after the first steps
        const float d = m == kNegInf ? kNegInf : m - top;
        l *= __builtin_amdgcn_exp2f(d);
        int up = 0;
        if constexpr (T == QLLAMA_KV_I8) {          // what is held shrinks with the weights, by less than 2 in all
          const float more = fminf(slack - d, 512.0f);
          up = min((int)more, kRaise - raise);
          raise += up;
          slack = raise == kRaise ? 0.0f : more - up;
        }
        const float by = __builtin_amdgcn_exp2f(d + up);
#pragma unroll
        for (int c = 0; c < DPL; c++) acc[c] *= by;
        m = top;
      }
      const float ref = m == kNegInf ? 0.0f : m;
      float p[SUB][4];
#pragma unroll
      for (int i = 0; i < SUB; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
          p[i][j] = __builtin_amdgcn_exp2f(sc[i][j] - ref);
          l += p[i][j];
          if constexpr (T == QLLAMA_KV_I8) p[i][j] *= f.v[i][j];
          else p[i][j] *= C::RAISED;
        }
      if constexpr (T == QLLAMA_KV_I8) {            // into f16's range
        float most = 0.0f;
#pragma unroll
        for (int i = 0; i < SUB; i++)
#pragma unroll
          for (int j = 0; j < 4; j++) most = fmaxf(most, fabsf(p[i][j]));      // a scale may be negative
        most = max_groups(most);
        const int room = 141 - (int)(__float_as_uint(most) >> 23);           // most < 2^(15 - room)
        if (__any(room < raise)) {                  // rare after the first step
          const int down = min(room - raise, 0);
          raise += down;
#pragma unroll
          for (int c = 0; c < DPL; c++)
#pragma unroll
            for (int i = 0; i < 4; i++) acc[c][i] = ldexpf(acc[c][i], down);
        }
#pragma unroll
        for (int i = 0; i < SUB; i++)
#pragma unroll
          for (int j = 0; j < 4; j++) p[i][j] = ldexpf(p[i][j], raise);
      }

      if constexpr (T == QLLAMA_KV_F32) {
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
          for (int c = 0; c < DPL; c++)
            acc[c] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(v.w[0][j][c / C::PD][c % C::PD]), p[0][j], acc[c], 0, 0, 0);
      } else {
        const float pf[8] = {p[0][0], p[0][1], p[0][2], p[0][3], p[SUB - 1][0], p[SUB - 1][1], p[SUB - 1][2], p[SUB - 1][3]};
        u4 pp[C::PARTS];
        if constexpr (C::HALF) {
          const Parts2 x = cut2(pf);
          pp[0] = x.p[0]; pp[1] = x.p[1];
        } else {
          const Parts3 x = cut3(pf);
          pp[0] = x.p[0]; pp[1] = x.p[1]; pp[2] = x.p[2];
        }
        if constexpr (T == QLLAMA_KV_I8) {
#pragma unroll
          for (int i = 0; i < SUB; i++)
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
              for (int x = 0; x < C::PIECES; x++)
#pragma unroll
                for (int w = 0; w < C::PW; w++) v.w[i][j][x][w] ^= 0x80808080u;
        }
#pragma unroll
        for (int c = 0; c < DPL; c++) {
          u4 vv;                                    // dim c of the lane's piece, 8 keys
#pragma unroll
          for (int i = 0; i < SUB; i++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
              const uint32_t *x = v.w[i][2 * j][c / C::PD], *y = v.w[i][2 * j + 1][c / C::PD];
              constexpr int PD = C::PD;
              if constexpr (T == QLLAMA_KV_I8) {
                const uint32_t xa = x[c % PD / 4], ya = y[c % PD / 4];
                vv[2 * i + j] = c % 4 == 0 ? codes<0x0c040c00>(ya, xa) : c % 4 == 1 ? codes<0x0c050c01>(ya, xa)
                              : c % 4 == 2 ? codes<0x0c060c02>(ya, xa) : codes<0x0c070c03>(ya, xa);
              } else {
                vv[2 * i + j] = c % 2 ? hi16s(y[c % PD / 2], x[c % PD / 2]) : lo16s(y[c % PD / 2], x[c % PD / 2]);
              }
            }
#pragma unroll
          for (int k = 0; k < C::PARTS; k++) acc[c] = mfma16<T>(vv, pp[k], acc[c]);
        }
      }
    };

    for (int s = from; s < to; s += 2) {
      step(s, k0, k1, f0, f1);
      if (s + 1 < to) step(s + 1, k1, k0, f1, f0);
    }
    l = sum_groups(l);

    // lane (n, g) holds head n; acc[c][i] is dim c mod PD of the piece of lane 4 g + i
    const bool whole = from == 0 && to == steps;
    const auto put = [&](float *o, float by) {
      by *= 1.0f / C::RAISED;
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int c = 0; c < DPL; c += 4) {
          float x[4] = {acc[c][i] * by, acc[c + 1][i] * by, acc[c + 2][i] * by, acc[c + 3][i] * by};
          if constexpr (T == QLLAMA_KV_I8) {
#pragma unroll
            for (int j = 0; j < 4; j++) x[j] = ldexpf(x[j], kCodeBits - raise);
          }
          const int d = 16 * C::PD * (c / C::PD) + C::PD * (4 * g + i) + c % C::PD;
          if (d < a.hd) __builtin_memcpy(o + d, x, sizeof x);
        }
    };
    if (n < rows) {
      if (whole) {
        put(a.o + r * a.o_stride + (long long)(h0 + row) * a.hd, l == 0.0f ? 0.0f : 1.0f / l);
        if (g == 0 && a.lse) a.lse[r * a.lse_stride + h0 + row] = l == 0.0f ? kNegInf : (m + __builtin_amdgcn_logf(l)) * 0.69314718056f;
      } else if constexpr (MEET) {
        float *o = parts + wave * (a.rows * (a.hd + 2)) + row * (a.hd + 2);
        put(o, 1.0f);
        if (g == 0) { o[a.hd] = m; o[a.hd + 1] = l; }
      } else {
        float *o = a.part + ((long long)id * 2 + (u == begin ? 0 : 1)) * (a.rows * (a.hd + 2)) + row * (a.hd + 2);
        put(o, 1.0f);
        if (g == 0) { o[a.hd] = m; o[a.hd + 1] = l; }
      }
    }
    if (!MEET && from == 0 && !whole && lane == 0)   // the tile goes on in the shares behind this one
      a.split[id] = make_int4(1 + (int)((steps - to + share - 1) / share), r, tile, u == begin ? 0 : 1);
    u += to - from;
    from = 0;
    tile++;
  }

  if constexpr (MEET) {
    const int kvh = (int)blockIdx.x / a.tiles, part = (int)blockIdx.x - kvh * a.tiles;
    const int h0 = kvh * a.G + part * 16, rows = a.G - part * 16 < 16 ? a.G - part * 16 : 16;
    float *o = a.o + r * a.o_stride + (long long)h0 * a.hd, *lse = a.lse + r * a.lse_stride + h0;
    const int each = (steps + waves - 1) / waves, n_parts = steps ? (steps + each - 1) / each : 0, one = a.hd + 2;
    __syncthreads();
    if (n_parts == 1) return;
    for (int i = threadIdx.x; i < rows * a.hd; i += 64 * waves) {
      const int row = i / a.hd, d = i - row * a.hd;
      const float *p = parts + row * one;
      float top = kNegInf, sum = 0.0f, x = 0.0f;
      for (int j = 0; j < n_parts; j++) top = fmaxf(top, p[j * a.rows * one + a.hd]);
      for (int j = 0; j < n_parts; j++) {
        const float f = part_weight(p[j * a.rows * one + a.hd], top);
        sum += p[j * a.rows * one + a.hd + 1] * f;
        x += p[j * a.rows * one + d] * f;
      }
      o[i] = sum == 0.0f ? 0.0f : x * (1.0f / sum);
      if (d == 0 && a.lse) lse[row] = sum == 0.0f ? kNegInf : (top + __builtin_amdgcn_logf(sum)) * 0.69314718056f;
    }
    return;
  }

  // a request without a token has no tile: its outputs are set here
  for (int e = id; e < a.n_req; e += kShares)
    if (a.lens[e] <= 0)
      for (int i = lane; i < a.n_heads * a.hd; i += 64) {
        a.o[e * a.o_stride + i] = 0.0f;
        if (a.lse && i < a.n_heads) a.lse[e * a.lse_stride + i] = kNegInf;
      }
}

// One block a share and row: where a tile begins in the share and goes on behind it, its
// parts put together in the order of their keys, 8 (hd <= 128) or 4 side by side.  A
// trip to the descriptor and one to the parts, with a launch in front: 5.2 us for eight
// tiles of 67 parts, 7.3 at 64 ragged requests (512 tiles of some 4 parts), 12.3 where
// 2048 shares make 16 tiles.
constexpr int kJoinThreads = 256, kAhead = 4;
__global__ __launch_bounds__(kJoinThreads) void k_paged_join(PaArgs a) {
  __shared__ float weight[kShares], lds[kJoinThreads / 32][256], red[2][kJoinThreads / 64];
  const int4 s = a.split[blockIdx.x];
  const int parts = s.x, r = s.y, tile = s.z, row = blockIdx.y;
  const int kvh = tile / a.tiles, h = kvh * a.G + (tile % a.tiles) * 16 + row;
  if (!parts || h >= (kvh + 1) * a.G) return;
  const int one = a.rows * (a.hd + 2);
  // the first part may follow another tile's in its share
  const float *part = a.part + 2LL * blockIdx.x * one + row * (a.hd + 2);
  const int first = s.w * one;
  const int width = a.hd <= 128 ? 32 : 64, groups = kJoinThreads / width;
  const int group = threadIdx.x / width, d = threadIdx.x % width * 4;
  // a thread's first values are under way while the weights are formed
  float y[kAhead][4];
#pragma unroll
  for (int j = 0; j < kAhead; j++) {
    const int i = group + j * groups;
    const float *p = part + (i < parts && d < a.hd ? 2LL * i * one + (i ? 0 : first) + d : first);
    __builtin_memcpy(y[j], p, sizeof y[j]);
  }
  float top = kNegInf, l = 0.0f;
  for (int i = threadIdx.x; i < parts; i += kJoinThreads) {
    const float *p = part + 2LL * i * one + (i ? 0 : first) + a.hd;
    weight[i] = p[0];
    if (i < kJoinThreads) l = p[1];
    top = fmaxf(top, weight[i]);
  }
  for (int d = 32; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
  if ((threadIdx.x & 63) == 0) red[0][threadIdx.x >> 6] = top;
  __syncthreads();
  for (int i = 0; i < kJoinThreads / 64; i++) top = fmaxf(top, red[0][i]);
  float sum = 0.0f;
  for (int i = threadIdx.x; i < parts; i += kJoinThreads) {
    weight[i] = part_weight(weight[i], top);
    sum += (i < kJoinThreads ? l : part[2LL * i * one + a.hd + 1]) * weight[i];
  }
  for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
  if ((threadIdx.x & 63) == 0) red[1][threadIdx.x >> 6] = sum;
  __syncthreads();
  sum = 0.0f;
  for (int i = 0; i < kJoinThreads / 64; i++) sum += red[1][i];

  if (d < a.hd) {
    float x[4] = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < kAhead; j++) {
      const int i = group + j * groups;
      if (i < parts) {
        const float f = weight[i];
#pragma unroll
        for (int c = 0; c < 4; c++) x[c] += y[j][c] * f;
      }
    }
#pragma unroll 8
    for (int i = group + kAhead * groups; i < parts; i += groups) {
      float z[4];
      __builtin_memcpy(z, part + 2LL * i * one + d, sizeof z);
#pragma unroll
      for (int c = 0; c < 4; c++) x[c] += z[c] * weight[i];
    }
#pragma unroll
    for (int c = 0; c < 4; c++) lds[group][d + c] = x[c];
  }
  __syncthreads();
  const float by = sum == 0.0f ? 0.0f : 1.0f / sum;
  for (int i = threadIdx.x; i < a.hd; i += kJoinThreads) {
    float x = 0.0f;
    for (int j = 0; j < groups; j++) x += lds[j][i];
    a.o[r * a.o_stride + (long long)h * a.hd + i] = x * by;
  }
  if (threadIdx.x == 0 && a.lse) a.lse[r * a.lse_stride + h] = sum == 0.0f ? kNegInf : (top + __builtin_amdgcn_logf(sum)) * 0.69314718056f;
}

int rows_of(const QPagedKV *c, int n_heads) {
  const int G = n_heads / c->n_kv;
  return G < 16 ? G : 16;
}

template <int T, int HDP>
int launch(const char *fn, const PaArgs &a, hipStream_t stream) {
  using C = Cfg<T, HDP>;
  const bool uni = a.page_size % 16 == 0, once = a.tiles == 1;
  const long long tiles = (long long)a.n_req * a.n_kv * a.tiles, room = ((long long)a.width * a.page_size + C::STEP - 1) / C::STEP;
  const size_t queries = (size_t)C::PARTS * a.rows * C::QROW, part = (size_t)a.rows * (a.hd + 2) * sizeof(float);
  // Short tables: a block a tile, whose waves meet, and no second launch: 8 waves while a CU
  // has one tile at most, else 4, with a limit on the steps that a wave takes.  Against shares, us
  // (8 KV heads, hd 128 if not said, lengths up to the number): bf16, 32 requests of 120 7.2 / 11.7, 64
  // of 340 17.8 / 22.7 (8 waves 21.3), 64 of 900 34.1 / 35.7, 128 of 340 29.3 / 34.4, 512 of 900 201 / 213;
  // 64 int8 ones of 340 15.9 / 21.7; hd 64, 24 f32 ones of 250 8.7 / 13.2, 128 of 450 30.6 / 35.3, 64 bf16 ones
  // of 1900 (16 steps) 36.1 / 34.5.  One request leaves CUs idle: of 100 6.7 / 8.8, of 340 10.1 / 9.0.
  // Among thousands of tiles whose waves have a step at most, or of int8, shares are better:
  // 256 of 60 24.1 / 18.6, 512 int8 ones of 300 82 / 77.  The rule knows the tables' width, not the
  // lengths in device memory: 32 requests of 120 behind tables of 2560 take 12.6, 64 of 340 22.6.
  const int waves = tiles > 256 ? 4 : C::MEETING;
  const long long each = (room + waves - 1) / waves;
  const bool few = tiles > 256 ? each <= 8 && each * HDP <= 1024 && (tiles <= 1024 || (each > 1 && T != QLLAMA_KV_I8)) : each * HDP <= (tiles < 32 ? 128 : 256);
  const bool meet = few && a.n_req <= 65535 && waves * (queries + part) <= 64 * 1024;
  void (*f)(PaArgs);
  if (meet)
    f = uni ? once ? k_paged_attn<T, HDP, true, true, true> : k_paged_attn<T, HDP, true, false, true>
            : once ? k_paged_attn<T, HDP, false, true, true> : k_paged_attn<T, HDP, false, false, true>;
  else
    f = uni ? once ? k_paged_attn<T, HDP, true, true, false> : k_paged_attn<T, HDP, true, false, false>
            : once ? k_paged_attn<T, HDP, false, true, false> : k_paged_attn<T, HDP, false, false, false>;
  const size_t lds = meet ? waves * (queries + part) : kWaves * queries;
  if (lds > 64 * 1024 &&              // past what a launch may take unasked
      hipFuncSetAttribute(reinterpret_cast<const void *>(f), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds) != hipSuccess) {
    (void)hipGetLastError();
    return qs::refuse(fn, "hipFuncSetAttribute failed");
  }
  if (meet) {
    QS_LAUNCH(fn, f, dim3(a.n_kv * a.tiles, a.n_req), dim3(64 * waves), lds, stream, a);
    return 0;
  }
  QS_LAUNCH(fn, f, dim3(kBlocks), dim3(kThreads), lds, stream, a);
  // shares that can hold a step, by the room of the tables
  const long long most = tiles * room;
  const int shares = most / kMinShare + 1 < kShares ? (int)(most / kMinShare + 1) : kShares;
  QS_LAUNCH(fn, k_paged_join, dim3(shares, a.rows), dim3(kJoinThreads), 0, stream, a);
  return 0;
}

template <int T>
int launch_hd(const char *fn, const PaArgs &a, hipStream_t stream) {
  return a.hd <= 64 ? launch<T, 64>(fn, a, stream) : a.hd <= 128 ? launch<T, 128>(fn, a, stream) : launch<T, 256>(fn, a, stream);
}

}  // namespace

extern "C" int qllama_test_page_of(const int32_t *table, int width, int page_size, int n_pages, int len, long long key, int *place) {
  len = clamp_len(len, width, page_size);
  *place = 0;
  if (key < 0 || len == 0) return -1;
  const int page = page_of(table[entry_of(key, len, page_size, place)], key, len, n_pages);
  if (page < 0) *place = 0;
  return page;
}

extern "C" size_t qllama_paged_attention_work(const QPagedKV *c, int n_req, int n_heads) {
  if (qs::bad_cache(c) || n_req < 0 || n_heads < 1 || n_heads > 65535 || n_heads % c->n_kv) return 0;
  return kShares * (sizeof(int4) + (size_t)2 * rows_of(c, n_heads) * (c->head_dim + 2) * sizeof(float));
}

extern "C" int qllama_paged_attention(const QPagedKV *c, const QPagedQuery *a, void *stream) {
  static const char fn[] = "qllama_paged_attention";
  if (const char *why = qs::bad_cache(c)) return qs::refuse(fn, why);
  if (!a || a->n_req < 0) return qs::refuse(fn, "null argument or n_req < 0");
  if (a->n_heads < 1 || a->n_heads > 65535 || a->n_heads % c->n_kv) return qs::refuse(fn, "n_heads must be a multiple of the cache's KV heads");
  if (a->n_req == 0) return 0;
  if (!a->q || !a->o || !a->table || !a->lens) return qs::refuse(fn, "null q, o, table or lens");
  const int64_t qd = (int64_t)a->n_heads * c->head_dim;
  if (a->q_stride < qd || a->o_stride < qd || (a->lse && a->lse_stride < a->n_heads)) return qs::refuse(fn, "a row stride below the row's length");
  if (a->width < 1 || a->table_stride < a->width || (int64_t)a->width * c->page_size > INT_MAX - 64)   // a step past it still fits
    return qs::refuse(fn, "bad table width (width * page_size must be below 2^31 - 64) or stride");
  if ((int64_t)a->n_req * (((int64_t)a->width * c->page_size + 15) / 16) > INT_MAX)
    return qs::refuse(fn, "n_req * width * page_size is too large");
  if (!(a->scale >= 0.0f) || a->scale > 2.35e38f)      // times log2 e within a float's range
    return qs::refuse(fn, "scale must be 0 .. 2.35e38");
  if (a->q == a->o) return qs::refuse(fn, "o must not be q");
  if (qs::misaligned(a->q, 4) || qs::misaligned(a->o, 4) || qs::misaligned(a->lse, 4) || qs::misaligned(a->table, 4) || qs::misaligned(a->lens, 4))
    return qs::refuse(fn, "a buffer is not aligned to its elements");
  if (!a->work || qs::misaligned(a->work, 16) || a->work_bytes < qllama_paged_attention_work(c, a->n_req, a->n_heads))
    return qs::refuse(fn, "work is missing, misaligned or smaller than qllama_paged_attention_work");
  qs::OnDevice on(c->k, (hipStream_t)stream);
  if (on.why) return qs::refuse(fn, on.why);
  const int es = c->type == QLLAMA_KV_F32 ? 4 : c->type == QLLAMA_KV_I8 ? 1 : 2;
  PaArgs p;
  p.k = static_cast<const char *>(c->k); p.v = static_cast<const char *>(c->v);
  p.ks = c->k_scale; p.vs = c->v_scale;
  p.q = a->q; p.o = a->o; p.lse = a->lse; p.table = a->table; p.lens = a->lens; p.split = static_cast<int4 *>(a->work);
  p.part = reinterpret_cast<float *>(p.split + kShares);
  p.pst = c->page_stride * es; p.hst = c->head_stride * es; p.sst = c->slot_stride * es;
  p.scp = c->scale_page_stride; p.sch = c->scale_head_stride; p.scs = c->scale_slot_stride;
  p.q_stride = a->q_stride; p.o_stride = a->o_stride; p.lse_stride = a->lse_stride; p.table_stride = a->table_stride;
  p.n_req = a->n_req; p.n_heads = a->n_heads; p.n_kv = c->n_kv; p.G = a->n_heads / c->n_kv; p.tiles = (p.G + 15) / 16;
  p.rows = rows_of(c, a->n_heads); p.hd = c->head_dim; p.n_pages = c->n_pages; p.page_size = c->page_size; p.width = a->width;
  p.qscale = (a->scale > 0.0f ? a->scale : 1.0f / __builtin_sqrtf((float)c->head_dim)) * 1.44269504089f;
  switch (c->type) {
    case QLLAMA_KV_F32: return launch_hd<QLLAMA_KV_F32>(fn, p, (hipStream_t)stream);
    case QLLAMA_KV_F16: return launch_hd<QLLAMA_KV_F16>(fn, p, (hipStream_t)stream);
    case QLLAMA_KV_BF16: return launch_hd<QLLAMA_KV_BF16>(fn, p, (hipStream_t)stream);
    default: return launch_hd<QLLAMA_KV_I8>(fn, p, (hipStream_t)stream);
  }
}
