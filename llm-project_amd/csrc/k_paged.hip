// k_paged.hip - pages and slots of a serving step, and new rows into their slots
// (qllama_paged_plan, qllama_paged_append; semantics in qserve.h).  No counterpart in
// the reference, whose cache is one dense array per sequence (llama.c:275-288).
#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include "qserve_host.h"

namespace {

// ---------------------------------------------------------------------------
// Plan
// ---------------------------------------------------------------------------
constexpr int kPlanThreads = 256;
constexpr int kPlanMaxReq = 8192;

struct PlanSums { long long a, b, c; };

__device__ inline PlanSums operator+(PlanSums x, PlanSums y) { return {x.a + y.a, x.b + y.b, x.c + y.c}; }

// Inclusive sums over the block's threads, and their total.
__device__ PlanSums plan_scan(PlanSums v, PlanSums *wave_sums, PlanSums *total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  for (int d = 1; d < 64; d <<= 1) {
    const PlanSums u = {__shfl_up(v.a, d), __shfl_up(v.b, d), __shfl_up(v.c, d)};
    if (lane >= d) v = v + u;
  }
  __syncthreads();                       // the previous scan's sums have been read
  if (lane == 63) wave_sums[w] = v;
  __syncthreads();
  PlanSums before = {0, 0, 0}, all = {0, 0, 0};
  for (int i = 0; i < kPlanThreads / 64; i++) {
    const PlanSums s = wave_sums[i];
    if (i < w) before = before + s;
    all = all + s;
  }
  *total = all;
  return v + before;
}

// Largest r with first[r] <= i, first ascending and first[0] = 0 <= i < first[n].
__device__ inline int plan_find(const int *first, int n, int i) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= i) lo = mid; else hi = mid;
  }
  return lo;
}

// Entries that n tokens fill (n <= width * page_size < 2^31).
__device__ inline int plan_pages(int n, int page_size) { return (int)(((unsigned)n + (unsigned)page_size - 1u) / (unsigned)page_size); }

// Place x + y of a ring of R, for x < R and y < R.
__device__ inline int plan_place(int x, int y, int R) {
  const unsigned s = (unsigned)x + (unsigned)y;
  return (int)(s >= (unsigned)R ? s - (unsigned)R : s);
}

// Every block forms the same prefix sums over all requests (they fit a few passes of
// 256 threads, which costs less than a second launch) and fills its share of the rows,
// the new pages and the returned pages; block 0 also writes what there is per request.
// Reads and in-place writes cannot meet: pages are taken from ring places [head, head +
// count) and returned to those behind, table entries below a request's first new one
// are read and those from it on written.  A chain of latencies, not bytes: 6.7 us at 250
// requests of a token each (two blocks: lengths, three scans, table and ring behind a
// search), 5.4 at 48 requests with 16384 rows (65 blocks; 0.2 MB); 13 us at 1000 requests and
// 63 at 8192, whose 32 passes every block makes.
__global__ __launch_bounds__(kPlanThreads) void k_paged_plan(QPagedPlan p) {
  extern __shared__ int lds[];
  int *row0 = lds, *take0 = lds + p.n_req + 1, *give0 = take0 + p.n_req + 1;
  __shared__ PlanSums wave_sums[kPlanThreads / 64];
  const int t = threadIdx.x;
  const int R = p.ring_size;
  int head = p.state[0], count = p.state[1];
  if (head < 0 || head >= R) head = 0;
  count = count < 0 ? 0 : count > R ? R : count;
  const long long room = (long long)p.width * p.page_size;

  PlanSums asked = {0, 0, 0}, given = {0, 0, 0};       // totals of the passes before
  for (int r0 = 0; r0 < p.n_req; r0 += kPlanThreads) {
    const int r = r0 + t;
    const bool there = r < p.n_req;
    const long long c = there ? p.cached[r] : 0, a = there ? p.added[r] : 0;
    const bool known = c >= 0 && c <= room;
    const long long have = known ? plan_pages((int)c, p.page_size) : 0;
    const bool fits = known && a >= 0 && c + a <= room;
    const bool ended = known && a < 0;
    const long long add = fits ? a : 0;
    const long long need = fits ? plan_pages((int)(c + a), p.page_size) - have : 0;
    PlanSums total;
    const PlanSums want = asked + plan_scan({need, add, 0}, wave_sums, &total);
    asked = asked + total;
    const bool pages_ok = need == 0 || want.a <= count, rows_ok = add == 0 || want.b <= p.max_rows;
    const bool in = fits && pages_ok && rows_ok;
    const PlanSums mine = {in ? need : 0, in ? add : 0, ended ? have : 0};
    const PlanSums upto = given + plan_scan(mine, wave_sums, &total);
    given = given + total;
    if (there) {
      row0[r] = (int)(upto.b - mine.b);
      take0[r] = (int)(upto.a - mine.a);
      const long long g = upto.c - mine.c;
      give0[r] = g > INT_MAX ? INT_MAX : (int)g;
      if (blockIdx.x == 0) {
        p.starts[r] = row0[r];
        p.lens[r] = known && !ended ? (int)(c + (in ? a : 0)) : 0;
        p.status[r] = !known ? 2 : ended || in ? 0 : !fits ? 1 : !pages_ok ? 3 : 4;
      }
    }
  }
  const int rows = (int)given.b, taken = (int)given.a;
  const int back = given.c > R - count ? R - count : (int)given.c;
  if (t == 0) {
    row0[p.n_req] = rows;
    take0[p.n_req] = taken;
    give0[p.n_req] = given.c > INT_MAX ? INT_MAX : (int)given.c;
    if (blockIdx.x == 0) {
      p.starts[p.n_req] = rows;
      p.state_out[0] = taken == R ? head : plan_place(head, taken, R);
      p.state_out[1] = count - taken + back;
    }
  }
  __syncthreads();

  const int step = gridDim.x * kPlanThreads, first = blockIdx.x * kPlanThreads + t;
  for (int i = first; i < p.max_rows; i += step) {
    int slot = -1, pos = 0, req = -1;
    if (i < rows) {
      req = plan_find(row0, p.n_req, i);
      const int c = p.cached[req];
      pos = c + (i - row0[req]);
      const int have = plan_pages(c, p.page_size), at = pos / p.page_size;
      const int page = at < have ? p.table[req * p.table_stride + at] : p.ring[plan_place(head, take0[req] + (at - have), R)];
      const long long s = (long long)page * p.page_size + pos % p.page_size;
      if (page >= 0 && s <= INT_MAX) slot = (int)s;
    }
    p.slots[i] = slot;
    p.positions[i] = pos;
    p.requests[i] = req;
  }
  for (int i = first; i < taken; i += step) {
    const int req = plan_find(take0, p.n_req, i);
    const int have = plan_pages(p.cached[req], p.page_size);
    p.table[req * p.table_stride + have + (i - take0[req])] = p.ring[plan_place(head, i, R)];
  }
  for (int i = first; i < back; i += step) {
    const int req = plan_find(give0, p.n_req, i);
    p.ring[plan_place(head, count + i, R)] = p.table[req * p.table_stride + (i - give0[req])];
  }
}

// ---------------------------------------------------------------------------
// Append
// ---------------------------------------------------------------------------
constexpr int kAppThreads = 256;

struct AppArgs {
  const float *q, *k, *v, *cos_t, *sin_t;
  float *q_out;
  void *kc, *vc;
  float *ks, *vs;
  const int *slots, *positions;
  int *bad;
  long long q_stride, k_stride, v_stride, q_out_stride, pst, hst, sst, scp, sch, scs;
  int rows, n_heads, n_kv, hd, n_pos, page_size, n_slots;
  int group, heads_per_block;           // lanes of a head (a power of two), heads of a block
};

template <bool VEC>
__device__ inline void load4(float (&x)[4], const float *p) {
  if constexpr (VEC) {
    const float4 f = *reinterpret_cast<const float4 *>(p);
    x[0] = f.x; x[1] = f.y; x[2] = f.z; x[3] = f.w;
  } else {
    for (int i = 0; i < 4; i++) x[i] = p[i];
  }
}

template <int T>
__device__ inline void store4(void *base, long long at, const float (&x)[4]) {
  if constexpr (T == QLLAMA_KV_F32) {
    *reinterpret_cast<float4 *>(static_cast<float *>(base) + at) = make_float4(x[0], x[1], x[2], x[3]);
  } else if constexpr (T == QLLAMA_KV_F16) {
    ushort4 o;
    o.x = __half_as_ushort(__float2half_rn(x[0])); o.y = __half_as_ushort(__float2half_rn(x[1]));
    o.z = __half_as_ushort(__float2half_rn(x[2])); o.w = __half_as_ushort(__float2half_rn(x[3]));
    *reinterpret_cast<ushort4 *>(static_cast<unsigned short *>(base) + at) = o;
  } else {
    ushort4 o;
    unsigned short *e = &o.x;
    for (int i = 0; i < 4; i++) {       // to nearest even; a NaN stays one
      const uint32_t u = __float_as_uint(x[i]);
      e[i] = (u & 0x7fffffffu) > 0x7f800000u ? (unsigned short)((u >> 16) | 0x40)
                                             : (unsigned short)((u + 0x7fffu + ((u >> 16) & 1)) >> 16);
    }
    *reinterpret_cast<ushort4 *>(static_cast<unsigned short *>(base) + at) = o;
  }
}

// quant.c:10-27's code: round to nearest even, clamp; NaN becomes 0
__device__ inline int code(float x) {
  if (x != x) return 0;
  return (int)fminf(fmaxf(rintf(x), -127.0f), 127.0f);
}

// One lane: four pairs (d, d + hd/2) of one head of one row; query heads first, then
// the keys', then the values'.  Memory bound: 4 (2 H + 2 KVH) hd bytes of a row and its
// cache bytes.  int8: the lanes of a head agree on its largest magnitude.  4001 rows of
// 32 + 2 x 8 heads of 128 into an f16 cache: 37.5 us, 4.9 TB/s (a 1 GiB copy: 5.1); 64
// rows 3.0 us, a launch and one trip to memory.  Other caches: 42.2 us f32 (4.7 TB/s), 38.1 bf16,
// 39.1 int8 (4.5 TB/s; 64 rows 3.4).
template <int T, bool VEC>
__global__ __launch_bounds__(kAppThreads) void k_paged_append(AppArgs a) {
  const int row = blockIdx.x;
  const int lane = threadIdx.x % a.group;
  const int head = blockIdx.y * a.heads_per_block + threadIdx.x / a.group;
  const int half = a.hd / 2, d = lane * 4;
  const int heads = a.n_heads + 2 * a.n_kv;
  const bool live = d < half && head < heads;

  const int slot = a.slots[row];
  const int pos = a.cos_t ? a.positions[row] : 0;
  const bool no_pos = a.cos_t && (pos < 0 || pos >= a.n_pos), no_slot = slot >= a.n_slots;
  if (a.bad && (no_pos || no_slot) && blockIdx.y == 0 && threadIdx.x == 0) atomicAdd(a.bad, 1);
  if (no_pos) return;                                   // the whole block: one row
  const bool is_q = head < a.n_heads, is_v = head >= a.n_heads + a.n_kv;
  const int h = is_q ? head : is_v ? head - a.n_heads - a.n_kv : head - a.n_heads;

  float x1[4] = {0, 0, 0, 0}, x2[4] = {0, 0, 0, 0};
  if (live) {
    const float *src = is_q ? a.q + row * a.q_stride : is_v ? a.v + row * a.v_stride : a.k + row * a.k_stride;
    src += (long long)h * a.hd + d;
    load4<VEC>(x1, src);
    load4<VEC>(x2, src + half);
    if (a.cos_t && !is_v) {
      float c[4], s[4];
      load4<VEC>(c, a.cos_t + (long long)pos * half + d);
      load4<VEC>(s, a.sin_t + (long long)pos * half + d);
      for (int i = 0; i < 4; i++) {
        const float y1 = x1[i] * c[i] - x2[i] * s[i], y2 = x2[i] * c[i] + x1[i] * s[i];
        x1[i] = y1;
        x2[i] = y2;
      }
    }
  }
  if (is_q) {
    if (live) {
      float *o = a.q_out + row * a.q_out_stride + (long long)h * a.hd + d;
      if constexpr (VEC) {
        store4<QLLAMA_KV_F32>(o, 0, x1);
        store4<QLLAMA_KV_F32>(o, half, x2);
      } else {
        for (int i = 0; i < 4; i++) { o[i] = x1[i]; o[half + i] = x2[i]; }
      }
    }
    if constexpr (T != QLLAMA_KV_I8) return;
  }
  const bool stored = live && !is_q && slot >= 0 && !no_slot;
  const int page = slot / a.page_size, off = slot % a.page_size;
  const long long at = page * a.pst + h * a.hst + off * a.sst + d;
  void *cache = is_v ? a.vc : a.kc;
  if constexpr (T == QLLAMA_KV_I8) {
    float m = 0.0f;
    for (int i = 0; i < 4; i++) m = fmaxf(m, fmaxf(fabsf(x1[i]), fabsf(x2[i])));
    for (int s = 1; s < a.group; s <<= 1) m = fmaxf(m, __shfl_xor(m, s));
    if (!stored) return;
    const float scale = m > 0.0f ? m * (1.0f / 127.0f) : 1.0f, inv = 1.0f / scale;
    char4 o1, o2;
    o1.x = code(x1[0] * inv); o1.y = code(x1[1] * inv); o1.z = code(x1[2] * inv); o1.w = code(x1[3] * inv);
    o2.x = code(x2[0] * inv); o2.y = code(x2[1] * inv); o2.z = code(x2[2] * inv); o2.w = code(x2[3] * inv);
    *reinterpret_cast<char4 *>(static_cast<signed char *>(cache) + at) = o1;
    *reinterpret_cast<char4 *>(static_cast<signed char *>(cache) + at + half) = o2;
    if (lane == 0) (is_v ? a.vs : a.ks)[page * a.scp + h * a.sch + off * a.scs] = scale;
  } else {
    if (!stored) return;
    store4<T>(cache, at, x1);
    store4<T>(cache, at + half, x2);
  }
}

}  // namespace

extern "C" int qllama_paged_plan(const QPagedPlan *p, void *stream) {
  static const char fn[] = "qllama_paged_plan";
  if (!p) return qs::refuse(fn, "null argument");
  if (p->n_req < 0 || p->n_req > kPlanMaxReq) return qs::refuse(fn, "n_req must be 0 .. 8192");
  if (p->width < 1 || p->page_size < 1 || (int64_t)p->width * p->page_size > INT_MAX)
    return qs::refuse(fn, "bad width or page size (width * page_size must fit in 31 bits)");
  if (p->ring_size < 1 || p->ring_size > (1 << 30) || p->max_rows < 0 || p->max_rows > (1 << 30) || p->table_stride < p->width)
    return qs::refuse(fn, "bad ring size, max_rows (each up to 2^30) or table stride");
  if (!p->state || !p->ring || !p->starts || !p->state_out || (p->n_req && (!p->cached || !p->added || !p->table || !p->lens || !p->status)) ||
      (p->max_rows && (!p->slots || !p->positions || !p->requests)))
    return qs::refuse(fn, "null buffer");
  if (p->state_out == p->state || (p->n_req && (p->lens == p->cached || p->lens == p->added || p->status == p->cached || p->status == p->added)))
    return qs::refuse(fn, "an output is one of the inputs");
  qs::OnDevice on(p->state, (hipStream_t)stream);
  if (on.why) return qs::refuse(fn, on.why);
  // a row or a page a thread, as far as the chip is filled
  const long long most = (long long)p->max_rows + p->n_req;
  const int grid = (int)(most > 256LL * kPlanThreads ? 256 : most < 1 ? 1 : (most + kPlanThreads - 1) / kPlanThreads);
  QS_LAUNCH(fn, k_paged_plan, dim3(grid), dim3(kPlanThreads), 3 * (p->n_req + 1) * sizeof(int), (hipStream_t)stream, *p);
  return 0;
}

template <int T>
static int append_launch(const char *fn, const AppArgs &a, bool vec, hipStream_t stream) {
  const int heads = a.n_heads + 2 * a.n_kv;
  const dim3 grid(a.rows, (heads + a.heads_per_block - 1) / a.heads_per_block);
  if (vec) QS_LAUNCH(fn, (k_paged_append<T, true>), grid, dim3(kAppThreads), 0, stream, a);
  else QS_LAUNCH(fn, (k_paged_append<T, false>), grid, dim3(kAppThreads), 0, stream, a);
  return 0;
}

extern "C" int qllama_paged_append(const QPagedKV *c, const QPagedRows *r, void *stream) {
  static const char fn[] = "qllama_paged_append";
  if (const char *why = qs::bad_cache(c)) return qs::refuse(fn, why);
  if (!r || r->rows < 0 || r->rows > (1 << 23)) return qs::refuse(fn, "null argument, or rows not 0 .. 2^23");
  if (r->rows == 0) return 0;
  if (!r->k || !r->v || !r->slots) return qs::refuse(fn, "null k, v or slots");
  const int H = r->q ? r->n_heads : 0;
  if (r->q && (!r->q_out || H < 1 || H > 65535)) return qs::refuse(fn, "q needs q_out and its number of heads");
  if (r->cos_t && (!r->sin_t || !r->positions || r->n_pos < 1)) return qs::refuse(fn, "a rotation needs cosines, sines and positions");
  const int64_t kvd = (int64_t)c->n_kv * c->head_dim, qd = (int64_t)H * c->head_dim;
  if (r->k_stride < kvd || r->v_stride < kvd || (H && (r->q_stride < qd || r->q_out_stride < qd))) return qs::refuse(fn, "a row stride below the row's length");
  if (qs::misaligned(r->k, 4) || qs::misaligned(r->v, 4) || qs::misaligned(r->q, 4) || qs::misaligned(r->q_out, 4) || qs::misaligned(r->slots, 4) ||
      qs::misaligned(r->positions, 4) || qs::misaligned(r->cos_t, 4) || qs::misaligned(r->sin_t, 4) || qs::misaligned(r->bad, 4))
    return qs::refuse(fn, "a buffer is not aligned to its elements");
  qs::OnDevice on(c->k, (hipStream_t)stream);
  if (on.why) return qs::refuse(fn, on.why);
  AppArgs a;
  a.q = r->q; a.k = r->k; a.v = r->v; a.cos_t = r->cos_t; a.sin_t = r->sin_t; a.q_out = r->q_out;
  a.kc = c->k; a.vc = c->v; a.ks = c->k_scale; a.vs = c->v_scale;
  a.slots = r->slots; a.positions = r->positions; a.bad = r->bad;
  a.q_stride = r->q_stride; a.k_stride = r->k_stride; a.v_stride = r->v_stride; a.q_out_stride = r->q_out_stride;
  a.pst = c->page_stride; a.hst = c->head_stride; a.sst = c->slot_stride;
  a.scp = c->scale_page_stride; a.sch = c->scale_head_stride; a.scs = c->scale_slot_stride;
  a.rows = r->rows; a.n_heads = H; a.n_kv = c->n_kv; a.hd = c->head_dim; a.n_pos = r->n_pos;
  a.page_size = c->page_size; a.n_slots = c->n_pages * c->page_size;
  a.group = 1;
  while (a.group * 8 < c->head_dim) a.group <<= 1;
  a.heads_per_block = kAppThreads / a.group;
  const auto off16 = [](const void *p, int64_t stride) { return p && (qs::misaligned(p, 16) || stride % 4); };
  const bool vec = !(off16(r->k, r->k_stride) || off16(r->v, r->v_stride) || (H && (off16(r->q, r->q_stride) || off16(r->q_out, r->q_out_stride))) ||
                     off16(r->cos_t, 0) || off16(r->sin_t, 0));
  switch (c->type) {
    case QLLAMA_KV_F32: return append_launch<QLLAMA_KV_F32>(fn, a, vec, (hipStream_t)stream);
    case QLLAMA_KV_F16: return append_launch<QLLAMA_KV_F16>(fn, a, vec, (hipStream_t)stream);
    case QLLAMA_KV_BF16: return append_launch<QLLAMA_KV_BF16>(fn, a, vec, (hipStream_t)stream);
    default: return append_launch<QLLAMA_KV_I8>(fn, a, vec, (hipStream_t)stream);
  }
}
