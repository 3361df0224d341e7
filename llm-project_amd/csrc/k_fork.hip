// k_fork.hip - pages that several requests hold, and rows of the cache to other slots
// (qllama_paged_fork, qllama_paged_move; semantics in qserve.h).  No counterpart in the
// reference, whose cache is one dense array per sequence (llama.c:275-288).
#include <hip/hip_runtime.h>

#include "qserve_host.h"

namespace {

// ---------------------------------------------------------------------------
// Fork
// ---------------------------------------------------------------------------
constexpr int kForkThreads = 256, kForkPlanThreads = 1024;
constexpr int kForkOne = 64, kForkOneWidth = 256;        // requests, and table entries of each, that one block takes

constexpr int kNoPage = -1, kNoCopy = -2, kRefused = -3;          // the ring names no page, none is needed, none is left

struct ForkArgs {
  QPagedFork p;
  unsigned long long *best, *first;      // of a page: the new holder with most of it, the first old one
  int *holders;                          // of a page, as far as they are counted
  int *got;                              // of a new request: the page for its copy, or one of those below
  int *freed;                            // of an old request: pages that it is the first to give back
  int *taken;                            // pages taken from the ring
};

__device__ inline int fork_len(const QPagedFork &p, int r) { return min(max(p.lens[r], 0), p.width * p.page_size); }
__device__ inline int fork_pages(const QPagedFork &p, int len) { return (int)(((unsigned)len + (unsigned)p.page_size - 1u) / (unsigned)p.page_size); }
// Source of new request i (-1: none) and its tokens.
__device__ inline int fork_source(const QPagedFork &p, int i, int *tokens) {
  int r = p.from[i];
  if (r < 0 || r >= p.n_old) r = -1;
  *tokens = r < 0 ? 0 : p.keep ? min(max(p.keep[i], 0), fork_len(p, r)) : fork_len(p, r);
  return r;
}
__device__ inline int fork_page(const QPagedFork &p, int r, int e) {
  const int page = p.table[r * p.table_stride + e];
  return page >= 0 && page < p.n_pages ? page : -1;
}
__device__ inline void fork_ring(const QPagedFork &p, int *head, int *count) {
  *head = p.state[0] < 0 || p.state[0] >= p.ring_size ? 0 : p.state[0];
  *count = min(max(p.state[1], 0), p.ring_size);
}
__device__ inline int ring_place(int x, int y, int R) {        // x + y of a ring of R, x < R, y <= R
  const unsigned s = (unsigned)x + (unsigned)y;
  return (int)(s >= (unsigned)R ? s - (unsigned)R : s);
}
__device__ inline unsigned long long fork_id(const QPagedFork &p, int r, int e) { return ~((unsigned long long)r * p.width + e); }
// What new request i holds of a page, above what others hold: more of its tokens, then a smaller i.
__device__ inline unsigned long long fork_rank(int covered, int i) { return (unsigned long long)covered << 32 | (0xffffffffu - (unsigned)i); }

// The steps of a fork, each over all entries of the requests' tables.  Where there are few
// requests with short tables one block takes all steps, a wave a request at a time; else every
// step is a launch, with a block a request.  One block against six launches, whose enqueueing
// takes the host 15 us more, us with 16, 256 and 1024 pages each: 2 old and 2 new requests 8
// against 14, 14 against 14, 36 against 22; 16 and 16 10 against 15, 20 against 16, 55 against 23;
// 32 and 32 17 against 17, 32 against 17 (with 512: 55 against 19); 256 and 256 with 40 more than
// 100 against 20.  How many pages a request has the host does not know, only how many its table
// has room for.
// Of what a step hands to the next: in the L2, also within one launch.
template <typename T>
__device__ inline T load(const T *p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
template <typename T>
__device__ inline void store(T *p, T x) { __hip_atomic_store(p, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

struct Span { int row, rows, entry, entries; };       // first request and entry, and steps between them

// The pages in hand are cleared, ...
__device__ inline void fork_clear(const ForkArgs &a, Span s) {
  const QPagedFork &p = a.p;
  for (int r = s.row; r < p.n_old; r += s.rows) {
    const int have = fork_pages(p, fork_len(p, r));
    for (int e = s.entry; e < have; e += s.entries) {
      const int page = fork_page(p, r, e);
      if (page < 0) continue;
      store(a.holders + page, p.extra[page] + 1);
      store(a.best + page, 0ull);
      store(a.first + page, 0ull);
    }
  }
}

// ... then the old holders are taken off, which leaves those outside the call, and new ones ranked, ...
__device__ inline void fork_rank_all(const ForkArgs &a, Span s) {
  const QPagedFork &p = a.p;
  for (int x = s.row; x < p.n_old + p.n_new; x += s.rows) {
    if (x < p.n_old) {
      const int have = fork_pages(p, fork_len(p, x));
      for (int e = s.entry; e < have; e += s.entries) {
        const int page = fork_page(p, x, e);
        if (page < 0) continue;
        atomicSub(a.holders + page, 1);
        atomicMax(a.first + page, fork_id(p, x, e));
      }
    } else {
      const int i = x - p.n_old;
      int tokens;
      const int r = fork_source(p, i, &tokens), want = fork_pages(p, tokens);
      for (int e = s.entry; e < want; e += s.entries) {
        const int page = fork_page(p, r, e);
        if (page >= 0) atomicMax(a.best + page, fork_rank(min(p.page_size, tokens - e * p.page_size), i));
      }
    }
  }
}

// ... copies decided and their pages taken, request by request, by one block; all threads return the pages taken, ...
__device__ int fork_copies(const ForkArgs &a) {
  const QPagedFork &p = a.p;
  __shared__ int wave_sums[kForkPlanThreads / 64];
  const int t = threadIdx.x, lane = t & 63, w = t >> 6;
  int head, count;
  fork_ring(p, &head, &count);
  int asked = 0;                         // by the requests before this pass
  for (int i0 = 0; i0 < p.n_new; i0 += kForkPlanThreads) {
    const int i = i0 + t;
    int tokens = 0, r = -1, page = -1, part = 0;
    if (i < p.n_new) {
      r = fork_source(p, i, &tokens);
      part = tokens % p.page_size;
      if (part) page = fork_page(p, r, tokens / p.page_size);
    }
    const bool copies = page >= 0 && (load(a.holders + page) > 0 || load(a.best + page) != fork_rank(part, i));
    const uint64_t wanting = __ballot(copies);
    __syncthreads();                     // the sums of the pass before have been read
    if (lane == 0) wave_sums[w] = __popcll(wanting);
    __syncthreads();
    // requests are admitted up to a border, so a request's place among the free pages is that among all that ask
    int place = asked + __popcll(wanting & ((1ull << lane) - 1));
    for (int j = 0; j < kForkPlanThreads / 64; j++) {
      if (j < w) place += wave_sums[j];
      asked += wave_sums[j];
    }
    const bool refused = copies && place >= count, in = copies && !refused;
    if (i < p.n_new) {
      const int got = in ? p.ring[ring_place(head, place, p.ring_size)] : -1;
      const bool there = in && got >= 0 && got < p.n_pages;
      store(a.got + i, refused ? kRefused : there ? got : in ? kNoPage : kNoCopy);
      p.lens_out[i] = refused ? 0 : tokens;
      p.status[i] = refused ? 3 : 0;
      p.src[i] = there ? page * p.page_size : -1;
      p.dst[i] = there ? got * p.page_size : -1;
      p.count[i] = there ? part : 0;
    }
  }
  return min(asked, count);
}

// ... what every new request holds written down, ...
__device__ inline void fork_hold(const ForkArgs &a, Span s) {
  const QPagedFork &p = a.p;
  for (int i = s.row; i < p.n_new; i += s.rows) {
    const int got = load(a.got + i);
    if (got == kRefused) continue;
    int tokens;
    const int r = fork_source(p, i, &tokens), want = fork_pages(p, tokens);
    for (int e = s.entry; e < want; e += s.entries) {
      int page = fork_page(p, r, e);
      if (got != kNoCopy && e == want - 1) page = got;
      else if (page >= 0) atomicAdd(a.holders + page, 1);
      p.table_out[i * p.table_out_stride + e] = page;
    }
  }
}

// Whether old request r is the one to give back the page of its entry e.
__device__ inline bool fork_gone(const ForkArgs &a, int r, int e, int page) { return page >= 0 && load(a.holders + page) <= 0 && load(a.first + page) == fork_id(a.p, r, e); }

// ... and pages that no one holds any more counted and put at the ring's back, row by row.
// The state behind the call: `taken` pages from the front, `all` to the back, as far as there is room.
__device__ inline void fork_state(const QPagedFork &p, int head, int count, int taken, long long all) {
  const int room = p.ring_size - count;
  p.state_out[0] = ring_place(head, taken, p.ring_size);
  p.state_out[1] = count - taken + (int)(all < room ? all : room);
}

__device__ inline void fork_between() {
  __builtin_amdgcn_s_waitcnt(0);         // what this wave has written is in the L2, from where the counts below are read
  __syncthreads();
}
// All steps by one block.  (With fences of the whole device between them it took 32 us.)
__global__ __launch_bounds__(kForkPlanThreads) void k_fork_one(ForkArgs a) {
  const QPagedFork &p = a.p;
  __shared__ int sums[kForkPlanThreads / 64], before[kForkPlanThreads];
  const int t = threadIdx.x, lane = t & 63, w = t >> 6;
  const Span all = {w, kForkPlanThreads / 64, lane, 64};
  if (p.extra_out != p.extra)
    for (int i = t; i < p.n_pages; i += kForkPlanThreads) p.extra_out[i] = p.extra[i];
  fork_clear(a, all);
  fork_between();
  fork_rank_all(a, all);
  fork_between();
  const int taken = fork_copies(a);
  fork_between();
  fork_hold(a, all);
  fork_between();
  for (int r = w; r < p.n_old; r += kForkPlanThreads / 64) {
    const int have = fork_pages(p, fork_len(p, r));
    int n = 0;
    for (int e0 = 0; e0 < have; e0 += 64) {
      const int page = e0 + lane < have ? fork_page(p, r, e0 + lane) : -1;
      if (page >= 0) p.extra_out[page] = max(load(a.holders + page) - 1, 0);
      n += __popcll(__ballot(fork_gone(a, r, e0 + lane, page)));
    }
    if (lane == 0) before[r] = n;
  }
  __syncthreads();
  const int mine = t < p.n_old ? before[t] : 0;
  int upto = mine;
  for (int d = 1; d < 64; d <<= 1) {
    const int x = __shfl_up(upto, d);
    if (lane >= d) upto += x;
  }
  if (lane == 63) sums[w] = upto;
  __syncthreads();
  for (int j = 0; j < w; j++) upto += sums[j];
  before[t] = upto - mine;
  int head, count;
  fork_ring(p, &head, &count);
  const int room = p.ring_size - count;
  if (t == kForkPlanThreads - 1) fork_state(p, head, count, taken, upto);
  __syncthreads();
  for (int r = w; r < p.n_old; r += kForkPlanThreads / 64) {
    const int have = fork_pages(p, fork_len(p, r));
    int at = before[r];
    for (int e0 = 0; e0 < have; e0 += 64) {
      const int page = e0 + lane < have ? fork_page(p, r, e0 + lane) : -1;
      const bool gone = fork_gone(a, r, e0 + lane, page);
      const uint64_t which = __ballot(gone);
      const int place = at + __popcll(which & ((1ull << lane) - 1));
      if (gone && place < room) p.ring[ring_place(ring_place(head, count, p.ring_size), place, p.ring_size)] = page;
      at += __popcll(which);
    }
  }
}

__device__ inline Span fork_block() { return {(int)blockIdx.x, (int)gridDim.x, (int)threadIdx.x, kForkThreads}; }
__global__ __launch_bounds__(kForkThreads) void k_fork_clear(ForkArgs a) {
  fork_clear(a, fork_block());
  if (a.p.extra_out != a.p.extra)
    for (int i = blockIdx.x * kForkThreads + threadIdx.x; i < a.p.n_pages; i += gridDim.x * kForkThreads) a.p.extra_out[i] = a.p.extra[i];
}
__global__ __launch_bounds__(kForkThreads) void k_fork_rank(ForkArgs a) { fork_rank_all(a, fork_block()); }
__global__ __launch_bounds__(kForkPlanThreads) void k_fork_copies(ForkArgs a) {
  const int taken = fork_copies(a);
  if (threadIdx.x == 0) *a.taken = taken;
}
__global__ __launch_bounds__(kForkThreads) void k_fork_hold(ForkArgs a) { fork_hold(a, fork_block()); }
__global__ __launch_bounds__(kForkThreads) void k_fork_count(ForkArgs a) {
  const QPagedFork &p = a.p;
  const int r = blockIdx.x, have = fork_pages(p, fork_len(p, r));
  int n = 0;
  for (int e0 = 0; e0 < have; e0 += kForkThreads) {
    const int e = e0 + threadIdx.x;
    const int page = e < have ? fork_page(p, r, e) : -1;
    if (page >= 0) p.extra_out[page] = max(load(a.holders + page) - 1, 0);
    n += __syncthreads_count(fork_gone(a, r, e, page));
  }
  if (threadIdx.x == 0) a.freed[r] = n;
}
__global__ __launch_bounds__(kForkThreads) void k_fork_free(ForkArgs a) {
  const QPagedFork &p = a.p;
  __shared__ int sums[kForkThreads / 64];
  const int r = blockIdx.x, t = threadIdx.x, lane = t & 63, w = t >> 6;
  int head, count;
  fork_ring(p, &head, &count);
  long long at = 0;                        // pages of the rows before
  for (int i0 = 0; i0 < r; i0 += kForkThreads) {
    int x = i0 + t < r ? a.freed[i0 + t] : 0;
    for (int d = 32; d; d >>= 1) x += __shfl_xor(x, d);
    __syncthreads();
    if (lane == 0) sums[w] = x;
    __syncthreads();
    for (int j = 0; j < kForkThreads / 64; j++) at += sums[j];
  }
  const int room = p.ring_size - count;
  if (t == 0 && r + 1 == p.n_old) fork_state(p, head, count, *a.taken, at + a.freed[r]);
  const int have = fork_pages(p, fork_len(p, r));
  for (int e0 = 0; e0 < have; e0 += kForkThreads) {
    const int e = e0 + t;
    const int page = e < have ? fork_page(p, r, e) : -1;
    const bool gone = fork_gone(a, r, e, page);
    const uint64_t all = __ballot(gone);
    __syncthreads();
    if (lane == 0) sums[w] = __popcll(all);
    __syncthreads();
    long long mine = at + __popcll(all & ((1ull << lane) - 1));
    for (int j = 0; j < kForkThreads / 64; j++) {
      if (j < w) mine += sums[j];
      at += sums[j];
    }
    if (gone && mine < room) p.ring[ring_place(ring_place(head, count, p.ring_size), (int)mine, p.ring_size)] = page;
  }
}

// ---------------------------------------------------------------------------
// Moves
// ---------------------------------------------------------------------------
constexpr int kMoveThreads = 256, kMoveCaches = 64, kAhead = 8;

struct MoveArgs {
  struct { char *k, *v; float *ks, *vs; } c[kMoveCaches];
  const int *src, *dst, *count, *starts;
  int *bad;
  long long pst, hst, sst;                // bytes
  long long scp, sch, scs;                // floats
  int n_moves, n_groups, n_kv, page_size, n_slots;
  int per_row, units;                     // of a row of one head; of a slot, keys and values
  int scales, first;                      // n_kv floats of keys and as many of values; whether the first launch counts bad moves
};

template <int U> struct Unit;
template <> struct Unit<16> { using type = uint4; };
template <> struct Unit<8> { using type = uint2; };

// Whether n slots from src can go to dst; *bad counts those that leave the cache.
__device__ inline bool move_fits(const MoveArgs &a, int src, int dst, int n, bool *bad) {
  *bad = false;
  if (src < 0 || dst < 0 || n <= 0) return false;
  *bad = n > a.n_slots || src > a.n_slots - n || dst > a.n_slots - n;
  return !*bad;
}

// Address of unit u of a slot (scales are 4-byte units behind the others).
__device__ inline long long move_at(const MoveArgs &a, int slot, int head, int x, int unit_bytes) {
  const int page = slot / a.page_size, place = slot - page * a.page_size;
  return page * a.pst + head * a.hst + place * a.sst + (long long)x * unit_bytes;
}
__device__ inline long long move_scale_at(const MoveArgs &a, int slot, int head) {
  const int page = slot / a.page_size, place = slot - page * a.page_size;
  return page * a.scp + head * a.sch + place * a.scs;
}

// Independent moves: a block a move and cache (and share of its slots), a thread a unit of
// 16 bytes of one slot's row of one head.  256 moves of 7 slots on average in 16 caches (8 heads of
// 64 bf16) take 18 us: 36 MB read and written in pieces of 128 bytes to 2 KB, 2 TB/s, 9 us at a
// copy's rate.  A wave a head, four heads under way at a time, took 24, a block for four caches
// with their loads under way together 30.
template <int U>
__global__ __launch_bounds__(kMoveThreads) void k_move(MoveArgs a) {
  using T = typename Unit<U>::type;
  const int i = blockIdx.x, src = a.src[i], dst = a.dst[i], n = a.count ? a.count[i] : 1;
  bool bad;
  const bool fits = move_fits(a, src, dst, n, &bad);
  if (bad && a.bad && a.first && blockIdx.y == 0 && blockIdx.z == 0 && threadIdx.x == 0) atomicAdd(a.bad, 1);
  if (!fits) return;
  const auto &c = a.c[blockIdx.y];
  const int per_slot = a.units + a.scales;
  const long long all = (long long)n * per_slot;
  const bool small = all <= INT_MAX;       // a division of 32 bits
  for (long long u = blockIdx.z * kMoveThreads + threadIdx.x; u < all; u += gridDim.z * kMoveThreads) {
    const int s = small ? (int)u / per_slot : (int)(u / per_slot);
    int x = (int)(u - (long long)s * per_slot);
    if (x < a.units) {
      char *base = x < a.units / 2 ? c.k : c.v;
      if (x >= a.units / 2) x -= a.units / 2;
      const int head = x / a.per_row, at = x - head * a.per_row;
      *reinterpret_cast<T *>(base + move_at(a, dst + s, head, at, U)) = *reinterpret_cast<const T *>(base + move_at(a, src + s, head, at, U));
    } else {
      x -= a.units;
      float *base = x < a.n_kv ? c.ks : c.vs;
      if (x >= a.n_kv) x -= a.n_kv;
      base[move_scale_at(a, dst + s, x)] = base[move_scale_at(a, src + s, x)];
    }
  }
}

// Moves one after another: a thread takes its unit through all moves of a group, eight
// loads at a time; what an earlier one of the eight stores goes to a later load of that
// slot in registers, so the result is that of single steps.
template <int U>
__global__ __launch_bounds__(kMoveThreads) void k_move_groups(MoveArgs a) {
  using T = typename Unit<U>::type;
  const int g = blockIdx.x;
  const int from = min(max(a.starts[g], 0), a.n_moves), to = min(max(a.starts[g + 1], 0), a.n_moves);
  const auto &c = a.c[blockIdx.y];
  int x = blockIdx.z * kMoveThreads + threadIdx.x;
  const bool counts = a.bad && a.first && blockIdx.y == 0 && blockIdx.z == 0 && threadIdx.x == 0;
  const bool live = x < a.units + a.scales, scale = x >= a.units;
  char *base = nullptr;
  int head = 0, at = 0;
  if (live && !scale) {
    base = x < a.units / 2 ? c.k : c.v;
    if (x >= a.units / 2) x -= a.units / 2;
    head = x / a.per_row;
    at = x - head * a.per_row;
  } else if (live) {
    x -= a.units;
    base = reinterpret_cast<char *>(x < a.n_kv ? c.ks : c.vs);
    head = x < a.n_kv ? x : x - a.n_kv;
  }
  for (int m = from; m < to; m += kAhead) {
    int src[kAhead], dst[kAhead];
    T v[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; j++) {
      src[j] = m + j < to ? a.src[m + j] : -1;
      dst[j] = m + j < to ? a.dst[m + j] : -1;
      bool bad;
      if (!move_fits(a, src[j], dst[j], 1, &bad)) src[j] = dst[j] = -1;
      if (bad && counts) atomicAdd(a.bad, 1);
    }
    if (!live) continue;
#pragma unroll
    for (int j = 0; j < kAhead; j++) {
      if (src[j] < 0) continue;
      if (scale) v[j].x = *reinterpret_cast<const uint32_t *>(base + 4 * move_scale_at(a, src[j], head));
      else v[j] = *reinterpret_cast<const T *>(base + move_at(a, src[j], head, at, U));
    }
#pragma unroll
    for (int j = 0; j < kAhead; j++)
#pragma unroll
      for (int k = 0; k < j; k++)
        if (src[j] >= 0 && dst[k] == src[j]) v[j] = v[k];
#pragma unroll
    for (int j = 0; j < kAhead; j++) {
      if (src[j] < 0) continue;
      if (scale) *reinterpret_cast<uint32_t *>(base + 4 * move_scale_at(a, dst[j], head)) = v[j].x;
      else *reinterpret_cast<T *>(base + move_at(a, dst[j], head, at, U)) = v[j];
    }
  }
}

}  // namespace

extern "C" size_t qllama_paged_fork_work(int n_old, int n_new, int n_pages) {
  if (n_old < 0 || n_old > 8192 || n_new < 0 || n_new > 8192 || n_pages < 1) return 0;
  return (size_t)n_pages * 20 + ((size_t)n_old + n_new + 1) * 4 + 16;
}

extern "C" int qllama_paged_fork(const QPagedFork *p, void *stream) {
  static const char fn[] = "qllama_paged_fork";
  if (!p) return qs::refuse(fn, "null argument");
  if (p->n_old < 0 || p->n_old > 8192 || p->n_new < 0 || p->n_new > 8192) return qs::refuse(fn, "n_old and n_new must be 0 .. 8192");
  if (p->width < 1 || p->page_size < 1 || (int64_t)p->width * p->page_size > INT_MAX)
    return qs::refuse(fn, "bad width or page size (width * page_size must fit in 31 bits)");
  if (p->n_pages < 1 || (int64_t)p->n_pages * p->page_size > INT_MAX) return qs::refuse(fn, "bad number of pages (n_pages * page_size must fit in 31 bits)");
  if (p->ring_size < 1 || p->ring_size > (1 << 30) || p->table_stride < p->width || p->table_out_stride < p->width)
    return qs::refuse(fn, "bad ring size (up to 2^30) or table stride");
  const void *all[] = {p->extra, p->state, p->ring, p->extra_out, p->state_out};
  const void *old[] = {p->lens, p->table}, *made[] = {p->from, p->table_out, p->lens_out, p->status, p->src, p->dst, p->count};
  for (const void *x : all)
    if (!x || qs::misaligned(x, 4)) return qs::refuse(fn, "a buffer is null or not aligned to its elements");
  for (const void *x : old)
    if (p->n_old && (!x || qs::misaligned(x, 4))) return qs::refuse(fn, "a buffer is null or not aligned to its elements");
  for (const void *x : made)
    if (p->n_new && (!x || qs::misaligned(x, 4))) return qs::refuse(fn, "a buffer is null or not aligned to its elements");
  if (qs::misaligned(p->keep, 4)) return qs::refuse(fn, "a buffer is null or not aligned to its elements");
  if (p->state_out == p->state) return qs::refuse(fn, "an output is one of the inputs");
  for (const void *x : {(const void *)p->table_out, (const void *)p->lens_out, (const void *)p->status, (const void *)p->src, (const void *)p->dst, (const void *)p->count})
    if (p->n_new && (x == p->table || x == p->lens || x == p->from || x == p->keep || x == p->extra || x == p->ring))
      return qs::refuse(fn, "an output is one of the inputs");
  if (!p->work || qs::misaligned(p->work, 16) || p->work_bytes < qllama_paged_fork_work(p->n_old, p->n_new, p->n_pages))
    return qs::refuse(fn, "work is missing, misaligned or smaller than qllama_paged_fork_work");
  qs::OnDevice on(p->state, (hipStream_t)stream);
  if (on.why) return qs::refuse(fn, on.why);
  ForkArgs a;
  a.p = *p;
  a.best = static_cast<unsigned long long *>(p->work);
  a.first = a.best + p->n_pages;
  a.holders = reinterpret_cast<int *>(a.first + p->n_pages);
  a.got = a.holders + p->n_pages;
  a.freed = a.got + p->n_new;
  a.taken = a.freed + p->n_old;
  const hipStream_t s = (hipStream_t)stream;
  const int copy = p->extra_out == p->extra ? 0 : (p->n_pages + kForkThreads - 1) / kForkThreads, clear = copy > 256 ? 256 : copy;
  if (p->n_old == 0 && copy > 64) {      // more counts than one block should copy
    QS_LAUNCH(fn, k_fork_clear, dim3(clear), dim3(kForkThreads), 0, s, a);
    a.p.extra = a.p.extra_out;
  }
  if (p->n_old == 0 || (p->n_old + p->n_new <= kForkOne && p->width <= kForkOneWidth && p->n_pages <= 16384)) {
    QS_LAUNCH(fn, k_fork_one, dim3(1), dim3(kForkPlanThreads), 0, s, a);
    return 0;
  }
  QS_LAUNCH(fn, k_fork_clear, dim3(p->n_old > clear ? p->n_old : clear), dim3(kForkThreads), 0, s, a);
  QS_LAUNCH(fn, k_fork_rank, dim3(p->n_old + p->n_new), dim3(kForkThreads), 0, s, a);
  QS_LAUNCH(fn, k_fork_copies, dim3(1), dim3(kForkPlanThreads), 0, s, a);
  if (p->n_new) QS_LAUNCH(fn, k_fork_hold, dim3(p->n_new), dim3(kForkThreads), 0, s, a);
  QS_LAUNCH(fn, k_fork_count, dim3(p->n_old), dim3(kForkThreads), 0, s, a);
  QS_LAUNCH(fn, k_fork_free, dim3(p->n_old), dim3(kForkThreads), 0, s, a);
  return 0;
}

extern "C" int qllama_paged_move(const QPagedKV *caches, int n_caches, const QPagedMoves *m, void *stream) {
  static const char fn[] = "qllama_paged_move";
  if (!caches || n_caches < 0 || !m) return qs::refuse(fn, "null argument or n_caches < 0");
  for (int i = 0; i < n_caches; i++) {
    const QPagedKV *c = caches + i;
    if (const char *why = qs::bad_cache(c)) return qs::refuse(fn, why);
    if (c->type != caches->type || c->n_pages != caches->n_pages || c->page_size != caches->page_size || c->n_kv != caches->n_kv ||
        c->head_dim != caches->head_dim || c->page_stride != caches->page_stride || c->head_stride != caches->head_stride ||
        c->slot_stride != caches->slot_stride ||
        (c->type == QLLAMA_KV_I8 && (c->scale_page_stride != caches->scale_page_stride || c->scale_head_stride != caches->scale_head_stride ||
                                     c->scale_slot_stride != caches->scale_slot_stride)))
      return qs::refuse(fn, "the caches must be alike in type, sizes and strides");
  }
  if (m->n_moves < 0 || m->n_moves > (1 << 23) || (m->starts && (m->n_groups < 0 || m->n_groups > (1 << 23))))
    return qs::refuse(fn, "n_moves and n_groups must be 0 .. 2^23");
  if (m->starts && m->count) return qs::refuse(fn, "moves in groups have no count");
  if (n_caches == 0 || m->n_moves == 0 || (m->starts && m->n_groups == 0)) return 0;
  if (!m->src || !m->dst || qs::misaligned(m->src, 4) || qs::misaligned(m->dst, 4) || qs::misaligned(m->count, 4) || qs::misaligned(m->starts, 4) ||
      qs::misaligned(m->bad, 4))
    return qs::refuse(fn, "a buffer is null or not aligned to its elements");
  qs::OnDevice on(caches->k, (hipStream_t)stream);
  if (on.why) return qs::refuse(fn, on.why);
  const QPagedKV *c = caches;
  const int es = c->type == QLLAMA_KV_F32 ? 4 : c->type == QLLAMA_KV_I8 ? 1 : 2;
  MoveArgs a;
  a.src = m->src; a.dst = m->dst; a.count = m->count; a.starts = m->starts; a.bad = m->bad;
  a.pst = c->page_stride * es; a.hst = c->head_stride * es; a.sst = c->slot_stride * es;
  a.scp = c->scale_page_stride; a.sch = c->scale_head_stride; a.scs = c->scale_slot_stride;
  a.n_moves = m->n_moves; a.n_groups = m->n_groups; a.n_kv = c->n_kv; a.page_size = c->page_size; a.n_slots = c->n_pages * c->page_size;
  a.scales = c->type == QLLAMA_KV_I8 ? 2 * c->n_kv : 0;
  // rows and strides are multiples of 8 elements: of 16 bytes but for int8
  const bool wide = ((c->head_dim * es) | a.pst | a.hst | a.sst) % 16 == 0;
  a.per_row = c->head_dim * es / (wide ? 16 : 8);
  a.units = 2 * c->n_kv * a.per_row;
  for (int first = 0; first < n_caches; first += kMoveCaches) {
    const int n = n_caches - first < kMoveCaches ? n_caches - first : kMoveCaches;
    for (int i = 0; i < n; i++) a.c[i] = {static_cast<char *>(caches[first + i].k), static_cast<char *>(caches[first + i].v), caches[first + i].k_scale, caches[first + i].v_scale};
    a.first = first == 0;
    if (m->starts) {
      const dim3 grid(m->n_groups, n, (a.units + a.scales + kMoveThreads - 1) / kMoveThreads);
      QS_LAUNCH(fn, (wide ? k_move_groups<16> : k_move_groups<8>), grid, dim3(kMoveThreads), 0, (hipStream_t)stream, a);
    } else {
      // few moves: their slots over several blocks
      const long long blocks = (long long)m->n_moves * n;
      const dim3 grid(m->n_moves, n, !m->count || blocks >= 1024 ? 1 : blocks >= 128 ? 4 : 16);
      QS_LAUNCH(fn, (wide ? k_move<16> : k_move<8>), grid, dim3(kMoveThreads), 0, (hipStream_t)stream, a);
    }
  }
  return 0;
}
