// k_rules.hip - penalties for tokens that were used, biases and masks on rows of logits
// (qllama_logit_rules; semantics in qserve.h).  No counterpart in the reference, whose
// sampler (sampler.c:54-143) takes logits as they are.
//
// Memory bound: 8 bytes a logit.  A block takes a slice of a row: its logits are under way
// in registers while the row's history is counted into LDS, a counter a token of the slice
// (every block of a row reads the whole history, 4 bytes a token out of L2), then every
// thread looks at its tokens' counters and the mask's bits.  The few tokens that a rule
// touches are evaluated in 64 bits.  192 rows of 128256 with histories of up to 8000 tokens,
// biases and masks: 44 us, 4.6 TB/s (a 1 GiB copy: 5.1); 9 rows each of 40 trees, 32000
// tokens: 21.6 us, 3.7 TB/s; 4 rows 5.1 us, a launch and three trips to memory.
#include <hip/hip_runtime.h>

#include "qserve_host.h"

namespace {

constexpr int kThreads = 512, kAhead = 8;
constexpr uint32_t kBiased = 1u << 30, kCount = kBiased - 1, kPrompt = 1u << 31;

__device__ inline float setting(const float *p, int r, float none) {
  const float x = p ? p[r] : none;
  return x == x ? x : none;
}

// K: float4s of a thread; VEC: rows are 16-byte aligned; USED: there is a history, a tree or a bias
template <int K, bool VEC, bool USED>
__global__ __launch_bounds__(kThreads) void k_rules(QLogitRules p) {
  constexpr int SLICE = 4 * K * kThreads;
  __shared__ __align__(16) uint32_t used[USED ? SLICE : 4];
  const int i = blockIdx.y, lo = blockIdx.x * SLICE, t = threadIdx.x, lane = t & 63;
  const int r = p.requests ? p.requests[i] : i;
  if (r < 0 || r >= p.n_req) return;
  const float *row = p.logits + i * p.stride + lo;
  float *out = p.out + i * p.out_stride + lo;
  const int n = min(SLICE, p.vocab - lo);

  float x[K][4];
#pragma unroll
  for (int k = 0; k < K; k++) {
    const int at = 4 * (k * kThreads + t);
    if (VEC && at + 4 <= n) {
      const float4 f = *reinterpret_cast<const float4 *>(row + at);
      x[k][0] = f.x; x[k][1] = f.y; x[k][2] = f.z; x[k][3] = f.w;
    } else {
#pragma unroll
      for (int j = 0; j < 4; j++) x[k][j] = at + j < n ? row[at + j] : 0.0f;
    }
  }
  const int m = p.allowed ? p.allowed_rows[i] : -1;
  const uint32_t *allowed = m >= 0 && m < p.n_masks ? p.allowed + m * p.allowed_stride : nullptr;
  uint32_t bits[K];
#pragma unroll
  for (int k = 0; k < K; k++) {
    const int at = 4 * (k * kThreads + t);
    bits[k] = allowed && at < n ? allowed[(lo + at) >> 5] >> (at & 31) : 0xfu;      // lo is a multiple of 32
  }

  const float rep0 = setting(p.repetition, r, 1.0f), pres = setting(p.presence, r, 0.0f), freq = setting(p.frequency, r, 0.0f);
  const float rep = rep0 > 0.0f ? rep0 : 1.0f;
  if constexpr (USED) {
#pragma unroll
    for (int k = 0; k < K; k++) *reinterpret_cast<uint4 *>(used + 4 * (k * kThreads + t)) = make_uint4(0, 0, 0, 0);
    __syncthreads();
    if (rep != 1.0f || pres != 0.0f || freq != 0.0f) {
      if (p.tokens) {
        const int *tokens = p.tokens + r * p.token_stride;
        const int len = min(max(p.n_tokens[r], 0), p.capacity), prompt = p.n_prompt ? min(max(p.n_prompt[r], 0), len) : 0;
        for (int j0 = t; j0 < len; j0 += kAhead * kThreads) {          // several loads under way at a time
          int token[kAhead];
#pragma unroll
          for (int k = 0; k < kAhead; k++) token[k] = j0 + k * kThreads < len ? tokens[j0 + k * kThreads] : -1;
#pragma unroll
          for (int k = 0; k < kAhead; k++) {
            const unsigned at = (unsigned)token[k] - (unsigned)lo;
            if (at < (unsigned)n && token[k] >= 0) {
              if (j0 + k * kThreads < prompt) atomicOr(used + at, kPrompt);
              else atomicAdd(used + at, 1u);
            }
          }
        }
      }
      if (p.mask && t < 64 * p.words) {
        const int a = min(max(p.starts[r], 0), p.rows), b = min(max(p.starts[r + 1], 0), p.rows);
        if ((p.mask[(int64_t)i * p.words + (t >> 6)] >> (t & 63) & 1) && a + t < b) {
          const int token = p.drafted[a + t];
          const unsigned at = (unsigned)token - (unsigned)lo;
          if (at < (unsigned)n && token >= 0) atomicAdd(used + at, 1u);
        }
      }
    }
    for (int j = t; j < p.n_bias; j += kThreads) {
      const int token = p.bias_tokens[r * p.bias_stride + j];
      const unsigned at = (unsigned)token - (unsigned)lo;
      if (at < (unsigned)n && token >= 0) atomicOr(used + at, kBiased);
    }
    __syncthreads();
  }

#pragma unroll
  for (int k = 0; k < K; k++) {
    const int at = 4 * (k * kThreads + t);
    if constexpr (USED) {
      const uint4 u4 = *reinterpret_cast<const uint4 *>(used + at);
      const uint32_t u[4] = {u4.x, u4.y, u4.z, u4.w};
#pragma unroll
      for (int j = 0; j < 4; j++) {
        float bias = 0.0f;
        // the wave looks for the first entry of each of its biased tokens, 64 at a time
        for (uint64_t todo = __ballot((u[j] & kBiased) != 0); todo; todo &= todo - 1) {
          const int who = __builtin_ctzll(todo), token = __shfl(lo + at + j, who);
          for (int b0 = 0; b0 < p.n_bias; b0 += 64) {
            const bool is = b0 + lane < p.n_bias && p.bias_tokens[r * p.bias_stride + b0 + lane] == token;
            const uint64_t found = __ballot(is);
            if (found) {
              if (lane == who) bias = p.bias[r * p.bias_stride + b0 + __builtin_ctzll(found)];
              break;
            }
          }
        }
        if (u[j]) {
          double y = x[k][j];
          const uint32_t times = u[j] & kCount;
          if (u[j] & ~kBiased) y = x[k][j] > 0.0f ? y / rep : y * rep;
          if (times) y -= (double)freq * times + pres;
          if (bias == bias) y += bias;
          x[k][j] = (float)y;
        }
      }
    }
#pragma unroll
    for (int j = 0; j < 4; j++)
      if (!(bits[k] >> j & 1)) x[k][j] = -__builtin_inff();
    if (VEC && at + 4 <= n) {
      *reinterpret_cast<float4 *>(out + at) = make_float4(x[k][0], x[k][1], x[k][2], x[k][3]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (at + j < n) out[at + j] = x[k][j];
    }
  }
}

template <int K>
int launch(const char *fn, const QLogitRules &p, bool vec, hipStream_t stream) {
  const bool used = p.tokens || p.mask || p.n_bias;
  const int slice = 4 * K * kThreads;
  void (*f)(QLogitRules) = vec ? used ? k_rules<K, true, true> : k_rules<K, true, false> : used ? k_rules<K, false, true> : k_rules<K, false, false>;
  QS_LAUNCH(fn, f, dim3((p.vocab + slice - 1) / slice, p.rows), dim3(kThreads), 0, stream, p);
  return 0;
}

}  // namespace

extern "C" int qllama_logit_rules(const QLogitRules *p, void *stream) {
  static const char fn[] = "qllama_logit_rules";
  if (!p) return qs::refuse(fn, "null argument");
  if (p->rows < 0 || p->rows > 65535 || p->vocab < 1 || p->vocab > (1 << 20) || p->n_req < 0) return qs::refuse(fn, "rows must be 0 .. 65535, vocab 1 .. 2^20, n_req not negative");
  if (p->rows == 0) return 0;
  if (!p->logits || !p->out || p->stride < p->vocab || p->out_stride < p->vocab) return qs::refuse(fn, "null logits or out, or a row stride below vocab");
  if (p->out == p->logits && p->out_stride != p->stride) return qs::refuse(fn, "out may be logits with the same stride only");
  if (p->tokens && (!p->n_tokens || p->capacity < 0 || p->capacity > (1 << 28) || p->token_stride < p->capacity))
    return qs::refuse(fn, "a history needs n_tokens, a capacity of 0 .. 2^28 and a stride of at least that");
  if (p->mask && (p->words < 1 || p->words > 4 || !p->starts || !p->drafted)) return qs::refuse(fn, "a tree's mask needs 1 .. 4 words, starts and drafted");
  if (p->n_bias < 0 || p->n_bias > 4096 || (p->n_bias && (!p->bias_tokens || !p->bias || p->bias_stride < p->n_bias)))
    return qs::refuse(fn, "n_bias must be 0 .. 4096, with bias_tokens, bias and a stride of at least that");
  if (p->allowed && (!p->allowed_rows || p->n_masks < 0 || p->allowed_stride < (p->vocab + 31) / 32)) return qs::refuse(fn, "masks need allowed_rows and a stride of vocab / 32 words");
  const void *four[] = {p->logits, p->out, p->requests, p->tokens, p->n_tokens, p->n_prompt, p->repetition, p->presence, p->frequency, p->starts,
                        p->drafted, p->bias_tokens, p->bias, p->allowed, p->allowed_rows};
  for (const void *x : four)
    if (qs::misaligned(x, 4)) return qs::refuse(fn, "a buffer is not aligned to its elements");
  if (qs::misaligned(p->mask, 8)) return qs::refuse(fn, "a buffer is not aligned to its elements");
  qs::OnDevice on(p->logits, (hipStream_t)stream);
  if (on.why) return qs::refuse(fn, on.why);
  const bool vec = !qs::misaligned(p->logits, 16) && !qs::misaligned(p->out, 16) && p->stride % 4 == 0 && p->out_stride % 4 == 0;
  // slices of 2048 to 8192 tokens: the largest that leave the chip two blocks a CU.  192 rows of 128256: slices of 4096 53
  // us, 8192 47, 16384 (whose counters take 64 KB of LDS: two blocks a CU, not four) 57
  const long long tokens = (long long)p->rows * p->vocab;
  if (tokens >= 512LL * 8192) return launch<4>(fn, *p, vec, (hipStream_t)stream);
  if (tokens >= 512LL * 4096) return launch<2>(fn, *p, vec, (hipStream_t)stream);
  return launch<1>(fn, *p, vec, (hipStream_t)stream);
}
