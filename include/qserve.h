// qserve.h - C ABI of the serving operators: one step of many requests over a paged
// key-value cache.  They stand beside qllama.h's single-sequence cache (LlamaKV),
// its op-level attention (qllama_gqa_decode_ex) and its sampler (sample_token), and
// have no counterpart in the reference.
//
// A step, in order: qllama_paged_plan gives every request the pages its new tokens
// need and names each new row's slot and position; qllama_paged_append rotates the
// rows' queries and keys and stores keys and values in their slots;
// qllama_paged_attention lets the newest token of every request attend to its pages;
// qllama_sample_rows draws a token from every row of logits.  The model's products between
// them may be qmatmul_device_noalloc's: that one always enqueues on qllama_stream(), with
// which no other stream is ordered, so that such a step runs on that stream as a whole or
// orders its own with it by events.
//
// All pointers are DEVICE memory, of one device in a call, unless stated
// otherwise.  Every call enqueues on the hipStream_t it is given (0 is HIP's default
// stream, qllama_stream() the library's), returns without waiting, allocates nothing,
// keeps nothing between calls and may be captured into a HIP graph.  The buffers'
// device need not be the current one; the stream has to be on it.  Calls return 0, or
// print "Error: ..." and return nonzero before anything is enqueued (but for a launch
// that the runtime itself refuses: a call's first kernel may have run by then, and its
// outputs are not to be used); none aborts.  An error that an earlier HIP call has
// left behind is not looked at, and stays unless the call is refused.  Calls that
// overlap need workspaces of their own.  What lies in device memory (lengths, tables,
// slots, settings) cannot be refused by the host: each call states what it does with
// values out of range, and none of them makes it read or write outside its buffers, as
// long as nothing else writes them while the call runs.  Float sums are held in 32
// bits or more and in a fixed order: equal inputs give equal bits.
#ifndef QSERVE_H
#define QSERVE_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

// ---------------------------------------------------------------------------
// The cache
// ---------------------------------------------------------------------------
#define QLLAMA_KV_F32  0   // as LlamaKV holds it
#define QLLAMA_KV_F16  1   // rounded to nearest even
#define QLLAMA_KV_BF16 2   // rounded to nearest even
#define QLLAMA_KV_I8   3   // int8 codes with a float scale per (slot, KV head), of either sign; the append's scale =
                           // max|x| * (1/127) (1 for a row of zeros), code = x * (1/scale) rounded to nearest even, as
                           // quant.c:10-27 up to the last bit of the scale

// A view of memory the caller owns: n_pages pages of page_size slots.  Element d of
// KV head h in slot s of page p is k[p * page_stride + h * head_stride + s *
// slot_stride + d] (strides in elements, alike for k and v).  head_dim is a multiple
// of 8, at most 256; strides are multiples of 8; k and v are 16-byte aligned.
// n_pages * page_size fits in 31 bits; offsets are 64-bit.  A page size that is a
// multiple of 16 lets the attention find a page once for 16 keys.
typedef struct {
  int type;                                       // QLLAMA_KV_*
  int n_pages, page_size, n_kv, head_dim;
  int64_t page_stride, head_stride, slot_stride;  // slot_stride >= head_dim
  void *k, *v;
  int64_t scale_page_stride, scale_head_stride, scale_slot_stride;  // QLLAMA_KV_I8: strides of the scales
  float *k_scale, *v_scale;                       // QLLAMA_KV_I8 only, else NULL
} QPagedKV;

// ---------------------------------------------------------------------------
// Pages and slots of a step
// ---------------------------------------------------------------------------
// Request r holds cached[r] tokens in its first ceil(cached[r] / page_size) table
// entries; added[r] tokens are to be added, or added[r] < 0: the request has ended.
// Free pages wait in a ring: state[0] is the position of the first, state[1] their
// number.
//   * An admitted request's new pages are taken from the ring's front, request by
//     request, and written behind its table entries; lens[r] = cached + added.
//   * The pages of ended requests are put at the ring's back, request by request, for
//     later calls (this one does not take them); lens[r] = 0; the table row is left.
//     What does not fit in the ring any more is dropped.
//   * Requests are admitted in order: r is refused when the pages that r and all requests
//     before it ask for, refused ones among them, exceed the free ones (status 3), or
//     their rows exceed max_rows (status 4); a request that needs no page is not held up
//     by missing pages.  cached + added > width * page_size: status 1.
//     Refused requests keep lens[r] = cached and add nothing.  cached < 0 or above
//     width * page_size: status 2, lens[r] = 0, nothing else.
//   * Admitted rows lie one behind another: starts[r] is the first of request r,
//     starts[n_req] their number.  Row i of them gets its slot (page * page_size +
//     place, -1 if the table entry is negative or the slot exceeds 31 bits), position
//     and request; rows behind the last get slot -1, position 0, request -1.
//   * state_out is the ring's new state.  state outside the ring counts as position 0
//     and as many pages as the ring has places, respectively.
// table and ring change in place; no other output may be one of the inputs.  A page that
// two requests hold (a shared beginning) is returned by each of them: such pages are the
// caller's to count, and to leave out of the rows of ended requests.
typedef struct {
  int n_req;              // 0 .. 8192
  int width;              // table entries of a request
  int page_size, ring_size;                  // ring_size and max_rows: up to 2^30
  int max_rows;           // room for rows in slots, positions and requests
  int64_t table_stride;   // entries between two rows of table, >= width
  const int32_t *cached, *added, *state;     // n_req, n_req, 2
  int32_t *table, *ring;                     // n_req x width, ring_size
  int32_t *lens, *status, *starts;           // n_req, n_req, n_req + 1
  int32_t *state_out;                        // 2
  int32_t *slots, *positions, *requests;     // max_rows
} QPagedPlan;
int qllama_paged_plan(const QPagedPlan *p, void *stream);

// ---------------------------------------------------------------------------
// New rows into their slots
// ---------------------------------------------------------------------------
// For every row i: q_out = R q, K[slot] = R k, V[slot] = v, rounded to the cache's
// type, where R turns the pairs (d, d + head_dim / 2) by the angle of position
// positions[i] (rope.c:48-68: x1 c - x2 s and x2 c + x1 s, each operation rounded),
// with cosines and sines from tables of n_pos rows of head_dim / 2.  cos_t NULL: no
// rotation.  q NULL: keys and values only.  q_out may be q.  Rows hold their heads one
// behind another; strides are in floats.  Row i without a slot (slots[i] < 0, padding)
// stores no key and value.  Rows whose position lies outside the tables write nothing
// at all, rows whose slot lies outside the cache no key and value; *bad (if not NULL)
// is increased by their number.  Slots of one call must differ.  A NaN becomes code 0
// in an int8 row, and does not count for its scale.
typedef struct {
  int rows, n_heads;                          // rows up to 2^23; n_heads: query heads (with q)
  const float *q, *k, *v;
  float *q_out;
  int64_t q_stride, k_stride, v_stride, q_out_stride;
  const int32_t *slots, *positions;
  const float *cos_t, *sin_t;
  int n_pos;
  int32_t *bad;
} QPagedRows;
int qllama_paged_append(const QPagedKV *c, const QPagedRows *r, void *stream);

// ---------------------------------------------------------------------------
// Attention of one new token per request
// ---------------------------------------------------------------------------
// For every request r and query head h (of KV head h / (n_heads / n_kv)), over the
// cached tokens j < lens[r]: o = sum_j w_j v_j, w = softmax_j(scale * q . k_j), and lse
// = ln sum_j e^(scale * q . k_j) (lse may be NULL).  Token j lies in slot j mod
// page_size of page table[r][j / page_size].  scale 0 stands for 1 / sqrt(head_dim);
// up to 2.35e38.  lens[r] <= 0 gives o = 0 and lse = -inf; lengths above width *
// page_size count as that; tokens of a page outside the cache are left out.  What lies
// in slots behind a request's tokens, NaN included, has no effect.  Products and sums
// in 32 bits: a 16-bit or int8 row enters a product as it is, a query or a weight
// (int8: times its value's scale) as two or three 16-bit parts that together hold 23
// (f16 and int8 caches, where a weight is held to 2^-37 of the largest at least) or 24
// bits.  A cached infinity gives NaN.
// width * page_size has to be below 2^31 - 64.  work: qllama_paged_attention_work bytes,
// 16-byte aligned.
typedef struct {
  int n_req, n_heads, width;
  int64_t q_stride, o_stride, lse_stride;     // floats between requests; heads lie one behind another
  int64_t table_stride;
  const float *q;
  float *o, *lse;
  const int32_t *table, *lens;
  float scale;
  void *work;
  size_t work_bytes;
} QPagedQuery;
int qllama_paged_attention(const QPagedKV *c, const QPagedQuery *a, void *stream);
// Bytes of work that a call over this cache needs (host arithmetic; 0 if it would be refused).
size_t qllama_paged_attention_work(const QPagedKV *c, int n_req, int n_heads);
// Where the attention looks for token `key` of a request of len tokens (all host
// memory): its page, -1 if there is none, and its place there.  For tests.
int qllama_test_page_of(const int32_t *table, int width, int page_size, int n_pages, int len, long long key, int *place);

// ---------------------------------------------------------------------------
// A token from every row of logits
// ---------------------------------------------------------------------------
// sample_token (sampler.c:54-143) for many rows, settings and given random numbers,
// with min-p: tokens ordered by (logit descending, index ascending), e_i = exp((l_i -
// l_0) / temperature), and the first n tokens are kept, where n is the smallest of
//   top_k (0 < top_k < vocab, else no limit),
//   the first n whose e add up to at least top_p of all (0 < top_p < 1, else no limit),
//   the number of tokens with e_i >= min_p (min_p > 2^-43, else no limit; above 1 as 1);
// the token is the first j whose e_0 + .. + e_j reach u times the kept sum.
// temperature <= 0 or NaN: the first index of the largest logit.  u outside [0, 1)
// counts as the nearest inside, NaN as 0; a NaN setting is no limit.  Logits of -inf
// and NaN are masked: never kept; a row with nothing else gives token -1, kept 0 and
// prob 0.  Logits of +inf share the row between them.
// Sums and comparisons in 64 bits (each e to 2^-37 + 2^-52 |l_0| / temperature of the
// largest), so a token differs from sample_token's only where that one's float rounding
// decides.
// prob: the token's probability among the kept ones; kept: n.  Both may be NULL.  The
// settings' arrays may be NULL: temperature 1, no limit.  work: qllama_sample_rows_work
// bytes, 16-byte aligned.
typedef struct {
  int rows, vocab;                            // rows up to 65535, vocab 1 .. 1048576
  int64_t stride;                             // floats between rows of logits, >= vocab
  const float *logits, *u;
  const float *temperature;
  const int32_t *top_k;
  const float *top_p, *min_p;
  int32_t *token, *kept;
  float *prob;
  void *work;
  size_t work_bytes;
} QSampleRows;
int qllama_sample_rows(const QSampleRows *s, void *stream);
size_t qllama_sample_rows_work(int rows, int vocab);
// The weight e of a token among its row's sums, in units of which the largest logit has 2^43
// to 1.045 times that (host arithmetic, as the kernels').  For tests.
unsigned long long qllama_test_sample_weight(float logit, float top, float temperature);

#ifdef __cplusplus
}
#endif

#endif
