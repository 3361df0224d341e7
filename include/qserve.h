// qserve.h - C ABI of the serving operators: one step of many requests over a paged
// key-value cache.  They stand beside qllama.h's single-sequence cache (LlamaKV),
// its op-level attention (qllama_gqa_decode_ex) and its sampler (sample_token), and
// have no counterpart in the reference.
//
// A step, in order: qllama_paged_plan gives every request the pages its new tokens
// need and names each new row's slot and position; qllama_paged_append rotates the
// rows' queries and keys and stores keys and values in their slots;
// qllama_paged_attention lets the newest token of every request attend to its pages;
// qllama_sample_rows draws a token from every row of logits.  A step that verifies drafted
// tokens adds qllama_tree_plan, qllama_tree_attention in place of the attention above, and
// qllama_tree_accept (below); qllama_logit_rules applies penalties, biases and masks before
// tokens are drawn, and qllama_paged_fork and qllama_paged_move continue requests over pages
// that they share.  The model's products between
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

// ---------------------------------------------------------------------------
// Several new tokens a request: drafted trees
// ---------------------------------------------------------------------------
// A step that verifies drafted tokens gives every request a forest of new rows.  Row j of
// request r is row i = starts[r] + j of the step, and token lens[r] - m + j of the
// request's pages, where m = starts[r + 1] - starts[r] is the number of its new rows and
// lens[r] its tokens with them (starts, lens, slots as qllama_paged_plan leaves them).
// In order: qllama_paged_plan, qllama_tree_plan, qllama_paged_append,
// qllama_tree_attention, (qllama_logit_rules,) qllama_sample_rows for every row,
// qllama_tree_accept, qllama_paged_move in every layer's cache, and qllama_paged_fork with
// keep = the accepted lengths, which gives the pages of rejected rows back.
//
// parents[r][j] is the row (0 .. j - 1, of the same request) that row j follows; any other
// value means none: the row follows the request's earlier tokens.  Rows behind the first
// `nodes` of a request have none.  starts outside 0 .. max_rows count as the nearest
// inside; rows that no request has are left as they were.

// positions[i] = lens[r] - m + depth of the row (0 for a row that follows none); bit b of
// mask[i] (bit b mod 64 of its word b / 64) is set for b = j and every row above j.  Rows
// behind the first 64 * words of a request get mask 0 and the position lens[r] - m + j.
// Such rows attend to nothing new, not even to themselves, so that trees need words >=
// ceil(nodes / 64), and have 256 rows at most.
typedef struct {
  int n_req;                // 0 .. 8192
  int nodes;                // rows of a request that parents has room for: 1 .. 1024
  int max_rows;             // rows of positions and mask
  int words;                // 64-bit words of a row of mask: 1 .. 4
  int64_t parent_stride;    // entries between two requests' parents, >= nodes
  const int32_t *starts, *lens, *parents;    // n_req + 1, n_req, n_req x nodes
  int32_t *positions;                        // max_rows
  uint64_t *mask;                            // max_rows x words
} QTreePlan;
int qllama_tree_plan(const QTreePlan *p, void *stream);

// What the chosen tokens confirm.  Row 0 of a request is accepted (its token was certain);
// then, as long as there is one, the first row c whose parent is the row accepted last and
// whose token tokens[c] is the one that was chosen behind that row (chosen[] >= 0).
// accepted[r] rows in all, lens_out[r] = lens[r] - m + accepted[r], last[r] = what was
// chosen behind the last of them (-1 if the request has no rows).  path[starts[r] + k] is
// the k-th accepted row of the step, -1 behind them; where it is not row k of its request,
// src and dst are the slots that its keys and values have to be moved between (dst: that
// of row k), else -1: groups of qllama_paged_move, with starts as they are.  Rows that no
// request has are left as they were.  Rows behind the first `nodes` follow none and are not
// accepted: where the rows attended with a mask, nodes has to be 64 * words at most (the
// stride as it is), as the rows behind those have attended to nothing new.  Every request of
// a call is verified: rows that are certain (a piece of a prompt) go without this call, in a
// step of their own, or have their next row's token in chosen.
typedef struct {
  int n_req, nodes, max_rows;                // as QTreePlan's
  int64_t parent_stride;
  const int32_t *starts, *lens, *parents;    // n_req + 1, n_req, n_req x nodes
  const int32_t *tokens, *chosen, *slots;    // max_rows
  int32_t *accepted, *last, *lens_out;       // n_req
  int32_t *path, *src, *dst;                 // max_rows
} QTreeAccept;
int qllama_tree_accept(const QTreeAccept *p, void *stream);

// qllama_paged_attention for all new rows: row i = starts[r] + j attends to the tokens t <
// lens[r] - m of its request and to those new rows b < m whose bit is set in mask[i]; mask
// NULL: to b = 0 .. j (the next piece of a prompt).  Bits behind a row's words count as 0.
// A row that attends to nothing gives o = 0 and lse = -inf.  A masked token has no effect,
// whatever its slot holds; an infinity or NaN among the values that a row attends to leaves
// that dim of its output infinite or NaN.  A score of -inf, of an infinite f32 key, is a
// weight of 0, one of +inf or NaN makes the row's outputs NaN; an infinite key in 16 bits
// may make them NaN either way.  Lengths, pages, scale, padding and precision are those of
// qllama_paged_attention, except that int8 rows also meet queries and weights held to 24
// bits, and that f32 rows of up to 128 dims, where `nodes` times the query heads of a KV
// head is above 32, enter the products, as queries and weights do, as three 16-bit parts
// that together are exact: what is left out of a product is below 1.001 x 2^-24 of it, as
// much as rounding it to 32 bits leaves out.  width * page_size and rows * n_heads have to
// be below 2^31 - 1024, n_req below 2^31 - 4096.  `nodes` is the number of rows of a request
// that the call is laid out for (0: rows / n_req), the same that qllama_tree_attention_work
// is asked for; any number of rows is right, other ones are slower.  Rows that no request
// has are left as they were.  starts outside 0 .. rows count as the nearest inside; a row
// that two requests name gets either result.  work: qllama_tree_attention_work bytes,
// 16-byte aligned.
typedef struct {
  int rows;                 // of q, o, lse and mask
  int n_req, n_heads, width, words, nodes;
  int64_t q_stride, o_stride, lse_stride;     // floats between rows; heads lie one behind another
  int64_t table_stride;
  const float *q;
  float *o, *lse;
  const uint64_t *mask;     // rows x words; NULL: words 0
  const int32_t *starts, *table, *lens;
  float scale;
  void *work;
  size_t work_bytes;
} QTreeQuery;
int qllama_tree_attention(const QPagedKV *c, const QTreeQuery *a, void *stream);
size_t qllama_tree_attention_work(const QPagedKV *c, int rows, int n_req, int n_heads, int nodes);

// ---------------------------------------------------------------------------
// Pages that several requests hold
// ---------------------------------------------------------------------------
// New request i continues old request from[i] (0 .. n_old - 1; any other value: it is
// empty) with its first min(keep[i], lens[from[i]]) tokens (keep NULL: all; below 0: none).
// Old requests that nothing continues end.  extra[p] counts who holds page p beyond one: 0
// for pages as qllama_paged_plan gives them and for free ones; holders that are no row of
// the call (a kept beginning of prompts) count too and keep what they have.
//   * Pages are held by every new request that continues over them.  A page that new
//     request i would write to next (its last one, unless full) and that others hold as
//     well is copied: i gets a free page for it, and src[i], dst[i] (slots) and count[i] (tokens)
//     say what to copy (-1, -1, 0: nothing), for qllama_paged_move without starts.  Of the
//     new requests that hold such a page, the one with the most of its tokens (the first
//     of these) keeps it without a copy, if no one outside the call holds it.
//   * Free pages are taken from the ring's front, request by request.  A request that needs a
//     copy is refused (status 3, lens_out 0, nothing held) when the copies that it and all
//     requests before it ask for, refused ones among them, exceed the free pages at the
//     start; one that needs none is never refused.  A page number of the ring outside 0 ..
//     n_pages - 1 is no page: the request that it falls to has -1 there, and nothing to copy.
//   * Pages that no one holds any more are put at the ring's back, in the order of the old
//     rows (a page that several held: where the first of them has it), for later calls.
//     What does not fit in the ring any more is dropped.
//   * lens_out[i] is the number of tokens, the first ceil(lens_out / page_size) entries of
//     table_out[i] the pages; entries behind them are left.  extra_out and state_out follow.
//     state outside the ring counts as in qllama_paged_plan; lens outside 0 .. width *
//     page_size as the nearest inside; a table entry outside 0 .. n_pages - 1 is no page:
//     it is carried over as -1, and not copied.
//   * What a refused request continued ends with the call, like every old request that
//     nothing continues, though it was only to be cut back into a page that others hold.  The
//     old requests are not lost: of the ring only places behind the count at the start change,
//     so that lens, table, extra (where extra_out is another), state and the ring are valid
//     as before the call, which can be made again from them with other requests, as long as
//     its results have not been used.
// extra_out may be extra; no other output may be one of the inputs.  work:
// qllama_paged_fork_work bytes, 16-byte aligned.
typedef struct {
  int n_old, n_new;         // 0 .. 8192
  int width;                // table entries of a request, old and new
  int page_size, n_pages;   // n_pages * page_size fits in 31 bits
  int ring_size;            // up to 2^30
  int64_t table_stride, table_out_stride;     // >= width
  const int32_t *lens, *table;                // n_old, n_old x width
  const int32_t *from, *keep;                 // n_new
  const int32_t *extra, *state;               // n_pages, 2
  int32_t *ring;                              // ring_size, changes in place
  int32_t *table_out, *lens_out, *status;     // n_new x width, n_new, n_new
  int32_t *extra_out, *state_out;             // n_pages, 2
  int32_t *src, *dst, *count;                 // n_new
  void *work;
  size_t work_bytes;
} QPagedFork;
int qllama_paged_fork(const QPagedFork *p, void *stream);
size_t qllama_paged_fork_work(int n_old, int n_new, int n_pages);

// Keys and values (and scales) of slot src[i] into slot dst[i], in n_caches caches at once
// (one a layer; alike in type, sizes and strides).  Without starts the moves are
// independent: count[i] slots from src[i] into as many from dst[i] (count NULL: 1), and no
// slot that a move writes may be read by any or written by another.  With starts, moves
// starts[g] .. starts[g + 1] - 1 happen one after another, and so a slot may be moved on
// into another's old place; groups are independent, and count has to be NULL.  Moves with
// a negative slot, or no count, do nothing; those that leave the cache do nothing either
// and increase *bad (if not NULL) by their number.  starts outside 0 .. n_moves count as
// the nearest inside.
typedef struct {
  int n_moves;              // 0 .. 2^23
  int n_groups;             // 0 .. 2^23; with starts
  const int32_t *src, *dst, *count;           // n_moves
  const int32_t *starts;                      // n_groups + 1
  int32_t *bad;
} QPagedMoves;
int qllama_paged_move(const QPagedKV *caches, int n_caches, const QPagedMoves *m, void *stream);

// ---------------------------------------------------------------------------
// Rules on logits
// ---------------------------------------------------------------------------
// For every row i of request r = requests[i] (NULL: r = i) and every token t:
//   x = logits[i][t];  if t is known, x = x > 0 ? x / repetition[r] : x * repetition[r];
//   x -= frequency[r] * n + (n > 0 ? presence[r] : 0);  x += the bias of t;
//   out[i][t] = x, or -inf where the row's mask does not allow t
// evaluated in 64 bits and rounded once.  n is how often t was generated, t is known if it
// was generated or stands in the prompt: tokens[r] holds n_tokens[r] tokens, the first
// n_prompt[r] (NULL: 0) of them the prompt.  With mask (a tree's, as QTreePlan's), the
// tokens drafted[starts[r] + b] of the bits b of mask[i] were generated too: list those of
// earlier steps alone in tokens.  bias_tokens[r] names n_bias tokens with a bias each; one
// that it names twice gets the first.  allowed_rows[i] names the row's mask, of n_masks:
// bit t mod 32 of word t / 32 is set for an allowed token; other numbers: no mask.
// Tokens outside 0 .. vocab - 1 are none; lengths outside 0 .. capacity count as the
// nearest inside.  A NaN setting, and a repetition that is not above 0, is none.  A row
// whose request lies outside 0 .. n_req - 1 is not written.  out may be logits (with the
// same stride), else they must not overlap.
typedef struct {
  int rows, vocab, n_req;                     // rows up to 65535, vocab 1 .. 1048576
  int64_t stride, out_stride;                 // floats between rows, >= vocab
  const float *logits;
  float *out;
  const int32_t *requests;                    // rows
  int capacity;                               // entries of a row of tokens: 0 .. 2^28
  int64_t token_stride;
  const int32_t *tokens, *n_tokens, *n_prompt;            // NULL: no history
  const float *repetition, *presence, *frequency;         // n_req; NULL: none
  int words;                                  // of a row of mask, 1 .. 4
  const int32_t *starts, *drafted;            // n_req + 1, rows
  const uint64_t *mask;                       // rows x words; NULL: none, and no starts, drafted
  int n_bias;                                 // 0 .. 4096
  int64_t bias_stride;
  const int32_t *bias_tokens;                 // n_req x n_bias
  const float *bias;
  int n_masks;
  int64_t allowed_stride;                     // words between masks, >= ceil(vocab / 32)
  const uint32_t *allowed;                    // NULL: none
  const int32_t *allowed_rows;                // rows
} QLogitRules;
int qllama_logit_rules(const QLogitRules *p, void *stream);

#ifdef __cplusplus
}
#endif

#endif
