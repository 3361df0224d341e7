// k_tattn.hip - entry points of the attention of several new tokens a request over a paged
// key-value cache (qllama_tree_attention; semantics in qserve.h, kernels in qdev_tattn.h).
#include <climits>

#include "qdev_tattn.h"
#include "qserve_host.h"

namespace {

// The tile that a call is laid out for: the smallest that holds `nodes` rows of a KV head's
// query heads, 0 to 4: 16, 32, 64, 128 or 256 columns (64 or 128 with heads of more than 128,
// whose outputs take the registers of a second group of columns).
int pick(const QPagedKV *c, int rows, int n_req, int n_heads, int nodes) {
  if (nodes == 0) nodes = n_req ? (rows + n_req - 1) / n_req : 1;
  const int64_t cols = (int64_t)nodes * (n_heads / c->n_kv);
  if (c->head_dim > 128) return cols <= 64 ? 2 : 3;
  // f32 rows of 65 to 128 dims have room for 16-bit parts (LDS) in tiles of 128 columns only, which pay from 33 on, half empty:
  // against f32 products in 64 columns, 8 requests with 45 rows of 4 heads 118 -> 99 us, 64 ragged ones with 16 269 -> 256, 8
  // with 12 60 -> 56, 2 of up to 20000 tokens with 16 125 -> 113; 32 ragged ones with 10 or 16 the same (149, 140)
  if (c->type == QLLAMA_KV_F32 && c->head_dim > 64 && cols > 32) return 3;
  if (cols <= 64) return cols <= 16 ? 0 : cols <= 32 ? 1 : 2;
  // 128 columns a tile unless 64 leave fewer of them empty, by a sixth of all
  const int64_t wide = (cols + 127) / 128 * 128, narrow = (cols + 63) / 64 * 64;
  return 7 * narrow < 6 * wide ? 2 : 3;
}

}  // namespace

extern "C" size_t qllama_tree_attention_work(const QPagedKV *c, int rows, int n_req, int n_heads, int nodes) {
  if (qs::bad_cache(c) || rows < 0 || n_req < 0 || n_heads < 1 || n_heads > 65535 || n_heads % c->n_kv || nodes < 0) return 0;
  const int hdp = c->head_dim <= 64 ? 64 : c->head_dim <= 128 ? 128 : 256, cols = 16 << pick(c, rows, n_req, n_heads, nodes);
  return qtree::kShares * sizeof(int4) + (size_t)(qtree::kShares * 16 / cols) * 2 * cols * (hdp + 2) * sizeof(float);
}

extern "C" int qllama_tree_attention(const QPagedKV *c, const QTreeQuery *a, void *stream) {
  static const char fn[] = "qllama_tree_attention";
  if (const char *why = qs::bad_cache(c)) return qs::refuse(fn, why);
  if (!a || a->n_req < 0 || a->rows < 0 || a->rows > (1 << 23) || a->nodes < 0) return qs::refuse(fn, "null argument, n_req or nodes < 0, or rows not 0 .. 2^23");
  if (a->n_heads < 1 || a->n_heads > 65535 || a->n_heads % c->n_kv) return qs::refuse(fn, "n_heads must be a multiple of the cache's KV heads");
  if (a->n_req == 0 || a->rows == 0) return 0;
  if (!a->q || !a->o || !a->table || !a->lens || !a->starts) return qs::refuse(fn, "null q, o, table, lens or starts");
  if (a->mask ? a->words < 1 || a->words > 4 : a->words != 0) return qs::refuse(fn, "a mask has 1 .. 4 words a row, no mask has 0");
  const int64_t qd = (int64_t)a->n_heads * c->head_dim;
  if (a->q_stride < qd || a->o_stride < qd || (a->lse && a->lse_stride < a->n_heads)) return qs::refuse(fn, "a row stride below the row's length");
  if (a->width < 1 || a->table_stride < a->width || (int64_t)a->width * c->page_size > INT_MAX - 1024)   // a step past it still fits
    return qs::refuse(fn, "bad table width (width * page_size must be below 2^31 - 1024) or stride");
  if ((int64_t)a->rows * a->n_heads > INT_MAX - 1024) return qs::refuse(fn, "rows * n_heads must be below 2^31 - 1024");
  if (a->n_req > INT_MAX - 4096) return qs::refuse(fn, "n_req is too large (2^31 - 4096 and more)");      // a step of the loops over requests past it still fits
  if (((double)a->rows * a->n_heads + c->n_kv) * a->n_req * ((double)a->width * c->page_size + 512) > 4e18) return qs::refuse(fn, "n_req * rows * width * page_size is too large");
  if (!(a->scale >= 0.0f) || a->scale > 2.35e38f)      // times log2 e within a float's range
    return qs::refuse(fn, "scale must be 0 .. 2.35e38");
  if (a->q == a->o) return qs::refuse(fn, "o must not be q");
  if (qs::misaligned(a->q, 4) || qs::misaligned(a->o, 4) || qs::misaligned(a->lse, 4) || qs::misaligned(a->table, 4) || qs::misaligned(a->lens, 4) ||
      qs::misaligned(a->starts, 4) || qs::misaligned(a->mask, 8))
    return qs::refuse(fn, "a buffer is not aligned to its elements");
  if (!a->work || qs::misaligned(a->work, 16) || a->work_bytes < qllama_tree_attention_work(c, a->rows, a->n_req, a->n_heads, a->nodes))
    return qs::refuse(fn, "work is missing, misaligned or smaller than qllama_tree_attention_work");
  qs::OnDevice on(c->k, (hipStream_t)stream);
  if (on.why) return qs::refuse(fn, on.why);
  const int es = c->type == QLLAMA_KV_F32 ? 4 : c->type == QLLAMA_KV_I8 ? 1 : 2;
  qtree::TaArgs p;
  p.k = static_cast<const char *>(c->k); p.v = static_cast<const char *>(c->v);
  p.ks = c->k_scale; p.vs = c->v_scale;
  p.q = a->q; p.o = a->o; p.lse = a->lse; p.mask = a->mask; p.starts = a->starts; p.table = a->table; p.lens = a->lens;
  p.split = static_cast<int4 *>(a->work);
  p.part = reinterpret_cast<float *>(p.split + qtree::kShares);
  p.pst = c->page_stride * es; p.hst = c->head_stride * es; p.sst = c->slot_stride * es;
  p.scp = c->scale_page_stride; p.sch = c->scale_head_stride; p.scs = c->scale_slot_stride;
  p.q_stride = a->q_stride; p.o_stride = a->o_stride; p.lse_stride = a->lse_stride; p.table_stride = a->table_stride;
  p.rows = a->rows; p.n_req = a->n_req; p.n_kv = c->n_kv; p.G = a->n_heads / c->n_kv; p.hd = c->head_dim;
  p.n_pages = c->n_pages; p.page_size = c->page_size; p.width = a->width; p.words = a->words;
  p.wide = ((c->head_dim * es) | p.pst | p.hst | p.sst) % 16 == 0;
  p.qscale = (a->scale > 0.0f ? a->scale : 1.0f / __builtin_sqrtf((float)c->head_dim)) * 1.44269504089f;
  const int tile = pick(c, a->rows, a->n_req, a->n_heads, a->nodes);
  switch (c->type) {
    case QLLAMA_KV_F32: return qtree::launch_f32(fn, p, tile, (hipStream_t)stream);
    case QLLAMA_KV_F16: return qtree::launch_f16(fn, p, tile, (hipStream_t)stream);
    case QLLAMA_KV_BF16: return qtree::launch_bf16(fn, p, tile, (hipStream_t)stream);
    default: return qtree::launch_i8(fn, p, tile, (hipStream_t)stream);
  }
}
