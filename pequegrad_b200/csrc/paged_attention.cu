// Attention of new tokens over the paged cache: the entry point.
//   o_r = sum_j softmax_j(scale * q_r . k_j) v_j    over the keys j <= position of row r; zero where there are none
#include <cmath>
#include <string>

#include "paged.cuh"

namespace pgb {

static int fail(int status, const std::string &msg) {
  set_error("paged_attention: " + msg);
  return status;
}

static int paged_attention(const pgb_tensor *q, const pgb_tensor *k_cache, const pgb_tensor *v_cache, const pgb_tensor *k_scale, const pgb_tensor *v_scale,
                           const pgb_tensor *q_start, const pgb_tensor *ctx_len, const pgb_tensor *page_table, float scale, const pgb_tensor *out,
                           cudaStream_t stream) {
  const char *what = "paged_attention";
  KvCache c;
  KvPlan p;
  int st = kv_parse_cache(what, k_cache, v_cache, k_scale, v_scale, false, c);
  if (st != PGB_OK) return st;
  if (!ctx_len) return fail(PGB_ERR_INVALID_ARG, "null plan");
  if ((st = kv_parse_plan(what, q_start, ctx_len, page_table, p)) != PGB_OK) return st;
  if (!q || !out) return fail(PGB_ERR_INVALID_ARG, "null tensor");
  if (q->dtype != PGB_F16 && q->dtype != PGB_BF16) {
    set_error(std::string("paged_attention not implemented for ") + dtype_name(q->dtype));
    return PGB_ERR_UNSUPPORTED;
  }
  if (out->dtype != q->dtype || (c.dtype != PGB_I8 && c.dtype != q->dtype))
    return fail(PGB_ERR_INVALID_ARG, "q, out and a 16-bit cache must share one dtype");
  if (q->ndim != 3 || q->shape[1] < 1 || q->shape[1] % c.heads) return fail(PGB_ERR_INVALID_ARG, "q must be [rows, heads, head dim], its heads a multiple of the cache's");
  if (!(scale > 0.f) || !std::isfinite(scale)) return fail(PGB_ERR_INVALID_ARG, "the scale must be positive and finite");
  PagedParams a{};
  const int64_t H = q->shape[1];
  if (H > 65535) return fail(PGB_ERR_UNSUPPORTED, "too many heads");
  if ((st = kv_parse_rows(what, "q", q, H, c.head_dim, false, &a.q_row, &a.q_head)) != PGB_OK) return st;
  if ((st = kv_parse_rows(what, "out", out, H, c.head_dim, true, &a.o_row, &a.o_head)) != PGB_OK) return st;
  if (out->shape[0] != q->shape[0]) return fail(PGB_ERR_INVALID_ARG, "q and out differ in rows");
  if (!kv_device_present()) return PGB_ERR_CUDA;
  // A row's queries are read before its result is written, and by nobody else: out may be q.
  const bool in_place = view_of(*out, 2) == view_of(*q, 2);
  if ((st = kv_apart(what, {{"out", out}},
                     {{"q", in_place ? nullptr : q}, {"k_cache", k_cache}, {"v_cache", v_cache}, {"k_scale", k_scale}, {"v_scale", v_scale},
                      {"q_start", q_start}, {"ctx_len", ctx_len}, {"page_table", page_table}})) != PGB_OK)
    return st;
  a.q = static_cast<const uint8_t *>(q->data);
  a.out = static_cast<uint8_t *>(out->data);
  a.rows = q->shape[0];
  a.heads = (int)H;
  a.group = (int)(H / c.heads);
  a.c = scale * 1.4426950408889634f;
  if (a.rows == 0 || p.n_seq == 0) return PGB_OK;
  if (c.n_pages == 0) p.width = 0;  // no page at all: no key for anyone, and nothing to point a load at
  // Rows of a sequence on average, times the query heads that share a key: what rides on one pass over the keys. Both kernels
  // are right for any number; the one of 16-row tiles reads the keys again for every further 16, the one of 256-row tiles takes
  // as long for any number up to 256. In us, 16-row tiles and 256-row tiles, 20 and 32 such rows (alone they have 4 to 64 sequences):
  //   16 bits, head dim 128:  4 x 300 tokens 26, 29 and 16, 16;  16 x 1000 100, 78 and 52, 52;  8 x 4000 (grouped) 95, 81 and 62, 65
  //   16 bits, head dim 64:   4 x 300 12, 14 and 13, 13;  64 x 500 59, 61 and 63, 64;  4 x 4000 31, 52 and 45, 46
  // Beside an int8 cache the large tiles' step is longer and the small tiles' bytes fewer; 20, 32 and 48 rows:
  //   head dim 64:   4 x 300 12, 12, 14 and 18;  64 x 500 49, 52, 74 and 107;  4 x 4000 25, 41, 41 and 70
  //   head dim 128:  16 x 1000 75, 64, 81 and 85;  8 x 4000 (grouped) 74, 73, 84 and 102;  but 4 x 1000 38, 40, 44 and 29
  const int64_t few = c.dtype == PGB_I8 ? 48 : 16;
  if (a.rows * a.group > few * p.n_seq && run_paged_chunk(a, c, p, q->dtype == PGB_F16, stream, &st)) return st;
  return run_paged_rows(a, c, p, q->dtype == PGB_F16, stream);
}

}  // namespace pgb

using namespace pgb;

extern "C" PGB_API int pgb_paged_attention(const pgb_tensor *q, const pgb_tensor *k_cache, const pgb_tensor *v_cache, const pgb_tensor *k_scale,
                                           const pgb_tensor *v_scale, const pgb_tensor *q_start, const pgb_tensor *ctx_len, const pgb_tensor *page_table,
                                           float scale, const pgb_tensor *out, void *stream) {
  try {
    return paged_attention(q, k_cache, v_cache, k_scale, v_scale, q_start, ctx_len, page_table, scale, out, (cudaStream_t)stream);
  } catch (...) {  // nothing throws across the boundary: what can is the allocation of a message
    return PGB_ERR_CUDA;
  }
}
