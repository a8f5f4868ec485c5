// Attention of new tokens over the paged cache.
//   o_r = sum_j softmax_j(scale * q_r . k_j) v_j    over the keys j <= position of row r; zero where there are none
// A warp per row and query head. A lane takes one key of 32 for the scores, and D / 32 values of the head for the output;
// running maximum and sum in fp32.
#include <cmath>
#include <string>

#include "kv_cache.cuh"
#include "vec.cuh"

namespace pgb {

struct PagedParams {
  const uint8_t *q;
  uint8_t *out;
  int64_t q_row, q_head, o_row, o_head;  // bytes
  int64_t rows;
  int heads, group;
  float c;  // scale * log2(e)
};

template <typename IoT>
__device__ __forceinline__ float cached_value(const KvPages &p, int dtype, int64_t at, int d, float s) {
  if (dtype == PGB_I8) return (float)reinterpret_cast<const int8_t *>(p.base + at)[d] * s;
  return to_compute<float, IoT>(reinterpret_cast<const IoT *>(p.base + at)[d]);
}

template <typename IoT, int D>
__global__ void __launch_bounds__(256) paged_attention_kernel(const __grid_constant__ PagedParams a, const __grid_constant__ KvCache c,
                                                              const __grid_constant__ KvPlan p) {
  const int lane = threadIdx.x & 31;
  const int64_t g = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (g >= a.rows * a.heads) return;
  const int64_t row = g / a.heads;
  const int head = (int)(g - row * a.heads), kvh = head / a.group;
  const int s = kv_sequence(p, row);
  if (s < 0) return;
  const int64_t last = min(kv_position(p, s, row), ((int64_t)p.width << c.log2_page) - 1);
  const IoT *q = reinterpret_cast<const IoT *>(a.q + row * a.q_row + head * a.q_head);
  float m = -INFINITY, l = 0.f, o[D / 32] = {};
  for (int64_t j0 = 0; j0 <= last; j0 += 32) {
    const int64_t j = j0 + lane;
    const int page = j <= last ? kv_page(p, c, s, j) : -1;
    const int slot = (int)(j & ((1 << c.log2_page) - 1));
    float x = -INFINITY;
    if (page >= 0) {
      const int64_t at = page * c.k.page + kvh * c.k.head + slot * c.k.slot;
      const float ks = c.k.scale ? c.k.scale[page * c.k.scale_page + kvh * c.k.scale_head + slot] : 1.f;
      x = 0.f;
      for (int d = 0; d < D; ++d) x = fmaf(to_compute<float, IoT>(q[d]), cached_value<IoT>(c.k, c.dtype, at, d, ks), x);
      x *= a.c;
    }
    float mx = x;
    for (int k = 16; k > 0; k >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, k));
    const float m_new = fmaxf(m, mx);
    const float alpha = m_new == -INFINITY ? 1.f : exp2f(m - m_new);
    const float e = page >= 0 ? exp2f(x - m_new) : 0.f;
    float sum = e;
    for (int k = 16; k > 0; k >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, k);
    l = l * alpha + sum;
    m = m_new;
    for (int i = 0; i < D / 32; ++i) o[i] *= alpha;
    for (int k = 0; k < 32; ++k) {
      const int pg = __shfl_sync(0xffffffffu, page, k), sl = __shfl_sync(0xffffffffu, slot, k);
      const float pe = __shfl_sync(0xffffffffu, e, k);
      if (pg < 0) continue;
      const int64_t at = pg * c.v.page + kvh * c.v.head + sl * c.v.slot;
      const float vs = c.v.scale ? c.v.scale[pg * c.v.scale_page + kvh * c.v.scale_head + sl] : 1.f;
      for (int i = 0; i < D / 32; ++i) o[i] = fmaf(pe, cached_value<IoT>(c.v, c.dtype, at, lane + 32 * i, vs), o[i]);
    }
  }
  IoT *out = reinterpret_cast<IoT *>(a.out + row * a.o_row + head * a.o_head);
  for (int i = 0; i < D / 32; ++i) out[lane + 32 * i] = from_compute<IoT, float>(l > 0.f ? o[i] / l : o[i]);
}

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
  a.q = static_cast<const uint8_t *>(q->data);
  a.out = static_cast<uint8_t *>(out->data);
  a.rows = q->shape[0];
  a.heads = (int)H;
  a.group = (int)(H / c.heads);
  a.c = scale * 1.4426950408889634f;
  if (a.rows == 0 || p.n_seq == 0) return PGB_OK;
  const int64_t grid = (a.rows * H + 7) / 8;
  if (grid > 2147483647LL) return fail(PGB_ERR_UNSUPPORTED, "too many rows");
  if (q->dtype == PGB_F16) {
    if (c.head_dim == 64) paged_attention_kernel<__half, 64><<<(unsigned)grid, 256, 0, stream>>>(a, c, p);
    else paged_attention_kernel<__half, 128><<<(unsigned)grid, 256, 0, stream>>>(a, c, p);
  } else {
    if (c.head_dim == 64) paged_attention_kernel<__nv_bfloat16, 64><<<(unsigned)grid, 256, 0, stream>>>(a, c, p);
    else paged_attention_kernel<__nv_bfloat16, 128><<<(unsigned)grid, 256, 0, stream>>>(a, c, p);
  }
  count_launch();
  return check_launch("paged_attention_kernel");
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
