// The paged key / value cache: storing new rows (16-bit copy, or int8 with a scale per token and head) and reading
// sequences back (gather, dequantise).
//
// Both move every byte once and compute next to nothing, so they are bound by memory; a step of decoding, with one row per
// sequence, is bound by the launch and three dependent loads (row offsets, table, data).
// One row for each of 32 sequences, 12 heads of 64: 11 us a call, all but 2 of them the host's. 2800 rows, 8 heads of 128, into
// int8 and 9600 tokens read back: 31 us for 67 MB.
//   store  s = max(max_d |x_d|, 1e-6) / 127,  c_d = clip(rint(x_d / s), -127, 127): the rule of pgb_quantize_i8, with the
//          maximum over one token's head instead of the whole tensor
//   read   x_d = c_d * s, one product in fp32, rounded once to the output's type
#include <string>

#include "gemm_ptx.cuh"
#include "kv_cache.cuh"

namespace pgb {

bool kv_device_present() {
  int n = 0;
  if (cudaGetDeviceCount(&n) != cudaSuccess || n <= 0) {
    cudaGetLastError();
    set_error("no CUDA device: this library has no CPU fallback");
    return false;
  }
  return true;
}

static int fail(int status, const char *what, const std::string &msg) {
  set_error(std::string(what) + ": " + msg);
  return status;
}

static int parse_pages(const char *what, const char *name, const pgb_tensor &t, const pgb_tensor *scale, bool writes, KvPages &p) {
  const int es = dtype_size(t.dtype);
  if (t.stride_bytes[3] != es) return fail(PGB_ERR_INVALID_ARG, what, std::string("the head dim of ") + name + " must be contiguous");
  if (reinterpret_cast<uintptr_t>(t.data) & 15) return fail(PGB_ERR_UNSUPPORTED, what, std::string(name) + " must be 16-byte aligned");
  for (int d = 0; d < 3; ++d) {
    if (t.stride_bytes[d] < 0 || t.stride_bytes[d] % 16)
      return fail(PGB_ERR_UNSUPPORTED, what, std::string(name) + " must have page, head and slot pitches that are multiples of 16 bytes");
  }
  if (writes && view_overlaps_itself(view_of(t, es))) return fail(PGB_ERR_INVALID_ARG, what, std::string(name) + " overlaps itself");
  p.base = static_cast<uint8_t *>(t.data);
  p.page = t.stride_bytes[0];
  p.head = t.stride_bytes[1];
  p.slot = t.stride_bytes[2];
  p.scale = nullptr;
  p.scale_page = p.scale_head = 0;
  if (!scale) return PGB_OK;
  if (scale->dtype != PGB_F32 || scale->ndim != 3 || scale->shape[0] != t.shape[0] || scale->shape[1] != t.shape[1] || scale->shape[2] != t.shape[2])
    return fail(PGB_ERR_INVALID_ARG, what, "the scales must be float32 [pages, heads, page size] as the cache is");
  if (scale->stride_bytes[2] != 4 || scale->stride_bytes[0] < 0 || scale->stride_bytes[1] < 0 || scale->stride_bytes[0] % 16 ||
      scale->stride_bytes[1] % 16 || (reinterpret_cast<uintptr_t>(scale->data) & 15))
    return fail(PGB_ERR_UNSUPPORTED, what, "the scales of a page must be contiguous and 16-byte aligned");
  if (writes && view_overlaps_itself(view_of(*scale, 4)))
    return fail(PGB_ERR_INVALID_ARG, what, "the scales overlap themselves");
  if (!scale->data && t.shape[0]) return fail(PGB_ERR_INVALID_ARG, what, "null scales");
  p.scale = static_cast<float *>(scale->data);
  p.scale_page = scale->stride_bytes[0] / 4;
  p.scale_head = scale->stride_bytes[1] / 4;
  return PGB_OK;
}

int kv_parse_cache(const char *what, const pgb_tensor *k_cache, const pgb_tensor *v_cache, const pgb_tensor *k_scale,
                   const pgb_tensor *v_scale, bool writes, KvCache &c) {
  if (!k_cache || !v_cache) return fail(PGB_ERR_INVALID_ARG, what, "null cache");
  if (k_cache->ndim != 4 || v_cache->ndim != 4) return fail(PGB_ERR_INVALID_ARG, what, "a cache is [pages, heads, page size, head dim]");
  for (int d = 0; d < 4; ++d)
    if (k_cache->shape[d] != v_cache->shape[d]) return fail(PGB_ERR_INVALID_ARG, what, "the key and value caches differ in shape");
  if (k_cache->dtype != v_cache->dtype) return fail(PGB_ERR_INVALID_ARG, what, "the key and value caches differ in dtype");
  c.dtype = k_cache->dtype;
  if (c.dtype != PGB_F16 && c.dtype != PGB_BF16 && c.dtype != PGB_I8) {
    set_error(std::string(what) + " not implemented for a cache of " + dtype_name(c.dtype));
    return PGB_ERR_UNSUPPORTED;
  }
  const bool i8 = c.dtype == PGB_I8;
  if (i8 != (k_scale != nullptr) || i8 != (v_scale != nullptr))
    return fail(PGB_ERR_INVALID_ARG, what, i8 ? "an int8 cache needs k_scale and v_scale" : "only an int8 cache has scales");
  const int64_t P = k_cache->shape[2], D = k_cache->shape[3];
  if (D != 64 && D != 128) return fail(PGB_ERR_UNSUPPORTED, what, "only head dims of 64 and 128 are implemented");
  if (P != 16 && P != 32 && P != 64 && P != 128) return fail(PGB_ERR_UNSUPPORTED, what, "the page size must be 16, 32, 64 or 128");
  if (k_cache->shape[0] < 0 || k_cache->shape[0] > 2147483647LL || k_cache->shape[1] < 1 || k_cache->shape[1] > 65535)
    return fail(PGB_ERR_UNSUPPORTED, what, "bad number of pages or heads");
  if (k_cache->shape[0] && (!k_cache->data || !v_cache->data)) return fail(PGB_ERR_INVALID_ARG, what, "null cache");
  c.n_pages = (int)k_cache->shape[0];
  c.heads = (int)k_cache->shape[1];
  c.head_dim = (int)D;
  c.log2_page = P == 16 ? 4 : (P == 32 ? 5 : (P == 64 ? 6 : 7));
  int st = parse_pages(what, "k_cache", *k_cache, k_scale, writes, c.k);
  if (st == PGB_OK) st = parse_pages(what, "v_cache", *v_cache, v_scale, writes, c.v);
  return st;
}

int kv_parse_plan(const char *what, const pgb_tensor *start, const pgb_tensor *ctx, const pgb_tensor *table, KvPlan &p) {
  if (!start || !table) return fail(PGB_ERR_INVALID_ARG, what, "null plan");
  if (start->dtype != PGB_I32 || table->dtype != PGB_I32 || (ctx && ctx->dtype != PGB_I32))
    return fail(PGB_ERR_INVALID_ARG, what, "row offsets, lengths and the page table must be int32");
  if (start->ndim != 1 || start->shape[0] < 1 || !is_contiguous(*start)) return fail(PGB_ERR_INVALID_ARG, what, "the row offsets must be a contiguous [sequences + 1]");
  const int64_t B = start->shape[0] - 1;
  if (ctx && (ctx->ndim != 1 || ctx->shape[0] != B || !is_contiguous(*ctx))) return fail(PGB_ERR_INVALID_ARG, what, "the lengths must be a contiguous [sequences]");
  if (table->ndim != 2 || table->shape[0] != B || table->shape[1] < 0) return fail(PGB_ERR_INVALID_ARG, what, "the page table must be [sequences, pages of a sequence]");
  if (table->shape[1] > 1 && table->stride_bytes[1] != 4) return fail(PGB_ERR_INVALID_ARG, what, "the rows of the page table must be contiguous");
  if (table->stride_bytes[0] < 0 || table->stride_bytes[0] % 4) return fail(PGB_ERR_INVALID_ARG, what, "bad stride in the page table");
  // positions are 32-bit numbers: 2^23 pages of at most 128 tokens
  if (B > 1000000 || table->shape[1] > (1 << 23)) return fail(PGB_ERR_UNSUPPORTED, what, "too many sequences or pages");
  if (B && (!start->data || (ctx && !ctx->data) || (table->shape[1] && !table->data))) return fail(PGB_ERR_INVALID_ARG, what, "null plan");
  for (const pgb_tensor *t : {start, ctx, table})
    if (t && (reinterpret_cast<uintptr_t>(t->data) & 3)) return fail(PGB_ERR_INVALID_ARG, what, "row offsets, lengths and the page table must be 4-byte aligned");
  p.start = static_cast<const int *>(start->data);
  p.ctx = ctx ? static_cast<const int *>(ctx->data) : nullptr;
  p.table = static_cast<const int *>(table->data);
  p.pitch = table->stride_bytes[0] / 4;
  p.n_seq = (int)B;
  p.width = (int)table->shape[1];
  return PGB_OK;
}

int kv_parse_rows(const char *what, const char *name, const pgb_tensor *t, int64_t heads, int head_dim, bool writes, int64_t *row,
                  int64_t *head) {
  if (!t) return fail(PGB_ERR_INVALID_ARG, what, std::string("null ") + name);
  const int es = dtype_size(t->dtype);
  if (t->ndim != 3 || t->shape[1] != heads || t->shape[2] != head_dim)
    return fail(PGB_ERR_INVALID_ARG, what, std::string(name) + " must be [rows, heads, head dim], with the heads and head dim of the cache");
  if (t->stride_bytes[2] != es) return fail(PGB_ERR_INVALID_ARG, what, std::string("the head dim of ") + name + " must be contiguous");
  if ((reinterpret_cast<uintptr_t>(t->data) & 15) || t->stride_bytes[0] < 0 || t->stride_bytes[1] < 0 ||
      (t->shape[0] > 1 && t->stride_bytes[0] % 16) || (heads > 1 && t->stride_bytes[1] % 16))
    return fail(PGB_ERR_UNSUPPORTED, what, std::string(name) + " must be 16-byte aligned with row and head pitches that are multiples of 16 bytes");
  if (writes && view_overlaps_itself(view_of(*t, es)))
    return fail(PGB_ERR_INVALID_ARG, what, std::string(name) + " overlaps itself");
  if (t->shape[0] < 0) return fail(PGB_ERR_INVALID_ARG, what, std::string(name) + " has a negative number of rows");
  if (t->shape[0] > 2147483647LL) return fail(PGB_ERR_UNSUPPORTED, what, "too many rows");
  if (t->shape[0] && !t->data) return fail(PGB_ERR_INVALID_ARG, what, std::string("null ") + name);
  *row = t->shape[0] > 1 ? t->stride_bytes[0] : 0;
  *head = heads > 1 ? t->stride_bytes[1] : 0;
  return PGB_OK;
}

int kv_apart(const char *what, std::initializer_list<KvOperand> written, std::initializer_list<KvOperand> read) {
  ByteView w[4];  // the cache's two tensors and their scales at most
  int n = 0;
  const KvOperand *of[4];
  auto alone = [&](const KvOperand &o, const ByteView &v) -> bool {
    for (int i = 0; i < n; ++i)
      if (views_share(w[i], v)) {
        set_error(std::string(what) + ": " + of[i]->name + " is written and shares memory with " + o.name);
        return false;
      }
    return true;
  };
  for (const KvOperand &o : written) {
    if (!o.t) continue;
    const ByteView v = view_of(*o.t, dtype_size(o.t->dtype));
    if (!alone(o, v)) return PGB_ERR_INVALID_ARG;
    w[n] = v;
    of[n++] = &o;
  }
  for (const KvOperand &o : read)
    if (o.t && !alone(o, view_of(*o.t, dtype_size(o.t->dtype)))) return PGB_ERR_INVALID_ARG;
  return PGB_OK;
}

struct KvRows {
  uint8_t *k, *v;
  int64_t k_row, k_head, v_row, v_head;  // bytes
  int64_t rows;
};

// Which row and head a group of lanes has: 64-bit division takes longer than the rest of the address work, and few calls need it.
__device__ __forceinline__ void row_and_head(int64_t g, int64_t rows, int heads, int64_t &row, int &head) {
  if (rows * heads <= 0xffffffffLL) {
    const uint32_t r = (uint32_t)g / (uint32_t)heads;
    row = r;
    head = (int)((uint32_t)g - r * (uint32_t)heads);
  } else {
    row = g / heads;
    head = (int)(g - row * heads);
  }
}

// For the read: TILE consecutive rows of one head, then the next head, so that a warp reads one stretch of a page. The rows that
// fill no tile come last, head by head.
template <int TILE>
__device__ __forceinline__ void row_and_head_tiled(int64_t g, int64_t rows, int heads, int64_t &row, int &head) {
  const int64_t whole = rows - rows % TILE;
  if (g >= whole * heads) {
    row_and_head(g - whole * heads, rows - whole, heads, row, head);
    row += whole;
    return;
  }
  int64_t block;
  row_and_head(g / TILE, whole / TILE, heads, block, head);
  row = block * TILE + g % TILE;
}

// Eight 16-bit values as fp32, and back.
template <bool HALF>
__device__ __forceinline__ void widen8(const uint4 &r, float (&x)[8]) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float2 f;
    if constexpr (HALF) f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
    else f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&w[i]));
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}
template <bool HALF>
__device__ __forceinline__ uint32_t narrow2(float lo, float hi) {
  uint32_t r;
  if (HALF) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// D / 8 lanes hold one token's head, eight values a lane. A value that is not finite makes the scale NaN, and with it
// everything that is read back of this token and head: an infinity has no int8 form, and must not come back as a number.
template <int D, bool HALF>
__device__ __forceinline__ uint2 quantise8(const uint4 &r, float &scale) {
  float x[8];
  widen8<HALF>(r, x);
  uint32_t m = 0;  // |x| ordered as bits: finite < infinity < NaN
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
#pragma unroll
  for (int k = D / 16; k > 0; k >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, k, D / 8));
  if (m >= 0x7f800000u) {
    scale = __uint_as_float(0x7fc00000u);
    return make_uint2(0u, 0u);
  }
  const float s = fmaxf(__uint_as_float(m), 1e-6f) / 127.0f;
  const float inv = 1.0f / s, thr = 0.49999f * s;
  scale = s;
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    bool recheck = false;
    w[i] = quant_i8_fast4<false>(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3], s, inv, thr, recheck);
    if (recheck) w[i] = quant_i8_pack4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3], s, inv);
  }
  return make_uint2(w[0], w[1]);
}

// A group of D / 8 lanes stores one token's head of K and of V: both loads are under way before the plan is looked up.
template <int D, bool HALF, bool I8>
__global__ void __launch_bounds__(256) kv_write_kernel(const __grid_constant__ KvRows x, const __grid_constant__ KvCache c,
                                                       const __grid_constant__ KvPlan p) {
  constexpr int kLanes = D / 8;
  const int64_t g = ((int64_t)blockIdx.x * 256 + threadIdx.x) / kLanes;
  const int lane = threadIdx.x % kLanes;
  const bool in = g < x.rows * c.heads;  // the lanes of a warp stay together for the shuffles
  int64_t row = 0;
  int head = 0;
  if (in) row_and_head(g, x.rows, c.heads, row, head);
  uint4 k = make_uint4(0, 0, 0, 0), v = k;
  if (in) {
    k = __ldcs(reinterpret_cast<const uint4 *>(x.k + row * x.k_row + head * x.k_head) + lane);
    v = __ldcs(reinterpret_cast<const uint4 *>(x.v + row * x.v_row + head * x.v_head) + lane);
  }
  int page = -1, slot = 0;
  if (in) {
    const int s = kv_sequence(p, row);
    if (s >= 0) {
      const int64_t pos = kv_position(p, s, row);
      page = kv_page(p, c, s, pos);
      slot = (int)(pos & ((1 << c.log2_page) - 1));
    }
  }
  if constexpr (I8) {
    float ks, vs;
    const uint2 kq = quantise8<D, HALF>(k, ks), vq = quantise8<D, HALF>(v, vs);
    if (page < 0) return;
    reinterpret_cast<uint2 *>(c.k.base + page * c.k.page + head * c.k.head + slot * c.k.slot)[lane] = kq;
    reinterpret_cast<uint2 *>(c.v.base + page * c.v.page + head * c.v.head + slot * c.v.slot)[lane] = vq;
    if (lane == 0) {
      c.k.scale[page * c.k.scale_page + head * c.k.scale_head + slot] = ks;
      c.v.scale[page * c.v.scale_page + head * c.v.scale_head + slot] = vs;
    }
  } else {
    if (page < 0) return;
    reinterpret_cast<uint4 *>(c.k.base + page * c.k.page + head * c.k.head + slot * c.k.slot)[lane] = k;
    reinterpret_cast<uint4 *>(c.v.base + page * c.v.page + head * c.v.head + slot * c.v.slot)[lane] = v;
  }
}

// Sixteen int8 values times their scale, in the output's type: 16 bits as two vectors, fp32 as four.
template <int OUT>  // PGB_F16, PGB_BF16 or PGB_F32
__device__ __forceinline__ void store_dequantised(uint8_t *dst, const uint4 &r, float s) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
  float x[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i] = (float)(int8_t)(w[i >> 2] >> (8 * (i & 3))) * s;
  uint4 *d = reinterpret_cast<uint4 *>(dst);
  if constexpr (OUT == PGB_F32) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      __stcs(d + i, make_uint4(__float_as_uint(x[4 * i]), __float_as_uint(x[4 * i + 1]), __float_as_uint(x[4 * i + 2]), __float_as_uint(x[4 * i + 3])));
  } else {
    uint32_t o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = narrow2<OUT == PGB_F16>(x[2 * i], x[2 * i + 1]);
    __stcs(d, make_uint4(o[0], o[1], o[2], o[3]));
    __stcs(d + 1, make_uint4(o[4], o[5], o[6], o[7]));
  }
}

// The mirror image of the store: a lane moves 16 bytes of K and of V (eight 16-bit or sixteen int8 values). 12 sequences of up
// to 8192 int8 tokens, 8 heads of 128, into bf16: 68 to 70 us, 0.75 of the copy rate (73 with a warp across four heads of a token). Two
// and four rows a thread, with all their loads under way at once, were slower (74 and 82 against 73).
template <int D, bool I8, int OUT>
__global__ void __launch_bounds__(256) kv_read_kernel(const __grid_constant__ KvRows y, const __grid_constant__ KvCache c,
                                                      const __grid_constant__ KvPlan p) {
  constexpr int kLanes = I8 ? D / 16 : D / 8;
  constexpr int kOutBytes = I8 ? (OUT == PGB_F32 ? 64 : 32) : 16;  // per lane
  const int64_t g = ((int64_t)blockIdx.x * 256 + threadIdx.x) / kLanes;
  const int lane = threadIdx.x % kLanes;
  if (g >= y.rows * c.heads) return;
  int64_t row;
  int head;
  row_and_head_tiled<32 / kLanes>(g, y.rows, c.heads, row, head);
  const int s = kv_sequence(p, row);
  if (s < 0) return;  // behind the last sequence: left as it was
  const int64_t pos = kv_position(p, s, row);
  const int page = kv_page(p, c, s, pos), slot = (int)(pos & ((1 << c.log2_page) - 1));
  uint4 k = make_uint4(0, 0, 0, 0), v = k;
  float ks = 0.f, vs = 0.f;
  if (page >= 0) {
    k = __ldcs(reinterpret_cast<const uint4 *>(c.k.base + page * c.k.page + head * c.k.head + slot * c.k.slot) + lane);
    v = __ldcs(reinterpret_cast<const uint4 *>(c.v.base + page * c.v.page + head * c.v.head + slot * c.v.slot) + lane);
    if constexpr (I8) {
      ks = __ldg(c.k.scale + page * c.k.scale_page + head * c.k.scale_head + slot);
      vs = __ldg(c.v.scale + page * c.v.scale_page + head * c.v.scale_head + slot);
    }
  }
  uint8_t *ko = y.k + row * y.k_row + head * y.k_head + lane * kOutBytes, *vo = y.v + row * y.v_row + head * y.v_head + lane * kOutBytes;
  if constexpr (I8) {
    store_dequantised<OUT>(ko, k, ks);
    store_dequantised<OUT>(vo, v, vs);
  } else {
    __stcs(reinterpret_cast<uint4 *>(ko), k);
    __stcs(reinterpret_cast<uint4 *>(vo), v);
  }
}

static int kv_write(const pgb_tensor *k, const pgb_tensor *v, const pgb_tensor *k_cache, const pgb_tensor *v_cache, const pgb_tensor *k_scale,
                    const pgb_tensor *v_scale, const pgb_tensor *q_start, const pgb_tensor *ctx_len, const pgb_tensor *page_table, cudaStream_t stream) {
  const char *what = "kv_write";
  KvCache c;
  KvPlan p;
  int st = kv_parse_cache(what, k_cache, v_cache, k_scale, v_scale, true, c);
  if (st != PGB_OK) return st;
  if (!ctx_len) return fail(PGB_ERR_INVALID_ARG, what, "null plan");
  if ((st = kv_parse_plan(what, q_start, ctx_len, page_table, p)) != PGB_OK) return st;
  if (!k || !v || (k->dtype != PGB_F16 && k->dtype != PGB_BF16) || v->dtype != k->dtype)
    return fail(PGB_ERR_INVALID_ARG, what, "k and v must both be float16 or both bfloat16");
  if (c.dtype != PGB_I8 && c.dtype != k->dtype) return fail(PGB_ERR_INVALID_ARG, what, "a 16-bit cache must have the dtype of k and v");
  KvRows x{};
  if ((st = kv_parse_rows(what, "k", k, c.heads, c.head_dim, false, &x.k_row, &x.k_head)) != PGB_OK) return st;
  if ((st = kv_parse_rows(what, "v", v, c.heads, c.head_dim, false, &x.v_row, &x.v_head)) != PGB_OK) return st;
  if (k->shape[0] != v->shape[0]) return fail(PGB_ERR_INVALID_ARG, what, "k and v differ in rows");
  x.k = static_cast<uint8_t *>(k->data);
  x.v = static_cast<uint8_t *>(v->data);
  x.rows = k->shape[0];
  if (!kv_device_present()) return PGB_ERR_CUDA;
  if ((st = kv_apart(what, {{"k_cache", k_cache}, {"v_cache", v_cache}, {"k_scale", k_scale}, {"v_scale", v_scale}},
                     {{"k", k}, {"v", v}, {"q_start", q_start}, {"ctx_len", ctx_len}, {"page_table", page_table}})) != PGB_OK)
    return st;
  if (x.rows == 0 || p.n_seq == 0 || c.n_pages == 0 || p.width == 0) return PGB_OK;
  const int64_t grid = (x.rows * c.heads * (c.head_dim / 8) + 255) / 256;
  if (grid > 2147483647LL) return fail(PGB_ERR_UNSUPPORTED, what, "too many rows");
  const bool half = k->dtype == PGB_F16, i8 = c.dtype == PGB_I8;
#define PGB_KV_WRITE(D, H, Q) kv_write_kernel<D, H, Q><<<(unsigned)grid, 256, 0, stream>>>(x, c, p)
  if (c.head_dim == 64) {
    if (!i8) PGB_KV_WRITE(64, true, false);
    else if (half) PGB_KV_WRITE(64, true, true);
    else PGB_KV_WRITE(64, false, true);
  } else {
    if (!i8) PGB_KV_WRITE(128, true, false);
    else if (half) PGB_KV_WRITE(128, true, true);
    else PGB_KV_WRITE(128, false, true);
  }
#undef PGB_KV_WRITE
  count_launch();
  return check_launch("kv_write_kernel");
}

static int kv_read(const pgb_tensor *k_cache, const pgb_tensor *v_cache, const pgb_tensor *k_scale, const pgb_tensor *v_scale, const pgb_tensor *kv_start,
                   const pgb_tensor *page_table, const pgb_tensor *k, const pgb_tensor *v, cudaStream_t stream) {
  const char *what = "kv_read";
  KvCache c;
  KvPlan p;
  int st = kv_parse_cache(what, k_cache, v_cache, k_scale, v_scale, false, c);
  if (st != PGB_OK) return st;
  if ((st = kv_parse_plan(what, kv_start, nullptr, page_table, p)) != PGB_OK) return st;
  if (!k || !v || k->dtype != v->dtype) return fail(PGB_ERR_INVALID_ARG, what, "k and v must have one dtype");
  const bool i8 = c.dtype == PGB_I8;
  if (i8 ? (k->dtype != PGB_F16 && k->dtype != PGB_BF16 && k->dtype != PGB_F32) : k->dtype != c.dtype)
    return fail(PGB_ERR_INVALID_ARG, what, i8 ? "an int8 cache is read as float16, bfloat16 or float32" : "a 16-bit cache is read in its own dtype");
  KvRows y{};
  if ((st = kv_parse_rows(what, "k", k, c.heads, c.head_dim, true, &y.k_row, &y.k_head)) != PGB_OK) return st;
  if ((st = kv_parse_rows(what, "v", v, c.heads, c.head_dim, true, &y.v_row, &y.v_head)) != PGB_OK) return st;
  if (k->shape[0] != v->shape[0]) return fail(PGB_ERR_INVALID_ARG, what, "k and v differ in rows");
  y.k = static_cast<uint8_t *>(k->data);
  y.v = static_cast<uint8_t *>(v->data);
  y.rows = k->shape[0];
  if (!kv_device_present()) return PGB_ERR_CUDA;
  if ((st = kv_apart(what, {{"k", k}, {"v", v}},
                     {{"k_cache", k_cache}, {"v_cache", v_cache}, {"k_scale", k_scale}, {"v_scale", v_scale}, {"kv_start", kv_start}, {"page_table", page_table}})) != PGB_OK)
    return st;
  if (y.rows == 0 || p.n_seq == 0) return PGB_OK;
  const int lanes = i8 ? c.head_dim / 16 : c.head_dim / 8;
  const int64_t grid = (y.rows * c.heads * lanes + 255) / 256;
  if (grid > 2147483647LL) return fail(PGB_ERR_UNSUPPORTED, what, "too many rows");
#define PGB_KV_READ(D, Q, O) kv_read_kernel<D, Q, O><<<(unsigned)grid, 256, 0, stream>>>(y, c, p)
  if (c.head_dim == 64) {
    if (!i8) PGB_KV_READ(64, false, PGB_F16);  // a copy of 16-bit values, whichever type they have
    else if (k->dtype == PGB_F16) PGB_KV_READ(64, true, PGB_F16);
    else if (k->dtype == PGB_BF16) PGB_KV_READ(64, true, PGB_BF16);
    else PGB_KV_READ(64, true, PGB_F32);
  } else {
    if (!i8) PGB_KV_READ(128, false, PGB_F16);
    else if (k->dtype == PGB_F16) PGB_KV_READ(128, true, PGB_F16);
    else if (k->dtype == PGB_BF16) PGB_KV_READ(128, true, PGB_BF16);
    else PGB_KV_READ(128, true, PGB_F32);
  }
#undef PGB_KV_READ
  count_launch();
  return check_launch("kv_read_kernel");
}

}  // namespace pgb

using namespace pgb;

extern "C" {

PGB_API int pgb_kv_write(const pgb_tensor *k, const pgb_tensor *v, const pgb_tensor *k_cache, const pgb_tensor *v_cache, const pgb_tensor *k_scale,
                         const pgb_tensor *v_scale, const pgb_tensor *q_start, const pgb_tensor *ctx_len, const pgb_tensor *page_table, void *stream) {
  try {
    return kv_write(k, v, k_cache, v_cache, k_scale, v_scale, q_start, ctx_len, page_table, (cudaStream_t)stream);
  } catch (...) {  // nothing throws across the boundary: what can is the allocation of a message
    return PGB_ERR_CUDA;
  }
}

PGB_API int pgb_kv_read(const pgb_tensor *k_cache, const pgb_tensor *v_cache, const pgb_tensor *k_scale, const pgb_tensor *v_scale,
                        const pgb_tensor *kv_start, const pgb_tensor *page_table, const pgb_tensor *k, const pgb_tensor *v, void *stream) {
  try {
    return kv_read(k_cache, v_cache, k_scale, v_scale, kv_start, page_table, k, v, (cudaStream_t)stream);
  } catch (...) {
    return PGB_ERR_CUDA;
  }
}

}  // extern "C"
