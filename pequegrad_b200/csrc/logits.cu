// Logits shaped before a token is picked: penalties for repeated tokens, sparse biases, a grammar's bit mask.
//
//   seen[v]  = v occurs in history[0, len)          count[v] = times v occurs in history[prompt, len)
//   x = logits[v];  if seen: x = x > 0 ? x / repetition : x * repetition
//   x = x - frequency * count[v] - presence * (count[v] > 0) + sum of bias[i] over bias_ids[i] == v
//   out[v] = mask bit v set ? x : -inf
// in fp32, each operation rounded as written, the result rounded once to the output's type.
//
// The work is one read and one write of the logits; the counts never leave the SM: a CTA owns a slice of one row's
// vocabulary, counts the history's tokens that fall into it with integer atomics in shared memory (their order does not
// change the result), and then streams its slice. Every CTA of a row reads the whole history, which the L2 serves.
#include <string>

#include "reduce_common.cuh"
#include "vec.cuh"

namespace pgb {

constexpr int kLogitThreads = 256;
constexpr uint32_t kSeen = 0x80000000u;  // bit 31 of a counter: the token occurs at all; the rest counts the generated ones

struct LogitParams {
  const void *x;
  void *y;
  int64_t x_pitch, y_pitch;  // elements
  int64_t V;
  const int *history, *history_len, *prompt_len;
  int64_t history_pitch;
  int L;
  const float *repetition, *frequency, *presence;
  const int *bias_ids;
  const float *bias;
  int64_t bias_ids_pitch, bias_pitch;
  int n_bias;
  const uint32_t *mask;
  int64_t mask_pitch;  // words
  int slice;           // vocabulary entries per CTA
};

template <typename IoT, int V>
__global__ void __launch_bounds__(kLogitThreads) logits_kernel(const __grid_constant__ LogitParams p) {
  extern __shared__ uint32_t smem[];
  const int64_t row = blockIdx.y;
  const int64_t v0 = (int64_t)blockIdx.x * p.slice;
  const int n = (int)min((int64_t)p.slice, p.V - v0);
  const bool counts = p.history != nullptr, biased = p.n_bias > 0;
  uint32_t *count = smem;
  float *bias = reinterpret_cast<float *>(smem + (counts ? p.slice : 0));
  if (counts)
    for (int i = threadIdx.x; i < n; i += kLogitThreads) count[i] = 0;
  if (biased)
    for (int i = threadIdx.x; i < n; i += kLogitThreads) bias[i] = 0.f;
  __syncthreads();
  if (counts) {
    const int len = p.history_len ? min(max(__ldg(p.history_len + row), 0), p.L) : p.L;
    const int prompt = p.prompt_len ? __ldg(p.prompt_len + row) : 0;
    const int *h = p.history + row * p.history_pitch;
    for (int i = threadIdx.x; i < len; i += kLogitThreads) {
      const int64_t at = (int64_t)__ldg(h + i) - v0;
      if (at < 0 || at >= n) continue;
      if (i >= prompt) {
        if ((atomicAdd(count + at, 1u) & kSeen) == 0) atomicOr(count + at, kSeen);
      } else {
        atomicOr(count + at, kSeen);
      }
    }
  }
  // A token may be biased more than once. One warp takes the list in order, and lanes that hold the same token leave the
  // sum to the first of them, which adds in list order: the result does not depend on timing.
  if (biased && threadIdx.x < 32) {
    const int *ids = p.bias_ids + row * p.bias_ids_pitch;
    const float *val = p.bias + row * p.bias_pitch;
    const int lane = threadIdx.x;
    for (int i0 = 0; i0 < p.n_bias; i0 += 32) {
      const bool in = i0 + lane < p.n_bias;
      const int64_t at = in ? (int64_t)__ldg(ids + i0 + lane) - v0 : -1;
      const float b = in ? __ldg(val + i0 + lane) : 0.f;
      const bool mine = at >= 0 && at < n;
      const uint32_t same = __match_any_sync(0xffffffffu, mine ? (int)at : -1);
      const bool first = mine && (__ffs(same) - 1) == lane;
      float sum = first ? bias[at] + b : 0.f;
      uint32_t rest = __reduce_or_sync(0xffffffffu, first ? same & ~(1u << lane) : 0u);
      while (rest) {  // the lanes that are not first in their group, in order
        const int src = __ffs(rest) - 1;
        const float other = __shfl_sync(0xffffffffu, b, src);
        if (first && ((same >> src) & 1)) sum = sum + other;
        rest &= rest - 1;
      }
      if (first) bias[at] = sum;
      __syncwarp();
    }
  }
  __syncthreads();
  const float rep = p.repetition ? __ldg(p.repetition + row) : 1.f;
  const float freq = p.frequency ? __ldg(p.frequency + row) : 0.f;
  const float pres = p.presence ? __ldg(p.presence + row) : 0.f;
  const IoT *x = (const IoT *)p.x + row * p.x_pitch + v0;
  IoT *y = (IoT *)p.y + row * p.y_pitch + v0;
  const uint32_t *mask = p.mask ? p.mask + row * p.mask_pitch : nullptr;
  auto shape = [&](float f, int i, uint32_t allowed) -> float {
    if (counts) {
      const uint32_t c = count[i];
      if (c) {
        f = f > 0.f ? f / rep : f * rep;
        const uint32_t made = c & ~kSeen;
        if (made) f = f - freq * (float)made - pres;
      }
    }
    if (biased) f = f + bias[i];
    return allowed ? f : -INFINITY;
  };
  const int nv = n / V * V;
  for (int i = threadIdx.x * V; i < nv; i += kLogitThreads * V) {
    float f[V];
    load_vec<float, IoT, V>(x + i, f);
    const int64_t v = v0 + i;  // V entries share a mask word: V divides 32 and v is a multiple of V
    const uint32_t bits = mask ? __ldg(mask + (v >> 5)) >> (v & 31) : 0xffffffffu;
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] = shape(f[e], i + e, (bits >> e) & 1);
    store_vec<IoT, float, V>(y + i, f);
  }
  for (int i = nv + threadIdx.x; i < n; i += kLogitThreads) {  // the ragged end of the row
    const int64_t v = v0 + i;
    const uint32_t bit = mask ? (__ldg(mask + (v >> 5)) >> (v & 31)) & 1 : 1u;
    y[i] = from_compute<IoT, float>(shape(to_compute<float, IoT>(x[i]), i, bit));
  }
}

static int bad(int status, const std::string &msg) {
  set_error("logits_process: " + msg);
  return status;
}

// An optional [rows] or [rows, n] operand of 32-bit values whose rows are contiguous.
static bool rows_of(const pgb_tensor *t, int dtype, int ndim, int64_t rows, int64_t *n, int64_t *pitch) {
  if (t->dtype != dtype || t->ndim != ndim || t->shape[0] != rows || (reinterpret_cast<uintptr_t>(t->data) & 3)) return false;
  if (ndim == 1) return rows <= 1 || t->stride_bytes[0] == 4;
  if ((t->shape[1] > 1 && t->stride_bytes[1] != 4) || t->stride_bytes[0] < 0 || t->stride_bytes[0] % 4) return false;
  *n = t->shape[1];
  *pitch = t->stride_bytes[0] / 4;
  return true;
}

static int logits_process(const pgb_tensor *logits, const pgb_tensor *history, const pgb_tensor *history_len, const pgb_tensor *prompt_len,
                          const pgb_tensor *repetition, const pgb_tensor *frequency, const pgb_tensor *presence, const pgb_tensor *bias_ids,
                          const pgb_tensor *bias, const pgb_tensor *mask, const pgb_tensor *out, cudaStream_t stream) {
  if (!logits || !out) return bad(PGB_ERR_INVALID_ARG, "null tensor");
  if (logits->dtype != PGB_F16 && logits->dtype != PGB_BF16 && logits->dtype != PGB_F32) {
    set_error(std::string("logits_process not implemented for ") + dtype_name(logits->dtype));
    return PGB_ERR_UNSUPPORTED;
  }
  const int es = dtype_size(logits->dtype);
  if (logits->ndim != 2 || out->ndim != 2 || logits->shape[0] != out->shape[0] || logits->shape[1] != out->shape[1] || out->dtype != logits->dtype)
    return bad(PGB_ERR_INVALID_ARG, "logits and out must be [rows, vocabulary] of one dtype");
  const int64_t rows = logits->shape[0], V = logits->shape[1];
  for (const pgb_tensor *t : {logits, out})
    if ((V > 1 && t->stride_bytes[1] != es) || t->stride_bytes[0] < 0 || t->stride_bytes[0] % es || (reinterpret_cast<uintptr_t>(t->data) & (es - 1)))
      return bad(PGB_ERR_INVALID_ARG, "the vocabulary dim must be contiguous");
  if (rows > 1 && out->stride_bytes[0] < V * es) return bad(PGB_ERR_INVALID_ARG, "out overlaps itself");
  if (V > 2147483647LL - 65536 || rows > 65535) return bad(PGB_ERR_UNSUPPORTED, "too many rows or vocabulary entries for one launch");
  LogitParams p{};
  int64_t n = 0;
  if (history) {
    if (!rows_of(history, PGB_I32, 2, rows, &n, &p.history_pitch) || n > 2147483647LL) return bad(PGB_ERR_INVALID_ARG, "history must be int32 [rows, tokens]");
    p.L = (int)n;
  } else if (history_len || prompt_len || repetition || frequency || presence) {
    return bad(PGB_ERR_INVALID_ARG, "penalties and lengths need a history");
  }
  for (const pgb_tensor *t : {history_len, prompt_len})
    if (t && !rows_of(t, PGB_I32, 1, rows, nullptr, nullptr)) return bad(PGB_ERR_INVALID_ARG, "lengths must be int32 [rows]");
  for (const pgb_tensor *t : {repetition, frequency, presence})
    if (t && !rows_of(t, PGB_F32, 1, rows, nullptr, nullptr)) return bad(PGB_ERR_INVALID_ARG, "penalties must be float32 [rows]");
  if ((bias_ids != nullptr) != (bias != nullptr)) return bad(PGB_ERR_INVALID_ARG, "bias and bias_ids come together");
  if (bias) {
    int64_t m = 0;
    if (!rows_of(bias_ids, PGB_I32, 2, rows, &n, &p.bias_ids_pitch) || !rows_of(bias, PGB_F32, 2, rows, &m, &p.bias_pitch) || n != m || n > 2147483647LL - 32)
      return bad(PGB_ERR_INVALID_ARG, "bias_ids must be int32 and bias float32, both [rows, entries]");
    p.n_bias = (int)n;
  }
  if (mask) {
    if (!rows_of(mask, PGB_I32, 2, rows, &n, &p.mask_pitch) || n < (V + 31) / 32)
      return bad(PGB_ERR_INVALID_ARG, "mask must be int32 [rows, at least a bit for each vocabulary entry]");
  }
  int devs = 0;
  if (cudaGetDeviceCount(&devs) != cudaSuccess || devs <= 0) {
    cudaGetLastError();
    set_error("no CUDA device: this library has no CPU fallback");
    return PGB_ERR_CUDA;
  }
  if (rows == 0 || V == 0) return PGB_OK;
  p.x = logits->data;
  p.y = out->data;
  p.V = V;
  p.x_pitch = rows > 1 ? logits->stride_bytes[0] / es : 0;
  p.y_pitch = rows > 1 ? out->stride_bytes[0] / es : 0;
  auto ptr = [](const pgb_tensor *t) { return t ? t->data : nullptr; };
  p.history = p.L > 0 ? (const int *)ptr(history) : nullptr;
  p.history_len = (const int *)ptr(history_len);
  p.prompt_len = (const int *)ptr(prompt_len);
  p.repetition = (const float *)ptr(repetition);
  p.frequency = (const float *)ptr(frequency);
  p.presence = (const float *)ptr(presence);
  p.bias_ids = (const int *)ptr(bias_ids);
  p.bias = (const float *)ptr(bias);
  p.mask = (const uint32_t *)ptr(mask);
  p.slice = 4096;
  const dim3 grid((unsigned)((V + p.slice - 1) / p.slice), (unsigned)rows);
  const size_t smem = ((p.history ? 1 : 0) + (p.n_bias ? 1 : 0)) * (size_t)p.slice * 4;
  const bool aligned = !(reinterpret_cast<uintptr_t>(p.x) & 15) && !(reinterpret_cast<uintptr_t>(p.y) & 15) && (p.x_pitch * es) % 16 == 0 && (p.y_pitch * es) % 16 == 0;
#define PGB_LOGITS(T, N)                                                  \
  do {                                                                    \
    if (aligned) logits_kernel<T, N><<<grid, kLogitThreads, smem, stream>>>(p); \
    else logits_kernel<T, 1><<<grid, kLogitThreads, smem, stream>>>(p);         \
  } while (0)
  if (logits->dtype == PGB_F32) PGB_LOGITS(float, 4);
  else if (logits->dtype == PGB_F16) PGB_LOGITS(__half, 8);
  else PGB_LOGITS(__nv_bfloat16, 8);
#undef PGB_LOGITS
  count_launch();
  return check_launch("logits_kernel");
}

}  // namespace pgb

using namespace pgb;

extern "C" PGB_API int pgb_logits_process(const pgb_tensor *logits, const pgb_tensor *history, const pgb_tensor *history_len, const pgb_tensor *prompt_len,
                                          const pgb_tensor *repetition, const pgb_tensor *frequency, const pgb_tensor *presence,
                                          const pgb_tensor *bias_ids, const pgb_tensor *bias, const pgb_tensor *mask, const pgb_tensor *out, void *stream) {
  try {
    return logits_process(logits, history, history_len, prompt_len, repetition, frequency, presence, bias_ids, bias, mask, out, (cudaStream_t)stream);
  } catch (...) {  // nothing throws across the boundary: what can is the allocation of a message
    return PGB_ERR_CUDA;
  }
}
