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
//
// 256 rows of 50257 halves with histories of up to 2000 tokens, 64 biases and a mask: 33 us (54 MB: 8 us at the copy rate). The
// copy alone takes 16 us through shared memory (results at another alignment than the logits), the history 10: thirteen CTAs
// of a row read it, and a CTA's chain of loads, atomics and two barriers is a few microseconds, of which 4 to 6 overlap on an SM.
#include <cstring>
#include <string>

#include "overlap.hpp"
#include "reduce_common.cuh"
#include "vec.cuh"

namespace pgb {

constexpr int kLogitThreads = 256;
// Vocabulary entries per CTA: two 16-byte vectors a thread.
template <typename IoT> constexpr int kLogitSlice = 2 * kLogitThreads * 16 / (int)sizeof(IoT);
// A shared-memory array of them, with room to shift them as a row's start requires.
template <typename IoT> constexpr int kLogitRoom = kLogitSlice<IoT> + 8;
constexpr uint32_t kSeen = 0x80000000u;  // bit 31 of a counter: the token occurs in the prompt; the rest counts the generated ones

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
};

// V consecutive values as they lie in memory
template <typename IoT, int V>
struct alignas(sizeof(IoT) * V) RawVec { IoT v[V]; };

template <typename IoT, int V>
__global__ void __launch_bounds__(kLogitThreads) logits_kernel(const __grid_constant__ LogitParams p) {
  constexpr int kSlice = kLogitSlice<IoT>, kArray = kLogitRoom<IoT>, kVecs = kSlice / (kLogitThreads * V);
  extern __shared__ __align__(16) uint32_t smem[];
  const int64_t row = blockIdx.y;
  const int64_t v0 = (int64_t)blockIdx.x * kSlice;
  const int n = (int)min((int64_t)kSlice, p.V - v0);
  const bool counts = p.history != nullptr, biased = p.n_bias > 0;
  uint32_t *count = smem;
  float *bias = reinterpret_cast<float *>(smem + (counts ? kArray : 0));
  // where x and y are not aligned alike, the results pass through shared memory
  IoT *staged = reinterpret_cast<IoT *>(smem + (counts + biased) * kArray);
  const IoT *x = (const IoT *)p.x + row * p.x_pitch + v0;
  IoT *y = (IoT *)p.y + row * p.y_pitch + v0;
  // Rows start anywhere (50257 halves in a row: at any even address). Whole 16-byte vectors of x are taken, from entry `first`
  // on; the few entries before and behind them one by one. The arrays in shared memory are shifted likewise, so that a
  // vector's counts and biases are whole vectors too.
  const int shift = (int)((reinterpret_cast<uintptr_t>(x) / sizeof(IoT)) % V), first = (V - shift) % V;
  const int n_vec = max(0, n - first) / V;
  count += shift;
  bias += shift;
  // the slice is on its way while the history is counted
  RawVec<IoT, V> raw[kVecs];
#pragma unroll
  for (int u = 0; u < kVecs; ++u) {
    const int k = u * kLogitThreads + threadIdx.x;
    if (k < n_vec) {
      const uint4 r = __ldcs(reinterpret_cast<const uint4 *>(x + first + k * V));
      memcpy(&raw[u], &r, 16);
    }
  }
  // The last warp takes the biases, where there are any, the others the history. Its first tokens are fetched before its
  // length is known: what lies behind the length is not used.
  const int counters = kLogitThreads - (biased ? 32 : 0);
  const int *h = p.history + row * p.history_pitch;
  int len = 0, prompt = 0, early[4] = {};
  if (counts && threadIdx.x < counters) {
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if ((int)threadIdx.x + u * counters < p.L) early[u] = __ldg(h + threadIdx.x + u * counters);
    len = p.history_len ? min(max(__ldg(p.history_len + row), 0), p.L) : p.L;
    prompt = p.prompt_len ? __ldg(p.prompt_len + row) : 0;
  }
  for (int i = threadIdx.x * 4; i < (counts + biased) * kArray; i += kLogitThreads * 4) *reinterpret_cast<uint4 *>(smem + i) = make_uint4(0, 0, 0, 0);
  __syncthreads();
  if (counts && threadIdx.x < counters) {
    auto put = [&](int i, int id) {
      const int64_t at = (int64_t)id - v0;
      if (at < 0 || at >= n) return;
      if (i >= prompt) atomicAdd(count + at, 1u);  // a count that is not zero says as much as the flag
      else atomicOr(count + at, kSeen);
    };
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if ((int)threadIdx.x + u * counters < len) put(threadIdx.x + u * counters, early[u]);
    int i = threadIdx.x + 4 * counters;
    for (; i + 3 * counters < len; i += 4 * counters) {  // four loads under way
      const int a = __ldg(h + i), b = __ldg(h + i + counters), c = __ldg(h + i + 2 * counters), d = __ldg(h + i + 3 * counters);
      put(i, a);
      put(i + counters, b);
      put(i + 2 * counters, c);
      put(i + 3 * counters, d);
    }
    for (; i < len; i += counters) put(i, __ldg(h + i));
  }
  // A token may be biased more than once. One warp takes the list in order, and lanes that hold the same token leave the
  // sum to the first of them, which adds in list order: the result does not depend on timing.
  if (biased && threadIdx.x >= counters) {
    const int *ids = p.bias_ids + row * p.bias_ids_pitch;
    const float *val = p.bias + row * p.bias_pitch;
    const int lane = threadIdx.x & 31;
    for (int i0 = 0; i0 < p.n_bias; i0 += 32) {
      const bool in = i0 + lane < p.n_bias;
      const int64_t at = in ? (int64_t)__ldg(ids + i0 + lane) - v0 : -1;
      const float b = in ? __ldg(val + i0 + lane) : 0.f;
      const bool mine = at >= 0 && at < n;
      if (!__any_sync(0xffffffffu, mine)) continue;
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
  const uint32_t *mask = p.mask ? p.mask + row * p.mask_pitch : nullptr;
  auto shape = [&](float f, uint32_t c, float b, uint32_t allowed) -> float {
    if (c) {
      f = f > 0.f ? f / rep : f * rep;
      const uint32_t made = c & ~kSeen;
      if (made) f = f - freq * (float)made - pres;
    }
    if (biased) f = f + b;
    return allowed ? f : -INFINITY;
  };
  // bit e of the result: may entry i + e follow
  auto allowed = [&](int i) -> uint32_t {
    if (!mask) return 0xffffffffu;
    const int64_t v = v0 + i, w = v >> 5;
    const uint32_t lo = __ldg(mask + w), hi = (v & 31) + V > 32 && (w + 1) * 32 < p.V ? __ldg(mask + w + 1) : 0u;
    return __funnelshift_r(lo, hi, (uint32_t)(v & 31));
  };
  const int y_shift = (int)((reinterpret_cast<uintptr_t>(y) / sizeof(IoT)) % V);
  const bool alike = y_shift == shift;
#pragma unroll
  for (int u = 0; u < kVecs; ++u) {
    const int k = u * kLogitThreads + threadIdx.x;
    if (k >= n_vec) continue;
    const int i = first + k * V;
    // counts and biases in 16-byte reads: word by word, eight lanes would meet in each bank
    uint32_t c[V] = {};
    float b[V] = {};
#pragma unroll
    for (int e = 0; e < V; e += 4) {
      if (counts) {
        const uint4 r = *reinterpret_cast<const uint4 *>(count + i + e);
        c[e] = r.x; c[e + 1] = r.y; c[e + 2] = r.z; c[e + 3] = r.w;
      }
      if (biased) {
        const float4 r = *reinterpret_cast<const float4 *>(bias + i + e);
        b[e] = r.x; b[e + 1] = r.y; b[e + 2] = r.z; b[e + 3] = r.w;
      }
    }
    const uint32_t bits = allowed(i);
    float f[V];
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] = shape(to_compute<float, IoT>(raw[u].v[e]), c[e], b[e], (bits >> e) & 1);
    if (alike) {
      store_vec<IoT, float, V>(y + i, f);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) staged[y_shift + i + e] = from_compute<IoT, float>(f[e]);
    }
  }
  // the entries before the first vector and behind the last
  const int head = min(first, n), tail = first + n_vec * V, rest = head + max(0, n - tail);
  if (threadIdx.x < rest) {
    const int i = threadIdx.x < head ? threadIdx.x : tail + threadIdx.x - head;
    const IoT f = from_compute<IoT, float>(shape(to_compute<float, IoT>(x[i]), counts ? count[i] : 0u, biased ? bias[i] : 0.f, allowed(i) & 1));
    if (alike) y[i] = f;
    else staged[y_shift + i] = f;
  }
  if (alike) return;
  __syncthreads();
  const int y_first = (V - y_shift) % V, y_vec = max(0, n - y_first) / V, y_tail = y_first + y_vec * V, y_head = min(y_first, n);
  for (int k = threadIdx.x; k < y_vec; k += kLogitThreads)
    *reinterpret_cast<uint4 *>(y + y_first + k * V) = *reinterpret_cast<const uint4 *>(staged + y_shift + y_first + k * V);
  if (threadIdx.x < y_head + max(0, n - y_tail)) {
    const int i = threadIdx.x < y_head ? threadIdx.x : y_tail + threadIdx.x - y_head;
    y[i] = staged[y_shift + i];
  }
}

static int bad(int status, const std::string &msg) {
  set_error("logits_process: " + msg);
  return status;
}

// An optional [rows] or [rows, n] operand of 32-bit values whose rows are contiguous. Only one without values may be null.
static bool rows_of(const pgb_tensor *t, int dtype, int ndim, int64_t rows, int64_t *n, int64_t *pitch) {
  if (t->dtype != dtype || t->ndim != ndim || t->shape[0] != rows || (reinterpret_cast<uintptr_t>(t->data) & 3)) return false;
  if (rows > 0 && (ndim == 1 || t->shape[1] > 0) && !t->data) return false;
  if (ndim == 1) return rows <= 1 || t->stride_bytes[0] == 4;
  if (t->shape[1] < 0 || (t->shape[1] > 1 && t->stride_bytes[1] != 4) || t->stride_bytes[0] < 0 || t->stride_bytes[0] % 4) return false;
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
  if (rows < 0 || V < 0) return bad(PGB_ERR_INVALID_ARG, "negative rows or vocabulary");
  if (rows && V && (!logits->data || !out->data)) return bad(PGB_ERR_INVALID_ARG, "null tensor");
  for (const pgb_tensor *t : {logits, out})
    if ((V > 1 && t->stride_bytes[1] != es) || t->stride_bytes[0] < 0 || t->stride_bytes[0] % es || (reinterpret_cast<uintptr_t>(t->data) & (es - 1)))
      return bad(PGB_ERR_INVALID_ARG, "the vocabulary dim must be contiguous");
  if (rows > 1 && out->stride_bytes[0] < V * es) return bad(PGB_ERR_INVALID_ARG, "out overlaps itself");
  if (V > 2147483647LL - 65536 || rows > 65535) return bad(PGB_ERR_UNSUPPORTED, "too many rows or vocabulary entries for one launch");
  LogitParams p{};
  int64_t n = 0;
  if (history) {
    if (!rows_of(history, PGB_I32, 2, rows, &n, &p.history_pitch) || n > 2147483647LL - 65536) return bad(PGB_ERR_INVALID_ARG, "history must be int32 [rows, tokens]");
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
  const ByteView written = view_of(*out, es);
  for (const pgb_tensor *t : {logits, history, history_len, prompt_len, repetition, frequency, presence, bias_ids, bias, mask}) {
    if (!t) continue;
    const ByteView v = view_of(*t, dtype_size(t->dtype));
    if (views_share(written, v) && !(t == logits && v == written))
      return bad(PGB_ERR_INVALID_ARG, "out shares memory with an operand (it may be logits itself, but no other view of it)");
  }
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
  // alike for every row where the bases are alike and the pitches differ by whole vectors, or there is one row
  const bool alike = (reinterpret_cast<uintptr_t>(p.x) - reinterpret_cast<uintptr_t>(p.y)) % 16 == 0 && ((p.x_pitch - p.y_pitch) * es) % 16 == 0;
  auto launch = [&](auto kernel, int slice, int room) {
    const size_t smem = ((p.history ? 1 : 0) + (p.n_bias ? 1 : 0)) * (size_t)room * 4 + (alike ? 0 : (size_t)room * es);
    kernel<<<dim3((unsigned)((V + slice - 1) / slice), (unsigned)rows), kLogitThreads, smem, stream>>>(p);
  };
  if (logits->dtype == PGB_F32) launch(logits_kernel<float, 4>, kLogitSlice<float>, kLogitRoom<float>);
  else if (logits->dtype == PGB_F16) launch(logits_kernel<__half, 8>, kLogitSlice<__half>, kLogitRoom<__half>);
  else launch(logits_kernel<__nv_bfloat16, 8>, kLogitSlice<__nv_bfloat16>, kLogitRoom<__nv_bfloat16>);
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
