// The paged key / value cache as the kernels see it: views of the pages, the plan that maps packed rows to sequences
// and positions, and the host-side checks that the entry points of the cache share.
//
// The reference's GPT-2 recomputes every position for each new token (examples/gpt2.py:406-438) and has no cache.
#pragma once
#include <initializer_list>
#include <string>

#include "gemm.hpp"
#include "overlap.hpp"
#include "reduce_common.cuh"

namespace pgb {

// Pages of K or of V: [n_pages, heads, page size, head dim], head dim contiguous, strides in bytes. An int8 cache has one
// fp32 scale per page, head and slot (slots contiguous, strides in elements).
struct KvPages {
  uint8_t *base;
  int64_t page, head, slot;
  float *scale;
  int64_t scale_page, scale_head;
};

struct KvCache {
  KvPages k, v;
  int n_pages, heads, log2_page, head_dim, dtype;
};

// start: row offsets of the sequences, [n_seq + 1]; ctx: cached tokens of each sequence, its new ones included (null where
// positions count from zero); table: the pages of each sequence, [n_seq, width], pitch in elements.
struct KvPlan {
  const int *start, *ctx, *table;
  int64_t pitch;
  int n_seq, width;
};

// The sequence that row r belongs to, or -1 for a row behind the last one. Decoding has one row per sequence, so r itself
// is tried first. Offsets that do not increase give some sequence, never an index out of range.
__device__ __forceinline__ int kv_sequence(const KvPlan &p, int64_t r) {
  if (r < p.n_seq && __ldg(p.start + r) <= r && __ldg(p.start + r + 1) > r) return (int)r;
  int lo = 0, hi = p.n_seq;  // start[lo] <= r < start[hi], once the ends are checked
  if (__ldg(p.start) > r || __ldg(p.start + hi) <= r) return -1;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(p.start + mid) <= r) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Position of row r of sequence s in its context; negative where the context is shorter than the new rows.
__device__ __forceinline__ int64_t kv_position(const KvPlan &p, int s, int64_t r) {
  if (!p.ctx) return r - __ldg(p.start + s);
  return (int64_t)__ldg(p.ctx + s) + r - __ldg(p.start + s + 1);
}

// The page that holds a position, or -1 where the table has none (a position outside the table, an entry outside the cache).
__device__ __forceinline__ int kv_page(const KvPlan &p, const KvCache &c, int s, int64_t pos) {
  const int64_t i = pos >> c.log2_page;
  if (pos < 0 || i >= p.width) return -1;
  const int page = __ldg(p.table + (int64_t)s * p.pitch + i);
  return page >= 0 && page < c.n_pages ? page : -1;
}

// Host side. Each returns a pgb_status and leaves the message in pgb_last_error(); `what` names the entry point.
int kv_parse_cache(const char *what, const pgb_tensor *k_cache, const pgb_tensor *v_cache, const pgb_tensor *k_scale,
                   const pgb_tensor *v_scale, bool writes, KvCache &c);
int kv_parse_plan(const char *what, const pgb_tensor *start, const pgb_tensor *ctx, const pgb_tensor *table, KvPlan &p);
// A [rows, heads, head dim] operand: head dim contiguous, rows and heads 16-byte aligned; strides in bytes.
int kv_parse_rows(const char *what, const char *name, const pgb_tensor *t, int64_t heads, int head_dim, bool writes, int64_t *row,
                  int64_t *head);
bool kv_device_present();
// No tensor of `written` may share memory with another one or with one of `read`: null tensors are passed over.
struct KvOperand {
  const char *name;
  const pgb_tensor *t;
};
int kv_apart(const char *what, std::initializer_list<KvOperand> written, std::initializer_list<KvOperand> read);

}  // namespace pgb
