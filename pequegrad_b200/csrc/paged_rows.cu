// Attention over the paged cache for few rows per sequence (decoding, speculated continuations).
//
// The work is reading the cache once: 16 rows of arithmetic ride on every key, so the kernel is bound by HBM, and with one
// short sequence by latency. A work item is (16 rows, key head): the rows are consecutive tokens times the query heads that
// share the key head. Its keys are split over the CTAs of a cluster and their warps, 16 or 32 keys at a time.
//   copies   each lane copies its own fragments into its own slots of shared memory with cp.async, several blocks ahead, and
//            reads them back itself: no barrier, and the copies in flight cost no registers. A key that nobody sees (behind
//            the context, no page) is filled with zeros, so that nothing stale meets a probability of zero.
//   products mma.sync m16n8k16: one token of one head uses a sixteenth of it, and still the tensor pipe waits for memory. The
//            contraction is taken in whatever order the 16-byte chunks of a row arrive (Q is held in that order), and the
//            columns of the output likewise, so both products take their operands as they lie in memory.
//   softmax  running maximum and sum per row in fp32; the warps' and then the CTAs' partial results are joined in shared and
//            distributed shared memory, in a fixed order. No scratch in global memory, nothing shared between launches.
//   int8     widened exactly to fp16; the key's scale multiplies its scores, the value's scale its probabilities, in fp32.
// Measured: 16 sequences of up to 32768 int8 tokens, 32 heads of 128 on 8: 183 us, 3.4 TB/s, half the copy rate; 64 of up to
// 1024 tokens, 12 heads of 64 in fp16: 38 us, 3.5 TB/s. What bounds them then is the latency of a warp's chain from copy to
// second product, with the twelve warps whose registers fit an SM (eight, whose stages do, with 128 values of 16 bits). Tiles of
// 8 rows (half the output's registers) gave 176 and 39 us, a cap at 128 registers for sixteen warps 329 (spills): neither is
// worth a second set of kernels.
#include <atomic>
#include <string>
#include <type_traits>

#include "paged.cuh"

namespace pgb {

template <int D, bool I8>
struct RowTile {
  // Warps that share an item's keys. Short rows: two, so that all the items of a batch run at once (64 sequences, 12 heads of
  // 64: 37 us against 41 with four); long ones: four (16 sequences of up to 32768 int8 tokens, 8 heads of 128: 184 us
  // against 191 with two and 254 with eight).
  static constexpr int kWarps = D == 64 ? 2 : 4;
  static constexpr int kEs = I8 ? 1 : 2;
  static constexpr int kKChunks = D * kEs / 64;              // 16-byte chunks of one key that a lane holds
  static constexpr int kVBytes = D * kEs / 8;                // bytes of one value row that a lane holds
  static constexpr int kVPiece = kVBytes < 16 ? 8 : 16;      // copied at once
  static constexpr int kVPieces = kVBytes / kVPiece;
  static constexpr int kK = 2 * kKChunks * 512, kV = 4 * kVPieces * 32 * kVPiece;
  static constexpr int kSub = kK + kV + (I8 ? 128 : 0);      // 16 keys of one warp; with int8 their 32 scales
  // Sub-blocks a warp takes at once: with short rows two, whose chains of products overlap and which share one turn of the
  // running maximum (64 sequences of 1024, 12 heads of 64: 43 us with one).
  static constexpr int kSubs = D == 64 ? 2 : 1;
  static constexpr int kStage = kSubs * kSub;
  static constexpr int kStages = kEs * kSubs == 4 ? 2 : (D * kEs > 128 || kSubs == 2 ? 3 : 4);
  static constexpr int kWarp = kStages * kStage;
  static constexpr int kJoin = kWarps * 16 * (D + 2) * 4;
  static constexpr int kSmem = (kWarps * kWarp > kJoin ? kWarps * kWarp : kJoin) + 16 * (D + 2) * 4;
  static constexpr int kFit = 233472 / (kSmem + 1024);  // CTAs that the shared memory of an SM holds
  static constexpr int kCtas = kFit < 12 / kWarps ? kFit : 12 / kWarps;  // and registers: twelve warps
};

__device__ __forceinline__ void copy8(uint32_t dst, const void *src, bool there) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(there ? 8 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <bool HALF>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (HALF)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <bool HALF>
__device__ __forceinline__ bool not_finite(uint32_t bits) {  // of one 16-bit float
  constexpr uint32_t e = HALF ? 0x7c00u : 0x7f80u;
  return (bits & e) == e;
}
__device__ __forceinline__ uint4 ld_shared16(uint32_t a) {
  uint4 r;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(a) : "memory");
  return r;
}
__device__ __forceinline__ uint2 ld_shared8(uint32_t a) {
  uint2 r;
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(r.x), "=r"(r.y) : "r"(a) : "memory");
  return r;
}
template <bool HALF, int D, bool I8>
__global__ void __launch_bounds__(RowTile<D, I8>::kWarps * 32, RowTile<D, I8>::kCtas) paged_rows_kernel(const __grid_constant__ PagedParams a, const __grid_constant__ KvCache c,
                                                                       const __grid_constant__ KvPlan p, unsigned splits, unsigned tiles_per_token, int by_slot) {
  using S = RowTile<D, I8>;
  constexpr int kRowWarps = S::kWarps;
  extern __shared__ __align__(16) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quad = lane >> 2, t = lane & 3;
  const int rank = (int)(blockIdx.x % splits);  // of the CTA in its cluster
  unsigned unit = blockIdx.x / splits;
  const int kvh = (int)(unit % c.heads);
  unit /= c.heads;
  const int sub = (int)(unit % tiles_per_token);  // which 16 query heads, where more than that share a key head
  const int tokens = a.group >= 16 ? 1 : 16 / a.group;  // tokens of a tile
  // One tile for each row (with one new token per sequence), of which those return that begin none; or one for each slot:
  // the slots of sequence s begin at start[s] / tokens + s, and it has at least as many as tiles.
  int64_t row0 = unit / tiles_per_token, first;
  int seq;
  if (by_slot) {
    const int64_t slot = row0;
    int hi = p.n_seq;
    seq = 0;
    while (hi - seq > 1) {
      const int mid = (seq + hi) >> 1;
      if (__ldg(p.start + mid) / tokens + mid <= slot) seq = mid;
      else hi = mid;
    }
    first = __ldg(p.start + seq);
    row0 = first + (slot - first / tokens - seq) * tokens;
  } else {
    seq = kv_sequence(p, row0);
    if (seq < 0) return;
    first = __ldg(p.start + seq);
    if ((row0 - first) % tokens) return;  // another tile's row
  }
  const int64_t end = min((int64_t)__ldg(p.start + seq + 1), a.rows);
  if (first < 0 || row0 < first || row0 >= end) return;
  // Row i of the tile: token i / group, query head i % group (of the 16 that start at sub * 16)
  const int heads_here = min(a.group - sub * 16, 16);
  const int n_tok = (int)min((int64_t)tokens, end - row0);
  const int n_rows = n_tok * heads_here;
  const int held = p.width << c.log2_page;  // at most 2^30
  const int pos0 = (int)max(kv_position(p, seq, row0), -((int64_t)1 << 31));
  const int n_keys = max(0, min(held, pos0 + n_tok));  // what the tile's last token sees
  const int n_blocks = (n_keys + 16 * S::kSubs - 1) / (16 * S::kSubs);

  // Q in the order in which the chunks of K arrive: value i of this lane's D / 4 is d = 16/es * (t + 4 (i es / 16)) + ...
  // Beside an int8 cache the products run in fp16: there a key widens in fewer steps than in bf16. A bf16 row of Q is brought
  // into fp16's range by a power of two, exactly but for values 2^-29 of the row's largest; its scores are scaled back.
  constexpr bool kHalfMma = HALF || I8;
  constexpr int kPer = 16 / S::kEs;  // values in a 16-byte chunk of K
  uint32_t q[D / 16][4];
  int lim[2];      // last key that the lane's two rows see
  float scale[2];  // of their scores
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int i = quad + 8 * h;
    const int tok = i / heads_here, head = i - tok * heads_here;
    const bool in = i < n_rows;
    lim[h] = in ? min(pos0 + tok, held - 1) : -1;
    scale[h] = a.c;
    const uint8_t *src = a.q + (row0 + (in ? tok : 0)) * a.q_row + ((int64_t)kvh * a.group + sub * 16 + (in ? head : 0)) * a.q_head;
#pragma unroll
    for (int j = 0; j < S::kKChunks; ++j) {
#pragma unroll
      for (int e = 0; e < kPer; e += 8) {
        uint4 r = make_uint4(0, 0, 0, 0);
        if (in) r = __ldg(reinterpret_cast<const uint4 *>(src + 2 * (kPer * (t + 4 * j) + e)));
        const int s = (j * kPer + e) / 4;
        q[s][h] = r.x; q[s][2 + h] = r.y;
        q[s + 1][h] = r.z; q[s + 1][2 + h] = r.w;
      }
    }
    if constexpr (I8 && !HALF) {
      uint32_t top = 0;  // largest |q| as bf16 bits
#pragma unroll
      for (int s = 0; s < D / 16; ++s)
#pragma unroll
        for (int e = 0; e < 2; ++e) top = max(top, max(q[s][2 * e + h] & 0x7fffu, (q[s][2 * e + h] >> 16) & 0x7fffu));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int up = min(14 + 127 - (int)(top >> 7), 100);  // the largest value lands in [2^14, 2^15)
      const float f = __uint_as_float((uint32_t)(up + 127) << 23);
      scale[h] *= __uint_as_float((uint32_t)(127 - up) << 23);
#pragma unroll
      for (int s = 0; s < D / 16; ++s)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          uint32_t &w = q[s][2 * e + h];
          w = out_pair<true>(__uint_as_float(w << 16) * f, __uint_as_float(w & 0xffff0000u) * f);
        }
    }
  }
  const int lim_min = pos0;  // the tile's first token: keys up to here are seen by all its rows

  const uint32_t base = (uint32_t)__cvta_generic_to_shared(smem) + warp * S::kWarp;
  const int step = (int)splits * kRowWarps, block0 = rank * kRowWarps + warp, page_mask = (1 << c.log2_page) - 1;
  const int *table = p.table + (int64_t)seq * p.pitch;
  const uint8_t *k_head = c.k.base + kvh * c.k.head + quad * c.k.slot + t * 16, *v_head = c.v.base + kvh * c.v.head + 2 * t * c.v.slot + quad * S::kVPiece;
  // the table's entry for block kb; looked up long before it is judged
  struct Entries { int page[S::kSubs]; };
  auto entry_of = [&](int kb) -> Entries {
    Entries e;
#pragma unroll
    for (int u = 0; u < S::kSubs; ++u) {
      const int key0 = (kb * S::kSubs + u) << 4;
      e.page[u] = key0 < n_keys ? __ldg(table + (key0 >> c.log2_page)) : -1;
    }
    return e;
  };
  // Starts the copies of 16 keys (of the page given) into their place. What the lane copies is what it reads.
  auto fetch_sub = [&](int key0, int page, uint32_t dst) {
    {
      const int slot0 = key0 & page_mask;
      const bool ok = (unsigned)page < (unsigned)c.n_pages;
      const int64_t pg = ok ? page : 0;
      const int there = ok ? n_keys - key0 : 0;  // keys that exist, if fewer than 16
      const uint8_t *k = k_head + pg * c.k.page + slot0 * c.k.slot, *v = v_head + pg * c.v.page + slot0 * c.v.slot;
      auto pieces = [&](auto whole) {
        constexpr bool kWhole = decltype(whole)::value;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const bool in = kWhole || quad + 8 * h < there;
#pragma unroll
          for (int j = 0; j < S::kKChunks; ++j)
            paged_copy16(dst + ((h * S::kKChunks + j) * 32 + lane) * 16, in ? k + h * 8 * c.k.slot + j * 64 : c.k.base, in);
        }
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const bool in = kWhole || 2 * t + (g & 1) + 8 * (g >> 1) < there;
#pragma unroll
          for (int j = 0; j < S::kVPieces; ++j) {
            const uint32_t to = dst + S::kK + ((g * S::kVPieces + j) * 32 + lane) * S::kVPiece;
            const uint8_t *from = in ? v + ((g & 1) + 8 * (g >> 1)) * c.v.slot + j * 8 * S::kVPiece : c.v.base;
            if (S::kVPiece == 16) paged_copy16(to, from, in);
            else copy8(to, from, in);
          }
        }
      };
      if (there >= 16) pieces(std::true_type{});
      else pieces(std::false_type{});
      if (I8 && lane < 8) {  // scales of the block: slots are contiguous, 16 of them 16-byte aligned
        const KvPages &w = lane < 4 ? c.k : c.v;
        const float *s = w.scale + pg * w.scale_page + kvh * w.scale_head + slot0 + (lane & 3) * 4;
        paged_copy16(dst + S::kK + S::kV + lane * 16, s, ok);
      }
    }
  };
  auto fetch = [&](int kb, const Entries &e, int stage) {
    if (kb < n_blocks) {
#pragma unroll
      for (int u = 0; u < S::kSubs; ++u) fetch_sub((kb * S::kSubs + u) << 4, e.page[u], base + stage * S::kStage + u * S::kSub);
    }
    copy_commit();  // empty groups keep the count
  };

  float o[D / 8][4];
#pragma unroll
  for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  // m is the reference of the exponents. Beside an int8 cache it counts the power of two of each key's value scale: the scaled
  // probabilities then stay within fp16, the largest of a row at order one, whatever ratios the scales have and whatever
  // lies where the row must not look. It is in the sums too, so O / l is what it was.
  constexpr float kNothing = -80.f;  // log2 of a scale whose values are nothing: a sum of 2^94s is within fp32
  // fp16 probabilities are held 2^14 times too large, at most 2^15 with a value's scale: what fp16 rounds coarsely or drops is
  // that much smaller then. The sum has the factor too.
  constexpr float kUp = kHalfMma ? 14.f : 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  bool met[2] = {false, false};  // the row has a key

  Entries pages[S::kStages];  // table entries of the blocks under way
#pragma unroll
  for (int i = 0; i < S::kStages; ++i) pages[i] = entry_of(block0 + i * step);
#pragma unroll
  for (int i = 0; i < S::kStages - 1; ++i) fetch(block0 + i * step, pages[i], i);
  int stage = 0;
  for (int kb = block0; kb < n_blocks; kb += step) {
    bool absent[S::kSubs], any_absent = false;
#pragma unroll
    for (int u = 0; u < S::kSubs; ++u) {
      absent[u] = (unsigned)pages[0].page[u] >= (unsigned)c.n_pages;
      any_absent |= absent[u];
    }
    fetch(kb + (S::kStages - 1) * step, pages[S::kStages - 1], stage == 0 ? S::kStages - 1 : stage - 1);
#pragma unroll
    for (int i = 0; i + 1 < S::kStages; ++i) pages[i] = pages[i + 1];
    pages[S::kStages - 1] = entry_of(kb + S::kStages * step);
    copy_wait<S::kStages - 1>();
    if (I8) __syncwarp();  // the scales were copied by other lanes
    const uint32_t src = base + stage * S::kStage;
    stage = stage + 1 == S::kStages ? 0 : stage + 1;

    constexpr int U = S::kSubs;
    float s[U][2][4] = {};  // of sub-block u, half h: [0..1] row quad, [2..3] row quad + 8; keys 2t, 2t + 1 of the half
#pragma unroll
    for (int j = 0; j < S::kKChunks; ++j)
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint4 r = ld_shared16(src + u * S::kSub + ((h * S::kKChunks + j) * 32 + lane) * 16);
          if constexpr (I8) {
            const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) mma16816<true>(s[u][h], q[4 * j + e], paged_widen2<true>(w[e], 0), paged_widen2<true>(w[e], 1));
          } else {
            mma16816<HALF>(s[u][h], q[2 * j], r.x, r.y);
            mma16816<HALF>(s[u][h], q[2 * j + 1], r.z, r.w);
          }
        }
    const int key0 = kb * (16 * U);
    const bool masked = key0 + 16 * U - 1 > lim_min || any_absent;  // warp-uniform
    float vs[U][4];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if constexpr (I8) {
        const uint32_t at = src + u * S::kSub + S::kK + S::kV + 8 * t;
        const uint2 k0 = ld_shared8(at), k1 = ld_shared8(at + 32), v0 = ld_shared8(at + 64), v1 = ld_shared8(at + 96);
        const float ks[4] = {__uint_as_float(k0.x), __uint_as_float(k0.y), __uint_as_float(k1.x), __uint_as_float(k1.y)};
        vs[u][0] = __uint_as_float(v0.x); vs[u][1] = __uint_as_float(v0.y); vs[u][2] = __uint_as_float(v1.x); vs[u][3] = __uint_as_float(v1.y);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[u][h][e] *= ks[2 * h + (e & 1)];
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[u][h][e] *= scale[e >> 1];
      if (masked) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int key = key0 + 16 * u + 8 * h + 2 * t + (e & 1);
            if (key > lim[e >> 1] || absent[u]) s[u][h][e] = -INFINITY;
            else met[e >> 1] = true;
            // a slot behind the context has a stale scale: its probability of zero must meet a number
            if (I8 && e < 2 && (key >= n_keys || absent[u])) vs[u][2 * h + e] = 0.f;
          }
      }
    }
    if (!masked) met[0] = met[1] = true;
    float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float ev = 0.f;
          if constexpr (I8) {
            const int top = (int)((__float_as_uint(vs[u][2 * h + e]) >> 23) & 255);
            ev = top == 255 ? kNothing : fmaxf((float)(top - 127), kNothing);
          }
          mx[0] = fmaxf(mx[0], I8 ? s[u][h][e] + ev : s[u][h][e]);
          mx[1] = fmaxf(mx[1], I8 ? s[u][h][2 + e] + ev : s[u][h][2 + e]);
        }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
      mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
    }
    if (__any_sync(0xffffffffu, mx[0] > m[0] || mx[1] > m[1])) {  // rare once the largest scores have been met
      float alpha[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float mn = fmaxf(m[r], mx[r]);
        alpha[r] = mn == -INFINITY ? 1.f : ex2f(m[r] - mn);
        m[r] = mn;
        l[r] *= alpha[r];
      }
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        o[i][0] *= alpha[0]; o[i][1] *= alpha[0];
        o[i][2] *= alpha[1]; o[i][3] *= alpha[1];
      }
    }
    const float ref[2] = {m[0] == -INFINITY ? 0.f : m[0] - kUp, m[1] == -INFINITY ? 0.f : m[1] - kUp};
    bool cleared = false;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      // The probabilities as the A operand of the second product: the accumulator's layout is the operand's.
      uint32_t pa[4];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float x = ex2f(s[u][h][2 * r] - ref[r]), y = ex2f(s[u][h][2 * r + 1] - ref[r]);
          l[r] += x + y;
          if (I8) {  // a token that a row does not see may have a scale that is no number
            x = x == 0.f ? 0.f : x * vs[u][2 * h];
            y = y == 0.f ? 0.f : y * vs[u][2 * h + 1];
          }
          pa[2 * h + r] = out_pair<kHalfMma>(x, y);
        }
      const uint32_t vsrc = src + u * S::kSub + S::kK + lane * S::kVPiece;
      auto value_words = [&](int g, int j) -> uint4 {
        const uint32_t at = vsrc + (g * S::kVPieces + j) * 32 * S::kVPiece;
        if constexpr (S::kVPiece == 16) {
          uint4 r = ld_shared16(at);
          // A new token that some rows must not see: NaN and infinities would reach them through a probability of zero.
          if (!I8 && masked && key0 + 16 * u + 2 * t + (g & 1) + 8 * (g >> 1) > lim_min) {
            uint32_t *w = reinterpret_cast<uint32_t *>(&r);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const bool lo = not_finite<HALF>(w[e] & 0xffffu), hi = not_finite<HALF>(w[e] >> 16);
              if (lo) w[e] &= 0xffff0000u;
              if (hi) w[e] &= 0xffffu;
              cleared |= lo || hi;
            }
          }
          return r;
        } else {
          const uint2 r = ld_shared8(at);
          return make_uint4(r.x, r.y, 0, 0);
        }
      };
#pragma unroll
      for (int j = 0; j < S::kVPieces; ++j) {
        const uint4 r0 = value_words(0, j), r1 = value_words(1, j), r2 = value_words(2, j), r3 = value_words(3, j);
        const uint32_t w0[4] = {r0.x, r0.y, r0.z, r0.w}, w1[4] = {r1.x, r1.y, r1.z, r1.w}, w2[4] = {r2.x, r2.y, r2.z, r2.w}, w3[4] = {r3.x, r3.y, r3.z, r3.w};
        constexpr int kWords = S::kVPiece / 4;
#pragma unroll
        for (int e = 0; e < kWords; ++e) {
          if constexpr (I8) {
            // bytes of two keys interleaved, then each pair widened: value d of keys 2t and 2t + 1 in one register
            const uint32_t lo01 = __byte_perm(w0[e], w1[e], 0x5140), hi01 = __byte_perm(w0[e], w1[e], 0x7362);
            const uint32_t lo23 = __byte_perm(w2[e], w3[e], 0x5140), hi23 = __byte_perm(w2[e], w3[e], 0x7362);
#pragma unroll
            for (int d = 0; d < 4; ++d)
              mma16816<true>(o[j * kWords * 4 + 4 * e + d], pa, paged_widen2<true>(d < 2 ? lo01 : hi01, d & 1), paged_widen2<true>(d < 2 ? lo23 : hi23, d & 1));
          } else {
            mma16816<HALF>(o[j * 8 + 2 * e], pa, __byte_perm(w0[e], w1[e], 0x5410), __byte_perm(w2[e], w3[e], 0x5410));
            mma16816<HALF>(o[j * 8 + 2 * e + 1], pa, __byte_perm(w0[e], w1[e], 0x7632), __byte_perm(w2[e], w3[e], 0x7632));
          }
        }
      }
    }
    if constexpr (!I8) {
      if (masked && __any_sync(0xffffffffu, cleared)) {  // rare: give back what was cleared, to the rows that see it
        __syncwarp();                                    // the values lie in other lanes' slots
        for (int key = max(0, lim_min + 1 - key0); key < min(16 * U, n_keys - key0); ++key) {
          const int g = (key & 1) + 2 * ((key >> 3) & 1), owner = (key & 7) >> 1;
#pragma unroll
          for (int i = 0; i < D / 8; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const uint32_t at = src + (key >> 4) * S::kSub + S::kK + ((g * S::kVPieces + i / 8) * 32 + (2 * t + e) * 4 + owner) * 16 + 2 * (i % 8);
              unsigned short bits;
              asm volatile("ld.shared.u16 %0, [%1];" : "=h"(bits) : "r"(at) : "memory");
              if (!not_finite<HALF>(bits)) continue;
              const float v = HALF ? __half2float(__ushort_as_half(bits)) : __uint_as_float((uint32_t)bits << 16);
              if (key0 + key <= lim[0]) o[i][e] += v;
              if (key0 + key <= lim[1]) o[i][2 + e] += v;
            }
        }
        __syncwarp();
      }
    }
  }
  copy_wait<0>();
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    met[r] = (__ballot_sync(0xffffffffu, met[r]) >> (lane & 28)) & 15;
  }
  __syncthreads();  // every warp is done with its stages: the memory now holds partial results

  // [warp][row][D], then m and l of [warp][row]. Accumulator i of a lane's columns 2t, 2t + 1 is value kCol * (2t + e) + i of
  // its piece (kCol values a column).
  float *part = reinterpret_cast<float *>(smem);
  float *part_m = part + kRowWarps * 16 * D, *part_l = part_m + kRowWarps * 16;
  constexpr int kCol = S::kVPiece / S::kEs;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int row = quad + 8 * r;
    if (row < n_rows) {
      float *dst = part + (warp * 16 + row) * D;
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        const int piece = i / kCol, d = piece * 8 * kCol + i % kCol;
        dst[d + kCol * (2 * t)] = o[i][2 * r];
        dst[d + kCol * (2 * t + 1)] = o[i][2 * r + 1];
      }
      if (t == 0) {
        // No key, or none with a score above -infinity: the sum says which, and the softmax is that of nothing (zeros) or no number.
        // With a score that is NaN, so is l.
        const bool low = m[r] == -INFINITY && l[r] == 0.f;
        part_m[warp * 16 + row] = low || m[r] != -INFINITY ? m[r] : 0.f;
        part_l[warp * 16 + row] = low ? (met[r] ? 1.f : 0.f) : l[r];
      }
    }
  }
  __syncthreads();
  // the warps of this CTA, and behind a cluster barrier its CTAs
  float *mine = reinterpret_cast<float *>(smem + S::kSmem) - 16 * (D + 2), *mine_m = mine + 16 * D, *mine_l = mine_m + 16;
  auto write = [&](int row, int d, float x) {  // two neighbours are written by two lanes
    const int tok = row / heads_here, head = row - tok * heads_here;
    uint8_t *out = a.out + (row0 + tok) * a.o_row + ((int64_t)kvh * a.group + sub * 16 + head) * a.o_head;
    const float y = __shfl_down_sync(__activemask(), x, 1);
    if (!(d & 1)) *reinterpret_cast<uint32_t *>(out + 2 * d) = out_pair<HALF>(x, y);
  };
  for (int i = threadIdx.x; i < n_rows * D; i += kRowWarps * 32) {
    const int row = i / D, d = i % D;
    float mm = -INFINITY;
#pragma unroll
    for (int w = 0; w < kRowWarps; ++w) mm = fmaxf(mm, part_m[w * 16 + row]);
    float x = 0.f, sum = 0.f;
    if (mm != -INFINITY) {
#pragma unroll
      for (int w = 0; w < kRowWarps; ++w) {
        const float e = ex2f(part_m[w * 16 + row] - mm);
        x += part[(w * 16 + row) * D + d] * e;
        sum += part_l[w * 16 + row] * e;
      }
    } else {
#pragma unroll
      for (int w = 0; w < kRowWarps; ++w) sum += part_l[w * 16 + row];
    }
    if (splits == 1) {
      write(row, d, mm == -INFINITY ? (sum == 0.f ? 0.f : NAN) : x / sum);
    } else {
      mine[row * D + d] = x;
      if (d == 0) { mine_m[row] = mm; mine_l[row] = sum; }
    }
  }
  if (splits == 1) return;
  paged_cluster_sync();
  const uint32_t at = (uint32_t)__cvta_generic_to_shared(mine), at_m = (uint32_t)__cvta_generic_to_shared(mine_m), at_l = (uint32_t)__cvta_generic_to_shared(mine_l);
  // each CTA writes its share of the outputs: 32 of them at a time
  for (int i = (rank * kRowWarps + warp) * 32 + lane; i < n_rows * D; i += splits * kRowWarps * 32) {
    const int row = i / D, d = i % D;
    float mm = -INFINITY;
    for (int s = 0; s < splits; ++s) mm = fmaxf(mm, paged_peer(at_m + 4 * row, s));
    float x = 0.f, sum = 0.f;
    if (mm != -INFINITY) {
      for (int s = 0; s < splits; ++s) {
        const float e = ex2f(paged_peer(at_m + 4 * row, s) - mm);
        x += paged_peer(at + 4 * i, s) * e;
        sum += paged_peer(at_l + 4 * row, s) * e;
      }
    } else {
      for (int s = 0; s < splits; ++s) sum += paged_peer(at_l + 4 * row, s);
    }
    write(row, d, mm == -INFINITY ? (sum == 0.f ? 0.f : NAN) : x / sum);
  }
  paged_cluster_sync();  // nobody's shared memory goes away while it is read
}

template <bool HALF, int D, bool I8>
static int launch(const PagedParams &a, const KvCache &c, const KvPlan &p, int splits, int tiles_per_token, bool by_slot, int64_t units, cudaStream_t stream) {
  using S = RowTile<D, I8>;
  const auto kernel = paged_rows_kernel<HALF, D, I8>;
  // the attribute belongs to the device: set once on each, again where two threads meet
  static std::atomic<bool> ready[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64 || !ready[dev].load(std::memory_order_relaxed)) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem);
    if (e != cudaSuccess) {
      set_error(std::string("paged_attention: cannot raise the shared-memory limit: ") + cudaGetErrorString(e));
      return PGB_ERR_CUDA;
    }
    if (dev >= 0 && dev < 64) ready[dev].store(true, std::memory_order_relaxed);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(units * splits));
  cfg.blockDim = dim3(S::kWarps * 32);
  cfg.dynamicSmemBytes = S::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = splits;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a, c, p, (unsigned)splits, (unsigned)tiles_per_token, by_slot ? 1 : 0);
  if (e != cudaSuccess) {
    cudaGetLastError();
    set_error(std::string("paged_rows_kernel: ") + cudaGetErrorString(e));
    return PGB_ERR_CUDA;
  }
  count_launch();
  return PGB_OK;
}

int run_paged_rows(const PagedParams &a, const KvCache &c, const KvPlan &p, bool half, cudaStream_t stream) {
  const int tiles_per_token = (a.group + 15) / 16;
  // Work is dealt out by rows or by slots, whichever are fewer (4 sequences of 4000 tokens, 16 heads of 128, 16 new tokens each: 77
  // and 55 us). Some of either have nothing to do; the tiles, of which each sequence that has rows adds at most one that is not
  // full, are what counts for the split.
  const int64_t tokens = a.group >= 16 ? 1 : 16 / a.group, k = p.n_seq < a.rows ? p.n_seq : a.rows;
  const bool by_slot = a.rows / tokens + p.n_seq < a.rows;
  const int64_t units = (by_slot ? a.rows / tokens + p.n_seq : a.rows) * tiles_per_token * c.heads;
  const int64_t tiles = ((a.rows - k) / tokens + k) * tiles_per_token * c.heads;
  // As many CTAs per item as leave no SM idle, up to a portable cluster; not more than have a block of keys for each warp, or two
  // where a tile has several tokens' rows to join (the same with 300 tokens: 25 us with one, 16 with two, 19 with four).
  int splits = 1;
  const int warps = c.head_dim == 64 ? 2 : 4;
  const int64_t blocks = ((int64_t)p.width << c.log2_page) / (c.head_dim == 64 ? 32 : 16);
  while (splits < 8 && tiles * splits < 4LL * sm_count() && blocks > (int64_t)splits * warps * (a.rows > p.n_seq ? 2 : 1)) splits *= 2;
  if (units * splits > 2147483647LL) {
    set_error("paged_attention: too many rows for one launch");
    return PGB_ERR_UNSUPPORTED;
  }
  const bool i8 = c.dtype == PGB_I8;
#define PGB_ROWS(H, D, Q) return launch<H, D, Q>(a, c, p, splits, tiles_per_token, by_slot, units, stream)
  if (half) {
    if (c.head_dim == 64) { if (i8) PGB_ROWS(true, 64, true); PGB_ROWS(true, 64, false); }
    if (i8) PGB_ROWS(true, 128, true);
    PGB_ROWS(true, 128, false);
  }
  if (c.head_dim == 64) { if (i8) PGB_ROWS(false, 64, true); PGB_ROWS(false, 64, false); }
  if (i8) PGB_ROWS(false, 128, true);
  PGB_ROWS(false, 128, false);
#undef PGB_ROWS
}

}  // namespace pgb
