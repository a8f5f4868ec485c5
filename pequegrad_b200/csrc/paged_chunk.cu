// Attention over the paged cache for chunks of new tokens, on the 5th-generation tensor cores.
//
// Work item = (key head, 256 packed rows): the rows of a sequence are its new tokens times the query heads that share the
// key head (token t, head g is row t * group + g), so grouped heads fill the tiles whatever their number. The two halves of
// 128 rows, A and B, meet every block of 128 keys together: a block is fetched, and for an int8 cache widened, once for
// both. One CTA per SM walks its share of the items; where there are fewer items than SMs, a cluster of CTAs splits the
// keys of one item and joins the partial results in distributed shared memory.
//   warps 0-3, 4-7  softmax of A and of B: thread = row. Scores from tensor memory into registers, mask, running maximum,
//                   exponentials, row sum, probabilities as 16-bit pairs back into tensor memory. O is rescaled there only when
//                   a row's maximum outgrew its reference by 2^8.
//   warps 8-11      keys and values. 16 bits: one warp issues a TMA box per page (an index that is no page reads as zeros).
//                   int8: each warp brings 32 keys a block into a raw ring with cp.async, widens them exactly to 16 bits and
//                   stores them as the tiles TMA would have written; scales go to the softmax warps through a small ring.
//   warps 12, 13    issue the MMAs of A and of B (one lane each), so that neither half waits for the other's softmax
//   warp 14         Q: where the group divides 128, by TMA (a box of group heads x 128 / group tokens is a half); otherwise by
//                   cp.async into the swizzled tiles (warps 9-11 help where keys come by TMA)
//   warp 15         finds the items, some ahead of their use: the search's loads and divisions stay out of the other roles' way
//                   and its code is there once
// Tensor memory: S_A [0, 128), S_B [128, 256), O_A, O_B behind them. With head dim 64 there is room for P beside S, and the
// scores of the next block are computed under the softmax of this one; with 128 P takes the place of S, and the two halves
// keep the tensor pipe and the exponentials busy in turn.
// int8 scales: the key's multiplies its scores, the value's its probabilities, both in fp32. In fp16 the products' range is
// kept by a reference of the exponents that counts the value scale's power of two, row by row; O / l is what it was.
// Masked places: a score that is left out is -inf by selection, its probability zero. Value rows behind the context are
// zeroed in shared memory, and values of new tokens that some rows must not see are cleared of NaN and infinities there;
// the rows that do see such a token get them back in the epilogue.
// Every wait is bounded; one that runs out sets the device error word and the CTA drains.
//
// Bound by the latency of a softmax warp's chain (two warps a scheduler) more than by either pipe. A step of 256 rows and 128
// keys takes 2.0 us with head dim 64 (610 TFLOP/s over the GPU, the tensor pipe at a fifth of its cycles in a profile),
// 3.2 us with 128 (780 TFLOP/s; S waits for the product that reads P), 3.5 and 5 us beside an int8 cache, whose scales are
// read twice a score, and for fp16 their exponents once (2 of 51 us for 10 steps). A launch and its first item cost 10 us before
// and behind the steps, each further item 4.
// Tried and slower: 128 scores held in registers (spills, 4.7 us a step with head dim 64, and the code leaves the instruction
// cache); one MMA warp for both halves; every role searching its items itself (74 against 50 us for 8 x 1024 tokens); giving S
// up with half of its exponentials to go instead of a quarter (no gain in 16 bits, 52 against 49 us beside an int8 cache).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <string>
#include <type_traits>

#include "paged.cuh"

namespace pgb {

constexpr int kChunkRows = 256;     // of an item
constexpr int kChunkThreads = 512;
constexpr uint32_t kChunkPolls = 1u << 20;  // eight seconds, when nothing comes
constexpr float kChunkLazy = 8.0f;  // log2 of the largest probability before a row's reference moves
// log2 of the smallest value scale that has a say in fp16 outputs: 127 times less is nothing there. With it zero scales have an
// exponent, and a row's sum stays within fp32.
constexpr float kChunkNothing = -40.0f;
constexpr int kScaleSlots = 4;
constexpr int kItemSlots = 4;  // items found ahead
constexpr int kItemReaders = 15;  // warps that read them: all but the one that finds them

template <int D, bool I8>
struct ChunkTile {
  static constexpr bool kAhead = D == 64;  // P beside S: the next scores are computed ahead
  static constexpr int kQ = kChunkRows * D * 2, kKV = 128 * D * 2, kRaw = 128 * D * 2;  // raw: K and V of a block, int8
  static constexpr int kStages = I8 ? (D == 64 ? 2 : 1) : (D == 64 ? 3 : 2);
  static constexpr int kRawStages = I8 ? (D == 64 ? 3 : 2) : 0;
  static constexpr int kRing = 2 * kStages * kKV + kRawStages * kRaw;
  static constexpr int kScales = I8 ? kScaleSlots * 3 * 128 * 4 : 0;
  static constexpr int kMl = 3 * kChunkRows * 4;  // m and l of the rows, weights of the parts
  static constexpr int kSmem = kQ + kRing + kScales + kMl + kItemSlots * 64 + 512 /*barriers*/ + 1024 /*alignment*/;
  static_assert(kRing >= kChunkRows * D * 4, "the partial results of a split item take the place of the rings");
  static_assert(kSmem <= 232448, "shared memory of one SM");
};

struct ChunkParams {
  PagedParams a;
  KvCache c;
  KvPlan p;
  int n_tiles;  // bound on the tiles of all sequences
  int splits;
  int *err;
  uint32_t polls;
  int skip_loads;
  int q_tma;  // Q has a tensor map
};

struct ChunkItem {
  int seq, head;
  int token, sub;        // of the first packed row: row of q, query head of the group
  int rows;              // packed rows of the item, at most 256
  int pos;               // position of that token
  int n_keys;            // keys that the item's last row sees
  int first_seen;        // last key that the item's first row sees
  int lo;                // first block of this CTA
  int steps, n_a, n_b;   // blocks of this CTA; those of half A and of half B

  __device__ __forceinline__ int blocks(int half) const { return half ? n_b : n_a; }
};

// x / group; without grouped heads there is nothing to divide
__device__ __forceinline__ int chunk_div(int x, int group) { return group == 1 ? x : (int)((unsigned)x / (unsigned)group); }

struct ChunkCursor {
  int hi = -1, lo = 0;  // tiles with keys in (lo, hi] are being dealt out; hi < 0: not begun
  int seq0 = 0, base = 0;
};

// Item `id` (tile id / heads, key head id % heads), found by a warp, sequences 32 at a time. The tiles are listed by the
// number of keys that their last row sees, in bands of an eighth, most first: heavy items that start first even out. Within
// a sequence that number grows with the tile, so how many of its tiles lie in a band takes no search. Items are asked for in
// ascending order, so the search resumes where it stopped. False past the last tile.
__device__ __forceinline__ bool chunk_item(const ChunkParams &P, int id, int rank, ChunkCursor &cur, ChunkItem &it) {
  constexpr int kAll = -2147483647 - 1;
  const int lane = threadIdx.x & 31;
  const int t = id / P.c.heads;
  it.head = id - t * P.c.heads;
  if (cur.hi < 0) {
    int most = 0;
    for (int s = lane; s < P.p.n_seq; s += 32) most = max(most, __ldg(P.p.ctx + s));
    most = __reduce_max_sync(0xffffffffu, most);
    cur.hi = 2147483647;
    cur.lo = most - (most >> 3);
  }
  for (;;) {
    if (cur.seq0 >= P.p.n_seq) {
      if (cur.lo == kAll) return false;
      cur.hi = cur.lo;
      cur.lo = cur.lo > 64 ? cur.lo - (cur.lo >> 3) : kAll;
      cur.seq0 = 0;
    }
    const int s = cur.seq0 + lane;
    int64_t start = 0, n = 0;
    int ctx = 0;
    if (s < P.p.n_seq) {
      start = __ldg(P.p.start + s);
      n = min((int64_t)__ldg(P.p.start + s + 1), P.a.rows) - start;
      ctx = __ldg(P.p.ctx + s);
      if (n < 0 || start < 0) n = 0;  // offsets that make no sense hold no rows
    }
    const int tiles = (int)((n * P.a.group + kChunkRows - 1) / kChunkRows);
    auto above = [&](int keys) -> int {  // tiles of this lane's sequence with more keys than that
      if (keys == kAll) return tiles;
      if (ctx <= keys) return 0;
      return tiles - (int)min((int64_t)max(0, tiles - 1), max((int64_t)0, (keys - (ctx - n)) * P.a.group / kChunkRows));
    };
    const int top = above(cur.hi), count = above(cur.lo) - top;
    int sum = count;
#pragma unroll
    for (int k = 1; k < 32; k <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, sum, k);
      if (lane >= k) sum += up;
    }
    const uint32_t hit = __ballot_sync(0xffffffffu, t < cur.base + sum);
    if (!hit) {
      cur.base += __shfl_sync(0xffffffffu, sum, 31);
      cur.seq0 += 32;
      continue;
    }
    const int src = __ffs(hit) - 1;
    const int tile = __shfl_sync(0xffffffffu, tiles - 1 - top - (t - cur.base - (sum - count)), src);
    n = __shfl_sync(0xffffffffu, n, src);
    it.seq = cur.seq0 + src;
    start = __shfl_sync(0xffffffffu, start, src);
    const int64_t row0 = (int64_t)tile * kChunkRows;
    const int64_t tok0 = row0 < 2147483647LL ? (int64_t)chunk_div((int)row0, P.a.group) : row0 / P.a.group;
    it.token = (int)(start + tok0);
    it.sub = (int)(row0 - tok0 * P.a.group);
    it.rows = (int)min((int64_t)kChunkRows, n * P.a.group - row0);
    const int held = P.p.width << P.c.log2_page;  // at most 2^30
    it.pos = (int)max(kv_position(P.p, it.seq, it.token), -((int64_t)1 << 31));
    auto keys = [&](int row) { return max(0, min(held, it.pos + chunk_div(it.sub + row, P.a.group) + 1)); };
    it.first_seen = keys(0) - 1;
    it.n_keys = keys(it.rows - 1);
    const int n_a = (keys(min(it.rows, 128) - 1) + 127) >> 7, n_all = (it.n_keys + 127) >> 7;
    it.lo = n_all * rank / P.splits;
    it.steps = n_all * (rank + 1) / P.splits - it.lo;
    it.n_a = max(0, min(it.steps, n_a - it.lo));
    it.n_b = it.rows > 128 ? it.steps : 0;
    return true;
  }
}

__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  uint64_t ua, ub, ud;
  memcpy(&ua, &a, 8); memcpy(&ub, &b, 8);
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(ud) : "l"(ua), "l"(ub));
  float2 d;
  memcpy(&d, &ud, 8);
  return d;
}
// maximum of three, NaN if one of them is
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float4 chunk_peer4(uint32_t addr, uint32_t rank) {
  uint32_t remote;
  float4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(remote) : "memory");
  return v;
}
// Waits for this thread's loads from tensor memory and ties their registers to the wait.
__device__ __forceinline__ void chunk_ld_wait(uint32_t (&v)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]), "+r"(v[10]),
                 "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]), "+r"(v[16]), "+r"(v[17]), "+r"(v[18]), "+r"(v[19]), "+r"(v[20]),
                 "+r"(v[21]), "+r"(v[22]), "+r"(v[23]), "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29]), "+r"(v[30]),
                 "+r"(v[31])::"memory");
}
// Bit 15 or 31 of the result is set where the low or high 16-bit float of w has an exponent of all ones: NaN or infinity.
template <bool HALF>
__device__ __forceinline__ uint32_t exponent_carry(uint32_t w) {
  return (w & (HALF ? 0x7c007c00u : 0x7f807f80u)) + (HALF ? 0x04000400u : 0x00800080u);
}
template <bool HALF>
__device__ __forceinline__ float half_of(uint32_t w, int hi) {
  const uint32_t u = hi ? w >> 16 : w & 0xffffu;
  if (HALF) return __half2float(__ushort_as_half((unsigned short)u));
  return __uint_as_float(u << 16);
}

template <bool HALF, int D, bool I8>
__global__ void __launch_bounds__(kChunkThreads, 1) paged_chunk_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                                                                       const __grid_constant__ ChunkParams P) {
  using S = ChunkTile<D, I8>;
  constexpr int kQWarps = I8 ? 1 : 4;  // 14 and, where keys come by TMA, 9-11
  constexpr bool kProducts = I8 && HALF;  // the exponents' reference counts value scales too
  // fp16 probabilities are held 2^7 times too large, at most 2^15 with the lag of the reference (products with value scales,
  // which may be twice as large, 2^6): what fp16 rounds coarsely or drops is that much smaller then. The sum has the factor too.
  constexpr float kUp = !HALF ? 0.f : kProducts ? 6.f : 7.f;
  constexpr int kKind = GEMM_F16;  // kind::f16 serves both 16-bit types; the descriptor tells them apart
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t *q_s = smem;                          // [half][d / 64][128 rows][128 bytes]
  uint8_t *k_s = q_s + S::kQ;                   // [stage][d / 64][128 keys][128 bytes]
  uint8_t *v_s = k_s + S::kStages * S::kKV;
  uint8_t *raw_s = v_s + S::kStages * S::kKV;   // [stage][K, V][128 keys][D bytes]
  float *scale_s = reinterpret_cast<float *>(raw_s + S::kRawStages * S::kRaw);  // [slot][128 of K, 128 of V, 128 exponents of V's]
  float *ml_s = scale_s + S::kScales / 4;       // [m, l][256], [part][rows that this CTA writes]
  int4 *item_s = reinterpret_cast<int4 *>(ml_s + 3 * kChunkRows);  // [slot][4]
  uint64_t *bars = reinterpret_cast<uint64_t *>(item_s + 4 * kItemSlots);
  uint64_t *q_full = bars, *q_empty = bars + 1;
  uint64_t *k_full = bars + 2, *k_empty = k_full + 4, *v_full = k_empty + 4, *v_empty = v_full + 4;  // [kStages]
  uint64_t *sc_full = v_empty + 4, *sc_empty = sc_full + kScaleSlots;
  uint64_t *s_full = sc_empty + kScaleSlots, *s_free = s_full + 2, *p_full = s_free + 2, *pv_done = p_full + 2;  // [half]
  uint64_t *item_full = pv_done + 2, *item_empty = item_full + kItemSlots, *drained = item_empty + kItemSlots;  // drained: [half]
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(drained + 2);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
  int *dead = const_cast<int *>(abort_flag) + 1;
  volatile int *poison = const_cast<volatile int *>(abort_flag) + 2;
  volatile uint32_t *moved = tmem_slot + 4;  // [half] steps whose products were issued

  // broadcast, so that the compiler knows it is the same for the warp: barrier addresses and descriptors stay uniform
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int rank = P.splits > 1 ? (int)(blockIdx.x % P.splits) : 0;
  const int n_items = P.n_tiles * P.c.heads;
  // Items are dealt out in rounds over the clusters (of one CTA, where keys are not split), in alternating direction.
  const int unit = (int)blockIdx.x / P.splits, units = (int)gridDim.x / P.splits;
  auto id_of = [&](int r) -> int { return r * units + ((r & 1) ? units - 1 - unit : unit); };

  if (threadIdx.x == 0) {
    mbar_init(q_full, P.q_tma ? 1 : kQWarps);
    mbar_init(q_empty, 2);
    for (int s = 0; s < S::kStages; ++s) {
      mbar_init(&k_full[s], I8 ? 4 : 1);
      mbar_init(&v_full[s], I8 ? 4 : 1);
      mbar_init(&k_empty[s], 2);  // the MMAs of A and of B
      mbar_init(&v_empty[s], 2);
    }
    for (int s = 0; s < kScaleSlots; ++s) {
      mbar_init(&sc_full[s], 4);
      mbar_init(&sc_empty[s], 8);
    }
    for (int s = 0; s < kItemSlots; ++s) {
      mbar_init(&item_full[s], 1);
      mbar_init(&item_empty[s], kItemReaders);
    }
    for (int h = 0; h < 2; ++h) {
      mbar_init(&s_full[h], 1);
      mbar_init(&s_free[h], 4);
      mbar_init(&p_full[h], 4);
      mbar_init(&pv_done[h], 1);
      mbar_init(&drained[h], 1);
    }
    *abort_flag = 0;
    *poison = 0;
    moved[0] = moved[1] = 0;
    *dead = *(volatile int *)P.err != 0;  // an earlier wait ran out and nobody has cleared the word: do nothing
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 12) tmem_alloc(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const bool run = *dead == 0;

  // last key that a row of the item sees
  auto last_seen = [&](const ChunkItem &it, int row) -> int {
    return min(it.pos + chunk_div(it.sub + min(row, it.rows - 1), P.a.group), (P.p.width << P.c.log2_page) - 1);
  };
  auto out_row = [&](const ChunkItem &it, int row) -> uint8_t * {
    const int pr = it.sub + row, tok = chunk_div(pr, P.a.group);
    return P.a.out + ((int64_t)it.token + tok) * P.a.o_row + ((int64_t)it.head * P.a.group + (pr - tok * P.a.group)) * P.a.o_head;
  };
  // 32 columns of a row of O from tensor memory, and, rarely, what was cleared from the values it sees given back.
  auto load_o = [&](const ChunkItem &it, uint32_t o_addr, int q, bool any, bool seen, bool slow, int lim, float (&o)[32]) {
    if (any) {
      uint32_t r[32];
      tmem_ld32_issue(o_addr + q * 32, r);
      chunk_ld_wait(r);
#pragma unroll
      for (int i = 0; i < 32; ++i) o[i] = seen ? __uint_as_float(r[i]) : 0.f;
    } else {
#pragma unroll
      for (int i = 0; i < 32; ++i) o[i] = 0.f;
    }
    if (slow) {
      const int end = min(min(lim + 1, it.n_keys), (it.lo + it.steps) << 7);
      for (int key = max(it.first_seen + 1, it.lo << 7); key < end; ++key) {
        const int page = kv_page(P.p, P.c, it.seq, key);
        if (page < 0) continue;
        const int sl = key & ((1 << P.c.log2_page) - 1);
        const uint32_t *v = reinterpret_cast<const uint32_t *>(P.c.v.base + page * P.c.v.page + it.head * P.c.v.head + sl * P.c.v.slot) + q * 16;
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const float x = half_of<HALF>(v[i >> 1], i & 1);
          if (!(fabsf(x) <= 3.4028234e38f)) o[i] += x;
        }
      }
    }
  };
  // Some wait for a whole item, which a context of 2^30 tokens makes seconds long. Each ends when a role that waits for one
  // step at a time gives up, or the role that finds the items sees nothing move, and raises the flag that every wait looks at.
  const uint32_t patient = P.polls < (1u << 20) ? P.polls : 1u << 31;
  // a wait of the whole warp; `role` goes into the error word
  auto wait = [&](uint64_t *bar, uint32_t parity, int role, uint32_t polls = 0) -> bool {
    const bool ok = __all_sync(0xffffffffu, attn_wait(bar, parity, abort_flag, polls ? polls : P.polls));
    if (!ok && lane == 0) {
      *abort_flag = 1;
      atomicCAS(P.err, 0, (role << 16) | (int)(blockIdx.x & 0xffff));
    }
    return ok;
  };
  // What a role keeps from round to round: its cursors and its counts of steps, products and items.
  ChunkCursor cur;
  ChunkItem it, s_it;
  uint32_t taken = 0, s_taken = 0;
  uint32_t g = 0, n = 0, s_g = 0, s_n = 0, s_items = 0;
  int s_j = 0;
  bool gone = false;  // after a wait that ran out, what was in flight has been seen out
  bool ok = run && !(P.skip_loads && (warp == 14 || (warp >= 8 && warp < 12)));

  // Alone, a CTA walks all its rounds with every role at its own pace. In a cluster the CTAs meet after each round and join.
  for (int pass = 0;; ++pass) {
  // The next item; false past the last. In a cluster a role does one item between two joins.
  auto read_item = [&](uint32_t &count, ChunkItem &to, bool release) -> bool {
    const uint32_t slot = count % kItemSlots;
    if (!wait(&item_full[slot], (count / kItemSlots) & 1, 46, patient)) { ok = false; return false; }
    const int4 a = item_s[4 * slot], b = item_s[4 * slot + 1], c = item_s[4 * slot + 2];
    if (release) {
      __syncwarp();
      if (lane == 0) mbar_arrive(&item_empty[slot]);
    }
    ++count;
    to.seq = a.x; to.head = a.y; to.token = a.z; to.sub = a.w;
    to.rows = b.x; to.pos = b.y; to.n_keys = b.z; to.first_seen = b.w;
    to.lo = c.x; to.steps = c.y; to.n_a = c.z; to.n_b = c.w;
    return to.seq >= 0;
  };
  bool first = true;
  auto take = [&]() -> bool {
    const bool more = ok && (P.splits == 1 || first) && read_item(taken, it, true);
    first = false;
    return more;
  };
  // ---- Q, by kQWarps warps in 16-byte pieces; rows that do not exist are zeros ----
  auto load_q = [&](int w) {
    constexpr int kUnits = D / 8, kRows = kQWarps * 32 / kUnits;  // pieces of a row; rows at once
    const int u = (w * 32 + lane) % kUnits, step_tok = chunk_div(kRows, P.a.group), step_head = kRows - step_tok * P.a.group;
    while (take()) {
      if (it.steps == 0 || (P.q_tma && w > 0)) continue;
      if (!(ok = wait(q_empty, (n & 1) ^ 1, 32, patient))) break;
      ++n;
      if (P.q_tma) {  // rows of other sequences behind the item's are loaded with it and not used; behind the last row, zeros
        if (lane == 0) {
          mbar_expect_tx(q_full, S::kQ);
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int d = 0; d < D / 64; ++d)
              tma_load_4d(q_s + h * (S::kQ / 2) + d * 16384, &map_q, 64 * d, it.head * P.a.group, it.token + h * chunk_div(128, P.a.group), 0, q_full);
        }
        __syncwarp();
        continue;
      }
      int row = (w * 32 + lane) / kUnits;
      int tok = chunk_div(it.sub + row, P.a.group), head = it.sub + row - tok * P.a.group;
      for (; row < kChunkRows; row += kRows) {
        const bool in = row < it.rows;
        const uint8_t *src = P.a.q + ((int64_t)it.token + (in ? tok : 0)) * P.a.q_row + ((int64_t)it.head * P.a.group + (in ? head : 0)) * P.a.q_head + u * 16;
        const uint32_t dst = smem_u32(q_s) + (row >> 7) * (S::kQ / 2) + (u >> 3) * 16384 + (row & 127) * 128 + (((u & 7) ^ (row & 7)) << 4);
        paged_copy16(dst, src, in);
        tok += step_tok;
        head += step_head;
        if (head >= P.a.group) { head -= P.a.group; ++tok; }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
    }
  };
  if (!run) {
  } else if (warp >= 12) {
    if (warp == 15) {
      // Waits until every reader has given a slot up. While it waits here, other roles may be waiting for items or whole items
      // of Q: it ends that wait, for all of them, when no product was issued during a full count of polls.
      auto given_up = [&](uint32_t slot, uint32_t parity) -> bool {
        for (uint32_t seen = ~0u;;) {
          const uint32_t now = __shfl_sync(0xffffffffu, moved[0] + moved[1], 0);
          if (now == seen) return wait(&item_empty[slot], parity, 47, 1);
          seen = now;
          if (__all_sync(0xffffffffu, attn_wait(&item_empty[slot], parity, abort_flag, P.polls))) return true;
        }
      };
      for (bool more = true; more && ok; ++taken) {
        const int id = id_of((int)taken);
        more = id < n_items && chunk_item(P, id, rank, cur, it);
        const uint32_t slot = taken % kItemSlots, parity = (taken / kItemSlots) & 1;
        if (!(ok = given_up(slot, parity ^ 1))) break;
        if (lane == 0) {
          item_s[4 * slot] = make_int4(more ? it.seq : -1, it.head, it.token, it.sub);
          item_s[4 * slot + 1] = make_int4(it.rows, it.pos, it.n_keys, it.first_seen);
          item_s[4 * slot + 2] = make_int4(it.lo, it.steps, it.n_a, it.n_b);
          mbar_arrive(&item_full[slot]);
        }
        __syncwarp();
        if (!more || P.splits > 1) ok = given_up(slot, parity);  // the last of all items, or of this pass: nobody waits for one after it
        if (P.splits > 1) {  // one between two joins
          ++taken;
          break;
        }
      }
    } else if (warp == 14) {
      load_q(0);
    } else {
    // ---- MMA of one half ----------------------------------------------------------------------------------------------
    // A half that has nothing in a step still waits for the step's operands before it gives them up: its arrivals must not
    // run ahead of the other half's.
    const int h = warp - 12;
    const uint32_t idesc_s = attn_idesc(HALF, false, 128), idesc_pv = attn_idesc(HALF, true, D);
    const uint32_t t_s = tmem + h * 128, t_p = S::kAhead ? tmem + 384 + h * 64 : t_s, t_o = tmem + 256 + h * D;
    // descriptors of the first tile of each operand; the others differ in the address field alone, by constants
    const uint64_t d_q = make_kmajor_sw128_desc(smem_u32(q_s) + h * (S::kQ / 2)), d_k = make_kmajor_sw128_desc(smem_u32(k_s));
    const uint64_t d_v = make_mnmajor_sw128_desc(smem_u32(v_s), 16384);
    // The cursor of the scores reads items without giving up their slots, which `take` does. So it never looks past the item
    // behind the last one taken: an item without blocks stops it until `take` has passed that. (Looking for the next item with
    // blocks through any number of others, it would wait for a slot that this warp holds.) And it reads every item before
    // `take` does, while the slot is the item's.
    bool s_more = false, s_first = true;
    auto s_seek = [&]() -> bool {
      while (ok && !s_more && s_taken <= taken && (P.splits == 1 || s_first)) {
        s_first = false;
        s_more = read_item(s_taken, s_it, false) && s_it.steps > 0;
      }
      return s_more;
    };
    // scores of the step at the S cursor
    auto issue_s = [&]() -> bool {
      if (s_j == 0 && !wait(q_full, s_items & 1, 34)) return false;
      const uint32_t ks = s_g % S::kStages;
      if (!wait(&k_full[ks], (s_g / S::kStages) & 1, 35)) return false;
      const bool active = s_j < s_it.blocks(h), last = s_j + 1 == s_it.steps;
      if (active) {
        if (S::kAhead) {
          if (!wait(&s_free[h], (s_n & 1) ^ 1, 36)) return false;
        } else if (n > 0 && !wait(&pv_done[h], (n - 1) & 1, 39)) {  // P lies where these scores go
          return false;
        }
        tc_fence_after();
      }
      if (lane == 0) {
        if (active) {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint32_t off = (kk >> 2) * (16384 >> 4) + 2 * (kk & 3);
            tc_mma<kKind>(t_s, d_q + off, d_k + ks * (S::kKV >> 4) + off, idesc_s, kk != 0);
          }
          tc_commit(&s_full[h]);
          tc_commit(&k_empty[ks]);
          if (last) tc_commit(q_empty);
        } else {
          mbar_arrive(&k_empty[ks]);
          if (last) tc_commit(q_empty);  // behind this half's earlier products
        }
      }
      __syncwarp();
      s_n += active;
      ++s_g;
      if (++s_j == s_it.steps) {
        ++s_items;
        s_j = 0;
        s_more = false;
      }
      return true;
    };
    // Scores of the steps before `limit`. Those of step g have to be under way before its product; where P lies beside S those
    // of step g + 1 too, otherwise these follow the product, which reads P where they go.
    auto scores_to = [&](uint32_t limit) {
      while (ok && s_g < limit && s_seek()) ok = issue_s();
    };
    for (s_seek(); take(); s_seek()) {
      for (int j = 0; j < it.steps && ok; ++j, ++g) {
        scores_to(g + (S::kAhead ? 2 : 1));
        if (!ok) break;
        const uint32_t vs = g % S::kStages, ph = (g / S::kStages) & 1;
        const bool active = j < it.blocks(h);
        if (active && !(ok = wait(&p_full[h], n & 1, 37))) break;
        if (!(ok = wait(&v_full[vs], ph, 38))) break;
        tc_fence_after();
        if (lane == 0) {
          if (active) {
#pragma unroll
            for (int kk = 0; kk < 8; ++kk)  // 16 keys per MMA: 8 columns of P, 16 rows of V
              tc_mma_ts(t_o, t_p + kk * 8, d_v + vs * (S::kKV >> 4) + kk * (2048 >> 4), idesc_pv, (j | kk) != 0);
            tc_commit(&pv_done[h]);
            tc_commit(&v_empty[vs]);
          } else {
            mbar_arrive(&v_empty[vs]);
          }
          moved[h] = g;
        }
        __syncwarp();
        n += active;
        if (!S::kAhead) scores_to(g + 2);
      }
    }
    }
  } else if (warp >= 8) {
    // ---- keys and values --------------------------------------------------------------------------------------------
    if constexpr (!I8) {
      if (warp == 8) {
        const int per = 128 >> P.c.log2_page;  // pages of a block, a lane each
        while (take()) {
          auto page_of = [&](int j) -> int {
            const int pos = ((it.lo + j) << 7) + (lane << P.c.log2_page);
            const int page = lane < per && pos < it.n_keys ? kv_page(P.p, P.c, it.seq, pos) : -1;
            return page < 0 ? P.c.n_pages : page;  // out of the tensor's range: zeros
          };
          int page = it.steps > 0 ? page_of(0) : 0;
          for (int j = 0; j < it.steps && ok; ++j, ++g) {
            const int next = j + 1 < it.steps ? page_of(j + 1) : 0;
            const uint32_t st = g % S::kStages, ph = ((g / S::kStages) & 1) ^ 1;
            const int box = 128 << P.c.log2_page;  // bytes of a page's 64 columns
            for (int kv = 0; kv < 2 && ok; ++kv) {
              uint64_t *full = kv ? &v_full[st] : &k_full[st];
              ok = wait(kv ? &v_empty[st] : &k_empty[st], ph, 33);
              if (!ok) break;
              if (lane == 0) mbar_expect_tx(full, S::kKV);
              __syncwarp();
              if (lane < per) {
                uint8_t *dst = (kv ? v_s : k_s) + st * S::kKV + lane * box;
#pragma unroll
                for (int d = 0; d < D / 64; ++d) tma_load_4d(dst + d * 16384, kv ? &map_v : &map_k, 64 * d, 0, it.head, page, full);
              }
              __syncwarp();
              if (kv) n = g + 1;
              else s_n = g + 1;  // blocks of V and of K that were asked for
            }
            page = next;
          }
        }
      } else {
        load_q(warp - 8);  // 1 to 3: an int8 cache needs these warps for its keys
      }
    } else {
      constexpr int kChunks = D / 16;         // 16-byte pieces of a key
      constexpr int kKeys = 32 / kChunks;     // keys that the warp's lanes reach at once
      const int w = warp - 8, key = w * 32 + lane;
      const uint32_t raw = smem_u32(raw_s) + w * 32 * D;
      while (take()) {
        // this lane's key of step j: its page, or -1
        auto page_of = [&](int j) -> int {
          const int pos = ((it.lo + j) << 7) + key;
          return j < it.steps && pos < it.n_keys ? kv_page(P.p, P.c, it.seq, pos) : -1;
        };
        auto fetch = [&](int j, int page, uint32_t stage, float &ks, float &vs) {
          ks = vs = 0.f;
          if (j < it.steps) {
            const int slot = (((it.lo + j) << 7) + key) & ((1 << P.c.log2_page) - 1);
            if (page >= 0) {
              ks = __ldg(P.c.k.scale + page * P.c.k.scale_page + it.head * P.c.k.scale_head + slot);
              vs = __ldg(P.c.v.scale + page * P.c.v.scale_page + it.head * P.c.v.scale_head + slot);
            }
            const uint32_t dst = raw + stage * S::kRaw;
#pragma unroll
            for (int i = 0; i < kChunks; ++i) {
              const int kk = i * kKeys + lane / kChunks, part = lane % kChunks;
              const int pg = __shfl_sync(0xffffffffu, page, kk), sl = __shfl_sync(0xffffffffu, slot, kk);
              const bool there = pg >= 0;
              const int64_t at = there ? pg : 0;
              paged_copy16(dst + kk * D + part * 16, P.c.k.base + at * P.c.k.page + it.head * P.c.k.head + sl * P.c.k.slot + part * 16, there);
              paged_copy16(dst + 128 * D + kk * D + part * 16, P.c.v.base + at * P.c.v.page + it.head * P.c.v.head + sl * P.c.v.slot + part * 16, there);
            }
          }
          asm volatile("cp.async.commit_group;" ::: "memory");
        };
        // widens the warp's 32 keys of a raw tile into the swizzled 16-bit tile
        auto widen = [&](uint32_t src, uint32_t dst) {
#pragma unroll
          for (int i = 0; i < kChunks; ++i) {
            const int kk = i * kKeys + lane / kChunks, part = lane % kChunks, row = w * 32 + kk;
            uint32_t x[4], y[8];
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(src + kk * D + part * 16) : "memory");
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              y[2 * e] = paged_widen2<HALF>(x[e], 0);
              y[2 * e + 1] = paged_widen2<HALF>(x[e], 1);
            }
            const uint32_t base = dst + (part >> 2) * 16384 + row * 128, u = 2 * (part & 3);
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(base + ((u ^ (row & 7)) << 4)), "r"(y[0]), "r"(y[1]), "r"(y[2]), "r"(y[3]) : "memory");
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(base + (((u + 1) ^ (row & 7)) << 4)), "r"(y[4]), "r"(y[5]), "r"(y[6]), "r"(y[7]) : "memory");
          }
        };
        constexpr int kDeep = S::kRawStages;
        float ks[kDeep], vs[kDeep];  // of the steps under way, the current one first
#pragma unroll
        for (int i = 0; i < kDeep - 1; ++i) fetch(i, page_of(i), (g + i) % kDeep, ks[i], vs[i]);
        int page = page_of(kDeep - 1);
        for (int j = 0; j < it.steps && ok; ++j, ++g) {
          fetch(j + kDeep - 1, page, (g + kDeep - 1) % kDeep, ks[kDeep - 1], vs[kDeep - 1]);
          page = page_of(j + kDeep);
          asm volatile("cp.async.wait_group %0;" ::"n"(kDeep - 1) : "memory");
          __syncwarp();
          const uint32_t src = raw + (g % kDeep) * S::kRaw;
          const uint32_t st = g % S::kStages, ph = ((g / S::kStages) & 1) ^ 1, slot = g % kScaleSlots;
          if (!(ok = wait(&k_empty[st], ph, 33))) break;
          widen(src, smem_u32(k_s) + st * S::kKV);
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) mbar_arrive(&k_full[st]);
          if (!(ok = wait(&sc_empty[slot], ((g / kScaleSlots) & 1) ^ 1, 40))) break;
          float *sc = scale_s + slot * (3 * 128);
          sc[key] = ks[0];
          sc[128 + key] = vs[0];
          const int e = (int)((__float_as_uint(vs[0]) >> 23) & 255);
          sc[256 + key] = e == 255 ? kChunkNothing : fmaxf((float)(e - 127), kChunkNothing);
          __syncwarp();
          if (lane == 0) mbar_arrive(&sc_full[slot]);
          if (!(ok = wait(&v_empty[st], ph, 33))) break;
          widen(src + 128 * D, smem_u32(v_s) + st * S::kKV);
          fence_proxy_async();
          __syncwarp();  // every lane has read its raw bytes: the next fetch may overwrite them
          if (lane == 0) mbar_arrive(&v_full[st]);
#pragma unroll
          for (int i = 0; i + 1 < kDeep; ++i) { ks[i] = ks[i + 1]; vs[i] = vs[i + 1]; }
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncwarp();
      }
    }
  } else {
    // ---- softmax ------------------------------------------------------------------------------------------------------
    const int h = warp >> 2, tid = threadIdx.x & 127, row = h * 128 + tid;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_addr = tmem + lanes + h * 128, o_addr = tmem + lanes + 256 + h * D;
    const uint32_t p_addr = tmem + lanes + (S::kAhead ? 384 + h * 64 : h * 128);
    const float c = P.a.c;
    const float2 c2 = make_float2(c, c);
    while (take()) {
      // last key that this row sees, and the warp's first row; rows that do not exist see what the last one does
      const int lim = last_seen(it, row);
      const int warp_lim = __shfl_sync(0xffffffffu, lim, 0);
      // Reference of the exponents, times c where it is a score, and the sum of their powers.
      float m = -INFINITY, l = 0.f;
      uint32_t met = 0;  // not zero: the row has a key
      auto page_of = [&](int j) -> int {  // of this lane's sixteen keys of step j; looked up a step early, used when it is there
        const int i = (((it.lo + j) << 7) + 16 * (lane & 7)) >> P.c.log2_page;
        return j < it.steps && (i << P.c.log2_page) < it.n_keys ? __ldg(P.p.table + (int64_t)it.seq * P.p.pitch + i) : 0;
      };
      int page_next = page_of(0);
      for (int j = 0; j < it.steps; ++j, ++g) {
        const int page_now = page_next;
        page_next = page_of(j + 1);
        const uint32_t slot = g % kScaleSlots;
        if (j >= it.blocks(h)) {
          if (I8) {  // not before the slot is filled: a half that has nothing to do must not get ahead of the other
            if (ok) ok = wait(&sc_full[slot], (g / kScaleSlots) & 1, 42);
            if (ok && lane == 0) mbar_arrive(&sc_empty[slot]);
          }
          continue;
        }
        if (ok) ok = wait(&s_full[h], n & 1, 41);
        if (I8 && ok) ok = wait(&sc_full[slot], (g / kScaleSlots) & 1, 42);
        if (!ok) continue;
        tc_fence_after();
        // Two passes over the row of S, 32 columns at a time, the next 32 on their way: the maximum, then the probabilities.
        // Reading tensor memory twice is cheaper than holding 128 scores: the loop's code stays in the instruction cache
        // and its registers leave room.
        uint32_t x0[32], x1[32];
        tmem_ld32_issue(s_addr, x0);
        const uint32_t absent = __ballot_sync(0xffffffffu, (unsigned)page_now >= (unsigned)P.c.n_pages) & 0xffu;  // a bit for each 16 keys without a page
        const int key0 = (it.lo + j) << 7;
        const bool masked = key0 + 127 > warp_lim || absent != 0;  // warp-uniform
        const int last = lim - key0;                               // last of the 128 that the row sees
        const float *sc = scale_s + slot * (3 * 128);
        // The largest exponent. Beside an int8 cache the probabilities take their values' scales with them into 16 bits: with fp16 it
        // is then the largest of the products that counts, each score with its value scale's power of two. Whatever ratios the scales
        // have, and wherever the tokens are that a row does not see, the largest product is of order one.
        float mx = -INFINITY;
        // The first pass scales int8 scores by their keys and puts -inf where the row must not look; it writes what it changed
        // back, so that the second pass takes every score as it finds it.
        auto top = [&](uint32_t (&x)[32], int c) {
          if (I8) {
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              const float4 k4 = *reinterpret_cast<const float4 *>(sc + c + i);
              const float2 u = mul2(make_float2(__uint_as_float(x[i]), __uint_as_float(x[i + 1])), make_float2(k4.x, k4.y));
              const float2 v = mul2(make_float2(__uint_as_float(x[i + 2]), __uint_as_float(x[i + 3])), make_float2(k4.z, k4.w));
              x[i] = __float_as_uint(u.x); x[i + 1] = __float_as_uint(u.y); x[i + 2] = __float_as_uint(v.x); x[i + 3] = __float_as_uint(v.y);
            }
          }
          if (masked) {
            // a bit for each of the 32 columns: up to the row's last, without the sixteens that have no page
            const int more = last - c;
            uint32_t keep = more >= 31 ? 0xffffffffu : more < 0 ? 0u : (2u << more) - 1;
            if ((absent >> (c >> 4)) & 1) keep &= 0xffff0000u;
            if ((absent >> (c >> 4)) & 2) keep &= 0xffffu;
            met |= keep;
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (!((keep >> i) & 1)) x[i] = 0xff800000u;  // -inf
          }
          if (I8 || masked) tmem_st32(s_addr + c, x);
          float mq[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            float y[8];
#pragma unroll
            for (int i = 0; i < 8; i += 4) {
              float4 z = make_float4(__uint_as_float(x[8 * q + i]), __uint_as_float(x[8 * q + i + 1]), __uint_as_float(x[8 * q + i + 2]), __uint_as_float(x[8 * q + i + 3]));
              if (kProducts) {
                const float4 e4 = *reinterpret_cast<const float4 *>(sc + 256 + c + 8 * q + i);
                const float2 u = fma2(make_float2(z.x, z.y), c2, make_float2(e4.x, e4.y)), v = fma2(make_float2(z.z, z.w), c2, make_float2(e4.z, e4.w));
                z = make_float4(u.x, u.y, v.x, v.y);
              }
              y[i] = z.x; y[i + 1] = z.y; y[i + 2] = z.z; y[i + 3] = z.w;
            }
            mq[q] = max3_nan(y[0], y[1], y[2]);
            mq[q] = max3_nan(mq[q], y[3], y[4]);
            mq[q] = max3_nan(mq[q], y[5], y[6]);
            mq[q] = max3_nan(mq[q], mq[q], y[7]);
          }
          mx = max3_nan(mx, max3_nan(mq[0], mq[1], mq[2]), mq[3]);
        };
#pragma unroll 1
        for (int c = 0; c < 128; c += 64) {
          chunk_ld_wait(x0);
          tmem_ld32_issue(s_addr + c + 32, x1);
          top(x0, c);
          chunk_ld_wait(x1);
          if (c == 0) tmem_ld32_issue(s_addr + 64, x0);
          top(x1, c + 32);
        }
        if (I8 || masked) tmem_st_wait();
        tmem_ld32_issue(s_addr, x0);
        if (!masked) met = 1;
        // A score that is no number makes the row's sum none either, and so does +infinity, whose exponent is infinity less itself.
        // (Both would be lost in the polynomial of the exponentials.)
        if (!(mx < INFINITY)) l = __uint_as_float(0x7fc00000u);
        const float m_cand = fmaxf(m, mx);
        const float unit = kProducts ? 1.f : c;  // scores are kept as they are: with exponents the step takes 3 % longer
        const bool grow = (m_cand - m) * unit > kChunkLazy;  // -inf -> finite: true; -inf -> -inf is NaN: false
        const float m_new = grow ? m_cand : m;
        const float m_use = m_new == -INFINITY ? 0.f : m_new;
        const float alpha = grow ? ex2f((m - m_use) * unit) : 1.f;
        const float nmc = fmaf(-m_use, unit, kUp);
        const float2 nmc2 = make_float2(nmc, nmc);
        m = m_new;
        if (n > 0) {
          // the product before must have read P and updated O
          ok = wait(&pv_done[h], (n - 1) & 1, 43);
          if (!ok) continue;
          tc_fence_after();
          if (j > 0 && __any_sync(0xffffffffu, alpha != 1.0f)) {
#pragma unroll
            for (int q4 = 0; q4 < D / 16; ++q4) {
              uint32_t o[16];
              tmem_ld16_issue(o_addr + q4 * 16, o);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
              tmem_st16(o_addr + q4 * 16, o);
            }
            tmem_st_wait();
          }
        }
        float2 sq[4] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        auto exps = [&](uint32_t (&x)[32], int c) {
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            const float s[4] = {__uint_as_float(x[i]), __uint_as_float(x[i + 1]), __uint_as_float(x[i + 2]), __uint_as_float(x[i + 3])};
            const float2 e0 = fma2(make_float2(s[0], s[1]), c2, nmc2), e1 = fma2(make_float2(s[2], s[3]), c2, nmc2);
            float2 p0 = make_float2(ex2f(e0.x), ex2f(e0.y));
            // a quarter of the exponentials on the FMA pipe, as in attention_sm100.cu
            float2 p1 = (i & 4) ? ex2_fma2(e1) : make_float2(ex2f(e1.x), ex2f(e1.y));
            if ((i & 4) && masked) {  // whose smallest value is not zero
              p1.x = s[2] == -INFINITY ? 0.f : p1.x;
              p1.y = s[3] == -INFINITY ? 0.f : p1.y;
            }
            sq[(i >> 1) & 2] = add2(sq[(i >> 1) & 2], p0);
            sq[((i >> 1) & 2) + 1] = add2(sq[((i >> 1) & 2) + 1], p1);
            if (I8) {
              const float4 v4 = *reinterpret_cast<const float4 *>(sc + 128 + c + i);
              float2 t0 = mul2(p0, make_float2(v4.x, v4.y)), t1 = mul2(p1, make_float2(v4.z, v4.w));
              if (masked) {  // a token that is not seen may have a scale that is no number
                t0 = make_float2(p0.x == 0.f ? 0.f : t0.x, p0.y == 0.f ? 0.f : t0.y);
                t1 = make_float2(p1.x == 0.f ? 0.f : t1.x, p1.y == 0.f ? 0.f : t1.y);
              }
              p0 = t0;
              p1 = t1;
            }
            pk[i >> 1] = out_pair<HALF>(p0.x, p0.y);
            pk[(i >> 1) + 1] = out_pair<HALF>(p1.x, p1.y);
          }
          tmem_st16(p_addr + (c >> 1), pk);  // where P shares S's columns: those of scores already in registers
        };
#pragma unroll 1
        for (int c = 0; c < 128; c += 64) {
          chunk_ld_wait(x0);
          tmem_ld32_issue(s_addr + c + 32, x1);
          exps(x0, c);
          chunk_ld_wait(x1);
          if (c == 0) tmem_ld32_issue(s_addr + 64, x0);
          else if (S::kAhead) {  // every score is in registers
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&s_free[h]);
          }
          exps(x1, c + 32);
        }
        const float2 s01 = add2(sq[0], sq[1]), s23 = add2(sq[2], sq[3]);
        l = l * alpha + ((s01.x + s01.y) + (s23.x + s23.y));
        if (I8) {
          __syncwarp();
          if (lane == 0) mbar_arrive(&sc_empty[slot]);
        }
        if (!I8 && (key0 + 127 > it.first_seen)) {
          // This block's values: thread = key. What lies behind the context is zeroed, what only some rows see is made finite.
          const uint32_t st = g % S::kStages;
          ok = wait(&v_full[st], (g / S::kStages) & 1, 44);
          if (!ok) continue;
          const int key = key0 + tid;
          uint8_t *vrow = v_s + st * S::kKV + tid * 128;
          auto piece = [&](int u) { return reinterpret_cast<uint4 *>(vrow + (u >> 3) * 16384 + (u & 7) * 16); };  // in any order
          if (key >= it.n_keys) {
#pragma unroll
            for (int u = 0; u < D / 8; ++u) *piece(u) = make_uint4(0, 0, 0, 0);
          } else if (key > it.first_seen) {
            uint32_t hit = 0;
#pragma unroll
            for (int u = 0; u < D / 8; ++u) {
              const uint4 x = *piece(u);
              hit |= exponent_carry<HALF>(x.x) | exponent_carry<HALF>(x.y) | exponent_carry<HALF>(x.z) | exponent_carry<HALF>(x.w);
            }
            if (hit & 0x80008000u) {
              *poison = 1;
              __threadfence_block();
#pragma unroll 1
              for (int u = 0; u < D / 8; ++u) {
                uint4 x = *piece(u);
                uint32_t *x4 = reinterpret_cast<uint32_t *>(&x);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const uint32_t bad = exponent_carry<HALF>(x4[e]);
                  if (bad & 0x8000u) x4[e] &= 0xffff0000u;
                  if (bad & 0x80000000u) x4[e] &= 0xffffu;
                }
                *piece(u) = x;
              }
            }
          }
          __threadfence_block();
          fence_proxy_async();
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[h]);
        ++n;
      }
      // ---- the item's rows ----
      if (!ok) continue;
      const bool any = it.blocks(h) > 0;
      if (any) {
        ok = wait(&pv_done[h], (n - 1) & 1, 45);
        if (!ok) continue;
        tc_fence_after();
      }
      // No key, or none with a score above -infinity: then the softmax is that of nothing (zeros) or no number. A part of a split
      // item says which in its sum, and nobody reads its O. (A score that is NaN leaves l NaN.)
      const bool low = m == -INFINITY && l == l;
      if (P.splits > 1) {  // joined below
        ml_s[row] = low || m != -INFINITY ? (kProducts ? m : m * c) : 0.f;
        ml_s[kChunkRows + row] = low ? (met ? 1.f : 0.f) : l;
        continue;
      }
      const float inv = low ? (met ? __uint_as_float(0x7fc00000u) : 0.f) : 1.0f / l;
      const bool slow = !I8 && any && *poison != 0;
      uint8_t *out = out_row(it, row);
#pragma unroll 1
      for (int q = 0; q < D / 32; ++q) {
        float o[32];
        load_o(it, o_addr, q, any, !low, slow, lim, o);
        if (row < it.rows) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) w[k] = out_pair<HALF>(o[8 * i + 2 * k] * inv, o[8 * i + 2 * k + 1] * inv);
            *reinterpret_cast<uint4 *>(out + q * 64 + i * 16) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      }
      tc_fence_before();
    }
  }

  tc_fence_before();
  __syncthreads();
  if (run && *abort_flag != 0 && !gone) {
    // Some role gave up. Copies and products that are in flight are waited for, with a limit again: nothing may write the
    // memory of a CTA that has gone. The roles that did not give up have to stop too: in a cluster there are rounds to come, and
    // what they would start there nobody sees out.
    gone = true;
    ok = false;
    auto see_out = [&](uint64_t *bar, uint32_t parity) {
      for (uint32_t i = 0; i < kChunkPolls && !mbar_try_wait(bar, parity); ++i) {}
    };
    if (warp < 8) {
      tmem_ld_wait();
      tmem_st_wait();
    } else if (!I8 && warp == 8) {
      for (uint32_t st = 0; st < S::kStages; ++st) {
        if (s_n > st) see_out(&k_full[(s_n - 1 - st) % S::kStages], ((s_n - 1 - st) / S::kStages) & 1);
        if (n > st) see_out(&v_full[(n - 1 - st) % S::kStages], ((n - 1 - st) / S::kStages) & 1);
      }
    } else if (warp == 14 && P.q_tma) {
      if (n > 0) see_out(q_full, (n - 1) & 1);
    } else if (warp == 12 || warp == 13) {
      if (lane == 0) tc_commit(&drained[warp - 12]);
      __syncwarp();
      see_out(&drained[warp - 12], 0);
    }
    __syncthreads();
  }
  if (P.splits == 1) break;
  // The round's item once more, for the warps whose role did not read it. A CTA whose wait ran out writes nothing, but stays
  // for every barrier of its cluster, since the others read its shared memory.
  const bool good = run && *abort_flag == 0;
  {
    const int4 a = item_s[4 * (pass % kItemSlots)], b = item_s[4 * (pass % kItemSlots) + 1], c = item_s[4 * (pass % kItemSlots) + 2];
    it.seq = a.x; it.head = a.y; it.token = a.z; it.sub = a.w;
    it.rows = b.x; it.pos = b.y; it.n_keys = b.z; it.first_seen = b.w;
    it.lo = c.x; it.steps = c.y; it.n_a = c.z; it.n_b = c.w;
  }
  if (good ? it.seq < 0 : id_of(pass) >= n_items) break;

  // ---- join the CTAs of the cluster ---------------------------------------------------------------------------------------
  // Every role is done with the item, so the rings are free: they take the partial rows, by columns of four, so that
  // neighbouring rows fall into neighbouring banks.
  tc_fence_after();
  if (good && warp < 8) {
    const int row = threadIdx.x, h = warp >> 2;
    const bool any = it.blocks(h) > 0, seen = any && ml_s[row] != -INFINITY;
    const uint32_t o_addr = tmem + ((uint32_t)((warp & 3) * 32) << 16) + 256 + h * D;
    const int lim = last_seen(it, row);
    const bool slow = !I8 && any && *poison != 0;
#pragma unroll 1
    for (int q = 0; q < D / 32; ++q) {
      float o[32];
      load_o(it, o_addr, q, any, seen, slow, lim, o);
      float4 *st = reinterpret_cast<float4 *>(k_s) + q * 8 * kChunkRows + row;
#pragma unroll
      for (int i = 0; i < 8; ++i) st[i * kChunkRows] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
    }
  }
  tc_fence_before();
  paged_cluster_sync();
  // each CTA writes its share of the rows: first how much each part counts, then the weighted sums, eight values a thread
  auto join = [&](auto parts) {
    constexpr int N = decltype(parts)::value, kShare = kChunkRows / N, kParts = D / 8;
    float *weight = ml_s + 2 * kChunkRows;
    const int r0 = rank * kShare, n_rows = min(kShare, it.rows - r0);
    if (threadIdx.x < kChunkRows) {
      const int row = threadIdx.x % kShare, part = threadIdx.x / kShare;
      float pm[N], pl[N], mm = -INFINITY, sum = 0.f;
#pragma unroll
      for (int s = 0; s < N; ++s) {
        pm[s] = paged_peer(smem_u32(ml_s + r0 + row), s);
        pl[s] = paged_peer(smem_u32(ml_s + kChunkRows + r0 + row), s);
      }
#pragma unroll
      for (int s = 0; s < N; ++s) mm = fmaxf(mm, pm[s]);
      float mine = 0.f;
#pragma unroll
      for (int s = 0; s < N; ++s) {
        const float e = pm[s] == -INFINITY ? 0.f : ex2f(pm[s] - mm);
        sum += pl[s] * e;
        if (s == part) mine = e;
      }
      if (mm == -INFINITY) {  // no part has a score above that: zeros without a key, else no number
        float keys = 0.f;
#pragma unroll
        for (int s = 0; s < N; ++s) keys += pl[s];
        mine = keys > 0.f ? __uint_as_float(0x7fc00000u) : 0.f;
        sum = 1.f;
      }
      weight[part * kShare + row] = mine / sum;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n_rows * kParts; i += kChunkThreads) {
      const int row = i / kParts, part = i % kParts;
      const uint32_t at = smem_u32(k_s) + ((part * 2) * kChunkRows + r0 + row) * 16;
      float4 x[N], y[N];
#pragma unroll
      for (int s = 0; s < N; ++s) {
        x[s] = chunk_peer4(at, s);
        y[s] = chunk_peer4(at + kChunkRows * 16, s);
      }
      float o[8] = {};
#pragma unroll
      for (int s = 0; s < N; ++s) {
        const float e = weight[s * kShare + row];
        o[0] += x[s].x * e; o[1] += x[s].y * e; o[2] += x[s].z * e; o[3] += x[s].w * e;
        o[4] += y[s].x * e; o[5] += y[s].y * e; o[6] += y[s].z * e; o[7] += y[s].w * e;
      }
      *reinterpret_cast<uint4 *>(out_row(it, r0 + row) + part * 16) =
          make_uint4(out_pair<HALF>(o[0], o[1]), out_pair<HALF>(o[2], o[3]), out_pair<HALF>(o[4], o[5]), out_pair<HALF>(o[6], o[7]));
    }
  };
  if (good) {
    if (P.splits == 2) join(std::integral_constant<int, 2>{});
    else if (P.splits == 4) join(std::integral_constant<int, 4>{});
    else join(std::integral_constant<int, 8>{});
  }
  fence_proxy_async();   // TMA may write next where the partial rows lay
  paged_cluster_sync();  // nobody's shared memory changes or goes away while it is read
  }
  if (warp == 12) tmem_dealloc(tmem, 512);
}

template <bool HALF, int D, bool I8>
static int launch(ChunkParams &P, const CUtensorMap &mq, const CUtensorMap &mk, const CUtensorMap &mv, int64_t items, int64_t blocks, cudaStream_t stream) {
  using S = ChunkTile<D, I8>;
  const auto kernel = paged_chunk_kernel<HALF, D, I8>;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) {
    cudaGetLastError();
    set_error("paged_attention: cannot tell the current device");
    return PGB_ERR_CUDA;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kChunkThreads);
  cfg.dynamicSmemBytes = S::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  // Per device: the shared-memory limit is raised, and how many clusters of 2, 4 and 8 run at a time is asked for, once; again
  // where two threads meet. The processor clusters' SMs do not divide evenly: 148 SMs hold fewer than 148 / 4 clusters of
  // four, and one cluster too many would wait for a whole round of the others.
  static std::atomic<uint32_t> capacity[64];
  uint32_t cap = capacity[dev].load(std::memory_order_relaxed);
  if (cap == 0) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem);
    for (int k = 3; k >= 1 && e == cudaSuccess; --k) {
      int n = 0;
      attr[0].val.clusterDim.x = 1u << k;
      cfg.gridDim = dim3(1u << k);
      e = cudaOccupancyMaxActiveClusters(&n, kernel, &cfg);
      cap = cap << 8 | (uint32_t)std::min(n, 255);
    }
    if (e != cudaSuccess) {
      cudaGetLastError();
      set_error(std::string("paged_attention: cannot set up the kernel: ") + cudaGetErrorString(e));
      return PGB_ERR_CUDA;
    }
    cap |= 1u << 31;
    capacity[dev].store(cap, std::memory_order_relaxed);
  }
  // CTAs per item: what makes the launch shortest, in steps of a block of keys. Of s CTAs' share of the longest item and of
  // all items (which have, by and large, 0.6 of the longest's keys) over the clusters that run at once, the longer counts;
  // each round costs one and a half steps to fill and drain, and four where CTAs join (12 heads of 64, contexts of 5003 and
  // 3000 int8 tokens, 36 items: 74, 49 and 53 us with 2, 4 and 8 CTAs).
  P.splits = 1;
  int64_t units = sm_count();
  double best = 0;
  for (int k = 0; k <= 3; ++k) {
    const int64_t s = 1 << k, n = k == 0 ? sm_count() : (cap >> (8 * (k - 1))) & (k == 3 ? 127 : 255);
    if (n == 0 || (k > 0 && blocks < 2 * s)) continue;
    const double part = (double)blocks / s, rounds = std::max(1.0, (double)items / n);
    const double t = std::max(part, 0.6 * part * items / n) + rounds * (k ? 4.0 : 1.5);
    if (k == 0 || t < best) {
      best = t;
      P.splits = (int)s;
      units = n;
    }
  }
  cfg.gridDim = dim3((unsigned)(std::min(items, units) * P.splits));
  attr[0].val.clusterDim.x = P.splits;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, mq, mk, mv, P);
  if (e != cudaSuccess) {
    cudaGetLastError();
    set_error(std::string("paged_chunk_kernel: ") + cudaGetErrorString(e));
    return PGB_ERR_CUDA;
  }
  count_launch();
  return PGB_OK;
}

// The pages as a 4-D tensor map: boxes of one page and 64 columns. False where TMA cannot address them.
static bool page_map(CUtensorMap *m, const KvCache &c, const KvPages &p) {
  const uint64_t P = (uint64_t)1 << c.log2_page;
  const uint64_t dims[4] = {(uint64_t)c.head_dim, P, (uint64_t)c.heads, (uint64_t)c.n_pages};
  // a dim of extent 1 still needs a valid stride
  const uint64_t slot = (uint64_t)p.slot;
  const uint64_t head = c.heads > 1 ? (uint64_t)p.head : slot * P;
  const uint64_t page = c.n_pages > 1 ? (uint64_t)p.page : head * c.heads;
  const uint64_t strides[3] = {slot, head, page};
  const uint32_t box[4] = {64, (uint32_t)P, 1, 1};
  for (uint64_t s : strides)
    if (s == 0 || s >= (1ull << 40)) return false;
  return encode_map_4d(m, c.dtype == PGB_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, p.base, dims, strides, box);
}

// Q as [rows, heads, head dim] with a box of one half's rows: the heads of a group times 128 / group tokens. False where the
// group does not divide 128 or TMA cannot address Q: its rows are copied one by one then.
static bool query_map(CUtensorMap *m, const PagedParams &a, const KvCache &c, bool half) {
  if (128 % a.group) return false;
  const uint64_t dims[4] = {(uint64_t)c.head_dim, (uint64_t)a.heads, (uint64_t)a.rows, 1};
  // a dim of extent 1 still needs a valid stride
  const uint64_t head = a.heads > 1 ? (uint64_t)a.q_head : (uint64_t)c.head_dim * 2;
  const uint64_t row = a.rows > 1 ? (uint64_t)a.q_row : head * a.heads;
  const uint64_t strides[3] = {head, row, row};
  const uint32_t box[4] = {64, (uint32_t)a.group, (uint32_t)(128 / a.group), 1};
  for (uint64_t s : strides)
    if (s == 0 || s >= (1ull << 40)) return false;
  return encode_map_4d(m, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, a.q, dims, strides, box);
}

bool run_paged_chunk(const PagedParams &a, const KvCache &c, const KvPlan &p, bool half, cudaStream_t stream, int *status) {
  ChunkParams P{};
  P.a = a;
  P.c = c;
  P.p = p;
  // tiles of 256 rows: each sequence that has rows adds at most one that is not full
  const int64_t k = std::min<int64_t>(p.n_seq, a.rows), tiles = (a.rows * a.group - k) / kChunkRows + k;
  if (tiles * c.heads > 1073741824LL || c.n_pages == 0) return false;
  CUtensorMap mq{}, mk{}, mv{};
  if (c.dtype != PGB_I8 && (!page_map(&mk, c, c.k) || !page_map(&mv, c, c.v))) return false;
  P.q_tma = query_map(&mq, a, c, half) ? 1 : 0;
  P.n_tiles = (int)tiles;
  const int64_t items = tiles * c.heads, blocks = ((int64_t)p.width << c.log2_page) / 128;
  P.err = gemm_error_word();
  if (!P.err) {
    set_error("paged_attention: cannot resolve the device error word");
    *status = PGB_ERR_CUDA;
    return true;
  }
  uint32_t drill_polls = 0;
  take_next_wait_test(&drill_polls, &P.skip_loads);
  P.polls = drill_polls ? drill_polls : kChunkPolls;
  const bool i8 = c.dtype == PGB_I8;
#define PGB_CHUNK(H, D, Q) launch<H, D, Q>(P, mq, mk, mv, items, blocks, stream)
  if (half) {
    if (c.head_dim == 64) *status = i8 ? PGB_CHUNK(true, 64, true) : PGB_CHUNK(true, 64, false);
    else *status = i8 ? PGB_CHUNK(true, 128, true) : PGB_CHUNK(true, 128, false);
  } else {
    if (c.head_dim == 64) *status = i8 ? PGB_CHUNK(false, 64, true) : PGB_CHUNK(false, 64, false);
    else *status = i8 ? PGB_CHUNK(false, 128, true) : PGB_CHUNK(false, 128, false);
  }
#undef PGB_CHUNK
  return true;
}

}  // namespace pgb
