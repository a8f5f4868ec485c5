// Shared by the two kernels of attention over the paged cache (paged_rows.cu, paged_chunk.cu) and their entry point
// (paged_attention.cu).
#pragma once
#include "attention_ptx.cuh"
#include "kv_cache.cuh"

namespace pgb {

struct PagedParams {
  const uint8_t *q;
  uint8_t *out;
  int64_t q_row, q_head, o_row, o_head;  // bytes
  int64_t rows;
  int heads, group;  // query heads; query heads per key head
  float c;           // scale * log2(e)
};

// Few rows per sequence: tiles of 16 rows, keys streamed once, split over a cluster. Right for any number of rows.
int run_paged_rows(const PagedParams &a, const KvCache &c, const KvPlan &p, bool half, cudaStream_t stream);
// Many rows per sequence: tiles of 256 rows on the tensor cores. False where the pages cannot be addressed by TMA, or there
// are none: nothing was launched. Right for any number of rows.
bool run_paged_chunk(const PagedParams &a, const KvCache &c, const KvPlan &p, bool half, cudaStream_t stream, int *status);

// 16 bytes into shared memory, zeros where there is nothing to copy
__device__ __forceinline__ void paged_copy16(uint32_t dst, const void *src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
// The same address in the shared memory of another CTA of the cluster
__device__ __forceinline__ float paged_peer(uint32_t addr, uint32_t rank) {
  uint32_t remote;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(remote) : "memory");
  return v;
}
__device__ __forceinline__ void paged_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Two of four int8 values (the low or the high pair of w) as exact 16-bit floats. fp16: the byte plus 128 is placed in the
// mantissa of 1024, and 1152 taken off. bf16: its low seven bits in the mantissa of 128, less 128 or, where the sign bit
// makes that 256, 256.
template <bool HALF>
__device__ __forceinline__ uint32_t paged_widen2(uint32_t w, int high) {
  uint32_t r;
  if (HALF) {
    const uint32_t u = __byte_perm(w ^ 0x80808080u, 0x64646464u, high ? 0x4342 : 0x4140);
    asm("sub.f16x2 %0, %1, %2;" : "=r"(r) : "r"(u), "r"(0x64806480u));
  } else {
    const uint32_t u = __byte_perm(w, 0u, high ? 0x4342 : 0x4140);
    const uint32_t a = (u & 0x007f007fu) | 0x43004300u, b = (u & 0x00800080u) | 0x43004300u;
    asm("sub.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  }
  return r;
}

}  // namespace pgb
