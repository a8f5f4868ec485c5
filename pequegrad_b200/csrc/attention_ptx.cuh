// Device helpers shared by the attention kernels (attention_sm100.cu, paged_chunk.cu): instruction descriptors, packed fp32
// arithmetic, exponentials, tensor-memory accesses, the bounded wait.
#pragma once
#include <cstring>

#include "gemm_ptx.cuh"

namespace pgb {

// f16 / bf16 instruction descriptor, M = 128, fp32 accumulate; bit 16 = B operand is MN-major
__device__ __forceinline__ uint32_t attn_idesc(bool is_half, bool b_mn_major, int n) {
  uint32_t d = 0;
  const uint32_t fmt = is_half ? 0u : 1u;
  d |= 1u << 4;
  d |= fmt << 7;
  d |= fmt << 10;
  if (b_mn_major) d |= 1u << 16;
  d |= (uint32_t)(n >> 3) << 17;
  d |= (uint32_t)(128 >> 4) << 24;
  return d;
}

__device__ __forceinline__ float ex2f(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  uint64_t ua, ub, uc, ud;
  memcpy(&ua, &a, 8); memcpy(&ub, &b, 8); memcpy(&uc, &c, 8);
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(ud) : "l"(ua), "l"(ub), "l"(uc));
  float2 d;
  memcpy(&d, &ud, 8);
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  uint64_t ua, ub, ud;
  memcpy(&ua, &a, 8); memcpy(&ub, &b, 8);
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(ud) : "l"(ua), "l"(ub));
  float2 d;
  memcpy(&d, &ud, 8);
  return d;
}
// D[tmem] (+)= A[tmem] * B[smem]: the A operand (M = 128 rows = lanes, 16-bit elements two per column) is read from
// tensor memory
__device__ __forceinline__ void tc_mma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
      "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// 2^x for a pair of exponent arguments on the FMA pipe instead of the SFU: n = round(x) taken from the low mantissa
// bits of x + 1.5 * 2^23, f = x - n in [-0.5, 0.5], a cubic for 2^f (relative error 7.5e-5, a sixth of the rounding
// of a 16-bit P), and n added into the exponent field. x below -126 is clamped (the result is then 2^-126, nothing in P).
__device__ __forceinline__ float2 ex2_fma2(float2 x) {
  const float kMagic = 12582912.f;
  x.x = fmaxf(x.x, -126.f);
  x.y = fmaxf(x.y, -126.f);
  const float2 r = add2(x, make_float2(kMagic, kMagic));
  const float2 n = add2(r, make_float2(-kMagic, -kMagic));
  const float2 f = add2(x, make_float2(-n.x, -n.y));
  float2 q = fma2(make_float2(0.05517144873738289f, 0.05517144873738289f), f, make_float2(0.2426108419895172f, 0.2426108419895172f));
  q = fma2(q, f, make_float2(0.6932609677314758f, 0.6932609677314758f));
  q = fma2(q, f, make_float2(0.9999281167984009f, 0.9999281167984009f));
  return make_float2(__uint_as_float(__float_as_uint(q.x) + (__float_as_uint(r.x) << 23)), __uint_as_float(__float_as_uint(q.y) + (__float_as_uint(r.y) << 23)));
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
template <bool HALF>
__device__ __forceinline__ uint32_t out_pair(float lo, float hi) {
  uint32_t r;
  if (HALF) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

__device__ __forceinline__ void tmem_ld16_issue(uint32_t taddr, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]),
        "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]),
      "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
// Bounded wait. try_wait lets the hardware park the thread for a short while instead of spinning through the issue
// slots that the softmax warps need. (A suspend-time hint of 2 us was measured and is slower.)
__device__ __forceinline__ bool attn_wait(uint64_t *bar, uint32_t parity, volatile int *abort_flag, uint32_t polls) {
  const uint32_t addr = smem_u32(bar);
  for (uint32_t i = 0; i < polls; ++i) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(addr), "r"(parity)
        : "memory");
    if (ok) return true;
    if ((i & 63) == 63 && *abort_flag) return false;
  }
  return false;
}

}  // namespace pgb
