// Warp-level matrix and conversion wrappers (mma.sync, ldmatrix, movmatrix, ex2)
// of the paged KV-cache kernels.
#pragma once

#include <stdint.h>

#include <type_traits>

#include "common.cuh"

namespace dli_sm100 {

// D[16x8] += A[16x16] B[16x8], 16-bit operands, fp32 accumulators.
template <typename T>
__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                          uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  } else {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
}
// D[16x8] += A[16x8] B[8x8], operands fp32 bits of which the MMA reads the top 19 (TF32).
__device__ __forceinline__ void mma_1688_tf32(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                              uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// x = hi + lo: hi rounded to nearest (ties away) at TF32's 11 significant bits, lo the
// rest of at most 12, whose last the MMA cuts off (2^-23 of x at most). No bits of lo are
// touched: it carries a NaN, and one of all ones (the GPU's own) plus a rounding unit
// would be -0. An infinity, and a value that rounds up to one, becomes a NaN, as the row
// of q or P would that has it; CACHED values keep hi at the largest TF32 number, and lo
// is the rest, an infinity included (an infinite k may count for nothing, an infinite v
// is an infinity): two more instructions of five.
template <bool CACHED = false>
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
  if constexpr (CACHED) {
    constexpr float kMost = 0x1.ffcp127f;
    hi = ((__float_as_uint(fminf(fabsf(x), kMost)) + 0x1000u) & 0x7FFFE000u) | (__float_as_uint(x) & 0x80000000u);
  } else {
    hi = (__float_as_uint(x) + 0x1000u) & 0xFFFFE000u;
  }
  lo = __float_as_uint(x - __uint_as_float(hi));
}
// A B to fp32's accuracy as three TF32 products, lo * lo (2^-22 of it at most) left out. The
// MMA cuts its sums off instead of rounding them, so the caller keeps its chains
// short: the leading product goes to `main`, the small ones to `low`.
__device__ __forceinline__ void mma_1688_f32(float (&main)[4], float (&low)[4], const uint32_t (&ah)[4],
                                             const uint32_t (&al)[4], float b0, float b1) {
  uint32_t h0, l0, h1, l1;
  split_tf32(b0, h0, l0);
  split_tf32(b1, h1, l1);
  mma_1688_tf32(low, al[0], al[1], al[2], al[3], h0, h1);
  mma_1688_tf32(low, ah[0], ah[1], ah[2], ah[3], l0, l1);
  mma_1688_tf32(main, ah[0], ah[1], ah[2], ah[3], h0, h1);
}
__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
// Transposes an 8x8 matrix of 16-bit values held one row pair per lane.
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
template <typename T>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  } else {
    __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  }
}
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// cap tanh(x / cap), times log2(e), from z = 2 log2(e) x / cap; cap2 = 2 cap log2(e).
// tanh = 1 - 2 / (1 + 2^z) is off by some 2^-22 of the cap, which would drown scores far
// below it: those (|z| < 1) take tanh's series, y - y^3/3 + 2y^5/15 - 17y^7/315 +
// 62y^9/2835 with y = z ln(2) / 2, whose next term is below 2^-22 of the sum.
constexpr float kHalfLn2 = 0.34657359f, kHalfLn2Sq = kHalfLn2 * kHalfLn2;
constexpr float kTanh0 = 0.5f * kHalfLn2, kTanh1 = -kHalfLn2Sq / 3.f, kTanh2 = kHalfLn2Sq * kHalfLn2Sq * (2.f / 15.f),
                kTanh3 = -kHalfLn2Sq * kHalfLn2Sq * kHalfLn2Sq * (17.f / 315.f),
                kTanh4 = kHalfLn2Sq * kHalfLn2Sq * kHalfLn2Sq * kHalfLn2Sq * (62.f / 2835.f);
__device__ __forceinline__ float capped_score(float z, float cap2) {
  const float s = z * z;
  float t = fmaf(s, kTanh4, kTanh3);
  t = fmaf(s, t, kTanh2);
  t = fmaf(s, t, kTanh1);
  t = fmaf(s, t, 1.f) * (z * (kTanh0 * cap2));
  const float e = fmaf(-cap2, rcp_approx(1.f + exp2_approx(z)), 0.5f * cap2);
  return fabsf(z) < 1.f ? t : e;
}
// Byte I of `w` (two E2M1 codes) as two halves, the low code in the low half.
template <int I>
__device__ __forceinline__ uint32_t e2m1x2_to_half2(uint32_t w) {
  uint32_t r;
  if constexpr (I == 0)
    asm("{.reg .b8 a,b,c,d; mov.b32 {a,b,c,d}, %1; cvt.rn.f16x2.e2m1x2 %0, a;}" : "=r"(r) : "r"(w));
  else if constexpr (I == 1)
    asm("{.reg .b8 a,b,c,d; mov.b32 {a,b,c,d}, %1; cvt.rn.f16x2.e2m1x2 %0, b;}" : "=r"(r) : "r"(w));
  else if constexpr (I == 2)
    asm("{.reg .b8 a,b,c,d; mov.b32 {a,b,c,d}, %1; cvt.rn.f16x2.e2m1x2 %0, c;}" : "=r"(r) : "r"(w));
  else
    asm("{.reg .b8 a,b,c,d; mov.b32 {a,b,c,d}, %1; cvt.rn.f16x2.e2m1x2 %0, d;}" : "=r"(r) : "r"(w));
  return r;
}
// Two E4M3 bytes (low 16 bits of `w`) as two halves.
__device__ __forceinline__ uint32_t e4m3x2_to_half2(uint32_t w) {
  uint32_t r;
  asm("{.reg .b16 a; cvt.u16.u32 a, %1; cvt.rn.f16x2.e4m3x2 %0, a;}" : "=r"(r) : "r"(w));
  return r;
}
__device__ __forceinline__ uint32_t mul_half2(uint32_t a, uint32_t b) {
  __half2 r = __hmul2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<uint32_t*>(&r);
}

}  // namespace dli_sm100
