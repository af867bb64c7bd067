// Device helpers of the tcgen05 attention kernels (attention.cu, attn_varlen.cu); the packed arithmetic serves kv_cache.cu too.
#pragma once
#include "common.cuh"

namespace mb {
namespace attn {

// ---- packed f32x2 helpers (sm_100): two IEEE single-precision ops per instruction
MB_DEV uint64_t pk2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1,%2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
MB_DEV void up2(uint64_t v, float& a, float& b) { asm("mov.b64 {%0,%1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
MB_DEV uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
MB_DEV uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
MB_DEV uint64_t sub2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
MB_DEV float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// 2^x for a pair by a degree-3 polynomial (own minimax fit of 2^f on [-1/2, 1/2], max relative
// error 7.5e-5, far below the bf16 rounding P is stored with): x is clamped to >= -126 (masked
// keys give ~1e-38), rounded to n by the 1.5 * 2^23 trick, and 2^n enters the exponent field.
MB_DEV void exp2_poly3(uint64_t x2, float& e0, float& e1) {
  float a, b;
  up2(x2, a, b);
  a = fmaxf(a, -126.f);
  b = fmaxf(b, -126.f);
  const uint64_t xc = pk2(a, b);
  const uint64_t magic = pk2(12582912.f, 12582912.f);
  const uint64_t t2 = add2(xc, magic);
  const uint64_t f = sub2(xc, sub2(t2, magic));
  uint64_t p = fma2(pk2(0.05517132207751274f, 0.05517132207751274f), f, pk2(0.24261054396629333f, 0.24261054396629333f));
  p = fma2(p, f, pk2(0.6932609677314758f, 0.6932609677314758f));
  p = fma2(p, f, pk2(0.9999281167984009f, 0.9999281167984009f));
  float t0, t1, p0, p1;
  up2(t2, t0, t1);
  up2(p, p0, p1);
  e0 = __int_as_float(__float_as_int(p0) + (int)((uint32_t)__float_as_int(t0) << 23));
  e1 = __int_as_float(__float_as_int(p1) + (int)((uint32_t)__float_as_int(t1) << 23));
}

MB_DEV void tmem_st16a(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
          taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// Elected-lane forms for a converged warp (lane 0 issues): cheaper to issue than a lane-0 branch.
MB_DEV void umma_ss_elect(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p, e;\n .reg .b32 r;\n setp.ne.b32 p, %4, 0;\n elect.sync r|e, 0xffffffff;\n"
      " @e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
MB_DEV void umma_ts_elect(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p, e;\n .reg .b32 r;\n setp.ne.b32 p, %4, 0;\n elect.sync r|e, 0xffffffff;\n"
      " @e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Four products in a row under one election: depth steps of 16 that lie 32 bytes apart in both operands (64 elements of
// one 128-byte swizzle atom column, K-major).
MB_DEV void umma_ss_x4_elect(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p, t, e;\n .reg .b32 r;\n .reg .b64 a, b;\n setp.ne.b32 p, %4, 0;\n setp.eq.b32 t, %3, %3;\n"
      " elect.sync r|e, 0xffffffff;\n"
      " @e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n"
      " add.s64 a, %1, 2;\n add.s64 b, %2, 2;\n"
      " @e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, t;\n"
      " add.s64 a, %1, 4;\n add.s64 b, %2, 4;\n"
      " @e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, t;\n"
      " add.s64 a, %1, 6;\n add.s64 b, %2, 6;\n"
      " @e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, t;\n}\n" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// The same with A in TMEM (8 columns a step) and B MN-major: 16 rows of 128 bytes a step.
MB_DEV void umma_ts_x4_elect(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p, t, e;\n .reg .b32 r, a;\n .reg .b64 b;\n setp.ne.b32 p, %4, 0;\n setp.eq.b32 t, %3, %3;\n"
      " elect.sync r|e, 0xffffffff;\n"
      " @e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
      " add.s32 a, %1, 8;\n add.s64 b, %2, 128;\n"
      " @e tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, t;\n"
      " add.s32 a, %1, 16;\n add.s64 b, %2, 256;\n"
      " @e tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, t;\n"
      " add.s32 a, %1, 24;\n add.s64 b, %2, 384;\n"
      " @e tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, t;\n}\n" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

}  // namespace attn
}  // namespace mb
