// Arithmetic of the tensor-core attention kernels' softmax: exponentials to base 2
// on the MUFU unit and on the FMA pipe, Blackwell's paired f32 forms, and the
// 32-byte row store.
#pragma once

#include <stdint.h>

namespace lc {
namespace softmax {

// One 32-byte store of eight 32-bit words (the address is 32-byte aligned).
__device__ __forceinline__ void st_global_v8_b32(void *dst, const uint32_t *v) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "r"(v[0]), "r"(v[1]),
               "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Packed pairs of f32 (Blackwell's f32x2 ALU forms: one instruction for two
// lanes of FMA, ADD or SUB).
__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpack2(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t ffma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t fadd2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t fsub2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// 2^x for a pair on the FMA pipe, for a share of the exponentials so the MUFU
// unit is not the limiter.  Range reduction: x = n + f with n = round(x) taken
// from the low mantissa bits of x + 1.5*2^23 and f in [-0.5, 0.5]; 2^f from a
// degree-3 polynomial fitted here by the Remez exchange algorithm for minimax
// relative error on [-0.5, 0.5] (max relative error 7.5e-5, below half an f16
// ulp); 2^n is added to the exponent field.  x is clamped at -125 so the
// exponent stays normal; the caller's x never exceeds 8.
__device__ __forceinline__ uint64_t ex2_poly2(uint64_t x2) {
  const float2 x = unpack2(x2);
  const uint64_t xc = pack2(fmaxf(x.x, -125.0f), fmaxf(x.y, -125.0f));
  const uint64_t magic = pack2(12582912.0f, 12582912.0f);
  const uint64_t t = fadd2(xc, magic);
  const uint64_t f = fsub2(xc, fsub2(t, magic));
  uint64_t q = ffma2(pack2(0.0551716685f, 0.0551716685f), f, pack2(0.242611125f, 0.242611125f));
  q = ffma2(q, f, pack2(0.693260968f, 0.693260968f));
  q = ffma2(q, f, pack2(0.999928057f, 0.999928057f));
  const float2 qq = unpack2(q), tt = unpack2(t);
  return pack2(__int_as_float(__float_as_int(qq.x) + (__float_as_int(tt.x) << 23)),
               __int_as_float(__float_as_int(qq.y) + (__float_as_int(tt.y) << 23)));
}

}  // namespace softmax
}  // namespace lc
