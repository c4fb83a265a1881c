// rk_act.cuh — activations of the serving operators: float32, float16 or
// bfloat16 in memory, float32 in registers.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "rk_common.cuh"

namespace rk {

RK_DEV float act_load(const float *p) { return *p; }
RK_DEV float act_load(const __half *p) { return __half2float(*p); }
RK_DEV float act_load(const __nv_bfloat16 *p) { return __bfloat162float(*p); }
RK_DEV void act_store(float *p, float v) { *p = v; }
RK_DEV void act_store(__half *p, float v) { *p = __float2half_rn(v); }
RK_DEV void act_store(__nv_bfloat16 *p, float v) { *p = __float2bfloat16_rn(v); }

// Two neighbours of 16 bits, the first in the low half.
template <class T>
RK_DEV float2 act_pair(uint32_t w);
template <>
RK_DEV float2 act_pair<__nv_bfloat16>(uint32_t w) {
  return make_float2(u2f(w << 16), u2f(w & 0xffff0000u));
}
template <>
RK_DEV float2 act_pair<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2 *>(&w));
}
template <class T>
RK_DEV uint32_t act_pack(float a, float b);
template <>
RK_DEV uint32_t act_pack<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&v);
}
template <>
RK_DEV uint32_t act_pack<__half>(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&v);
}

// Scales below this are stored as zero, with zeros for their values: their
// reciprocal would leave float32's range.
constexpr uint32_t K_TINY = 0x03800000u;  // 2^-120

// clamp(RoundToEven(x · inv), ±127); NaN gives 0.
RK_DEV int quant127(float x, float inv) {
  const float p = __fmul_rn(x, inv);
  if (p != p) return 0;
  return int(rintf(fminf(127.0f, fmaxf(-127.0f, p))));
}

// The same for x · inv within ±127.5, as the low byte of the result: adding
// 1.5·2^23 rounds to even and leaves the integer in the low bits, at full rate
// (rintf and the conversion to int run at a quarter of it).
RK_DEV uint32_t quant127_bits(float x, float inv) { return f2u(__fadd_rn(__fmul_rn(x, inv), 12582912.0f)); }
// Four of them as bytes.
RK_DEV uint32_t pack_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// |x| of a finite x, else 0.
RK_DEV float finite_abs(float x) {
  const float a = fabsf(x);
  return a < u2f(0x7f800000u) ? a : 0.0f;
}

}  // namespace rk
