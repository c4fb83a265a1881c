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

// Scales below this are stored as zero, with zeros for their values: their
// reciprocal would leave float32's range.
constexpr uint32_t K_TINY = 0x03800000u;  // 2^-120

// clamp(RoundToEven(x · inv), ±127); NaN gives 0.
RK_DEV int quant127(float x, float inv) {
  const float p = __fmul_rn(x, inv);
  if (p != p) return 0;
  return int(rintf(fminf(127.0f, fmaxf(-127.0f, p))));
}

// |x| of a finite x, else 0.
RK_DEV float finite_abs(float x) {
  const float a = fabsf(x);
  return a < u2f(0x7f800000u) ? a : 0.0f;
}

}  // namespace rk
