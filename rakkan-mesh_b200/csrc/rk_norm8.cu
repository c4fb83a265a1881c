// rk_norm8.cu — residual addition and RMSNorm with an 8-bit output.
#include "rk_act.cuh"
#include "rk_serve.cuh"

namespace rk {

// A CTA per row, a warp per group in turn: h is formed, stored and squared
// on the first reading, the groups' magnitudes and integers on the second.
constexpr int kNormThreads = 256;

template <class T>
__global__ void __launch_bounds__(kNormThreads) k_norm8_rows(Norm8Args a) {
  __shared__ float sh[kNormThreads / 32];
  const int64_t row = blockIdx.x;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const T *x = static_cast<const T *>(a.x) + row * a.x_stride;
  const T *res = a.residual ? static_cast<const T *>(a.residual) + row * a.r_stride : nullptr;
  const T *w = static_cast<const T *>(a.weight);
  auto h_of = [&](int j) { return res ? __fadd_rn(act_load(x + j), act_load(res + j)) : act_load(x + j); };
  float ss = 0.0f;
  for (int j = threadIdx.x; j < a.cols; j += kNormThreads) {
    const float h = h_of(j);
    ss = fmaf(h, h, ss);
  }
  for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  if (lane == 0) sh[warp] = ss;
  __syncthreads();
  ss = 0.0f;
  for (int i = 0; i < kNormThreads / 32; i++) ss += sh[i];
  const float r = __frcp_rn(__fsqrt_rn(ss / (float)a.cols + a.eps));
  const int groups = a.cols / a.group;
  for (int g = warp; g < groups; g += kNormThreads / 32) {
    float m = 0.0f;
    for (int j = lane; j < a.group; j += 32) {
      const int c = g * a.group + j;
      m = fmaxf(m, fabsf(__fmul_rn(h_of(c), act_load(w + c))));
    }
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    float base = __fmul_rn(m, u2f(K_1_127));
    if (base < u2f(K_TINY)) base = 0.0f;
    const float inv = base > 0.0f ? __fdiv_rn(1.0f, base) : 0.0f;
    for (int j = lane; j < a.group; j += 32) {
      const int c = g * a.group + j;
      a.q[row * a.cols + c] = (int8_t)quant127(__fmul_rn(h_of(c), act_load(w + c)), inv);
    }
    if (lane == 0) a.scales[row * groups + g] = __fmul_rn(base, r);
  }
  if (!a.sum_out) return;
  __syncthreads();  // sum_out may be x or the residual
  T *sum = static_cast<T *>(a.sum_out) + row * a.s_stride;
  for (int j = threadIdx.x; j < a.cols; j += kNormThreads) act_store(sum + j, h_of(j));
}

cudaError_t launch_add_rmsnorm_q8(const Norm8Args &a, int type, int, cudaStream_t st) {
  switch (type) {
    case RK_ACT_F32: return launch_k(k_norm8_rows<float>, a.rows, kNormThreads, 0, st, a);
    case RK_ACT_F16: return launch_k(k_norm8_rows<__half>, a.rows, kNormThreads, 0, st, a);
    default: return launch_k(k_norm8_rows<__nv_bfloat16>, a.rows, kNormThreads, 0, st, a);
  }
}

cudaError_t init_norm8_attributes() { return cudaSuccess; }

}  // namespace rk
