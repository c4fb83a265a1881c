// rk_w4.cu — products of a 4-bit matrix with group scales and 8-bit vectors.
#include "rk_act.cuh"
#include "rk_serve.cuh"

namespace rk {

// A warp per (row, vector): lane j takes every 32nd block of 32 columns.
constexpr int kW4Warps = 4;

RK_DEV float scale_at(const void *s, int type, int64_t i) {
  if (type == RK_ACT_F32) return static_cast<const float *>(s)[i];
  if (type == RK_ACT_F16) return __half2float(static_cast<const __half *>(s)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16 *>(s)[i]);
}

template <class T>
__global__ void __launch_bounds__(32 * kW4Warps) k_w4_rows(W4Args a) {
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * kW4Warps + (threadIdx.x >> 5), v = blockIdx.y;
  if (row >= a.rows) return;
  const int blocks = a.cols / 32, groups = a.cols / a.group, xgroups = a.cols / a.x_group;
  float acc = 0.0f;
  for (int b = lane; b < blocks; b += 32) {
    const int64_t g = row * groups + 32 * b / a.group;
    const int z = a.zeros ? a.zeros[g] : 8;
    const uint8_t *w = a.w + row * (a.cols / 2) + 16 * b;
    const int8_t *x = a.x + v * a.cols + 32 * b;
    int dot = 0;
    for (int j = 0; j < 16; j++) dot += ((w[j] & 15) - z) * x[j] + ((w[j] >> 4) - z) * x[j + 16];
    acc = fmaf((float)dot, scale_at(a.scales, a.scale_type, g) * a.x_scales[v * xgroups + 32 * b / a.x_group], acc);
  }
  for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
  if (lane == 0) act_store(static_cast<T *>(a.out) + v * a.out_stride + row, acc);
}

cudaError_t launch_w4_mulvec(const W4Args &a, int type, int, cudaStream_t st) {
  for (int v = 0; v < a.n; v += 32768) {  // grid.y's limit
    W4Args b = a;
    b.n = a.n - v < 32768 ? a.n - v : 32768;
    b.x += (int64_t)v * a.cols;
    b.x_scales += (int64_t)v * (a.cols / a.x_group);
    b.out = static_cast<char *>(a.out) + (int64_t)v * a.out_stride * (type == RK_ACT_F32 ? 4 : 2);
    const dim3 grid((a.rows + kW4Warps - 1) / kW4Warps, b.n);
    cudaError_t e = type == RK_ACT_F32   ? launch_k(k_w4_rows<float>, grid, 32 * kW4Warps, 0, st, b)
                    : type == RK_ACT_F16 ? launch_k(k_w4_rows<__half>, grid, 32 * kW4Warps, 0, st, b)
                                         : launch_k(k_w4_rows<__nv_bfloat16>, grid, 32 * kW4Warps, 0, st, b);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

cudaError_t init_w4_attributes() { return cudaSuccess; }

}  // namespace rk
