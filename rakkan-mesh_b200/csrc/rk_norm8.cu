// rk_norm8.cu — residual addition and RMSNorm with an 8-bit output.
//
//   h = x + residual,  u = h·w,  base = max|u| / 127 over a group,
//   q = round(u / base),  scale = base / sqrt(mean(h²) + eps).
// The integers do not depend on the row's norm (it cancels in u / base), so a
// row is read once: h and u stay in registers, the integers are stored while
// the sum of squares is still on its way through the CTA, and only the scales
// wait for it. The bytes of x, residual, sum and q bound the call.
//
// A CTA takes a row, a thread K pieces of VEC neighbours (16 bytes, or single
// values where rows or groups do not lie on 16-byte boundaries); a group is a
// power of two of lanes, whose largest magnitude is found by shuffles, or the
// whole row. Other groups take a kernel that keeps h in shared memory.
// 4096 rows of 5120 bfloat16 values in groups of 128 take 25.9 us, 5.7 TB/s; one
// row of 4096 float32 values 3.1 us, most of it the launch.
#include "rk_act.cuh"
#include "rk_serve.cuh"
#include "rk_warp.cuh"

namespace rk {

// VEC values as they lie in memory.
template <class T, int VEC>
struct Piece {
  uint4 bits;
  RK_DEV void load(const T *p) { bits = *reinterpret_cast<const uint4 *>(p); }
  RK_DEV void values(float *v) const {
    const uint32_t w[4] = {bits.x, bits.y, bits.z, bits.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
      if constexpr (sizeof(T) == 4) {
        v[i] = u2f(w[i]);
      } else {
        const float2 h = act_pair<T>(w[i]);
        v[2 * i] = h.x;
        v[2 * i + 1] = h.y;
      }
    }
  }
};
template <class T>
struct Piece<T, 1> {
  T bits;
  RK_DEV void load(const T *p) { bits = *p; }
  RK_DEV void values(float *v) const { v[0] = act_load(&bits); }
};
template <int VEC>
RK_DEV void norm_store(float *p, const float *v) {
  if constexpr (VEC == 4) *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
  else *p = v[0];
}
template <int VEC, class T>
RK_DEV void norm_store(T *p, const float *v) {
  if constexpr (VEC == 8) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) w[i] = act_pack<T>(v[2 * i], v[2 * i + 1]);
    *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
    act_store(p, v[0]);
  }
}

// 1 / sqrt(mean + eps) within a few units in the last place (the integers do
// not depend on it).
RK_DEV float norm_recip(float ss, float inv_cols, float eps) { return rsqrtf(fmaf(ss, inv_cols, eps)); }
// base of a group's largest magnitude, and the factor of its values.
RK_DEV float norm_base(float m, float &inv) {
  float base = __fmul_rn(m, u2f(K_1_127));
  if (base < u2f(K_TINY)) base = 0.0f;
  inv = base > 0.0f ? __frcp_rn(base) : 0.0f;
  return base;
}

// log_lanes: of the lanes of a group (0 to 5); -1: the group is the row. A CTA
// takes every gridDim.x-th row and loads the next one before it waits for a
// row's sum (41.9 us for 4096x5120 bfloat16 with a CTA a row and no loads in
// flight meanwhile).
template <class T, int VEC, int K>
__global__ void __launch_bounds__(K <= 2 ? 1024 : 512) k_norm8(Norm8Args a, int log_lanes) {
  __shared__ float sh[2][32], sh_max[2][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const auto at_of = [&](int k) { return VEC * ((int)threadIdx.x + k * (int)blockDim.x); };
  Piece<T, VEC> x[K], res[K], w[K];
  const auto load = [&](int64_t row) {
#pragma unroll
    for (int k = 0; k < K; k++)
      if (at_of(k) < a.cols) {
        x[k].load(static_cast<const T *>(a.x) + row * a.x_stride + at_of(k));
        if (a.residual) res[k].load(static_cast<const T *>(a.residual) + row * a.r_stride + at_of(k));
      }
  };
  load(blockIdx.x);
#pragma unroll
  for (int k = 0; k < K; k++)
    if (at_of(k) < a.cols) w[k].load(static_cast<const T *>(a.weight) + at_of(k));
  // Values within ±127 of their base need no clamp; a thread with a NaN or an
  // infinity among its h (then its squares' sum is one), weights or products
  // (then its largest is one, and it times the factor of zero a NaN) does.
  bool odd_weights = false;
#pragma unroll
  for (int k = 0; k < K; k++)
    if (at_of(k) < a.cols) {
      float f[VEC];
      w[k].values(f);
#pragma unroll
      for (int i = 0; i < VEC; i++) odd_weights |= !(fabsf(f[i]) < INFINITY);
    }

  int flip = 0;
  const int groups = a.cols / a.group;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, flip ^= 1) {
    int8_t *q = a.q + row * a.cols;
    float u[K][VEC], ss = 0.0f, top[K], base[K], all = 0.0f;
#pragma unroll
    for (int k = 0; k < K; k++) {
      top[k] = 0.0f;
#pragma unroll
      for (int i = 0; i < VEC; i++) u[k][i] = 0.0f;
      if (at_of(k) < a.cols) {
        float h[VEC], f[VEC];
        x[k].values(h);
        if (a.residual) {
          res[k].values(f);
#pragma unroll
          for (int i = 0; i < VEC; i++) h[i] = __fadd_rn(h[i], f[i]);
        }
        if (a.sum_out) norm_store<VEC>(static_cast<T *>(a.sum_out) + row * a.s_stride + at_of(k), h);
        w[k].values(f);
#pragma unroll
        for (int i = 0; i < VEC; i++) {
          ss = fmaf(h[i], h[i], ss);
          u[k][i] = __fmul_rn(h[i], f[i]);
          top[k] = fmaxf(top[k], fabsf(u[k][i]));
        }
      }
      all = fmaxf(all, top[k]);
    }
    if (row + gridDim.x < a.rows) load(row + gridDim.x);
    const bool odd = odd_weights || !(ss < INFINITY) || !(all < INFINITY);
    auto store = [&](int k, float inv) {
      const int at = at_of(k);
      if (at >= a.cols) return;
      uint32_t v[VEC];
      if (odd) {
#pragma unroll
        for (int i = 0; i < VEC; i++) v[i] = (uint32_t)quant127(u[k][i], inv);
      } else {
#pragma unroll
        for (int i = 0; i < VEC; i++) v[i] = quant127_bits(u[k][i], inv);
      }
      if constexpr (VEC == 1) {
        q[at] = (int8_t)v[0];
      } else {
        uint32_t p[VEC / 4];
#pragma unroll
        for (int i = 0; i < VEC / 4; i++) p[i] = pack_bytes(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
        if constexpr (VEC == 8) *reinterpret_cast<uint2 *>(q + at) = make_uint2(p[0], p[1]);
        else *reinterpret_cast<uint32_t *>(q + at) = p[0];
      }
    };
    ss = warp_sum(ss);
    if (log_lanes < 0) all = warp_max(all);
    if (lane == 0) {
      sh[flip][warp] = ss;
      sh_max[flip][warp] = all;
    }
    if (log_lanes >= 0) {
#pragma unroll
      for (int o = 0; o < 5; o++)
        if (o < log_lanes)
#pragma unroll
          for (int k = 0; k < K; k++) top[k] = fmaxf(top[k], __shfl_xor_sync(0xffffffffu, top[k], 1 << o));
#pragma unroll
      for (int k = 0; k < K; k++) {
        float inv;
        base[k] = norm_base(top[k], inv);
        store(k, inv);
      }
    }
    __syncthreads();  // one a row: the next row's sums go to the other half
    ss = lane < warps ? sh[flip][lane] : 0.0f;
    const float r = norm_recip(warp_sum(ss), a.inv_cols, a.eps);
    if (log_lanes < 0) {
      float inv;
      const float b = norm_base(warp_max(lane < warps ? sh_max[flip][lane] : 0.0f), inv);
#pragma unroll
      for (int k = 0; k < K; k++) store(k, inv);
      if (threadIdx.x == 0) a.scales[row] = __fmul_rn(b, r);
    } else if ((threadIdx.x & ((1 << log_lanes) - 1)) == 0) {
      float *scales = a.scales + row * groups;
#pragma unroll
      for (int k = 0; k < K; k++)
        if (at_of(k) < a.cols) scales[((int)threadIdx.x + k * (int)blockDim.x) >> log_lanes] = __fmul_rn(base[k], r);
    }
  }
}

// Any group: h in shared memory where a row fits (else read again), a warp
// per group in turn.
constexpr int kNormThreads = 256, kNormShared = 12000;

template <class T>
__global__ void __launch_bounds__(kNormThreads) k_norm8_any(Norm8Args a) {
  __shared__ float sh[kNormThreads / 32], keep[kNormShared];
  const int64_t row = blockIdx.x;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const bool kept = a.cols <= kNormShared;
  const T *x = static_cast<const T *>(a.x) + row * a.x_stride;
  const T *res = a.residual ? static_cast<const T *>(a.residual) + row * a.r_stride : nullptr;
  const T *w = static_cast<const T *>(a.weight);
  auto h_of = [&](int j) { return res ? __fadd_rn(act_load(x + j), act_load(res + j)) : act_load(x + j); };
  float ss = 0.0f;
  for (int j = threadIdx.x; j < a.cols; j += kNormThreads) {
    const float h = h_of(j);
    if (kept) keep[j] = h;
    ss = fmaf(h, h, ss);
  }
  ss = warp_sum(ss);
  if (lane == 0) sh[warp] = ss;
  __syncthreads();
  ss = 0.0f;
  for (int i = 0; i < kNormThreads / 32; i++) ss += sh[i];
  const float r = norm_recip(ss, a.inv_cols, a.eps);
  const int groups = a.cols / a.group;
  for (int g = warp; g < groups; g += kNormThreads / 32) {
    float m = 0.0f;
    for (int j = lane; j < a.group; j += 32) {
      const int c = g * a.group + j;
      m = fmaxf(m, fabsf(__fmul_rn(kept ? keep[c] : h_of(c), act_load(w + c))));
    }
    float inv;
    const float base = norm_base(warp_max(m), inv);
    for (int j = lane; j < a.group; j += 32) {
      const int c = g * a.group + j;
      a.q[row * a.cols + c] = (int8_t)quant127(__fmul_rn(kept ? keep[c] : h_of(c), act_load(w + c)), inv);
    }
    if (lane == 0) a.scales[row * groups + g] = __fmul_rn(base, r);
  }
  if (!a.sum_out) return;
  __syncthreads();  // sum_out may be x or the residual
  T *sum = static_cast<T *>(a.sum_out) + row * a.s_stride;
  for (int j = threadIdx.x; j < a.cols; j += kNormThreads) act_store(sum + j, kept ? keep[j] : h_of(j));
}

template <class T, int VEC>
static cudaError_t norm_pieces(const Norm8Args &a, int sms, int lanes, cudaStream_t st, bool &taken) {
  // Few rows: as many threads as pieces. Many: CTAs of up to 512, several of
  // which share an SM.
  const int pieces = a.cols / VEC, most = a.rows >= 2 * sms ? 512 : 1024;
  const auto threads = [&](int k) { return ((pieces + k - 1) / k + 31) / 32 * 32; };
  // As many CTAs as the SMs hold at the registers that the bounds leave.
  const auto ctas = [&](int t, int regs) {
    const int n = 65536 / (regs * t), by_threads = 2048 / t;
    const int64_t all = (int64_t)sms * (n < by_threads ? n : by_threads);
    return (unsigned)(a.rows < all ? a.rows : all);
  };
  taken = true;
  int t;
  if ((t = threads(1)) <= most) return launch_k(k_norm8<T, VEC, 1>, ctas(t, 64), t, 0, st, a, lanes);
  if ((t = threads(2)) <= most) return launch_k(k_norm8<T, VEC, 2>, ctas(t, 64), t, 0, st, a, lanes);
  if ((t = threads(4)) <= 512) return launch_k(k_norm8<T, VEC, 4>, ctas(t, 128), t, 0, st, a, lanes);
  if ((t = threads(8)) <= 512) return launch_k(k_norm8<T, VEC, 8>, ctas(t, 128), t, 0, st, a, lanes);
  taken = false;
  return cudaSuccess;
}

template <class T>
static cudaError_t norm_typed(const Norm8Args &a, int sms, cudaStream_t st) {
  constexpr int VEC = 16 / sizeof(T);
  const auto on16 = [](const void *p, int64_t stride) {
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && stride % VEC == 0;
  };
  const bool vec = a.cols % VEC == 0 && on16(a.x, a.x_stride) && on16(a.weight, 0) && (!a.residual || on16(a.residual, a.r_stride)) &&
                   (!a.sum_out || on16(a.sum_out, a.s_stride)) && (reinterpret_cast<uintptr_t>(a.q) & 7) == 0;
  const auto lanes_of = [&](int v) {  // log2; -1: the row; -2: no power of two of lanes
    if (a.group == a.cols) return -1;
    for (int k = 0; k <= 5; k++)
      if (a.group == v << k) return k;
    return -2;
  };
  bool taken = false;
  cudaError_t e = cudaSuccess;
  if (vec && lanes_of(VEC) >= -1) e = norm_pieces<T, VEC>(a, sms, lanes_of(VEC), st, taken);
  else if (lanes_of(1) >= -1) e = norm_pieces<T, 1>(a, sms, lanes_of(1), st, taken);
  return taken ? e : launch_k(k_norm8_any<T>, a.rows, kNormThreads, 0, st, a);
}

cudaError_t launch_add_rmsnorm_q8(const Norm8Args &a, int type, int sms, cudaStream_t st) {
  switch (type) {
    case RK_ACT_F32: return norm_typed<float>(a, sms, st);
    case RK_ACT_F16: return norm_typed<__half>(a, sms, st);
    default: return norm_typed<__nv_bfloat16>(a, sms, st);
  }
}

cudaError_t init_norm8_attributes() { return cudaSuccess; }

}  // namespace rk
