// rk_attn8.cu — attention over the 8-bit paged cache: the kernels with one
// float16 term, the join, and the launches.
#include "rk_attn8.cuh"

namespace rk {

// Joins the parts of the unit that crosses into CTA blockIdx.x + 1: the CTAs
// it crosses into share its rows.
constexpr int kJoinThreads = 128, kJoinParts = 256;

__global__ void __launch_bounds__(kJoinThreads) k_attn8_join(Attn8Args a, int type, A8Grid grid) {
  __shared__ float s_g[kJoinParts];
  __shared__ float s_red[2][kJoinThreads / 32];
  griddep_wait();
  const A8Record *records = static_cast<const A8Record *>(a.ws);
  const float *parts = reinterpret_cast<const float *>(records + grid.ctas);
  const int b = blockIdx.x + 1, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const A8Record rec = records[b];
  if (rec.first < 0) return;
  const int hs = a.c.head_size, G = a.heads / a.c.kv_heads, n = rec.last - rec.first + 1;
  const int64_t size = a8_part_floats(hs);
  auto part_of = [&](int i) { return parts + (2LL * (rec.first + i) + (i == 0 ? 1 : 0)) * size; };
  for (int row = b - rec.first - 1; row < rec.rows; row += n - 1) {
    float mm = -INFINITY, MM = -INFINITY;
    for (int i = tid; i < n; i += kJoinThreads) {
      const float *s = part_of(i) + 64 * hs + 4 * row;
      mm = fmaxf(mm, s[0]);
      MM = fmaxf(MM, s[1]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, o));
      MM = fmaxf(MM, __shfl_xor_sync(0xffffffffu, MM, o));
    }
    __syncthreads();
    if (lane == 0) {
      s_red[0][warp] = mm;
      s_red[1][warp] = MM;
    }
    __syncthreads();
    for (int w = 0; w < kJoinThreads / 32; w++) {
      mm = fmaxf(mm, s_red[0][w]);
      MM = fmaxf(MM, s_red[1][w]);
    }
    const float msafe = mm == -INFINITY ? 0.0f : mm, Msafe = MM == -INFINITY ? 0.0f : MM;
    float ll = 0.0f, v0 = 0.0f, v1 = 0.0f;  // dimensions tid and tid + 128
    for (int i0 = 0; i0 < n; i0 += kJoinParts) {
      const int k = min(kJoinParts, n - i0);
      __syncthreads();
      for (int i = tid; i < k; i += kJoinThreads) {
        const float *s = part_of(i0 + i) + 64 * hs + 4 * row;
        s_g[i] = exp2f(s[1] - Msafe);
        ll += s[2] * exp2f(s[0] - msafe);
      }
      __syncthreads();
      if (tid < hs) {
#pragma unroll 8
        for (int i = 0; i < k; i++) v0 = fmaf(part_of(i0 + i)[row * hs + tid], s_g[i], v0);
        if (hs > kJoinThreads)
#pragma unroll 8
          for (int i = 0; i < k; i++) v1 = fmaf(part_of(i0 + i)[row * hs + tid + kJoinThreads], s_g[i], v1);
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ll += __shfl_xor_sync(0xffffffffu, ll, o);
    __syncthreads();
    if (lane == 0) s_red[0][warp] = ll;
    __syncthreads();
    ll = 0.0f;
    for (int w = 0; w < kJoinThreads / 32; w++) ll += s_red[0][w];
    const float scale = ll == 0.0f ? 0.0f : exp2f(Msafe - 14.0f - msafe) / ll;
    const int qrow = rec.row0 + row;
    const int64_t oi = (int64_t)(rec.q0 + qrow / G) * a.out_stride + (int64_t)(rec.head * G + qrow % G) * hs;
    if (tid < hs) o_store(a.out, type, oi + tid, v0 * scale);
    if (tid + kJoinThreads < hs) o_store(a.out, type, oi + tid + kJoinThreads, v1 * scale);
  }
}

// The workspace is sized for the most CTAs that any type's kernel has.
int64_t attn8_workspace(const rk_kv8 &c, int, int sms) {
  const int64_t ctas = (int64_t)sms * a8_ctas(c.head_size, 1, 1);
  return ctas * (int64_t)sizeof(A8Record) + 2 * ctas * a8_part_floats(c.head_size) * 4;
}

cudaError_t launch_kv8_attention(const Attn8Args &a, int type, int sms, cudaStream_t st) {
  const int hs = a.c.head_size, G = a.heads / a.c.kv_heads;
  // Two tiles of 8 rows a warp halve the conversions a row costs, once the
  // requests have more than 8 rows a kv head on average. float16 takes two
  // terms below that, where they cost little beside the loads: one term's
  // rounding is not far below the output's own.
  const bool rows = (int64_t)a.tokens * G > 8LL * a.n;
  const int terms = type == RK_ACT_F32 || (type == RK_ACT_F16 && !rows) ? 2 : 1;
  const int nt = terms == 1 && rows && hs <= 128 ? 2 : 1;
  A8Grid g{sms * a8_ctas(hs, terms, nt), 4, a.c.block == 16 ? 4 : a.c.block == 32 ? 5 : a.c.block == 64 ? 6 : 7};
  // Short tables: a unit's tiles are few for one CTA, and without units cut in
  // two there is nothing to join.
  const bool whole = (int64_t)a.max_blocks * a.c.block <= 512;
  if (whole) g.min_tiles = 0;
  cudaError_t e = terms == 2 ? attn8_main_two(a, type, g, st) : A8<1>::at(hs, A8<1>::Launch{a, type, nt, g, st});
  if (e != cudaSuccess || whole) return e;
  // The join may be placed while the main kernel's last CTAs run; it waits
  // for them before it reads.
  const bool pdl = g_pdl;
  g_pdl = true;
  e = launch_k(k_attn8_join, g.ctas - 1, kJoinThreads, 0, st, a, type, g);
  g_pdl = pdl;
  return e;
}

cudaError_t init_attn8_attributes() {
  const cudaError_t e = attn8_init_two();
  return e != cudaSuccess ? e : A8<1>::init();
}

}  // namespace rk
