// rk_attn8.cu — attention over the 8-bit paged cache: the kernels for 16-bit
// queries, the join, and the launches.
#include "rk_attn8.cuh"

namespace rk {

// Joins the parts of the unit that crosses into CTA blockIdx.x + 1: the CTAs
// it crosses into share its rows.
__global__ void __launch_bounds__(128) k_attn8_join(Attn8Args a, int type, A8Grid grid) {
  griddep_wait();
  const A8Record *records = static_cast<const A8Record *>(a.ws);
  const float *parts = reinterpret_cast<const float *>(records + grid.ctas);
  const int b = blockIdx.x + 1;
  const int first = records[b].first;
  if (first < 0) return;
  const A8Record rec = records[b];
  const int hs = a.c.head_size, G = a.heads / a.c.kv_heads, n = rec.last - first + 1;
  const int64_t size = a8_part_floats(hs);
  auto part_of = [&](int i) { return parts + (2LL * (first + i) + (i == 0 ? 1 : 0)) * size; };
  for (int row = b - first - 1; row < rec.rows; row += n - 1) {
    float mm = -INFINITY, MM = -INFINITY;
    for (int i = 0; i < n; i++) {
      const float *s = part_of(i) + 64 * hs + 4 * row;
      mm = fmaxf(mm, s[0]);
      MM = fmaxf(MM, s[1]);
    }
    const float msafe = mm == -INFINITY ? 0.0f : mm, Msafe = MM == -INFINITY ? 0.0f : MM;
    const int qrow = rec.row0 + row;
    const int64_t oi = (int64_t)(rec.q0 + qrow / G) * a.out_stride + (int64_t)(rec.head * G + qrow % G) * hs;
    for (int d = threadIdx.x; d < hs; d += 128) {
      float ll = 0.0f, v = 0.0f;
#pragma unroll 4
      for (int i = 0; i < n; i++) {
        const float *p = part_of(i), *s = p + 64 * hs + 4 * row;
        ll += s[2] * exp2f(s[0] - msafe);
        v = fmaf(p[row * hs + d], exp2f(s[1] - Msafe), v);
      }
      o_store(a.out, type, oi + d, ll == 0.0f ? 0.0f : v * (exp2f(Msafe - 14.0f - msafe) / ll));
    }
  }
}

// As many CTAs as fit the SMs (A8Shape::CTAS), and
// at least four tiles a CTA, one for each warp.
static A8Grid attn8_grid(int hs, int sms) { return A8Grid{sms * (hs > 128 ? 1 : hs > 64 ? 2 : hs > 32 ? 3 : 4), 4}; }

int64_t attn8_workspace(const rk_kv8 &c, int, int sms) {
  const int64_t ctas = attn8_grid(c.head_size, sms).ctas;
  return ctas * (int64_t)sizeof(A8Record) + 2 * ctas * a8_part_floats(c.head_size) * 4;
}

cudaError_t launch_kv8_attention(const Attn8Args &a, int type, int sms, cudaStream_t st) {
  const A8Grid g = attn8_grid(a.c.head_size, sms);
  cudaError_t e = type == RK_ACT_F32 ? attn8_main_f32(a, type, g, st)
                                     : A8<false>::at(a.c.head_size, A8<false>::Launch{a, type, g, st});
  if (e != cudaSuccess) return e;
  // The join may be placed while the main kernel's last CTAs run; it waits
  // for them before it reads.
  const bool pdl = g_pdl;
  g_pdl = true;
  e = launch_k(k_attn8_join, g.ctas - 1, 128, 0, st, a, type, g);
  g_pdl = pdl;
  return e;
}

cudaError_t init_attn8_attributes() {
  const cudaError_t e = attn8_init_f32();
  return e != cudaSuccess ? e : A8<false>::init();
}

}  // namespace rk
