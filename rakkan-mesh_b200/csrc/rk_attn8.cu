// rk_attn8.cu — attention over the 8-bit paged cache: the kernels with one
// float16 term, the join, and the launches.
#include "rk_attn8.cuh"

namespace rk {

// Joins the parts of the unit that crosses into CTA c of the main kernel
// (c = blockIdx.x + 1). The CTAs of all its crossings share its rows. A row of a
// few parts is one warp's, a row of many all four's: a warp's lanes read its
// parts' (m, M, l) side by side, then the sums, four dimensions a lane, with
// all loads under way at once; each step is a round trip to L2, and there is
// little else to the call.
constexpr int kJoinWarps = 4, kJoinFew = 8;

template <int J>  // pieces of 128 dimensions
__global__ void __launch_bounds__(32 * kJoinWarps) k_attn8_join(Attn8Args a, int type, A8Grid grid) {
  __shared__ float4 s_v[kJoinWarps][J][32];
  __shared__ float s_st[kJoinWarps][3];
  griddep_wait();
  const A8Record *records = static_cast<const A8Record *>(a.ws);
  const float *parts = reinterpret_cast<const float *>(records + grid.ctas);
  const int b = blockIdx.x + 1, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const A8Record rec = records[b];
  if (rec.first < 0) return;
  const int hs = a.c.head_size, G = a.heads / a.c.kv_heads, n = rec.last - rec.first + 1;
  const int64_t size = a8_part_floats(hs);
  // Part i is CTA first + i's: its second slot where the unit begins, else its first.
  const float *p0 = parts + 2LL * rec.first * size;
  auto part_of = [&](int i) { return p0 + (2LL * i + (i == 0)) * size; };
  const bool few = n <= kJoinFew;
  const int nth = (b - rec.first - 1) * gridDim.y + blockIdx.y, step = (n - 1) * gridDim.y;
  const int row0 = few ? nth * kJoinWarps + warp : nth, row_step = few ? step * kJoinWarps : step;
  const int my0 = few ? 0 : warp, my_step = few ? 1 : kJoinWarps;  // parts of this warp
  for (int row = row0; row < rec.rows; row += row_step) {
    float mm = -INFINITY, MM = -INFINITY, ll = 0.0f;
    float4 v[J] = {};
    for (int i0 = my0; i0 < n; i0 += 32 * my_step) {
      const int k = min(32, (n - i0 + my_step - 1) / my_step);
      float m = -INFINITY, M = -INFINITY, l = 0.0f;
      if (lane < k) {
        const float4 s = *reinterpret_cast<const float4 *>(part_of(i0 + lane * my_step) + 64 * hs + 4 * row);
        m = s.x, M = s.y, l = s.z;
      }
      const float m1 = fmaxf(mm, warp_max(m)), M1 = fmaxf(MM, warp_max(M));
      const float ms = m1 == -INFINITY ? 0.0f : m1, Ms = M1 == -INFINITY ? 0.0f : M1;
      const float g = exp2f(M - Ms), old = exp2f(MM - Ms);
      ll = ll * exp2f(mm - ms) + warp_sum(l * exp2f(m - ms));
      mm = m1, MM = M1;
#pragma unroll
      for (int j = 0; j < J; j++) v[j].x *= old, v[j].y *= old, v[j].z *= old, v[j].w *= old;
      for (int i1 = 0; i1 < k; i1 += 8) {
        float4 x[8][J];
#pragma unroll
        for (int i = 0; i < 8; i++)
#pragma unroll
          for (int j = 0; j < J; j++) {
            const int d = 4 * lane + 128 * j;
            x[i][j] = i1 + i < k && d < hs ? *reinterpret_cast<const float4 *>(part_of(i0 + (i1 + i) * my_step) + row * hs + d)
                                           : make_float4(0, 0, 0, 0);
          }
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const float w = __shfl_sync(0xffffffffu, g, min(i1 + i, 31));
#pragma unroll
          for (int j = 0; j < J; j++)
            if (i1 + i < k) {
              v[j].x = fmaf(x[i][j].x, w, v[j].x);
              v[j].y = fmaf(x[i][j].y, w, v[j].y);
              v[j].z = fmaf(x[i][j].z, w, v[j].z);
              v[j].w = fmaf(x[i][j].w, w, v[j].w);
            }
        }
      }
    }
    if (!few) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < J; j++) s_v[warp][j][lane] = v[j];
      if (lane == 0) s_st[warp][0] = mm, s_st[warp][1] = MM, s_st[warp][2] = ll;
      __syncthreads();
      if (warp > 0) continue;
      float m1 = mm, M1 = MM;
#pragma unroll
      for (int w = 1; w < kJoinWarps; w++) m1 = fmaxf(m1, s_st[w][0]), M1 = fmaxf(M1, s_st[w][1]);
      const float ms = m1 == -INFINITY ? 0.0f : m1, Ms = M1 == -INFINITY ? 0.0f : M1;
      ll = 0.0f;
#pragma unroll
      for (int j = 0; j < J; j++) v[j] = make_float4(0, 0, 0, 0);
#pragma unroll
      for (int w = 0; w < kJoinWarps; w++) {
        ll += s_st[w][2] * exp2f(s_st[w][0] - ms);
        const float g = exp2f(s_st[w][1] - Ms);
#pragma unroll
        for (int j = 0; j < J; j++) {
          const float4 x = s_v[w][j][lane];
          v[j].x = fmaf(x.x, g, v[j].x), v[j].y = fmaf(x.y, g, v[j].y);
          v[j].z = fmaf(x.z, g, v[j].z), v[j].w = fmaf(x.w, g, v[j].w);
        }
      }
      mm = m1, MM = M1;
    }
    const float scale = ll == 0.0f ? 0.0f : exp2f((MM == -INFINITY ? 0.0f : MM) - 14.0f - (mm == -INFINITY ? 0.0f : mm)) / ll;
    const int qrow = rec.row0 + row;
    const int64_t oi = (int64_t)(rec.q0 + qrow / G) * a.out_stride + (int64_t)(rec.head * G + qrow % G) * hs;
#pragma unroll
    for (int j = 0; j < J; j++) {
      const int d = 4 * lane + 128 * j;
      if (d >= hs) break;
      o_store4(a.out, type, oi + d, make_float4(v[j].x * scale, v[j].y * scale, v[j].z * scale, v[j].w * scale), grid.vec_out);
    }
  }
}

// The workspace is sized for the most CTAs that any type's kernel has.
int64_t attn8_workspace(const rk_kv8 &c, int sms) {
  const int64_t ctas = (int64_t)sms * a8_ctas(c.head_size, 1, 1);
  return ctas * (int64_t)sizeof(A8Record) + 2 * ctas * a8_part_floats(c.head_size) * 4;
}

cudaError_t launch_kv8_attention(const Attn8Args &a, int type, int sms, cudaStream_t st) {
  const int hs = a.c.head_size, G = a.heads / a.c.kv_heads;
  // Two tiles of 8 rows a warp halve the conversions a row costs, once the
  // requests have more than 16 rows a kv head on average (16 requests over 2048
  // tokens, G = 4: 34.0 us with them and 29.8 without at 16 rows, 39.2 and
  // 44.7 at 20, 65.5 and 75.9 at 64, bfloat16; float32 49.7 and 54.8 at 20, 85.0
  // and 95.2 at 64).
  const bool rows = (int64_t)a.tokens * G > 8LL * a.n;
  const int nt = (int64_t)a.tokens * G > 16LL * a.n && hs <= 128 ? 2 : 1;
  // The precision goes by the type alone, so that a row's does not depend on
  // what else the call holds. One term's rounding (2^-12 of a weight) is an
  // eighth of bfloat16's of the output, but not far below float16's own.
  const int terms = type == RK_ACT_BF16 ? 1 : 2;
  A8Grid g{sms * a8_ctas(hs, terms, nt), 4, a.c.block == 16 ? 4 : a.c.block == 32 ? 5 : a.c.block == 64 ? 6 : 7,
           a.q_stride % 8 == 0 && (reinterpret_cast<uintptr_t>(a.q) & 15) == 0,
           a.out_stride % 4 == 0 && (reinterpret_cast<uintptr_t>(a.out) & (type == RK_ACT_F32 ? 15 : 7)) == 0,
           G > 1 && (int64_t)a.tokens * G * G < 1LL << 32 ? 0xffffffffu / G + 1 : 0};
  // Short tables: a unit's tiles are few for one CTA, and without units cut in
  // two there is nothing to join.
  const bool whole = (int64_t)a.max_blocks * a.c.block <= RK_KV8_NO_WORKSPACE;
  if (whole) g.min_tiles = 0;
  cudaError_t e = terms == 2 ? attn8_main_two(a, type, nt, g, st) : A8<1>::at(hs, A8<1>::Launch{a, type, nt, g, st});
  if (e != cudaSuccess || whole) return e;
  // The join may be placed while the main kernel's last CTAs run; it waits
  // for them before it reads.
  const bool pdl = g_pdl;
  g_pdl = true;
  // Units of up to 64 rows are joined by eight CTAs for each crossing.
  e = launch_k(hs > 128 ? k_attn8_join<2> : k_attn8_join<1>, dim3(g.ctas - 1, rows ? 8 : 1), 32 * kJoinWarps, 0, st, a, type, g);
  g_pdl = pdl;
  return e;
}

cudaError_t init_attn8_attributes() {
  const cudaError_t e = attn8_init_two();
  return e != cudaSuccess ? e : A8<1>::init();
}

}  // namespace rk
