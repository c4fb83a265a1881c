// rk_w4.cu — products of a 4-bit matrix with group scales and 8-bit vectors.
//
//   out[v][row] = Σ over segments  sw · sx · Σ_k (u_k − z) x_k
// A segment is a run of columns with one weight scale and one vector scale.
// Up to 16 vectors the bytes of the weights bound the product (half a byte a
// weight), so what a warp does for them has to stay below an SM's share of
// the memory bandwidth: about 44 instructions for 256 bytes. The sums run on
// mma.m16n8k32 on signed bytes (16 rows, 8 vectors; one vector fills one
// column, the others ride along), exact in int32. The weights are laid out
// once, at upload, in the order in which a warp's lanes hold the operand, and
// as two's complement nibbles of u − 8: the upper half of a byte, its lower
// half masked away, is then 16 (u − 8) as a signed byte, so unpacking eight
// weights takes three instructions and the 16 goes into the scale. A zero point other than
// 8 takes 16 (z − 8) Σ x off, with Σ x from one more product by a constant operand.
//
// Work. A warp takes MT tiles of 16 rows and a share of their columns, as few
// shares as give every SM sixteen warps (a warp's beginning and end cost as
// much as ten column pairs): first among a CTA's eight warps, which else take
// tiles of their own, then among the CTAs of a cluster. The float32 sums of a
// tile's shares meet in shared memory, in order.
#include <cooperative_groups.h>

#include "rk_act.cuh"
#include "rk_serve.cuh"

namespace cg = cooperative_groups;

namespace rk {

constexpr int kW4Warps = 8;

// Rows are padded to 16 and columns to 128, with zeros. Columns of a lane's
// nibbles, for column pair kp (64 columns), word 2s + h
// (32-column step s, row r + 8h of the tile): low halves 8c .. 8c + 3 of the
// step, high halves 8c + 4 .. 8c + 7. Its vector bytes are eight neighbours.
RK_DEV int w4_col(int kp, int s, int c) { return 64 * kp + 32 * s + 8 * c; }

__global__ void k_w4_layout(const uint8_t *w, int rows, int cols, int kpairs, uint32_t *out, int64_t words) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= words) return;
  const int word = i & 3, lane = (i >> 2) & 31, r = lane >> 2, c = lane & 3;
  const int64_t tile = (i >> 7) / kpairs;
  const int kp = (int)((i >> 7) % kpairs), s = word >> 1;
  const int64_t row = tile * 16 + r + 8 * (word & 1);
  uint32_t v = 0;
  if (row < rows)
    for (int b = 0; b < 8; b++) {
      const int col = w4_col(kp, s, c) + b;
      if (col >= cols) break;
      const uint8_t x = w[row * (cols / 2) + (col / 32) * 16 + col % 16];  // columns j and j + 16 of a block share byte j
      const uint32_t u = (col % 32 < 16 ? x & 15 : x >> 4) ^ 8;
      v |= u << (b < 4 ? 8 * b : 8 * (b - 4) + 4);
    }
  out[i] = v;
}

// [rows][groups] into [tile][group][16], `fill` behind the last row.
template <class T>
__global__ void k_w4_tile(const T *in, int rows, int groups, T fill, T *out, int64_t n) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n) return;
  const int64_t row = (i >> 4) / groups * 16 + (i & 15);
  out[i] = row < rows ? in[row * groups + (i >> 4) % groups] : fill;
}

cudaError_t launch_w4_layout(const uint8_t *w, const void *scales, const uint8_t *zeros, int rows, int cols, int group,
                             int scale_bytes, uint8_t *w_out, void *s_out, uint8_t *z_out, cudaStream_t st) {
  const int kpairs = (cols + 127) / 128 * 2, groups = cols / group, tiles = (rows + 15) / 16;
  const int64_t words = (int64_t)tiles * kpairs * 128, n = (int64_t)tiles * groups * 16;
  const auto grid = [](int64_t k) { return dim3((unsigned)((k + 255) / 256)); };
  cudaError_t e = launch_k(k_w4_layout, grid(words), 256, 0, st, w, rows, cols, kpairs, reinterpret_cast<uint32_t *>(w_out), words);
  if (e == cudaSuccess) {
    if (scale_bytes == 4)
      e = launch_k(k_w4_tile<uint32_t>, grid(n), 256, 0, st, static_cast<const uint32_t *>(scales), rows, groups, 0u,
                   static_cast<uint32_t *>(s_out), n);
    else
      e = launch_k(k_w4_tile<uint16_t>, grid(n), 256, 0, st, static_cast<const uint16_t *>(scales), rows, groups, (uint16_t)0,
                   static_cast<uint16_t *>(s_out), n);
  }
  if (e == cudaSuccess && zeros) e = launch_k(k_w4_tile<uint8_t>, grid(n), 256, 0, st, zeros, rows, groups, (uint8_t)8, z_out, n);
  return e;
}

RK_DEV void imma(int *c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Scales and zero points go through shared memory, a warp's own, for
// kW4Chunk columns at a time: read from global memory where a segment ends
// they cost a round trip for each (25.7 and 62.9 us for 28672x4096 by one vector
// and 4096x14336 by 16).
constexpr int kW4Chunk = 1024;
// Groups that a chunk meets (its first column is a multiple of 128).
__host__ __device__ inline int w4_chunk_groups(int group) {
  return kW4Chunk % group == 0 && group <= 128 ? kW4Chunk / group : kW4Chunk / group + 2;
}
// Bytes of a warp's buffer: scales [groups][16 MT], zero points, vector scales [groups][8 NT].
struct W4Smem {
  int zeros, x, size;
};
__host__ __device__ inline W4Smem w4_smem(const W4Args &a, int mt, int nt) {
  const int g = w4_chunk_groups(a.group) * 16 * mt;
  W4Smem s;
  s.zeros = g * (a.scale_type == RK_ACT_F32 ? 4 : 2);
  s.x = s.zeros + (a.zeros ? g : 0);
  s.size = s.x + w4_chunk_groups(a.x_group) * 8 * nt * 4;
  return s;
}

RK_DEV void w4_copy16(void *dst, const void *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
}
RK_DEV void w4_copy4(void *dst, const void *src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
}

RK_DEV float w4_scale(const char *s, int type, int i) {
  if (type == RK_ACT_F32) return reinterpret_cast<const float *>(s)[i];
  const unsigned short h = reinterpret_cast<const unsigned short *>(s)[i];
  return type == RK_ACT_F16 ? __half2float(__ushort_as_half(h)) : u2f((uint32_t)h << 16);
}

// MT tiles of 16 rows, NT of 8 vectors; SEG columns share their scales.
template <int MT, int NT, int SEG, bool ZEROS, class T>
__global__ void __launch_bounds__(32 * kW4Warps, MT > 1 ? 2 : 3) k_w4(W4Args a, int quads, int split, int log_kw, int bufs) {
  constexpr int AHEAD = 2;  // stretches of 128 columns in flight
  extern __shared__ __align__(16) char sm[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = lane >> 2, c = lane & 3;
  // Of the CTA's eight warps, 2^log_kw share the columns of a tile; so do the
  // CTAs of a cluster, `split` of them (a power of two as well).
  const int tiles = (a.rows + 15) / 16, rank = blockIdx.x & (split - 1), kw = 1 << log_kw;
  const int cta_tile0 = blockIdx.x / split * (kW4Warps >> log_kw) * MT, tile0 = cta_tile0 + (warp >> log_kw) * MT;
  const int v0 = blockIdx.y * 8 * NT;
  // This warp's columns, in whole stretches of 128.
  const int log_shares = __ffs(split) - 1 + log_kw, share = (rank << log_kw) + (warp & (kw - 1));
  const int q0 = (quads * share) >> log_shares, q1 = (quads * (share + 1)) >> log_shares;  // quads <= 2^11, shares <= 2^6

  // A tile behind the last and a vector behind the last are computed from
  // the last one's, and not stored.
  const uint4 *w[MT];
  int tile[MT];
#pragma unroll
  for (int m = 0; m < MT; m++) {
    tile[m] = min(tile0 + m, tiles - 1);
    w[m] = reinterpret_cast<const uint4 *>(a.w) + ((int64_t)tile[m] * quads + q0) * 64 + lane;
  }
  const int8_t *x[NT];
#pragma unroll
  for (int n = 0; n < NT; n++) x[n] = a.x + (int64_t)min(v0 + 8 * n + r, a.n - 1) * a.cols + 128 * q0 + 8 * c;
  uint4 wbuf[AHEAD][MT][2];
  uint2 xbuf[AHEAD][NT][4];
  auto fetch = [&](int i, int q) {  // the next stretch, q, into buffer i
    if (q < q1) {
#pragma unroll
      for (int m = 0; m < MT; m++) {
        wbuf[i][m][0] = __ldcs(w[m]);
        wbuf[i][m][1] = __ldcs(w[m] + 32);
        w[m] += 64;
      }
#pragma unroll
      for (int n = 0; n < NT; n++) {
#pragma unroll
        for (int s = 0; s < 4; s++) {
          // Only rows of less than whole stretches end inside one (their weights are zeros there).
          if (SEG == 128 || 128 * q + 32 * s < a.cols) xbuf[i][n][s] = __ldg(reinterpret_cast<const uint2 *>(x[n] + 32 * s));
        }
        x[n] += 128;
      }
    }
  };
  if (SEG < 128)
#pragma unroll
    for (int i = 0; i < AHEAD; i++)
#pragma unroll
      for (int n = 0; n < NT; n++) xbuf[i][n][0] = xbuf[i][n][1] = xbuf[i][n][2] = xbuf[i][n][3] = make_uint2(0, 0);
#pragma unroll
  for (int i = 0; i < AHEAD; i++) fetch(i, q0 + i);

  const int groups = a.cols / a.group, xgroups = a.cols / a.x_group;
  const W4Smem lay = w4_smem(a, MT, NT);
  const int es = a.scale_type == RK_ACT_F32 ? 4 : 2;
  char *mine = sm + warp * bufs * lay.size;
  auto stage = [&](int q, char *to) {  // the scales of the chunk from stretch q on
    if (q < q1) {
      const int col = 128 * q, last = min(128 * min(q + kW4Chunk / 128, q1), a.cols) - 1;
      const int g0 = col / a.group, ng = last / a.group - g0 + 1;
#pragma unroll
      for (int m = 0; m < MT; m++) {
        const char *src = static_cast<const char *>(a.scales) + ((int64_t)tile[m] * groups + g0) * 16 * es;
        for (int i = lane; i < ng * es; i += 32) w4_copy16(to + (m * ng * es + i) * 16, src + 16 * i);
        if (ZEROS)
          for (int i = lane; i < ng; i += 32)
            w4_copy16(to + lay.zeros + (m * ng + i) * 16, a.zeros + ((int64_t)tile[m] * groups + g0 + i) * 16);
      }
      const int x0 = col / a.x_group, nx = last / a.x_group - x0 + 1;
      for (int j = c; j < nx; j += 4)
#pragma unroll
        for (int n = 0; n < NT; n++)
          w4_copy4(to + lay.x + (j * 8 * NT + 8 * n + r) * 4, a.x_scales + (int64_t)min(v0 + 8 * n + r, a.n - 1) * xgroups + x0 + j);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  stage(q0, mine);

  float acc[MT][NT][4] = {};
  int buf = 0;
  for (int qc = q0; qc < q1; qc += kW4Chunk / 128) {
    const int qn = min(q1, qc + kW4Chunk / 128);
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncwarp();
    const char *now = mine + buf * lay.size;
    if (bufs > 1) {
      buf ^= 1;
      stage(qn, mine + buf * lay.size);
    }
    // Where the chunk's columns lie in their groups.
    const int col0 = 128 * qc, ng = (min(128 * qn, a.cols) - 1) / a.group - col0 / a.group + 1;
    int g_left = a.group - col0 % a.group, x_left = a.x_group - col0 % a.x_group;
    const char *sw_at = now + r * es, *z_at = now + lay.zeros + r, *sx_at = now + lay.x + 8 * c;

    for (int qb = qc; qb < qn; qb += AHEAD) {
#pragma unroll
      for (int i = 0; i < AHEAD; i++) {
        const int q = qb + i;
        if (q >= qn) break;
        int sum[MT][NT][4], ones[NT][4];
#pragma unroll
        for (int s = 0; s < 4; s++) {
          if (SEG < 128 && 128 * q + 32 * s >= a.cols) break;
          const bool first = s * 32 % SEG == 0, last = (s + 1) * 32 % SEG == 0;
          if (first) {
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
              for (int e = 0; e < 4; e++) {
                ones[n][e] = 0;
#pragma unroll
                for (int m = 0; m < MT; m++) sum[m][n][e] = 0;
              }
          }
#pragma unroll
          for (int m = 0; m < MT; m++) {
            const uint4 cw = wbuf[i][m][s >> 1];
            const uint32_t p = s & 1 ? cw.z : cw.x, u = s & 1 ? cw.w : cw.y;
            const uint32_t a0 = (p << 4) & 0xf0f0f0f0u, a2 = p & 0xf0f0f0f0u;
            const uint32_t a1 = (u << 4) & 0xf0f0f0f0u, a3 = u & 0xf0f0f0f0u;
#pragma unroll
            for (int n = 0; n < NT; n++) imma(sum[m][n], a0, a1, a2, a3, xbuf[i][n][s].x, xbuf[i][n][s].y);
          }
          if (ZEROS)
#pragma unroll
            for (int n = 0; n < NT; n++)
              imma(ones[n], 0x10101010u, 0x10101010u, 0x10101010u, 0x10101010u, xbuf[i][n][s].x, xbuf[i][n][s].y);
          if (last) {  // a segment ends
            float2 sx[NT];
#pragma unroll
            for (int n = 0; n < NT; n++) sx[n] = *reinterpret_cast<const float2 *>(sx_at + 32 * n);
#pragma unroll
            for (int m = 0; m < MT; m++) {
              const char *sp = sw_at + m * ng * 16 * es;
              const float sw[2] = {w4_scale(sp, a.scale_type, 0) * 0.0625f, w4_scale(sp, a.scale_type, 8) * 0.0625f};
              int z[2] = {0, 0};
              if (ZEROS) {
                z[0] = 8 - (int)*reinterpret_cast<const uint8_t *>(z_at + m * ng * 16);
                z[1] = 8 - (int)*reinterpret_cast<const uint8_t *>(z_at + m * ng * 16 + 8);
              }
#pragma unroll
              for (int n = 0; n < NT; n++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                  const int v = ZEROS ? sum[m][n][e] + z[e >> 1] * ones[n][e] : sum[m][n][e];
                  acc[m][n][e] = fmaf((float)v, sw[e >> 1] * (e & 1 ? sx[n].y : sx[n].x), acc[m][n][e]);
                }
            }
            if ((g_left -= SEG) == 0) sw_at += 16 * es, z_at += 16, g_left = a.group;
            if ((x_left -= SEG) == 0) sx_at += 32 * NT, x_left = a.x_group;
          }
        }
        fetch(i, q + AHEAD);
      }
    }
  }

  // The warps' sums, in order, then the cluster's CTAs', in order.
  __syncthreads();
  float *part = reinterpret_cast<float *>(sm);  // [warps][rows][vectors]
  constexpr int TILE = 16 * MT * 8 * NT;
#pragma unroll
  for (int m = 0; m < MT; m++)
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int e = 0; e < 4; e++)
        part[warp * TILE + (16 * m + r + 8 * (e >> 1)) * 8 * NT + 8 * n + 2 * c + (e & 1)] = acc[m][n][e];
  __syncthreads();
  const int all = TILE * (kW4Warps >> log_kw);
  for (int i = threadIdx.x; i < all; i += 32 * kW4Warps) {
    const int at = (i / TILE << log_kw) * TILE + i % TILE;
    float v = part[at];
    for (int k = 1; k < kw; k++) v += part[at + k * TILE];
    part[at] = v;
  }
  if (split > 1) cg::this_cluster().sync();
  else __syncthreads();
  if (rank == 0) {
    for (int i = threadIdx.x; i < all; i += 32 * kW4Warps) {
      // Neighbouring threads store neighbouring rows of a vector.
      const int row = i % (16 * MT), vec = i / (16 * MT) % (8 * NT), t = i / TILE;
      const int at = (t << log_kw) * TILE + row * 8 * NT + vec;
      float v = part[at];
      for (int k = 1; k < split; k++) v += cg::this_cluster().map_shared_rank(part, k)[at];
      const int64_t to = (int64_t)(cta_tile0 + t * MT) * 16 + row;
      if (to < a.rows && v0 + vec < a.n) act_store(static_cast<T *>(a.out) + (int64_t)(v0 + vec) * a.out_stride + to, v);
    }
  }
  if (split > 1) cg::this_cluster().sync();  // a member's shared memory stays until it has been read
}

template <int MT, int NT, int SEG, bool ZEROS>
static cudaError_t w4_run(const W4Args &a, int type, int split, int log_kw, cudaStream_t st) {
  const int quads = (a.cols + 127) / 128, tiles = (a.rows + 15) / 16;
  const int per_cta = (kW4Warps >> log_kw) * MT;
  const dim3 grid((unsigned)((tiles + per_cta - 1) / per_cta * split), (unsigned)((a.n + 8 * NT - 1) / (8 * NT)));
  const dim3 cl(split, 1, 1);
  // One buffer of scales where a chunk takes the longest share.
  const int64_t shares = split << log_kw;
  const int bufs = (quads + shares - 1) / shares * 128 <= kW4Chunk ? 1 : 2;
  const size_t stage = (size_t)kW4Warps * bufs * w4_smem(a, MT, NT).size, part = (size_t)kW4Warps * 16 * MT * 8 * NT * 4;
  const size_t smem = stage > part ? stage : part;
  switch (type) {
    case RK_ACT_F32: return launch_kc(k_w4<MT, NT, SEG, ZEROS, float>, grid, 32 * kW4Warps, cl, smem, st, a, quads, split, log_kw, bufs);
    case RK_ACT_F16: return launch_kc(k_w4<MT, NT, SEG, ZEROS, __half>, grid, 32 * kW4Warps, cl, smem, st, a, quads, split, log_kw, bufs);
    default:
      return launch_kc(k_w4<MT, NT, SEG, ZEROS, __nv_bfloat16>, grid, 32 * kW4Warps, cl, smem, st, a, quads, split, log_kw, bufs);
  }
}

template <int MT, int NT>
static cudaError_t w4_seg(const W4Args &a, int type, int split, int log_kw, cudaStream_t st) {
  const int seg = a.group % 128 == 0 && a.x_group % 128 == 0 ? 128 : a.group % 64 == 0 && a.x_group % 64 == 0 ? 64 : 32;
  if (a.zeros) {
    if (seg == 128) return w4_run<MT, NT, 128, true>(a, type, split, log_kw, st);
    if (seg == 64) return w4_run<MT, NT, 64, true>(a, type, split, log_kw, st);
    return w4_run<MT, NT, 32, true>(a, type, split, log_kw, st);
  }
  if (seg == 128) return w4_run<MT, NT, 128, false>(a, type, split, log_kw, st);
  if (seg == 64) return w4_run<MT, NT, 64, false>(a, type, split, log_kw, st);
  return w4_run<MT, NT, 32, false>(a, type, split, log_kw, st);
}

cudaError_t launch_w4_mulvec(const W4Args &a, int type, int sms, cudaStream_t st) {
  const int tiles = (a.rows + 15) / 16;
  // More than 8 vectors: two tiles of 16 rows share a warp's vectors and
  // their scales.
  const int mt = a.n > 8 ? 2 : 1;
  // Shares of the columns until every SM has sixteen warps, as long as a warp
  // keeps 256 columns.
  const int64_t units = (tiles + mt - 1) / mt;
  int log_kw = 0, split = 1;
  const auto more = [&] { return (units * split << log_kw) < 16 * sms && a.cols / (split * 2 << log_kw) >= 256; };
  while (log_kw < 3 && more()) log_kw++;
  while (log_kw == 3 && split < 8 && more()) split *= 2;
  const int64_t width = 65535LL * 8;  // of grid.y
  for (int64_t v = 0; v < a.n; v += width) {
    W4Args b = a;
    b.n = (int)(a.n - v < width ? a.n - v : width);
    b.x += v * a.cols;
    b.x_scales += v * (a.cols / a.x_group);
    b.out = static_cast<char *>(a.out) + v * a.out_stride * (type == RK_ACT_F32 ? 4 : 2);
    const cudaError_t e = mt == 2 ? w4_seg<2, 2>(b, type, split, log_kw, st) : w4_seg<1, 1>(b, type, split, log_kw, st);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

// The most shared memory of any matrix: float32 scales of groups of 32, two buffers.
template <int MT, int NT, int SEG, bool ZEROS>
static cudaError_t w4_attr() {
  const int most = kW4Warps * 2 * (kW4Chunk / 32 * (16 * MT * (4 + ZEROS) + 8 * NT * 4));
  const cudaFuncAttribute at = cudaFuncAttributeMaxDynamicSharedMemorySize;
  cudaError_t e = cudaFuncSetAttribute(k_w4<MT, NT, SEG, ZEROS, float>, at, most);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(k_w4<MT, NT, SEG, ZEROS, __half>, at, most);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(k_w4<MT, NT, SEG, ZEROS, __nv_bfloat16>, at, most);
  return e;
}
template <int MT, int NT>
static cudaError_t w4_attrs() {
  cudaError_t e = w4_attr<MT, NT, 32, false>();
  if (e == cudaSuccess) e = w4_attr<MT, NT, 64, false>();
  if (e == cudaSuccess) e = w4_attr<MT, NT, 128, false>();
  if (e == cudaSuccess) e = w4_attr<MT, NT, 32, true>();
  if (e == cudaSuccess) e = w4_attr<MT, NT, 64, true>();
  if (e == cudaSuccess) e = w4_attr<MT, NT, 128, true>();
  return e;
}

cudaError_t init_w4_attributes() {
  const cudaError_t e = w4_attrs<1, 1>();
  return e != cudaSuccess ? e : w4_attrs<2, 2>();
}

}  // namespace rk
