// rk_w4.cu — products of a 4-bit matrix with group scales and 8-bit vectors.
//
//   out[v][row] = Σ over segments  sw · sx · Σ_k (u_k − z) x_k
// A segment is a run of columns with one weight scale and one vector scale.
// Up to 16 vectors the bytes of the weights bound the product (half a byte a
// weight), so what a warp does for them has to stay below an SM's share of
// the memory bandwidth: about 180 instructions for a KB. The sums run on
// mma.m16n8k32 on signed bytes (16 rows, 8 vectors; one vector fills one
// column, the others ride along), exact in int32.
//
// Layout. At upload the matrix becomes a stream of records, one for each tile
// of 16 rows and stretch of 128 columns: 1 KB of weights in the order in which
// a warp's lanes hold the operand, then the scales (and zero points) of the
// stretch's segments, repeated where a group is wider, so that a record is
// one contiguous copy and needs no arithmetic on groups. Weights are two's
// complement nibbles of u − 8: the upper half of a byte, its lower half masked
// away, is then 16 (u − 8) as a signed byte, so unpacking eight weights takes
// three instructions, and the 16 goes into the vectors' scales. A zero point
// other than 8 adds (8 − z) · 16 Σ x, with Σ x made once for each segment.
//
// Work. One CTA of sixteen warps an SM goes through tiles of 16 rows. KW warps
// of it (a team) share a tile's columns, or a cluster's CTAs do where there
// are few rows; each warp keeps its share of the columns from tile to tile, so
// the vectors and their scales are brought into shared memory once. The
// records come through a ring of each warp in shared memory, which runs on
// over the tiles: no load waits for a tile's end. (A CTA for each tile took
// 22.3 us for 28672x4096 by one vector: its beginning and end cost as much as
// ten column pairs a warp, and the last wave of CTAs left SMs idle.) The
// float32 sums of a tile's shares meet in shared memory, in order, while the
// warps are at the next tile.
#include "rk_act.cuh"
#include "rk_serve.cuh"

namespace rk {

constexpr int kW4Warps = 16;
constexpr int kW4Smem = 227 * 1024;

// Columns of the weights' segments, of both's.
static int w4_width(int group) { return group % 128 == 0 ? 128 : group % 64 == 0 ? 64 : 32; }
static int w4_segment(const W4Args &a) {
  const int w = w4_width(a.group), x = w4_width(a.x_group);
  return w < x ? w : x;
}
// Bytes of a segment's scales in a record: for r < 8, rows r and r + 8, each
// the scale (and 8 − z: in the upper half of a 16-bit scale's word, or in a
// word of its own).
__host__ __device__ constexpr int w4_entry(bool s32, bool zeros) { return 32 * (s32 ? 2 : 1) * (zeros ? 2 : 1); }
static int w4_record(int group, bool s32, bool zeros) { return 1024 + 128 / w4_width(group) * w4_entry(s32, zeros); }
int64_t w4_bytes(int rows, int cols, int group, int scale_type, bool zeros) {
  return (int64_t)((rows + 15) / 16) * ((cols + 127) / 128) * w4_record(group, scale_type == RK_ACT_F32, zeros);
}

// The stream from the caller's order, a word a thread. Rows are padded to 16
// and columns to 128 with zeros. Word `word` of lane (r, c) in 64 columns has
// the nibbles of row r + 8 (word % 2) and step s = word / 2 of 32 columns: low
// halves columns 8c .. 8c + 3 of the step, high halves 8c + 4 .. 8c + 7, so
// that a lane's vector bytes are eight neighbours.
__global__ void k_w4_stream(const uint8_t *w, const void *scales, const uint8_t *zeros, int rows, int cols, int group, bool s32,
                            int width, int record, uint32_t *out, int64_t words) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= words) return;
  const int quads = (cols + 127) / 128;
  const int64_t rec = i / (record / 4), tile = rec / quads;
  const int q = (int)(rec % quads), at = (int)(i % (record / 4));
  uint32_t v = 0;
  if (at < 256) {
    const int word = at & 3, lane = (at >> 2) & 31, r = lane >> 2, c = lane & 3;
    const int64_t row = tile * 16 + r + 8 * (word & 1);
    if (row < rows)
      for (int b = 0; b < 8; b++) {
        const int col = 128 * q + 64 * (at >> 7) + 32 * (word >> 1) + 8 * c + b;
        if (col >= cols) break;
        const uint8_t x = w[row * (cols / 2) + (col / 32) * 16 + col % 16];  // columns j and j + 16 of a block share byte j
        const uint32_t u = (col % 32 < 16 ? x & 15 : x >> 4) ^ 8;
        v |= u << (b < 4 ? 8 * b : 8 * (b - 4) + 4);
      }
  } else {
    const int per_row = (s32 ? 4 : 2) + (zeros ? (s32 ? 4 : 2) : 0);  // bytes
    const int byte = 4 * (at - 256), entry = byte / (16 * per_row), in = byte % (16 * per_row);
    const int col = 128 * q + width * entry;
    const auto row_of = [&](int b) { return tile * 16 + b / (2 * per_row) + 8 * (b / per_row % 2); };
    const auto group_at = [&](int64_t row) { return row * (cols / group) + col / group; };
    if (col < cols) {
      if (s32) {
        const int64_t row = row_of(in);
        if (row < rows)
          v = in % per_row == 0 ? static_cast<const uint32_t *>(scales)[group_at(row)] : (uint32_t)(8 - (int)zeros[group_at(row)]);
      } else if (zeros) {
        const int64_t row = row_of(in);
        if (row < rows)
          v = static_cast<const uint16_t *>(scales)[group_at(row)] | (uint32_t)(8 - (int)zeros[group_at(row)]) << 16;
      } else {
        for (int h = 0; h < 2; h++) {
          const int64_t row = row_of(in + 2 * h);
          if (row < rows) v |= (uint32_t)static_cast<const uint16_t *>(scales)[group_at(row)] << (16 * h);
        }
      }
    }
  }
  out[i] = v;
}

cudaError_t launch_w4_stream(const uint8_t *w, const void *scales, const uint8_t *zeros, int rows, int cols, int group,
                             int scale_type, uint8_t *out, cudaStream_t st) {
  const bool s32 = scale_type == RK_ACT_F32;
  const int64_t words = w4_bytes(rows, cols, group, scale_type, zeros != nullptr) / 4;
  return launch_k(k_w4_stream, dim3((unsigned)((words + 255) / 256)), 256, 0, st, w, scales, zeros, rows, cols, group, s32,
                  w4_width(group), w4_record(group, s32, zeros != nullptr), reinterpret_cast<uint32_t *>(out), words);
}

RK_DEV void imma(int *c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The same from sums of zero.
RK_DEV void imma_first(int *c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(0));
}

// Shared memory by 32-bit addresses.
RK_DEV uint32_t s_addr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
RK_DEV uint32_t lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a));
  return v;
}
RK_DEV uint2 lds64(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
  return v;
}
RK_DEV uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
RK_DEV void copy16_s(uint32_t dst, const void *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
RK_DEV void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
RK_DEV void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// Stores v at `to` (an address in this CTA's shared memory) of the cluster's first CTA.
RK_DEV void store_first(uint32_t to, float v) {
  asm volatile(
      "{\n\t.reg .b32 p;\n\t"
      "mapa.shared::cluster.u32 p, %0, 0;\n\t"
      "st.shared::cluster.f32 [p], %1;\n\t}" ::"r"(to),
      "f"(v)
      : "memory");
}

// How a product is dealt out, and its shared memory.
struct W4Plan {
  int quads;      // stretches of 128 columns
  int log_kw;     // log2 of the warps of a team
  int split;      // CTAs of a cluster, which share a tile's columns (then teams are whole CTAs)
  int teams;      // of all CTAs or clusters
  int cta_quads;  // stretches of a CTA, at most
  int x_stride;   // bytes between vectors in shared memory; 0: they stay in global memory
  int record, log_width;  // of the stream: bytes of a record, log2 of a segment's columns
  int at_xs, at_ring, at_part, at_far, size;
};
// Stages of a warp's ring.
__host__ __device__ constexpr int w4_depth(int nt) { return nt > 1 ? 3 : 4; }

// NT tiles of 8 vectors; SEG columns share their scales; XS: the vectors lie
// in shared memory; S32: float32 scales.
template <int NT, int SEG, bool ZEROS, bool XS, bool S32>
__global__ void __launch_bounds__(32 * kW4Warps, 1) k_w4(W4Args a, W4Plan p, int out_type) {
  constexpr int DEPTH = w4_depth(NT), TILE = 16 * 8 * NT, SEGS = 128 / SEG, ENTRY = w4_entry(S32, ZEROS);
  constexpr int XSB = ZEROS ? 8 : 4;  // bytes of a vector's entry for a segment: its scale / 16 (and 16 Σ x)
  extern __shared__ __align__(128) char sm[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = lane >> 2, c = lane & 3;
  const int kw = 1 << p.log_kw, tiles = (a.rows + 15) / 16;
  const int rank = blockIdx.x & (p.split - 1);
  const int team = p.split > 1 ? blockIdx.x / p.split : blockIdx.x * (kW4Warps >> p.log_kw) + (warp >> p.log_kw);
  const int v0 = blockIdx.y * 8 * NT, nv = min(8 * NT, a.n - v0);
  // The CTA's columns, and this warp's.
  const int cq0 = p.quads * rank / p.split, cq1 = p.quads * (rank + 1) / p.split;
  const int share = warp & (kw - 1);
  const int q0 = cq0 + (((cq1 - cq0) * share) >> p.log_kw), q1 = cq0 + (((cq1 - cq0) * (share + 1)) >> p.log_kw);

  // The ring. Records left to copy, and left of the tile's share.
  const int len = q1 - q0, my_tiles = team < tiles ? (tiles - 1 - team) / p.teams + 1 : 0;
  const uint32_t ring = s_addr(sm) + p.at_ring + warp * DEPTH * p.record, ring_end = ring + DEPTH * p.record;
  int c_left = len * my_tiles, c_tile = len;
  uint32_t c_to = ring + 16 * lane;
  const uint8_t *c_from = a.w + ((int64_t)team * p.quads + q0) * p.record + 16 * lane;
  const int64_t c_jump = ((int64_t)p.teams * p.quads - len) * p.record;
  const bool c_tail = 1024 + 16 * lane < p.record;
  auto copy = [&] {
    if (c_left > 0) {
      copy16_s(c_to, c_from);
      copy16_s(c_to + 512, c_from + 512);
      if (c_tail) copy16_s(c_to + 1024, c_from + 1024);
      c_from += p.record;
      c_to += p.record;
      if (c_to >= ring_end) c_to = ring + 16 * lane;
      c_left--;
      if (--c_tile == 0) {
        c_tile = len;
        c_from += c_jump;
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < DEPTH - 1; i++) copy();

  // The CTA's columns of the vectors, and their entries: [segment][8 NT].
  const int x0 = 128 * cq0, x_cols = min(a.cols, 128 * cq1) - x0;
  if (XS)
    for (int i = threadIdx.x; i < nv * (x_cols / 16); i += 32 * kW4Warps) {
      const int v = i / (x_cols / 16), j = i % (x_cols / 16);
      *reinterpret_cast<uint4 *>(sm + v * p.x_stride + 16 * j) =
          __ldg(reinterpret_cast<const uint4 *>(a.x + (int64_t)(v0 + v) * a.cols + x0) + j);
    }
  for (int i = threadIdx.x; i < x_cols / SEG * 8 * NT; i += 32 * kW4Warps) {
    const int v = v0 + min(i % (8 * NT), nv - 1), col = x0 + SEG * (i / (8 * NT));
    const float s = __ldg(a.x_scales + (int64_t)v * (a.cols / a.x_group) + col / a.x_group) * 0.0625f;
    if (ZEROS) {
      const uint4 *at = reinterpret_cast<const uint4 *>(a.x + (int64_t)v * a.cols + col);
      int sum = 0;
#pragma unroll
      for (int k = 0; k < SEG / 16; k++) {
        const uint4 u = __ldg(at + k);
        sum = __dp4a((int)u.x, 0x10101010, sum);
        sum = __dp4a((int)u.y, 0x10101010, sum);
        sum = __dp4a((int)u.z, 0x10101010, sum);
        sum = __dp4a((int)u.w, 0x10101010, sum);
      }
      *reinterpret_cast<float2 *>(sm + p.at_xs + XSB * i) = make_float2(s, __int_as_float(sum));
    } else {
      *reinterpret_cast<float *>(sm + p.at_xs + XSB * i) = s;
    }
  }
  __syncthreads();

  // A vector behind the last is computed from the last one's, and not stored.
  uint32_t xr[NT];
  const int8_t *xg[NT];
#pragma unroll
  for (int n = 0; n < NT; n++) {
    const int v = min(8 * n + r, nv - 1);
    xr[n] = s_addr(sm) + v * p.x_stride + 128 * (q0 - cq0) + 8 * c;
    xg[n] = a.x + (int64_t)(v0 + v) * a.cols + 128 * q0 + 8 * c;
  }
  const uint32_t x_first = s_addr(sm) + p.at_xs + (q0 - cq0) * SEGS * 8 * NT * XSB + 2 * c * XSB;
  // Where a step's scales lie in a record (SEG may be narrower than the weights' segments).
  uint32_t s_at[4];
#pragma unroll
  for (int s = 0; s < 4; s++) s_at[s] = 1024 + ((32 * s) >> p.log_width) * ENTRY + r * (ENTRY / 8);
  const bool bf16 = a.scale_type == RK_ACT_BF16;
  const auto half_scale = [&](uint32_t h) { return bf16 ? u2f(h << 16) : __half2float(__ushort_as_half((unsigned short)h)); };

  float *part = reinterpret_cast<float *>(sm + p.at_part), *far = reinterpret_cast<float *>(sm + p.at_far);
  uint32_t now = ring;
  int flip = 0, far_tile = -1;
  constexpr int MINE = (TILE + 32 * kW4Warps - 1) / (32 * kW4Warps);  // of a tile's sums, where the team is the CTA
  float kept[MINE];
  // Element i of a tile's sums: neighbours are neighbouring rows of a vector.
  auto put = [&](int t, int i, float v) {
    const int64_t row = (int64_t)t * 16 + i % 16;
    const int vec = i / 16;
    if (row >= a.rows || vec >= nv) return;
    const int64_t to = (int64_t)(v0 + vec) * a.out_stride + row;
    if (out_type == RK_ACT_F32) act_store(static_cast<float *>(a.out) + to, v);
    else if (out_type == RK_ACT_F16) act_store(static_cast<__half *>(a.out) + to, v);
    else act_store(static_cast<__nv_bfloat16 *>(a.out) + to, v);
  };
  auto join_far = [&] {  // the first CTA of a cluster: the other CTAs' sums of tile far_tile have come
#pragma unroll
    for (int k = 0; k < MINE; k++) {
      const int i = threadIdx.x + k * 32 * kW4Warps;
      if (i >= TILE) break;
      float v = kept[k];
      for (int o = 1; o < p.split; o++) v += far[((flip ^ 1) * (p.split - 1) + o - 1) * TILE + i];
      put(far_tile, i, v);
    }
  };

  for (int t = team; t < tiles; t += p.teams) {
    float acc[NT][4] = {};
    uint32_t x_at = x_first, xq[NT];
    const int8_t *xp[NT];
#pragma unroll
    for (int n = 0; n < NT; n++) xq[n] = xr[n], xp[n] = xg[n];
    for (int q = q0; q < q1; q++) {
      asm volatile("cp.async.wait_group %0;" ::"n"(DEPTH - 2) : "memory");
      __syncwarp();
      copy();
      const uint4 w01 = lds128(now + 16 * lane), w23 = lds128(now + 512 + 16 * lane);
      int sum[NT][4];
#pragma unroll
      for (int s = 0; s < 4; s++) {
        if (SEG < 128 && 128 * q + 32 * s >= a.cols) break;  // rows may end inside a stretch
        const uint4 w = s < 2 ? w01 : w23;
        const uint32_t lo = s & 1 ? w.z : w.x, hi = s & 1 ? w.w : w.y;  // rows r and r + 8
        const uint32_t a0 = (lo << 4) & 0xf0f0f0f0u, a1 = (hi << 4) & 0xf0f0f0f0u, a2 = lo & 0xf0f0f0f0u, a3 = hi & 0xf0f0f0f0u;
#pragma unroll
        for (int n = 0; n < NT; n++) {
          const uint2 xv = XS ? lds64(xq[n] + 32 * s) : __ldg(reinterpret_cast<const uint2 *>(xp[n] + 32 * s));
          if (s * 32 % SEG == 0) imma_first(sum[n], a0, a1, a2, a3, xv.x, xv.y);
          else imma(sum[n], a0, a1, a2, a3, xv.x, xv.y);
        }
        if ((s + 1) * 32 % SEG == 0) {  // a segment ends
          float sw[2];
          int z[2] = {0, 0};
          if constexpr (S32 && ZEROS) {
            const uint4 e = lds128(now + s_at[s]);
            sw[0] = u2f(e.x), z[0] = (int)e.y, sw[1] = u2f(e.z), z[1] = (int)e.w;
          } else if constexpr (S32) {
            const uint2 e = lds64(now + s_at[s]);
            sw[0] = u2f(e.x), sw[1] = u2f(e.y);
          } else if constexpr (ZEROS) {
            const uint2 e = lds64(now + s_at[s]);
            sw[0] = half_scale(e.x & 0xffff), z[0] = (int)e.x >> 16, sw[1] = half_scale(e.y & 0xffff), z[1] = (int)e.y >> 16;
          } else {
            const uint32_t e = lds32(now + s_at[s]);
            sw[0] = half_scale(e & 0xffff), sw[1] = half_scale(e >> 16);
          }
#pragma unroll
          for (int n = 0; n < NT; n++) {
            float f[2];  // of vectors 2c and 2c + 1
            if constexpr (ZEROS) {
              const uint4 e = lds128(x_at + 8 * n * XSB);
              f[0] = u2f(e.x), f[1] = u2f(e.z);
              sum[n][0] += z[0] * (int)e.y;
              sum[n][1] += z[0] * (int)e.w;
              sum[n][2] += z[1] * (int)e.y;
              sum[n][3] += z[1] * (int)e.w;
            } else {
              const uint2 e = lds64(x_at + 8 * n * XSB);
              f[0] = u2f(e.x), f[1] = u2f(e.y);
            }
#pragma unroll
            for (int e = 0; e < 4; e++) acc[n][e] = fmaf((float)sum[n][e], sw[e >> 1] * f[e & 1], acc[n][e]);
          }
          x_at += 8 * NT * XSB;
        }
      }
#pragma unroll
      for (int n = 0; n < NT; n++) xq[n] += 128, xp[n] += 128;
      now += p.record;
      if (now == ring_end) now = ring;
    }
    // The team's sums: one barrier a tile, since the next tile's go to the
    // other half, and are read behind the next barrier.
    float *mine = part + (flip * kW4Warps + warp) * TILE;
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int e = 0; e < 4; e++) mine[(8 * n + 2 * c + (e & 1)) * 16 + r + 8 * (e >> 1)] = acc[n][e];
    if (p.log_kw == 0) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(warp >> p.log_kw), "r"(32 << p.log_kw) : "memory");
    const float *first = part + (flip * kW4Warps + (warp & ~(kw - 1))) * TILE;
    if (p.split == 1) {
      for (int i = share * 32 + lane; i < TILE; i += 32 << p.log_kw) {
        float v = first[i];
        for (int k = 1; k < kw; k++) v += first[k * TILE + i];
        put(t, i, v);
      }
      flip ^= 1;
    } else {
      float here[MINE];
#pragma unroll
      for (int k = 0; k < MINE; k++) {
        const int i = threadIdx.x + k * 32 * kW4Warps;
        here[k] = 0.0f;
        if (i < TILE) {
          here[k] = first[i];
          for (int o = 1; o < kw; o++) here[k] += first[o * TILE + i];
        }
      }
      // The other CTAs' sums of the tile before have come: they are waited for a tile late.
      if (far_tile >= 0) {
        cluster_wait();
        if (rank == 0) join_far();
      } else {  // every CTA of the cluster has begun, before its memory is written
        cluster_arrive();
        cluster_wait();
      }
#pragma unroll
      for (int k = 0; k < MINE; k++) {
        const int i = threadIdx.x + k * 32 * kW4Warps;
        if (rank == 0) kept[k] = here[k];
        else if (i < TILE) store_first(s_addr(far + (flip * (p.split - 1) + rank - 1) * TILE + i), here[k]);
      }
      cluster_arrive();
      far_tile = t;
      flip ^= 1;
    }
  }
  if (p.split > 1 && far_tile >= 0) {
    cluster_wait();
    if (rank == 0) join_far();
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

// Shared memory of a plan (teams, log_kw, split set); the vectors go to
// shared memory if that fits.
static void w4_layout_smem(const W4Args &a, W4Plan &p) {
  const int nt = a.n > 8 ? 2 : 1, nv = a.n < 8 * nt ? a.n : 8 * nt;
  p.cta_quads = (p.quads + p.split - 1) / p.split;
  const int xs = (128 * p.cta_quads / w4_segment(a) * 8 * nt * (a.zeros ? 8 : 4) + 127) / 128 * 128;
  const int ring = (kW4Warps * w4_depth(nt) * p.record + 127) / 128 * 128;
  const int part = 2 * kW4Warps * 16 * 8 * nt * 4, far = 2 * (p.split - 1) * 16 * 8 * nt * 4;
  p.x_stride = 128 * p.cta_quads + 32;  // rows of eight lanes' reads fall on different banks
  if ((int64_t)nv * p.x_stride + 128 + xs + ring + part + far > kW4Smem) p.x_stride = 0;
  p.at_xs = (nv * p.x_stride + 127) / 128 * 128;
  p.at_ring = p.at_xs + xs;
  p.at_part = p.at_ring + ring;
  p.at_far = p.at_part + part;
  p.size = p.at_far + far;
}

// f<NT, SEG, ZEROS, XS, S32>() of the instance for a product.
template <int NT, bool XS, bool S32, class F>
static cudaError_t w4_seg(int seg, bool zeros, F f) {
  if (zeros) {
    if (seg == 128) return f.template operator()<NT, 128, true, XS, S32>();
    if (seg == 64) return f.template operator()<NT, 64, true, XS, S32>();
    return f.template operator()<NT, 32, true, XS, S32>();
  }
  if (seg == 128) return f.template operator()<NT, 128, false, XS, S32>();
  if (seg == 64) return f.template operator()<NT, 64, false, XS, S32>();
  return f.template operator()<NT, 32, false, XS, S32>();
}
template <class F>
static cudaError_t w4_at(int nt, bool xs, bool s32, int seg, bool zeros, F f) {
  if (nt > 1) {
    if (xs) return s32 ? w4_seg<2, true, true>(seg, zeros, f) : w4_seg<2, true, false>(seg, zeros, f);
    return s32 ? w4_seg<2, false, true>(seg, zeros, f) : w4_seg<2, false, false>(seg, zeros, f);
  }
  if (xs) return s32 ? w4_seg<1, true, true>(seg, zeros, f) : w4_seg<1, true, false>(seg, zeros, f);
  return s32 ? w4_seg<1, false, true>(seg, zeros, f) : w4_seg<1, false, false>(seg, zeros, f);
}

struct W4Launch {
  const W4Args &a;
  int type;
  const W4Plan &p;
  cudaStream_t st;
  template <int NT, int SEG, bool ZEROS, bool XS, bool S32>
  cudaError_t operator()() const {
    const int ctas = p.split > 1 ? p.teams * p.split : p.teams / (kW4Warps >> p.log_kw);
    const dim3 grid(ctas, (unsigned)((a.n + 8 * NT - 1) / (8 * NT))), cl(p.split, 1, 1);
    return launch_kc(k_w4<NT, SEG, ZEROS, XS, S32>, grid, 32 * kW4Warps, cl, p.size, st, a, p, type);
  }
};

cudaError_t launch_w4_mulvec(const W4Args &a, int type, int sms, cudaStream_t st) {
  const int tiles = (a.rows + 15) / 16;
  const bool s32 = a.scale_type == RK_ACT_F32;
  W4Plan best{};
  double least = 0;
  // The time of a plan in stretches: a team's tiles, each its longest share and
  // an end (about two stretches' instructions; another four for the exchange in
  // a cluster); vectors that stay in global memory take four times as long.
  const auto take = [&](int log_kw, int split) {
    W4Plan p{};
    p.quads = (a.cols + 127) / 128;
    p.log_kw = log_kw;
    p.split = split;
    p.record = w4_record(a.group, s32, a.zeros);
    p.log_width = w4_width(a.group) == 128 ? 7 : w4_width(a.group) == 64 ? 6 : 5;
    w4_layout_smem(a, p);
    if (p.size > kW4Smem) return;
    const int units = split > 1 ? sms / split : sms * (kW4Warps >> log_kw);
    const int rounds = (tiles + units - 1) / units;
    const int share = (p.cta_quads + (1 << log_kw) - 1) >> log_kw;
    const double cost = rounds * (share * (p.x_stride ? 1.0 : 4.0) + 2 + (split > 1 ? 4 : 0));
    const int per_cta = kW4Warps >> log_kw;
    p.teams = split > 1 ? (tiles < units ? tiles : units) : (tiles < units ? (tiles + per_cta - 1) / per_cta * per_cta : units);
    if (least == 0 || cost < least) {
      least = cost;
      best = p;
    }
  };
  for (int k = 4; k >= 0; k--) take(k, 1);
  for (int s = 2; s <= 8; s *= 2) take(4, s);
  if (least == 0) return cudaErrorInvalidValue;
  const int64_t width = 65535LL * 8;  // of grid.y
  for (int64_t v = 0; v < a.n; v += width) {
    W4Args b = a;
    b.n = (int)(a.n - v < width ? a.n - v : width);
    b.x += v * a.cols;
    b.x_scales += v * (a.cols / a.x_group);
    b.out = static_cast<char *>(a.out) + v * a.out_stride * (type == RK_ACT_F32 ? 4 : 2);
    const cudaError_t e = w4_at(a.n > 8 ? 2 : 1, best.x_stride > 0, s32, w4_segment(a), a.zeros, W4Launch{b, type, best, st});
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

struct W4Init {
  template <int NT, int SEG, bool ZEROS, bool XS, bool S32>
  cudaError_t operator()() const {
    return cudaFuncSetAttribute(k_w4<NT, SEG, ZEROS, XS, S32>, cudaFuncAttributeMaxDynamicSharedMemorySize, kW4Smem);
  }
};

cudaError_t init_w4_attributes() {
  for (int i = 0; i < 16; i++)
    for (int seg = 32; seg <= 128; seg *= 2) {
      const cudaError_t e = w4_at(1 + (i & 1), (i & 2) != 0, (i & 4) != 0, seg, (i & 8) != 0, W4Init{});
      if (e != cudaSuccess) return e;
    }
  return cudaSuccess;
}

}  // namespace rk
