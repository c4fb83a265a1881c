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
// Work. CTAs of sixteen warps, at most one an SM, go through tiles of 16 rows.
// KW warps of a CTA (a team) share a tile's columns; each warp keeps its share
// of the columns from tile to tile, so the vectors and their scales are brought
// into shared memory once (vectors that do not fit come with each record, from
// L2, and so do scales that do not). Where teams are fewer than the SMs' warps
// each takes one tile, and whole CTAs of teams leave SMs without work: 112 of
// 148 have some at 28672x4096, 128 at 4096x14336.
// The records come through a ring of each warp in shared memory, which runs on
// over the tiles of a team: its loads do not wait for a tile's end. Sharing a tile's columns over
// the CTAs of a cluster was tried for vectors that do not fit and for few rows:
// the exchange cost 1 to 3 us a tile. (A CTA for each tile took
// 22.3 us for 28672x4096 by one vector: its beginning and end cost as much as
// ten column pairs a warp, and the last wave of CTAs left SMs idle.) The
// float32 sums of a tile's shares meet in shared memory, in order, while the
// warps are at the next tile.
// 28672x4096 takes 14.4 us by one vector (4.3 TB/s; some 4 us are the launch,
// the vectors and the only tile's end, the rest 112 SMs' streams), 128256x4096 44.4 us (6.1 TB/s, 0.93 of a plain
// copy's rate), 4096x14336 by 16 vectors in groups of 32 15.8 us.
#include "rk_act.cuh"
#include "rk_serve.cuh"
#include "rk_warp.cuh"

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

RK_DEV uint32_t s_addr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
RK_DEV void copy4_s(uint32_t dst, const void *src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
// How a product is dealt out, and its shared memory.
struct W4Plan {
  int quads;      // stretches of 128 columns
  int log_kw;     // log2 of the warps of a team
  int teams;      // of all CTAs
  int vectors;    // W4_KEPT, ...
  int x_stride;   // bytes between kept vectors
  int record, log_width;  // of the stream: bytes of a record, log2 of a segment's columns
  int stage;      // bytes of a ring stage: a record, and the vectors' columns that come with it
  int at_xs, at_ring, at_part, size;
};
// Stages of a warp's ring.
__host__ __device__ constexpr int w4_depth(int nt) { return nt > 1 ? 3 : 4; }

// Where the vectors lie: in shared memory, or they come with the records, or
// their scales do too.
enum { W4_KEPT = 2, W4_PASSING = 1, W4_ALL_PASSING = 0 };

// NT tiles of 8 vectors; SEG columns share their scales; S32: float32 scales.
template <int NT, int SEG, bool ZEROS, int VECTORS, bool S32>
__global__ void __launch_bounds__(32 * kW4Warps, 1) k_w4(W4Args a, W4Plan p, int out_type) {
  constexpr int DEPTH = w4_depth(NT), TILE = 16 * 8 * NT, SEGS = 128 / SEG, ENTRY = w4_entry(S32, ZEROS);
  constexpr bool XS = VECTORS == W4_KEPT, ENTRIES = VECTORS != W4_ALL_PASSING, SUMS = ZEROS && ENTRIES;
  constexpr int XSB = SUMS ? 8 : 4;  // bytes of a vector's entry for a segment: its scale / 16 (and 16 Σ x)
  extern __shared__ __align__(128) char sm[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = lane >> 2, c = lane & 3;
  const int kw = 1 << p.log_kw, tiles = (a.rows + 15) / 16;
  const int team = blockIdx.x * (kW4Warps >> p.log_kw) + (warp >> p.log_kw);
  const int v0 = blockIdx.y * 8 * NT, nv = min(8 * NT, a.n - v0);
  const int share = warp & (kw - 1);  // this warp's columns
  const int q0 = (p.quads * share) >> p.log_kw, q1 = (p.quads * (share + 1)) >> p.log_kw;

  // The ring. Records left to copy, and left of the tile's share.
  const int len = q1 - q0, my_tiles = team < tiles ? (tiles - 1 - team) / p.teams + 1 : 0;
  const uint32_t ring = s_addr(sm) + p.at_ring + warp * DEPTH * p.stage, ring_end = ring + DEPTH * p.stage;
  int c_left = len * my_tiles, c_tile = len;
  uint32_t c_to = ring + 16 * lane;
  const uint8_t *c_from = a.w + ((int64_t)team * p.quads + q0) * p.record + 16 * lane;
  const int64_t c_jump = ((int64_t)p.teams * p.quads - len) * p.record;
  const bool c_tail = 1024 + 16 * lane < p.record;
  // Vectors that come with the records: 16-byte piece lane % 8 of vector lane / 8 + 4i.
  const int8_t *c_x = a.x + (int64_t)(v0 + (lane >> 3)) * a.cols + 128 * q0 + 16 * (lane & 7);
  const uint32_t c_xto = p.record + (lane >> 3) * 128 + 16 * ((lane & 7) ^ (((lane >> 3) & 3) << 1)) - 16 * lane;
  const bool c_tail_x = SEG < 128 && 128 * (q1 - 1) + 16 * (lane & 7) >= a.cols;  // behind the row's end in its last stretch
  auto copy = [&] {
    if (c_left > 0) {
      copy16(c_to, c_from);
      copy16(c_to + 512, c_from + 512);
      if (c_tail) copy16(c_to + 1024, c_from + 1024);
      if (!XS) {
#pragma unroll
        for (int i = 0; i < 2 * NT; i++)
          if ((lane >> 3) + 4 * i < nv && !(c_tile == 1 && c_tail_x)) copy16(c_to + c_xto + 512 * i, c_x + (int64_t)4 * i * a.cols);
        c_x += 128;
        if (c_tile == 1) c_x -= 128 * len;
      }
      if (!ENTRIES) {
        const int col = 128 * (q1 - c_tile);
#pragma unroll
        for (int i = lane; i < SEGS * 8 * NT; i += 32) {
          const int v = i % (8 * NT), at = col + SEG * (i / (8 * NT));
          if (v < nv && at < a.cols)
            copy4_s(c_to - 16 * lane + p.stage - SEGS * 8 * NT * 4 + 4 * i,
                    a.x_scales + (int64_t)(v0 + v) * (a.cols / a.x_group) + at / a.x_group);
        }
      }
      c_from += p.record;
      c_to += p.stage;
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

  // The vectors, and their entries: [segment][8 NT].
  if (XS)
    for (int i = threadIdx.x; i < nv * (a.cols / 16); i += 32 * kW4Warps) {
      const int v = i / (a.cols / 16), j = i % (a.cols / 16);
      *reinterpret_cast<uint4 *>(sm + v * p.x_stride + 16 * j) =
          __ldg(reinterpret_cast<const uint4 *>(a.x + (int64_t)(v0 + v) * a.cols) + j);
    }
  for (int i = threadIdx.x; ENTRIES && i < a.cols / SEG * 8 * NT; i += 32 * kW4Warps) {
    const int v = v0 + min(i % (8 * NT), nv - 1), col = SEG * (i / (8 * NT));
    const float s = __ldg(a.x_scales + (int64_t)v * (a.cols / a.x_group) + col / a.x_group) * 0.0625f;
    if (SUMS) {
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

  // A vector behind the last is computed from the last one's (or from what
  // lies in the ring), and not stored.
  uint32_t xr[NT], x_step[4];
#pragma unroll
  for (int n = 0; n < NT; n++)
    xr[n] = XS ? s_addr(sm) + min(8 * n + r, nv - 1) * p.x_stride + 128 * q0 + 8 * c : p.record + (8 * n + r) * 128 + 8 * (c & 1);
#pragma unroll
  for (int s = 0; s < 4; s++) x_step[s] = XS ? 32 * s : 16 * ((2 * s + (c >> 1)) ^ ((r & 3) << 1));
  const uint32_t x_first = s_addr(sm) + p.at_xs + q0 * SEGS * 8 * NT * XSB + 2 * c * XSB;
  // Where a step's scales lie in a record (SEG may be narrower than the weights' segments).
  uint32_t s_at[4];
#pragma unroll
  for (int s = 0; s < 4; s++) s_at[s] = 1024 + ((32 * s) >> p.log_width) * ENTRY + r * (ENTRY / 8);
  const bool bf16 = a.scale_type == RK_ACT_BF16;
  const auto half_scale = [&](uint32_t h) { return bf16 ? u2f(h << 16) : __half2float(__ushort_as_half((unsigned short)h)); };

  float *part = reinterpret_cast<float *>(sm + p.at_part);
  uint32_t now = ring;
  int flip = 0;
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

  for (int t = team; t < tiles; t += p.teams) {
    float acc[NT][4] = {};
    uint32_t x_now = 0, x_at = x_first;
    for (int q = q0; q < q1; q++) {
      asm volatile("cp.async.wait_group %0;" ::"n"(DEPTH - 2) : "memory");
      __syncwarp();
      copy();
      const uint4 w01 = lds128(now + 16 * lane), w23 = lds128(now + 512 + 16 * lane);
      if (!ENTRIES) x_at = now + p.stage - SEGS * 8 * NT * 4 + 8 * c;
      int sum[NT][4], ones[NT][4];
#pragma unroll
      for (int s = 0; s < 4; s++) {
        if (SEG < 128 && 128 * q + 32 * s >= a.cols) break;  // rows may end inside a stretch
        const uint4 w = s < 2 ? w01 : w23;
        const uint32_t lo = s & 1 ? w.z : w.x, hi = s & 1 ? w.w : w.y;  // rows r and r + 8
        const uint32_t a0 = (lo << 4) & 0xf0f0f0f0u, a1 = (hi << 4) & 0xf0f0f0f0u, a2 = lo & 0xf0f0f0f0u, a3 = hi & 0xf0f0f0f0u;
#pragma unroll
        for (int n = 0; n < NT; n++) {
          const uint2 xv = lds64((XS ? x_now : now) + xr[n] + x_step[s]);
          if (s * 32 % SEG == 0) mma16832_first(sum[n], {a0, a1, a2, a3}, xv.x, xv.y);
          else mma16832(sum[n], {a0, a1, a2, a3}, xv.x, xv.y);
          if constexpr (ZEROS && !ENTRIES) {
            constexpr uint32_t all = 0x10101010u;
            if (s * 32 % SEG == 0) mma16832_first(ones[n], {all, all, all, all}, xv.x, xv.y);
            else mma16832(ones[n], {all, all, all, all}, xv.x, xv.y);
          }
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
            if constexpr (SUMS) {
              const uint4 e = lds128(x_at + 8 * n * XSB);
              f[0] = u2f(e.x), f[1] = u2f(e.z);
              sum[n][0] += z[0] * (int)e.y;
              sum[n][1] += z[0] * (int)e.w;
              sum[n][2] += z[1] * (int)e.y;
              sum[n][3] += z[1] * (int)e.w;
            } else {
              const uint2 e = lds64(x_at + 8 * n * XSB);
              f[0] = u2f(e.x), f[1] = u2f(e.y);
              if (!ENTRIES) f[0] *= 0.0625f, f[1] *= 0.0625f;
              if (ZEROS)
#pragma unroll
                for (int k = 0; k < 4; k++) sum[n][k] += z[k >> 1] * ones[n][k];
            }
#pragma unroll
            for (int e = 0; e < 4; e++) acc[n][e] = fmaf((float)sum[n][e], sw[e >> 1] * f[e & 1], acc[n][e]);
          }
          x_at += 8 * NT * XSB;
        }
      }
      x_now += 128;
      now += p.stage;
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
    for (int i = share * 32 + lane; i < TILE; i += 32 << p.log_kw) {
      float v = first[i];
      for (int k = 1; k < kw; k++) v += first[k * TILE + i];
      put(t, i, v);
    }
    flip ^= 1;
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

// Shared memory of a plan; the vectors go there if they fit.
static void w4_layout_smem(const W4Args &a, W4Plan &p) {
  const int nt = a.n > 8 ? 2 : 1, nv = a.n < 8 * nt ? a.n : 8 * nt;
  const int64_t xs = ((int64_t)a.cols / w4_segment(a) * 8 * nt * (a.zeros ? 8 : 4) + 127) / 128 * 128;
  const int part = 2 * kW4Warps * 16 * 8 * nt * 4;
  const auto ring = [&] { return (kW4Warps * w4_depth(nt) * p.stage + 127) / 128 * 128; };
  p.vectors = W4_KEPT;
  p.stage = p.record;
  p.x_stride = 128 * p.quads + 32;  // rows of eight lanes' reads fall on different banks
  int64_t entries = xs;
  if ((int64_t)nv * p.x_stride + 128 + xs + ring() + part > kW4Smem) {
    p.vectors = W4_PASSING;
    p.stage += 8 * nt * 128;
    p.x_stride = 0;
    if (xs + ring() + part > kW4Smem) {
      p.vectors = W4_ALL_PASSING;
      p.stage += 128 / w4_segment(a) * 8 * nt * 4;
      entries = 0;
    }
  }
  p.at_xs = (nv * p.x_stride + 127) / 128 * 128;
  p.at_ring = (int)(p.at_xs + entries);
  p.at_part = p.at_ring + ring();
  p.size = p.at_part + part;
}

// f<NT, SEG, ZEROS, VECTORS, S32>() of the instance for a product.
template <int NT, int VECTORS, bool S32, class F>
static cudaError_t w4_seg(int seg, bool zeros, F f) {
  if (zeros) {
    if (seg == 128) return f.template operator()<NT, 128, true, VECTORS, S32>();
    if (seg == 64) return f.template operator()<NT, 64, true, VECTORS, S32>();
    return f.template operator()<NT, 32, true, VECTORS, S32>();
  }
  if (seg == 128) return f.template operator()<NT, 128, false, VECTORS, S32>();
  if (seg == 64) return f.template operator()<NT, 64, false, VECTORS, S32>();
  return f.template operator()<NT, 32, false, VECTORS, S32>();
}
template <int NT, bool S32, class F>
static cudaError_t w4_vec(int vectors, int seg, bool zeros, F f) {
  if (vectors == W4_KEPT) return w4_seg<NT, W4_KEPT, S32>(seg, zeros, f);
  return vectors == W4_PASSING ? w4_seg<NT, W4_PASSING, S32>(seg, zeros, f) : w4_seg<NT, W4_ALL_PASSING, S32>(seg, zeros, f);
}
template <class F>
static cudaError_t w4_at(int nt, int vectors, bool s32, int seg, bool zeros, F f) {
  if (nt > 1) return s32 ? w4_vec<2, true>(vectors, seg, zeros, f) : w4_vec<2, false>(vectors, seg, zeros, f);
  return s32 ? w4_vec<1, true>(vectors, seg, zeros, f) : w4_vec<1, false>(vectors, seg, zeros, f);
}

struct W4Launch {
  const W4Args &a;
  int type;
  const W4Plan &p;
  cudaStream_t st;
  template <int NT, int SEG, bool ZEROS, int VECTORS, bool S32>
  cudaError_t operator()() const {
    const dim3 grid(p.teams / (kW4Warps >> p.log_kw), (unsigned)((a.n + 8 * NT - 1) / (8 * NT)));
    return launch_k(k_w4<NT, SEG, ZEROS, VECTORS, S32>, grid, 32 * kW4Warps, p.size, st, a, p, type);
  }
};

cudaError_t launch_w4_mulvec(const W4Args &a, int type, int sms, cudaStream_t st) {
  const int tiles = (a.rows + 15) / 16;
  const bool s32 = a.scale_type == RK_ACT_F32;
  W4Plan p{};
  p.quads = (a.cols + 127) / 128;
  p.record = w4_record(a.group, s32, a.zeros);
  p.log_width = w4_width(a.group) == 128 ? 7 : w4_width(a.group) == 64 ? 6 : 5;
  w4_layout_smem(a, p);
  if (p.size > kW4Smem) return cudaErrorInvalidValue;
  // Teams of the size that ends soonest, counted in stretches: the tiles of a
  // team, each its longest share and an end, which costs about two stretches.
  int least = 0x7fffffff;
  for (int log_kw = 4; log_kw >= 0; log_kw--) {
    const int per_cta = kW4Warps >> log_kw, units = sms * per_cta;
    const int64_t cost = (int64_t)((tiles + units - 1) / units) * (((p.quads + (1 << log_kw) - 1) >> log_kw) + 2);
    if (cost < least) {
      least = (int)cost;
      p.log_kw = log_kw;
      p.teams = tiles < units ? (tiles + per_cta - 1) / per_cta * per_cta : units;
    }
  }
  const int64_t width = 65535LL * 8;  // of grid.y
  for (int64_t v = 0; v < a.n; v += width) {
    W4Args b = a;
    b.n = (int)(a.n - v < width ? a.n - v : width);
    b.x += v * a.cols;
    b.x_scales += v * (a.cols / a.x_group);
    b.out = static_cast<char *>(a.out) + v * a.out_stride * (type == RK_ACT_F32 ? 4 : 2);
    const cudaError_t e = w4_at(a.n > 8 ? 2 : 1, p.vectors, s32, w4_segment(a), a.zeros, W4Launch{b, type, p, st});
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

struct W4Init {
  template <int NT, int SEG, bool ZEROS, int VECTORS, bool S32>
  cudaError_t operator()() const {
    return cudaFuncSetAttribute(k_w4<NT, SEG, ZEROS, VECTORS, S32>, cudaFuncAttributeMaxDynamicSharedMemorySize, kW4Smem);
  }
};

cudaError_t init_w4_attributes() {
  for (int i = 0; i < 24; i++)
    for (int seg = 32; seg <= 128; seg *= 2) {
      const cudaError_t e = w4_at(1 + (i & 1), i / 8, (i & 2) != 0, seg, (i & 4) != 0, W4Init{});
      if (e != cudaSuccess) return e;
    }
  return cudaSuccess;
}

}  // namespace rk
