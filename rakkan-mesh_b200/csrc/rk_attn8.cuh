// rk_attn8.cuh — the kernels of attention over the 8-bit paged cache.
//
// For each row (a query token and head) and visible token t, with the
// cache's integers kq, vq and their pages' scales ks, vs:
//   a_t = scale · ks · (q · kq_t),   out = Σ 2^(a_t·log2e) vs vq_t / Σ 2^(a_t·log2e).
// The cache is read once for the query heads of a kv head. At one token a
// request that read bounds the call (one byte a value, 4·G flop for it with
// G query heads a kv head), and CUDA cores cannot keep up with it from G = 4
// on; so both products run on mma.m16n8k16 with the integers as float16
// (exact), and no shared memory lies between a load and its product: each
// warp streams its own tiles from global memory into the registers that the
// products read.
//
// Fragments. A 16-column step of a product may take its columns in any order
// as long as both operands agree. Lane (r, c) = (lane / 4, lane % 4) holds
// columns {2c, 2c+1, 2c+8, 2c+9} of a step; they are given to four
// neighbouring bytes, so that a lane's bytes of several steps are one 16-, 8-
// or 4-byte load: of a key row, dimensions; of a transposed value row,
// tokens. The scores' columns (tokens) land where the second product wants
// its rows, which fixes the token of a key row (token_of).
//
// Precision. A float32 row of queries is scaled by a power of two to a
// largest magnitude near 2^13 and split into two float16 terms (22 bits)
// that fill both halves of the 16 rows (8 query rows, high and low terms);
// 16-bit queries are one exact term (16 query rows). The softmax weights
// likewise, with the value scale in the weight: w_t = 2^(s_t + E - M + 14)·f
// for vs = f·2^E, with M the running maximum of s_t + E + 1 and so
// w_t <= 2^14. The denominator has a running maximum of its own (m), so
// that pages of any two scales are weighed rightly. 16-bit types round a
// weight once to float16 (2^-12 of itself, an eighth of bfloat16's own
// rounding of the result, and half of float16's on average over tokens).
//
// Work. A unit is a request's kv head and up to four tiles of query rows; its
// keys are cut into tiles of 32 tokens (16 at head size 256). The tiles of all
// units in a row are dealt out in equal runs, one to a CTA, so that lengths
// need not be alike and one long request fills the GPU as well as many short
// ones. Within a CTA the warps take different row tiles of the same tokens
// (their loads meet in L1) or, where there are fewer, different tokens. A unit
// that crosses CTAs leaves its parts in the workspace, and a second kernel
// joins them.
#pragma once
#include "rk_act.cuh"
#include "rk_matvec.cuh"
#include "rk_serve.cuh"

namespace rk {

constexpr int kA8Warps = 4;
constexpr int kA8Threads = 32 * kA8Warps;

template <int HS>
struct A8Shape {
  static constexpr int TT = HS > 128 ? 16 : 32;  // tokens of a tile
  static constexpr int CTAS = HS > 128 ? 1 : HS > 64 ? 2 : HS > 32 ? 3 : 4;  // of an SM, by their registers
  static constexpr int KS = HS / 16;             // 16-column steps over a head
  static constexpr int PITCH = HS + 8;           // floats between rows of a merge buffer
};

// A part's place in the workspace: 4 row tiles of 16 rows, each HS sums and
// (m, M, l), behind the records of all CTAs.
struct A8Record {
  int first, last;       // CTAs of the unit (first < 0: no unit crosses into this CTA)
  int req, head, row0;   // request, kv head, first query row
  int rows;              // query rows in the unit
  int q0;                // first row of q of the request
  int pad;
};
__host__ __device__ inline int64_t a8_part_floats(int hs) { return 64LL * (hs + 4); }

struct A8Grid {
  int ctas;       // CTAs of the main kernel
  int min_tiles;  // fewest tiles worth a CTA
};

RK_DEV uint32_t prmt(uint32_t a, uint32_t b, uint32_t s) {
  uint32_t d;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(s));
  return d;
}

// Four int8 as two pairs of float16: 1024 + (q + 128) has the byte in its
// low bits, and subtracting 1152 is exact.
RK_DEV void i8_to_h2(uint32_t w, uint32_t &p01, uint32_t &p23) {
  const uint32_t u = w ^ 0x80808080u;
  const __half2 off = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
  uint32_t a = prmt(u, 0x64646464u, 0x4140), b = prmt(u, 0x64646464u, 0x4342);
  __half2 ha = __hsub2(*reinterpret_cast<__half2 *>(&a), off), hb = __hsub2(*reinterpret_cast<__half2 *>(&b), off);
  p01 = *reinterpret_cast<uint32_t *>(&ha);
  p23 = *reinterpret_cast<uint32_t *>(&hb);
}

RK_DEV void mma16816(float *c, const uint32_t *a, uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

RK_DEV float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

RK_DEV uint32_t pack_h2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&h);
}
// The part of (a, b) that pack_h2 left.
RK_DEV uint32_t pack_rest(float a, float b, uint32_t p) {
  const __half2 h = *reinterpret_cast<const __half2 *>(&p);
  return pack_h2(a - __low2float(h), b - __high2float(h));
}

// A lane's words of one row of HS bytes: word s is step s's four bytes.
// Whole 64-byte stretches as 16 bytes a lane, then 32 as 8, then 16 as 4.
template <int HS>
RK_DEV void load_row(const int8_t *row, int c, uint32_t *w) {
  constexpr int N64 = HS / 64, R = HS % 64;
#pragma unroll
  for (int i = 0; i < N64; i++) {
    const uint4 v = __ldg(reinterpret_cast<const uint4 *>(row + 64 * i + 16 * c));
    w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
  }
  if constexpr (R >= 32) {
    const uint2 v = __ldg(reinterpret_cast<const uint2 *>(row + 64 * N64 + 8 * c));
    w[4 * N64] = v.x, w[4 * N64 + 1] = v.y;
  }
  if constexpr (R % 32 != 0)
    w[HS / 16 - 1] = __ldg(reinterpret_cast<const uint32_t *>(row + HS - 16 + 4 * c));
}
// The dimension of byte b (0..3) of lane c's word s.
template <int HS>
RK_DEV int dim_of(int s, int c, int b) {
  constexpr int N64 = HS / 64, R = HS % 64;
  if (s < 4 * N64) return 64 * (s / 4) + 16 * c + 4 * (s % 4) + b;
  if (R >= 32 && s < 4 * N64 + 2) return 64 * N64 + 8 * c + 4 * (s - 4 * N64) + b;
  return HS - 16 + 4 * c + b;
}

RK_DEV float q_load(const void *q, int type, int64_t i) {
  if (type == RK_ACT_F32) return static_cast<const float *>(q)[i];
  if (type == RK_ACT_F16) return __half2float(static_cast<const __half *>(q)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16 *>(q)[i]);
}
RK_DEV void o_store(void *o, int type, int64_t i, float v) {
  if (type == RK_ACT_F32) static_cast<float *>(o)[i] = v;
  else if (type == RK_ACT_F16) static_cast<__half *>(o)[i] = __float2half_rn(v);
  else static_cast<__nv_bfloat16 *>(o)[i] = __float2bfloat16_rn(v);
}

// A request's share of the work.
struct A8Req {
  int q0, nq;      // its rows of q
  int len;         // its tokens, at most the table's
  long long last;  // position of its last query (lens - 1, the table's end apart)
  int tile0, tiles;
  int units;       // of one kv head
  int rw;          // row tiles of a unit (1, 2 or 4)
};

template <int HS, bool SPLIT>
RK_DEV A8Req a8_req(const Attn8Args &a, int i) {
  constexpr int TT = A8Shape<HS>::TT, R = SPLIT ? 8 : 16;
  A8Req q;
  if (a.q_start) {
    q.q0 = min(max(a.q_start[i], 0), a.tokens);
    q.nq = min(max(a.q_start[i + 1], q.q0), a.tokens) - q.q0;
  } else {
    q.q0 = i;
    q.nq = 1;
  }
  const int len = a.lens[i];
  q.last = (long long)len - 1;
  q.len = (int)max(0LL, min((long long)len, (long long)a.max_blocks * a.c.block));
  const long long from = a.window > 0 ? max(0LL, q.last - (q.nq - 1) + 1 - a.window) : 0;
  q.tile0 = (int)min((long long)q.len, from) / TT;
  q.tiles = max(1, (q.len + TT - 1) / TT - q.tile0);
  const int rts = (int)(((long long)q.nq * (a.heads / a.c.kv_heads) + R - 1) / R);
  q.rw = rts >= 4 ? 4 : rts >= 2 ? 2 : 1;
  q.units = (rts + q.rw - 1) / q.rw;
  return q;
}

template <int HS, bool SPLIT, bool WIDE>
__global__ void __launch_bounds__(kA8Threads, A8Shape<HS>::CTAS) k_attn8(Attn8Args a, int type, A8Grid grid) {
  using Shape = A8Shape<HS>;
  constexpr int TT = Shape::TT, KS = Shape::KS, PITCH = Shape::PITCH, R = SPLIT ? 8 : 16;
  constexpr int NH = TT / 16, ND = HS / 8;  // 16-token halves of a tile; 8-dimension columns of the output
  extern __shared__ __align__(16) float sm[];
  float *s_o = sm;                                     // [warps][16][PITCH]
  float *s_st = sm + kA8Warps * 16 * PITCH;            // [warps][16][4]
  __shared__ long long s_scan[kA8Warps + 1];
  __shared__ long long s_before;
  __shared__ int s_req;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, r = lane >> 2, c = lane & 3;
  const int G = a.heads / a.c.kv_heads, H = a.c.kv_heads, B = a.c.block;
  griddep_trigger();

  // The run of tiles of this CTA: a scan over the requests' tiles.
  const int per_t = (a.n + kA8Threads - 1) / kA8Threads;
  const int i0 = min(a.n, tid * per_t), i1 = min(a.n, i0 + per_t);
  long long mine = 0;
  for (int i = i0; i < i1; i++) {
    const A8Req q = a8_req<HS, SPLIT>(a, i);
    mine += (long long)H * q.units * q.tiles;
  }
  long long incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long u = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += u;
  }
  if (lane == 31) s_scan[warp] = incl;
  __syncthreads();
  long long excl = incl - mine, total = 0;
  for (int w = 0; w < kA8Warps; w++) {
    if (w < warp) excl += s_scan[w];
    total += s_scan[w];
  }
  const long long per = max((long long)grid.min_tiles, (total + grid.ctas - 1) / grid.ctas);
  const long long begin = per * blockIdx.x, end = min(total, begin + per);
  A8Record *records = static_cast<A8Record *>(a.ws);
  float *parts = reinterpret_cast<float *>(records + grid.ctas);
  if (begin >= end) {
    if (tid == 0) records[blockIdx.x].first = -1;
    return;
  }
  if (begin >= excl && begin < excl + mine) {
    long long p = excl;
    for (int i = i0; i < i1; i++) {
      const A8Req q = a8_req<HS, SPLIT>(a, i);
      const long long size = (long long)H * q.units * q.tiles;
      if (begin < p + size) {
        s_req = i;
        s_before = p;
        break;
      }
      p += size;
    }
  }
  __syncthreads();
  int req = s_req;
  long long base = s_before;  // where the request's tiles begin
  A8Req q = a8_req<HS, SPLIT>(a, req);

  for (long long at = begin; at < end;) {
    // The unit at `at`, and this CTA's tiles of it.
    while (at >= base + (long long)H * q.units * q.tiles) {
      base += (long long)H * q.units * q.tiles;
      q = a8_req<HS, SPLIT>(a, ++req);
    }
    const int u = (int)((at - base) / q.tiles);
    const int head = u / q.units, rg = u % q.units;
    const long long u0 = base + (long long)u * q.tiles, u1 = u0 + q.tiles;
    const int t0 = (int)(at - u0), t1 = (int)(min(end, u1) - u0);
    const int rw = q.rw, tw = kA8Warps / rw, wr = warp % rw, wt = warp / rw;
    const int row0 = (rg * rw + wr) * R;        // of the request's nq·G rows (token-major)
    const int all_rows = q.nq * G;

    // Limits of this lane's rows: visible tokens are (low, high]. Rows past
    // the last see all (their queries are zeros, their sums are not stored).
    int high[2], low[2], high_max = -1;
    float f[2];
#pragma unroll
    for (int j = 0; j < 2; j++) {
      const int row = row0 + r + 8 * (SPLIT ? 0 : j);
      const long long pos = q.last - (q.nq - 1) + row / G;
      high[j] = 0x7fffffff;
      low[j] = -1;
      if (row < all_rows) {
        high[j] = (int)max(-1LL, min(pos, (long long)q.len - 1));
        if (a.window > 0) low[j] = (int)max(-1LL, min(pos - a.window, (long long)q.len));
        high_max = max(high_max, high[j]);
      }
    }
    int high_min = min(high[0], high[1]), low_max = max(low[0], low[1]);
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) {
      high_max = max(high_max, __shfl_xor_sync(0xffffffffu, high_max, o));
      high_min = min(high_min, __shfl_xor_sync(0xffffffffu, high_min, o));
      low_max = max(low_max, __shfl_xor_sync(0xffffffffu, low_max, o));
    }

    // Query fragments.
    uint32_t qa[KS][4];
#pragma unroll
    for (int j = 0; j < (SPLIT ? 1 : 2); j++) {
      const int row = row0 + r + 8 * j;
      const bool have = row < all_rows;
      const int64_t qi = have ? (int64_t)(q.q0 + row / G) * a.q_stride + (int64_t)(head * G + row % G) * HS : 0;
      float top = 0.0f;
      bool wrong = false;
#pragma unroll
      for (int s = 0; s < KS; s++)
#pragma unroll
        for (int b = 0; b < 4; b++) {
          const float v = have ? fabsf(q_load(a.q, type, qi + dim_of<HS>(s, c, b))) : 0.0f;
          top = fmaxf(top, v);
          wrong |= !(v < INFINITY);
        }
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      wrong = (__ballot_sync(0xffffffffu, wrong) >> (lane & 28) & 15) != 0;
      // 2^-e brings the row's largest magnitude into [2^13, 2^14).
      int e = top > 0.0f && !wrong ? int(f2u(top) >> 23) - 127 - 13 : 0;
      e = max(e, -112);
      const float down = u2f(uint32_t(127 - e) << 23);
      f[j] = wrong ? u2f(kCanonNaN) : u2f(uint32_t(127 + e) << 23) * (a.scale * 1.44269504088896f);
#pragma unroll
      for (int s = 0; s < KS; s++) {
        float v[4];
#pragma unroll
        for (int b = 0; b < 4; b++)
          v[b] = have && !wrong ? q_load(a.q, type, qi + dim_of<HS>(s, c, b)) * down : 0.0f;
        qa[s][j] = pack_h2(v[0], v[1]);
        qa[s][2 + j] = pack_h2(v[2], v[3]);
        if constexpr (SPLIT) {
          qa[s][1] = pack_rest(v[0], v[1], qa[s][0]);
          qa[s][3] = pack_rest(v[2], v[3], qa[s][2]);
        }
      }
    }
    if (SPLIT) f[1] = f[0];

    float o[ND][4], m[2] = {-INFINITY, -INFINITY}, M[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
#pragma unroll
    for (int d = 0; d < ND; d++) o[d][0] = o[d][1] = o[d][2] = o[d][3] = 0.0f;

    // One tile: where its halves lie, and their scales.
    const int *table = a.table + (int64_t)req * a.max_blocks;
    int64_t ph[NH];
    uint32_t kw[NH][2][KS], vw[NH][ND];
    float ks[NH], vs[NH];
    bool live[NH];
    auto place = [&](int t) {
#pragma unroll
      for (int s = 0; s < NH; s++) {
        if (WIDE && s > 0) {
          ph[s] = ph[0];
          live[s] = live[0];
          continue;
        }
        const int tok = (q.tile0 + t) * TT + 16 * s;
        int page = tok <= high_max ? __ldg(table + tok / B) : -1;
        live[s] = page >= 0 && page < a.c.blocks;
        if (tok <= high_max && !live[s]) atomicExch(a.err, DEV_ERR_RANGE);
        ph[s] = live[s] ? (int64_t)page * H + head : 0;
      }
    };
    auto load_k = [&](int t) {
#pragma unroll
      for (int s = 0; s < NH; s++) {
        const int o0 = ((q.tile0 + t) * TT + (WIDE ? 0 : 16 * s)) % B;
#pragma unroll
        for (int j = 0; j < 2; j++) {
          const int tok = o0 + (WIDE ? 8 * (r >> 1) + 4 * s : 4 * (r >> 1)) + 2 * j + (r & 1);
          load_row<HS>(a.c.k + (ph[s] * B + tok) * HS, c, kw[s][j]);
        }
        ks[s] = live[s] ? __ldg(a.c.k_scale + ph[s]) : 0.0f;
        vs[s] = live[s] ? __ldg(a.c.v_scale + ph[s]) : 0.0f;
      }
    };
    auto load_v = [&](int t) {
      if constexpr (WIDE) {
        const int8_t *v = a.c.v + (ph[0] * HS + r) * B + ((q.tile0 + t) * TT) % B + 8 * c;
#pragma unroll
        for (int d = 0; d < ND; d++) {
          const uint2 w = __ldg(reinterpret_cast<const uint2 *>(v + (int64_t)8 * d * B));
          vw[0][d] = w.x;
          vw[1][d] = w.y;
        }
      } else {
#pragma unroll
        for (int s = 0; s < NH; s++) {
          const int8_t *v = a.c.v + (ph[s] * HS + r) * B + ((q.tile0 + t) * TT + 16 * s) % B + 4 * c;
#pragma unroll
          for (int d = 0; d < ND; d++) vw[s][d] = __ldg(reinterpret_cast<const uint32_t *>(v + (int64_t)8 * d * B));
        }
      }
    };
    auto in_reach = [&](int t) {  // of any row of the warp
      return t < t1 && (q.tile0 + t) * TT <= high_max;
    };

    int t = t0 + wt;
    if (in_reach(t)) {
      place(t);
      load_k(t);
      load_v(t);
    }
    for (; in_reach(t); t += tw) {
      const int tok0 = (q.tile0 + t) * TT;
      float sc[NH][2][4];
#pragma unroll
      for (int s = 0; s < NH; s++)
#pragma unroll
        for (int j = 0; j < 2; j++) {
          sc[s][j][0] = sc[s][j][1] = sc[s][j][2] = sc[s][j][3] = 0.0f;
#pragma unroll
          for (int k = 0; k < KS; k++) {
            uint32_t b0, b1;
            i8_to_h2(kw[s][j][k], b0, b1);
            mma16816(sc[s][j], qa[k], b0, b1);
          }
        }
      float cks[NH], cvs[NH];
      bool whole = tok0 + TT - 1 <= high_min && tok0 > low_max, clive[NH];
#pragma unroll
      for (int s = 0; s < NH; s++) {
        cks[s] = ks[s];
        cvs[s] = vs[s];
        clive[s] = live[s];
        whole &= live[s];
      }
      const bool more = in_reach(t + tw);
      if (more) {
        place(t + tw);
        load_k(t + tw);
      }

      // Scores in powers of two, their maxima, and the tile's weights.
      float mx[NH][2];
#pragma unroll
      for (int s = 0; s < NH; s++) {
        const float f0 = f[0] * cks[s], f1 = f[1] * cks[s];
#pragma unroll
        for (int j = 0; j < 2; j++) {
          if constexpr (SPLIT) {
            sc[s][j][0] = (sc[s][j][0] + sc[s][j][2]) * f0;
            sc[s][j][1] = (sc[s][j][1] + sc[s][j][3]) * f0;
          } else {
            sc[s][j][0] *= f0;
            sc[s][j][1] *= f0;
            sc[s][j][2] *= f1;
            sc[s][j][3] *= f1;
          }
          if (!whole) {
            const int tok = tok0 + (WIDE ? 8 * c + 4 * s : 16 * s + 4 * c) + 2 * j;
#pragma unroll
            for (int e = 0; e < (SPLIT ? 2 : 4); e++) {
              const int k = tok + (e & 1);
              if (!clive[s] || k > high[e >> 1] || k <= low[e >> 1]) sc[s][j][e] = -INFINITY;
            }
          }
        }
        mx[s][0] = fmaxf(fmaxf(sc[s][0][0], sc[s][0][1]), fmaxf(sc[s][1][0], sc[s][1][1]));
        mx[s][1] = SPLIT ? mx[s][0] : fmaxf(fmaxf(sc[s][0][2], sc[s][0][3]), fmaxf(sc[s][1][2], sc[s][1][3]));
      }
      if (WIDE && NH == 2) {
        mx[0][0] = mx[NH - 1][0] = fmaxf(mx[0][0], mx[NH - 1][0]);
        mx[0][1] = mx[NH - 1][1] = fmaxf(mx[0][1], mx[NH - 1][1]);
      }
#pragma unroll
      for (int s = 0; s < (WIDE ? 1 : NH); s++)
#pragma unroll
        for (int j = 0; j < (SPLIT ? 1 : 2); j++) {
          mx[s][j] = fmaxf(mx[s][j], __shfl_xor_sync(0xffffffffu, mx[s][j], 1));
          mx[s][j] = fmaxf(mx[s][j], __shfl_xor_sync(0xffffffffu, mx[s][j], 2));
        }
      // vs = vf · 2^ve.
      float ve[NH], vf[NH];
#pragma unroll
      for (int s = 0; s < NH; s++) {
        const int e = max(int(f2u(cvs[s]) >> 23) - 127, -126);
        ve[s] = cvs[s] > 0.0f ? (float)e : -1e30f;  // a scale of zero: weights of zero
        vf[s] = cvs[s] * u2f(uint32_t(127 - min(e, 126)) << 23) * (e > 126 ? 0.5f : 1.0f);
      }
      float ms[2], Ms[2], top[2];
      bool grew = false;
#pragma unroll
      for (int j = 0; j < (SPLIT ? 1 : 2); j++) {
        float mn = m[j], Mn = M[j];
#pragma unroll
        for (int s = 0; s < (WIDE ? 1 : NH); s++) {
          mn = fmaxf(mn, mx[s][j]);
          if (cvs[s] > 0.0f) Mn = fmaxf(Mn, mx[s][j] + (ve[s] + 1.0f));
        }
        ms[j] = mn == -INFINITY ? 0.0f : mn;
        Ms[j] = Mn == -INFINITY ? 0.0f : Mn;
        top[j] = Mn;
        l[j] *= ex2(m[j] - ms[j]);
        grew |= Mn > M[j];
        m[j] = mn;
      }
      if (SPLIT) ms[1] = ms[0], Ms[1] = Ms[0], top[1] = top[0];
      if (__any_sync(0xffffffffu, grew)) {
        const float g0 = ex2(M[0] - Ms[0]), g1 = SPLIT ? g0 : ex2(M[1] - Ms[1]);
#pragma unroll
        for (int d = 0; d < ND; d++) {
          o[d][0] *= g0;
          o[d][1] *= g0;
          o[d][2] *= g1;
          o[d][3] *= g1;
        }
#pragma unroll
        for (int j = 0; j < 2; j++) M[j] = top[j];
      }
#pragma unroll
      for (int s = 0; s < NH; s++) {
        uint32_t pa[4];
#pragma unroll
        for (int j = 0; j < 2; j++) {
          float w[4];
#pragma unroll
          for (int e = 0; e < (SPLIT ? 2 : 4); e++) {
            const float v = sc[s][j][e];
            l[e >> 1] += ex2(v - ms[e >> 1]);
            w[e] = ex2(v + (ve[s] + 14.0f - Ms[e >> 1])) * vf[s];
          }
          pa[2 * j] = pack_h2(w[0], w[1]);
          pa[2 * j + 1] = SPLIT ? pack_rest(w[0], w[1], pa[2 * j]) : pack_h2(w[2], w[3]);
        }
#pragma unroll
        for (int d = 0; d < ND; d++) {
          uint32_t b0, b1;
          i8_to_h2(vw[s][d], b0, b1);
          mma16816(o[d], pa, b0, b1);
        }
      }
      if (more) load_v(t + tw);
    }

    // The warps' sums meet in shared memory.
#pragma unroll
    for (int j = 0; j < 2; j++) {
      l[j] += __shfl_xor_sync(0xffffffffu, l[j], 1);
      l[j] += __shfl_xor_sync(0xffffffffu, l[j], 2);
    }
    __syncthreads();  // the last unit's readers are done
    float *so = s_o + warp * 16 * PITCH, *st = s_st + warp * 64;
#pragma unroll
    for (int d = 0; d < ND; d++) {
      if constexpr (SPLIT) {
        *reinterpret_cast<float2 *>(so + r * PITCH + 8 * d + 2 * c) = make_float2(o[d][0] + o[d][2], o[d][1] + o[d][3]);
      } else {
        *reinterpret_cast<float2 *>(so + r * PITCH + 8 * d + 2 * c) = make_float2(o[d][0], o[d][1]);
        *reinterpret_cast<float2 *>(so + (r + 8) * PITCH + 8 * d + 2 * c) = make_float2(o[d][2], o[d][3]);
      }
    }
    if (c == 0) {
#pragma unroll
      for (int j = 0; j < (SPLIT ? 1 : 2); j++) {
        st[4 * (r + 8 * j)] = m[j];
        st[4 * (r + 8 * j) + 1] = M[j];
        st[4 * (r + 8 * j) + 2] = l[j];
      }
    }
    __syncthreads();
    const bool starts = at == u0, ends = u1 <= end;
    float *part = parts + (2LL * blockIdx.x + (starts ? 1 : 0)) * a8_part_floats(HS);
    const int unit_row0 = rg * rw * R, unit_rows = min(rw * R, all_rows - unit_row0);
    for (int row = warp; row < unit_rows; row += kA8Warps) {
      const int tile = row / R, rr = row % R;
      float mm = -INFINITY, MM = -INFINITY;
      for (int w = 0; w < tw; w++) {
        mm = fmaxf(mm, s_st[(tile + w * rw) * 64 + 4 * rr]);
        MM = fmaxf(MM, s_st[(tile + w * rw) * 64 + 4 * rr + 1]);
      }
      const float msafe = mm == -INFINITY ? 0.0f : mm, Msafe = MM == -INFINITY ? 0.0f : MM;
      float ll = 0.0f, g[kA8Warps];
#pragma unroll
      for (int w = 0; w < kA8Warps; w++) {
        if (w >= tw) break;
        const float *s = s_st + (tile + w * rw) * 64 + 4 * rr;
        ll += s[2] * exp2f(s[0] - msafe);
        g[w] = exp2f(s[1] - Msafe);
      }
      const int qrow = unit_row0 + row;
      const float scale = ll == 0.0f ? 0.0f : exp2f(Msafe - 14.0f - msafe) / ll;
      const int64_t oi = (int64_t)(q.q0 + qrow / G) * a.out_stride + (int64_t)(head * G + qrow % G) * HS;
      for (int d = lane; d < HS; d += 32) {
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < kA8Warps; w++) {
          if (w >= tw) break;
          v = fmaf(s_o[(tile + w * rw) * 16 * PITCH + rr * PITCH + d], g[w], v);
        }
        if (starts && ends) o_store(a.out, type, oi + d, v * scale);
        else part[row * HS + d] = v;
      }
      if (!(starts && ends) && lane == 0) {
        float *s = part + 64 * HS + 4 * row;
        s[0] = mm;
        s[1] = MM;
        s[2] = ll;
      }
    }
    if (at == begin && tid == 0) {
      A8Record rec;
      rec.first = starts ? -1 : (int)(u0 / per);
      rec.last = (int)((u1 - 1) / per);
      rec.req = req;
      rec.head = head;
      rec.row0 = unit_row0;
      rec.rows = unit_rows;
      rec.q0 = q.q0;
      rec.pad = 0;
      records[blockIdx.x] = rec;
    }
    at = min(end, u1);
  }
}

// The instances for one of the two query forms (each in a file of its own,
// to be compiled side by side).
template <bool SPLIT>
struct A8 {
  template <class F>
  static cudaError_t at(int hs, F f) {
    switch (hs) {
      case 16: return f.template operator()<16>();
      case 32: return f.template operator()<32>();
      case 48: return f.template operator()<48>();
      case 64: return f.template operator()<64>();
      case 80: return f.template operator()<80>();
      case 96: return f.template operator()<96>();
      case 112: return f.template operator()<112>();
      case 128: return f.template operator()<128>();
      case 256: return f.template operator()<256>();
    }
    return cudaErrorInvalidValue;
  }
  template <int HS>
  static constexpr int smem() { return kA8Warps * 16 * (A8Shape<HS>::PITCH + 4) * 4; }

  struct Init {
    template <int HS>
    cudaError_t operator()() const {
      cudaError_t e = cudaFuncSetAttribute(k_attn8<HS, SPLIT, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem<HS>());
      if constexpr (A8Shape<HS>::TT == 32)
        if (e == cudaSuccess)
          e = cudaFuncSetAttribute(k_attn8<HS, SPLIT, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem<HS>());
      return e;
    }
  };
  struct Launch {
    const Attn8Args &a;
    int type;
    A8Grid g;
    cudaStream_t st;
    template <int HS>
    cudaError_t operator()() const {
      if constexpr (A8Shape<HS>::TT == 32)
        if (a.c.block >= 32)
          return launch_k(k_attn8<HS, SPLIT, true>, g.ctas, kA8Threads, smem<HS>(), st, a, type, g);
      return launch_k(k_attn8<HS, SPLIT, false>, g.ctas, kA8Threads, smem<HS>(), st, a, type, g);
    }
  };
  static cudaError_t init() {
    cudaError_t e = cudaSuccess;
    for (int hs : {16, 32, 48, 64, 80, 96, 112, 128, 256})
      if (e == cudaSuccess) e = at(hs, Init{});
    return e;
  }
};

cudaError_t attn8_init_f32();
cudaError_t attn8_main_f32(const Attn8Args &a, int type, A8Grid g, cudaStream_t st);

}  // namespace rk
