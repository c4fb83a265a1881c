// rk_attn8.cuh — the kernels of attention over the 8-bit paged cache.
//
// For each row (a query token and head) and visible token t, with the
// cache's integers kq, vq and their pages' scales ks, vs:
//   a_t = scale · ks · (q · kq_t),   out = Σ 2^(a_t·log2e) vs vq_t / Σ 2^(a_t·log2e).
// The cache is read once for the query heads of a kv head. At one token a
// request that read bounds the call (one byte a value, 4·G flop for it with
// G query heads a kv head), and CUDA cores cannot keep up with it from G = 4
// on; so both products run on the tensor cores, the scores on the bytes as they
// are, the weighted values with the bytes as float16 (exact). Each warp streams
// its own tiles through two slots of shared memory (cp.async), one under way
// while it works on the other: tiles loaded into registers instead took 78.6
// us for one token of 32 sequences of up to 4096 tokens (97,000 in all, 8 kv
// heads of 128, G = 4), which takes 42.8 now: 4.7 TB/s. With 16384 tokens each it is 6.0.
// With many rows a request the instructions around the products bound it, some
// 1000 for 16 rows by 32 tokens: 512 rows over 8192 tokens 366 us, 182 TFLOP/s.
//
// Fragments. Keys and transposed values are the 16-row operand, queries and
// weights the 8-column one: a tile of 8 query rows then fills the columns,
// and half as many products and registers do as with queries in the rows
// (91 us that way, with tiles in registers). A step of a product may
// take its terms in any order as long as both operands agree. So of a step of
// two 16-long halves lane (r, c) = (lane / 4, lane % 4) is given four neighbouring
// bytes of each, and its bytes of several steps are one 16-, 8- or 4-byte
// load: of a key row, dimensions; of a transposed value row, tokens. The scores
// come out as (token, query); a transposing move of 8x8 registers makes them
// the second product's column operand, which fixes the token of each key row.
//
// Precision. The scores' product is mma.m16n8k32 on signed bytes: the keys
// as they are, a row of queries as integers of two signed bytes (bfloat16,
// the row's largest at 32639: off by at most 2^-16 of it) or three (float32 and
// float16, 2^-24), each its own exact product, joined in float32. (float16
// products would want the keys converted: 58.3 us in place of 48.9 at the time.)
// The softmax weights are float16, one term for bfloat16 (2^-12 of itself:
// an eighth of bfloat16's own rounding of the result) and two for the others
// (22 bits): float16's rounding of the result is 2^-11, and one term raised
// the error of float16 pieces from 2.1e-4 to 2.8e-4. The type alone decides:
// what a row gives does not lose precision by what else the call holds. (8 x 64
// rows of float16 over up to 2048 tokens take 69 us, 54 with one term.) With
// one term the products' own sums run over all tiles; their adder does not
// round, which costs 7e-6 of the result over 4600 tokens, against bfloat16's
// 2e-3. The value scale is in the weight: w_t = 2^(s_t - M + E + 14) f for vs = f 2^E, M within a power of two
// of the running maximum of s_t + E + 1 and so w_t < 2^16. The denominator has
// a reference of its own (m), so that pages of any two scales are weighed
// rightly.
//
// Work. A unit is a request's kv head and up to four tiles of query rows; its
// keys are cut into tiles of 32 tokens. The tiles of all units in a row are dealt
// out in runs of equal work, one to a CTA, so that lengths need not be alike
// and one long request fills the GPU as well as many short ones. Within a CTA
// the warps take different row tiles of the same tokens, which they copy
// together, or, where there are fewer, different tokens. A unit that crosses
// CTAs leaves its parts in the workspace, and a second kernel joins them.
#pragma once
#include <type_traits>

#include "rk_act.cuh"
#include "rk_matvec.cuh"
#include "rk_serve.cuh"
#include "rk_warp.cuh"

namespace rk {

constexpr int kA8Warps = 4;
constexpr int kA8Threads = 32 * kA8Warps;

constexpr int kA8Tile = 32;  // tokens
// What a unit's beginning and end cost a CTA, in tiles of one warp (about 5 us
// against 0.6 us a tile where memory bounds them): a CTA that begins a second
// unit gets so many fewer. With 6, 9, 12 and 16 one token of the 32 sequences
// takes 43.1, 43.1, 42.6 and 43.4 us, 8 x 64 rows over up to 2048 tokens (one
// term) 55.5, 54.7, 53.9 and 54.0; heads of 128 in both, and the one value
// serves the other sizes, where it was not varied.
constexpr int kA8Begin = 12;
template <int HS>
struct A8Shape {
  static constexpr int KS = HS / 16;        // 16-long steps over a head
  static constexpr int PITCH = HS + 4;      // floats between rows of a merge buffer
  static constexpr int KBYTES = kA8Tile * HS, TILE = 2 * KBYTES;  // of a tile: keys [32][HS], values [HS][32]
};
// Shared memory of a CTA: the rings of two tiles (of one warp, or of at least
// two that share a tile where a warp has two tiles of rows), then those warps'
// queries; between two units, the merge buffers.
template <int HS, int NT, int DIGITS>
struct A8Smem {
  static constexpr int RINGS = kA8Warps / NT * 2 * A8Shape<HS>::TILE;
  static constexpr int QUERY = NT > 1 ? NT * DIGITS * (HS / 16 + HS / 16 % 2) * 128 : 0;  // of a warp
  static constexpr int MERGE = kA8Warps * 8 * NT * (A8Shape<HS>::PITCH + 4) * 4;
  static constexpr int ALL = RINGS + kA8Warps * QUERY > MERGE ? RINGS + kA8Warps * QUERY : MERGE;
};
// CTAs of an SM, by their registers and shared memory (TERMS float16 terms,
// NT tiles of 8 rows a warp).
__host__ __device__ constexpr int a8_ctas(int hs, int terms, int nt) {
  return hs > 128 ? 1 : nt > 1 ? (hs > 64 ? 2 : 3) : hs > 64 ? 3 : 4;
}

// A part's place in the workspace: up to 64 rows, each HS sums and
// (m, M, l), behind the records of all CTAs.
struct A8Record {
  int first, last;       // CTAs of the unit (first < 0: no unit crosses into this CTA)
  int head, row0;        // kv head, first query row
  int rows;              // query rows in the unit
  int q0;                // first row of q of the request
  int pad[2];
};
__host__ __device__ inline int64_t a8_part_floats(int hs) { return 64LL * (hs + 4); }

struct A8Grid {
  int ctas;       // CTAs of the main kernel
  int min_tiles;  // fewest warp tiles worth a CTA; 0: a CTA takes whole units
  int log_block;  // of the page's tokens
  bool vec_q;     // rows of q lie on 16-byte boundaries
  bool vec_out;   // four neighbours of out on a boundary of their size
  uint32_t by_group;  // ceil(2^32 / G), for quotients below 2^32 / G (0: divide)
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

RK_DEV void mma16816(float *c, const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
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
// An 8x8 tile of 16-bit values, a pair of neighbours a lane, transposed.
RK_DEV uint32_t transpose_h2(uint32_t v) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
  return d;
}
// The part of (a, b) that pack_h2 left.
RK_DEV uint32_t pack_rest(float a, float b, uint32_t p) {
  const __half2 h = *reinterpret_cast<const __half2 *>(&p);
  return pack_h2(a - __low2float(h), b - __high2float(h));
}

RK_DEV void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
RK_DEV void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Key rows of 128 and 256 bytes would meet in the same banks; the 64-byte
// stretches of odd rows change places in pairs.
template <int HS>
RK_DEV int key_swizzle(int row) { return HS % 128 == 0 ? (row & 1) << 6 : 0; }

// A lane's words of one key row: word s is step s's four bytes. Whole 64-byte
// stretches as 16 bytes a lane, then 32 as 8, then 16 as 4.
template <int HS>
RK_DEV void load_row(uint32_t row, int swizzle, int c, uint32_t *w) {
  constexpr int N64 = HS / 64, R = HS % 64;
#pragma unroll
  for (int i = 0; i < N64; i++) {
    const uint4 v = lds128(row + (i % 2 ? (64 ^ swizzle) + 64 * (i - 1) : swizzle + 64 * i) + 16 * c);
    w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
  }
  if constexpr (R >= 32) {
    const uint2 v = lds64(row + 64 * N64 + 8 * c);
    w[4 * N64] = v.x, w[4 * N64 + 1] = v.y;
  }
  if constexpr (R % 32 != 0) w[HS / 16 - 1] = lds32(row + HS - 16 + 4 * c);
}
// A lane's values of a query row as they lie in memory, in load_row's order:
// 16, 8 and 4 neighbours, as 16-byte pieces where the rows allow it. float32
// fills the four words of a word's values, 16-bit types the first two.
template <int N>
RK_DEV void load_bits(const float *q, bool vec, uint32_t (*w)[4]) {
#pragma unroll
  for (int i = 0; i < N / 4; i++) {
    if (vec) {
      const uint4 x = __ldg(reinterpret_cast<const uint4 *>(q) + i);
      w[i][0] = x.x, w[i][1] = x.y, w[i][2] = x.z, w[i][3] = x.w;
    } else {
#pragma unroll
      for (int b = 0; b < 4; b++) w[i][b] = f2u(__ldg(q + 4 * i + b));
    }
  }
}
template <int N, int W>
RK_DEV void load_bits(const uint16_t *q, bool vec, uint32_t (*w)[W]) {
  if (!vec) {
#pragma unroll
    for (int i = 0; i < N; i += 2) w[i / 4][i / 2 % 2] = __ldg(q + i) | (uint32_t)__ldg(q + i + 1) << 16;
  } else if constexpr (N >= 8) {
#pragma unroll
    for (int i = 0; i < N / 8; i++) {
      const uint4 x = __ldg(reinterpret_cast<const uint4 *>(q) + i);
      w[2 * i][0] = x.x, w[2 * i][1] = x.y, w[2 * i + 1][0] = x.z, w[2 * i + 1][1] = x.w;
    }
  } else {
    const uint2 x = __ldg(reinterpret_cast<const uint2 *>(q));
    w[0][0] = x.x, w[0][1] = x.y;
  }
}
template <int HS, class F>
RK_DEV void by_stretch(int c, F f) {  // f<N>(first dimension, first word)
  constexpr int N64 = HS / 64, R = HS % 64;
#pragma unroll
  for (int i = 0; i < N64; i++) f.template operator()<16>(64 * i + 16 * c, 4 * i);
  if constexpr (R >= 32) f.template operator()<8>(64 * N64 + 8 * c, 4 * N64);
  if constexpr (R % 32 != 0) f.template operator()<4>(HS - 16 + 4 * c, HS / 16 - 1);
}
template <class T, int W>
struct LoadQuery {
  const T *q;
  bool vec;
  uint32_t (*bits)[W];
  template <int N>
  RK_DEV void operator()(int d, int word) const {
    load_bits<N>(q + d, vec, bits + word);
  }
};
RK_DEV void o_store(void *o, int type, int64_t i, float v) {
  if (type == RK_ACT_F32) static_cast<float *>(o)[i] = v;
  else if (type == RK_ACT_F16) static_cast<__half *>(o)[i] = __float2half_rn(v);
  else static_cast<__nv_bfloat16 *>(o)[i] = __float2bfloat16_rn(v);
}
// Four neighbours; vec: on a boundary of their size.
RK_DEV void o_store4(void *o, int type, int64_t i, float4 v, bool vec) {
  if (!vec) {
    o_store(o, type, i, v.x), o_store(o, type, i + 1, v.y);
    o_store(o, type, i + 2, v.z), o_store(o, type, i + 3, v.w);
  } else if (type == RK_ACT_F32) {
    *reinterpret_cast<float4 *>(static_cast<float *>(o) + i) = v;
  } else {
    const uint2 w = type == RK_ACT_F16 ? make_uint2(act_pack<__half>(v.x, v.y), act_pack<__half>(v.z, v.w))
                                       : make_uint2(act_pack<__nv_bfloat16>(v.x, v.y), act_pack<__nv_bfloat16>(v.z, v.w));
    *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(o) + i) = w;
  }
}

// A request's share of the work.
struct A8Req {
  int q0, nq;      // its rows of q
  int len;         // its tokens, at most the table's
  int last;        // position of its last query (lens - 1, the table's end apart)
  int tile0, tiles;
  int units;       // of one kv head
  int rw;          // row tiles of a unit (1, 2 or 4)
};

template <int HS, int R>
RK_DEV A8Req a8_req(const Attn8Args &a, int lb, int i) {
  constexpr int TT = kA8Tile;
  A8Req q;
  if (a.q_start) {
    q.q0 = min(max(a.q_start[i], 0), a.tokens);
    q.nq = min(max(a.q_start[i + 1], q.q0), a.tokens) - q.q0;
  } else {
    q.q0 = i;
    q.nq = 1;
  }
  const int len = max(a.lens[i], 0);
  q.last = len - 1;
  q.len = a.max_blocks < (len >> lb) + 1 ? min(len, a.max_blocks << lb) : len;
  const int first = q.last - (q.nq - 1);
  q.tile0 = a.window > 0 && first >= a.window ? min(q.len, first - a.window + 1) / TT : 0;
  q.tiles = max(1, q.len / TT + (q.len % TT != 0) - q.tile0);
  const long long rows = (long long)q.nq * (a.heads / a.c.kv_heads);
  const int rts = (int)((rows + R - 1) / R);
  q.rw = rts >= 4 ? 4 : rts >= 2 || R > 8 ? 2 : 1;
  q.units = (rts + q.rw - 1) / q.rw;
  return q;
}

template <int HS, int TERMS, int NT>
__global__ void __launch_bounds__(kA8Threads, a8_ctas(HS, TERMS, NT)) k_attn8(Attn8Args a, int type, A8Grid grid) {
  using Shape = A8Shape<HS>;
  constexpr int TT = kA8Tile, KS = Shape::KS, PITCH = Shape::PITCH, R = 8 * NT, ND = HS / 8;
  constexpr int DIGITS = TERMS + 1;  // signed bytes of a query
  using Smem = A8Smem<HS, NT, DIGITS>;
  extern __shared__ __align__(128) char sm[];
  // The rings; between two units, the merge buffers [warps][R][PITCH] and [warps][R][4].
  float *s_o = reinterpret_cast<float *>(sm), *s_st = s_o + kA8Warps * R * PITCH;
  __shared__ long long s_scan[kA8Warps + 1];
  __shared__ long long s_before;
  __shared__ int s_req;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, r = lane >> 2, c = lane & 3;
  const int G = a.heads / a.c.kv_heads, H = a.c.kv_heads, lb = grid.log_block;
  const auto token_of = [&](int row) { return grid.by_group ? (int)__umulhi(row, grid.by_group) : row / G; };
  griddep_trigger();

  // The run of tiles (or of whole units) of this CTA: a scan over the
  // requests' sizes.
  const bool by_unit = grid.min_tiles == 0;
  const int per_t = (a.n + kA8Threads - 1) / kA8Threads;
  const int i0 = min(a.n, tid * per_t), i1 = min(a.n, i0 + per_t);
  // A unit's length: its tiles, each as many warp tiles as it has row tiles,
  // and kA8Begin in front of them.
  auto length_of = [&](const A8Req &q) { return by_unit ? 1 : q.tiles * q.rw + kA8Begin; };
  auto size_of = [&](const A8Req &q) { return (long long)H * q.units * length_of(q); };
  long long mine = 0;
  for (int i = i0; i < i1; i++) mine += size_of(a8_req<HS, R>(a, lb, i));
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
  const long long per = max((long long)max(grid.min_tiles, 1), (total + grid.ctas - 1) / grid.ctas);
  const long long begin = per * blockIdx.x, end = min(total, begin + per);
  A8Record *records = static_cast<A8Record *>(a.ws);
  float *parts = reinterpret_cast<float *>(records + grid.ctas);
  if (tid == 0 && !by_unit) records[blockIdx.x].first = -1;
  if (begin >= end) return;
  if (begin >= excl && begin < excl + mine) {
    long long p = excl;
    for (int i = i0; i < i1; i++) {
      const long long size = size_of(a8_req<HS, R>(a, lb, i));
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
  long long base = s_before;  // where the request's run begins
  A8Req q = a8_req<HS, R>(a, lb, req);

  for (long long at = begin; at < end;) {
    // The unit at `at`, and this CTA's tiles of it.
    while (at >= base + size_of(q)) {
      base += size_of(q);
      q = a8_req<HS, R>(a, lb, ++req);
    }
    const int step = length_of(q);
    const long long in = at - base;
    const int u = in >> 32 ? (int)(in / step) : (int)((uint32_t)in / (uint32_t)step);
    const int head = u / q.units, rg = u % q.units;
    const long long u0 = base + (long long)u * step, u1 = u0 + step;
    // A tile is that CTA's in whose run it begins.
    const int rw = q.rw, log_rw = rw >> 1, tw = kA8Warps / rw;
    const int t0 = by_unit ? 0 : (max(0, (int)(at - u0) - kA8Begin) + rw - 1) >> log_rw;
    const int t1 = by_unit ? q.tiles : ((int)(min(end, u1) - u0) - kA8Begin + rw - 1) >> log_rw;
    if (t1 <= 0) break;  // the run ends before the unit's first tile
    if (t0 >= q.tiles) {  // and begins behind the start of its last
      at = u1;
      continue;
    }
    const int wr = warp % rw, wt = warp / rw;
    const int row0 = (rg * rw + wr) * R;        // of the request's nq·G rows (token-major)
    const int all_rows = q.nq * G;

    const int unit_row0 = rg * rw * R, unit_rows = min(rw * R, all_rows - unit_row0);

    // Limits of this lane's query columns: visible tokens are (low, high].
    // Columns past the last row see all (their queries are zeros, their sums
    // are not stored).
    const int pos0 = q.last - (q.nq - 1);
    int high[NT][2], low[NT][2], high_max = -1, high_min = 0x7fffffff, low_max = -1;
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int e = 0; e < 2; e++) {
        const int row = row0 + 8 * n + 2 * c + e;
        high[n][e] = 0x7fffffff;
        low[n][e] = -1;
        if (row < all_rows) {
          const int pos = pos0 + token_of(row);
          high[n][e] = max(-1, min(pos, q.len - 1));
          if (a.window > 0 && pos >= a.window) low[n][e] = pos - a.window;
          high_max = max(high_max, high[n][e]);
        }
        high_min = min(high_min, high[n][e]);
        low_max = max(low_max, low[n][e]);
      }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      high_max = max(high_max, __shfl_xor_sync(0xffffffffu, high_max, o));
      high_min = min(high_min, __shfl_xor_sync(0xffffffffu, high_min, o));
      low_max = max(low_max, __shfl_xor_sync(0xffffffffu, low_max, o));
    }
    // The same of the whole unit: the tiles that its warps go through together.
    const int reach = max(-1, min(pos0 + token_of(unit_row0 + unit_rows - 1), q.len - 1));
    const int pos_first = pos0 + token_of(unit_row0);
    const int seen = a.window > 0 && pos_first >= a.window ? min(q.len, pos_first - a.window + 1) : 0;  // its first token
    const int t_first = max(t0, seen / TT - q.tile0);
    const int t_end = min(t1, reach / TT + (reach >= 0) - q.tile0);

    // A group of rw warps shares the tiles t_first + wt, + tw, ..., and copies
    // each together while it works on the one before. page[h] is the page of
    // the copied tile's tokens 16h.. (one page from 32 tokens on). A page
    // outside the cache is left out: page 0 is copied in its place, and masked;
    // so is a page of 16 tokens that no row of the unit sees (in front of the
    // windows or behind the last row), whose entry is not read.
    char *ring = sm + wt * 2 * Shape::TILE;
    const int *table = a.table + (int64_t)req * a.max_blocks;
    const uint32_t page_bytes = (uint32_t)(H * HS) << lb;
    // A lane's piece of 16 bytes: of the keys, 32 side by side; of the values,
    // dimension lane / 2, half lane % 2 of the tile's tokens.
    const int8_t *k_lane = a.c.k + (((int64_t)head * HS) << lb) + 16 * lane;
    const int8_t *v_lane = a.c.v + (((int64_t)head * HS + (lane >> 1)) << lb) + 16 * (lane & 1);
    const int key_piece = (16 * lane) ^ key_swizzle<HS>(16 * lane / HS);
    const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring);
    int page[2];  // -1: left out
    float ks = 0.0f, vs = 0.0f;  // scales of the next tile, of the page of this lane's tokens
    bool live = false;
    auto look_up = [&](int t) {
      page[0] = page[1] = -1;
      if (t < t_end) {
        const int tok = (q.tile0 + t) * TT;
        bool wrong = false;
        if (lb > 4 || tok + 16 > seen) {
          page[0] = __ldg(table + (tok >> lb));
          wrong = (unsigned)page[0] >= (unsigned)a.c.blocks;
          if (wrong) page[0] = -1;
        }
        if (lb > 4) {
          page[1] = page[0];
        } else if (tok + 16 <= reach) {
          page[1] = __ldg(table + (tok >> lb) + 1);
          if ((unsigned)page[1] >= (unsigned)a.c.blocks) wrong = true, page[1] = -1;
        }
        if (wrong) atomicExch(a.err, DEV_ERR_RANGE);
      }
    };
    // The copies of a tile: piece i of a lane, by constant offsets where the
    // warp copies all, every rw-th by a loop.
    auto copy_pieces = [&](auto log, uint32_t dst, const int8_t *k0, const int8_t *k1, const int8_t *v0) {
      constexpr int LB = decltype(log)::value;
      auto copy_piece = [&](int i) {
        const int8_t *k = LB > 4 || (KS % 2 ? 32 * i + lane < HS : 2 * i < KS) ? k0 : k1;
        copy16(dst + key_piece + 512 * i, k + 512 * i);
        copy16(dst + Shape::KBYTES + 16 * lane + 512 * i, v0 + (16 << LB) * i);
      };
      if (rw == 1) {
#pragma unroll
        for (int i = 0; i < KS; i++) copy_piece(i);
      } else {
#pragma unroll 1
        for (int i = wr; i < KS; i += rw) copy_piece(i);
      }
    };
    auto copy_tile = [&](int t, int stage) {  // page[] is the tile's
      if (t < t_end) {
        const uint32_t dst = ring_at + stage * Shape::TILE;
        const int in_page = ((q.tile0 + t) * TT) & ((1 << lb) - 1);
        const int64_t p0 = (int64_t)((uint64_t)(uint32_t)max(page[0], 0) * page_bytes);
        const int8_t *k0 = k_lane + p0 + in_page * HS, *v0 = v_lane + p0 + in_page;
        if (lb == 6) {
          copy_pieces(std::integral_constant<int, 6>(), dst, k0, k0, v0);
        } else if (lb == 5) {
          copy_pieces(std::integral_constant<int, 5>(), dst, k0, k0, v0);
        } else if (lb == 7) {
          copy_pieces(std::integral_constant<int, 7>(), dst, k0, k0, v0);
        } else {
          const int64_t p1 = (int64_t)((uint64_t)(uint32_t)max(page[1], 0) * page_bytes);
          copy_pieces(std::integral_constant<int, 4>(), dst, k0, k_lane + p1 - 16 * HS, lane & 1 ? v_lane + p1 - 16 : v0);
        }
      }
      copy_commit();
    };
    auto load_scales = [&](int t) {
      const int p = page[r >> 2];
      live = t < t_end && p >= 0;
      const int64_t ph = (int64_t)max(p, 0) * H + head;
      ks = live ? __ldg(a.c.k_scale + ph) : 0.0f;
      vs = live ? __ldg(a.c.v_scale + ph) : 0.0f;
    };
    // The queries' loads, under way while the first tile is looked up.
    constexpr int QW = TERMS == 1 ? 2 : 4;  // one term: bfloat16 only
    uint32_t qbits[NT][KS][QW];
#pragma unroll
    for (int n = 0; n < NT; n++) {
      const int row = row0 + 8 * n + r;
#pragma unroll
      for (int s = 0; s < KS; s++)
#pragma unroll
        for (int b = 0; b < QW; b++) qbits[n][s][b] = 0;
      if (row < all_rows) {
        const int tq = token_of(row);
        const int64_t qi = (q.q0 + tq) * a.q_stride + (head * G + row - tq * G) * HS;
        if constexpr (TERMS == 2)
          if (type == RK_ACT_F32) by_stretch<HS>(c, LoadQuery<float, QW>{static_cast<const float *>(a.q) + qi, grid.vec_q, qbits[n]});
        if (TERMS == 1 || type != RK_ACT_F32)
          by_stretch<HS>(c, LoadQuery<uint16_t, QW>{static_cast<const uint16_t *>(a.q) + qi, grid.vec_q, qbits[n]});
      }
    }
    int t = t_first + wt;
    look_up(t);
    load_scales(t);
    copy_tile(t, 0);
    look_up(t + tw);

    // Query fragments: in registers, or (two tiles of rows) in shared memory.
    uint32_t qb[NT > 1 ? 1 : NT][DIGITS][KS + KS % 2];
    uint2 *const q_mine = reinterpret_cast<uint2 *>(sm + Smem::RINGS + warp * Smem::QUERY) + lane;
    const uint32_t q_at = (uint32_t)__cvta_generic_to_shared(q_mine);
    float f[NT][2];
#pragma unroll
    for (int n = 0; n < NT; n++) {
      float v[KS][4];
#pragma unroll
      for (int s = 0; s < KS; s++) {
        if constexpr (TERMS == 2)
          if (type == RK_ACT_F32) {
#pragma unroll
            for (int b = 0; b < 4; b++) v[s][b] = u2f(qbits[n][s][b]);
            continue;
          }
#pragma unroll
        for (int b = 0; b < 2; b++) {
          const float2 x = TERMS == 2 ? act_pair<__half>(qbits[n][s][b]) : act_pair<__nv_bfloat16>(qbits[n][s][b]);
          v[s][2 * b] = x.x, v[s][2 * b + 1] = x.y;
        }
      }
      // The largest magnitude, as bits: infinities and NaN come out on top.
      uint32_t most = 0;
#pragma unroll
      for (int s = 0; s < KS; s++)
#pragma unroll
        for (int b = 0; b < 4; b++) most = max(most, f2u(v[s][b]) & 0x7fffffffu);
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
      // The row as integers of DIGITS signed bytes, its largest at the top. (Of
      // a row that is not finite any integers: its factor makes its scores NaN.)
      // Three bytes hold 127·65793; two less, since the product's rounding may add one.
      constexpr float LIMIT = DIGITS == 2 ? 127 * 257 : 127 * 65793 - 2;
      const float top = fmaxf(u2f(most), u2f(27u << 23));  // 2^-100: the quotients stay finite
      const float up = LIMIT / top;
      const float fr = most >= 0x7f800000u ? u2f(kCanonNaN) : (top * (1.0f / LIMIT)) * (a.scale * 1.44269504088896f);
      f[n][0] = __shfl_sync(0xffffffffu, fr, 8 * c);
      f[n][1] = __shfl_sync(0xffffffffu, fr, 8 * c + 4);
#pragma unroll
      for (int s = 0; s < KS; s++) {
        uint32_t w[4];
#pragma unroll
        for (int b = 0; b < 4; b++)
          w[b] = DIGITS == 2 ? f2u(fmaf(v[s][b], up, 12582912.0f)) : (uint32_t)__float2int_rn(v[s][b] * up);
        // The lowest byte as a signed one; the rest is a multiple of 256: the
        // next byte of w + 128, and that of w + 128 + 128·256.
        qb[NT > 1 ? 0 : n][DIGITS - 1][s] = pack_bytes(w[0], w[1], w[2], w[3]);
#pragma unroll
        for (int b = 0; b < 4; b++) w[b] += 0x80u;
        qb[NT > 1 ? 0 : n][DIGITS - 2][s] = prmt(prmt(w[0], w[1], 0x0051), prmt(w[2], w[3], 0x0051), 0x5410);
        if constexpr (DIGITS == 3) {
#pragma unroll
          for (int b = 0; b < 4; b++) w[b] += 0x8000u;
          qb[NT > 1 ? 0 : n][0][s] = prmt(prmt(w[0], w[1], 0x0062), prmt(w[2], w[3], 0x0062), 0x5410);
        }
      }
      if (KS % 2)
#pragma unroll
        for (int x = 0; x < DIGITS; x++) qb[NT > 1 ? 0 : n][x][KS] = 0;
      if constexpr (NT > 1)
#pragma unroll
        for (int x = 0; x < DIGITS; x++)
#pragma unroll
          for (int s = 0; s < KS; s += 2)
            q_mine[((n * DIGITS + x) * ((KS + 1) / 2) + s / 2) * 32] = make_uint2(qb[0][x][s], qb[0][x][s + 1]);
    }

    float o[NT][ND / 2][4], m[NT][2], M[NT][2], l[NT][2];
#pragma unroll
    for (int n = 0; n < NT; n++) {
#pragma unroll
      for (int d = 0; d < ND / 2; d++) o[n][d][0] = o[n][d][1] = o[n][d][2] = o[n][d][3] = 0.0f;
      m[n][0] = m[n][1] = M[n][0] = M[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.0f;
    }
    for (int it = 0; t < t_end; t += tw, it ^= 1) {
      copy_wait<0>();
      if (rw == 1) __syncwarp();
      else asm volatile("bar.sync %0, %1;" ::"r"(1 + wt), "r"(32 * rw) : "memory");
      float cks = ks, cvs = vs;
      const bool clive = live;
      load_scales(t + tw);
      copy_tile(t + tw, it ^ 1);
      look_up(t + 2 * tw);
      const int tok0 = (q.tile0 + t) * TT;
      if (tok0 > high_max) continue;  // in reach of other warps' rows only

      const uint32_t kt = ring_at + it * Shape::TILE + (8 * (r >> 1) + (r & 1)) * HS, vt = ring_at + it * Shape::TILE + Shape::KBYTES + r * TT + 8 * c;
      float sc[2][NT][4];
#pragma unroll
      for (int s = 0; s < 2; s++) {
        // Token of row r (and r + 8) of the 16: 8 (r/2) + 4s + r%2 (and + 2).
        uint32_t kw[2][KS + KS % 2];
#pragma unroll
        for (int j = 0; j < 2; j++) {
          load_row<HS>(kt + (4 * s + 2 * j) * HS, key_swizzle<HS>(r), c, kw[j]);
          if (KS % 2) kw[j][KS] = 0;
        }
        int si[DIGITS][NT][4];
#pragma unroll
        for (int k = 0; k < KS; k += 2) {
          const uint32_t ka[4] = {kw[0][k], kw[1][k], kw[0][k + 1], kw[1][k + 1]};
#pragma unroll
          for (int n = 0; n < NT; n++)
#pragma unroll
            for (int x = 0; x < DIGITS; x++) {
              uint2 b;
              if constexpr (NT > 1) b = lds64(q_at + ((n * DIGITS + x) * ((KS + 1) / 2) + k / 2) * 256);
              else b = make_uint2(qb[n][x][k], qb[n][x][k + 1]);
              if (k == 0) mma16832_first(si[x][n], ka, b.x, b.y);
              else mma16832(si[x][n], ka, b.x, b.y);
            }
        }
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int x = 0; x < 4; x++) {
            if constexpr (DIGITS == 2) sc[s][n][x] = (float)(256 * si[0][n][x] + si[1][n][x]);
            else sc[s][n][x] = fmaf((float)si[0][n][x], 65536.0f, (float)(256 * si[1][n][x] + si[DIGITS - 1][n][x]));
          }
      }
      // A scale that is not finite makes the scores NaN, where the page is
      // visible, and leaves the weights of zero elsewhere.
      if (!(fabsf(cks) < INFINITY && fabsf(cvs) < INFINITY)) cks = u2f(kCanonNaN), cvs = 0.0f;
      // vs = vf · 2^ve, vf with the sign; a scale of zero: weights of zero.
      const int ex = max(int(f2u(cvs) >> 23 & 255) - 127, -126);
      const float ve = cvs != 0.0f ? (float)ex : -1e30f;
      const float vf = cvs * u2f(uint32_t(127 - min(ex, 126)) << 23) * (ex > 126 ? 0.5f : 1.0f);
      const bool whole = __all_sync(0xffffffffu, clive) && tok0 + TT - 1 <= high_min && tok0 > low_max;

      // Scores in powers of two. m and M are references that stay while no
      // score passes them by much, so that most tiles need no exchange
      // between lanes.
      bool grew = false;
#pragma unroll
      for (int n = 0; n < NT; n++) {
        const float f0 = f[n][0] * cks, f1 = f[n][1] * cks;
#pragma unroll
        for (int s = 0; s < 2; s++) {
          sc[s][n][0] *= f0;
          sc[s][n][1] *= f1;
          sc[s][n][2] *= f0;
          sc[s][n][3] *= f1;
          if (!whole) {
            const int tok = tok0 + 8 * (r >> 1) + 4 * s + (r & 1);
#pragma unroll
            for (int x = 0; x < 4; x++) {
              const int k = tok + (x & 2);
              if (!clive || k > high[n][x & 1] || k <= low[n][x & 1]) sc[s][n][x] = -INFINITY;
            }
          }
        }
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const float mx = fmaxf(fmaxf(sc[0][n][e], sc[0][n][2 + e]), fmaxf(sc[1][n][e], sc[1][n][2 + e]));
          grew |= mx > m[n][e] + 20.0f || mx + ve > M[n][e];
        }
      }
      if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int e = 0; e < 2; e++) {
            float mn = fmaxf(fmaxf(sc[0][n][e], sc[0][n][2 + e]), fmaxf(sc[1][n][e], sc[1][n][2 + e]));
            float Mn = ve > -1e29f ? mn + (ve + 1.0f) : -INFINITY;
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) {
              mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, x));
              Mn = fmaxf(Mn, __shfl_xor_sync(0xffffffffu, Mn, x));
            }
            mn = fmaxf(mn, m[n][e]);
            Mn = fmaxf(Mn, M[n][e]);
            l[n][e] *= ex2(m[n][e] - (mn == -INFINITY ? 0.0f : mn));
            const float g = ex2(M[n][e] - (Mn == -INFINITY ? 0.0f : Mn));
#pragma unroll
            for (int d = 0; d < ND / 2; d++) {
              o[n][d][e] *= g;
              o[n][d][2 + e] *= g;
            }
            m[n][e] = mn;
            M[n][e] = Mn;
          }
      }
      uint32_t pb[2][NT][TERMS][2];
#pragma unroll
      for (int n = 0; n < NT; n++) {
        float ms[2], kap[2];
#pragma unroll
        for (int e = 0; e < 2; e++) {
          ms[e] = m[n][e] == -INFINITY ? 0.0f : m[n][e];
          kap[e] = ex2(fminf(ms[e] - (M[n][e] == -INFINITY ? 0.0f : M[n][e]) + 14.0f + ve, 120.0f)) * vf;
        }
#pragma unroll
        for (int s = 0; s < 2; s++) {
          float w[4];
#pragma unroll
          for (int x = 0; x < 4; x++) {
            const float p = ex2(sc[s][n][x] - ms[x & 1]);
            l[n][x & 1] += p;
            w[x] = p * kap[x & 1];
          }
#pragma unroll
          for (int j = 0; j < 2; j++) {
            const uint32_t h = pack_h2(w[2 * j], w[2 * j + 1]);
            pb[s][n][0][j] = transpose_h2(h);
            if constexpr (TERMS == 2) pb[s][n][1][j] = transpose_h2(pack_rest(w[2 * j], w[2 * j + 1], h));
          }
        }
      }
#pragma unroll
      for (int d = 0; d < ND / 2; d++) {
        // Tokens 8c .. 8c + 7 of two dimensions.
        const uint2 v0 = lds64(vt + 16 * d * TT);
        const uint2 v1 = lds64(vt + (16 * d + 8) * TT);
        // Two terms: a tile's sums of their own, added outside. The products'
        // adder does not round, and over thousands of tokens that shows
        // (6.7e-6 of a float32 result over 4600).
        float part[NT][4] = {};
#pragma unroll
        for (int s = 0; s < 2; s++) {
          uint32_t va[4];
          i8_to_h2(s ? v0.y : v0.x, va[0], va[2]);
          i8_to_h2(s ? v1.y : v1.x, va[1], va[3]);
#pragma unroll
          for (int n = 0; n < NT; n++)
#pragma unroll
            for (int x = TERMS - 1; x >= 0; x--) mma16816(TERMS == 2 ? part[n] : o[n][d], va, pb[s][n][x][0], pb[s][n][x][1]);
        }
        if (TERMS == 2)
#pragma unroll
          for (int n = 0; n < NT; n++)
#pragma unroll
            for (int x = 0; x < 4; x++) o[n][d][x] += part[n][x];
      }
    }
    copy_wait<0>();

    // The warps' sums meet in shared memory.
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int e = 0; e < 2; e++)
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], x);
    __syncthreads();  // the rings are free
    float *so = s_o + warp * R * PITCH, *st = s_st + warp * R * 4;
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int e = 0; e < 2; e++) {
        float *row = so + (8 * n + 2 * c + e) * PITCH + r;
#pragma unroll
        for (int d = 0; d < ND / 2; d++) {
          row[16 * d] = o[n][d][e];
          row[16 * d + 8] = o[n][d][2 + e];
        }
        if (r == 0) {
          float *x = st + 4 * (8 * n + 2 * c + e);
          x[0] = m[n][e];
          x[1] = M[n][e];
          x[2] = l[n][e];
        }
      }
    __syncthreads();
    const bool starts = t0 == 0, ends = t1 == q.tiles;
    float *part = parts + (2LL * blockIdx.x + (starts ? 1 : 0)) * a8_part_floats(HS);
    // Rows warp, warp + 4, ..., at most 16: lane i makes the i-th's factors.
    const int my_row = warp + kA8Warps * lane;
    float my_g[kA8Warps] = {}, my_scale = 0.0f;
    int64_t my_at = 0;
    if (my_row < unit_rows) {
      const float4 *s = reinterpret_cast<const float4 *>(s_st) + my_row;
      float mm = -INFINITY, MM = -INFINITY, ll = 0.0f;
      for (int w = 0; w < tw; w++) {
        mm = fmaxf(mm, s[w * rw * R].x);
        MM = fmaxf(MM, s[w * rw * R].y);
      }
      const float msafe = mm == -INFINITY ? 0.0f : mm, Msafe = MM == -INFINITY ? 0.0f : MM;
#pragma unroll
      for (int w = 0; w < kA8Warps; w++) {
        if (w >= tw) break;
        const float4 x = s[w * rw * R];
        ll += x.z * ex2(x.x - msafe);
        my_g[w] = ex2(x.y - Msafe);
      }
      my_scale = ll == 0.0f ? 0.0f : ex2(Msafe - 14.0f - msafe) / ll;
      const int qrow = unit_row0 + my_row, tq = token_of(qrow);
      my_at = (q.q0 + tq) * a.out_stride + (head * G + qrow - tq * G) * HS;
      if (!(starts && ends)) reinterpret_cast<float4 *>(part + 64 * HS)[my_row] = make_float4(mm, MM, ll, 0.0f);
    }
    for (int i = 0, row = warp; row < unit_rows; i++, row += kA8Warps) {
      const int64_t oi = __shfl_sync(0xffffffffu, my_at, i);
      const float scale = __shfl_sync(0xffffffffu, my_scale, i);
      float g[kA8Warps];
#pragma unroll
      for (int w = 0; w < kA8Warps; w++) g[w] = __shfl_sync(0xffffffffu, my_g[w], i);
      const float *so_row = s_o + row * PITCH;
      for (int d = 4 * lane; d < HS; d += 128) {
        float4 v = make_float4(0, 0, 0, 0);
#pragma unroll
        for (int w = 0; w < kA8Warps; w++) {
          if (w >= tw) break;
          const float4 x = *reinterpret_cast<const float4 *>(so_row + w * rw * R * PITCH + d);
          v.x = fmaf(x.x, g[w], v.x), v.y = fmaf(x.y, g[w], v.y);
          v.z = fmaf(x.z, g[w], v.z), v.w = fmaf(x.w, g[w], v.w);
        }
        if (starts && ends) o_store4(a.out, type, oi + d, make_float4(v.x * scale, v.y * scale, v.z * scale, v.w * scale), grid.vec_out);
        else *reinterpret_cast<float4 *>(part + row * HS + d) = v;
      }
    }
    if (!starts && tid == 0) {  // the CTA's first unit, begun in another one
      A8Record rec;
      rec.first = (int)((u0 + kA8Begin) / per);
      rec.last = (int)((u1 - rw) / per);
      rec.head = head;
      rec.row0 = unit_row0;
      rec.rows = unit_rows;
      rec.q0 = q.q0;
      rec.pad[0] = rec.pad[1] = 0;
      records[blockIdx.x] = rec;
    }
    at = min(end, u1);
    __syncthreads();  // the merge buffers are free
  }
}

// The instances for one number of float16 terms (each in a file of its own,
// to be compiled side by side).
template <int TERMS>
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
  // Two tiles of 8 rows a warp where the registers allow it: heads up to 128.
  template <int HS>
  static constexpr bool two_tiles() { return HS <= 128; }
  struct Init {
    template <int HS>
    cudaError_t operator()() const {
      cudaError_t e = cudaFuncSetAttribute(k_attn8<HS, TERMS, 1>, cudaFuncAttributeMaxDynamicSharedMemorySize, A8Smem<HS, 1, TERMS + 1>::ALL);
      if constexpr (two_tiles<HS>())
        if (e == cudaSuccess)
          e = cudaFuncSetAttribute(k_attn8<HS, TERMS, 2>, cudaFuncAttributeMaxDynamicSharedMemorySize, A8Smem<HS, 2, TERMS + 1>::ALL);
      return e;
    }
  };
  struct Launch {
    const Attn8Args &a;
    int type, nt;
    A8Grid g;
    cudaStream_t st;
    template <int HS>
    cudaError_t operator()() const {
      if constexpr (two_tiles<HS>())
        if (nt == 2) return launch_k(k_attn8<HS, TERMS, 2>, g.ctas, kA8Threads, (A8Smem<HS, 2, TERMS + 1>::ALL), st, a, type, g);
      return launch_k(k_attn8<HS, TERMS, 1>, g.ctas, kA8Threads, (A8Smem<HS, 1, TERMS + 1>::ALL), st, a, type, g);
    }
  };
  static cudaError_t init() {
    cudaError_t e = cudaSuccess;
    for (int hs : {16, 32, 48, 64, 80, 96, 112, 128, 256})
      if (e == cudaSuccess) e = at(hs, Init{});
    return e;
  }
};

cudaError_t attn8_init_two();
cudaError_t attn8_main_two(const Attn8Args &a, int type, int nt, A8Grid g, cudaStream_t st);

}  // namespace rk
