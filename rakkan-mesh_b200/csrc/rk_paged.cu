// rk_paged.cu — page tables from request lengths, and the append of new keys
// and values into the 8-bit paged cache.
#include <cstring>

#include "rk_act.cuh"
#include "rk_matvec.cuh"
#include "rk_serve.cuh"

namespace rk {

// ---------------------------------------------------------------------------
// Page tables
// ---------------------------------------------------------------------------
// Two prefix sums over the requests (rows, then pages) and one value per row
// of the step. A step is a few kilobytes, so the call is all latency: one
// launch, in which every CTA makes both sums for itself from L2 (8 bytes a
// request) instead of waiting for another CTA's, and then writes its share
// of the rows, each thread finding its row's request by bisection. A step of
// 1024 requests of up to 96 new tokens takes 5.6 us, one of one request 3.6.
constexpr int kTabThreads = 512;

RK_DEV long long warp_scan(long long v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  return v;
}

// The sum of v over the threads before this one; *total: over all of them.
RK_DEV long long cta_scan(long long v, long long *sh, long long *total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long in = warp_scan(v, lane);
  __syncthreads();
  if (lane == 31) sh[warp] = in;
  __syncthreads();
  if (warp == 0) {
    const long long w = lane < kTabThreads / 32 ? sh[lane] : 0;
    const long long s = warp_scan(w, lane);
    if (lane < kTabThreads / 32) sh[lane] = s;
  }
  __syncthreads();
  *total = sh[kTabThreads / 32 - 1];
  return in - v + (warp ? sh[warp - 1] : 0);
}

__global__ void __launch_bounds__(kTabThreads) k_page_tables(TablesArgs a) {
  extern __shared__ int sm[];
  __shared__ long long sh[32];
  __shared__ int s_taken, s_refused;
  int *s_start = sm;             // [n + 1] first row of a request
  int *s_page = sm + a.n + 1;    // [n] place of its first new page behind the head; -1: refused
  const int n = a.n, B = a.block, tid = threadIdx.x;
  const int head = a.free_head ? *a.free_head : 0;
  const long long avail = head < 0 || head > a.n_free ? 0 : a.n_free - head;
  const long long room = (long long)a.max_blocks * B;
  const int per = (n + kTabThreads - 1) / kTabThreads, i0 = min(n, tid * per), i1 = min(n, i0 + per);
  if (tid == 0) s_taken = s_refused = 0;

  long long rows = 0, total, pages = 0, all_pages;
  for (int i = i0; i < i1; i++) rows += max(0, a.add[i]);
  long long at = cta_scan(rows, sh, &total);
  auto need_of = [&](int i, long long end, long long &ctx, long long &add) {
    ctx = max(0, a.ctx[i]);
    add = max(0, a.add[i]);
    const bool fits = end + add <= a.max_tokens && ctx + add <= room;
    return fits ? (ctx + add + B - 1) / B - (ctx + B - 1) / B : -1;
  };
  long long ctx, add, end = at;
  for (int i = i0; i < i1; i++) {
    const long long need = need_of(i, end, ctx, add);
    end += add;
    if (need > 0) pages += need;
  }
  long long before = cta_scan(pages, sh, &all_pages);
  end = at;
  int taken = 0, refused = 0;
  for (int i = i0; i < i1; i++) {
    const long long need = need_of(i, end, ctx, add);
    const bool served = need == 0 || (need > 0 && before + need <= avail);
    s_start[i] = (int)min(end, (long long)a.max_tokens);
    s_page[i] = served ? (int)min(before, 0x7fffffffLL) : -1;
    end += add;
    if (need > 0) before += need;
    if (served && need > 0) taken = (int)before;
    refused += !served;
    if (blockIdx.x == 0) {
      a.q_start[i] = s_start[i];
      a.lens[i] = served ? (int)(ctx + add) : 0;
    }
  }
  if (tid == 0) s_start[n] = (int)min(total, (long long)a.max_tokens);
  if (blockIdx.x == 0) {
    if (taken) atomicMax(&s_taken, taken);
    if (refused) atomicAdd(&s_refused, refused);
  }
  __syncthreads();
  const int used = s_start[n];
  if (blockIdx.x == 0 && tid == 0) {
    a.q_start[n] = used;
    a.info[0] = used;
    a.info[1] = s_taken;
    a.info[2] = s_refused;
    a.info[3] = head + s_taken;
  }

  for (long long t = (long long)blockIdx.x * kTabThreads + tid; t < a.max_tokens; t += (long long)gridDim.x * kTabThreads) {
    int slot = -1, pos = 0;
    if (t < used) {
      int lo = 0, hi = n;  // s_start[lo] <= t < s_start[hi]
      while (hi - lo > 1) {
        const int m = (lo + hi) >> 1;
        if (s_start[m] <= t) lo = m;
        else hi = m;
      }
      const int c = max(0, a.ctx[lo]);
      // Saturates for a refused request's far positions.
      pos = (int)min((long long)c + (t - s_start[lo]), 0x7fffffffLL);
      const int first = s_page[lo];
      if (first >= 0) {
        const int b = pos / B, old = (c + B - 1) / B;
        int *entry = a.table + (int64_t)lo * a.max_blocks + b;
        int page;
        if (b < old) {
          page = *entry;
        } else {
          page = a.free_pages[head + first + (b - old)];
          if (pos % B == 0) *entry = page;
        }
        const long long s = (long long)page * B + pos % B;
        if (page >= 0 && s <= 0x7fffffffLL) slot = (int)s;
      }
    }
    a.slots[t] = slot;
    a.positions[t] = pos;
  }
}

cudaError_t launch_page_tables(const TablesArgs &a, int sms, cudaStream_t st) {
  const long long want = ((long long)a.max_tokens + kTabThreads - 1) / kTabThreads;
  const int grid = want < 1 ? 1 : want > 2 * sms ? 2 * sms : (int)want;
  return launch_k(k_page_tables, grid, kTabThreads, sizeof(int) * (2 * (size_t)a.n + 1), st, a);
}

// ---------------------------------------------------------------------------
// Append
// ---------------------------------------------------------------------------
// A run is the consecutive rows of one page. One CTA takes a run's part for
// one kv head, of the keys or of the values: it finds the largest magnitude,
// then scales, rounds and stores. The bytes of the rows and of the cache bound
// the call. A run of up to 8192 values (a page of 64 tokens at head size 128) is
// loaded once, into registers; longer ones and rows off 16-byte boundaries are
// read twice, the second time from L1 or L2. The prompts of 16 sequences (8470
// tokens, 8 heads of 128, bfloat16) take 21.5 us, 2.4 TB/s, and 32.5 with every
// run read twice; what is left is each run's chain of load, maximum, store, and
// 59% of the issue slots. Values are stored transposed: the
// rounded bytes go through shared memory, from which 4 dimensions of 4 tokens
// become 4 words, with the tokens in the fast lanes, so that a page row's words
// are stored side by side. A CTA looks for the runs that begin in its `chunk`
// of rows (at most 32).
constexpr int kAppThreads = 128, kAppPieces = 8;  // a thread's pieces of eight values
constexpr int kAppHeld = kAppThreads * kAppPieces * 8;

RK_DEV float cta_max(float m, float *sh) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = m;
  __syncthreads();
  m = sh[0];
#pragma unroll
  for (int w = 1; w < kAppThreads / 32; w++) m = fmaxf(m, sh[w]);
  return m;
}

// e / d and e % d for a divisor that many e share.
struct Divisor {
  uint32_t d, m;
  RK_HD explicit Divisor(uint32_t n) : d(n), m(0xffffffffu / n + 1) {}  // d > 1, e·d < 2^32
  RK_DEV uint32_t quotient(uint32_t e) const { return __umulhi(e, m); }
  RK_DEV uint32_t rest(uint32_t e, uint32_t q) const { return e - q * d; }
};

// N neighbours of a row; vec: on a 16-byte boundary (N = 4 of 16 bits: of 8).
template <int N>
RK_DEV void load_n(const float *p, bool vec, float *v) {
  if (vec) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const float4 x = __ldg(reinterpret_cast<const float4 *>(p + i));
      v[i] = x.x, v[i + 1] = x.y, v[i + 2] = x.z, v[i + 3] = x.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = __ldg(p + i);
  }
}
template <int N, class T>
RK_DEV void load_n(const T *p, bool vec, float *v) {
  if (!vec) {
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = act_load(p + i);
    return;
  }
  uint32_t w[N / 2];
  if constexpr (N == 8) {
    const uint4 x = __ldg(reinterpret_cast<const uint4 *>(p));
    w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
  } else {
    const uint2 x = __ldg(reinterpret_cast<const uint2 *>(p));
    w[0] = x.x, w[1] = x.y;
  }
#pragma unroll
  for (int i = 0; i < N / 2; i++) {
    const float2 f = act_pair<T>(w[i]);
    v[2 * i] = f.x, v[2 * i + 1] = f.y;
  }
}
// The larger of top and |w|, as bits: of two values of 16 bits, each half by itself.
template <class T>
RK_DEV uint32_t max_bits(uint32_t top, uint32_t w) {
  if constexpr (sizeof(T) == 4) return max(top, w & 0x7fffffffu);
  else return __vmaxu2(top, w & 0x7fff7fffu);
}
// Their bytes; odd: infinities or NaN are among the run's values.
RK_DEV uint32_t quant4(const float *x, float inv, bool odd) {
  if (odd)
    return pack_bytes((uint32_t)quant127(x[0], inv), (uint32_t)quant127(x[1], inv), (uint32_t)quant127(x[2], inv),
                      (uint32_t)quant127(x[3], inv));
  return pack_bytes(quant127_bits(x[0], inv), quant127_bits(x[1], inv), quant127_bits(x[2], inv), quant127_bits(x[3], inv));
}
// Stored bytes times a ratio within ±1 (-1 makes 128 of -128, which stays 127).
RK_DEV uint32_t requant4(uint32_t w, float ratio) {
  const auto again = [&](uint32_t b) { return f2u(__fadd_rn(fminf(__fmul_rn((float)(int8_t)b, ratio), 127.0f), 12582912.0f)); };
  return pack_bytes(again(w), again(w >> 8), again(w >> 16), again(w >> 24));
}
// Bytes [from, to) of a word.
RK_DEV void store_bytes(int8_t *p, uint32_t w, int from, int to) {
  if (from <= 0 && to >= 4) {
    *reinterpret_cast<uint32_t *>(p) = w;
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; i++)
    if (i >= from && i < to) p[i] = (int8_t)(w >> (8 * i));
}

template <class T>
__global__ void __launch_bounds__(kAppThreads, sizeof(T) == 4 ? 4 : 6) k_kv8_append(AppendArgs a, int chunk, int log_block) {
  __shared__ float sh[kAppThreads / 32];
  __shared__ __align__(16) uint32_t s_rows[(kAppHeld + 128 * 4) / 4];  // rounded values, rows hs + 4 bytes apart
  // The CTAs of one run side by side: its rows lie together in memory.
  const int hs = a.c.head_size, H = a.c.kv_heads, B = 1 << log_block, lane = threadIdx.x & 31;
  const int part = blockIdx.x % (2 * H), head = part >> 1;
  const bool values = part & 1;
  const int cap = a.c.blocks << log_block;
  const T *x = static_cast<const T *>(values ? a.v : a.k) + (int64_t)head * hs;
  const int64_t stride = values ? a.v_stride : a.k_stride;
  const Divisor by8(hs >> 3);  // hs / 8 is at least 2
  const bool vec = stride * sizeof(T) % 16 == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0;
  int8_t *cache = values ? a.c.v : a.c.k;
  float *scales = values ? a.c.v_scale : a.c.k_scale;
  const int t0 = blockIdx.x / (2 * H) * chunk;

  // The rows at which runs begin, of this chunk.
  const int mine = t0 + lane < a.tokens && lane < chunk ? a.slots[t0 + lane] : -1;
  const int ahead = t0 + lane > 0 && mine >= 0 ? a.slots[t0 + lane - 1] : -1;
  const bool fits = mine >= 0 && mine < cap;
  if (mine >= cap && head == 0 && !values && threadIdx.x < 32) atomicExch(a.err, DEV_ERR_RANGE);
  unsigned begins =
      __ballot_sync(0xffffffffu, fits && !(ahead >= 0 && ahead < cap && ahead >> log_block == mine >> log_block));
  for (; begins; begins &= begins - 1) {
    const int t = t0 + __ffs(begins) - 1;
    const int slot = __shfl_sync(0xffffffffu, mine, __ffs(begins) - 1);
    const int page = slot >> log_block, first = slot & (B - 1);
    const int64_t ph = (int64_t)page * H + head;
    const float had = first > 0 ? scales[ph] : 0.0f;
    int rows = 0;          // of the run
    bool regular = true;   // its slots follow one another
    for (bool more = true; more;) {
      int s[4];  // one round trip for 128 rows
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int u = t + rows + 32 * i + lane;
        s[i] = u < a.tokens ? a.slots[u] : -1;
      }
      int n = 0;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const unsigned in = __ballot_sync(0xffffffffu, s[i] >= 0 && s[i] < cap && s[i] >> log_block == page);
        const int k = !more ? 0 : in == 0xffffffffu ? 32 : __ffs(~in) - 1;
        regular &= __all_sync(0xffffffffu, lane >= k || s[i] == slot + rows + 32 * i + lane);
        n += k;
        more &= k == 32;
      }
      rows += n;
    }

    // Held runs: magnitudes compare as their bits do, two of 16 bits at once,
    // and an infinity or a NaN comes out on top; such a run is read again.
    bool held = vec && regular && rows * hs <= kAppHeld, odd = false;
    const int pieces = rows * (hs >> 3);
    uint4 kept[kAppPieces][sizeof(T) / 2];
    float m = 0.0f;
    if (held) {
#pragma unroll
      for (int i = 0; i < kAppPieces; i++) {
        const int e = threadIdx.x + i * kAppThreads;
#pragma unroll
        for (int j = 0; j < sizeof(T) / 2; j++) kept[i][j] = make_uint4(0, 0, 0, 0);
        if (e < pieces) {
          const int r = by8.quotient(e);
          const uint4 *p = reinterpret_cast<const uint4 *>(x + (int64_t)(t + r) * stride + 8 * by8.rest(e, r));
#pragma unroll
          for (int j = 0; j < sizeof(T) / 2; j++) kept[i][j] = __ldg(p + j);
        }
      }
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < kAppPieces; i++)
#pragma unroll
        for (int j = 0; j < sizeof(T) / 2; j++) {
          const uint4 w = kept[i][j];
          top = max_bits<T>(max_bits<T>(max_bits<T>(max_bits<T>(top, w.x), w.y), w.z), w.w);
        }
      if (sizeof(T) == 2) top = max(top & 0xffff, top >> 16);
      T value;
      memcpy(&value, &top, sizeof(T));
      m = act_load(&value);
      odd = !(m < INFINITY);
      if (odd) m = 0.0f;
      held = !__syncthreads_or(odd);
    }
    if (!held) {
      m = 0.0f;
#pragma unroll 4
      for (int e = threadIdx.x; e < pieces; e += kAppThreads) {
        const int r = by8.quotient(e);
        float v[8];
        load_n<8>(x + (int64_t)(t + r) * stride + 8 * by8.rest(e, r), vec, v);
#pragma unroll
        for (int i = 0; i < 8; i++) {
          m = fmaxf(m, finite_abs(v[i]));
          odd |= !(fabsf(v[i]) < INFINITY);
        }
      }
      odd = __syncthreads_or(odd);
    }
    m = cta_max(m, sh);
    float scale = fmaxf(fabsf(had), __fmul_rn(m, u2f(K_1_127)));  // of a NaN and m: m's
    if (scale < u2f(K_TINY)) scale = 0.0f;
    const float inv = scale > 0.0f ? __fdiv_rn(1.0f, scale) : 0.0f;
    int8_t *pg = cache + ph * B * hs;

    if (had != scale) {  // earlier rows, to the larger scale
      float ratio = scale > 0.0f ? __fdiv_rn(had, scale) : 0.0f;
      if (ratio != ratio) ratio = 0.0f;
      if (!values) {
        for (int e = threadIdx.x; e < first * hs / 4; e += kAppThreads) {
          uint32_t *w = reinterpret_cast<uint32_t *>(pg) + e;
          *w = requant4(*w, ratio);
        }
      } else {
        const int words = (first + 3) >> 2;
        for (int e = threadIdx.x; e < words * hs; e += kAppThreads) {
          const int d = e / words, o = 4 * (e % words);
          int8_t *p = pg + d * B + o;
          store_bytes(p, requant4(*reinterpret_cast<const uint32_t *>(p), ratio), 0, first - o);
        }
      }
    }
    // Values to the page: f(row, dimension) are four dimensions' bytes of a row.
    // A word of the page is four tokens, the first and last perhaps in part.
    auto to_page = [&](auto f) {
      const int o0 = first & ~3, words = (first + rows + 3 - o0) >> 2;
      const Divisor by_words(max(words, 2));
      for (int e = threadIdx.x; e < words * (hs >> 2); e += kAppThreads) {
        const int n = words > 1 ? by_words.quotient(e) : e;
        const int o = words > 1 ? o0 + 4 * by_words.rest(e, n) : o0, d = 4 * n, r = o - first;
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; j++) w[j] = r + j >= 0 && r + j < rows ? f(r + j, d) : 0;
        // Byte i of the four rows: dimension d + i.
        const uint32_t lo01 = __byte_perm(w[0], w[1], 0x5140), hi01 = __byte_perm(w[0], w[1], 0x7362);
        const uint32_t lo23 = __byte_perm(w[2], w[3], 0x5140), hi23 = __byte_perm(w[2], w[3], 0x7362);
        const uint32_t t4[4] = {__byte_perm(lo01, lo23, 0x5410), __byte_perm(lo01, lo23, 0x7632), __byte_perm(hi01, hi23, 0x5410),
                                __byte_perm(hi01, hi23, 0x7632)};
        int8_t *to = pg + (d << log_block) + o;
        if (r >= 0 && r + 4 <= rows) {
#pragma unroll
          for (int i = 0; i < 4; i++) *reinterpret_cast<uint32_t *>(to + (i << log_block)) = t4[i];
        } else {
#pragma unroll
          for (int i = 0; i < 4; i++) store_bytes(to + (i << log_block), t4[i], -r, rows - r);
        }
      }
    };
    if (!regular) {  // a row after the other: of rows of one slot, the last stays
      for (int r = 0; r < rows; r++) {
        const int o = a.slots[t + r] & (B - 1);
        __syncthreads();
        for (int d = threadIdx.x; d < hs; d += kAppThreads)
          pg[values ? d * B + o : o * hs + d] = (int8_t)quant127(act_load(x + (int64_t)(t + r) * stride + d), inv);
      }
    } else if (held) {
#pragma unroll
      for (int i = 0; i < kAppPieces; i++) {
        const int e = threadIdx.x + i * kAppThreads;
        if (e < pieces) {
          float v[8];
          const uint32_t *w = reinterpret_cast<const uint32_t *>(kept[i]);
#pragma unroll
          for (int j = 0; j < 4; j++) {
            if constexpr (sizeof(T) == 4) {
              v[2 * j] = u2f(w[2 * j]), v[2 * j + 1] = u2f(w[2 * j + 1]);
            } else {
              const float2 f = act_pair<T>(w[j]);
              v[2 * j] = f.x, v[2 * j + 1] = f.y;
            }
          }
          const uint32_t w0 = quant4(v, inv, false), w1 = quant4(v + 4, inv, false);
          if (!values) {
            reinterpret_cast<uint2 *>(pg + first * hs)[e] = make_uint2(w0, w1);
          } else {
            const int r = by8.quotient(e), at = r * ((hs >> 2) + 1) + 2 * by8.rest(e, r);
            s_rows[at] = w0;
            s_rows[at + 1] = w1;
          }
        }
      }
      if (values) {
        __syncthreads();
        to_page([&](int r, int d) { return s_rows[r * ((hs >> 2) + 1) + (d >> 2)]; });
      }
    } else if (!values) {
#pragma unroll 4
      for (int e = threadIdx.x; e < pieces; e += kAppThreads) {
        const int r = by8.quotient(e);
        float v[8];
        load_n<8>(x + (int64_t)(t + r) * stride + 8 * by8.rest(e, r), vec, v);
        reinterpret_cast<uint2 *>(pg + first * hs)[e] = make_uint2(quant4(v, inv, odd), quant4(v + 4, inv, odd));
      }
    } else {
      __syncthreads();  // its bytes before the run have been written
      to_page([&](int r, int d) {
        float v[4];
        load_n<4>(x + (int64_t)(t + r) * stride + d, vec, v);
        return quant4(v, inv, odd);
      });
    }
    __syncthreads();  // every thread has read the old scale
    if (threadIdx.x == 0) scales[ph] = scale;
  }
}

cudaError_t launch_kv8_append(const AppendArgs &a, int type, int sms, cudaStream_t st) {
  const long long ctas = 2LL * a.tokens * a.c.kv_heads;
  int chunk = 1;  // rows a CTA looks through: more once every SM has several CTAs
  while (chunk < 32 && chunk < a.c.block && ctas / chunk > 32LL * sms) chunk *= 2;
  const long long ctas_all = (long long)((a.tokens + chunk - 1) / chunk) * 2 * a.c.kv_heads;
  if (ctas_all > 0x7fffffff) return cudaErrorInvalidValue;
  const dim3 grid((unsigned)ctas_all);
  const int lb = a.c.block == 16 ? 4 : a.c.block == 32 ? 5 : a.c.block == 64 ? 6 : 7;
  switch (type) {
    case RK_ACT_F32: return launch_k(k_kv8_append<float>, grid, kAppThreads, 0, st, a, chunk, lb);
    case RK_ACT_F16: return launch_k(k_kv8_append<__half>, grid, kAppThreads, 0, st, a, chunk, lb);
    default: return launch_k(k_kv8_append<__nv_bfloat16>, grid, kAppThreads, 0, st, a, chunk, lb);
  }
}

cudaError_t init_paged_attributes() {
  return cudaFuncSetAttribute(k_page_tables, cudaFuncAttributeMaxDynamicSharedMemorySize,
                              (int)(sizeof(int) * (2 * RK_MAX_REQUESTS + 1)));
}

}  // namespace rk
