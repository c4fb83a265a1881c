// rk_paged.cu — page tables from request lengths, and the append of new keys
// and values into the 8-bit paged cache.
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
// of the rows, each thread finding its row's request by bisection.
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
  const int want = (a.max_tokens + kTabThreads - 1) / kTabThreads;
  const int grid = want < 1 ? 1 : want > 2 * sms ? 2 * sms : want;
  return launch_k(k_page_tables, grid, kTabThreads, sizeof(int) * (2 * (size_t)a.n + 1), st, a);
}

// ---------------------------------------------------------------------------
// Append
// ---------------------------------------------------------------------------
// A run is the consecutive rows of one page. One CTA takes a run's part for
// one kv head, of the keys or of the values: it finds the largest magnitude
// (first reading), then scales, rounds and stores (second reading, from L2
// or L1). A CTA looks for the runs that begin in its `chunk` of rows.
constexpr int kAppThreads = 128;

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

template <class T>
__global__ void __launch_bounds__(kAppThreads) k_kv8_append(AppendArgs a, int chunk) {
  __shared__ float sh[kAppThreads / 32];
  const int head = blockIdx.y, lane = threadIdx.x & 31;
  const bool values = blockIdx.z != 0;
  const int B = a.c.block, hs = a.c.head_size, H = a.c.kv_heads;
  const int cap = a.c.blocks * B;
  const T *x = static_cast<const T *>(values ? a.v : a.k) + (int64_t)head * hs;
  const int64_t stride = values ? a.v_stride : a.k_stride;
  int8_t *cache = values ? a.c.v : a.c.k;
  float *scales = values ? a.c.v_scale : a.c.k_scale;
  const int t0 = blockIdx.x * chunk, t1 = min(a.tokens, t0 + chunk);

  for (int t = t0; t < t1; t++) {
    const int slot = a.slots[t];
    if (slot < 0) continue;
    if (slot >= cap) {
      if (threadIdx.x == 0 && head == 0 && !values) atomicExch(a.err, DEV_ERR_RANGE);
      continue;
    }
    const int page = slot / B, first = slot % B;
    if (t > 0) {
      const int p = a.slots[t - 1];
      if (p >= 0 && p < cap && p / B == page) continue;  // within a run that begins earlier
    }
    int rows = 1;  // of the run
    for (;;) {
      const int u = t + rows + lane;
      const int s = u < a.tokens ? a.slots[u] : -1;
      const unsigned in = __ballot_sync(0xffffffffu, s >= 0 && s < cap && s / B == page);
      if (in != 0xffffffffu) {
        rows += __ffs(~in) - 1;
        break;
      }
      rows += 32;
    }
    float m = 0.0f;
    for (int e = threadIdx.x; e < rows * hs; e += kAppThreads)
      m = fmaxf(m, finite_abs(act_load(x + (int64_t)(t + e / hs) * stride + e % hs)));
    m = cta_max(m, sh);
    const int64_t ph = (int64_t)page * H + head;
    const float had = first > 0 ? scales[ph] : 0.0f;
    float scale = fmaxf(had, __fmul_rn(m, u2f(K_1_127)));
    if (scale < u2f(K_TINY)) scale = 0.0f;
    const float inv = scale > 0.0f ? __fdiv_rn(1.0f, scale) : 0.0f;
    int8_t *pg = cache + ph * B * hs;
    const int64_t step_o = values ? 1 : hs, step_d = values ? B : 1;  // of a token, of a dimension
    if (had != scale) {
      const float ratio = scale > 0.0f ? __fdiv_rn(had, scale) : 0.0f;
      for (int e = threadIdx.x; e < first * hs; e += kAppThreads) {
        int8_t *q = pg + (values ? (e % first) * step_o + (e / first) * step_d : e);
        *q = (int8_t)quant127((float)*q, ratio);
      }
    }
    for (int e = threadIdx.x; e < rows * hs; e += kAppThreads) {
      const int r = values ? e % rows : e / hs, d = values ? e / rows : e % hs;
      const int o = a.slots[t + r] % B;
      pg[o * step_o + d * step_d] = (int8_t)quant127(act_load(x + (int64_t)(t + r) * stride + d), inv);
    }
    __syncthreads();  // every thread has read the old scale
    if (threadIdx.x == 0) scales[ph] = scale;
  }
}

cudaError_t launch_kv8_append(const AppendArgs &a, int type, int sms, cudaStream_t st) {
  const long long ctas = 2LL * a.tokens * a.c.kv_heads;
  int chunk = 1;  // rows a CTA looks through: more once every SM has several CTAs
  while (chunk < a.c.block && ctas / chunk > 32LL * sms) chunk *= 2;
  const dim3 grid((a.tokens + chunk - 1) / chunk, a.c.kv_heads, 2);
  switch (type) {
    case RK_ACT_F32: return launch_k(k_kv8_append<float>, grid, kAppThreads, 0, st, a, chunk);
    case RK_ACT_F16: return launch_k(k_kv8_append<__half>, grid, kAppThreads, 0, st, a, chunk);
    default: return launch_k(k_kv8_append<__nv_bfloat16>, grid, kAppThreads, 0, st, a, chunk);
  }
}

cudaError_t init_paged_attributes() {
  return cudaFuncSetAttribute(k_page_tables, cudaFuncAttributeMaxDynamicSharedMemorySize,
                              (int)(sizeof(int) * (2 * RK_MAX_REQUESTS + 1)));
}

}  // namespace rk
