// rk_attn8.cu — attention over the 8-bit paged cache.
#include "rk_act.cuh"
#include "rk_matvec.cuh"
#include "rk_serve.cuh"

namespace rk {

// A warp per (row, query head): lane j scores every 32nd key, the softmax
// runs over the 32 scores at a time, and each lane adds up its own
// dimensions of the weighted values.
constexpr int kAttnWarps = 4;

// The request of row t: the last i with q_start[i] <= t.
RK_DEV int request_of(const int *q_start, int n, int t) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int m = (lo + hi) >> 1;
    if (q_start[m] <= t) lo = m;
    else hi = m;
  }
  return lo;
}

template <class T>
__global__ void __launch_bounds__(32 * kAttnWarps) k_attn8_rows(Attn8Args a) {
  const int lane = threadIdx.x & 31, t = blockIdx.x, head = blockIdx.y * kAttnWarps + (threadIdx.x >> 5);
  if (head >= a.heads) return;
  const int B = a.c.block, hs = a.c.head_size, H = a.c.kv_heads, kvh = head / (a.heads / H);
  int req = t, pos;
  if (a.q_start) {
    req = request_of(a.q_start, a.n, t);
    if (t < a.q_start[0] || t >= a.q_start[req + 1]) return;
    pos = a.lens[req] - (a.q_start[req + 1] - t);
  } else {
    if (t >= a.n) return;
    pos = a.lens[req] - 1;
  }
  const T *q = static_cast<const T *>(a.q) + t * a.q_stride + (int64_t)head * hs;
  T *out = static_cast<T *>(a.out) + t * a.out_stride + (int64_t)head * hs;
  const int end = (int)min((long long)pos + 1, (long long)a.max_blocks * B);
  const int begin = a.window > 0 ? max(0, pos + 1 - a.window) : 0;
  float m = -INFINITY, l = 0.0f, acc[8];
  for (int d = 0; d < 8; d++) acc[d] = 0.0f;
  for (int k0 = begin; k0 < end; k0 += 32) {
    const int k = k0 + lane;
    float s = -INFINITY, vs = 0.0f;
    const int8_t *vp = nullptr;
    if (k < end) {
      const int page = a.table[(int64_t)req * a.max_blocks + k / B];
      if (page < 0 || page >= a.c.blocks) {
        atomicExch(a.err, DEV_ERR_RANGE);
      } else {
        const int64_t ph = (int64_t)page * H + kvh;
        const int8_t *kp = a.c.k + (ph * B + k % B) * hs;
        float dot = 0.0f;
        for (int d = 0; d < hs; d++) dot = fmaf(act_load(q + d), (float)kp[d], dot);
        s = dot * a.c.k_scale[ph] * a.scale;
        vs = a.c.v_scale[ph];
        vp = a.c.v + ph * B * hs + k % B;
      }
    }
    float top = s;
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float mn = fmaxf(m, top);
    if (mn == -INFINITY) continue;
    const float fix = exp2f((m - mn) * 1.44269504f);
    const float p = exp2f((s - mn) * 1.44269504f);
    m = mn;
    l *= fix;
    for (int d = 0; d < 8; d++) acc[d] *= fix;
    for (int j = 0; j < 32; j++) {
      const float pj = __shfl_sync(0xffffffffu, p, j);
      const float w = pj * __shfl_sync(0xffffffffu, vs, j);
      const int8_t *vj = (const int8_t *)__shfl_sync(0xffffffffu, (unsigned long long)vp, j);
      l += pj;
      if (vj)
        for (int d = 0; d < 8; d++)
          if (lane + 32 * d < hs) acc[d] = fmaf(w, (float)vj[(int64_t)(lane + 32 * d) * B], acc[d]);
    }
  }
  bool wrong = false;
  for (int d = lane; d < hs; d += 32) wrong |= !(fabsf(act_load(q + d)) < INFINITY);
  wrong = __any_sync(0xffffffffu, wrong) && end > begin;
  for (int d = 0; d < 8; d++)
    if (lane + 32 * d < hs) act_store(out + lane + 32 * d, wrong ? u2f(kCanonNaN) : l > 0.0f ? acc[d] / l : 0.0f);
}

int64_t attn8_workspace(const rk_kv8 &, int, int) { return 0; }

cudaError_t launch_kv8_attention(const Attn8Args &a, int type, int, cudaStream_t st) {
  const dim3 grid(a.tokens, (a.heads + kAttnWarps - 1) / kAttnWarps);
  switch (type) {
    case RK_ACT_F32: return launch_k(k_attn8_rows<float>, grid, 32 * kAttnWarps, 0, st, a);
    case RK_ACT_F16: return launch_k(k_attn8_rows<__half>, grid, 32 * kAttnWarps, 0, st, a);
    default: return launch_k(k_attn8_rows<__nv_bfloat16>, grid, 32 * kAttnWarps, 0, st, a);
  }
}

cudaError_t init_attn8_attributes() { return cudaSuccess; }

}  // namespace rk
