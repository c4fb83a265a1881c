// rk_serve.cu — C entry points of the serving operators: argument checks,
// the stream and the device, then a launch. They enqueue and return; nothing
// is allocated and no state is kept between calls (the 4-bit matrix handle
// aside), so any of them can be captured into a CUDA graph.
#include <cstdarg>
#include <cstdio>
#include <mutex>
#include <new>

#include "rk_serve.cuh"

namespace rk {
int internal_fail(int code, const char *msg);
void internal_device_view(const rk_device *d, int *ordinal, int *sms, void **stream, int **err_word);
void internal_device_count(rk_device *d, int64_t bytes);
int internal_device_check(rk_device *d);

cudaError_t init_serve_attributes() {
  cudaError_t e = init_paged_attributes();
  if (e == cudaSuccess) e = init_attn8_attributes();
  if (e == cudaSuccess) e = init_norm8_attributes();
  if (e == cudaSuccess) e = init_w4_attributes();
  return e;
}
}  // namespace rk

using namespace rk;

namespace {

int bad(const char *fmt, ...) {
  char buf[256];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  return internal_fail(RK_ERR_ARGS, buf);
}

// The device of a call: made current for its launches, and the caller's
// current device put back afterwards.
struct OnDevice {
  int ordinal = 0, sms = 0, before = -1;
  cudaStream_t st = nullptr;
  int *err = nullptr;
  cudaError_t e;
  OnDevice(const rk_device *d, void *stream) {
    void *own;
    internal_device_view(d, &ordinal, &sms, &own, &err);
    st = static_cast<cudaStream_t>(stream ? stream : own);
    e = cudaGetDevice(&before);
    if (e == cudaSuccess && before != ordinal) e = cudaSetDevice(ordinal);
  }
  ~OnDevice() {
    if (before >= 0 && before != ordinal) cudaSetDevice(before);
  }
  int done(cudaError_t launched, const char *what) const {
    const cudaError_t r = e != cudaSuccess ? e : launched;
    if (r == cudaSuccess) return RK_OK;
    char buf[256];
    snprintf(buf, sizeof buf, "%s: %s", what, cudaGetErrorString(r));
    return internal_fail(RK_ERR_CUDA, buf);
  }
};

// Held while a call's kernels that hand a workspace on are enqueued, so that
// those of two threads on one stream do not mix; by device.
std::mutex g_pairs[16];

bool aligned(const void *p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
size_t act_size(int type) { return type == RK_ACT_F32 ? 4 : 2; }
bool act_type(int type) { return type >= RK_ACT_F32 && type <= RK_ACT_BF16; }
bool block_ok(int b) { return b == 16 || b == 32 || b == 64 || b == 128; }

int check_cache(const rk_kv8 *c) {
  if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale) return bad("kv8: null cache");
  if (!block_ok(c->block)) return bad("kv8: pages of %d tokens (16, 32, 64 or 128)", c->block);
  if (c->head_size < 16 || c->head_size % 16 || (c->head_size > 128 && c->head_size != 256))
    return bad("kv8: head size %d (a multiple of 16 up to 128, or 256)", c->head_size);
  if (c->kv_heads < 1 || c->kv_heads > 65535) return bad("kv8: %d kv heads", c->kv_heads);
  if (c->blocks < 1 || (int64_t)c->blocks * c->block > 0x7fffffff) return bad("kv8: %d pages", c->blocks);
  if (!aligned(c->k, 16) || !aligned(c->v, 16) || !aligned(c->k_scale, 4) || !aligned(c->v_scale, 4))
    return bad("kv8: a misaligned cache buffer");
  return RK_OK;
}

}  // namespace

extern "C" int rk_device_check(rk_device *d, void *stream) {
  if (!d) return bad("null argument");
  OnDevice on(d, stream);
  const int rc = on.done(on.e == cudaSuccess ? cudaStreamSynchronize(on.st) : on.e, "device check");
  return rc ? rc : internal_device_check(d);
}

extern "C" int rk_page_tables(rk_device *d, int n, int block, const int32_t *ctx_lens, const int32_t *new_lens,
                              const int32_t *free_pages, const int32_t *free_head, int n_free, int32_t *table,
                              int max_blocks, int32_t *lens, int32_t *q_start, int32_t *slots, int32_t *positions,
                              int max_tokens, int32_t *info, void *stream) {
  if (!d || !q_start || !info) return bad("page tables: null argument");
  if (n < 0 || n > RK_MAX_REQUESTS) return bad("page tables: %d requests (at most %d)", n, RK_MAX_REQUESTS);
  if (!block_ok(block)) return bad("page tables: pages of %d tokens (16, 32, 64 or 128)", block);
  if (n_free < 0 || max_blocks < 0 || max_tokens < 0) return bad("page tables: a negative size");
  if ((n > 0 && (!ctx_lens || !new_lens || !lens)) || (n > 0 && max_blocks > 0 && !table) ||
      (n_free > 0 && !free_pages) || (max_tokens > 0 && (!slots || !positions)))
    return bad("page tables: null argument");
  for (const void *p : {(const void *)ctx_lens, (const void *)new_lens, (const void *)free_pages,
                        (const void *)free_head, (const void *)table, (const void *)lens, (const void *)q_start,
                        (const void *)slots, (const void *)positions, (const void *)info})
    if (!aligned(p, 4)) return bad("page tables: a misaligned buffer");
  // Every CTA reads the inputs for itself, while others write.
  const struct { const int32_t *p; int64_t n; bool out; const char *name; } bufs[] = {
      {ctx_lens, n, false, "ctx_lens"}, {new_lens, n, false, "new_lens"}, {free_pages, n_free, false, "free_pages"},
      {free_head, free_head ? 1 : 0, false, "free_head"}, {table, (int64_t)n * max_blocks, true, "table"}, {lens, n, true, "lens"},
      {q_start, (int64_t)n + 1, true, "q_start"}, {slots, max_tokens, true, "slots"}, {positions, max_tokens, true, "positions"},
      {info, 4, true, "info"}};
  for (const auto &a : bufs)
    for (const auto &b : bufs) {
      const uintptr_t pa = reinterpret_cast<uintptr_t>(a.p), pb = reinterpret_cast<uintptr_t>(b.p);
      if (&a != &b && b.out && a.n > 0 && b.n > 0 && pa < pb + 4 * (uint64_t)b.n && pb < pa + 4 * (uint64_t)a.n)
        return bad("page tables: %s and %s overlap", a.name, b.name);
    }
  OnDevice on(d, stream);
  TablesArgs a{n, block, n_free, max_blocks, max_tokens, ctx_lens, new_lens, free_pages, free_head,
               table, lens, q_start, slots, positions, info};
  return on.done(on.e == cudaSuccess ? launch_page_tables(a, on.sms, on.st) : on.e, "page tables");
}

extern "C" int rk_kv8_append(rk_device *d, const rk_kv8 *c, int type, int tokens, const void *k, int64_t k_stride,
                             const void *v, int64_t v_stride, const int32_t *slots, void *stream) {
  if (!d) return bad("kv8 append: null argument");
  if (int rc = check_cache(c)) return rc;
  if (!act_type(type)) return bad("kv8 append: unknown type %d", type);
  if (tokens < 0 || tokens > RK_KV8_MAX_ROWS) return bad("kv8 append: %d rows (at most %d)", tokens, RK_KV8_MAX_ROWS);
  if (tokens == 0) return RK_OK;
  if (!k || !v || !slots) return bad("kv8 append: null argument");
  const int64_t width = (int64_t)c->kv_heads * c->head_size;
  if (k_stride < width || v_stride < width) return bad("kv8 append: rows overlap (strides %lld, %lld; %lld values)",
                                                       (long long)k_stride, (long long)v_stride, (long long)width);
  if (!aligned(k, act_size(type)) || !aligned(v, act_size(type)) || !aligned(slots, 4))
    return bad("kv8 append: a misaligned buffer");
  OnDevice on(d, stream);
  AppendArgs a{*c, k, v, k_stride, v_stride, slots, tokens, on.err};
  return on.done(on.e == cudaSuccess ? launch_kv8_append(a, type, on.sms, on.st) : on.e, "kv8 append");
}

extern "C" int64_t rk_kv8_attention_workspace(rk_device *d, const rk_kv8 *c, int heads) {
  if (!d) return bad("kv8 attention: null argument");
  if (int rc = check_cache(c)) return rc;
  if (heads < 1 || heads % c->kv_heads) return bad("kv8 attention: %d heads over %d kv heads", heads, c->kv_heads);
  int ordinal, sms, *err;
  void *own;
  internal_device_view(d, &ordinal, &sms, &own, &err);
  return attn8_workspace(*c, sms);
}

extern "C" int rk_kv8_attention(rk_device *d, const rk_kv8 *c, int type, int n, int heads, int tokens, const void *q,
                                int64_t q_stride, const int32_t *q_start, const int32_t *lens, const int32_t *table,
                                int max_blocks, float scale, int window, void *out, int64_t out_stride,
                                void *workspace, int64_t workspace_bytes, void *stream) {
  if (!d) return bad("kv8 attention: null argument");
  if (int rc = check_cache(c)) return rc;
  if (!act_type(type)) return bad("kv8 attention: unknown type %d", type);
  if (heads < 1 || heads % c->kv_heads) return bad("kv8 attention: %d heads over %d kv heads", heads, c->kv_heads);
  if (n < 0 || n > RK_MAX_REQUESTS) return bad("kv8 attention: %d requests (at most %d)", n, RK_MAX_REQUESTS);
  if (tokens < 0 || max_blocks < 0 || window < 0) return bad("kv8 attention: a negative size");
  if (tokens > RK_KV8_MAX_ROWS || (int64_t)tokens * heads > 0x7fffffff)
    return bad("kv8 attention: %d rows of %d heads (at most %d rows, 2^31 - 1 in all)", tokens, heads, RK_KV8_MAX_ROWS);
  if (!q_start && tokens < n) return bad("kv8 attention: %d rows for %d requests of one each", tokens, n);
  if (!(scale >= 0.0f) || scale > 3.0e38f) return bad("kv8 attention: scale %g", (double)scale);
  if (n == 0 || tokens == 0) return RK_OK;
  if (!q || !lens || !out || (max_blocks > 0 && !table)) return bad("kv8 attention: null argument");
  const int64_t width = (int64_t)heads * c->head_size;
  if (q_stride < width || out_stride < width) return bad("kv8 attention: rows overlap");
  if (!aligned(q, act_size(type)) || !aligned(out, act_size(type)) || !aligned(q_start, 4) || !aligned(lens, 4) ||
      !aligned(table, 4))
    return bad("kv8 attention: a misaligned buffer");
  OnDevice on(d, stream);
  const int64_t need = (int64_t)max_blocks * c->block <= RK_KV8_NO_WORKSPACE ? 0 : attn8_workspace(*c, on.sms);
  if (workspace_bytes < need || (need > 0 && (!workspace || !aligned(workspace, 16))))
    return bad("kv8 attention: a workspace of %lld bytes, 16-byte aligned (%lld given)", (long long)need,
               (long long)workspace_bytes);
  Attn8Args a{*c, n, heads, tokens, max_blocks, window, q, out, q_stride, out_stride, q_start, lens, table, scale,
              workspace, on.err};
  if (scale == 0.0f) a.scale = (float)(1.0 / __builtin_sqrt((double)c->head_size));
  std::unique_lock<std::mutex> pair(g_pairs[on.ordinal & 15], std::defer_lock);
  if (need > 0) pair.lock();
  return on.done(on.e == cudaSuccess ? launch_kv8_attention(a, type, on.sms, on.st) : on.e, "kv8 attention");
}

extern "C" int rk_add_rmsnorm_q8(rk_device *d, int type, int rows, int cols, int group, const void *x,
                                 int64_t x_stride, const void *residual, int64_t r_stride, const void *weight,
                                 float eps, void *sum_out, int64_t s_stride, int8_t *q, float *scales, void *stream) {
  if (!d) return bad("norm q8: null argument");
  if (!act_type(type)) return bad("norm q8: unknown type %d", type);
  if (rows < 0 || cols < 1 || cols > RK_MAX_COLS) return bad("norm q8: %d×%d out of range", rows, cols);
  if (group == 0) group = cols;
  if (group < 1 || cols % group) return bad("norm q8: groups of %d in %d columns", group, cols);
  if (!(eps >= 0.0f)) return bad("norm q8: eps %g", (double)eps);
  if (rows == 0) return RK_OK;
  if (!x || !weight || !q || !scales) return bad("norm q8: null argument");
  if (x_stride < cols || (residual && r_stride < cols) || (sum_out && s_stride < cols))
    return bad("norm q8: rows overlap");
  if ((sum_out == x && sum_out && s_stride != x_stride) || (sum_out && sum_out == residual && s_stride != r_stride))
    return bad("norm q8: sums in place with another stride");
  const size_t es = act_size(type);
  if (!aligned(x, es) || !aligned(residual, es) || !aligned(weight, es) || !aligned(sum_out, es) || !aligned(scales, 4))
    return bad("norm q8: a misaligned buffer");
  OnDevice on(d, stream);
  Norm8Args a{rows, cols, group, x, residual, weight, sum_out, x_stride, r_stride, s_stride, eps, 1.0f / (float)cols, q, scales};
  return on.done(on.e == cudaSuccess ? launch_add_rmsnorm_q8(a, type, on.sms, on.st) : on.e, "norm q8");
}

// ---------------------------------------------------------------------------
// 4-bit matrices
// ---------------------------------------------------------------------------
struct rk_w4 {
  rk_device *d = nullptr;
  int rows = 0, cols = 0, group = 0, scale_type = 0;
  bool zeros = false;
  uint8_t *w = nullptr;
  int64_t bytes = 0;
};

extern "C" int rk_w4_upload(rk_device *d, int rows, int cols, int group, int scale_type, const uint8_t *w,
                            const void *scales, const uint8_t *zeros, rk_w4 **out) {
  if (!d || !w || !scales || !out) return bad("w4: null argument");
  if (!act_type(scale_type)) return bad("w4: unknown scale type %d", scale_type);
  if (rows < 1 || cols < 32 || cols % 32 || cols > RK_MAX_COLS || rows > RK_MAX_ROWS)
    return bad("w4: matrix %d×%d out of range", rows, cols);
  if (group < 32 || group % 32 || cols % group) return bad("w4: groups of %d in %d columns", group, cols);
  const size_t groups = (size_t)rows * (cols / group);
  if (zeros)
    for (size_t i = 0; i < groups; i++)
      if (zeros[i] > 15) return bad("w4: zero point %d is not four bits", zeros[i]);
  OnDevice on(d, nullptr);
  // The caller's order goes through a buffer of its own, freed at the end.
  const size_t wb = (size_t)rows * cols / 2, sb = groups * act_size(scale_type);
  const auto up = [](size_t n) { return (n + 255) & ~size_t(255); };
  const size_t total = up(w4_bytes(rows, cols, group, scale_type, zeros != nullptr));
  uint8_t *buf = nullptr, *raw = nullptr;
  cudaError_t e = on.e;
  if (e == cudaSuccess) e = cudaMalloc(&buf, total);
  if (e == cudaSuccess) e = cudaMalloc(&raw, up(wb) + up(sb) + groups);
  uint8_t *raw_s = raw + up(wb), *raw_z = zeros ? raw_s + up(sb) : nullptr;
  if (e == cudaSuccess) e = cudaMemcpyAsync(raw, w, wb, cudaMemcpyHostToDevice, on.st);
  if (e == cudaSuccess) e = cudaMemcpyAsync(raw_s, scales, sb, cudaMemcpyHostToDevice, on.st);
  if (e == cudaSuccess && zeros) e = cudaMemcpyAsync(raw_z, zeros, groups, cudaMemcpyHostToDevice, on.st);
  if (e == cudaSuccess) e = launch_w4_stream(raw, raw_s, raw_z, rows, cols, group, scale_type, buf, on.st);
  if (e == cudaSuccess) e = cudaStreamSynchronize(on.st);
  cudaFree(raw);
  rk_w4 *m = e == cudaSuccess ? new (std::nothrow) rk_w4() : nullptr;
  if (!m) {
    cudaFree(buf);
    if (e == cudaSuccess || e == cudaErrorMemoryAllocation) return internal_fail(RK_ERR_NOMEM, "w4: out of memory");
    return on.done(e, "w4 upload");
  }
  m->d = d;
  m->rows = rows;
  m->cols = cols;
  m->group = group;
  m->scale_type = scale_type;
  m->zeros = zeros != nullptr;
  m->w = buf;
  m->bytes = (int64_t)total;
  internal_device_count(d, m->bytes);
  *out = m;
  return RK_OK;
}

extern "C" void rk_w4_free(rk_w4 *m) {
  if (!m) return;
  OnDevice on(m->d, nullptr);
  cudaFree(m->w);  // waits for the device's work, so products in flight have ended
  internal_device_count(m->d, -m->bytes);
  delete m;
}

extern "C" int64_t rk_w4_bytes(const rk_w4 *m) { return m ? m->bytes : 0; }

extern "C" int rk_w4_mulvec(rk_w4 *m, int n, const int8_t *x, const float *x_scales, int x_group, int type, void *out,
                            int64_t out_stride, void *stream) {
  if (!m) return bad("w4: null argument");
  if (!act_type(type)) return bad("w4: unknown type %d", type);
  if (x_group == 0) x_group = m->cols;
  if (x_group < 32 || x_group % 32 || m->cols % x_group)
    return bad("w4: vectors in groups of %d in %d columns", x_group, m->cols);
  if (n < 0 || n > (1 << 20)) return bad("w4: %d vectors", n);
  if (n == 0) return RK_OK;
  if (!x || !x_scales || !out) return bad("w4: null argument");
  if (out_stride < m->rows) return bad("w4: output rows overlap");
  if (!aligned(x, 16) || !aligned(x_scales, 4) || !aligned(out, act_size(type))) return bad("w4: a misaligned buffer");
  OnDevice on(m->d, stream);
  W4Args a{m->rows, m->cols, m->group, x_group, n, m->scale_type, m->zeros, m->w, x, x_scales, out,
           out_stride};
  return on.done(on.e == cudaSuccess ? launch_w4_mulvec(a, type, on.sms, on.st) : on.e, "w4 product");
}
