// rk_serve.cuh — launch interface of the serving operators (page tables,
// 8-bit paged cache, residual RMSNorm with 8-bit output, 4-bit products).
#pragma once
#include <cstdint>
#include <cuda_runtime.h>

#include "../../include/rakkan_cuda.h"

namespace rk {

struct TablesArgs {
  int n, block, n_free, max_blocks, max_tokens;
  const int *ctx, *add, *free_pages, *free_head;
  int *table, *lens, *q_start, *slots, *positions, *info;
};
cudaError_t launch_page_tables(const TablesArgs &a, int sms, cudaStream_t st);

struct AppendArgs {
  rk_kv8 c;
  const void *k, *v;
  int64_t k_stride, v_stride;
  const int *slots;
  int tokens;
  int *err;
};
cudaError_t launch_kv8_append(const AppendArgs &a, int type, int sms, cudaStream_t st);

struct Attn8Args {
  rk_kv8 c;
  int n, heads, tokens, max_blocks, window;
  const void *q;
  void *out;
  int64_t q_stride, out_stride;
  const int *q_start, *lens, *table;
  float scale;
  void *ws;
  int *err;
};
int64_t attn8_workspace(const rk_kv8 &c, int sms);  // of any number of heads
cudaError_t launch_kv8_attention(const Attn8Args &a, int type, int sms, cudaStream_t st);

struct Norm8Args {
  int rows, cols, group;
  const void *x, *residual, *weight;
  void *sum_out;
  int64_t x_stride, r_stride, s_stride;
  float eps, inv_cols;  // 1 / cols
  int8_t *q;
  float *scales;
};
cudaError_t launch_add_rmsnorm_q8(const Norm8Args &a, int type, int sms, cudaStream_t st);

struct W4Args {
  int rows, cols, group, x_group, n;
  int scale_type;
  bool zeros;        // zero points in the stream (else 8)
  const uint8_t *w;  // the stream of launch_w4_stream
  const int8_t *x;
  const float *x_scales;
  void *out;
  int64_t out_stride;
};
// Bytes of a matrix's stream, and the stream from the caller's order (device
// buffers; zeros may be null).
int64_t w4_bytes(int rows, int cols, int group, int scale_type, bool zeros);
cudaError_t launch_w4_stream(const uint8_t *w, const void *scales, const uint8_t *zeros, int rows, int cols, int group,
                             int scale_type, uint8_t *out, cudaStream_t st);
cudaError_t launch_w4_mulvec(const W4Args &a, int type, int sms, cudaStream_t st);

// Dynamic shared memory opt-ins (once per device, at open).
cudaError_t init_serve_attributes();
cudaError_t init_paged_attributes();
cudaError_t init_attn8_attributes();
cudaError_t init_norm8_attributes();
cudaError_t init_w4_attributes();

}  // namespace rk
