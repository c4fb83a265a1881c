// rk_attn8_f32.cu — attention over the 8-bit paged cache: the kernels for
// float32 queries (two float16 terms).
#include "rk_attn8.cuh"

namespace rk {

cudaError_t attn8_init_f32() { return A8<true>::init(); }
cudaError_t attn8_main_f32(const Attn8Args &a, int type, A8Grid g, cudaStream_t st) {
  return A8<true>::at(a.c.head_size, A8<true>::Launch{a, type, g, st});
}

}  // namespace rk
