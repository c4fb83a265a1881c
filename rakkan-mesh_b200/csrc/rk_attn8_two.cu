// rk_attn8_two.cu — attention over the 8-bit paged cache: the kernels with
// two float16 terms.
#include "rk_attn8.cuh"

namespace rk {

cudaError_t attn8_init_two() { return A8<2>::init(); }
cudaError_t attn8_main_two(const Attn8Args &a, int type, int nt, A8Grid g, cudaStream_t st) {
  return A8<2>::at(a.c.head_size, A8<2>::Launch{a, type, nt, g, st});
}

}  // namespace rk
