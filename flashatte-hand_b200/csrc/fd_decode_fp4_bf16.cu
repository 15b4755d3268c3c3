// fd_decode_fp4_bf16.cu - bf16-query instantiations of the 4-bit-cache decode kernel.
#include "fd_decode_fp4.cuh"

namespace fd {

cudaError_t launch_fp4_bf16(const Fp4DecodeParams& p, int head_dim, int grid, cudaStream_t stream) {
  return launch_fp4<__nv_bfloat16, __nv_bfloat16>(p, head_dim, grid, stream);
}

}  // namespace fd
