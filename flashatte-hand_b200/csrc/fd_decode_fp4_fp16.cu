// fd_decode_fp4_fp16.cu - fp16-query instantiations of the 4-bit-cache decode kernel.
#include "fd_decode_fp4.cuh"

namespace fd {

cudaError_t launch_fp4_fp16(const Fp4DecodeParams& p, int head_dim, int grid, cudaStream_t stream) {
  return launch_fp4<__half, __half>(p, head_dim, grid, stream);
}

}  // namespace fd
