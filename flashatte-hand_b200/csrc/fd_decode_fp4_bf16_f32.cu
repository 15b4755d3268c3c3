// fd_decode_fp4_bf16_f32.cu - bf16-query instantiations of the 4-bit-cache decode kernel, fp32 output.
#include "fd_decode_fp4.cuh"

namespace fd {

cudaError_t launch_fp4_bf16_f32(const Fp4DecodeParams& p, int head_dim, int grid, cudaStream_t stream) {
  return launch_fp4<__nv_bfloat16, float>(p, head_dim, grid, stream);
}

}  // namespace fd
