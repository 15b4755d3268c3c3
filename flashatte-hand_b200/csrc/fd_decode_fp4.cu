// fd_decode_fp4.cu - dispatch of the 4-bit-cache decode kernel to its
// instantiations (fd_decode_fp4_{bf16,fp16}[_f32].cu, split so that nvcc
// compiles them in parallel).
#include "fd_decode_fp4.cuh"

namespace fd {

// 16 query rows a pass double the multiplications of each byte of K and V but
// halve the passes (32 sequences of 4096 tokens, 16 rows a KV head: 63 us in
// one pass, 77 in two; up to 8 rows the second half would be idle: 47 us
// against 60); at head dim 256 their accumulators do not fit registers.
int fp4_rows(int head_dim, int64_t qrows) { return head_dim == 256 || qrows <= 8 ? 8 : 16; }

int fp4_max_grid(int head_dim, int rows, int sms) {
  int per_sm;
  switch (head_dim) {
    case 64: per_sm = rows == 16 ? Fp4Geo<64, 2>::kCtas : Fp4Geo<64, 1>::kCtas; break;
    case 128: per_sm = rows == 16 ? Fp4Geo<128, 2>::kCtas : Fp4Geo<128, 1>::kCtas; break;
    default: per_sm = Fp4Geo<256, 1>::kCtas; break;
  }
  return per_sm * sms;
}

cudaError_t launch_decode_fp4(const Fp4DecodeParams& p, int head_dim, int q_dtype, bool out_fp32,
                              int grid, cudaStream_t stream) {
  if (q_dtype == 0)
    return out_fp32 ? launch_fp4_bf16_f32(p, head_dim, grid, stream)
                    : launch_fp4_bf16(p, head_dim, grid, stream);
  return out_fp32 ? launch_fp4_fp16_f32(p, head_dim, grid, stream)
                  : launch_fp4_fp16(p, head_dim, grid, stream);
}

}  // namespace fd
