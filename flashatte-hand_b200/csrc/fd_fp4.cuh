// fd_fp4.cuh - the 4-bit block-scaled cache format, shared by its kernels.
//
// A row of D values of one KV head is D / 16 blocks of 16 e2m1 codes (two per
// byte, the even element in the low half).  e2m1 has 1 sign, 2 exponent and 1
// mantissa bit: 0 .5 1 1.5 2 3 4 6.  Each block has an e4m3 scale and each KV
// head an fp32 scale g, so that value = e2m1 * e4m3 * g.  Quantising a block
// with largest magnitude a: scale s = e4m3(a / (6 g)), saturated at 448, code
// = e2m1(x / (s g)), both rounded to nearest even; s = 0 stores zeros.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp4.h>
#include <cuda_fp8.h>

#include <cstdint>

#include "fd_fp8.cuh"

namespace fd {

constexpr int kFp4Block = 16;  // values that share an e4m3 scale

// The four bytes of `w` (8 codes) as four f16 pairs, exactly.
__device__ __forceinline__ void e2m1x8_to_half2x4(uint32_t w, uint32_t (&h)[4]) {
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\tmov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\tcvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\tcvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(w));
}

// Two e4m3 bytes (low 16 bits) as an f16 pair, exactly.
__device__ __forceinline__ uint32_t e4m3x2_to_half2(uint32_t v) {
  uint32_t d;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(d) : "r"(v));
  return d;
}

__device__ __forceinline__ uint32_t hmul2_bits(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

__device__ __forceinline__ float e4m3_to_float(uint32_t v) { return e4m3x2_to_float2(v).x; }

}  // namespace fd
