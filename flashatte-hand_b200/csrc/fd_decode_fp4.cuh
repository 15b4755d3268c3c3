// fd_decode_fp4.cuh - persistent split-KV paged decode over a 4-bit
// block-scaled cache (format: fd_fp4.cuh).  Device code and launch templates;
// fd_decode_fp4_*.cu instantiate it.
//
//   s_t = scale * k_scale * sum_d q_d (e2m1_td * kblock_td),  O = sum_t p_t v_t
//
// with v_t = v_scale * e2m1 * vblock and p = softmax(s).  A token and KV head
// costs D / 2 + D / 16 bytes of K and of V (72 + 72 at D = 128, against 512 in
// 16 bits), so the HBM-bound time is 0.28 of the 16-bit cache's; what it must
// not be bound by is the unpacking, which is the same count of values in a
// quarter of the time.
//
// Mathematics.  e2m1 * e4m3 has at most 6 significant bits and lies in
// [2^-10, 2688]: the product is exact in f16.  So K and V are dequantised to
// f16 without error and multiplied by the tensor cores (mma.sync m16n8k16,
// f16 in, fp32 out); the head scales and the softmax scale are fp32 factors
// of the logits and of O.  The query is f16 after scaling each row by a power
// of two that brings its largest magnitude to [2^13, 2^14): exact for fp16
// rows (not scaled) and for the bf16 values down to 2^-28 of the row's
// largest (smaller ones keep an absolute error of 2^-39 of it).  P enters
// as two f16 parts, the rounded value and the rounded rest: 2^-24 of each, and
// 2^-32 of the row's largest below that, so that fp32 outputs are worth their
// bits, as over the 16-bit caches.  Up to four query rows the parts lie side by
// side in a tile's 8 columns (FOLD), beyond that each is multiplied with V.
// One part alone (2^-11 of each weight): 64 sequences of 4096 tokens with 4
// rows 67.6 us instead of 70.1 (76.5 unfolded), config 3 with 8 rows 114
// instead of 131, 16 rows of 4 speculated tokens 40.8 instead of 45.8.
//
// Why mma.sync and not tcgen05: the dequantised tiles would have to be
// written to shared memory (2 bytes a value) and read back by the tensor
// core, 4 of the 4.6 bytes of shared-memory traffic a value; at HBM speed
// that is 170 B a cycle and SM, above the 128 it has.  In registers the
// operands go straight from the unpacking to the multiplication.
//
// Layout of the fragments.  S^T[token, row] = K . Q^T with 16 tokens x 8
// query rows a tile.  Lane (r = lane / 4, c = lane % 4) holds K's rows r and
// r + 8: it takes the D / 4 consecutive values c * D / 4 .. of the row, i.e.
// whole scale blocks, and the query fragment uses the same order, so the sum
// over d needs no shuffles.  O^T[d, row] = V^T . P^T: lane (r, c) takes the
// D / 8 consecutive values r * D / 8 .. of four tokens; a byte of one token
// and the byte of its neighbour give the pairs (t, t + 1) that the fragment
// wants.  P^T comes from S^T by movmatrix.  The tokens of a tile are numbered
// so that rows of both parities meet in a quarter-warp (tau below): with the
// swizzle of the rings K's and V's loads are free of bank conflicts.
//
// Loads.  A row of codes is D / 2 = 64 bytes at a stride of Hkv * 64: a TMA
// box of such rows was measured to move one row in about 5 cycles of the SM
// (4.0 TB/s in all at D = 128, 1.8 TB/s with the 32-byte rows of D = 64,
// however many boxes were in flight, from L2 as from HBM).  So the lanes copy
// 16 bytes each with cp.async, eight rows an instruction, past L1: 6.5 to 6.8
// TB/s for the loads alone.
//
// A CTA is four warps, and a schedule tile four 32-token stages, one a warp:
// HW = 2 neighbouring KV heads of the same tokens (1 where their number is odd,
// and in short launches), so that the warps together read 128-byte runs (one
// head a CTA costs 1.27 times the DRAM traffic, 104 instead of 69 us on config
// 2), times 4 / HW stages along the sequence.  Each warp has a ring and a
// softmax state of its own, and nothing in the loop waits for another warp.
// The ring runs across segments (a segment is the CTA's part of a sequence's
// heads): the next one's first loads are in flight while this one is written
// out.  Work split and the joining of segments on different CTAs are those of
// fd_decode_sm100.cuh, a head of a segment at a time.
//
// What bounds it.  32 tokens of K and V of a head at D = 128 are 4.6 KB, 765
// cycles of a quarter SM's share of the HBM, and with up to four rows 506
// instructions of a warp: 128 conversions of code pairs and 87 other ones on the
// half-rate ALU, 128 half-rate f16 multiplications, 32 mma, 38 loads and stores
// (with 5 to 8 rows 16 mma and some 20 others more).  Two warps a scheduler
// overlap these to 850 cycles (5.9 to 6.0 TB/s; no fewer from L2); three (3 CTAs
// an SM, 168 registers) were 10 to 17 % slower, with more segments for each.  So the loop is written for few instructions (the
// half-rate ones most of all): every five ALU instructions of it are a percent.
//
// Measured on a B200 (6.56 TB/s is its copy rate): 64 sequences of 4096 tokens,
// 32 over 8 heads, D = 128: 69.5 us as launches replayed back to back, 4.3 TB/s,
// and 75 as calls one after another on changing inputs; two of 262144: 119 us,
// 5.1 TB/s, and 137.  The fixed part of a launch is 20 us (first data after 6.4
// us: schedule 1.7, first page ids 2.0, query 1.0, data 1.6; 2 to 3 us for a
// segment's end, 1.5 to 6 for a joining, the rest ramps and imbalance).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "fd_fp4.cuh"
#include "fd_kernels.h"
#include "fd_ptx.cuh"
#include "fd_schedule.cuh"

namespace fd {

namespace {

constexpr int kFp4Threads = 128;
constexpr int kFp4Warps = kFp4Threads / 32;
constexpr int kSubTokens = 32;  // tokens of a stage
constexpr int kOffEntries = 34; // 16 stages' offsets, and a stage of none
constexpr int kSegRing = 8;     // segments that the loads may be ahead
// P is 2^kLift where its logit is the reference's largest, and its reference
// is raised when one is 2^kRaise: in f16's range with room at both ends.
constexpr int kLift = 7, kRaise = 15;
static_assert(kTileTokens == kFp4Warps * kSubTokens, "a schedule tile is a stage of each warp");

template <int D, int NT> struct Fp4Geo {
  static constexpr int kRowBytes = D / 2;
  static constexpr int kScaleBytes = D / 16;
  static constexpr int kTileBytes = kSubTokens * kRowBytes;
  static constexpr int kTileScales = kSubTokens * kScaleBytes;
  static constexpr int kStageBytes = 2 * kTileBytes + 2 * kTileScales;
  static constexpr int kRows = 8 * NT;
  // CTAs per SM (D = 64: 50.3 us for 64 sequences of 4096 tokens, 51.8 with 2),
  // and stages of a ring: enough for the HBM's latency; 4 at D = 128 and 5 at
  // D = 64 were within 1 % and not better
  static constexpr int kCtas = D == 64 ? 3 : 2;
  static constexpr int kStages = D == 64 ? 4 : D == 128 ? 3 : 2;
  static constexpr int kRowPad = D + 4;  // floats of a row of the join buffer
  static constexpr int kJoinWarp = kRows * kRowPad * 4 + kRows * 2 * 4;  // O, then maximum and sum of each row
  // the ring; what a warp's lanes share of its loads (page offsets of 16
  // stages, segments ahead); the join; lengths
  static constexpr int kOffOffs = kFp4Warps * kStages * kStageBytes;     // [warps][kOffEntries] code and scale offsets
  static constexpr int kOffSegs = kOffOffs + kFp4Warps * kOffEntries * 16;        // [warps][kSegRing]
  static constexpr int kOffJoin = kOffSegs + kFp4Warps * kSegRing * 32;  // [kFp4Warps - 1]
  static constexpr int kOffMisc = kOffJoin + (kFp4Warps - 1) * kJoinWarp;
  static constexpr int kOffPrefix = kOffMisc + 32;
  static constexpr int kOffLens = kOffPrefix + (kMaxBatchPerLaunch + 1) * 4;
  static constexpr int kSmemBytes = kOffLens + kMaxBatchPerLaunch * 4;
  static_assert(kSegRing > kStages + 1, "the loads run at most kStages segments ahead");
  static_assert(kSmemBytes + 1024 <= 233472 / kCtas, "shared memory of the resident CTAs");
  static_assert(kStageBytes % 16 == 0 && kOffMisc % 16 == 0 && kJoinWarp % 16 == 0, "alignment");
};

// 16 bytes from global to shared memory past L1, or zeros where `any` is 0.
__device__ __forceinline__ void copy16_or_zeros(uint32_t dst, const uint8_t* src, int any) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.eq.s32 p, %2, 0;\n\tcp.async.cg.shared.global [%0], [%1], 16, p;\n\t}" ::"r"(dst),
      "l"(src), "r"(any)
      : "memory");
}
// Two such copies where `any` is not 0, nothing otherwise.
__device__ __forceinline__ void copy16x2_if(uint32_t dst0, const uint8_t* src0, uint32_t dst1, const uint8_t* src1,
                                            int any) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.s32 p, %4, 0;\n\t"
      "@p cp.async.cg.shared.global [%0], [%1], 16;\n\t"
      "@p cp.async.cg.shared.global [%2], [%3], 16;\n\t}" ::"r"(dst0),
      "l"(src0), "r"(dst1), "l"(src1), "r"(any)
      : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                        uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
  return d;
}

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// (lo, hi) + f * h, with f an f16 number, rounded to f16.  For h = pack_half2(lo,
// hi) and f = -1: what that rounding left of both, exactly before its own.
constexpr uint16_t kMinusOne = 0xBC00;
__device__ __forceinline__ uint32_t pack_rest2(float lo, float hi, uint32_t h, uint16_t f) {
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\t"
      "fma.rn.f32.f16 %0, a, %3, %0;\n\tfma.rn.f32.f16 %1, b, %3, %1;\n\t}"
      : "+f"(lo), "+f"(hi)
      : "r"(h), "h"(f));
  return pack_half2(lo, hi);
}

// p + n * step in one instruction of the FMA pipe (a 64-bit addition is two of
// the ALU's, which bounds the loop).
__device__ __forceinline__ const uint8_t* plus_multiple(const uint8_t* p, uint32_t step, uint32_t n) {
  if (n == 0) return p;
  uint64_t d;
  asm("mad.wide.u32 %0, %1, %2, %3;" : "=l"(d) : "r"(step), "r"(n), "l"(reinterpret_cast<uint64_t>(p)));
  return reinterpret_cast<const uint8_t*>(d);
}

// (v's low half, twice), (its high half, twice): written like this the compiler
// makes them operand selections of the multiplication, no instructions.
__device__ __forceinline__ uint32_t low_twice(uint32_t v) {
  uint32_t d;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tmov.b32 %0, {lo, lo};\n\t}" : "=r"(d) : "r"(v));
  return d;
}
__device__ __forceinline__ uint32_t high_twice(uint32_t v) {
  uint32_t d;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tmov.b32 %0, {hi, hi};\n\t}" : "=r"(d) : "r"(v));
  return d;
}
// A shift by 4 that stays a multiplication, off the ALU.
__device__ __forceinline__ uint32_t times16(uint32_t v) {
  uint32_t d;
  asm("mad.lo.u32 %0, %1, 16, 0;" : "=r"(d) : "r"(v));
  return d;
}

// The low halves of a's bytes with the high halves of b's, in one instruction
// (from & and | the compiler makes two).
__device__ __forceinline__ uint32_t low_high(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, 0x0F0F0F0F, 0xE4;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

// 0xFF at the bytes of w that are NaN in e4m3
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return __vcmpeq4(w & 0x7F7F7F7Fu, 0x7F7F7F7Fu); }

// Keeps a value of the lane in its register: not computed again in the loop.
__device__ __forceinline__ void keep(int& v) { asm volatile("" : "+r"(v)); }
__device__ __forceinline__ void keep(uint32_t& v) { asm volatile("" : "+r"(v)); }

// Read from shared memory here and now: not hoisted, not kept in registers.
__device__ __forceinline__ int volatile_at(const int* p) { return *reinterpret_cast<const volatile int*>(p); }
__device__ __forceinline__ int4 volatile_at(const int4* p) {
  int4 v;
  asm volatile("ld.shared.v4.s32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(smem_u32(p))
               : "memory");
  return v;
}

template <typename T> __device__ __forceinline__ float2 pair_to_float2(uint32_t w);
template <> __device__ __forceinline__ float2 pair_to_float2<__nv_bfloat16>(uint32_t w) {
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w));
}
template <> __device__ __forceinline__ float2 pair_to_float2<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

// N words (1, 2 or 4) from shared memory in one load.
template <int N> __device__ __forceinline__ void load_words(const uint8_t* p, uint32_t (&w)[N]) {
  if constexpr (N == 1) {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else if constexpr (N == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x; w[1] = v.y;
  } else {
    static_assert(N == 4, "1, 2 or 4 words");
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  }
}

template <typename O> __device__ __forceinline__ uint32_t pack_out(float lo, float hi) {
  if constexpr (std::is_same<O, __half>::value) {
    return pack_half2(lo, hi);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

// N consecutive values, rounded once, in 16-byte stores.
template <typename O, int N> __device__ __forceinline__ void store_row(O* dst, const float (&x)[N]) {
  if constexpr (sizeof(O) == 4) {
#pragma unroll
    for (int i = 0; i < N; i += 4)
      *reinterpret_cast<float4*>(dst + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
  } else {
    static_assert(N % 8 == 0, "whole 16-byte stores");
#pragma unroll
    for (int i = 0; i < N; i += 8)
      *reinterpret_cast<uint4*>(dst + i) =
          make_uint4(pack_out<O>(x[i], x[i + 1]), pack_out<O>(x[i + 2], x[i + 3]), pack_out<O>(x[i + 4], x[i + 5]),
                     pack_out<O>(x[i + 6], x[i + 7]));
  }
}

// N = 2 or 4 consecutive values, as wide as they are: partials past L1, and
// the output, rounded once.
template <int N> __device__ __forceinline__ void load_vec(const float* src, float (&x)[N]) {
  if constexpr (N == 4) {
    const float4 y = __ldcg(reinterpret_cast<const float4*>(src));
    x[0] = y.x; x[1] = y.y; x[2] = y.z; x[3] = y.w;
  } else {
    static_assert(N == 2, "2 or 4 values");
    const float2 y = __ldcg(reinterpret_cast<const float2*>(src));
    x[0] = y.x; x[1] = y.y;
  }
}
template <typename O, int N> __device__ __forceinline__ void store_vec(O* dst, const float (&x)[N]) {
  if constexpr (sizeof(O) == 4) {
    if constexpr (N == 4) *reinterpret_cast<float4*>(dst) = make_float4(x[0], x[1], x[2], x[3]);
    else *reinterpret_cast<float2*>(dst) = make_float2(x[0], x[1]);
  } else {
    if constexpr (N == 4)
      *reinterpret_cast<uint2*>(dst) = make_uint2(pack_out<O>(x[0], x[1]), pack_out<O>(x[2], x[3]));
    else *reinterpret_cast<uint32_t*>(dst) = pack_out<O>(x[0], x[1]);
  }
}

// Place of 16-byte chunk `chunk` of row `row` in a tile of RB-byte rows: the
// chunks of a row are exchanged by the row, so that the loads of K (16 bytes
// of 8 rows) and of V (8 bytes of 4 rows) touch every bank once.
template <int RB> __device__ __forceinline__ int swizzled(int row, int chunk) {
  if constexpr (RB == 32) return chunk ^ ((row >> 2) & 1);
  else if constexpr (RB == 64) return chunk ^ ((row >> 1) & 3);
  else return chunk ^ (row & 7);
}

// MULTI: several query tokens, or a causal mask.  FOLD: at most four query rows;
// the second halves of the 8 columns hold them again, for P's second part.
template <typename T, typename OutT, int D, int NT, bool MULTI, bool FOLD>
__global__ void __launch_bounds__(kFp4Threads, Fp4Geo<D, NT>::kCtas)
    decode_fp4_kernel(const __grid_constant__ Fp4DecodeParams p) {
  using G = Fp4Geo<D, NT>;
  constexpr int RB = G::kRowBytes, SB = G::kScaleBytes;
  constexpr int KW = D / 32;        // words of K a lane takes from a row
  constexpr int VW = D / 64;        // words of V a lane takes from a token
  constexpr int MT = D / 16;        // 16-dim tiles of O^T
  constexpr int KS = D / 16;        // 16-dim steps of S^T
  constexpr int kParts = FOLD ? 1 : 2;  // products of V with parts of P
  static_assert(!FOLD || NT == 1, "four rows, twice");
  extern __shared__ __align__(16) uint8_t smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int r = lane >> 2, c = lane & 3;
  // the query row of the pass in column 2 c + e of tile nt
  auto row_of = [&](int nt, int e) { return FOLD ? (2 * c + e) & 3 : nt * 8 + 2 * c + e; };

  uint8_t* ring = smem + warp * G::kStages * G::kStageBytes;
  longlong2* offs = reinterpret_cast<longlong2*>(smem + G::kOffOffs) + warp * kOffEntries;
  int4* seg_ring = reinterpret_cast<int4*>(smem + G::kOffSegs) + warp * kSegRing * 2;
  unsigned long long* launch_epoch = reinterpret_cast<unsigned long long*>(smem + G::kOffMisc);
  volatile int* last_flag = reinterpret_cast<volatile int*>(smem + G::kOffMisc + 8);  // [2]
  int* align_word = reinterpret_cast<int*>(smem + G::kOffMisc + 16);
  int* prefix = reinterpret_cast<int*>(smem + G::kOffPrefix);
  int* lens = reinterpret_cast<int*>(smem + G::kOffLens);

  const int batch = p.batch, cta = blockIdx.x;
  const float neg_inf = -__int_as_float(0x7f800000);

  // ------------------------------------------------------------ prologue
  if (tid == 0) pdl_launch_dependents();
  const CostModel cm{p.cost_tile, p.cost_seg, 0};
  pdl_wait_prerequisites();
  unsigned long long epoch_ld = 0;
  if (tid == 0) epoch_ld = *reinterpret_cast<volatile unsigned long long*>(p.epoch_word);
  // Short launches: where every CTA's share is m = ceil(pairs / grid) whole
  // (sequence, KV head, row tile) pairs of at most align_tiles / m tiles of
  // kTileTokens, each CTA takes m whole pairs, a head at a time: no pair is
  // cut, so no partial, arrival or joining lengthens a launch that is one
  // latency chain (see fd_decode_sm100.cuh).
  const int pairs = batch * p.num_heads_k * p.row_tiles;
  const int align_m = (pairs + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x);
  const int align_max = p.align_tiles / align_m;
  bool is_short = align_max > 0;
  for (int b = tid; b < batch; b += kFp4Threads) {
    const int stored = __ldg(p.seqlens + b);
    const int64_t max_len = p.bt_stride * static_cast<int64_t>(p.page);
    const int64_t want = static_cast<int64_t>(stored < 0 ? 0 : stored) + p.len_add;
    const int64_t cap = max_len < 0x1fffffff ? max_len : 0x1fffffff;
    const int len = static_cast<int>(want > cap ? cap : want);
    lens[b] = len;
    is_short = is_short && seq_tiles(len) <= align_max;
  }
  const bool aligned = __syncthreads_and(is_short) != 0;
  const int HW = aligned ? 1 : p.heads, TW = kFp4Warps / HW;  // warps over heads, warps over tokens
  const int hw = warp & (HW - 1), tw = warp / HW;
  const int step = TW * kSubTokens;                           // tokens of a schedule tile
  // A pair of the schedule is (sequence, HW KV heads, row tile).  It counts
  // tiles of kTileTokens; a tile here is `step` tokens of HW heads, so lengths
  // are given to it times HW.
  for (int b = tid; b < batch; b += kFp4Threads) {
    const int len = lens[b] * HW;
    lens[b] = len;
    prefix[b + 1] = aligned ? cm.max_lead() + p.align_tiles * cm.full() + 1 : cm.pair_cost(len);
  }
  if (tid == 0) {
    prefix[0] = 0;
    *launch_epoch = epoch_ld & kEpochMax;
    *align_word = aligned ? align_m : 0;
  }
  __syncthreads();
  if (warp == 0) {
    int carry = 0;
    for (int base = 1; base <= batch; base += 32) {
      const int idx = base + lane;
      int v = idx <= batch ? prefix[idx] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
      }
      v += carry;
      if (idx <= batch) prefix[idx] = v;
      carry = __shfl_sync(0xffffffffu, v, 31);
    }
  }
  __syncthreads();
  // The schedule is asked at segment ends only: what it needs is read from
  // shared memory there, so that the loop's registers hold none of it.
  auto schedule = [&]() {
    Schedule x;
    x.cost_prefix = prefix;
    x.lens = lens;
    x.max_len = 0;
    x.total = static_cast<int64_t>(p.num_heads_k / HW * p.row_tiles) * volatile_at(prefix + p.batch);
    x.batch = p.batch;
    x.hkv = p.num_heads_k / HW * p.row_tiles;
    x.cm = CostModel{p.cost_tile, p.cost_seg, 0};
    x.behind_lead = true;
    x.align_m = volatile_at(align_word);
    x.align_cost = x.cm.max_lead() + p.align_tiles * x.cm.full() + 1;
    if (x.align_m > 0) {
      x.grid = (x.batch * x.hkv + x.align_m - 1) / x.align_m;
    } else {
      // every range longer than a tile: none inside a pair is empty
      const int64_t g = div_u32(x.total, x.cm.full() + 1);
      x.grid = static_cast<int>(g < 1 ? 1 : (g < gridDim.x ? g : gridDim.x));
    }
    return x;
  };

  // ------------------------------------------------------------ loads
  // The cursor of the loads, a ring ahead of the multiplication: pc_left
  // tiles of the segment entered last (seg_ring[seg_w - 1]) are left, the
  // next is its pc_k-th.  offs[2 i + g] are the byte offsets (codes; block
  // scales) of tokens 16 g .. of the warp's stage 16 n + i of the segment, plus
  // 16, or 0 where there is no page: no codes are copied then, and zeros as
  // scales; next_* the page id and row (-1: no tokens) of the same entry of
  // batch n + 1.  offs[32 .. 33] are a stage of none, for the rounds after the
  // last.
  int pc_left = 0, pc_end = 0, pc_k = 0, next_id = 0, next_row = -1, seg_w = 0;
  // A copy instruction moves 16 bytes a lane: half the lanes rows of K, half
  // of V, so that a lane needs one pointer; kCopies of them are 16 tokens.
  constexpr int kChunks = RB / 16;          // 16-byte chunks of a row of codes
  constexpr int kRowsPer = 16 / kChunks;    // rows of K, and of V, of one instruction
  constexpr int kCopies = 16 / kRowsPer;
  const int64_t row_bytes = static_cast<int64_t>(p.num_heads_k) * RB;
  const int lr = (lane & 15) / kChunks, lc = lane % kChunks;
  const uint8_t* code_src = (lane < 16 ? p.k_cache : p.v_cache) + lr * row_bytes + lc * 16 - 16;
  const uint32_t copy_step = kRowsPer * static_cast<uint32_t>(row_bytes);
  // ring places of the lane's row in the first copies; the swizzle of copy i
  // is that of copy i % kDstVariants
  constexpr int kDstVariants = RB == 128 ? 4 : 2;
  uint32_t code_dst[kDstVariants];
#pragma unroll
  for (int i = 0; i < kDstVariants; ++i) {
    code_dst[i] = smem_u32(ring) + (lane < 16 ? 0 : G::kTileBytes) + lr * RB +
                  swizzled<RB>(i * kRowsPer + lr, lc) * 16;
    keep(code_dst[i]);
  }
  // block scales: kScaleChunks 16-byte chunks of K, then of V (in two
  // instructions at D = 256); sg: the chunk's group of 16 tokens
  constexpr int kScaleChunks = G::kTileScales / 16;  // 8, 16 or 32
  constexpr int kScaleCopies = 2 * kScaleChunks > 32 ? 2 : 1;
  const int sx = lane % kScaleChunks, sg = sx / (kScaleChunks / 2);
  const uint8_t* scale_src =
      (kScaleCopies == 1 && lane >= kScaleChunks ? p.v_block : p.k_block) + (sx % (kScaleChunks / 2)) * 16 - 16;
  const uint32_t scale_dst = smem_u32(ring) + 2 * G::kTileBytes + lane * 16;
  auto entry = [&](int i) { return seg_ring + (i & (kSegRing - 1)) * 2; };
  auto segment_of = [&](int i) {
    const int4 x = volatile_at(entry(i)), y = volatile_at(entry(i) + 1);
    Segment g;
    g.b = x.x; g.kvh = x.y; g.tile0 = x.z; g.ntiles = x.w;
    g.seqlen = y.x; g.pair = y.y; g.nseg = y.z; g.cfirst = y.w;
    return g;
  };
  auto fetch_ids = [&](int k0) {  // batch of stages k0 ..
    const int4 x = volatile_at(entry(seg_w - 1));
    const int tok = (x.z + k0 + (lane >> 1)) * step + tw * kSubTokens + (lane & 1) * 16;
    next_row = -1;
    if (k0 + (lane >> 1) < x.w && tok < pc_end) {
      const uint32_t pg = static_cast<uint32_t>(tok) / static_cast<uint32_t>(p.page);
      next_row = static_cast<int>(static_cast<uint32_t>(tok) - pg * static_cast<uint32_t>(p.page));
      next_id = __ldg(p.block_table + x.x * p.bt_stride + pg);
    }
  };
  auto turn_batch = [&](int k0) {  // next_* become offs, and the batch after it is fetched
    __syncwarp();
    longlong2 o;
    o.x = o.y = 0;
    if (next_row >= 0 && (next_id < 0 || next_id >= p.num_blocks)) {
      report_status(p.err, kStatusBadPage);  // its rows are read as zeros
    } else if (next_row >= 0) {
      const int head = volatile_at(entry(seg_w - 1)).y / p.row_tiles * HW + hw;
      o.x = (static_cast<int64_t>(next_id) * p.page + next_row) * row_bytes + head * RB + 16;
      o.y = ((static_cast<int64_t>(next_id) * p.num_heads_k + head) * p.page + next_row) * SB + 16;
    }
    offs[lane] = o;
    __syncwarp();
    fetch_ids(k0 + 16);
  };
  auto enter = [&](const Segment& g) {  // publish a segment and prepare its loads
    __syncwarp();
    if (lane == 0) {
      entry(seg_w)[0] = make_int4(g.b, g.kvh, g.tile0, g.ntiles);
      entry(seg_w)[1] = make_int4(g.seqlen, g.pair, g.nseg, g.cfirst);
    }
    __syncwarp();
    ++seg_w;
    pc_left = g.ntiles;
    pc_end = g.seqlen / HW;
    pc_k = 0;
    fetch_ids(0);
    turn_batch(0);
  };
  // Copies a stage, entries o2[0 .. 1] of offs, to the ring at byte `at`.
  auto copy_stage = [&](const longlong2* o2, uint32_t at) {
#pragma unroll
    for (int g = 0; g < 2; ++g) {  // 16 tokens of one page
      const int64_t off = o2[g].x;
      const int valid = static_cast<int>(off) & 16;
      const uint8_t* src = code_src + off;
#pragma unroll
      for (int i = 0; i < kCopies; i += 2)
        copy16x2_if(code_dst[i % kDstVariants] + at + (g * 16 + i * kRowsPer) * RB, plus_multiple(src, copy_step, i),
                    code_dst[(i + 1) % kDstVariants] + at + (g * 16 + (i + 1) * kRowsPer) * RB,
                    plus_multiple(src, copy_step, i + 1), valid);
    }
    if (2 * kScaleChunks >= 32 || lane < 2 * kScaleChunks) {
      const int64_t off = o2[sg].y;
      const int any = static_cast<int>(off) & 16;
      const uint8_t* src = scale_src + off;
      copy16_or_zeros(scale_dst + at, src, any);
      if constexpr (kScaleCopies == 2)
        copy16_or_zeros(scale_dst + at + G::kTileScales, src + (p.v_block - p.k_block), any);
    }
  };
  if (lane < 2) offs[32 + lane] = make_longlong2(0, 0);
  {
    const Schedule sched = schedule();
    Segment g;
    if (sched.first(cta, g)) enter(g);
  }
  // ------------------------------------------------------------ segments
  uint32_t at = 0;  // byte of the ring's next stage
  // The lane's places in a stage.  tau: token of row r of an 8-token half
  // tile (neighbours swapped in every second pair); tx, ty: tau of rows 2 c
  // and 2 c + 1.  Rows 8, 16 and 24 further on have the same swizzle.
  const int tau = r ^ ((r >> 1) & 1);
  const int tx = (2 * c) ^ (c & 1), ty = (2 * c + 1) ^ (c & 1);
  int k_at, k_at2 = 0, v_at[2];
  if constexpr (D == 256) {
    k_at = tau * RB + swizzled<RB>(tau, 2 * c) * 16;
    k_at2 = tau * RB + swizzled<RB>(tau, 2 * c + 1) * 16;
    v_at[0] = tx * RB + swizzled<RB>(tx, r) * 16;
    v_at[1] = ty * RB + swizzled<RB>(ty, r) * 16;
  } else if constexpr (D == 128) {
    k_at = tau * RB + swizzled<RB>(tau, c) * 16;
    v_at[0] = tx * RB + swizzled<RB>(tx, r >> 1) * 16 + (r & 1) * 8;
    v_at[1] = ty * RB + swizzled<RB>(ty, r >> 1) * 16 + (r & 1) * 8;
  } else {
    k_at = tau * RB + swizzled<RB>(tau, c >> 1) * 16 + (c & 1) * 8;
    v_at[0] = tx * RB + swizzled<RB>(tx, r >> 2) * 16 + (r & 3) * 4;
    v_at[1] = ty * RB + swizzled<RB>(ty, r >> 2) * 16 + (r & 3) * 4;
  }
  int ks_at = 2 * G::kTileBytes + tau * SB + c * (D / 64);
  int vs_at[2] = {2 * G::kTileBytes + G::kTileScales + tx * SB + r * (D / 8) / 16,
                        2 * G::kTileBytes + G::kTileScales + ty * SB + r * (D / 8) / 16};
  keep(k_at), keep(k_at2), keep(v_at[0]), keep(v_at[1]), keep(ks_at), keep(vs_at[0]), keep(vs_at[1]);

  for (int seg_r = 0; seg_r < seg_w; ++seg_r) {
    int ntiles, k_mask;  // from stage k_mask on some row does not see some token
    {
      const Segment g = segment_of(seg_r);
      ntiles = g.ntiles;
      // t0 + kSubTokens > the keys that every row sees, for t0 = t + k * step
      const int t = g.tile0 * step + tw * kSubTokens;
      const int all_seen = g.seqlen / HW - ((MULTI && p.causal) ? p.seqlen_q - 1 : 0);
      k_mask = ((all_seen - kSubTokens - t) >> (HW == 2 ? 6 : 7)) + 1;
    }
    // sequence, KV head, first query row of the pass and its rows
    struct Place {
      int b, kvh, row_base, nrows;
    };
    auto place = [&]() {
      const int4 x = volatile_at(entry(seg_r));
      Place g;
      g.b = x.x;
      g.kvh = x.y / p.row_tiles * HW + hw;
      g.row_base = (p.row_tile0 + x.y % p.row_tiles) * p.rows;
      g.nrows = p.qrows - g.row_base < G::kRows ? p.qrows - g.row_base : G::kRows;
      return g;
    };
    // ---- query fragments: lane (r, c) holds values c * D / 4 .. of row r.
    // The logits' factor is made positive (its sign goes to the query, and a
    // factor of zero too), so that the largest product is the largest logit.
    uint32_t qf[NT][KS][2];
    float qfac[NT][2];  // per column of the lane (query rows 2 c, 2 c + 1 of each 8)
    {
      const Place pl = place();
      const int b = pl.b, kvh = pl.kvh, row_base = pl.row_base, nrows = pl.nrows;
      const float factor = __ldg(p.k_scale + kvh) * p.scale_log2;
      const float sign = factor > 0.f ? 1.f : (factor < 0.f ? -1.f : factor);
      float row_inv[NT];  // 2^-k of the row's scaling
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int n = FOLD ? r & 3 : nt * 8 + r;
        row_inv[nt] = 1.f;
        uint4 raw[D / 32];
        if (n < nrows) {
          const int h = row_base + n, qi = MULTI ? h / p.group : 0, g = h - qi * p.group;
          const uint4* src = reinterpret_cast<const uint4*>(
              static_cast<const T*>(p.q) +
              ((static_cast<int64_t>(b) * p.seqlen_q + qi) * p.num_heads + kvh * p.group + g) * D + c * (D / 4));
#pragma unroll
          for (int i = 0; i < D / 32; ++i) raw[i] = __ldg(src + i);
        } else {
#pragma unroll
          for (int i = 0; i < D / 32; ++i) raw[i] = make_uint4(0, 0, 0, 0);
        }
        float sc = sign;
        if constexpr (std::is_same<T, __nv_bfloat16>::value) {
          float mx = 0.f;
#pragma unroll
          for (int i = 0; i < D / 32; ++i) {
            const uint32_t x[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float2 f = pair_to_float2<T>(x[j]);
              mx = fmaxf(mx, fmaxf(fabsf(f.x), fabsf(f.y)));
            }
          }
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          if (mx > 0.f && mx <= 3.4e38f) {
            int k = 13 - (((__float_as_int(mx) >> 23) & 0xff) - 127);
            k = k > 126 ? 126 : (k < -126 ? -126 : k);
            sc = __int_as_float((k + 127) << 23) * sign;
            row_inv[nt] = __int_as_float((127 - k) << 23);
          }
        }
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
          const uint32_t x[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t h = x[j];
            if constexpr (std::is_same<T, __nv_bfloat16>::value) {
              const float2 f = pair_to_float2<T>(x[j]);
              h = pack_half2(f.x * sc, f.y * sc);
            } else {
              h = hmul2_bits(h, pack_half2(sc, sc));
            }
            qf[nt][2 * i + (j >> 1)][j & 1] = h;  // step s: values 4 s .. 4 s + 3 of the lane's
          }
        }
      }
      const float f = factor == 0.f ? 1.f : fabsf(factor);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          // not 0, whose product with a masked key's -infinity is NaN (the
          // smallest normal number does not change logits that are 0 to 2^-90)
          const float x = f * __shfl_sync(0xffffffffu, row_inv[nt], (2 * c + e) * 4);
          qfac[nt][e] = x < 1.17549435e-38f ? 1.17549435e-38f : x;
        }
    }

    float acc[MT][NT][4];
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][nt][e] = 0.f;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = -3e38f;  // below any logit; while no key was seen every P is 0
      l[nt][0] = l[nt][1] = 0.f;
    }

    // Before the first segment's first tile the ring is filled, by rounds that
    // only issue: one place in the code, which is long, and cold when a launch
    // starts.  (The query is read first: behind a full ring it waited 2 us.)
    // The rounds run in batches between which the cursor needs attention (its
    // segment or its page offsets end), so that the inner loop holds none of
    // that: its branches and the jumps over its code cost 100 cycles a round.
    for (int k = seg_r == 0 ? -G::kStages : 0; k < ntiles;) {
      const bool more = pc_left > 0;
      int n = ntiles - k;
      if (more) {
        const int turn = 16 - (pc_k & 15), calm = pc_left < turn ? pc_left : turn;
        n = n < calm ? n : calm;
      }
      const longlong2* o2 = offs + (more ? (pc_k & 15) * 2 : 32);
      const int o2_step = more ? 2 : 0;
#pragma unroll 1
      for (const int stop = k + n; k < stop; ++k) {
        if (k >= 0) {
          copy_wait<G::kStages - 1>();
          __syncwarp();  // every lane's copies of the stage have landed
          const uint8_t* st = ring + at;

          // ---- S^T = K . Q^T, two tiles of 16 tokens side by side
          float s[2][NT][4];
          uint32_t kw[2][2][KW];               // [tile][rows r, r + 8]: the lane's codes
          uint32_t kf[2][2][(D + 127) / 128];  // and the f16 pairs of their block scales
#pragma unroll
          for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int e = 0; e < 4; ++e) s[mt][nt][e] = 0.f;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const int row = mt * 16 + half * 8;
              const uint8_t* sc = st + ks_at + row * SB;
              if constexpr (D == 256) {
                uint32_t x[4], y[4];
                load_words<4>(st + k_at + row * RB, x);
                load_words<4>(st + k_at2 + row * RB, y);
#pragma unroll
                for (int i = 0; i < 4; ++i) { kw[mt][half][i] = x[i]; kw[mt][half][4 + i] = y[i]; }
                const uint32_t q = *reinterpret_cast<const uint32_t*>(sc);
                kf[mt][half][0] = e4m3x2_to_half2(q);
                kf[mt][half][1] = e4m3x2_to_half2(q >> 16);
              } else if constexpr (D == 128) {
                load_words<4>(st + k_at + row * RB, kw[mt][half]);
                kf[mt][half][0] = e4m3x2_to_half2(*reinterpret_cast<const uint16_t*>(sc));
              } else {
                load_words<2>(st + k_at + row * RB, kw[mt][half]);
                kf[mt][half][0] = e4m3x2_to_half2(*sc);
              }
            }
          }
#pragma unroll
          for (int wi = 0; wi < KW; ++wi) {
            const int blk = wi / 2;  // two words a block
#pragma unroll
            for (int mt = 0; mt < 2; ++mt) {
              uint32_t h[2][4];
#pragma unroll
              for (int half = 0; half < 2; ++half) {
                const uint32_t pair = kf[mt][half][blk / 2];
                const uint32_t f = blk & 1 ? high_twice(pair) : low_twice(pair);
                e2m1x8_to_half2x4(kw[mt][half][wi], h[half]);
#pragma unroll
                for (int j = 0; j < 4; ++j) h[half][j] = hmul2_bits(h[half][j], f);
              }
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                mma_f16(s[mt][nt], h[0][0], h[1][0], h[0][1], h[1][1], qf[nt][2 * wi][0], qf[nt][2 * wi][1]);
                mma_f16(s[mt][nt], h[0][2], h[1][2], h[0][3], h[1][3], qf[nt][2 * wi + 1][0], qf[nt][2 * wi + 1][1]);
              }
            }
          }

          // ---- softmax over the warp's 32 tokens (log2 domain)
          if (__any_sync(0xffffffffu, k >= k_mask)) {
            const int t0 = (volatile_at(entry(seg_r)).z + k) * step + tw * kSubTokens;
            const int len = volatile_at(entry(seg_r) + 1).x / HW, base = MULTI ? place().row_base : 0;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                // causal: row (qi, g) sees the keys up to its own position
                const int seen =
                    len + ((MULTI && p.causal) ? (base + row_of(nt, e)) / p.group - (p.seqlen_q - 1) : 0);
#pragma unroll
                for (int mt = 0; mt < 2; ++mt) {
                  if (t0 + mt * 16 + tau >= seen) s[mt][nt][e] = neg_inf;
                  if (t0 + mt * 16 + tau + 8 >= seen) s[mt][nt][e + 2] = neg_inf;
                }
              }
            // Block scales of V must not be NaN where P is 0.  Behind the sequence's
            // end they are what memory held: cleared.
            uint32_t* sb = reinterpret_cast<uint32_t*>(ring + at + 2 * G::kTileBytes + G::kTileScales + lane * SB);
            if (t0 + lane >= len) {
#pragma unroll
              for (int i = 0; i < SB / 4; ++i) sb[i] = 0;
            }
            __syncwarp();
            if constexpr (MULTI) {
              // A NaN of the sequence must not reach the rows that do not see its
              // token: it is taken out of the stage, and put into O's block of the
              // rows that do see it.
              bool any = false;
#pragma unroll
              for (int i = 0; i < SB / 4; ++i) any = any || nan_bytes(sb[i]) != 0;
              unsigned tokens = __ballot_sync(0xffffffffu, any);
              if (tokens != 0) {
#pragma unroll 1
                for (; tokens != 0; tokens &= tokens - 1) {
                  const int u = __ffs(tokens) - 1;
                  const uint8_t* row = st + 2 * G::kTileBytes + G::kTileScales + u * SB + r * (D / 8) / 16;
#pragma unroll
                  for (int j = 0; j < (D + 127) / 128; ++j) {  // the lane's blocks, of MT / that many tiles each
                    constexpr int kPer = MT / ((D + 127) / 128);
                    if (nan_bytes(row[j]) == 0) continue;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                      for (int e = 0; e < 2; ++e) {
                        const int seen =
                            len + (p.causal ? (base + row_of(nt, e)) / p.group - (p.seqlen_q - 1) : 0);
                        if (t0 + u >= seen) continue;
#pragma unroll
                        for (int i = j * kPer; i < (j + 1) * kPer; ++i)
                          acc[i][nt][e] = acc[i][nt][e + 2] = __int_as_float(0x7fffffff);
                      }
                  }
                }
                __syncwarp();
#pragma unroll
                for (int i = 0; i < SB / 4; ++i) sb[i] &= ~nan_bytes(sb[i]);
                __syncwarp();
              }
            }
          }
          // The reference of the exponents need not be the maximum less kLift: it
          // is raised (and O, l rescaled) only when a logit exceeds it by more than
          // kRaise, so that P stays inside f16 and most stages need no reduction
          // over the tokens' lanes.  The product rounded up bounds the exact ones
          // that the exponents subtract the reference from, however large.
          bool above = false;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float mx = fmaxf(fmaxf(s[0][nt][e], s[0][nt][e + 2]), fmaxf(s[1][nt][e], s[1][nt][e + 2]));
              above = above || __fmul_ru(mx, qfac[nt][e]) - m[nt][e] > kRaise;
            }
          if (__any_sync(0xffffffffu, above)) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                float mx = fmaxf(fmaxf(s[0][nt][e], s[0][nt][e + 2]), fmaxf(s[1][nt][e], s[1][nt][e + 2]));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                const float m_new = fmaxf(m[nt][e], __fmul_ru(mx, qfac[nt][e]) - kLift);
                const float alpha = m_new == m[nt][e] ? 1.f : fast_exp2(m[nt][e] - m_new);
                m[nt][e] = m_new;
                l[nt][e] *= alpha;
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                  acc[i][nt][e] *= alpha;
                  acc[i][nt][e + 2] *= alpha;
                }
              }
          }
          uint32_t pt[2][NT][kParts][2];  // P^T fragments of each 16 tokens
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
              for (int mt = 0; mt < 2; ++mt) {
                s[mt][nt][e] = fast_exp2(fmaf(s[mt][nt][e], qfac[nt][e], -m[nt][e]));
                s[mt][nt][e + 2] = fast_exp2(fmaf(s[mt][nt][e + 2], qfac[nt][e], -m[nt][e]));
              }
              l[nt][e] += (s[0][nt][e] + s[0][nt][e + 2]) + (s[1][nt][e] + s[1][nt][e + 2]);
            }
#pragma unroll
            for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
              for (int half = 0; half < 2; ++half) {
                const float x = s[mt][nt][2 * half], y = s[mt][nt][2 * half + 1];
                const uint32_t h = pack_half2(x, y);
                if constexpr (FOLD) {  // the first part in columns 0 .. 3, the second in 4 .. 7
                  pt[mt][nt][0][half] = transpose8x8(pack_rest2(x, y, h, c < 2 ? 0 : kMinusOne));
                } else {
                  pt[mt][nt][0][half] = transpose8x8(h);
                  pt[mt][nt][1][half] = transpose8x8(pack_rest2(x, y, h, kMinusOne));
                }
              }
            }
          }

          // ---- O^T += V^T . P^T
#pragma unroll
          for (int ks = 0; ks < 2; ++ks) {
            uint32_t v[4][VW], sc[4];  // tokens tx, ty, tx + 8, ty + 8 of the 16
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              const int row = ks * 16 + (u >> 1) * 8;
              load_words<VW>(st + G::kTileBytes + v_at[u & 1] + row * RB, v[u]);
              const uint8_t* sb = st + vs_at[u & 1] + row * SB;
              sc[u] = D == 256 ? *reinterpret_cast<const uint16_t*>(sb) : *sb;
            }
#pragma unroll
            for (int wi = 0; wi < VW; ++wi) {
              uint32_t w0, w1;  // the block scales of the word's block, of two tokens each
              if constexpr (D == 256) {
                w0 = __byte_perm(sc[0], sc[1], wi < 2 ? 0x0040 : 0x0051);
                w1 = __byte_perm(sc[2], sc[3], wi < 2 ? 0x0040 : 0x0051);
              } else {
                w0 = sc[0] + sc[1] * 256u;
                w1 = sc[2] + sc[3] * 256u;
              }
              const uint32_t f0 = e4m3x2_to_half2(w0), f1 = e4m3x2_to_half2(w1);
              // even codes of both tokens in one word, odd codes in another
              uint32_t e0[4], o0[4], e1[4], o1[4];
              e2m1x8_to_half2x4(low_high(v[0][wi], times16(v[1][wi])), e0);
              e2m1x8_to_half2x4(low_high(v[0][wi] >> 4, v[1][wi]), o0);
              e2m1x8_to_half2x4(low_high(v[2][wi], times16(v[3][wi])), e1);
              e2m1x8_to_half2x4(low_high(v[2][wi] >> 4, v[3][wi]), o1);
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const uint32_t a0 = hmul2_bits(e0[j], f0), a1 = hmul2_bits(o0[j], f0);
                const uint32_t a2 = hmul2_bits(e1[j], f1), a3 = hmul2_bits(o1[j], f1);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                  for (int part = kParts - 1; part >= 0; --part)
                    mma_f16(acc[wi * 4 + j][nt], a0, a1, a2, a3, pt[ks][nt][part][0], pt[ks][nt][part][1]);
              }
            }
          }
        }
        // ---- refill the stage
        __syncwarp();  // every lane has read it
        copy_stage(o2, at);
        o2 += o2_step;
        copy_commit();  // one group a stage, empty ones too, so that the count of groups stays fixed
        at = at == (G::kStages - 1) * G::kStageBytes ? 0 : at + G::kStageBytes;
      }
      if (more) {
        pc_k += n;
        pc_left -= n;
        if (pc_left == 0) {
          const Schedule sched = schedule();
          Segment nx;
          if (sched.next(segment_of(seg_w - 1), sched.range_start(cta + 1), nx)) enter(nx);
        } else if ((pc_k & 15) == 0) {
          turn_batch(pc_k);
        }
      }
    }

    // ---- the rows' sums; warps that share a head are joined on its first
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], 4);
        l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], 8);
        l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], 16);
      }
    if constexpr (FOLD) {  // the sums of both parts, in columns 0 .. 3
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][0][e] += __shfl_xor_sync(0xffffffffu, acc[i][0][e], 2);
    }
    if (TW > 1) {
      // Lane (r, c) holds dims r * D / 8 + 2 i (entries e) and + 2 i + 1
      // (entries e + 2) of rows 2 c + e.
      if (tw > 0) {
        float* buf = reinterpret_cast<float*>(smem + G::kOffJoin + (warp - HW) * G::kJoinWarp);
        float* ml = buf + G::kRows * G::kRowPad;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int row = nt * 8 + 2 * c + e;
            float4* d = reinterpret_cast<float4*>(buf + row * G::kRowPad + r * (D / 8));
#pragma unroll
            for (int i = 0; i < MT; i += 2)
              d[i / 2] = make_float4(acc[i][nt][e], acc[i][nt][e + 2], acc[i + 1][nt][e], acc[i + 1][nt][e + 2]);
            if (r == 0) {
              ml[row * 2] = m[nt][e];
              ml[row * 2 + 1] = l[nt][e];
            }
          }
      }
      __syncthreads();
      if (tw == 0) {
        for (int o = 1; o < TW; ++o) {
          const float* buf = reinterpret_cast<const float*>(smem + G::kOffJoin + (warp + (o - 1) * HW) * G::kJoinWarp);
          const float* ml = buf + G::kRows * G::kRowPad;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int row = nt * 8 + 2 * c + e;
              const float mo = ml[row * 2], mm = fmaxf(m[nt][e], mo);
              // equal references weigh 1, so that NaN sums stay
              const float fa = m[nt][e] == mm ? 1.f : fast_exp2(m[nt][e] - mm);
              const float fb = mo == mm ? 1.f : fast_exp2(mo - mm);
              m[nt][e] = mm;
              l[nt][e] = fmaf(l[nt][e], fa, ml[row * 2 + 1] * fb);
              const float4* d = reinterpret_cast<const float4*>(buf + row * G::kRowPad + r * (D / 8));
#pragma unroll
              for (int i = 0; i < MT; i += 2) {
                const float4 x = d[i / 2];
                acc[i][nt][e] = fmaf(acc[i][nt][e], fa, x.x * fb);
                acc[i][nt][e + 2] = fmaf(acc[i][nt][e + 2], fa, x.y * fb);
                acc[i + 1][nt][e] = fmaf(acc[i + 1][nt][e], fa, x.z * fb);
                acc[i + 1][nt][e + 2] = fmaf(acc[i + 1][nt][e + 2], fa, x.w * fb);
              }
            }
        }
      }
      __syncthreads();  // the buffers are free again
    }

    // ---- write: the output, or a partial of a pair cut by range boundaries
    const Place pl = place();
    const int b = pl.b, kvh = pl.kvh, row_base = pl.row_base, nrows = pl.nrows;
    const int4 sb = volatile_at(entry(seg_r) + 1);
    const int pair = sb.y, nseg = sb.z, cfirst = sb.w;
    const int64_t part = (static_cast<int64_t>(cta) + pair) * HW + hw;
    const float vs = __ldg(p.v_scale + kvh);
    const int rows = p.rows;
    // out and lse places of row `row`
    auto out_at = [&](int row) {
      const int h = row_base + row, qi = MULTI ? h / p.group : 0, g = h - qi * p.group;
      return static_cast<OutT*>(p.out) +
             ((static_cast<int64_t>(b) * p.seqlen_q + qi) * p.num_heads + kvh * p.group + g) * D;
    };
    auto put_lse = [&](int row, float lse2) {
      const int h = row_base + row, qi = MULTI ? h / p.group : 0, g = h - qi * p.group;
      if (p.lse != nullptr)
        p.lse[(static_cast<int64_t>(b) * p.num_heads + kvh * p.group + g) * p.seqlen_q + qi] =
            lse2 * 0.69314718055994531f;
    };
    if (tw == 0) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int row = nt * 8 + 2 * c + e;
          if (row >= nrows) continue;
          const bool some = !(l[nt][e] == 0.f);  // a row that saw a key (NaN stays NaN)
          const float inv = some ? vs / l[nt][e] : 0.f;
          // (the lift is taken out of both, so that the logarithm is of a small number)
          const float lse2 = some ? (m[nt][e] + kLift) + fast_log2(l[nt][e] * (1.f / (1 << kLift))) : neg_inf;
          float o[D / 8];
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            o[2 * i] = some ? acc[i][nt][e] * inv : 0.f;
            o[2 * i + 1] = some ? acc[i][nt][e + 2] * inv : 0.f;
          }
          if (nseg == 1) {
            store_row<OutT, D / 8>(out_at(row) + r * (D / 8), o);
            if (r == 0) put_lse(row, lse2);
          } else {
            store_row<float, D / 8>(p.part_o + (part * rows + row) * D + r * (D / 8), o);
            if (r == 0) p.part_lse[part * rows + row] = lse2;
          }
        }
    }
    if (nseg == 1) continue;
    constexpr int kAt = D == 256 ? 2 : 4;
    int last = 0;
    if (tw == 0) {
      __threadfence();
      __syncwarp();
      if (lane == 0) {
        unsigned long long* ticket = p.tickets + static_cast<int64_t>(pair) * HW + hw;
        last = ticket_add(ticket, pair_stamp(*launch_epoch), nseg) ? 1 : 0;
        // every segment of the pair has counted itself: clear for later launches
        if (last) *reinterpret_cast<volatile unsigned long long*>(ticket) = 0ull;
      }
      last = __shfl_sync(0xffffffffu, last, 0);
    }
    // With more rows or partials than one round takes, the head's other warps
    // take a share: of the rows, or else of the partials.
    const int row_ways = nrows > kAt ? TW : 1;
    const int part_ways = row_ways == 1 && nseg > kAt ? TW : 1;
    if (row_ways * part_ways > 1) {
      if (tw == 0 && lane == 0) last_flag[hw] = last;
      __syncthreads();
      last = last_flag[hw];
      __syncthreads();
    }
    if (!last && part_ways == 1) continue;  // (warps tw > 0 that have no share, too)
    __threadfence();
    // The last of the pair's segments joins them: partial j of the head is
    // part (cfirst + j + pair) * HW + hw.  A round is kAt partials of kAt rows
    // (of the warp's rows, partials), all their loads in flight: lane
    // kAt v + u holds the weight of partial u of row v, relative to a running
    // maximum.  Short code on purpose: it runs once, and cold instructions
    // cost more than the loads (16 partials unrolled took 2 to 10 us longer).
    const int64_t first = (static_cast<int64_t>(cfirst) + pair) * HW + hw;
    const int64_t lse_step = static_cast<int64_t>(HW) * rows;
    constexpr int kVec = D >= 128 ? 4 : 2, kPieces = D / (32 * kVec);
    const int lu = lane & (kAt - 1), lv = lane / kAt;
    const int row_tw = row_ways > 1 ? tw : 0, part_tw = part_ways > 1 ? tw : 0;
#pragma unroll 1
    for (int row0 = row_tw; row0 < nrows; row0 += kAt * row_ways) {
      float mm = neg_inf, den = 0.f;  // of row lv
      // rows past the last are read as the first, and not written
      int row_at[kAt];
#pragma unroll
      for (int v = 0; v < kAt; ++v) row_at[v] = (row0 + v * row_ways < nrows ? v * row_ways : 0) * D;
      float o[kAt][kPieces][kVec];
#pragma unroll
      for (int v = 0; v < kAt; ++v)
#pragma unroll
        for (int q = 0; q < kPieces; ++q)
#pragma unroll
          for (int i = 0; i < kVec; ++i) o[v][q][i] = 0.f;
#pragma unroll 1
      for (int j0 = part_tw * kAt; last && j0 < nseg; j0 += kAt * part_ways) {
        const int64_t at_row = first * rows + row0 + j0 * lse_step;
        const bool mine = lv < kAt && row0 + lv * row_ways < nrows && j0 + lu < nseg;
        const float lj = mine ? __ldcg(p.part_lse + at_row + lv * row_ways + lu * lse_step) : neg_inf;
        float x[kAt][kAt][kPieces][kVec];
        const float* src = p.part_o + at_row * D + lane * kVec;
#pragma unroll
        for (int u = 0; u < kAt; ++u) {
#pragma unroll
          for (int v = 0; v < kAt; ++v) {
            if (j0 + u < nseg) {
#pragma unroll
              for (int q = 0; q < kPieces; ++q) load_vec(src + row_at[v] + q * 32 * kVec, x[v][u][q]);
            }
          }
          src += lse_step * D;
        }
        float m_new = fmaxf(lj, __shfl_xor_sync(0xffffffffu, lj, 1));
        if constexpr (kAt == 4) m_new = fmaxf(m_new, __shfl_xor_sync(0xffffffffu, m_new, 2));
        m_new = fmaxf(mm, m_new);
        const float w = lj == neg_inf ? 0.f : fast_exp2(lj - m_new);  // 0: empty, or past the last
        const float alpha = m_new == mm ? 1.f : fast_exp2(mm - m_new);
        mm = m_new;
        float sum = w + __shfl_xor_sync(0xffffffffu, w, 1);
        if constexpr (kAt == 4) sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        den = fmaf(den, alpha, sum);
#pragma unroll
        for (int v = 0; v < kAt; ++v) {
          const float av = __shfl_sync(0xffffffffu, alpha, v * kAt);
#pragma unroll
          for (int q = 0; q < kPieces; ++q)
#pragma unroll
            for (int i = 0; i < kVec; ++i) o[v][q][i] *= av;
#pragma unroll
          for (int u = 0; u < kAt; ++u) {
            const float wu = __shfl_sync(0xffffffffu, w, v * kAt + u);
            if (j0 + u >= nseg) continue;  // (one whose weight is 0 counts, for its NaNs)
#pragma unroll
            for (int q = 0; q < kPieces; ++q)
#pragma unroll
              for (int i = 0; i < kVec; ++i) o[v][q][i] = fmaf(wu, x[v][u][q][i], o[v][q][i]);
          }
        }
      }
      if (part_ways > 1) {  // one round of rows: what the other warps joined goes to the first
        float* buf = reinterpret_cast<float*>(smem + G::kOffJoin + (warp - HW) * G::kJoinWarp);
        if (tw > 0 && last) {
          float* ml = buf + G::kRows * G::kRowPad;
          if (lv < kAt && lu == 0) ml[2 * lv] = mm, ml[2 * lv + 1] = den;
#pragma unroll
          for (int v = 0; v < kAt; ++v)
#pragma unroll
            for (int q = 0; q < kPieces; ++q)
#pragma unroll
              for (int i = 0; i < kVec; ++i) buf[v * G::kRowPad + (q * 32 + lane) * kVec + i] = o[v][q][i];
        }
        __syncthreads();
        if (tw == 0 && last) {
#pragma unroll 1
          for (int u = 1; u < TW; ++u) {
            const float* from =
                reinterpret_cast<const float*>(smem + G::kOffJoin + (warp + (u - 1) * HW) * G::kJoinWarp);
            const float* ml = from + G::kRows * G::kRowPad + 2 * (lv < kAt ? lv : 0);
            const float m_new = fmaxf(mm, ml[0]);
            const float fa = mm == m_new ? 1.f : fast_exp2(mm - m_new);
            const float fb = ml[0] == m_new ? 1.f : fast_exp2(ml[0] - m_new);
            mm = m_new;
            den = fmaf(den, fa, ml[1] * fb);
#pragma unroll
            for (int v = 0; v < kAt; ++v) {
              const float av = __shfl_sync(0xffffffffu, fa, v * kAt), bv = __shfl_sync(0xffffffffu, fb, v * kAt);
#pragma unroll
              for (int q = 0; q < kPieces; ++q)
#pragma unroll
                for (int i = 0; i < kVec; ++i)
                  o[v][q][i] = fmaf(o[v][q][i], av, from[v * G::kRowPad + (q * 32 + lane) * kVec + i] * bv);
            }
          }
        }
        __syncthreads();  // the buffers are free again
        if (tw > 0 || !last) break;
      }
      const bool some = !(den == 0.f);
      const float inv = some ? 1.f / den : 0.f;
      if (lv < kAt && lu == 0 && row0 + lv * row_ways < nrows)
        put_lse(row0 + lv * row_ways, some ? mm + fast_log2(den) : neg_inf);
#pragma unroll
      for (int v = 0; v < kAt; ++v) {
        const float iv = __shfl_sync(0xffffffffu, inv, v * kAt);
        if (row0 + v * row_ways >= nrows) continue;
        OutT* dst = out_at(row0 + v * row_ways) + lane * kVec;
#pragma unroll
        for (int q = 0; q < kPieces; ++q) {
#pragma unroll
          for (int i = 0; i < kVec; ++i) o[v][q][i] *= iv;
          store_vec(dst + q * 32 * kVec, o[v][q]);
        }
      }
    }
  }
  // Every CTA counts itself once it has read the epoch; the last one hands
  // the next launch a new epoch (see fd_decode_sm100.cuh).  Here at the end,
  // the counter's round trips delay no load.
  if (tid == 0) {
    const unsigned long long e = *launch_epoch;
    if (ticket_arrive(p.epoch_word + 1, e, static_cast<int>(gridDim.x))) {
      p.epoch_word[0] = e % kEpochMax + 1ull;
      p.epoch_word[1] = 0ull;
    }
  }
}

template <typename T, typename OutT, int D, int NT, bool MULTI, bool FOLD>
cudaError_t launch_fp4_typed(const Fp4DecodeParams& p, int grid, cudaStream_t stream) {
  using G = Fp4Geo<D, NT>;
  auto kern = decode_fp4_kernel<T, OutT, D, NT, MULTI, FOLD>;
  static unsigned long long configured = 0;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const unsigned long long bit = 1ull << (dev & 63);
  if ((__atomic_load_n(&configured, __ATOMIC_ACQUIRE) & bit) == 0) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, G::kSmemBytes);
    if (e != cudaSuccess) return e;
    __atomic_fetch_or(&configured, bit, __ATOMIC_RELEASE);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(kFp4Threads);
  cfg.dynamicSmemBytes = G::kSmemBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = p.pdl ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, p);
}

template <typename T, typename OutT, int D>
cudaError_t launch_fp4_dim(const Fp4DecodeParams& p, int grid, cudaStream_t stream) {
  const bool multi = p.seqlen_q > 1 || p.causal;
  if (p.qrows <= 4)
    return multi ? launch_fp4_typed<T, OutT, D, 1, true, true>(p, grid, stream)
                 : launch_fp4_typed<T, OutT, D, 1, false, true>(p, grid, stream);
  if constexpr (D < 256) {
    if (p.rows == 16)
      return multi ? launch_fp4_typed<T, OutT, D, 2, true, false>(p, grid, stream)
                   : launch_fp4_typed<T, OutT, D, 2, false, false>(p, grid, stream);
  }
  return multi ? launch_fp4_typed<T, OutT, D, 1, true, false>(p, grid, stream)
               : launch_fp4_typed<T, OutT, D, 1, false, false>(p, grid, stream);
}

template <typename T, typename OutT>
cudaError_t launch_fp4(const Fp4DecodeParams& p, int head_dim, int grid, cudaStream_t stream) {
  switch (head_dim) {
    case 64: return launch_fp4_dim<T, OutT, 64>(p, grid, stream);
    case 128: return launch_fp4_dim<T, OutT, 128>(p, grid, stream);
    default: return launch_fp4_dim<T, OutT, 256>(p, grid, stream);
  }
}

}  // namespace

}  // namespace fd
