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
// largest (smaller ones keep an absolute error of 2^-39 of it).  P is rounded
// to f16 (11 bits, relative to each warp's running maximum).
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
// TMA swizzle K's and V's loads are free of bank conflicts at D = 128, 256.
//
// A CTA is four warps; each has its own ring of 32-token stages filled by TMA
// (its lane 0 issues; page ids come from one lookup per 32 stages) and its
// own softmax state, so the loop has no CTA-wide synchronisation.  The four
// states are joined when a segment (the CTA's part of a pair) ends, after the
// next segment's first loads were issued.  Work split and the joining of
// segments on different CTAs are those of fd_decode_sm100.cuh.
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

template <int D, int NT> struct Fp4Geo {
  static constexpr int kRowBytes = D / 2;
  static constexpr int kScaleBytes = D / 16;
  static constexpr int kTileBytes = kSubTokens * kRowBytes;
  // Block scales of 16 tokens; TMA destinations are 128-byte aligned, so the
  // 64 bytes of D = 64 are spread when they come in boxes of 16 tokens.
  static constexpr int kHalfScales = 16 * kScaleBytes < 128 ? 128 : 16 * kScaleBytes;
  static constexpr int kTileScales = 2 * kHalfScales;
  static constexpr int kStageBytes = 2 * kTileBytes + 2 * kTileScales;
  static constexpr int kRows = 8 * NT;
  // CTAs per SM, and stages that fit beside them
  static constexpr int kCtas = D == 256 ? 2 : (NT == 1 ? 4 : 3);
  static constexpr int kStages = D == 64 ? 4 : 2;
  static constexpr int kRowPad = D + 4;  // floats of a row of the join buffer
  static constexpr int kOffJoin = kFp4Warps * kStages * kStageBytes;       // [2][kRows][kRowPad] floats
  static constexpr int kOffMl = kOffJoin + 2 * kRows * kRowPad * 4;        // [warps][kRows][2] floats
  static constexpr int kOffBars = kOffMl + kFp4Warps * kRows * 2 * 4;
  static constexpr int kOffMisc = kOffBars + kFp4Warps * kStages * 8;
  static constexpr int kOffPrefix = kOffMisc + 64;
  static constexpr int kOffLens = kOffPrefix + (kMaxBatchPerLaunch + 1) * 4;
  static constexpr int kSmemBytes = kOffLens + kMaxBatchPerLaunch * 4 + 1024;  // slack for alignment
  static_assert(kTileBytes % 1024 == 0 && kTileScales % 128 == 0, "TMA destinations");
  static_assert(kStageBytes % (8 * kRowBytes) == 0, "a stage starts on a swizzle period");
  static_assert(kSmemBytes <= 232448 / kCtas, "shared memory of the resident CTAs");
  static_assert(kOffBars % 8 == 0 && kOffMisc % 8 == 0, "alignment");
};

__device__ __forceinline__ void tma_load_3d(const CUtensorMap* map, uint64_t* bar, void* dst, int c0,
                                            int c1, int c2, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%3, %4, %5}], [%2], %6;" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "l"(policy)
      : "memory");
}

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                        uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
  return d;
}

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <typename T> __device__ __forceinline__ float2 pair_to_float2(uint32_t w);
template <> __device__ __forceinline__ float2 pair_to_float2<__nv_bfloat16>(uint32_t w) {
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w));
}
template <> __device__ __forceinline__ float2 pair_to_float2<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

template <typename O> __device__ __forceinline__ O fp4_out(float x);
template <> __device__ __forceinline__ float fp4_out<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 fp4_out<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half fp4_out<__half>(float x) { return __float2half_rn(x); }

// N words (1, 2, 4 or 8) from shared memory in the widest loads.
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

// 16-byte chunk of row `row` that the TMA put chunk `chunk` at: the swizzle
// exchanges chunks by address bits 7.., i.e. by the row.
template <int RB> __device__ __forceinline__ int swizzled(int row, int chunk) {
  if constexpr (RB == 32) return chunk ^ ((row >> 2) & 1);
  else if constexpr (RB == 64) return chunk ^ ((row >> 1) & 3);
  else return chunk ^ (row & 7);
}

template <typename T, typename OutT, int D, int NT, bool MULTI>
__global__ void __launch_bounds__(kFp4Threads, Fp4Geo<D, NT>::kCtas)
    decode_fp4_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                      const __grid_constant__ CUtensorMap tm_kb, const __grid_constant__ CUtensorMap tm_vb,
                      const Fp4DecodeParams p) {
  using G = Fp4Geo<D, NT>;
  constexpr int RB = G::kRowBytes, SB = G::kScaleBytes;
  constexpr int KW = D / 32;        // words of K a lane takes from a row
  constexpr int VW = D / 64;        // words of V a lane takes from a token
  constexpr int MT = D / 16;        // 16-dim tiles of O^T
  constexpr int KS = D / 16;        // 16-dim steps of S^T
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + (((raw_addr + 1023u) & ~1023u) - raw_addr);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int r = lane >> 2, c = lane & 3;

  uint8_t* ring = smem + warp * G::kStages * G::kStageBytes;
  float* join = reinterpret_cast<float*>(smem + G::kOffJoin);
  float* ml = reinterpret_cast<float*>(smem + G::kOffMl);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + G::kOffBars) + warp * G::kStages;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + G::kOffMisc);
  volatile int* last_flag = reinterpret_cast<volatile int*>(smem + G::kOffMisc + 4);
  unsigned long long* launch_epoch = reinterpret_cast<unsigned long long*>(smem + G::kOffMisc + 8);
  int* prefix = reinterpret_cast<int*>(smem + G::kOffPrefix);
  int* lens = reinterpret_cast<int*>(smem + G::kOffLens);

  const int batch = p.batch, cta = blockIdx.x;
  const int vheads = p.num_heads_k * p.row_tiles;  // a pair is (sequence, KV head, row tile)
  const int64_t max_len = p.bt_stride * static_cast<int64_t>(p.page);
  const float neg_inf = -__int_as_float(0x7f800000);
  // bytes from the block scales of a stage's token 0 to those of token 16
  const int half_scales = p.chunk == 16 ? G::kHalfScales : 16 * SB;

  // ------------------------------------------------------------ prologue
  if (tid == 0) {
    pdl_launch_dependents();
    uint64_t* all = reinterpret_cast<uint64_t*>(smem + G::kOffBars);
    for (int i = 0; i < kFp4Warps * G::kStages; ++i) mbar_init(all + i, 1);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
    tma_prefetch_desc(&tm_kb);
    tma_prefetch_desc(&tm_vb);
  }
  const CostModel cm{p.cost_tile, p.cost_seg, p.cost_floor};
  pdl_wait_prerequisites();
  unsigned long long epoch_ld = 0;
  if (tid == 0) epoch_ld = *reinterpret_cast<volatile unsigned long long*>(p.epoch_word);
  for (int b = tid; b < batch; b += kFp4Threads) {
    const int stored = __ldg(p.seqlens + b);
    const int64_t want = static_cast<int64_t>(stored < 0 ? 0 : stored) + p.len_add;
    const int64_t cap = max_len < 0x7fffffff ? max_len : 0x7fffffff;
    const int len = static_cast<int>(want > cap ? cap : want);
    lens[b] = len;
    prefix[b + 1] = cm.pair_cost(len);
  }
  if (tid == 0) {
    prefix[0] = 0;
    *launch_epoch = epoch_ld & kEpochMax;
  }
  fence_proxy_async_smem();
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
  // Every CTA counts itself once it has read the epoch; the last one hands
  // the next launch a new epoch (see fd_decode_sm100.cuh).
  if (tid == 0) {
    const unsigned long long e = *launch_epoch;
    if (ticket_arrive(p.epoch_word + 1, e, static_cast<int>(gridDim.x))) {
      p.epoch_word[0] = e % kEpochMax + 1ull;
      p.epoch_word[1] = 0ull;
    }
  }
  Schedule sched;
  sched.cost_prefix = prefix;
  sched.lens = lens;
  sched.max_len = max_len;
  sched.total = static_cast<int64_t>(vheads) * prefix[batch];
  sched.batch = batch;
  sched.hkv = vheads;
  sched.cm = cm;
  sched.align_m = 0;
  sched.align_cost = 0;
  {
    // every range longer than the costliest tile: none inside a pair is empty
    const int64_t g = div_u32(sched.total, cm.max_lead() + cm.full() + 1);
    sched.grid = static_cast<int>(g < 1 ? 1 : (g < gridDim.x ? g : gridDim.x));
  }
  const int64_t range_end = sched.range_start(cta + 1);

  // ------------------------------------------------------------ loads
  const uint64_t policy = policy_evict_first();
  // Page ids of the warp's next 32 stages, one per lane (two with 16-token
  // boxes); num_blocks, which the TMA fills with zeros, for a bad id.
  int page_ids[2] = {0, 0};
  int64_t stage_no = 0;  // stages this warp has used so far (ring position and parity)
  struct Walk {
    int b, kvh, tok0, end, count;  // this warp's stages: tokens tok0 + 128 k .. < end, k < count
  };
  auto walk_of = [&](const Segment& s) {
    Walk w;
    w.b = s.b;
    w.kvh = s.kvh / p.row_tiles;
    w.tok0 = s.tile0 * kTileTokens + warp * kSubTokens;
    const int64_t stop = static_cast<int64_t>(s.tile0 + s.ntiles) * kTileTokens;
    w.end = static_cast<int>(stop < s.seqlen ? stop : s.seqlen);
    w.count = w.end > w.tok0 ? (w.end - w.tok0 + kTileTokens - 1) / kTileTokens : 0;
    return w;
  };
  auto load_ids = [&](const Walk& w, int k0) {
    const int tok = w.tok0 + (k0 + lane) * kTileTokens;
    const int32_t* row = p.block_table + w.b * p.bt_stride;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int t = tok + 16 * u;
      int id = 0;
      if (k0 + lane < w.count && t < w.end && (u == 0 || p.chunk == 16)) {
        id = __ldg(row + static_cast<uint32_t>(t) / static_cast<uint32_t>(p.page));
        if (id < 0 || id >= p.num_blocks) {
          report_status(p.err, kStatusBadPage);
          id = static_cast<int>(p.num_blocks);
        }
      }
      page_ids[u] = id;
    }
  };
  auto issue = [&](const Walk& w, int k, int64_t no) {
    const int id0 = __shfl_sync(0xffffffffu, page_ids[0], k & 31);
    const int id1 = __shfl_sync(0xffffffffu, page_ids[1], k & 31);
    if (lane == 0) {
      const int slot = static_cast<int>(no % G::kStages);
      uint8_t* st = ring + slot * G::kStageBytes;
      uint64_t* bar = bars + slot;
      const int t = w.tok0 + k * kTileTokens;
      const int row0 = static_cast<int>(static_cast<uint32_t>(t) % static_cast<uint32_t>(p.page));
      const bool wide = p.chunk == kSubTokens;
      const int boxes = wide || t + 16 >= w.end ? 1 : 2;
      const int box_tokens = wide ? kSubTokens : 16;
      mbar_arrive_expect_tx(bar, static_cast<uint32_t>(boxes * box_tokens * 2 * (RB + SB)));
      for (int u = 0; u < boxes; ++u) {
        const int id = u == 0 ? id0 : id1;
        const int row = u == 0 ? row0
                               : static_cast<int>(static_cast<uint32_t>(t + 16) % static_cast<uint32_t>(p.page));
        tma_load_4d(&tm_k, bar, st + u * 16 * RB, 0, w.kvh, row, id, policy);
        tma_load_4d(&tm_v, bar, st + G::kTileBytes + u * 16 * RB, 0, w.kvh, row, id, policy);
        tma_load_3d(&tm_kb, bar, st + 2 * G::kTileBytes + u * G::kHalfScales, row * (SB / 4), w.kvh, id, policy);
        tma_load_3d(&tm_vb, bar, st + 2 * G::kTileBytes + G::kTileScales + u * G::kHalfScales,
                    row * (SB / 4), w.kvh, id, policy);
      }
    }
  };
  // First loads of a segment.
  auto start = [&](const Walk& w) {
    load_ids(w, 0);
    for (int k = 0; k < G::kStages && k < w.count; ++k) issue(w, k, stage_no + k);
  };

  // ------------------------------------------------------------ segments
  Segment seg{};
  bool have = sched.first(cta, seg);
  Walk w{};
  if (have) {
    w = walk_of(seg);
    start(w);
  }
  bool failed = false;
  while (have) {
    const int row_tile = seg.kvh - w.kvh * p.row_tiles;
    const int row_base = row_tile * p.rows;
    const int nrows = p.qrows - row_base < G::kRows ? p.qrows - row_base : G::kRows;
    // ---- query fragments: lane (r, c) holds values c * D / 4 .. of row r
    uint32_t qf[NT][KS][2];
    float row_inv[NT];  // 2^-k of the row's scaling
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int n = nt * 8 + r;
      row_inv[nt] = 1.f;
      uint4 raw[D / 32];
      if (n < nrows) {
        const int h = row_base + n, qi = MULTI ? h / p.group : 0, g = h - qi * p.group;
        const uint4* src = reinterpret_cast<const uint4*>(
            static_cast<const T*>(p.q) +
            ((static_cast<int64_t>(seg.b) * p.seqlen_q + qi) * p.num_heads + w.kvh * p.group + g) * D + c * (D / 4));
#pragma unroll
        for (int i = 0; i < D / 32; ++i) raw[i] = __ldg(src + i);
      } else {
#pragma unroll
        for (int i = 0; i < D / 32; ++i) raw[i] = make_uint4(0, 0, 0, 0);
      }
      float sc = 1.f;
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
          sc = __int_as_float((k + 127) << 23);
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
          }
          qf[nt][2 * i + (j >> 1)][j & 1] = h;  // step s: values 4 s .. 4 s + 3 of the lane's
        }
      }
    }
    // Per column of the lane (query rows 2 c, 2 c + 1 of each 8): the factor
    // of the logits, and how far from the end the row's last key lies.
    float qfac[NT][2];
    int seen[NT][2];
    {
      const float f = __ldg(p.k_scale + w.kvh) * p.scale_log2;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          qfac[nt][e] = f * __shfl_sync(0xffffffffu, row_inv[nt], (2 * c + e) * 4);
          const int h = row_base + nt * 8 + 2 * c + e;
          seen[nt][e] = seg.seqlen + ((MULTI && p.causal) ? h / p.group - (p.seqlen_q - 1) : 0);
        }
      }
    }
    const int all_seen = seg.seqlen - ((MULTI && p.causal) ? p.seqlen_q - 1 : 0);  // by every row

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
      m[nt][0] = m[nt][1] = neg_inf;
      l[nt][0] = l[nt][1] = 0.f;
    }
    // token of row i of an 8-token half tile: neighbours swapped in every second pair
    const int tau = r ^ ((r >> 1) & 1);
    const int tx = (2 * c) ^ (c & 1), ty = (2 * c + 1) ^ (c & 1);  // tau(2 c), tau(2 c + 1)

    for (int k = 0; k < w.count; ++k) {
      const int64_t no = stage_no + k;
      const int slot = static_cast<int>(no % G::kStages);
      if (!failed && !mbar_wait_bounded(bars + slot, static_cast<uint32_t>((no / G::kStages) & 1), abort_flag,
                                        p.timeout_ns))
        failed = true;
      failed = __any_sync(0xffffffffu, failed);
      if (failed) break;
      const uint8_t* st = ring + slot * G::kStageBytes;
      const uint8_t* sk = st + 2 * G::kTileBytes;
      const uint8_t* sv = sk + G::kTileScales;
      const int t0 = w.tok0 + k * kTileTokens;

      // ---- S^T = K . Q^T, two tiles of 16 tokens
      float s[2][NT][4];
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[mt][nt][e] = 0.f;
        const int ra = mt * 16 + tau, rb = ra + 8;
        uint32_t ka[KW], kb[KW];
        if constexpr (KW == 8) {
          uint32_t x[4], y[4];
          load_words<4>(st + ra * RB + swizzled<RB>(ra, 2 * c) * 16, x);
          load_words<4>(st + ra * RB + swizzled<RB>(ra, 2 * c + 1) * 16, y);
#pragma unroll
          for (int i = 0; i < 4; ++i) { ka[i] = x[i]; ka[4 + i] = y[i]; }
          load_words<4>(st + rb * RB + swizzled<RB>(rb, 2 * c) * 16, x);
          load_words<4>(st + rb * RB + swizzled<RB>(rb, 2 * c + 1) * 16, y);
#pragma unroll
          for (int i = 0; i < 4; ++i) { kb[i] = x[i]; kb[4 + i] = y[i]; }
        } else if constexpr (KW == 4) {
          load_words<4>(st + ra * RB + swizzled<RB>(ra, c) * 16, ka);
          load_words<4>(st + rb * RB + swizzled<RB>(rb, c) * 16, kb);
        } else {
          load_words<2>(st + ra * RB + swizzled<RB>(ra, c >> 1) * 16 + (c & 1) * 8, ka);
          load_words<2>(st + rb * RB + swizzled<RB>(rb, c >> 1) * 16 + (c & 1) * 8, kb);
        }
        // block scales of the lane's values: D / 64 bytes of a row
        uint32_t wa, wb;
        const uint8_t* sa = sk + mt * half_scales + tau * SB;
        if constexpr (D == 256) {
          wa = *reinterpret_cast<const uint32_t*>(sa + 4 * c);
          wb = *reinterpret_cast<const uint32_t*>(sa + 8 * SB + 4 * c);
        } else if constexpr (D == 128) {
          wa = *reinterpret_cast<const uint16_t*>(sa + 2 * c);
          wb = *reinterpret_cast<const uint16_t*>(sa + 8 * SB + 2 * c);
        } else {
          wa = sa[c];
          wb = sa[8 * SB + c];
        }
#pragma unroll
        for (int wi = 0; wi < KW; ++wi) {
          const int blk = wi / 2;  // two words a block
          const uint32_t pa = e4m3x2_to_half2(wa >> (16 * (blk / 2))), pb = e4m3x2_to_half2(wb >> (16 * (blk / 2)));
          const uint32_t fa = __byte_perm(pa, pa, blk & 1 ? 0x3232 : 0x1010);
          const uint32_t fb = __byte_perm(pb, pb, blk & 1 ? 0x3232 : 0x1010);
          uint32_t ha[4], hb[4];
          e2m1x8_to_half2x4(ka[wi], ha);
          e2m1x8_to_half2x4(kb[wi], hb);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            ha[j] = hmul2_bits(ha[j], fa);
            hb[j] = hmul2_bits(hb[j], fb);
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma_f16(s[mt][nt], ha[0], hb[0], ha[1], hb[1], qf[nt][2 * wi][0], qf[nt][2 * wi][1]);
            mma_f16(s[mt][nt], ha[2], hb[2], ha[3], hb[3], qf[nt][2 * wi + 1][0], qf[nt][2 * wi + 1][1]);
          }
        }
      }

      // ---- softmax over the stage (log2 domain)
      const bool edge = t0 + kSubTokens > all_seen;  // some row does not see some token
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x = s[mt][nt][e] * qfac[nt][e & 1];
            const int t = t0 + mt * 16 + tau + (e >> 1) * 8;
            s[mt][nt][e] = edge && t >= seen[nt][e & 1] ? neg_inf : x;
          }
      }
      uint32_t pt[2][NT][2];  // P^T fragments of each 16 tokens
      bool moved = false;
      float alpha[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float mx = fmaxf(fmaxf(s[0][nt][e], s[0][nt][e + 2]), fmaxf(s[1][nt][e], s[1][nt][e + 2]));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
          const float m_new = fmaxf(m[nt][e], mx);
          const float m_use = m_new == neg_inf ? 0.f : m_new;
          alpha[nt][e] = fast_exp2(m[nt][e] - m_use);
          moved = moved || m_new != m[nt][e];
          m[nt][e] = m_new;
          float sum = 0.f;
#pragma unroll
          for (int mt = 0; mt < 2; ++mt) {
            s[mt][nt][e] = fast_exp2(s[mt][nt][e] - m_use);
            s[mt][nt][e + 2] = fast_exp2(s[mt][nt][e + 2] - m_use);
            sum += s[mt][nt][e] + s[mt][nt][e + 2];
          }
          l[nt][e] = fmaf(l[nt][e], alpha[nt][e], sum);
        }
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
          pt[mt][nt][0] = transpose8x8(pack_half2(s[mt][nt][0], s[mt][nt][1]));
          pt[mt][nt][1] = transpose8x8(pack_half2(s[mt][nt][2], s[mt][nt][3]));
        }
      }
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[i][nt][e] *= alpha[nt][e & 1];
      }

      // ---- O^T += V^T . P^T
      const bool tail = t0 + kSubTokens > seg.seqlen;
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        const int rows[4] = {ks * 16 + tx, ks * 16 + ty, ks * 16 + tx + 8, ks * 16 + ty + 8};
        uint32_t v[4][VW];
        uint32_t sc[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int row = rows[u];
          const uint8_t* base = st + G::kTileBytes + row * RB;
          const uint8_t* sb = sv + ks * half_scales + (row - ks * 16) * SB;
          if constexpr (D == 256) {
            load_words<4>(base + swizzled<RB>(row, r) * 16, v[u]);
            sc[u] = *reinterpret_cast<const uint16_t*>(sb + 2 * r);
          } else if constexpr (D == 128) {
            load_words<2>(base + swizzled<RB>(row, r >> 1) * 16 + (r & 1) * 8, v[u]);
            sc[u] = sb[r];
          } else {
            load_words<1>(base + swizzled<RB>(row, r >> 2) * 16 + (r & 3) * 4, v[u]);
            sc[u] = sb[r >> 1];
          }
          // Rows past the sequence hold whatever memory held, NaN scales too,
          // and 0 * NaN would reach O: their scales are zeroed.
          if (tail && t0 + row >= seg.seqlen) sc[u] = 0u;
        }
#pragma unroll
        for (int wi = 0; wi < VW; ++wi) {
          const int sh = D == 256 ? 8 * (wi >> 1) : 0;  // the word's block
          const uint32_t f0 = e4m3x2_to_half2(((sc[0] >> sh) & 0xFFu) | (((sc[1] >> sh) & 0xFFu) << 8));
          const uint32_t f1 = e4m3x2_to_half2(((sc[2] >> sh) & 0xFFu) | (((sc[3] >> sh) & 0xFFu) << 8));
          // even codes of both tokens in one word, odd codes in another
          uint32_t e0[4], o0[4], e1[4], o1[4];
          e2m1x8_to_half2x4((v[0][wi] & 0x0F0F0F0Fu) | ((v[1][wi] << 4) & 0xF0F0F0F0u), e0);
          e2m1x8_to_half2x4(((v[0][wi] >> 4) & 0x0F0F0F0Fu) | (v[1][wi] & 0xF0F0F0F0u), o0);
          e2m1x8_to_half2x4((v[2][wi] & 0x0F0F0F0Fu) | ((v[3][wi] << 4) & 0xF0F0F0F0u), e1);
          e2m1x8_to_half2x4(((v[2][wi] >> 4) & 0x0F0F0F0Fu) | (v[3][wi] & 0xF0F0F0F0u), o1);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t a0 = hmul2_bits(e0[j], f0), a1 = hmul2_bits(o0[j], f0);
            const uint32_t a2 = hmul2_bits(e1[j], f1), a3 = hmul2_bits(o1[j], f1);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              mma_f16(acc[wi * 4 + j][nt], a0, a1, a2, a3, pt[ks][nt][0], pt[ks][nt][1]);
          }
        }
      }

      // ---- refill the stage
      const int kn = k + G::kStages;
      __syncwarp();  // every lane has read the stage
      if (kn < w.count) {
        if ((kn & 31) == 0) load_ids(w, kn);
        issue(w, kn, no + G::kStages);
      }
    }
    stage_no += w.count;

    // ---- next segment's first loads
    Segment nx{};
    const bool have_nx = sched.next(seg, range_end, nx);
    const Walk done = w;
    if (have_nx && !failed) {
      w = walk_of(nx);
      start(w);
    }

    // ---- join the warps
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float x = l[nt][e];
        x += __shfl_xor_sync(0xffffffffu, x, 4);
        x += __shfl_xor_sync(0xffffffffu, x, 8);
        x += __shfl_xor_sync(0xffffffffu, x, 16);
        if (r == 0) {
          float* d = ml + (warp * G::kRows + nt * 8 + 2 * c + e) * 2;
          d[0] = m[nt][e];
          d[1] = x;
        }
      }
    __syncthreads();
    const bool stop = *abort_flag != 0;
    // O of this warp relative to the CTA's maximum
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = nt * 8 + 2 * c + e;
        float mm = neg_inf;
#pragma unroll
        for (int i = 0; i < kFp4Warps; ++i) mm = fmaxf(mm, ml[(i * G::kRows + row) * 2]);
        const float f = m[nt][e] == mm ? 1.f : fast_exp2(m[nt][e] - mm);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          acc[i][nt][e] *= f;
          acc[i][nt][e + 2] *= f;
        }
      }
    // Lane (r, c) holds dims r * D / 8 + 2 i (entries e) and + 2 i + 1
    // (entries e + 2) of rows 2 c + e.  Warps 2, 3 leave their sums for 0, 1,
    // which add them; the two halves are added when they are written out.
    auto at = [&](int half, int nt, int e) {
      return join + (half * G::kRows + nt * 8 + 2 * c + e) * G::kRowPad + r * (D / 8);
    };
#pragma unroll
    for (int phase = 0; phase < 2; ++phase) {
      if ((phase == 0) == (warp >= 2)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float4* d = reinterpret_cast<float4*>(at(warp & 1, nt, e));
#pragma unroll
            for (int i = 0; i < MT; i += 2) {
              float4 x = make_float4(acc[i][nt][e], acc[i][nt][e + 2], acc[i + 1][nt][e], acc[i + 1][nt][e + 2]);
              if (phase == 1) {
                const float4 y = d[i / 2];
                x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
              }
              d[i / 2] = x;
            }
          }
      }
      __syncthreads();
    }

    // ---- write: the output, or a partial of a pair cut by range boundaries
    constexpr int kLanes = D / 4;                        // threads of a row, 4 dims each
    constexpr int kRowsPerPass = kFp4Threads / kLanes;
    const int d4 = (tid % kLanes) * 4;
    const int64_t part = static_cast<int64_t>(cta) + seg.pair;
    const bool direct = seg.nseg == 1;
    auto write_row = [&](int row, float4 o, float lse2) {
      const int h = row_base + row, qi = MULTI ? h / p.group : 0, g = h - qi * p.group;
      const int64_t head = done.kvh * p.group + g;
      OutT* dst = static_cast<OutT*>(p.out) +
                  ((static_cast<int64_t>(done.b) * p.seqlen_q + qi) * p.num_heads + head) * D + d4;
      dst[0] = fp4_out<OutT>(o.x);
      dst[1] = fp4_out<OutT>(o.y);
      dst[2] = fp4_out<OutT>(o.z);
      dst[3] = fp4_out<OutT>(o.w);
      if (p.lse != nullptr && d4 == 0)
        p.lse[(static_cast<int64_t>(done.b) * p.num_heads + head) * p.seqlen_q + qi] =
            lse2 == neg_inf ? neg_inf : lse2 * 0.69314718055994531f;
    };
    const float vs = __ldg(p.v_scale + done.kvh);
    if (!stop) {
      for (int row = tid / kLanes; row < nrows; row += kRowsPerPass) {
        float mm = neg_inf, ll = 0.f;
#pragma unroll
        for (int i = 0; i < kFp4Warps; ++i) mm = fmaxf(mm, ml[(i * G::kRows + row) * 2]);
#pragma unroll
        for (int i = 0; i < kFp4Warps; ++i) {
          const float mi = ml[(i * G::kRows + row) * 2];
          ll = fmaf(mi == mm ? 1.f : fast_exp2(mi - mm), ml[(i * G::kRows + row) * 2 + 1], ll);
        }
        const float4 x = *reinterpret_cast<const float4*>(join + row * G::kRowPad + d4);
        const float4 y = *reinterpret_cast<const float4*>(join + (G::kRows + row) * G::kRowPad + d4);
        const bool some = !(ll == 0.f);  // a row that saw a key (NaN stays NaN)
        const float inv = some ? vs / ll : 0.f;
        const float4 o = some ? make_float4((x.x + y.x) * inv, (x.y + y.y) * inv, (x.z + y.z) * inv,
                                            (x.w + y.w) * inv)
                              : make_float4(0.f, 0.f, 0.f, 0.f);
        const float lse2 = some ? mm + fast_log2(ll) : neg_inf;
        if (direct) {
          write_row(row, o, lse2);
        } else {
          *reinterpret_cast<float4*>(p.part_o + (part * p.rows + row) * D + d4) = o;
          if (d4 == 0) p.part_lse[part * p.rows + row] = lse2;
        }
      }
    }
    if (!direct && !stop) {
      __threadfence();
      __syncthreads();
      if (tid == 0) {
        const int is_last = ticket_arrive(p.tickets + seg.pair, *launch_epoch, seg.nseg) ? 1 : 0;
        if (is_last) *reinterpret_cast<volatile unsigned long long*>(p.tickets + seg.pair) = 0ull;
        *last_flag = is_last;
      }
      __syncthreads();
      if (*last_flag) {
        __threadfence();
        const int64_t base = static_cast<int64_t>(seg.cfirst) + seg.pair;
        const float* plse = p.part_lse + base * p.rows;
        const float* po = p.part_o + base * p.rows * D + d4;
        for (int row = tid / kLanes; row < nrows; row += kRowsPerPass) {
          float mm = neg_inf;
          for (int j = 0; j < seg.nseg; ++j) mm = fmaxf(mm, __ldcg(plse + static_cast<int64_t>(j) * p.rows + row));
          float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
          float den = 0.f;
          constexpr int kBatch = 8;
          for (int j0 = 0; j0 < seg.nseg; j0 += kBatch) {
            float4 x[kBatch];
            float lj[kBatch];
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
              const int64_t j = j0 + u;
              lj[u] = neg_inf;
              x[u] = make_float4(0.f, 0.f, 0.f, 0.f);
              if (j < seg.nseg) {
                lj[u] = __ldcg(plse + j * p.rows + row);
                x[u] = __ldcg(reinterpret_cast<const float4*>(po + (j * p.rows + row) * D));
              }
            }
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
              const float wj = lj[u] == neg_inf ? 0.f : fast_exp2(lj[u] - mm);
              if (lj[u] != neg_inf) {
                o.x = fmaf(wj, x[u].x, o.x);
                o.y = fmaf(wj, x[u].y, o.y);
                o.z = fmaf(wj, x[u].z, o.z);
                o.w = fmaf(wj, x[u].w, o.w);
                den += wj;
              }
            }
          }
          const bool some = !(den == 0.f);
          const float inv = some ? 1.f / den : 0.f;
          o.x *= inv; o.y *= inv; o.z *= inv; o.w *= inv;
          write_row(row, o, some ? mm + fast_log2(den) : neg_inf);
        }
      }
    }
    __syncthreads();  // join, ml and last_flag are reused by the next segment
    seg = nx;
    have = have_nx && !stop;
    if (__syncthreads_or(failed)) break;
  }
  if (*abort_flag) {
    if (tid == 0) {
      report_status(p.err, kStatusTimeout);
      // Let copies in flight land before the CTA's shared memory is released (bounded: 2 ms).
      const uint64_t t0 = globaltimer_ns();
      while (globaltimer_ns() - t0 < 2000000ull) {
      }
    }
    __syncthreads();
  }
}

template <typename T, typename OutT, int D, int NT, bool MULTI>
cudaError_t launch_fp4_typed(const Fp4TensorMaps& m, const Fp4DecodeParams& p, int grid, cudaStream_t stream) {
  using G = Fp4Geo<D, NT>;
  auto kern = decode_fp4_kernel<T, OutT, D, NT, MULTI>;
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
  return cudaLaunchKernelEx(&cfg, kern, m.k, m.v, m.k_block, m.v_block, p);
}

template <typename T, typename OutT>
cudaError_t launch_fp4(const Fp4TensorMaps& m, const Fp4DecodeParams& p, int head_dim, int grid,
                       cudaStream_t stream) {
  const bool multi = p.seqlen_q > 1 || p.causal;
  const bool two = p.rows == 16;
  switch (head_dim) {
    case 64:
      if (two)
        return multi ? launch_fp4_typed<T, OutT, 64, 2, true>(m, p, grid, stream)
                     : launch_fp4_typed<T, OutT, 64, 2, false>(m, p, grid, stream);
      return multi ? launch_fp4_typed<T, OutT, 64, 1, true>(m, p, grid, stream)
                   : launch_fp4_typed<T, OutT, 64, 1, false>(m, p, grid, stream);
    case 128:
      if (two)
        return multi ? launch_fp4_typed<T, OutT, 128, 2, true>(m, p, grid, stream)
                     : launch_fp4_typed<T, OutT, 128, 2, false>(m, p, grid, stream);
      return multi ? launch_fp4_typed<T, OutT, 128, 1, true>(m, p, grid, stream)
                   : launch_fp4_typed<T, OutT, 128, 1, false>(m, p, grid, stream);
    default:
      return multi ? launch_fp4_typed<T, OutT, 256, 1, true>(m, p, grid, stream)
                   : launch_fp4_typed<T, OutT, 256, 1, false>(m, p, grid, stream);
  }
}

}  // namespace

}  // namespace fd
