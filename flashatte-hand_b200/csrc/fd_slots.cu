// fd_slots.cu - packed new tokens into the paged cache by slot, and cache
// rows back out by slot.
//
// A slot is page * page_size + row.  The append takes rows [T, Hkv, D] (any
// token stride, e.g. a slice of a fused projection) and stores row t at slot
// slot_map[t] of a 16-bit, e4m3 or 4-bit block-scaled cache; the gather is
// its inverse and returns the values the cache stands for.  Slots below zero
// are padding (skipped by the append, zeros from the gather); a slot past the
// pool is skipped the same way and reported (FD_ERR_BAD_PAGE).
//
// Both are single passes: one thread handles 16 consecutive values of K and of
// V (two 16-byte loads each), which is one scale block of the 4-bit format, so
// a block's largest magnitude never leaves its thread.  A CTA takes several
// rows, so that what depends on the unit alone (head, scales) is read once.
//
// Measured on a B200 (copy rate 6.56 TB/s): 59k tokens of 8 heads of 128
// values in bf16 into the 4-bit cache 62.7 us, 4.9 TB/s of bytes read and
// written; the quantising bounds it (schedulers issue in 74 % of the cycles,
// the half-rate ALU works in 56 %).  Back 66.5 us, 5.2 TB/s, bound by the
// latency of slot, codes and store (two rows at a time: 80 registers, 81 us;
// six CTAs an SM: spilled, 112 us; lanes exchanging halves for whole-sector
// stores: 64 registers, 72 us).  The same rows into an e4m3 cache 75 us (its
// divisions are whole ones) and back 64; into a 16-bit one 81, 5.9 TB/s, and
// back 79.  12k 16-bit rows 9.0 us for 50 MB, 5.6 TB/s; a decode step's rows 3
// us, a launch.
#include <cuda_runtime.h>

#include <cstdint>

#include "fd_fp4.cuh"
#include "fd_kernels.h"
#include "fd_ptx.cuh"

namespace fd {

namespace {

constexpr int kSlotThreads = 256;

template <typename T> __device__ __forceinline__ float2 to_float2(uint32_t w);
template <> __device__ __forceinline__ float2 to_float2<__nv_bfloat16>(uint32_t w) {
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w));
}
template <> __device__ __forceinline__ float2 to_float2<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

__device__ __forceinline__ void unpack(const uint4& a, const uint4& b, uint32_t (&w)[8]) {
  w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
  w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
}

// A cache row: its page and its row in the page; page < 0 if there is none.
struct Place {
  int64_t page;
  int row;
};

__device__ __forceinline__ Place place_of_slot(int64_t slot, int page, int64_t num_blocks, int* err,
                                               bool report) {
  Place at{-1, 0};
  if (slot < 0) return at;
  int64_t pg;
  if ((page & (page - 1)) == 0) {
    pg = slot >> (31 - __clz(page));
    at.row = static_cast<int>(slot) & (page - 1);
  } else if (slot <= static_cast<int64_t>(UINT32_MAX)) {  // a 64-bit division is a long sequence
    const uint32_t s = static_cast<uint32_t>(slot), q = s / static_cast<uint32_t>(page);
    pg = q;
    at.row = static_cast<int>(s - q * static_cast<uint32_t>(page));
  } else {
    pg = slot / page;
    at.row = static_cast<int>(slot - pg * page);
  }
  if (pg < num_blocks) at.page = pg;
  else if (report) report_status(err, kStatusBadPage);
  return at;
}

// Where row `r` of an append goes: through the slot map, or (dense appends)
// position max(cache_seqlens[b], 0) + t of sequence b through its block table.
__device__ __forceinline__ Place place_of_row(const SlotParams& p, int64_t r, bool report) {
  if (p.slot_map != nullptr) return place_of_slot(p.slot_map[r], p.page, p.num_blocks, p.err, report);
  const int b = static_cast<int>(r / p.seqlen_new);
  const int stored = p.seqlens[b];
  const int64_t pos = static_cast<int64_t>(stored < 0 ? 0 : stored) + (r - static_cast<int64_t>(b) * p.seqlen_new);
  const int64_t idx = pos / p.page;
  Place at{-1, static_cast<int>(pos - idx * p.page)};
  if (idx < p.bt_stride) {
    const int pg = p.block_table[b * p.bt_stride + idx];
    if (pg >= 0 && pg < p.num_blocks) at.page = pg;
    else if (report) report_status(p.err, kStatusBadPage);
  }
  return at;
}

// x / d, correctly rounded, for r = 1 / d correctly rounded and nothing near
// the ends of the range: one Newton correction of x r with the exact
// remainder (Markstein's theorem).  Rounding to e2m1 then sees the tie cases
// exactly, which a plain product with the reciprocal would miss.  The remainder
// is taken with its sign turned: +0 for x = +0 and -0 alike, so that -0 keeps
// its sign (x - q d would add +0 to it).
__device__ __forceinline__ float divide(float x, float d, float r) {
  const float q = x * r;
  return fmaf(-fmaf(q, d, -x), r, q);
}

__device__ __forceinline__ uint32_t e2m1x2(float lo, float hi) {
  return static_cast<uint32_t>(
      __nv_cvt_float2_to_fp4x2(make_float2(lo, hi), __NV_E2M1, cudaRoundNearest));
}

// One block of 16 values to 8 bytes of codes and a scale byte.  A block with
// a NaN gets a NaN scale and zero codes: all of it reads back as NaN.
template <typename T>
__device__ __forceinline__ uint2 quantize_block(const uint32_t (&w)[8], float head_scale, uint8_t& scale) {
  // The largest magnitude: 16-bit floats without their sign order as whole
  // numbers, NaN above infinity above all else.
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = __vmaxu2(top, w[i] & 0x7FFF7FFFu);
  top = top > (top << 16) ? top & 0xFFFF0000u : top << 16;
  const float amax = to_float2<T>(top).y;
  const uint32_t s8 = static_cast<uint32_t>(
      __nv_cvt_float_to_fp8(__fdiv_rn(amax, 6.f * head_scale), __NV_SATFINITE, __NV_E4M3));
  scale = static_cast<uint8_t>(s8);
  const float s = e4m3_to_float(s8);
  if (!(s > 0.f)) return make_uint2(0u, 0u);
  const float d = s * head_scale;
  uint32_t c[2] = {0u, 0u};
  // the quotients are at most amax / d: with both well inside the range (and
  // no infinity among the values) no step of divide() leaves it
  if (amax < 1e30f && d > 1e-25f && d < 1e25f && amax < d * 1e25f) {
    const float r = __frcp_rn(d);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 f = to_float2<T>(w[i]);
      c[i >> 2] |= e2m1x2(divide(f.x, d, r), divide(f.y, d, r)) << (8 * (i & 3));
    }
  } else {
#pragma unroll 1
    for (int i = 0; i < 8; ++i) {
      uint32_t x = w[0];
#pragma unroll
      for (int j = 1; j < 8; ++j) x = i == j ? w[j] : x;
      const float2 f = to_float2<T>(x);
      const uint32_t byte = e2m1x2(f.x / d, f.y / d) << (8 * (i & 3));
      if (i < 4) c[0] |= byte; else c[1] |= byte;
    }
  }
  return make_uint2(c[0], c[1]);
}

template <typename T>
__device__ __forceinline__ uint4 quantize_e4m3(const uint32_t (&w)[8], float scale) {
  uint32_t c[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 a = to_float2<T>(w[2 * i]), b = to_float2<T>(w[2 * i + 1]);
    c[i] = e4m3x2(a.x / scale, a.y / scale) | (e4m3x2(b.x / scale, b.y / scale) << 16);
  }
  return make_uint4(c[0], c[1], c[2], c[3]);
}

enum CacheKind { kNative = 0, kE4m3 = 1, kFp4 = 2 };

// A row is `units` = num_heads_k * head_dim / 16 units of 16 values.  A CTA
// covers rows_per_cta rows, rows_at of them side by side (one row in several
// rounds if it has more units than the CTA threads), so that what depends on
// the unit alone is computed once a thread.
template <typename F>
__device__ __forceinline__ void for_units(const SlotParams& p, F&& body) {
  const int units = p.num_heads_k * (p.head_dim / 16);
  const int dr = units < kSlotThreads ? threadIdx.x / units : 0;
  if (dr >= p.rows_at) return;
  const int64_t r0 = static_cast<int64_t>(blockIdx.x) * p.rows_per_cta;
  const int64_t r1 = r0 + p.rows_per_cta < p.rows ? r0 + p.rows_per_cta : p.rows;
  for (int u = threadIdx.x - dr * units; u < units; u += kSlotThreads)
    body(u, units, r0 + dr, r1);
}

template <typename T, int KIND>
__global__ void __launch_bounds__(kSlotThreads) append_slots_kernel(const SlotParams p) {
  for_units(p, [&](int u, int units, int64_t r0, int64_t r1) {
    const int per_head = p.head_dim / 16, h = u / per_head;
    const T* kr = static_cast<const T*>(p.k) + u * 16;
    const T* vr = static_cast<const T*>(p.v) + u * 16;
    float kg = 1.f, vg = 1.f;
    if constexpr (KIND != kNative) {
      kg = __ldg(p.k_scale + h);
      vg = __ldg(p.v_scale + h);
    }
    for (int64_t r = r0; r < r1; r += p.rows_at) {
      const uint4* ks = reinterpret_cast<const uint4*>(kr + r * p.k_stride);
      const uint4* vs = reinterpret_cast<const uint4*>(vr + r * p.v_stride);
      const uint4 k0 = __ldcs(ks), k1 = __ldcs(ks + 1), v0 = __ldcs(vs), v1 = __ldcs(vs + 1);
      const Place at = place_of_row(p, r, u == 0);
      if (at.page < 0) continue;
      const int64_t dst = (at.page * p.page + at.row) * units + u;  // unit of the cache
      if constexpr (KIND == kNative) {
        uint4* kd = static_cast<uint4*>(p.k_cache) + dst * 2;
        uint4* vd = static_cast<uint4*>(p.v_cache) + dst * 2;
        kd[0] = k0; kd[1] = k1;
        vd[0] = v0; vd[1] = v1;
      } else {
        uint32_t kw[8], vw[8];
        unpack(k0, k1, kw);
        unpack(v0, v1, vw);
        if constexpr (KIND == kE4m3) {
          static_cast<uint4*>(p.k_cache)[dst] = quantize_e4m3<T>(kw, kg);
          static_cast<uint4*>(p.v_cache)[dst] = quantize_e4m3<T>(vw, vg);
        } else {
          const int64_t sd = ((at.page * p.num_heads_k + h) * p.page + at.row) * per_head + (u - h * per_head);
          uint8_t s;
          static_cast<uint2*>(p.k_cache)[dst] = quantize_block<T>(kw, kg, s);
          p.k_block[sd] = s;
          static_cast<uint2*>(p.v_cache)[dst] = quantize_block<T>(vw, vg, s);
          p.v_block[sd] = s;
        }
      }
    }
  });
}

// 16-bit rows that are not 16-byte aligned or not a multiple of 16 values.
__global__ void __launch_bounds__(kSlotThreads) append_slots_narrow_kernel(const SlotParams p) {
  const int n = p.num_heads_k * p.head_dim;
  const int64_t r = blockIdx.x;
  const Place at = place_of_row(p, r, threadIdx.x == 0);
  if (at.page < 0) return;
  const uint16_t* ks = static_cast<const uint16_t*>(p.k) + r * p.k_stride;
  const uint16_t* vs = static_cast<const uint16_t*>(p.v) + r * p.v_stride;
  const int64_t dst = (at.page * p.page + at.row) * n;
  for (int i = threadIdx.x; i < n; i += kSlotThreads) {
    static_cast<uint16_t*>(p.k_cache)[dst + i] = ks[i];
    static_cast<uint16_t*>(p.v_cache)[dst + i] = vs[i];
  }
}

template <typename O> struct Out16;
template <> struct Out16<__nv_bfloat16> {
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};
template <> struct Out16<__half> {
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};

template <typename O>
__device__ __forceinline__ void store16(void* base, int64_t unit, const float (&x)[16]) {
  if constexpr (sizeof(O) == 4) {
    float4* d = static_cast<float4*>(base) + unit * 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) d[i] = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
  } else {
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = Out16<O>::pack(x[2 * i], x[2 * i + 1]);
    uint4* d = static_cast<uint4*>(base) + unit * 2;
    d[0] = make_uint4(w[0], w[1], w[2], w[3]);
    d[1] = make_uint4(w[4], w[5], w[6], w[7]);
  }
}

// The 16 values of unit `src` of a cache.
template <typename C, int KIND>
__device__ __forceinline__ void load16(const void* cache, int64_t src, float scale, float block_scale,
                                       float (&x)[16]) {
  if constexpr (KIND == kNative) {
    const uint4* s = static_cast<const uint4*>(cache) + src * 2;
    uint32_t w[8];
    unpack(__ldg(s), __ldg(s + 1), w);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 f = to_float2<C>(w[i]);
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  } else if constexpr (KIND == kE4m3) {
    const uint4 q = __ldg(static_cast<const uint4*>(cache) + src);
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 a = e4m3x2_to_float2(w[i]), b = e4m3x2_to_float2(w[i] >> 16);
      x[4 * i] = a.x * scale;
      x[4 * i + 1] = a.y * scale;
      x[4 * i + 2] = b.x * scale;
      x[4 * i + 3] = b.y * scale;
    }
  } else {
    const uint2 q = __ldg(static_cast<const uint2*>(cache) + src);
    const uint32_t w[2] = {q.x, q.y};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint32_t h[4];
      e2m1x8_to_half2x4(w[i], h);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        // e2m1 * e4m3 is exact in fp32; the head's scale rounds once
        const float2 f = to_float2<__half>(h[j]);
        x[8 * i + 2 * j] = f.x * block_scale * scale;
        x[8 * i + 2 * j + 1] = f.y * block_scale * scale;
      }
    }
  }
}

template <typename C, typename O, int KIND>
__global__ void __launch_bounds__(kSlotThreads) gather_slots_kernel(const SlotParams p) {
  for_units(p, [&](int u, int units, int64_t r0, int64_t r1) {
    const int per_head = p.head_dim / 16, h = u / per_head;
    float kg = 1.f, vg = 1.f;
    if constexpr (KIND != kNative) {
      kg = __ldg(p.k_scale + h);
      vg = __ldg(p.v_scale + h);
    }
    for (int64_t r = r0; r < r1; r += p.rows_at) {
      const Place at = place_of_slot(p.slot_map[r], p.page, p.num_blocks, p.err, u == 0);
      float k[16], v[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) k[j] = v[j] = 0.f;
      if (at.page >= 0) {
        const int64_t src = (at.page * p.page + at.row) * units + u;
        float kb = 1.f, vb = 1.f;
        if constexpr (KIND == kFp4) {
          const int64_t sd = ((at.page * p.num_heads_k + h) * p.page + at.row) * per_head + (u - h * per_head);
          kb = e4m3_to_float(__ldg(p.k_block + sd));
          vb = e4m3_to_float(__ldg(p.v_block + sd));
        }
        load16<C, KIND>(p.k_cache, src, kg, kb, k);
        load16<C, KIND>(p.v_cache, src, vg, vb, v);
      }
      store16<O>(p.k_out, r * units + u, k);
      store16<O>(p.v_out, r * units + u, v);
    }
  });
}

// Rows side by side in a CTA, rows per CTA (up to 8 rounds, while the grid
// still covers the device several times) and the grid.
unsigned slot_grid(SlotParams& p) {
  const int units = p.num_heads_k * (p.head_dim / 16);
  p.rows_at = units < kSlotThreads ? kSlotThreads / units : 1;
  const int64_t rounds = p.rows / (static_cast<int64_t>(p.rows_at) * p.sms * 16);
  p.rows_per_cta = p.rows_at * static_cast<int>(rounds < 1 ? 1 : (rounds < 8 ? rounds : 8));
  return static_cast<unsigned>((p.rows + p.rows_per_cta - 1) / p.rows_per_cta);
}

template <typename T>
cudaError_t launch_append_typed(SlotParams p, int kind, cudaStream_t stream) {
  const unsigned grid = slot_grid(p);
  if (kind == kNative) append_slots_kernel<T, kNative><<<grid, kSlotThreads, 0, stream>>>(p);
  else if (kind == kE4m3) append_slots_kernel<T, kE4m3><<<grid, kSlotThreads, 0, stream>>>(p);
  else append_slots_kernel<T, kFp4><<<grid, kSlotThreads, 0, stream>>>(p);
  return cudaGetLastError();
}

template <typename C, int KIND>
cudaError_t launch_gather_typed(SlotParams p, int out_dtype, cudaStream_t stream) {
  const unsigned grid = slot_grid(p);
  if (out_dtype == 0) gather_slots_kernel<C, __nv_bfloat16, KIND><<<grid, kSlotThreads, 0, stream>>>(p);
  else if (out_dtype == 1) gather_slots_kernel<C, __half, KIND><<<grid, kSlotThreads, 0, stream>>>(p);
  else gather_slots_kernel<C, float, KIND><<<grid, kSlotThreads, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_append_slots(const SlotParams& p, int src_dtype, int cache_dtype,
                                cudaStream_t stream) {
  if (p.rows <= 0) return cudaSuccess;
  const int kind = cache_dtype == 4 ? kFp4 : cache_dtype == 3 ? kE4m3 : kNative;
  return src_dtype == 0 ? launch_append_typed<__nv_bfloat16>(p, kind, stream)
                        : launch_append_typed<__half>(p, kind, stream);
}

cudaError_t launch_append_slots_narrow(const SlotParams& p, cudaStream_t stream) {
  if (p.rows <= 0) return cudaSuccess;
  append_slots_narrow_kernel<<<static_cast<unsigned>(p.rows), kSlotThreads, 0, stream>>>(p);
  return cudaGetLastError();
}

cudaError_t launch_gather_slots(const SlotParams& p, int cache_dtype, int out_dtype,
                                cudaStream_t stream) {
  if (p.rows <= 0) return cudaSuccess;
  switch (cache_dtype) {
    case 0: return launch_gather_typed<__nv_bfloat16, kNative>(p, out_dtype, stream);
    case 1: return launch_gather_typed<__half, kNative>(p, out_dtype, stream);
    case 3: return launch_gather_typed<__half, kE4m3>(p, out_dtype, stream);
    default: return launch_gather_typed<__half, kFp4>(p, out_dtype, stream);
  }
}

}  // namespace fd
