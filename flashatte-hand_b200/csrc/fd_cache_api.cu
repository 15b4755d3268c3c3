// fd_cache_api.cu - the C entry points of the paged cache beside the decode
// ones in fd_api.cu: pages and slots (fd_pages.cu), rows by slot (fd_slots.cu)
// and the 4-bit block-scaled cache (fd_decode_fp4.cuh).
#include <cuda.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

#include "../../include/flashdecode.h"
#include "fd_kernels.h"
#include "fd_trace.h"

namespace {

using fd::report_error;

constexpr int kMaxDevices = 64;

// Split cost model of the 4-bit cache (units and meaning as in fd_api.cu: a
// tile, 128 tokens of one head or 64 of two, costs 8 and a bit).  A pair costs
// its CTA about 5 us beside its tiles (query, joining, partials, arrival), five
// tiles' time.  From 45 to 60 it makes little difference; config 3 takes 135 us
// at 30, 130 at 52 and 135 at 90, 4 speculated tokens of 32 sequences 48.2,
// 46.5 and 48.2 us.
constexpr int kCostTile4 = 2;
constexpr int kCostSeg4 = 52;
// Short launches take whole pairs where no CTA gets more than 12 tiles: 64
// sequences of up to 600 tokens 23.4 -> 22.2 us, eight 1k-token sequences alike,
// but config 1 (16 tiles) 16.2 -> 20.6.
constexpr int kAlignTiles4 = 12;
int cost_tile4() { static const int v = fd::env_int("FD_COST_TILE4", kCostTile4, 0, 64); return v; }
int cost_seg4() { static const int v = fd::env_int("FD_COST_SEG4", kCostSeg4, 1, 256); return v; }
int align_tiles4() { static const int v = fd::env_int("FD_ALIGN_TILES4", kAlignTiles4, 0, 4096); return v; }

// A partial for every (sequence, KV head, row tile), and for every KV head of
// the first and last segment of each CTA.
fd::WorkspaceLayout fp4_workspace(int64_t batch, int64_t num_heads_k, int64_t qrows, int rows, int grid_max,
                                  int head_dim) {
  return fd::workspace_layout(batch, num_heads_k * ((qrows + rows - 1) / rows), rows, 2 * grid_max, head_dim);
}

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

int current_device(int* dev, int** status) {
  if (cudaGetDevice(dev) != cudaSuccess || *dev < 0 || *dev >= kMaxDevices)
    return report_error(FD_ERR_CUDA, "no current CUDA device");
  *status = fd::device_status_word();
  if (*status == nullptr) return report_error(FD_ERR_CUDA, "cannot find the device status word");
  return FD_OK;
}

bool is_16bit(int dtype) { return dtype == FD_DTYPE_BF16 || dtype == FD_DTYPE_FP16; }

// What the appends and the gather check alike: sizes, scales, alignment of
// the caches.
int check_cache(const void* k_cache, const void* v_cache, const void* k_block, const void* v_block,
                const float* k_scale, const float* v_scale, int64_t num_heads_k, int64_t headdim,
                int64_t page, int64_t num_blocks, int cache_dtype) {
  if (k_cache == nullptr || v_cache == nullptr)
    return report_error(FD_ERR_INVALID_ARG, "null tensor pointer");
  if (num_heads_k <= 0 || headdim <= 0 || page <= 0 || num_blocks <= 0)
    return report_error(FD_ERR_INVALID_ARG, "sizes must be positive");
  if (!is_16bit(cache_dtype) && cache_dtype != FD_DTYPE_E4M3 && cache_dtype != FD_DTYPE_E2M1)
    return report_error(FD_ERR_INVALID_ARG, "cache dtype must be bf16, fp16, e4m3 or e2m1");
  if (!is_16bit(cache_dtype) && (k_scale == nullptr || v_scale == nullptr))
    return report_error(FD_ERR_INVALID_ARG, "e4m3 and e2m1 caches need k_scale and v_scale");
  if (cache_dtype == FD_DTYPE_E2M1 && (k_block == nullptr || v_block == nullptr))
    return report_error(FD_ERR_INVALID_ARG, "e2m1 caches need k_block_scale and v_block_scale");
  if (page > INT32_MAX || num_blocks > INT32_MAX || num_heads_k > 65535 || headdim > 65535 ||
      num_heads_k * headdim > (1 << 24))
    return report_error(FD_ERR_UNSUPPORTED, "size exceeds the supported range");
  return FD_OK;
}

fd::SlotParams slot_params(void* k_cache, void* v_cache, void* k_block, void* v_block,
                           const float* k_scale, const float* v_scale, int64_t num_heads_k,
                           int64_t headdim, int64_t page, int64_t num_blocks, int dev, int* status) {
  fd::SlotParams p{};
  p.sms = fd::device_sms(dev);
  p.k_cache = k_cache;
  p.v_cache = v_cache;
  p.k_block = static_cast<uint8_t*>(k_block);
  p.v_block = static_cast<uint8_t*>(v_block);
  p.k_scale = k_scale;
  p.v_scale = v_scale;
  p.num_blocks = num_blocks;
  p.num_heads_k = static_cast<int>(num_heads_k);
  p.head_dim = static_cast<int>(headdim);
  p.page = static_cast<int>(page);
  p.err = status;
  return p;
}

// The append of `p.rows` rows, by slot map or by table, into any cache.
int append_rows(fd::SlotParams p, int src_dtype, int cache_dtype, cudaStream_t stream) {
  const bool wide = p.head_dim % 16 == 0 && aligned(p.k, 16) && aligned(p.v, 16) && aligned(p.k_cache, 16) &&
                    aligned(p.v_cache, 16) && p.k_stride % 8 == 0 && p.v_stride % 8 == 0;
  if (!wide && !is_16bit(cache_dtype))
    return report_error(FD_ERR_UNSUPPORTED,
                        "quantised append: head dim must be a multiple of 16, rows and caches "
                        "16-byte aligned");
  if (p.rows > INT32_MAX) return report_error(FD_ERR_UNSUPPORTED, "size exceeds 32-bit index range");
  if (p.sms <= 0) return report_error(FD_ERR_CUDA, "cannot query SM count");
  const cudaError_t e = wide ? fd::launch_append_slots(p, src_dtype, cache_dtype, stream)
                             : fd::launch_append_slots_narrow(p, stream);
  if (e != cudaSuccess) return report_error(FD_ERR_CUDA, "append launch: %s", cudaGetErrorString(e));
  return fd::report_ok();
}

}  // namespace

extern "C" {

int fd_append_kv_slots(const void* k_new, int64_t k_token_stride, const void* v_new,
                       int64_t v_token_stride, void* k_cache, void* v_cache, void* k_block_scale,
                       void* v_block_scale, const float* k_scale, const float* v_scale,
                       const int64_t* slot_map, int64_t num_tokens, int64_t num_heads_k,
                       int64_t headdim, int64_t page_block_size, int64_t num_blocks, int src_dtype,
                       int cache_dtype, void* stream) {
  fd::TraceRange trace("append_slots");
  int st = check_cache(k_cache, v_cache, k_block_scale, v_block_scale, k_scale, v_scale, num_heads_k,
                       headdim, page_block_size, num_blocks, cache_dtype);
  if (st != FD_OK) return st;
  if (!is_16bit(src_dtype)) return report_error(FD_ERR_INVALID_ARG, "new rows must be bf16 or fp16");
  if (is_16bit(cache_dtype) && cache_dtype != src_dtype)
    return report_error(FD_ERR_INVALID_ARG, "a 16-bit cache takes rows of its own type");
  if (num_tokens < 0) return report_error(FD_ERR_INVALID_ARG, "num_tokens is negative");
  if (num_tokens == 0) return fd::report_ok();
  if (k_new == nullptr || v_new == nullptr || slot_map == nullptr)
    return report_error(FD_ERR_INVALID_ARG, "null tensor pointer");
  if (k_token_stride < num_heads_k * headdim || v_token_stride < num_heads_k * headdim)
    return report_error(FD_ERR_INVALID_ARG, "token strides overlap the rows");
  int dev = 0;
  int* status = nullptr;
  st = current_device(&dev, &status);
  if (st != FD_OK) return st;
  fd::SlotParams p = slot_params(k_cache, v_cache, k_block_scale, v_block_scale, k_scale, v_scale,
                                 num_heads_k, headdim, page_block_size, num_blocks, dev, status);
  p.k = k_new;
  p.v = v_new;
  p.k_stride = k_token_stride;
  p.v_stride = v_token_stride;
  p.slot_map = slot_map;
  p.rows = num_tokens;
  return append_rows(p, src_dtype, cache_dtype, static_cast<cudaStream_t>(stream));
}

int fd_gather_kv_slots(const void* k_cache, const void* v_cache, const void* k_block_scale,
                       const void* v_block_scale, const float* k_scale, const float* v_scale,
                       const int64_t* slot_map, int64_t num_tokens, void* k_out, void* v_out,
                       int64_t num_heads_k, int64_t headdim, int64_t page_block_size,
                       int64_t num_blocks, int cache_dtype, int out_dtype, void* stream) {
  fd::TraceRange trace("gather_slots");
  int st = check_cache(k_cache, v_cache, k_block_scale, v_block_scale, k_scale, v_scale, num_heads_k,
                       headdim, page_block_size, num_blocks, cache_dtype);
  if (st != FD_OK) return st;
  if (!is_16bit(out_dtype) && out_dtype != FD_DTYPE_FP32)
    return report_error(FD_ERR_INVALID_ARG, "out_dtype must be bf16, fp16 or fp32");
  if (num_tokens < 0) return report_error(FD_ERR_INVALID_ARG, "num_tokens is negative");
  if (num_tokens == 0) return fd::report_ok();
  if (slot_map == nullptr || k_out == nullptr || v_out == nullptr)
    return report_error(FD_ERR_INVALID_ARG, "null tensor pointer");
  if (headdim % 16 != 0 || !aligned(k_cache, 16) || !aligned(v_cache, 16) || !aligned(k_out, 16) ||
      !aligned(v_out, 16))
    return report_error(FD_ERR_UNSUPPORTED,
                        "gather: head dim must be a multiple of 16, caches and outputs 16-byte aligned");
  if (num_tokens > INT32_MAX) return report_error(FD_ERR_UNSUPPORTED, "size exceeds 32-bit index range");
  int dev = 0;
  int* status = nullptr;
  st = current_device(&dev, &status);
  if (st != FD_OK) return st;
  fd::SlotParams p = slot_params(const_cast<void*>(k_cache), const_cast<void*>(v_cache),
                                 const_cast<void*>(k_block_scale), const_cast<void*>(v_block_scale),
                                 k_scale, v_scale, num_heads_k, headdim, page_block_size, num_blocks,
                                 dev, status);
  if (p.sms <= 0) return report_error(FD_ERR_CUDA, "cannot query SM count");
  p.k_out = k_out;
  p.v_out = v_out;
  p.slot_map = slot_map;
  p.rows = num_tokens;
  const cudaError_t e = fd::launch_gather_slots(p, cache_dtype, out_dtype, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return report_error(FD_ERR_CUDA, "gather launch: %s", cudaGetErrorString(e));
  return fd::report_ok();
}

int fd_append_kv_paged_fp4(const void* k_new, const void* v_new, void* k_cache, void* v_cache,
                           void* k_block_scale, void* v_block_scale, const float* k_scale,
                           const float* v_scale, const int32_t* cache_seqlens,
                           const int32_t* block_table, int64_t block_table_stride,
                           int64_t batch_size, int64_t seqlen_new, int64_t num_heads_k,
                           int64_t headdim, int64_t page_block_size, int64_t num_blocks,
                           int src_dtype, void* stream) {
  fd::TraceRange trace("append_fp4");
  int st = check_cache(k_cache, v_cache, k_block_scale, v_block_scale, k_scale, v_scale, num_heads_k,
                       headdim, page_block_size, num_blocks, FD_DTYPE_E2M1);
  if (st != FD_OK) return st;
  if (k_new == nullptr || v_new == nullptr || cache_seqlens == nullptr || block_table == nullptr)
    return report_error(FD_ERR_INVALID_ARG, "null tensor pointer");
  if (batch_size <= 0 || seqlen_new <= 0 || block_table_stride <= 0)
    return report_error(FD_ERR_INVALID_ARG, "sizes must be positive");
  if (!is_16bit(src_dtype)) return report_error(FD_ERR_INVALID_ARG, "new rows must be bf16 or fp16");
  if (seqlen_new > 65535 || batch_size > INT32_MAX || batch_size * seqlen_new > INT32_MAX)
    return report_error(FD_ERR_UNSUPPORTED, "size exceeds 32-bit index range");
  int dev = 0;
  int* status = nullptr;
  st = current_device(&dev, &status);
  if (st != FD_OK) return st;
  fd::SlotParams p = slot_params(k_cache, v_cache, k_block_scale, v_block_scale, k_scale, v_scale,
                                 num_heads_k, headdim, page_block_size, num_blocks, dev, status);
  p.k = k_new;
  p.v = v_new;
  p.k_stride = p.v_stride = num_heads_k * headdim;
  p.seqlens = cache_seqlens;
  p.block_table = block_table;
  p.bt_stride = block_table_stride;
  p.seqlen_new = static_cast<int>(seqlen_new);
  p.rows = batch_size * seqlen_new;
  return append_rows(p, src_dtype, FD_DTYPE_E2M1, static_cast<cudaStream_t>(stream));
}

int fd_assign_pages(int32_t* block_table, int64_t block_table_stride, const int32_t* cache_seqlens,
                    const int32_t* new_lens, const int32_t* free_pages, int32_t* free_count,
                    int64_t batch_size, int64_t page_block_size, int64_t num_blocks,
                    int32_t* seqlens_out, int32_t* cu_new, int64_t* slot_map, int64_t num_slots,
                    void* stream) {
  fd::TraceRange trace("assign_pages");
  if (block_table == nullptr || cache_seqlens == nullptr || new_lens == nullptr || free_pages == nullptr ||
      free_count == nullptr || seqlens_out == nullptr || cu_new == nullptr ||
      (slot_map == nullptr && num_slots > 0))
    return report_error(FD_ERR_INVALID_ARG, "null tensor pointer");
  if (batch_size <= 0 || page_block_size <= 0 || num_blocks <= 0 || block_table_stride <= 0 || num_slots < 0)
    return report_error(FD_ERR_INVALID_ARG, "sizes must be positive");
  if (batch_size > fd::kMaxPagedRequests)
    return report_error(FD_ERR_UNSUPPORTED, "at most %d requests", fd::kMaxPagedRequests);
  if (page_block_size > INT32_MAX || num_blocks > INT32_MAX || num_slots > INT32_MAX ||
      block_table_stride > INT32_MAX)
    return report_error(FD_ERR_UNSUPPORTED, "size exceeds 32-bit index range");
  int dev = 0;
  int* status = nullptr;
  const int st = current_device(&dev, &status);
  if (st != FD_OK) return st;
  const int sms = fd::device_sms(dev);
  if (sms <= 0) return report_error(FD_ERR_CUDA, "cannot query SM count");
  fd::AssignPagesParams p;
  p.block_table = block_table;
  p.seqlens = cache_seqlens;
  p.new_lens = new_lens;
  p.free_pages = free_pages;
  p.free_count = free_count;
  p.seqlens_out = seqlens_out;
  p.cu_new = cu_new;
  p.slot_map = slot_map;
  p.bt_stride = block_table_stride;
  p.num_blocks = num_blocks;
  p.num_slots = num_slots;
  p.batch = static_cast<int>(batch_size);
  p.page = static_cast<int>(page_block_size);
  p.err = status;
  const cudaError_t e = fd::launch_assign_pages(p, sms, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return report_error(FD_ERR_CUDA, "assign launch: %s", cudaGetErrorString(e));
  return fd::report_ok();
}

int fd_release_pages(int32_t* block_table, int64_t block_table_stride,
                     const int32_t* cache_seqlens, const int32_t* keep_lens, int32_t* free_pages,
                     int32_t* free_count, int64_t batch_size, int64_t page_block_size,
                     int64_t num_blocks, void* stream) {
  fd::TraceRange trace("release_pages");
  if (block_table == nullptr || cache_seqlens == nullptr || keep_lens == nullptr || free_pages == nullptr ||
      free_count == nullptr)
    return report_error(FD_ERR_INVALID_ARG, "null tensor pointer");
  if (batch_size <= 0 || page_block_size <= 0 || num_blocks <= 0 || block_table_stride <= 0)
    return report_error(FD_ERR_INVALID_ARG, "sizes must be positive");
  if (batch_size > fd::kMaxPagedRequests)
    return report_error(FD_ERR_UNSUPPORTED, "at most %d requests", fd::kMaxPagedRequests);
  if (page_block_size > INT32_MAX || num_blocks > INT32_MAX || block_table_stride > INT32_MAX)
    return report_error(FD_ERR_UNSUPPORTED, "size exceeds 32-bit index range");
  int dev = 0;
  int* status = nullptr;
  const int st = current_device(&dev, &status);
  if (st != FD_OK) return st;
  const int sms = fd::device_sms(dev);
  if (sms <= 0) return report_error(FD_ERR_CUDA, "cannot query SM count");
  fd::ReleasePagesParams p;
  p.block_table = block_table;
  p.seqlens = cache_seqlens;
  p.keep_lens = keep_lens;
  p.free_pages = free_pages;
  p.free_count = free_count;
  p.bt_stride = block_table_stride;
  p.num_blocks = num_blocks;
  p.batch = static_cast<int>(batch_size);
  p.page = static_cast<int>(page_block_size);
  p.err = status;
  const cudaError_t e = fd::launch_release_pages(p, sms, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return report_error(FD_ERR_CUDA, "release launch: %s", cudaGetErrorString(e));
  return fd::report_ok();
}

size_t fd_decode_workspace_size_fp4(int64_t batch_size, int64_t seqlen_q, int64_t num_heads,
                                    int64_t num_heads_k, int64_t headdim) {
  if (batch_size <= 0 || seqlen_q <= 0 || num_heads <= 0 || num_heads_k <= 0 ||
      num_heads % num_heads_k != 0 || (headdim != 64 && headdim != 128 && headdim != 256))
    return 0;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return 0;
  const int sms = fd::device_sms(dev);
  if (sms <= 0) return 0;
  const int64_t nb = batch_size < fd::kMaxBatchPerLaunch ? batch_size : fd::kMaxBatchPerLaunch;
  const int64_t qrows = seqlen_q * (num_heads / num_heads_k);
  const int rows = fd::fp4_rows(static_cast<int>(headdim), qrows);
  return fp4_workspace(nb, num_heads_k, qrows, rows, fd::fp4_max_grid(static_cast<int>(headdim), rows, sms),
                       static_cast<int>(headdim)).total;
}

int fd_decode_paged_fp4(const void* q, void* k_cache, void* v_cache, void* k_block_scale,
                        void* v_block_scale, const float* k_scale, const float* v_scale,
                        const void* k_new, const void* v_new, int64_t seqlen_new, void* out,
                        float* lse, const int32_t* cache_seqlens, const int32_t* block_table,
                        int64_t block_table_stride, int64_t batch_size, int64_t seqlen_q,
                        int64_t num_heads, int64_t num_heads_k, int64_t headdim,
                        int64_t page_block_size, int64_t num_blocks, int q_dtype, int out_dtype,
                        float softmax_scale, int causal, int64_t max_seqlen_k, void* workspace,
                        size_t workspace_bytes, void* stream) {
  fd::TraceRange trace("decode_fp4");
  if (q == nullptr || out == nullptr || cache_seqlens == nullptr || block_table == nullptr)
    return report_error(FD_ERR_INVALID_ARG, "null tensor pointer");
  if ((k_new == nullptr) != (v_new == nullptr))
    return report_error(FD_ERR_INVALID_ARG, "k_new and v_new must be given together");
  if (batch_size <= 0 || seqlen_q <= 0 || num_heads <= 0 || num_heads_k <= 0 || block_table_stride <= 0)
    return report_error(FD_ERR_INVALID_ARG, "sizes must be positive");
  if (num_heads % num_heads_k != 0)
    return report_error(FD_ERR_INVALID_ARG, "num_heads %lld not a multiple of num_heads_k %lld",
                        (long long)num_heads, (long long)num_heads_k);
  if (!is_16bit(q_dtype)) return report_error(FD_ERR_INVALID_ARG, "query dtype must be bf16 or fp16");
  if (out_dtype != q_dtype && out_dtype != FD_DTYPE_FP32)
    return report_error(FD_ERR_INVALID_ARG, "out_dtype must equal the query dtype or be fp32");
  if (!std::isfinite(softmax_scale))
    return report_error(FD_ERR_INVALID_ARG, "softmax_scale must be finite");
  if (k_new != nullptr && (seqlen_new <= 0 || seqlen_new > 65535))
    return report_error(FD_ERR_INVALID_ARG, "seqlen_new out of range");
  int st = check_cache(k_cache, v_cache, k_block_scale, v_block_scale, k_scale, v_scale, num_heads_k,
                       headdim, page_block_size, num_blocks, FD_DTYPE_E2M1);
  if (st != FD_OK) return st;
  if (headdim != 64 && headdim != 128 && headdim != 256)
    return report_error(FD_ERR_UNSUPPORTED, "e2m1 cache: head dim must be 64, 128 or 256 (got %lld)",
                        (long long)headdim);
  if (page_block_size % 16 != 0)
    return report_error(FD_ERR_UNSUPPORTED, "e2m1 cache: page size must be a multiple of 16");
  if (seqlen_q > 65535 || num_heads > 65535 || batch_size > INT32_MAX ||
      batch_size * seqlen_q * num_heads > INT32_MAX || block_table_stride > INT32_MAX ||
      (k_new != nullptr && batch_size * seqlen_new > INT32_MAX))
    return report_error(FD_ERR_UNSUPPORTED, "size exceeds 32-bit index range");
  if (!aligned(q, 16) || !aligned(out, 16) || !aligned(k_cache, 16) || !aligned(v_cache, 16) ||
      !aligned(k_block_scale, 16) || !aligned(v_block_scale, 16) || !aligned(k_new, 16) || !aligned(v_new, 16))
    return report_error(FD_ERR_UNSUPPORTED, "e2m1 cache: tensors must be 16-byte aligned");
  int dev = 0;
  int* status = nullptr;
  st = current_device(&dev, &status);
  if (st != FD_OK) return st;
  const int sms = fd::device_sms(dev);
  if (sms <= 0) return report_error(FD_ERR_CUDA, "cannot query SM count");

  const int D = static_cast<int>(headdim);
  const int group = static_cast<int>(num_heads / num_heads_k);
  const int64_t qrows = seqlen_q * group;
  const int rows = fd::fp4_rows(D, qrows);
  const int64_t row_tiles = (qrows + rows - 1) / rows;
  // neighbouring KV heads of a token are read together where their count allows
  const int heads = num_heads_k % 2 == 0 ? 2 : 1;
  const int64_t head_sets = num_heads_k / heads;
  const int grid_max = fd::fp4_max_grid(D, rows, sms);
  const int64_t nb_max = batch_size < fd::kMaxBatchPerLaunch ? batch_size : fd::kMaxBatchPerLaunch;
  const fd::WorkspaceLayout wl = fp4_workspace(nb_max, num_heads_k, qrows, rows, grid_max, D);
  cudaStream_t cs = static_cast<cudaStream_t>(stream);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  if (ws == nullptr) {
    const char* why = "";
    ws = static_cast<uint8_t*>(fd::library_workspace(dev, wl.total, cs, &why));
    if (ws == nullptr) return report_error(FD_ERR_WORKSPACE, "%zu-byte workspace: %s", wl.total, why);
  } else if (workspace_bytes < wl.total) {
    return report_error(FD_ERR_WORKSPACE, "workspace %zu bytes < required %zu", workspace_bytes, wl.total);
  } else if (!aligned(ws, 256)) {
    return report_error(FD_ERR_WORKSPACE, "workspace not 256-byte aligned");
  }

  // (a length counts up to 2^29 - 1 tokens, as the kernel clamps it)
  const int64_t rows_max = block_table_stride * page_block_size;
  const int64_t kv_max = rows_max < 0x1fffffff ? rows_max : 0x1fffffff;
  const int64_t len_bound = max_seqlen_k > 0 && max_seqlen_k < kv_max ? max_seqlen_k : kv_max;
  // the schedule's tiles are kTileTokens / heads tokens of `heads` heads
  const int64_t tiles_bound = (len_bound * heads + fd::kTileTokens - 1) / fd::kTileTokens;
  const int lead = cost_seg4();
  const int64_t per_seq_cost = lead + ((kv_max * heads + fd::kTileTokens - 1) / fd::kTileTokens + 1) *
                                                 (8 + static_cast<int64_t>(cost_tile4()));
  // (whole pairs are taken a head at a time: `heads` as many)
  const int64_t aligned_cost = heads * (lead + static_cast<int64_t>(align_tiles4()) * (8 + cost_tile4()) + 1);
  int64_t tiles_per_launch = row_tiles;
  int64_t per_launch = fd::seqs_per_launch(per_seq_cost, aligned_cost, head_sets * row_tiles, grid_max);
  if (per_launch == 0) {  // not one sequence's rows: as many of its row tiles as fit, a launch each
    tiles_per_launch = fd::seqs_per_launch(per_seq_cost, aligned_cost, head_sets, grid_max);
    if (tiles_per_launch > row_tiles) tiles_per_launch = row_tiles;
    per_launch = 1;
  }
  if (tiles_per_launch == 0)
    return report_error(FD_ERR_UNSUPPORTED, "a block table of %lld tokens is too wide for %lld KV heads",
                        (long long)rows_max, (long long)num_heads_k);

  int len_add = 0;
  if (k_new != nullptr) {  // everything the attention would refuse has been checked
    st = fd_append_kv_paged_fp4(k_new, v_new, k_cache, v_cache, k_block_scale, v_block_scale, k_scale, v_scale,
                                cache_seqlens, block_table, block_table_stride, batch_size, seqlen_new,
                                num_heads_k, headdim, page_block_size, num_blocks, q_dtype, stream);
    if (st != FD_OK) return st;
    len_add = static_cast<int>(seqlen_new);
  }
  const int64_t es = 2, oes = out_dtype == FD_DTYPE_FP32 ? 4 : 2;
  for (int64_t b0 = 0; b0 < batch_size; b0 += per_launch) {
    const int64_t nb = batch_size - b0 < per_launch ? batch_size - b0 : per_launch;
    for (int64_t t0 = 0; t0 < row_tiles; t0 += tiles_per_launch) {
      const int64_t nt = row_tiles - t0 < tiles_per_launch ? row_tiles - t0 : tiles_per_launch;
      fd::Fp4DecodeParams p{};
      p.q = static_cast<const uint8_t*>(q) + b0 * seqlen_q * num_heads * headdim * es;
      p.k_cache = static_cast<const uint8_t*>(k_cache);
      p.v_cache = static_cast<const uint8_t*>(v_cache);
      p.k_block = static_cast<const uint8_t*>(k_block_scale);
      p.v_block = static_cast<const uint8_t*>(v_block_scale);
      p.out = static_cast<uint8_t*>(out) + b0 * seqlen_q * num_heads * headdim * oes;
      p.lse = lse != nullptr ? lse + b0 * num_heads * seqlen_q : nullptr;
      p.k_scale = k_scale;
      p.v_scale = v_scale;
      p.seqlens = cache_seqlens + b0;
      p.block_table = block_table + b0 * block_table_stride;
      p.bt_stride = block_table_stride;
      p.num_blocks = num_blocks;
      p.batch = static_cast<int>(nb);
      p.num_heads = static_cast<int>(num_heads);
      p.num_heads_k = static_cast<int>(num_heads_k);
      p.group = group;
      p.page = static_cast<int>(page_block_size);
      p.seqlen_q = static_cast<int>(seqlen_q);
      p.causal = causal ? 1 : 0;
      p.qrows = static_cast<int>(qrows);
      p.row_tiles = static_cast<int>(nt);
      p.row_tile0 = static_cast<int>(t0);
      p.rows = rows;
      p.heads = heads;
      p.len_add = len_add;
      p.scale_log2 = softmax_scale * 1.4426950408889634f;
      p.tickets = reinterpret_cast<unsigned long long*>(ws + wl.tickets_off);
      p.part_lse = reinterpret_cast<float*>(ws + wl.lse_off);
      p.part_o = reinterpret_cast<float*>(ws + wl.o_off);
      p.epoch_word = reinterpret_cast<unsigned long long*>(ws + wl.epoch_off);
      p.err = status;
      p.cost_tile = cost_tile4();
      p.cost_seg = lead;
      p.align_tiles = align_tiles4();
      p.pdl = fd::pdl_enabled() ? 1 : 0;
      const int64_t work = nb * head_sets * nt * tiles_bound;
      const int grid = static_cast<int>(work < grid_max ? work : grid_max);
      const cudaError_t e = fd::launch_decode_fp4(p, D, q_dtype, out_dtype == FD_DTYPE_FP32, grid, cs);
      if (e != cudaSuccess) return report_error(FD_ERR_CUDA, "e2m1 launch: %s", cudaGetErrorString(e));
    }
  }
  return fd::report_ok();
}

}  // extern "C"
