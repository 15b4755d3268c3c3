// fd_pages.cu - block tables and slot maps built on the GPU.
//
// A serving step gives request b (L_b tokens stored) a_b new tokens.  With
// pages of P tokens it holds ceil(L_b / P) pages and needs
// n_b = ceil((L_b + a_b) / P) - ceil(L_b / P) more.  With e_b the sum of n
// over the requests before b, request b takes entries e_b .. e_b + n_b - 1
// from the top of the pool's stack of free pages, and token t of the step's
// packed tokens (request by request) gets the cache slot
// table[b, pos / P] * P + pos % P.  All of it is integer prefix sums and
// look-ups: the kernel is bound by its launch and a few dependent loads for a
// decode step, and by the slot map's stores for long prompts.
//
// Every CTA scans the lengths itself (8192 requests at most: they fit its
// shared memory, and a scan of 256 values costs less than a second launch),
// then takes its share of the slots and of the new table entries.  The new
// lengths and the pool's count are written by the CTA that finishes its scan
// last, so that the caller may update the lengths in place.
//
// Measured on a B200 (assign and release of what it took, device time of both
// launches): one token for each of 4 requests 8.2 us, 4 for each of 256
// 12 us; 1.1 million prompt tokens of 256 requests (a slot map of 16.8 MB,
// 66 000 pages) 23 us, of which the assign is about half.  Both are chains of
// lengths, scan, table and stores; two launches that do nothing take 4 us.
#include <cuda_runtime.h>

#include <cstdint>

#include "fd_kernels.h"
#include "fd_ptx.cuh"

namespace fd {

namespace {

constexpr int kPagesThreads = 256;
constexpr int kReleaseThreads = 512;
constexpr int kReleaseBatch = 8;  // table entries per thread and round

// Inclusive sum of (x, y) over the block, in thread order; `sums` holds one
// pair per warp.  Returns the block's totals in (tx, ty).
template <int THREADS>
__device__ __forceinline__ void block_scan2(int64_t& x, int64_t& y, int64_t& tx, int64_t& ty,
                                            longlong2* sums) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t u = __shfl_up_sync(0xffffffffu, x, o), v = __shfl_up_sync(0xffffffffu, y, o);
    if (lane >= o) { x += u; y += v; }
  }
  __syncthreads();  // the previous use of `sums` has been read
  if (lane == 31) sums[warp] = make_longlong2(x, y);
  __syncthreads();
  int64_t bx = 0, by = 0;
  tx = ty = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    const longlong2 s = sums[w];
    if (w < warp) { bx += s.x; by += s.y; }
    tx += s.x;
    ty += s.y;
  }
  x += bx;
  y += by;
}

__device__ __forceinline__ int clamp_i32(int64_t v) {
  return static_cast<int>(v < INT32_MAX ? v : INT32_MAX);
}

// Largest i in [0, n) with prefix[i] <= v, for prefix[0] = 0 <= v.
__device__ __forceinline__ int find_owner(const int* prefix, int n, int v) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (prefix[mid] <= v) lo = mid; else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ int pages_of(int len, int page) {
  return static_cast<int>((static_cast<uint32_t>(len) + static_cast<uint32_t>(page) - 1u) /
                          static_cast<uint32_t>(page));
}

__global__ void __launch_bounds__(kPagesThreads) assign_pages_kernel(const AssignPagesParams p) {
  extern __shared__ int pages_smem[];
  __shared__ longlong2 sums[kPagesThreads / 32];
  __shared__ int taken_pages, last_cta;
  const int B = p.batch, page = p.page, tid = threadIdx.x;
  int* tok = pages_smem;        // [B + 1] new tokens before request b
  int* pre = tok + B + 1;       // [B + 1] pages wanted before request b
  int* len = pre + B + 1;       // [B] stored length, or ~length if the request gets nothing
  if (tid == 0) taken_pages = 0;
  const int64_t row_tokens = p.bt_stride * static_cast<int64_t>(page);
  int free = *reinterpret_cast<volatile const int32_t*>(p.free_count);
  free = free < 0 ? 0 : (free < p.num_blocks ? free : static_cast<int>(p.num_blocks));

  // Each thread scans a run of consecutive requests.
  const int per = (B + kPagesThreads - 1) / kPagesThreads;
  const int b0 = tid * per < B ? tid * per : B, b1 = b0 + per < B ? b0 + per : B;
  auto wanted = [&](int b, int& L, int& a, bool& fits) {
    L = p.seqlens[b];
    a = p.new_lens[b];
    L = L < 0 ? 0 : L;
    a = a < 0 ? 0 : a;
    const int64_t end = static_cast<int64_t>(L) + a;
    fits = end <= row_tokens && end <= INT32_MAX;
    return fits ? pages_of(static_cast<int>(end), page) - pages_of(L, page) : 0;
  };
  int64_t nt = 0, np = 0;
  for (int b = b0; b < b1; ++b) {
    int L, a;
    bool fits;
    np += wanted(b, L, a, fits);
    nt += a;
  }
  const int64_t mine_t = nt, mine_p = np;
  int64_t all_t, all_p;
  block_scan2<kPagesThreads>(nt, np, all_t, all_p, sums);
  nt -= mine_t;
  np -= mine_p;
  bool refused = false;
  int most = 0;
  for (int b = b0; b < b1; ++b) {
    int L, a;
    bool fits;
    const int n = wanted(b, L, a, fits);
    tok[b] = clamp_i32(nt);
    pre[b] = clamp_i32(np);
    nt += a;
    np += n;
    const bool granted = fits && (n == 0 || np <= free);
    if (granted && n > 0) most = static_cast<int>(np);
    refused = refused || !granted;
    len[b] = granted ? L : ~L;
  }
  if (tid == 0) {
    tok[B] = clamp_i32(all_t);
    pre[B] = clamp_i32(all_p);
  }
  if (most > 0) atomicMax(&taken_pages, most);
  __syncthreads();

  // This CTA has read the lengths and the count: they may change now.
  if (tid == 0) {
    int last = 1;
    if (gridDim.x > 1) {
      __threadfence();
      last = atomicAdd(p.free_count + 1, 1) == static_cast<int>(gridDim.x) - 1;
      __threadfence();
    }
    last_cta = last;
  }
  __syncthreads();
  const int taken = taken_pages;
  if (last_cta) {
    for (int b = tid; b < B; b += kPagesThreads) {
      const int L = len[b];
      int a = p.new_lens[b];
      a = a < 0 ? 0 : a;
      p.seqlens_out[b] = L < 0 ? ~L : L + a;
    }
    for (int b = tid; b <= B; b += kPagesThreads) p.cu_new[b] = tok[b];
    if (refused || (tid == 0 && all_t > p.num_slots)) report_status(p.err, kStatusNoPages);
    if (tid == 0) {
      p.free_count[0] = free - taken;
      p.free_count[1] = 0;
    }
  }

  const int stride_all = static_cast<int>(gridDim.x) * kPagesThreads;
  const int first = static_cast<int>(blockIdx.x) * kPagesThreads + tid;
  // k-th page of the step
  auto fresh_page = [&](int k) {
    const int id = p.free_pages[free - 1 - k];
    if (id >= 0 && id < p.num_blocks) return id;
    report_status(p.err, kStatusBadPage);
    return -1;
  };
  for (int64_t k = first; k < taken; k += stride_all) {
    const int b = find_owner(pre, B, static_cast<int>(k));
    p.block_table[b * p.bt_stride + pages_of(len[b], page) + (k - pre[b])] = fresh_page(static_cast<int>(k));
  }
  // Slots, four consecutive tokens a thread: one search, then steps along the
  // page, the pages and the requests.
  const int total = tok[B];
  const bool wide = (reinterpret_cast<uintptr_t>(p.slot_map) & 15u) == 0;
  for (int64_t t0 = static_cast<int64_t>(first) * 4; t0 < p.num_slots; t0 += static_cast<int64_t>(stride_all) * 4) {
    long long slot[4] = {-1, -1, -1, -1};
    if (t0 < total) {
      int b = find_owner(tok, B, static_cast<int>(t0));
      int end = 0, row = 0, j = 0, have = 0;  // the request's last token + 1; the token's row of page column j
      int64_t base = -1;                      // slot of the page's row 0
      bool enter = true;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int t = static_cast<int>(t0) + i;
        if (t >= total) break;
        if (!enter && t >= end) {
          do ++b; while (t >= tok[b + 1]);
          enter = true;
        }
        const int L = len[b];
        bool fetch = false;
        if (enter) {
          end = tok[b + 1];
          if (L >= 0) {
            const uint32_t pos = static_cast<uint32_t>(L) + static_cast<uint32_t>(t - tok[b]);
            j = static_cast<int>(pos / static_cast<uint32_t>(page));
            row = static_cast<int>(pos - static_cast<uint32_t>(j) * static_cast<uint32_t>(page));
            have = pages_of(L, page);
            fetch = true;
          }
          enter = false;
        } else if (++row == page) {
          row = 0;
          ++j;
          fetch = true;
        }
        if (L < 0) continue;
        if (fetch) {
          int id;
          if (j < have) {
            id = p.block_table[b * p.bt_stride + j];
            if (id < 0 || id >= p.num_blocks) {
              report_status(p.err, kStatusBadPage);
              id = -1;
            }
          } else {
            id = fresh_page(pre[b] + j - have);
          }
          base = id < 0 ? -1 : static_cast<int64_t>(id) * page;
        }
        if (base >= 0) slot[i] = base + row;
      }
    }
    if (wide && t0 + 4 <= p.num_slots) {
      longlong2* d = reinterpret_cast<longlong2*>(p.slot_map + t0);
      d[0] = make_longlong2(slot[0], slot[1]);
      d[1] = make_longlong2(slot[2], slot[3]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (t0 + i < p.num_slots) p.slot_map[t0 + i] = slot[i];
    }
  }
}

// Pages beyond ceil(keep_b / P) of each request go back to the stack.  They
// are pushed in reverse order (last request first, last page first), so that
// giving back what one assign took leaves the stack as it was.  With f the
// number of a page among the R given back, its place is count + R - 1 - f:
// the CTAs work apart, and the last to finish writes the count.  An entry
// outside the pool leaves a hole there, which that CTA closes.  (One CTA
// for all 66 000 pages took 165 us longer.)  Only if the
// stack has no room for all (a page released twice) does one CTA push them in
// order, since then each one's place depends on all before it.
__global__ void __launch_bounds__(kReleaseThreads) release_pages_kernel(const ReleasePagesParams p) {
  extern __shared__ int pages_smem[];
  __shared__ longlong2 sums[kReleaseThreads / 32];
  const int B = p.batch, page = p.page, tid = threadIdx.x;
  int* pre = pages_smem;      // [B + 1] pages given back before request b
  int* from = pre + B + 1;    // [B] first table column given back
  int count = p.free_count[0];
  count = count < 0 ? 0 : (count < p.num_blocks ? count : static_cast<int>(p.num_blocks));
  const int per = (B + kReleaseThreads - 1) / kReleaseThreads;
  const int b0 = tid * per < B ? tid * per : B, b1 = b0 + per < B ? b0 + per : B;
  auto columns = [&](int b, int& first) {
    const int64_t cap = p.bt_stride;
    const int L = p.seqlens[b], keep = p.keep_lens[b];
    const int have = L <= 0 ? 0 : pages_of(L, page);
    first = keep <= 0 ? 0 : pages_of(keep, page);
    const int end = have < cap ? have : static_cast<int>(cap);
    return end > first ? end - first : 0;
  };
  int64_t n = 0, unused = 0;
  for (int b = b0; b < b1; ++b) {
    int first;
    n += columns(b, first);
  }
  const int64_t mine = n;
  int64_t total, unused_total;
  block_scan2<kReleaseThreads>(n, unused, total, unused_total, sums);
  n -= mine;
  for (int b = b0; b < b1; ++b) {
    int first;
    const int m = columns(b, first);
    pre[b] = clamp_i32(n);
    from[b] = first;
    n += m;
  }
  if (tid == 0) pre[B] = clamp_i32(total);
  __syncthreads();
  const int R = pre[B];
  if (static_cast<int64_t>(count) + R <= p.num_blocks) {
    int bad = 0;
    const int stride_all = static_cast<int>(gridDim.x) * kReleaseThreads;
    for (int64_t f = static_cast<int64_t>(blockIdx.x) * kReleaseThreads + tid; f < R; f += stride_all) {
      const int b = find_owner(pre, B, static_cast<int>(f));
      int32_t* e = p.block_table + b * p.bt_stride + from[b] + (f - pre[b]);
      int id = *e;
      *e = -1;
      if (id < 0 || id >= p.num_blocks) {
        report_status(p.err, kStatusBadPage);
        id = -1;
        bad = 1;
      }
      p.free_pages[count + R - 1 - f] = id;
    }
    bad = __syncthreads_or(bad);
    __shared__ int arrivals;
    if (tid == 0) {
      // CTAs done in the low half, those that met a bad entry in the high
      __threadfence();
      const int add = 1 + (bad ? 1 << 16 : 0);
      arrivals = gridDim.x > 1 ? atomicAdd(p.free_count + 1, add) + add : add;
      __threadfence();
    }
    __syncthreads();
    if ((arrivals & 0xFFFF) != static_cast<int>(gridDim.x)) return;
    int good_all = R;
    if (arrivals >> 16) {  // close the holes, in order
      good_all = 0;
      for (int64_t base = 0; base < R; base += kReleaseThreads) {
        const int64_t i = base + tid;
        const int id = i < R ? __ldcg(p.free_pages + count + i) : -1;
        int64_t good = id >= 0 ? 1 : 0, none = 0, all, all_none;
        const int64_t mine_good = good;
        block_scan2<kReleaseThreads>(good, none, all, all_none, sums);
        // every entry of this round has been read, and places only move down
        if (id >= 0) p.free_pages[count + good_all + good - mine_good] = id;
        good_all += static_cast<int>(all);
      }
    }
    if (tid == 0) {
      p.free_count[0] = count + good_all;
      p.free_count[1] = 0;
    }
    return;
  }
  if (blockIdx.x != 0) return;
  int64_t pushed = 0;
  for (int64_t base = 0; base < R; base += kReleaseThreads * kReleaseBatch) {
    // entry u of the thread: number base + tid * batch + u from the end
    int ids[kReleaseBatch];
    int64_t good = 0, none = 0;
#pragma unroll
    for (int u = 0; u < kReleaseBatch; ++u) {
      const int64_t f = R - 1 - (base + tid * kReleaseBatch + u);
      ids[u] = -1;
      if (f >= 0) {
        const int b = find_owner(pre, B, static_cast<int>(f));
        int32_t* e = p.block_table + b * p.bt_stride + from[b] + (f - pre[b]);
        const int id = *e;
        *e = -1;
        if (id >= 0 && id < p.num_blocks) {
          ids[u] = id;
          ++good;
        } else {
          report_status(p.err, kStatusBadPage);
        }
      }
    }
    const int64_t my_good = good;
    int64_t all, all_none;
    block_scan2<kReleaseThreads>(good, none, all, all_none, sums);
    int64_t at = count + pushed + good - my_good;
#pragma unroll
    for (int u = 0; u < kReleaseBatch; ++u) {
      if (ids[u] < 0) continue;
      if (at < p.num_blocks) p.free_pages[at] = ids[u];
      else report_status(p.err, kStatusBadPage);  // more pages than the pool has
      ++at;
    }
    pushed += all;
  }
  if (tid == 0) {
    const int64_t c = count + pushed;
    p.free_count[0] = static_cast<int>(c < p.num_blocks ? c : p.num_blocks);
  }
}

constexpr size_t assign_smem(int batch) { return (3 * static_cast<size_t>(batch) + 2) * sizeof(int); }
constexpr size_t release_smem(int batch) { return (2 * static_cast<size_t>(batch) + 1) * sizeof(int); }

// Shared memory above the default limit (static and dynamic together) has to be
// allowed, once per device: what the largest call takes, so that no call lowers
// the limit under another thread's.
cudaError_t allow_smem(const void* kernel, size_t most, unsigned long long* allowed) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const unsigned long long bit = 1ull << (dev & 63);
  if ((__atomic_load_n(allowed, __ATOMIC_ACQUIRE) & bit) != 0) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(most));
  if (e == cudaSuccess) __atomic_fetch_or(allowed, bit, __ATOMIC_RELEASE);
  return e;
}

}  // namespace

cudaError_t launch_assign_pages(const AssignPagesParams& p, int sms, cudaStream_t stream) {
  static unsigned long long allowed = 0;
  const cudaError_t e =
      allow_smem(reinterpret_cast<const void*>(assign_pages_kernel), assign_smem(kMaxPagedRequests), &allowed);
  if (e != cudaSuccess) return e;
  int64_t grid = (p.num_slots + 4 * kPagesThreads - 1) / (4 * kPagesThreads);
  grid = grid < 1 ? 1 : (grid < 2 * sms ? grid : 2 * sms);
  assign_pages_kernel<<<static_cast<unsigned>(grid), kPagesThreads, assign_smem(p.batch), stream>>>(p);
  return cudaGetLastError();
}

cudaError_t launch_release_pages(const ReleasePagesParams& p, int sms, cudaStream_t stream) {
  static unsigned long long allowed = 0;
  const cudaError_t e =
      allow_smem(reinterpret_cast<const void*>(release_pages_kernel), release_smem(kMaxPagedRequests), &allowed);
  if (e != cudaSuccess) return e;
  // a CTA for every 8 pages of a thread that the table could hold
  const int64_t most = (p.batch * p.bt_stride + 8 * kReleaseThreads - 1) / (8 * kReleaseThreads);
  const unsigned grid = static_cast<unsigned>(most < sms ? most : sms);
  release_pages_kernel<<<grid, kReleaseThreads, release_smem(p.batch), stream>>>(p);
  return cudaGetLastError();
}

}  // namespace fd
