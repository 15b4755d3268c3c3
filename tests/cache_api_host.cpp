// The launches that the paged-cache entry points make, without a GPU: their
// host code (fd_cache_api.cu) linked with stand-ins for the device, the
// launchers and the library's scratch.  Every launch prints a line.
//   cache_api_host <SMs> decode B sq Hq Hkv D page width
//   cache_api_host <SMs> append | append_paged | gather
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <cstring>

#include "../flashatte-hand_b200/csrc/fd_kernels.h"
#include "../include/flashdecode.h"

static int g_sms = 148;
static int g_word = 0;

extern "C" {
cudaError_t CUDARTAPI cudaGetDevice(int* dev) { *dev = 0; return cudaSuccess; }
const char* CUDARTAPI cudaGetErrorString(cudaError_t) { return "error"; }
}

namespace fd {
int* device_status_word() { return &g_word; }
int device_sms(int) { return g_sms; }
bool pdl_enabled() { return true; }
int env_int(const char*, int dflt, int, int) { return dflt; }
int report_ok() { return FD_OK; }
int report_error(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vprintf(fmt, ap);
  va_end(ap);
  printf("\n");
  return code;
}
void* library_workspace(int, size_t, cudaStream_t, const char**) { return reinterpret_cast<void*>(4096); }
WorkspaceLayout workspace_layout(int64_t, int64_t, int64_t, int, int) { return WorkspaceLayout{0, 64, 128, 256, 512, 1024}; }
// Sequences of a launch: a cost line of all of them times grid + 1 below 2^32.
int64_t seqs_per_launch(int64_t per_seq, int64_t aligned, int64_t pairs, int grid) {
  const int64_t c = per_seq > aligned ? per_seq : aligned;
  const int64_t n = static_cast<int64_t>(UINT32_MAX) / (c * pairs * (grid + 1)), m = INT32_MAX / c;
  const int64_t least = n < m ? n : m;
  return least < kMaxBatchPerLaunch ? least : kMaxBatchPerLaunch;
}
int fp4_rows(int head_dim, int64_t qrows) { return head_dim == 256 || qrows <= 8 ? 8 : 16; }
int fp4_max_grid(int head_dim, int, int sms) { return (head_dim == 64 ? 3 : 2) * sms; }
cudaError_t launch_decode_fp4(const Fp4DecodeParams& p, int, int, bool, int grid, cudaStream_t) {
  printf("decode seq %lld batch %d tiles %d %d rows %d heads %d grid %d cost %d %d align %d\n",
         static_cast<long long>(reinterpret_cast<uintptr_t>(p.seqlens) - 4096) / 4, p.batch, p.row_tile0, p.row_tiles,
         p.rows, p.heads, grid, p.cost_tile, p.cost_seg, p.align_tiles);
  return cudaSuccess;
}
cudaError_t launch_append_slots(const SlotParams& p, int, int, cudaStream_t) {
  printf("append rows %lld sms %d\n", static_cast<long long>(p.rows), p.sms);
  return cudaSuccess;
}
cudaError_t launch_append_slots_narrow(const SlotParams& p, cudaStream_t) { return launch_append_slots(p, 0, 0, nullptr); }
cudaError_t launch_gather_slots(const SlotParams& p, int, int, cudaStream_t) {
  printf("gather rows %lld sms %d\n", static_cast<long long>(p.rows), p.sms);
  return cudaSuccess;
}
cudaError_t launch_assign_pages(const AssignPagesParams&, int, cudaStream_t) { return cudaSuccess; }
cudaError_t launch_release_pages(const ReleasePagesParams&, int, cudaStream_t) { return cudaSuccess; }
}  // namespace fd

int main(int argc, char** argv) {
  if (argc < 3) return 2;
  g_sms = std::atoi(argv[1]);
  void* at = reinterpret_cast<void*>(4096);  // never followed
  float* f = static_cast<float*>(at);
  int32_t* i32 = static_cast<int32_t*>(at);
  int64_t* i64 = static_cast<int64_t*>(at);
  int status = -1;
  if (std::strcmp(argv[2], "decode") == 0 && argc == 10) {
    int64_t v[7];
    for (int i = 0; i < 7; ++i) v[i] = std::atoll(argv[3 + i]);
    status = fd_decode_paged_fp4(at, at, at, at, at, f, f, nullptr, nullptr, 0, at, f, i32, i32, v[6], v[0], v[1], v[2],
                                 v[3], v[4], v[5], 1000, FD_DTYPE_BF16, FD_DTYPE_BF16, 0.1f, 0, 0, nullptr, 0, nullptr);
  } else if (std::strcmp(argv[2], "append") == 0) {
    status = fd_append_kv_slots(at, 256, at, 256, at, at, at, at, f, f, i64, 100000, 2, 128, 16, 1000, FD_DTYPE_BF16,
                                FD_DTYPE_E2M1, nullptr);
  } else if (std::strcmp(argv[2], "append_paged") == 0) {
    status = fd_append_kv_paged_fp4(at, at, at, at, at, at, f, f, i32, i32, 4, 2, 1, 2, 128, 16, 1000, FD_DTYPE_BF16,
                                    nullptr);
  } else if (std::strcmp(argv[2], "gather") == 0) {
    status = fd_gather_kv_slots(at, at, at, at, f, f, i64, 100000, at, at, 2, 128, 16, 1000, FD_DTYPE_E2M1,
                                FD_DTYPE_BF16, nullptr);
  }
  printf("status %d\n", status);
  return 0;
}
