// What the translation units of the library share: the thread-local error text, the current device's state, the launch
// count, and each unit's part of ga_init().
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <cstring>
#include <utility>

namespace ga {
namespace api {

int fail(const char* fmt, ...);         // records the text for ga_last_error(), returns 1
int device(int* dev, int* sm);          // current device, which ga_init() has prepared, and its SMs
// Tensor map of a 16-bit pool for boxes of 64 dims x `box` tokens of one head and page, 128-byte swizzle; false: it has none.
bool encode_map(CUtensorMap* map, const void* base, int hd, int page, int kvh, int pages, long long s_tok, long long s_head,
                long long s_page, int box);
void launches(int n);                   // what ga_last_launch_count() reports
int init_paged();                       // paged.cu: shared memory limits on the current device
int init_pages();                       // pages.cu: the same

#define GA_TRY(expr)                                                                                   \
  do {                                                                                                 \
    cudaError_t e_ = (expr);                                                                           \
    if (e_ != cudaSuccess) return ::ga::api::fail("%s failed: %s", #expr, cudaGetErrorString(e_));     \
  } while (0)

// Launch with programmatic stream serialization: the kernel may be scheduled while its predecessor in the stream
// drains, and orders itself with griddepcontrol.wait.
template <typename... KArgs, typename... Args>
cudaError_t launch_serial(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, Args&&... args) {
  cudaLaunchConfig_t cfg;
  std::memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
}

}  // namespace api
}  // namespace ga
