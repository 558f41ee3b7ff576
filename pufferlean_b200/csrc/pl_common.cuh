// Shared definitions for the B200 PPO+Muon update library: status codes, the per-thread
// error message behind pl_last_error(), launch checks, and small device helpers.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <stdio.h>

#include "../../include/pufferlean_b200.h"

namespace pl {

// Records a formatted message as this thread's last error and returns `code`.
int set_error(int code, const char* fmt, ...);
void clear_error();
int check_cuda(cudaError_t e, const char* what);

#define PL_CUDA(call)                                          \
  do {                                                         \
    cudaError_t _e = (call);                                   \
    if (_e != cudaSuccess) return ::pl::check_cuda(_e, #call); \
  } while (0)

#define PL_LAUNCH(what)                                        \
  do {                                                         \
    cudaError_t _e = cudaGetLastError();                       \
    if (_e != cudaSuccess) return ::pl::check_cuda(_e, what);  \
  } while (0)

#define PL_REQUIRE(cond, code, ...)                            \
  do {                                                         \
    if (!(cond)) return ::pl::set_error((code), __VA_ARGS__);  \
  } while (0)

static inline long ceil_div(long a, long b) { return (a + b - 1) / b; }
static inline long round_up(long a, long b) { return (a + b - 1) / b * b; }

#ifdef __CUDACC__
// Programmatic dependent launch. A kernel launched with launch_early may start while the kernel before it in the stream
// finishes; grid_wait holds it until that kernel is complete and its writes are seen (so every global access comes
// after it), grid_next lets the kernel after it start likewise. Both do nothing in an ordinary launch.
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
template <typename... P, typename... A>
static inline cudaError_t launch_early(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, A&&... args) {
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}
#endif

// Per-device word that kernels with bounded waits set when a wait runs out (0 = none).
unsigned* device_error_word();
// Reads and clears the word (synchronizes the device). Returns PL_OK or PL_ERR_DEVICE_TIMEOUT.
int device_error_check();

}  // namespace pl

#define PL_ERR_MBAR_TIMEOUT 0x100u
