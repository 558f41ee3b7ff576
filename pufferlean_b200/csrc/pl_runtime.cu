// Library runtime: error reporting, device selection, launch accounting, the per-device error
// word that bounded device-side waits write to.
#include <stdarg.h>
#include <string.h>

#include <atomic>
#include <mutex>

#include "pl_common.cuh"
#include "pl_runtime.h"

namespace pl {

static thread_local char g_err[1024] = "";
static std::atomic<uint64_t> g_launches{0};

int set_error(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
  return code;
}
void clear_error() { g_err[0] = 0; }

int check_cuda(cudaError_t e, const char* what) {
  if (e == cudaErrorNoDevice || e == cudaErrorInsufficientDriver)
    return set_error(PL_ERR_NO_DEVICE, "%s: %s (no usable CUDA device; this library has no CPU fallback)", what,
                     cudaGetErrorString(e));
  if (e == cudaErrorMemoryAllocation) return set_error(PL_ERR_NOMEM, "%s: %s", what, cudaGetErrorString(e));
  return set_error(PL_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

void count_launch(uint64_t n) { g_launches.fetch_add(n, std::memory_order_relaxed); }

// The word is a variable of the module, so that its first use allocates and clears nothing: that would end a stream
// capture that a library call runs in.
static __device__ unsigned g_err_word;

unsigned* device_error_word() {
  static std::atomic<unsigned*> at[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return nullptr;
  if (unsigned* p = at[dev].load(std::memory_order_relaxed)) return p;
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;  // the address itself may be asked for during a capture
  if (cudaThreadExchangeStreamCaptureMode(&mode) != cudaSuccess) return nullptr;
  void* p = nullptr;
  const cudaError_t e = cudaGetSymbolAddress(&p, g_err_word);
  cudaThreadExchangeStreamCaptureMode(&mode);
  if (e != cudaSuccess) return nullptr;
  at[dev].store((unsigned*)p, std::memory_order_relaxed);
  return (unsigned*)p;
}

int device_error_check() {
  unsigned* w = device_error_word();
  if (!w) return PL_OK;
  unsigned v = 0;
  PL_CUDA(cudaMemcpy(&v, w, sizeof(unsigned), cudaMemcpyDeviceToHost));
  if (v) {
    cudaMemset(w, 0, sizeof(unsigned));
    return set_error(PL_ERR_DEVICE_TIMEOUT, "a device-side bounded wait ran out (code 0x%x)", v);
  }
  return PL_OK;
}

// Requires a usable device; the library never computes on the host in place of the GPU.
int require_device() {
  int n = 0;
  cudaError_t e = cudaGetDeviceCount(&n);
  if (e != cudaSuccess || n == 0)
    return set_error(PL_ERR_NO_DEVICE, "no usable CUDA device (%s); this library has no CPU fallback",
                     e == cudaSuccess ? "count 0" : cudaGetErrorString(e));
  return PL_OK;
}

}  // namespace pl

extern "C" {

const char* pl_last_error(void) { return pl::g_err; }

int pl_device_count(void) {
  int n = 0;
  if (cudaGetDeviceCount(&n) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  return n;
}

int pl_set_device(int device) {
  PL_CUDA(cudaSetDevice(device));
  return PL_OK;
}

int pl_get_device(int* device) {
  PL_REQUIRE(device, PL_ERR_INVALID, "pl_get_device: NULL");
  PL_CUDA(cudaGetDevice(device));
  return PL_OK;
}

int pl_device_check(void) {
  int rc = pl::require_device();
  if (rc) return rc;
  PL_CUDA(cudaDeviceSynchronize());  // streams that do not wait for the default one too
  return pl::device_error_check();
}

uint64_t pl_kernel_launch_count(void) { return pl::g_launches.load(); }

}  // extern "C"

namespace pl {
static void* g_scratch[64][64];
static size_t g_scratch_sz[64][64];
static std::mutex g_scratch_mu;

void* scratch(int slot, size_t bytes) {
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || slot < 0 || slot >= 64) {
    set_error(PL_ERR_INVALID, "scratch slot %d / device %d out of range", slot, dev);
    return nullptr;
  }
  std::lock_guard<std::mutex> g(g_scratch_mu);
  if (bytes == 0) bytes = 16;
  if (g_scratch_sz[dev][slot] < bytes) {
    if (g_scratch[dev][slot]) cudaFree(g_scratch[dev][slot]);
    g_scratch[dev][slot] = nullptr;
    g_scratch_sz[dev][slot] = 0;
    void* p = nullptr;
    cudaError_t e = cudaMalloc(&p, bytes);
    if (e != cudaSuccess) {
      check_cuda(e, "cudaMalloc(scratch)");
      return nullptr;
    }
    g_scratch[dev][slot] = p;
    g_scratch_sz[dev][slot] = bytes;
  }
  return g_scratch[dev][slot];
}

struct SmemLimit {
  const void* kernel;
  size_t bytes;
};
static SmemLimit g_smem[64][256];
static int g_smem_n[64];
static std::mutex g_smem_mu;

int raise_smem_on(int device, const void* kernel, size_t bytes, int (*set)(const void*, size_t)) {
  if (device < 0 || device >= 64) return set(kernel, bytes);
  std::lock_guard<std::mutex> g(g_smem_mu);
  SmemLimit* t = g_smem[device];
  int i = 0;
  while (i < g_smem_n[device] && t[i].kernel != kernel) i++;
  if (i < g_smem_n[device] && t[i].bytes >= bytes) return PL_OK;
  const int rc = set(kernel, bytes);
  if (rc == PL_OK && i < 256) {
    t[i] = SmemLimit{kernel, bytes};
    if (i == g_smem_n[device]) g_smem_n[device]++;
  }
  return rc;
}

static int set_smem(const void* kernel, size_t bytes) {
  PL_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
  return PL_OK;
}
int raise_smem(const void* kernel, size_t bytes) {
  int dev = 0;
  PL_CUDA(cudaGetDevice(&dev));
  return raise_smem_on(dev, kernel, bytes, set_smem);
}
}  // namespace pl
