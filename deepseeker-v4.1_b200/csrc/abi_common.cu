// Error reporting and small device queries shared by every entry point.
#include <stdarg.h>
#include <string.h>

#include "ds_common.cuh"

namespace {
thread_local char g_last_error[512] = "";
}

namespace ds {

int set_error(int status, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_last_error, sizeof(g_last_error), fmt, ap);
  va_end(ap);
  return status;
}

int cuda_status(cudaError_t e, const char* what) {
  return set_error(DS_ECUDA, "CUDA error %d (%s) in %s", (int)e, cudaGetErrorString(e), what);
}

int sm_count() {
  static int cached[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (cached[dev] == 0) {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) n = 148;
    cached[dev] = n;
  }
  return cached[dev];
}

int current_device() {
  int dev = 0;
  return cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < 64 ? dev : -1;
}

// Two threads that meet here on a first call both do the work, with the same
// outcome.
int allow_smem(SmemOnce* done, const void* kernel, size_t bytes) {
  const int dev = current_device();
  if (dev >= 0 && __atomic_load_n(&done->set[dev], __ATOMIC_ACQUIRE)) return DS_OK;
  DS_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
  DS_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
  if (dev >= 0) __atomic_store_n(&done->set[dev], 1, __ATOMIC_RELEASE);
  return DS_OK;
}

int* symbol_address(SymbolOnce* known, const void* symbol) {
  const int dev = current_device();
  if (dev >= 0) {
    int* p = __atomic_load_n(&known->at[dev], __ATOMIC_ACQUIRE);
    if (p) return p;
  }
  void* p = nullptr;
  if (cudaGetSymbolAddress(&p, symbol) != cudaSuccess) return nullptr;
  if (dev >= 0) __atomic_store_n(&known->at[dev], static_cast<int*>(p), __ATOMIC_RELEASE);
  return static_cast<int*>(p);
}

namespace {
__global__ void take_word_kernel(int* word, int* out) { *out = atomicExch(word, 0); }
}  // namespace

int take_error_word(int* word, int32_t* err, cudaStream_t s) {
  int* got = nullptr;
  DS_CHECK_CUDA(cudaMallocAsync(reinterpret_cast<void**>(&got), sizeof(int), s));
  take_word_kernel<<<1, 1, 0, s>>>(word, got);
  cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) e = cudaMemcpyAsync(err, got, sizeof(int), cudaMemcpyDefault, s);
  const cudaError_t freed = cudaFreeAsync(got, s);
  return e != cudaSuccess ? cuda_status(e, "take_error_word") : freed != cudaSuccess ? cuda_status(freed, "take_error_word") : DS_OK;
}

}  // namespace ds

extern "C" const char* ds_last_error_string(void) { return g_last_error; }

extern "C" int ds_version(void) { return 100; }
