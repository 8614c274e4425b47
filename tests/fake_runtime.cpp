// The few calls of the CUDA runtime that kernel_room.cu reaches, for the CPU: a kernel's limit
// of dynamic shared memory, set by a first caller who stays in the call until `second_done`
// or two seconds have come.
#include <cuda_runtime_api.h>

#include <chrono>
#include <condition_variable>
#include <mutex>

constexpr int kOptIn = 232448, kFixed = 1024;
std::mutex m;
std::condition_variable changed;
int limit = 49152;
bool first_in = false, second_done = false;

extern "C" {
cudaError_t cudaFuncSetAttribute(const void*, cudaFuncAttribute which, int value) {
  if (which != cudaFuncAttributeMaxDynamicSharedMemorySize) return cudaSuccess;
  std::unique_lock<std::mutex> l(m);
  limit = value;
  if (!first_in) {                       // the first caller stays in here while another comes and goes
    first_in = true;
    changed.notify_all();
    changed.wait_for(l, std::chrono::seconds(2), [] { return second_done; });
  }
  return cudaSuccess;
}
cudaError_t cudaFuncGetAttributes(cudaFuncAttributes* a, const void*) {
  *a = cudaFuncAttributes{};
  a->sharedSizeBytes = kFixed;
  return cudaSuccess;
}
cudaError_t cudaDeviceGetAttribute(int* v, cudaDeviceAttr which, int) {
  *v = which == cudaDevAttrMaxSharedMemoryPerBlockOptin ? kOptIn : 148;
  return cudaSuccess;
}
cudaError_t cudaGetDevice(int* d) { *d = 0; return cudaSuccess; }
cudaError_t cudaSetDevice(int) { return cudaSuccess; }
const char* cudaGetErrorString(cudaError_t) { return ""; }
cudaError_t cudaOccupancyMaxActiveBlocksPerMultiprocessorWithFlags(int* n, const void*, int, size_t, unsigned) { *n = 1; return cudaSuccess; }
void** __cudaRegisterFatBinary(void*) { return nullptr; }
void __cudaRegisterFatBinaryEnd(void**) {}
void __cudaUnregisterFatBinary(void**) {}
char __cudaInitModule(void**) { return 1; }
}
