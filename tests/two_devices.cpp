// A stand-in for the HIP runtime with two devices whose memory is the host's, for tests
// of host code without a GPU: it keeps the current device, gives out memory, copies it,
// launches nothing, and lists the device that was current at every allocation, launch
// and device synchronization.  Loaded (RTLD_GLOBAL) before libneedle_hip.so, whose calls
// it then answers.
#include <hip/hip_runtime_api.h>

#include <cstdlib>
#include <cstring>
#include <map>
#include <string>

namespace {
int current = 0;
std::string events;
std::map<const void*, void*> variables;
struct {
  dim3 grid, block;
  size_t shared;
  hipStream_t stream;
} launch;

void note(const char* what) { events += std::string(what) + ":" + std::to_string(current) + " "; }
}  // namespace

extern "C" {

const char* double_events() { return events.c_str(); }
void double_clear() { events.clear(); }

hipError_t hipGetDeviceCount(int* n) { return *n = 2, hipSuccess; }
hipError_t hipGetDevice(int* d) { return *d = current, hipSuccess; }
hipError_t hipSetDevice(int d) { return current = d, hipSuccess; }
hipError_t hipGetDevicePropertiesR0600(hipDeviceProp_tR0600* p, int) {
  std::memset(p, 0, sizeof *p);
  std::strcpy(p->gcnArchName, "gfx950");
  p->totalGlobalMem = (size_t)1 << 34;
  p->multiProcessorCount = 256;
  return hipSuccess;
}
hipError_t hipDeviceSynchronize() { return note("synchronize"), hipSuccess; }
hipError_t hipGetLastError() { return hipSuccess; }
const char* hipGetErrorString(hipError_t) { return "error"; }
hipError_t hipMemGetInfo(size_t* free, size_t* total) {
  return *free = *total = (size_t)1 << 34, hipSuccess;
}

hipError_t hipMalloc(void** p, size_t n) {
  note("allocate");
  *p = std::calloc(n, 1);
  return *p ? hipSuccess : hipErrorOutOfMemory;
}
hipError_t hipFree(void* p) { return std::free(p), hipSuccess; }
hipError_t hipHostMalloc(void** p, size_t n, unsigned) {
  *p = std::calloc(n, 1);
  return *p ? hipSuccess : hipErrorOutOfMemory;
}
hipError_t hipHostFree(void* p) { return std::free(p), hipSuccess; }
hipError_t hipMemcpy(void* to, const void* from, size_t n, hipMemcpyKind) {
  return std::memcpy(to, from, n), hipSuccess;
}
hipError_t hipMemcpyAsync(void* to, const void* from, size_t n, hipMemcpyKind, hipStream_t) {
  return std::memcpy(to, from, n), hipSuccess;
}
hipError_t hipMemcpy2DAsync(void* to, size_t tp, const void* from, size_t fp, size_t w, size_t h,
                            hipMemcpyKind, hipStream_t) {
  for (size_t i = 0; i < h; ++i) std::memcpy((char*)to + i * tp, (const char*)from + i * fp, w);
  return hipSuccess;
}
hipError_t hipMemset(void* p, int v, size_t n) { return std::memset(p, v, n), hipSuccess; }
hipError_t hipMemsetAsync(void* p, int v, size_t n, hipStream_t) {
  return std::memset(p, v, n), hipSuccess;
}
hipError_t hipMemsetD32Async(hipDeviceptr_t p, int v, size_t n, hipStream_t) {
  for (size_t i = 0; i < n; ++i) static_cast<int*>(p)[i] = v;
  return hipSuccess;
}

hipError_t hipStreamCreateWithFlags(hipStream_t* s, unsigned) {
  return *s = reinterpret_cast<hipStream_t>(std::malloc(1)), hipSuccess;
}
hipError_t hipStreamDestroy(hipStream_t s) { return std::free(s), hipSuccess; }
hipError_t hipStreamSynchronize(hipStream_t) { return hipSuccess; }

hipError_t hipLaunchKernel(const void*, dim3, dim3, void**, size_t, hipStream_t) {
  return note("launch"), hipSuccess;
}
hipError_t __hipPushCallConfiguration(dim3 grid, dim3 block, size_t shared, hipStream_t s) {
  return launch = {grid, block, shared, s}, hipSuccess;
}
hipError_t __hipPopCallConfiguration(dim3* grid, dim3* block, size_t* shared, hipStream_t* s) {
  *grid = launch.grid, *block = launch.block, *shared = launch.shared, *s = launch.stream;
  return hipSuccess;
}

void** __hipRegisterFatBinary(const void*) {
  static void* module;
  return &module;
}
void __hipUnregisterFatBinary(void**) {}
void __hipRegisterFunction(void**, const void*, char*, const char*, unsigned, void*, void*, void*,
                           void*, int*) {}
void __hipRegisterVar(void**, void* var, char*, char*, int, size_t size, int, int) {
  variables[var] = std::calloc(size, 1);
}
hipError_t hipGetSymbolAddress(void** p, const void* var) { return *p = variables[var], hipSuccess; }

}  // extern "C"
