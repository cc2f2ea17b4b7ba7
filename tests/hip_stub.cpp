// A device runtime on the host: two devices, memory that is the host's, kernels
// that are counted and not run. What the library's host side asks for and
// refuses is tested with it where there is no GPU.
#include <hip/hip_runtime_api.h>

#include <cstdlib>
#include <cstring>
#include <map>
#include <string>

namespace {
constexpr int kDevices = 2;
int current = 0;
std::map<void*, int> owner;  // device of each allocation and stream
std::map<std::string, long> launches;
}  // namespace

extern "C" {

int stub_device_of(void* p) { return owner.count(p) ? owner[p] : -1; }
void stub_set_device(int device) { current = device; }
int stub_device() { return current; }
long stub_launches(const char* name) { return launches[name]; }

hipError_t hipGetDeviceCount(int* n) { return *n = kDevices, hipSuccess; }
hipError_t hipGetDevice(int* d) { return *d = current, hipSuccess; }
hipError_t hipSetDevice(int d) {
  if (d < 0 || d >= kDevices) return hipErrorInvalidDevice;
  return current = d, hipSuccess;
}
hipError_t hipGetDeviceProperties(hipDeviceProp_t* p, int) {
  memset(p, 0, sizeof(*p));
  strcpy(p->name, "stub");
  strcpy(p->gcnArchName, "gfx950");
  p->multiProcessorCount = 256;
  return hipSuccess;
}
hipError_t hipGetLastError() { return hipSuccess; }
const char* hipGetErrorString(hipError_t) { return "stub"; }
const char* hipGetErrorName(hipError_t) { return "stub"; }

hipError_t hipMalloc(void** p, size_t n) {
  if (posix_memalign(p, 4096, n ? n : 1) != 0) return hipErrorOutOfMemory;
  memset(*p, 0, n);
  owner[*p] = current;
  return hipSuccess;
}
hipError_t hipFree(void* p) {
  owner.erase(p);
  free(p);
  return hipSuccess;
}
hipError_t hipMemcpy(void* to, const void* from, size_t n, hipMemcpyKind) {
  memmove(to, from, n);
  return hipSuccess;
}
hipError_t hipMemcpyAsync(void* to, const void* from, size_t n, hipMemcpyKind k, hipStream_t) {
  return hipMemcpy(to, from, n, k);
}
hipError_t hipMemset(void* p, int v, size_t n) {
  memset(p, v, n);
  return hipSuccess;
}
hipError_t hipMemsetAsync(void* p, int v, size_t n, hipStream_t) { return hipMemset(p, v, n); }
hipError_t hipGetSymbolAddress(void** p, const void*) { return hipMalloc(p, 64); }

hipError_t hipStreamCreateWithFlags(hipStream_t* s, unsigned) {
  return hipMalloc(reinterpret_cast<void**>(s), 1);
}
hipError_t hipStreamDestroy(hipStream_t s) { return hipFree(s); }
hipError_t hipStreamSynchronize(hipStream_t) { return hipSuccess; }
hipError_t hipStreamIsCapturing(hipStream_t, hipStreamCaptureStatus* s) {
  return *s = hipStreamCaptureStatusNone, hipSuccess;
}
hipError_t hipStreamWaitEvent(hipStream_t, hipEvent_t, unsigned) { return hipSuccess; }
hipError_t hipEventCreate(hipEvent_t* e) { return hipMalloc(reinterpret_cast<void**>(e), 1); }
hipError_t hipEventCreateWithFlags(hipEvent_t* e, unsigned) { return hipEventCreate(e); }
hipError_t hipEventDestroy(hipEvent_t e) { return hipFree(e); }
hipError_t hipEventRecord(hipEvent_t, hipStream_t) { return hipSuccess; }

hipError_t hipModuleLoadData(hipModule_t* m, const void*) {
  return hipMalloc(reinterpret_cast<void**>(m), 1);
}
hipError_t hipModuleUnload(hipModule_t m) { return hipFree(m); }
hipError_t hipModuleGetFunction(hipFunction_t* f, hipModule_t, const char* name) {
  return *f = reinterpret_cast<hipFunction_t>(strdup(name)), hipSuccess;
}
hipError_t hipModuleLaunchKernel(hipFunction_t f, unsigned, unsigned, unsigned, unsigned, unsigned,
                                 unsigned, unsigned, hipStream_t s, void**, void**) {
  if (owner[s] != current) return hipErrorInvalidResourceHandle;
  ++launches[reinterpret_cast<const char*>(f)];
  return hipSuccess;
}

}  // extern "C"
