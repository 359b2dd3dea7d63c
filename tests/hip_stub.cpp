// A HIP runtime without a device, for tests of the library's host side on the CPU: device memory is
// host memory, work is done at once, launches are recorded and not run.  It stands in for the real
// one by its soname (the process that loads it must not have loaded that one).
//   stub_fail_at(k)   the k-th fallible call from now on fails (1: the next), 0: none
//   stub_calls()      fallible calls since the last stub_fail_at
//   stub_live()       allocations not freed yet
//   stub_launches()   launches recorded since stub_clear(); stub_launch(i) names one:
//                     "kernel<arguments> x y z threads"
//   stub_kernels()    kernels the library has; stub_kernel(i) names one
//   stub_error(e)     leaves e behind as the calling thread's last error
#include <cxxabi.h>
#include <hip/hip_runtime_api.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include <iterator>
#include <map>
#include <mutex>
#include <string>
#include <vector>

namespace {

std::mutex g_lock;
std::map<const void*, std::string> g_names;
std::vector<std::string> g_launches;
long g_fail_at = 0, g_calls = 0, g_live = 0;
thread_local hipError_t g_last = hipSuccess;
thread_local int g_device = 0;

hipError_t done(hipError_t e) {
  if (e != hipSuccess) g_last = e;
  return e;
}
// One fallible call: an error where its turn to fail has come.
hipError_t turn() {
  std::lock_guard<std::mutex> l(g_lock);
  return done(++g_calls == g_fail_at ? hipErrorOutOfMemory : hipSuccess);
}
hipError_t take(void** p, size_t bytes) {
  *p = nullptr;
  const hipError_t e = turn();
  if (e != hipSuccess) return e;
  if (!(*p = calloc(1, bytes ? bytes : 1))) return done(hipErrorOutOfMemory);
  std::lock_guard<std::mutex> l(g_lock);
  ++g_live;
  return hipSuccess;
}
hipError_t drop(void* p) {
  if (p) {
    free(p);
    std::lock_guard<std::mutex> l(g_lock);
    --g_live;
  }
  return hipSuccess;
}

}  // namespace

extern "C" {

void stub_fail_at(long k) {
  std::lock_guard<std::mutex> l(g_lock);
  g_fail_at = k;
  g_calls = 0;
}
long stub_calls() { return g_calls; }
long stub_live() { return g_live; }
void stub_error(int e) { g_last = (hipError_t)e; }
void stub_clear() {
  std::lock_guard<std::mutex> l(g_lock);
  g_launches.clear();
}
long stub_launches() { return (long)g_launches.size(); }
const char* stub_launch(long i) { return g_launches[i].c_str(); }
long stub_kernels() { return (long)g_names.size(); }
const char* stub_kernel(long i) { return std::next(g_names.begin(), i)->second.c_str(); }

void** __hipRegisterFatBinary(const void*) {
  static void* module;
  return &module;
}
void __hipUnregisterFatBinary(void**) {}
void __hipRegisterVar(void**, void*, char*, char*, int, size_t, int, int) {}
void __hipRegisterFunction(void**, const void* host, char*, const char* name, unsigned, void*, void*, void*, void*,
                           int*) {
  std::string mangled = name;  // (the demangler need not know the 16-bit types)
  for (const auto& t : {std::make_pair("DF16b", "8bfloat16"), std::make_pair("DF16_", "4half")})
    for (size_t i; (i = mangled.find(t.first)) != std::string::npos;) mangled.replace(i, 5, t.second);
  int bad = 0;
  char* plain = abi::__cxa_demangle(mangled.c_str(), nullptr, nullptr, &bad);
  std::string s = bad ? name : plain;
  free(plain);
  // without the result's type, the namespace and the parameters
  if (s.compare(0, 5, "void ") == 0) s.erase(0, 5);
  const std::string anonymous = "(anonymous namespace)::";
  if (s.compare(0, anonymous.size(), anonymous) == 0) s.erase(0, anonymous.size());
  for (size_t i = 0, depth = 0; i < s.size(); ++i) {
    depth += s[i] == '<' ? 1 : s[i] == '>' ? -1 : 0;
    if (s[i] == '(' && depth == 0) s.resize(i);
  }
  g_names[host] = s;
}

hipError_t __hipPushCallConfiguration(dim3, dim3, size_t, hipStream_t);
hipError_t __hipPopCallConfiguration(dim3*, dim3*, size_t*, hipStream_t*);
static thread_local struct {
  dim3 grid, block;
  size_t lds;
  hipStream_t stream;
} g_config;
hipError_t __hipPushCallConfiguration(dim3 grid, dim3 block, size_t lds, hipStream_t st) {
  g_config = {grid, block, lds, st};
  return hipSuccess;
}
hipError_t __hipPopCallConfiguration(dim3* grid, dim3* block, size_t* lds, hipStream_t* st) {
  *grid = g_config.grid;
  *block = g_config.block;
  *lds = g_config.lds;
  *st = g_config.stream;
  return hipSuccess;
}
hipError_t hipLaunchKernel(const void* f, dim3 grid, dim3 block, void**, size_t, hipStream_t) {
  // a launch counts its threads in 32 bits, and its workgroups down and behind in 16
  if ((unsigned long long)grid.x * block.x > 0xffffffffull || grid.y > 65535 || grid.z > 65535)
    return done(hipErrorInvalidConfiguration);
  char b[128];
  snprintf(b, sizeof b, " %u %u %u %u", grid.x, grid.y, grid.z, block.x * block.y * block.z);
  std::lock_guard<std::mutex> l(g_lock);
  g_launches.push_back(g_names[f] + b);
  return hipSuccess;
}

hipError_t hipGetLastError() {
  const hipError_t e = g_last;
  g_last = hipSuccess;
  return e;
}
const char* hipGetErrorString(hipError_t e) { return e == hipErrorOutOfMemory ? "out of memory" : "an error"; }
hipError_t hipGetDeviceCount(int* n) {
  *n = 2;
  return hipSuccess;
}
hipError_t hipGetDevice(int* d) {
  *d = g_device;
  return hipSuccess;
}
hipError_t hipSetDevice(int d) {
  if (d < 0 || d > 1) return done(hipErrorInvalidDevice);
  g_device = d;
  return hipSuccess;
}
hipError_t hipGetDevicePropertiesR0600(hipDeviceProp_t* p, int) {
  memset(p, 0, sizeof *p);
  strcpy(p->gcnArchName, "gfx950:sramecc+:xnack-");
  p->multiProcessorCount = 256;
  p->warpSize = 64;
  p->maxThreadsPerMultiProcessor = 2048;
  p->totalGlobalMem = (size_t)288 << 30;
  return hipSuccess;
}
hipError_t hipDeviceSynchronize() { return hipSuccess; }
hipError_t hipFuncSetAttribute(const void*, hipFuncAttribute, int) { return turn(); }
hipError_t hipOccupancyMaxActiveBlocksPerMultiprocessor(int* n, const void*, int, size_t) {
  *n = 1;
  return turn();
}
hipError_t hipGetSymbolAddress(void** p, const void*) {
  static char scratch[1 << 20];
  *p = scratch;
  return hipSuccess;
}

hipError_t hipMalloc(void** p, size_t bytes) { return take(p, bytes); }
hipError_t hipFree(void* p) { return drop(p); }
hipError_t hipHostMalloc(void** p, size_t bytes, unsigned) { return take(p, bytes); }
hipError_t hipHostFree(void* p) { return drop(p); }
hipError_t hipHostGetDevicePointer(void** dev, void* host, unsigned) {
  *dev = host;
  return turn();
}
hipError_t hipMemcpy(void* to, const void* from, size_t bytes, hipMemcpyKind) {
  memcpy(to, from, bytes);
  return hipSuccess;
}
hipError_t hipMemcpyAsync(void* to, const void* from, size_t bytes, hipMemcpyKind k, hipStream_t) {
  return hipMemcpy(to, from, bytes, k);
}
hipError_t hipMemcpy2D(void* to, size_t tp, const void* from, size_t fp, size_t w, size_t h, hipMemcpyKind) {
  for (size_t i = 0; i < h; ++i) memcpy((char*)to + i * tp, (const char*)from + i * fp, w);
  return hipSuccess;
}
hipError_t hipMemset(void* p, int v, size_t bytes) {
  // (fresh memory is zero, and large stretches of it stay untouched)
  if (v != 0 || bytes < (64u << 20)) memset(p, v, bytes);
  return hipSuccess;
}
hipError_t hipMemsetAsync(void* p, int v, size_t bytes, hipStream_t) {
  const hipError_t e = turn();
  return e == hipSuccess ? hipMemset(p, v, bytes) : e;
}
hipError_t hipMemset2DAsync(void* p, size_t pitch, int v, size_t w, size_t h, hipStream_t) {
  for (size_t i = 0; i < h; ++i) memset((char*)p + i * pitch, v, w);
  return hipSuccess;
}

static int g_handle;  // what events and streams point to
hipError_t hipStreamCreateWithFlags(hipStream_t* s, unsigned) {
  *s = (hipStream_t)&g_handle;
  return hipSuccess;
}
hipError_t hipStreamDestroy(hipStream_t) { return hipSuccess; }
hipError_t hipStreamSynchronize(hipStream_t) { return turn(); }
hipError_t hipStreamWaitEvent(hipStream_t, hipEvent_t, unsigned) { return hipSuccess; }
hipError_t hipEventCreate(hipEvent_t* e) {
  *e = (hipEvent_t)&g_handle;
  return hipSuccess;
}
hipError_t hipEventCreateWithFlags(hipEvent_t* e, unsigned) { return hipEventCreate(e); }
hipError_t hipEventDestroy(hipEvent_t) { return hipSuccess; }
hipError_t hipEventRecord(hipEvent_t, hipStream_t) { return hipSuccess; }
hipError_t hipEventSynchronize(hipEvent_t) { return hipSuccess; }
hipError_t hipEventElapsedTime(float* ms, hipEvent_t, hipEvent_t) {
  *ms = 1.f;
  return hipSuccess;
}

}  // extern "C"
