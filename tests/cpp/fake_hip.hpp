// A stand-in for the HIP runtime under the library's host code: a program that
// includes this defines the runtime's functions that libmolot_amd.so calls, so
// that its calls run without a GPU.  Kernels do not run: their launches are
// recorded in order, with the thread and the call (fake::call) that made them.
// Device memory is addresses that are never read.
#pragma once

#include <hip/hip_runtime.h>

#include <chrono>
#include <cstdint>
#include <cstdlib>
#include <cstring>
#include <map>
#include <mutex>
#include <string>
#include <thread>
#include <vector>

namespace fake {

struct Launch {
  std::string kernel;  // (mangled)
  dim3 grid, block;
  hipStream_t stream;
  int call;
};
struct State {
  std::mutex mu;
  std::map<const void*, std::string> names;
  std::vector<Launch> launches;
  std::vector<size_t> mallocs;   // sizes asked for and given
  std::vector<size_t> refused;
  size_t most = SIZE_MAX;        // allocations past it are refused,
  int left = INT32_MAX;          // and after so many more
  int live = 0;                  // allocations not freed
  uintptr_t next = 1ull << 40;
  bool capturing = false;
  int pause_us = 0;              // after every launch
};
inline State& state() {
  static State* s = new State;  // (the library registers its kernels before main)
  return *s;
}
inline thread_local int call = 0;
inline thread_local hipError_t last_error = hipSuccess;
inline void reset() {
  State& s = state();
  s.launches.clear();
  s.mallocs.clear();
  s.refused.clear();
}
inline hipError_t record(const void* fn, dim3 grid, dim3 block, hipStream_t stream) {
  State& s = state();
  int pause;
  {
    std::lock_guard<std::mutex> lk(s.mu);
    s.launches.push_back({s.names[fn], grid, block, stream, call});
    pause = s.pause_us;
  }
  if (pause) std::this_thread::sleep_for(std::chrono::microseconds(pause));
  return hipSuccess;
}
struct Config {
  dim3 grid, block;
  size_t lds;
  hipStream_t stream;
};
inline thread_local std::vector<Config> configs;

}  // namespace fake

extern "C" {

void** __hipRegisterFatBinary(const void*) {
  static void* handle = nullptr;
  return &handle;
}
void __hipUnregisterFatBinary(void**) {}
void __hipRegisterFunction(void**, const void* host, char*, const char* name, unsigned, void*, void*,
                           void*, void*, int*) {
  fake::state().names[host] = name;
}
void __hipRegisterVar(void**, void*, char*, char*, int, size_t, int, int) {}

hipError_t __hipPushCallConfiguration(dim3 grid, dim3 block, size_t lds, hipStream_t stream) {
  fake::configs.push_back({grid, block, lds, stream});
  return hipSuccess;
}
hipError_t __hipPopCallConfiguration(dim3* grid, dim3* block, size_t* lds, hipStream_t* stream) {
  const fake::Config c = fake::configs.back();
  fake::configs.pop_back();
  *grid = c.grid, *block = c.block, *lds = c.lds, *stream = c.stream;
  return hipSuccess;
}
hipError_t hipLaunchKernel(const void* fn, dim3 grid, dim3 block, void**, size_t, hipStream_t stream) {
  return fake::record(fn, grid, block, stream);
}
hipError_t hipExtLaunchKernel(const void* fn, dim3 grid, dim3 block, void**, size_t, hipStream_t stream,
                              hipEvent_t, hipEvent_t, int) {
  return fake::record(fn, grid, block, stream);
}
hipError_t hipMalloc(void** p, size_t bytes) {
  fake::State& s = fake::state();
  std::lock_guard<std::mutex> lk(s.mu);
  if (bytes > s.most || s.left <= 0) {
    s.refused.push_back(bytes);
    return fake::last_error = hipErrorOutOfMemory;
  }
  s.mallocs.push_back(bytes);
  --s.left;
  ++s.live;
  *p = reinterpret_cast<void*>(s.next);
  s.next += (bytes + 255) / 256 * 256;
  return hipSuccess;
}
hipError_t hipFree(void* p) {
  fake::State& s = fake::state();
  std::lock_guard<std::mutex> lk(s.mu);
  s.live -= p != nullptr;
  return hipSuccess;
}
// (what the classes of include/molot_amd use besides)
hipError_t hipMemset(void*, int, size_t) { return hipSuccess; }
hipError_t hipMemcpyAsync(void*, const void*, size_t, hipMemcpyKind, hipStream_t) { return hipSuccess; }
hipError_t hipHostMalloc(void** p, size_t bytes, unsigned) {
  *p = std::malloc(bytes);
  return hipSuccess;
}
hipError_t hipHostFree(void* p) {
  std::free(p);
  return hipSuccess;
}
hipError_t hipPointerGetAttributes(hipPointerAttribute_t* attr, const void*) {
  attr->type = hipMemoryTypeDevice;
  return hipSuccess;
}
hipError_t hipEventRecord(hipEvent_t, hipStream_t) { return hipSuccess; }
hipError_t hipGetLastError() {
  const hipError_t e = fake::last_error;
  fake::last_error = hipSuccess;
  return e;
}
const char* hipGetErrorString(hipError_t) { return "an error of the runtime"; }
hipError_t hipGetDevice(int* dev) {
  *dev = 0;
  return hipSuccess;
}
hipError_t hipDeviceGetAttribute(int* v, hipDeviceAttribute_t, int) {
  *v = 256;  // (asked for the CUs alone)
  return hipSuccess;
}
hipError_t hipStreamIsCapturing(hipStream_t, hipStreamCaptureStatus* st) {
  *st = fake::state().capturing ? hipStreamCaptureStatusActive : hipStreamCaptureStatusNone;
  return hipSuccess;
}
hipError_t hipStreamCreateWithFlags(hipStream_t* s, unsigned) {
  *s = nullptr;
  return hipSuccess;
}
hipError_t hipStreamDestroy(hipStream_t) { return hipSuccess; }
hipError_t hipStreamSynchronize(hipStream_t) { return hipSuccess; }
hipError_t hipMemcpyFromSymbolAsync(void* dst, const void*, size_t bytes, size_t, hipMemcpyKind,
                                    hipStream_t) {
  for (size_t i = 0; i < bytes / sizeof(int); ++i) static_cast<int*>(dst)[i] = (int)(i % 8);
  return hipSuccess;
}
hipError_t hipGetSymbolAddress(void** p, const void*) {
  *p = reinterpret_cast<void*>(1ull << 39);
  return hipSuccess;
}
hipError_t hipEventCreate(hipEvent_t* e) {
  *e = nullptr;
  return hipSuccess;
}
hipError_t hipEventDestroy(hipEvent_t) { return hipSuccess; }
hipError_t hipEventSynchronize(hipEvent_t) { return hipSuccess; }
hipError_t hipEventElapsedTime(float* ms, hipEvent_t, hipEvent_t) {
  *ms = 0.f;
  return hipSuccess;
}

}  // extern "C"
