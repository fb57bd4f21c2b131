// What the C entry points of every source file need to check arguments and to launch kernels.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <stdio.h>

#include <atomic>

#include "../../include/xfc_mi355x.h"

namespace {

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int check_launch() {
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) {
    fprintf(stderr, "xfc: kernel launch failed: %s\n", hipGetErrorString(e));
    return XFC_ERR_HIP;
  }
  return XFC_OK;
}

constexpr int MAX_DEVICES = 64;
int current_device() {
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= MAX_DEVICES) dev = 0;
  return dev;
}

constexpr int FULL_LDS = 160 * 1024;

// Dynamic LDS above the default limit needs the attribute once per kernel and device.
template <auto Kernel>
hipError_t raise_lds_limit(int lds) {
  static std::atomic<bool> raised[MAX_DEVICES];
  const int dev = current_device();
  if (lds <= 48 * 1024 || raised[dev].load(std::memory_order_acquire)) return hipSuccess;
  hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(Kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  if (e == hipSuccess) raised[dev].store(true, std::memory_order_release);
  return e;
}

// Launches Kernel and returns XFC_OK or XFC_ERR_HIP; nothing is launched when the LDS limit cannot be raised.
template <auto Kernel, class A>
int launch_k(dim3 g, dim3 b, int lds, hipStream_t st, const A& args) {
  const hipError_t e = raise_lds_limit<Kernel>(lds);
  if (e != hipSuccess) {
    fprintf(stderr, "xfc: cannot raise the dynamic LDS limit to %d bytes: %s\n", lds, hipGetErrorString(e));
    return XFC_ERR_HIP;
  }
  hipLaunchKernelGGL(Kernel, g, b, lds, st, args);
  return check_launch();
}

int num_cus() {
  static std::atomic<int> n[MAX_DEVICES];
  const int dev = current_device();
  int v = n[dev].load(std::memory_order_relaxed);
  if (v == 0) {
    int cnt = 0;
    if (hipDeviceGetAttribute(&cnt, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cnt <= 0) cnt = 256;
    v = cnt;
    n[dev].store(v, std::memory_order_relaxed);
  }
  return v;
}

bool dims_ok(int64_t v) { return v >= 0 && v <= 0x7fffffff; }

}  // namespace
