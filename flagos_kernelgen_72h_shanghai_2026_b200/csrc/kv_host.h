// kv_host.h — host-side checks and launch shared by the sources of libdsa_kv.so.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <atomic>
#include <mutex>

#include "dsa_kv.h"
#include "kv_common.cuh"

namespace kv {

constexpr int64_t kMaxIndex = 0x7fffffff;  // 32-bit indices on the device

inline bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }
inline int index_size(int dt) { return dt == DSA_KV_INT32 ? 4 : dt == DSA_KV_INT64 ? 8 : 0; }
inline bool is_16bit(int dt) { return dt == DSA_KV_BF16 || dt == DSA_KV_FP16; }
inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// 0 <= a * b * c < 2^31 for sizes that are not negative.
inline bool fits(int64_t a, int64_t b, int64_t c) {
  if (a == 0 || b == 0 || c == 0) return true;
  if (a > kMaxIndex || b > kMaxIndex || c > kMaxIndex) return false;
  return (double)a * (double)b * (double)c <= (double)kMaxIndex;
}

// Strides of a dense tensor: a multiple of 8 elements wherever they are used,
// and rows of an output that do not lie on one another by a stride of 0.
inline int check_dense(const dsa_kv_dense_t& t, int64_t B, int64_t Q, int64_t H, bool output) {
  if (!t.ptr) return DSA_KV_ERR_NULL_POINTER;
  if (!aligned(t.ptr, 16)) return DSA_KV_ERR_ALIGNMENT;
  const int64_t n[3] = {B, Q, H}, s[3] = {t.stride_b, t.stride_q, t.stride_h};
  for (int i = 0; i < 3; ++i) {
    if (n[i] <= 1) continue;
    if (s[i] % 8 != 0) return DSA_KV_ERR_ALIGNMENT;
    if (s[i] < 0 || (output && s[i] == 0)) return DSA_KV_ERR_BAD_SHAPE;
  }
  return DSA_KV_OK;
}
inline Dense dense(const dsa_kv_dense_t& t) {
  Dense d;
  d.ptr = static_cast<uint8_t*>(t.ptr);
  d.sb = t.stride_b * 2;
  d.sq = t.stride_q * 2;
  d.sh = t.stride_h * 2;
  return d;
}

// Uses of a cache: scales (and, read by plain loads, codes) may be broadcast by
// strides of 0; what is written may not, and tensor maps take codes as they lie.
enum CacheUse { kCacheRead, kCacheWritten, kCacheMapped };
inline int check_cache(const dsa_kv_cache_t& c, CacheUse use) {
  if (c.reserved0 != 0) return DSA_KV_ERR_BAD_ARGS_SIZE;
  if (c.code_dtype != DSA_KV_INT8 && c.code_dtype != DSA_KV_E4M3) return DSA_KV_ERR_BAD_DTYPE;
  if (c.P < 0 || c.H < 1 || c.block_size < 1) return DSA_KV_ERR_BAD_SHAPE;
  if (c.D < 16 || c.D > 256 || c.D % 16 != 0) return DSA_KV_ERR_BAD_HEAD_DIM;
  if (c.P > kMaxIndex || c.H > kMaxIndex || c.block_size > kMaxIndex) return DSA_KV_ERR_UNSUPPORTED;
  if (c.P == 0) return DSA_KV_OK;  // no page is ever followed
  if (!c.k_codes || !c.v_codes || !c.k_scale || !c.v_scale) return DSA_KV_ERR_NULL_POINTER;
  if (!aligned(c.k_codes, 16) || !aligned(c.v_codes, 16) || !aligned(c.k_scale, 4) || !aligned(c.v_scale, 4))
    return DSA_KV_ERR_ALIGNMENT;
  const int64_t n[3] = {c.P, c.H, c.block_size};
  for (int i = 0; i < 3; ++i) {
    if (n[i] <= 1) continue;
    if (c.k_stride[i] % 16 != 0 || c.v_stride[i] % 16 != 0) return DSA_KV_ERR_ALIGNMENT;
    const int64_t least = use == kCacheRead ? 0 : 1, least_scale = use == kCacheWritten ? 1 : 0;
    if (c.k_stride[i] < least || c.v_stride[i] < least || c.k_scale_stride[i] < least_scale ||
        c.v_scale_stride[i] < least_scale)
      return DSA_KV_ERR_BAD_SHAPE;
    if (use == kCacheMapped && (c.k_stride[i] >= (int64_t)1 << 40 || c.v_stride[i] >= (int64_t)1 << 40))
      return DSA_KV_ERR_UNSUPPORTED;
  }
  return DSA_KV_OK;
}

// The current device, whose context is made the calling thread's: the driver's
// own entry points do not do that for a thread's first call.
inline bool bind_device(int* dev) {
  thread_local int bound = -1;
  if (cudaGetDevice(dev) != cudaSuccess) return false;
  if (bound != *dev) {
    if (cudaSetDevice(*dev) != cudaSuccess) return false;
    bound = *dev;
  }
  return true;
}

constexpr int kMaxDevices = 64;
inline bool sm_count(int dev, int* sms) {
  static std::atomic<int> known[kMaxDevices];
  if (dev < 0 || dev >= kMaxDevices) return false;
  *sms = known[dev].load(std::memory_order_relaxed);
  if (*sms > 0) return true;
  if (cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return false;
  known[dev].store(*sms, std::memory_order_relaxed);
  return true;
}

// A driver entry point, looked up once (the library does not link libcuda).
inline void* driver_entry(std::atomic<void*>* cached, const char* name) {
  void* f = cached->load(std::memory_order_acquire);
  if (f) return f;
  cudaDriverEntryPointQueryResult found;
  if (cudaGetDriverEntryPointByVersion(name, &f, 12000, cudaEnableDefault, &found) != cudaSuccess ||
      found != cudaDriverEntryPointSuccess)
    return nullptr;
  cached->store(f, std::memory_order_release);
  return f;
}

// The driver's handle of a kernel on a device: a table that is only ever added
// to. Launching by it skips the runtime's own look-up of the kernel on every
// call.
inline CUfunction kernel_handle(const void* fn, int dev) {
  constexpr int kSlots = 1024;
  struct Slot {
    std::atomic<const void*> fn;
    std::atomic<int> dev;
    std::atomic<CUfunction> handle;
  };
  static Slot table[kSlots];
  static std::mutex lock;
  const size_t at = ((reinterpret_cast<uintptr_t>(fn) >> 4) + (size_t)dev * 131) % kSlots;
  for (size_t i = at, n = 0; n < kSlots; ++n, i = (i + 1) % kSlots) {
    const void* have = table[i].fn.load(std::memory_order_acquire);
    if (!have) break;
    if (have == fn && table[i].dev.load(std::memory_order_relaxed) == dev)
      return table[i].handle.load(std::memory_order_relaxed);
  }
  cudaFunction_t f;
  if (cudaGetFuncBySymbol(&f, fn) != cudaSuccess) return nullptr;
  std::lock_guard<std::mutex> hold(lock);
  for (size_t i = at, n = 0; n < kSlots; ++n, i = (i + 1) % kSlots) {
    const void* have = table[i].fn.load(std::memory_order_relaxed);
    if (have == fn && table[i].dev.load(std::memory_order_relaxed) == dev) break;
    if (have) continue;
    table[i].dev.store(dev, std::memory_order_relaxed);
    table[i].handle.store(f, std::memory_order_relaxed);
    table[i].fn.store(fn, std::memory_order_release);
    break;
  }
  return f;
}

// Launch on the current device, in clusters of `cluster` CTAs, with
// programmatic stream serialisation: the kernel waits for the previous one
// (griddepcontrol.wait) before its first global access. Without it a rotation
// of one token took 4.1 instead of 3.4 us call after call, a write followed by a
// read 10.6 instead of 7.7 us.
template <typename... A>
int launch(void (*fn)(A...), int64_t grid, int threads, size_t smem, int cluster, void* stream, const A&... args) {
  if (grid > kMaxIndex) return DSA_KV_ERR_UNSUPPORTED;
  static std::atomic<void*> entry{nullptr};
  using LaunchFn = CUresult (*)(const CUlaunchConfig*, CUfunction, void**, void**);
  const LaunchFn launch_ex = reinterpret_cast<LaunchFn>(driver_entry(&entry, "cuLaunchKernelEx"));
  int dev;
  if (!launch_ex || !bind_device(&dev)) return DSA_KV_ERR_CUDA;
  const CUfunction f = kernel_handle(reinterpret_cast<const void*>(fn), dev);
  if (!f) return DSA_KV_ERR_CUDA;
  CUlaunchAttribute attr[2] = {};
  attr[0].id = CU_LAUNCH_ATTRIBUTE_PROGRAMMATIC_STREAM_SERIALIZATION;
  attr[0].value.programmaticStreamSerializationAllowed = 1;
  attr[1].id = CU_LAUNCH_ATTRIBUTE_CLUSTER_DIMENSION;
  attr[1].value.clusterDim.x = (unsigned)cluster;
  attr[1].value.clusterDim.y = 1;
  attr[1].value.clusterDim.z = 1;
  CUlaunchConfig cfg = {};
  cfg.gridDimX = (unsigned)grid;
  cfg.gridDimY = cfg.gridDimZ = 1;
  cfg.blockDimX = (unsigned)threads;
  cfg.blockDimY = cfg.blockDimZ = 1;
  cfg.sharedMemBytes = (unsigned)smem;
  cfg.hStream = static_cast<CUstream>(stream);
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  void* params[] = {const_cast<void*>(static_cast<const void*>(&args))...};
  return launch_ex(&cfg, f, params, nullptr) == CUDA_SUCCESS ? DSA_KV_OK : DSA_KV_ERR_CUDA;
}

}  // namespace kv
