// kv_host.h — host-side checks and launch shared by the sources of libdsa_kv.so.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

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

inline int check_cache(const dsa_kv_cache_t& c, bool written) {
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
    const int64_t least = written ? 1 : 0;
    if (c.k_stride[i] < least || c.v_stride[i] < least || c.k_scale_stride[i] < least ||
        c.v_scale_stride[i] < least)
      return DSA_KV_ERR_BAD_SHAPE;
  }
  return DSA_KV_OK;
}

// Launch in clusters of `cluster` CTAs, with programmatic stream serialisation:
// the kernel waits for the previous one (griddepcontrol.wait) before its first
// global access.
template <typename... A, typename... B>
int launch(void (*fn)(A...), int64_t grid, int threads, size_t smem, int cluster, void* stream, const B&... args) {
  if (grid > kMaxIndex) return DSA_KV_ERR_UNSUPPORTED;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, fn, args...) == cudaSuccess ? DSA_KV_OK : DSA_KV_ERR_CUDA;
}

}  // namespace kv
