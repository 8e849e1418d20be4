// kv_copy_kernel.cuh — quantised write into, and dequantised read from, the
// paged cache (dsa_kv_write_launch, dsa_kv_read_launch, include/dsa_kv.h).
//
// Both move vectors of D values (a token's key or value of one head) and are
// bound by memory: 2D + (D + 4) bytes a vector. LPH = 8, 16 or 32 lanes hold
// a vector, 8 values each: 16 bytes on the dense side, 8 on the cache's. A
// warp takes 32 / LPH neighbouring vectors at a time, U times.
#pragma once

#include "kv_common.cuh"

namespace kv {

struct CopyParams {
  Dense k, v;
  CacheSide kc, vc;
  const void* page_table;
  const void* pos;        // q_pos [B, Q] (write), kv_lens [B] (read)
  int64_t P;
  uint32_t n;             // vectors: tokens * 2 * H
  FastDiv H2, H, Q, bs;   // 2 * heads, heads, tokens per batch row, block_size
  int64_t NB;
  int32_t D;
  int32_t page_bytes, pos_bytes;
};

template <typename T, int LPH, int U, bool E4M3>
__global__ void __launch_bounds__(kCtaThreads) write_kernel(const CopyParams p) {
  constexpr int VPW = 32 / LPH;
  pdl_wait();
  const int lane = threadIdx.x & 31, i = lane % LPH, grp = lane / LPH;
  const uint32_t n0 = (blockIdx.x * kCtaWarps + (threadIdx.x >> 5)) * (VPW * U) + grp;
  const bool active = 8 * i < p.D;
  uint4 raw[U];
  uint8_t* dst[U];
  float* sdst[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t n = n0 + u * VPW;
    raw[u] = make_uint4(0, 0, 0, 0);
    dst[u] = nullptr;
    if (n >= p.n) continue;
    uint32_t token, r, b, q;
    p.H2.divmod(n, &token, &r);
    p.Q.divmod(token, &b, &q);
    const bool is_v = r >= p.H.d;
    const uint32_t h = is_v ? r - p.H.d : r;
    if (active) raw[u] = ld_stream((is_v ? p.v : p.k).row(b, q, h) + 16 * i);
    const int64_t pos = load_index(p.pos, token, p.pos_bytes);
    if (pos < 0 || pos >= p.NB * (int64_t)p.bs.d) continue;
    const int64_t block = p.NB * (int64_t)p.bs.d <= 0x7fffffff ? (int64_t)p.bs.div((uint32_t)pos) : pos / p.bs.d;
    const int64_t page = load_index(p.page_table, b * p.NB + block, p.page_bytes);
    if (page < 0 || page >= p.P) continue;
    const int64_t off = pos - block * p.bs.d;
    const CacheSide& c = is_v ? p.vc : p.kc;
    dst[u] = c.codes + page * c.sp + h * c.sh + off * c.st + 8 * i;
    sdst[u] = c.scale + page * c.ssp + h * c.ssh + off * c.sst;
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    // The largest magnitude of 16-bit floats is the largest of their bits
    // without the sign; a NaN is above infinity, which is above the rest.
    const uint32_t a = __vmaxu2(__vmaxu2(raw[u].x & 0x7fff7fffu, raw[u].y & 0x7fff7fffu),
                                __vmaxu2(raw[u].z & 0x7fff7fffu, raw[u].w & 0x7fff7fffu));
    uint32_t m = max(a & 0xffffu, a >> 16);
#pragma unroll
    for (int o = 1; o < LPH; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (!dst[u]) continue;
    const float amax = Half16<T>::unpack(m).x;
    float scale = fmaxf(__fdiv_rn(amax, E4M3 ? 448.0f : 127.0f), kMinScale);
    float f[8];
    unpack8<T>(raw[u], f);
    const float inv = __frcp_rn(scale);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = __fmul_rn(f[e], inv);
    uint2 codes;
    codes.x = E4M3 ? to_e4m3x4(f[0], f[1], f[2], f[3]) : to_s8x4(f[0], f[1], f[2], f[3]);
    codes.y = E4M3 ? to_e4m3x4(f[4], f[5], f[6], f[7]) : to_s8x4(f[4], f[5], f[6], f[7]);
    if (m >= Half16<T>::kInf) {
      scale = __int_as_float(0x7fc00000);
      codes = make_uint2(0, 0);
    }
    if (active) *reinterpret_cast<uint2*>(dst[u]) = codes;
    if (i == 0) *sdst[u] = scale;
  }
}

template <typename T, int LPH, int U, bool E4M3>
__global__ void __launch_bounds__(kCtaThreads) read_kernel(const CopyParams p) {
  constexpr int VPW = 32 / LPH;
  pdl_wait();
  const int lane = threadIdx.x & 31, i = lane % LPH, grp = lane / LPH;
  const uint32_t n0 = (blockIdx.x * kCtaWarps + (threadIdx.x >> 5)) * (VPW * U) + grp;
  const bool active = 8 * i < p.D;
  uint2 codes[U];
  float scale[U];
  uint8_t* dst[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t n = n0 + u * VPW;
    codes[u] = make_uint2(0, 0);
    scale[u] = 0.f;
    dst[u] = nullptr;
    if (n >= p.n || !active) continue;
    uint32_t token, r, b, s;
    p.H2.divmod(n, &token, &r);
    p.Q.divmod(token, &b, &s);
    int64_t len = load_index(p.pos, b, p.pos_bytes);
    const uint32_t block = p.bs.div(s);
    if (s >= len || block >= p.NB) continue;
    const bool is_v = r >= p.H.d;
    const uint32_t h = is_v ? r - p.H.d : r;
    dst[u] = (is_v ? p.v : p.k).row(b, s, h) + 16 * i;
    const int64_t page = load_index(p.page_table, b * p.NB + block, p.page_bytes);
    if (page < 0 || page >= p.P) continue;
    const uint32_t off = s - block * p.bs.d;
    const CacheSide& c = is_v ? p.vc : p.kc;
    codes[u] = ld_stream8(c.codes + page * c.sp + h * c.sh + off * c.st + 8 * i);
    scale[u] = __ldg(c.scale + page * c.ssp + h * c.ssh + off * c.sst);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (!dst[u]) continue;
    float f[8];
    decode4<E4M3>(codes[u].x, f);
    decode4<E4M3>(codes[u].y, f + 4);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = f[e] * scale[u];
    *reinterpret_cast<uint4*>(dst[u]) = pack8<T>(f);
  }
}

}  // namespace kv
