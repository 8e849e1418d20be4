// kv_rope_kernel.cuh — per-head RMSNorm of queries and keys with the rotation
// by position (dsa_kv_rope_launch, include/dsa_kv.h).
//
// Per head x[D]:  y = x * rsqrt(mean(x^2) + eps) * gamma in fp32, then
// (a, b) -> (a cos - b sin, b cos + a sin) over the rotated pairs, rounded
// once to 16 bits. Bound by memory: every value is read and written once.
//
// LPH = 8, 16 or 32 lanes hold a head, 8 values (16 bytes) each, so a warp
// holds 32 / LPH heads at a time. The sum of squares is reduced by xor
// shuffles over those lanes. With pairs (i, i + rot/2) the partner of a lane's
// 8 values is another lane's 8 values, fetched as four packed words by
// shuffles before the norm; adjacent pairs lie within the lane.
#pragma once

#include "kv_common.cuh"

namespace kv {

struct RopeParams {
  Dense q, k, q_out, k_out;
  const void* q_gamma;
  const void* k_gamma;
  const float* cos_sin;
  const void* positions;
  int64_t max_pos;
  uint32_t tasks;         // tokens * strips
  FastDiv strips, Q;      // strips of heads per token (queries first), tokens per batch row
  uint32_t strips_q;
  uint32_t Hq, Hk;
  int32_t D, rot;
  int32_t gamma_dtype, pos_bytes;
  float eps, inv_d;
};

__device__ __forceinline__ void load_gamma8(const void* g, int i, int dtype, float f[8]) {
  if (dtype == DSA_KV_FP32) {
    const float4* p = reinterpret_cast<const float4*>(g) + 2 * i;
    const float4 a = __ldg(p), b = __ldg(p + 1);
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  } else {
    const uint4 raw = __ldg(reinterpret_cast<const uint4*>(g) + i);
    if (dtype == DSA_KV_BF16)
      unpack8<__nv_bfloat16>(raw, f);
    else
      unpack8<__half>(raw, f);
  }
}

// A warp takes a strip of U * 32 / LPH heads of one token: heads u * HPW + grp.
template <typename T, int LPH, int U, bool INTERLEAVED>
__global__ void __launch_bounds__(kCtaThreads) rope_kernel(const RopeParams p) {
  constexpr int HPW = 32 / LPH;
  pdl_wait();
  const uint32_t task = blockIdx.x * kCtaWarps + (threadIdx.x >> 5);
  if (task >= p.tasks) return;
  const int lane = threadIdx.x & 31, i = lane % LPH, grp = lane / LPH;
  uint32_t token, strip, b, q;
  p.strips.divmod(task, &token, &strip);
  p.Q.divmod(token, &b, &q);
  const bool is_k = strip >= p.strips_q;
  const uint32_t head0 = (is_k ? strip - p.strips_q : strip) * (HPW * U) + grp;
  const uint32_t heads = is_k ? p.Hk : p.Hq;
  const Dense& in = is_k ? p.k : p.q;
  const Dense& out = is_k ? p.k_out : p.q_out;
  const bool active = 8 * i < p.D;

  const uint8_t* src = in.row(b, q, head0) + 16 * i;
  uint4 raw[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    raw[u] = make_uint4(0, 0, 0, 0);
    if (active && head0 + u * HPW < heads) raw[u] = ld_stream(src + (int64_t)(u * HPW) * in.sh);
  }
  const int64_t pos = load_index(p.positions, token, p.pos_bytes);
  if (pos < 0) return;  // padding: the whole warp leaves
  const bool known = pos < p.max_pos;
  float gamma[8] = {};
  if (active) load_gamma8(is_k ? p.k_gamma : p.q_gamma, i, p.gamma_dtype, gamma);

  // Angles of this lane's values. Halves: 8 cosines and 8 sines, the sine
  // negated in the first half. Adjacent pairs: 4 of each.
  constexpr int NA = INTERLEAVED ? 4 : 8;
  float cs[NA], sn[NA];
  const int hl = p.rot >> 4;  // lanes of the first half
  const bool rotated = 8 * i < p.rot && known;
  const int partner = INTERLEAVED || !rotated ? lane : i < hl ? lane + hl : lane - hl;
  if (rotated) {
    const float* row = p.cos_sin + pos * p.rot + (INTERLEAVED ? 4 * i : 8 * (i < hl ? i : i - hl));
#pragma unroll
    for (int e = 0; e < NA; e += 4) {
      const float4 c = __ldg(reinterpret_cast<const float4*>(row + e));
      const float4 s = __ldg(reinterpret_cast<const float4*>(row + (p.rot >> 1) + e));
      cs[e] = c.x; cs[e + 1] = c.y; cs[e + 2] = c.z; cs[e + 3] = c.w;
      sn[e] = s.x; sn[e + 1] = s.y; sn[e + 2] = s.z; sn[e + 3] = s.w;
    }
    if (!INTERLEAVED && i < hl) {
#pragma unroll
      for (int e = 0; e < NA; ++e) sn[e] = -sn[e];
    }
  }
  // The partner's values are scaled by the partner's gamma.
  float gp[8];
  if (!INTERLEAVED) {
#pragma unroll
    for (int e = 0; e < 8; ++e) gp[e] = __shfl_sync(0xffffffffu, gamma[e], partner);
  }

  uint8_t* dst = out.row(b, q, head0) + 16 * i;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float y[8], ss = 0.f;
    unpack8<T>(raw[u], y);
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = fmaf(y[e], y[e], ss);
#pragma unroll
    for (int o = 1; o < LPH; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float inv = __frsqrt_rn(fmaf(ss, p.inv_d, p.eps));
    float z[8];
    if (!INTERLEAVED) {
      uint4 pr;
      pr.x = __shfl_sync(0xffffffffu, raw[u].x, partner);
      pr.y = __shfl_sync(0xffffffffu, raw[u].y, partner);
      pr.z = __shfl_sync(0xffffffffu, raw[u].z, partner);
      pr.w = __shfl_sync(0xffffffffu, raw[u].w, partner);
      unpack8<T>(pr, z);
    }
    if (!active || head0 + u * HPW >= heads) continue;
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = y[e] * inv * gamma[e];
    if (rotated) {
      if constexpr (INTERLEAVED) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float a = y[2 * e], c = y[2 * e + 1];
          y[2 * e] = a * cs[e] - c * sn[e];
          y[2 * e + 1] = c * cs[e] + a * sn[e];
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = y[e] * cs[e] + (z[e] * inv * gp[e]) * sn[e];
      }
    }
    if (!known) {
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = __int_as_float(0x7fc00000);
    }
    *reinterpret_cast<uint4*>(dst + (int64_t)(u * HPW) * out.sh) = pack8<T>(y);
  }
}

}  // namespace kv
