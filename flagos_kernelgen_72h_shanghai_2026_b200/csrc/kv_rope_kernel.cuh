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
// shuffles; adjacent pairs lie within the lane. Gamma, cosine and sine are
// multiplied once per task into two factors for each value: 75 instead of 180
// instructions for a warp's two heads of 128, which had bound the kernel (62 %
// of the issue slots). 8192 tokens x 40 heads x 128, bf16: 38.3 us, 4.5 TB/s.
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
  uint32_t strips_q, strip;  // strips of queries; heads of a strip
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

// A warp takes a strip of heads of one token, U * 32 / LPH at a time.
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
  const uint32_t head0 = (is_k ? strip - p.strips_q : strip) * p.strip;
  const uint32_t end = min(is_k ? p.Hk : p.Hq, head0 + p.strip);
  const Dense& in = is_k ? p.k : p.q;
  const Dense& out = is_k ? p.k_out : p.q_out;
  const bool active = 8 * i < p.D;
  const int64_t pos = load_index(p.positions, token, p.pos_bytes);

  uint4 raw[U];
  auto load = [&](uint32_t h) {
    const uint8_t* src = in.row(b, q, h) + 16 * i;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      raw[u] = make_uint4(0, 0, 0, 0);
      if (active && h + u * HPW < end) raw[u] = ld_stream(src + (int64_t)(u * HPW) * in.sh);
    }
  };
  load(head0 + grp);
  if (pos < 0) return;  // padding: the whole warp leaves

  // Factors of this lane's 8 values and of their partners:
  //   out = inv_rms * (A x + B x_partner)
  // first of a pair: A = gamma cos, B = -gamma_partner sin; second: +sin.
  const int hl = p.rot >> 4;  // lanes of the first half
  const bool rotated = 8 * i < p.rot;
  const int partner = INTERLEAVED || !rotated ? lane : i < hl ? lane + hl : lane - hl;
  f32x2 A[4], Bp[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) A[e] = Bp[e] = 0;
  if (active) {
    const void* gamma = is_k ? p.k_gamma : p.q_gamma;
    float ga[8];
    load_gamma8(gamma, i, p.gamma_dtype, ga);
    if (pos >= p.max_pos) {  // no angles
#pragma unroll
      for (int e = 0; e < 4; ++e) A[e] = pair(__int_as_float(0x7fc00000), __int_as_float(0x7fc00000));
    } else if (!rotated) {
#pragma unroll
      for (int e = 0; e < 4; ++e) A[e] = pair(ga[2 * e], ga[2 * e + 1]);
    } else if constexpr (INTERLEAVED) {
      const float* row = p.cos_sin + pos * p.rot + 4 * i;
      const float4 c = __ldg(reinterpret_cast<const float4*>(row));
      const float4 s = __ldg(reinterpret_cast<const float4*>(row + (p.rot >> 1)));
      const float cs[4] = {c.x, c.y, c.z, c.w}, sn[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        A[e] = pair(ga[2 * e] * cs[e], ga[2 * e + 1] * cs[e]);
        Bp[e] = pair(-ga[2 * e + 1] * sn[e], ga[2 * e] * sn[e]);
      }
    } else {
      float gp[8];
      load_gamma8(gamma, partner % LPH, p.gamma_dtype, gp);
      const float* row = p.cos_sin + pos * p.rot + 8 * (i < hl ? i : i - hl);
      const float sign = i < hl ? -1.f : 1.f;
#pragma unroll
      for (int e = 0; e < 4; e += 2) {
        const float4 c = __ldg(reinterpret_cast<const float4*>(row + 2 * e));
        const float4 s = __ldg(reinterpret_cast<const float4*>(row + (p.rot >> 1) + 2 * e));
        A[e] = pair(ga[2 * e] * c.x, ga[2 * e + 1] * c.y);
        A[e + 1] = pair(ga[2 * e + 2] * c.z, ga[2 * e + 3] * c.w);
        Bp[e] = pair(gp[2 * e] * (sign * s.x), gp[2 * e + 1] * (sign * s.y));
        Bp[e + 1] = pair(gp[2 * e + 2] * (sign * s.z), gp[2 * e + 3] * (sign * s.w));
      }
    }
  }

  for (uint32_t h = head0 + grp;;) {
    uint8_t* dst = out.row(b, q, h) + 16 * i;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t w[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
      f32x2 x[4], ss = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 t = Half16<T>::unpack(w[e]);
        x[e] = pair(t.x, t.y);
        ss = fma2(x[e], x[e], ss);
      }
      const float2 s2 = both(ss);
      float sum = s2.x + s2.y;
#pragma unroll
      for (int o = 1; o < LPH; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      const float inv = rsqrtf(fmaf(sum, p.inv_d, p.eps));
      const f32x2 inv2 = pair(inv, inv);
      uint32_t y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float2 t;
        if (INTERLEAVED) {
          t = both(x[e]);
          t = make_float2(t.y, t.x);
        } else {
          t = Half16<T>::unpack(__shfl_sync(0xffffffffu, w[e], partner));
        }
        t = both(mul2(inv2, fma2(Bp[e], pair(t.x, t.y), mul2(A[e], x[e]))));
        y[e] = Half16<T>::pack(t.x, t.y);
      }
      if (active && h + u * HPW < end)
        *reinterpret_cast<uint4*>(dst + (int64_t)(u * HPW) * out.sh) = make_uint4(y[0], y[1], y[2], y[3]);
    }
    h += U * HPW;
    if (h - grp >= end) break;
    load(h);
  }
}

}  // namespace kv
