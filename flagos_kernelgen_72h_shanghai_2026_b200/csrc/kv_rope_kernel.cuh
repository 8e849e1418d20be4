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
// multiplied into two factors for each value, once for a token's queries and
// once for its keys: 123 instead of 181 instructions in all for a warp's two
// heads of 128, which had bound the kernel.
//
// 8192 tokens x 40 heads x 128, bf16: 34.0 us, 5.1 TB/s, 62 % of the issue
// slots. One warp per 16 heads and token, without the next step's loads in
// flight, took 38.3 us: the chain position, angles, values was waited for in
// every CTA (19 warps per SM active, most of them on loads). What is left is
// the same wait at a smaller scale.
#pragma once

#include "kv_common.cuh"

namespace kv {

constexpr int kRopeThreads = 256, kRopeWarps = kRopeThreads / 32;
constexpr int kRopeCtas = 2;    // CTAs per SM

struct RopeParams {
  Dense q, k, q_out, k_out;
  const void* q_gamma;
  const void* k_gamma;
  const float* cos_sin;
  const void* positions;
  int64_t max_pos;
  uint32_t steps, tokens;  // steps of all tokens, tokens
  FastDiv per_token, Q;    // steps of a token (queries first), tokens of a batch row
  uint32_t steps_q;        // steps of a token's queries
  uint32_t Hq, Hk;
  int32_t D, rot;
  int32_t gamma_dtype, pos_bytes;
  float eps, inv_d;
};

__device__ __forceinline__ void load_gamma8(const void* g, int i, int dtype, float f[8]) {
  if (dtype == DSA_KV_FP32) {
    const float4* p = reinterpret_cast<const float4*>(g) + 2 * i;
    const float4 a = p[0], b = p[1];
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  } else {
    const uint4 raw = reinterpret_cast<const uint4*>(g)[i];
    if (dtype == DSA_KV_BF16)
      unpack8<__nv_bfloat16>(raw, f);
    else
      unpack8<__half>(raw, f);
  }
}

// A step is U * 32 / LPH heads of one token. Every warp walks through a share
// of its own of all steps, queries of a token first, then its keys, and has the
// next step's values (and, where they change, its angles) on the way while it
// works on this one.
template <typename T, int LPH, int U, bool INTERLEAVED>
__global__ void __launch_bounds__(kRopeThreads, kRopeCtas) rope_kernel(const RopeParams p) {
  constexpr int HPW = 32 / LPH;
  constexpr int NA = INTERLEAVED ? 4 : 8;  // angles of a lane's values
  pdl_wait();
  const uint32_t warps = gridDim.x * kRopeWarps, warp = blockIdx.x * kRopeWarps + (threadIdx.x >> 5);
  uint32_t step = (uint32_t)((uint64_t)p.steps * warp / warps);
  const uint32_t last = (uint32_t)((uint64_t)p.steps * (warp + 1) / warps);
  if (step == last) return;
  const int lane = threadIdx.x & 31, i = lane % LPH, grp = lane / LPH;
  const bool active = 8 * i < p.D;
  const int hl = p.rot >> 4;  // lanes of the first half
  const bool rotated = 8 * i < p.rot;
  const int partner = INTERLEAVED || !rotated ? lane : i < hl ? lane + hl : lane - hl;

  uint32_t token, st, b, q;  // of the step whose values are loaded next
  p.per_token.divmod(step, &token, &st);
  p.Q.divmod(token, &b, &q);
  auto load_pos = [&](uint32_t t) -> int64_t {
    return t < p.tokens ? load_index(p.positions, t, p.pos_bytes) : -1;
  };
  int64_t pos = load_pos(token), pos1 = load_pos(token + 1);  // of this token and of the next one
  auto load = [&](uint4 (&raw)[U], bool wanted) {
    const bool is_k = st >= p.steps_q;
    const uint32_t h = (is_k ? st - p.steps_q : st) * (HPW * U) + grp, heads = is_k ? p.Hk : p.Hq;
    const Dense& in = is_k ? p.k : p.q;
    const uint8_t* src = in.row(b, q, h) + 16 * i;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      raw[u] = make_uint4(0, 0, 0, 0);
      if (wanted && active && h + u * HPW < heads) raw[u] = ld_stream(src + (int64_t)(u * HPW) * in.sh);
    }
  };
  float cs[NA], sn[NA];
  auto load_angles = [&](int64_t at) {
    if (!rotated || at < 0 || at >= p.max_pos) return;
    const float* row = p.cos_sin + at * p.rot + (INTERLEAVED ? 4 * i : 8 * (i < hl ? i : i - hl));
#pragma unroll
    for (int e = 0; e < NA; e += 4) {
      const float4 c = *reinterpret_cast<const float4*>(row + e);
      const float4 s = *reinterpret_cast<const float4*>(row + (p.rot >> 1) + e);
      cs[e] = c.x; cs[e + 1] = c.y; cs[e + 2] = c.z; cs[e + 3] = c.w;
      sn[e] = s.x; sn[e + 1] = s.y; sn[e + 2] = s.z; sn[e + 3] = s.w;
    }
  };
  // Factors of this lane's 8 values and of their partners:
  //   out = inv_rms * (A x + B x_partner)
  // first of a pair: A = gamma cos, B = -gamma_partner sin; second: +sin.
  f32x2 A[4], Bp[4];
  auto factors = [&](bool is_k, int64_t at) {
#pragma unroll
    for (int e = 0; e < 4; ++e) A[e] = Bp[e] = 0;
    if (!active) return;
    const void* gamma = is_k ? p.k_gamma : p.q_gamma;
    float ga[8];
    load_gamma8(gamma, i, p.gamma_dtype, ga);
    if (at >= p.max_pos) {  // no angles
#pragma unroll
      for (int e = 0; e < 4; ++e) A[e] = pair(__int_as_float(0x7fc00000), __int_as_float(0x7fc00000));
    } else if (!rotated) {
#pragma unroll
      for (int e = 0; e < 4; ++e) A[e] = pair(ga[2 * e], ga[2 * e + 1]);
    } else if constexpr (INTERLEAVED) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        A[e] = pair(ga[2 * e] * cs[e], ga[2 * e + 1] * cs[e]);
        Bp[e] = pair(-ga[2 * e + 1] * sn[e], ga[2 * e] * sn[e]);
      }
    } else {
      float gp[8];
      load_gamma8(gamma, partner % LPH, p.gamma_dtype, gp);
      const float sign = i < hl ? -1.f : 1.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        A[e] = pair(ga[2 * e] * cs[2 * e], ga[2 * e + 1] * cs[2 * e + 1]);
        Bp[e] = pair(gp[2 * e] * (sign * sn[2 * e]), gp[2 * e + 1] * (sign * sn[2 * e + 1]));
      }
    }
  };
  auto head = [&](const uint4& raw, uint8_t* dst, bool wanted) {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
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
    if (wanted) *reinterpret_cast<uint4*>(dst) = make_uint4(y[0], y[1], y[2], y[3]);
  };
  auto work = [&](const uint4 (&raw)[U], uint32_t wb, uint32_t wq, uint32_t wst) {
    const bool is_k = wst >= p.steps_q;
    const uint32_t h = (is_k ? wst - p.steps_q : wst) * (HPW * U), heads = is_k ? p.Hk : p.Hq;
    const Dense& out = is_k ? p.k_out : p.q_out;
    uint8_t* dst = out.row(wb, wq, h + grp) + 16 * i;
    // A step that is not full leaves its empty places out: at the first one, or
    // (adjacent pairs) on a path of its own. The other way round each is slower,
    // 41.9 for 36.4 us and 41.0 for 34.9 us (16384 tokens x 40 heads x 64).
    if (INTERLEAVED && h + HPW * U <= heads) {
#pragma unroll
      for (int u = 0; u < U; ++u) head(raw[u], dst + (int64_t)(u * HPW) * out.sh, active);
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (h + u * HPW >= heads) break;
        head(raw[u], dst + (int64_t)(u * HPW) * out.sh, active && h + grp + u * HPW < heads);
      }
    }
  };

  uint4 now[U], next[U];
  load(now, true);
  load_angles(pos);
  factors(st >= p.steps_q, pos);
  for (;;) {
    const uint32_t wb = b, wq = q, wst = st;
    const bool more = ++step < last;
    bool turn = false;  // to the next token
    if (more) {
      if (++st == p.per_token.d) {
        st = 0;
        turn = true;
        ++token;
        if (++q == p.Q.d) {
          q = 0;
          ++b;
        }
      }
      load(next, (turn ? pos1 : pos) >= 0);
      if (turn || st == p.steps_q) load_angles(turn ? pos1 : pos);
    }
    if (pos >= 0) work(now, wb, wq, wst);  // a padded token: its rows are left as they are
    if (!more) return;
    if (turn) {
      pos = pos1;
      pos1 = load_pos(token + 1);
    }
    if (turn || st == p.steps_q) factors(st >= p.steps_q, pos);
#pragma unroll
    for (int u = 0; u < U; ++u) now[u] = next[u];
  }
}

}  // namespace kv
