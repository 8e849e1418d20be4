// kv_copy_kernel.cuh — quantised write into, and dequantised read from, the
// paged cache (dsa_kv_write_launch, dsa_kv_read_launch, include/dsa_kv.h).
//
// Both move vectors of D values (a token's key or value of one head) and are
// bound by memory: 2D + (D + 4) bytes a vector. LPH = 8, 16 or 32 lanes hold
// a vector, 8 values each: 16 bytes on the dense side, 8 on the cache's.
//
// A warp takes tpw tokens (one, unless the heads do not fill it) and, of both
// keys and values, U steps of hps heads. Position, page and addresses are
// worked out once for the 2U vectors that a lane then moves: with one vector
// per look-up the kernels were bound by that arithmetic (170 instructions for
// two vectors of a read, 75 % of the issue slots at 3.8 TB/s). Read of 8 x up to
// 8192 tokens x 8 heads x 128 (e4m3 to bf16): 52.8 us, 6.0 TB/s; write of
// 2 x 4096 tokens: 11.0 us, 4.2 TB/s.
#pragma once

#include "kv_common.cuh"

namespace kv {

// Four warps to a CTA: eight took 2.6 instead of 2.2 us for 64 tokens, 7.7
// instead of 7.0 us for a chunk of 4 x 512 written and 4 x 4000 tokens read, and
// as long for large calls; two are slower there.
constexpr int kCopyThreads = 128;

struct CopyParams {
  Dense k, v;
  CacheSide kc, vc;
  const void* page_table;
  const void* pos;        // q_pos [B, Q] (write), kv_lens [B] (read)
  int64_t P;
  uint32_t tasks;         // warps with work
  uint32_t tokens;        // B * Q
  uint32_t H, log_hps, log_tpw;  // heads; log2 of heads per step and of tokens per warp
  FastDiv strips, Q, bs;  // strips of U * hps heads, tokens per batch row, block_size
  int64_t NB;
  int32_t D;
  int32_t page_bytes, pos_bytes;
};

// A lane's place: token, first head, step of heads; false where it has none.
struct Place {
  uint32_t token, b, q, h;
};
template <int LPH, int U>
__device__ __forceinline__ bool place(const CopyParams& p, int lane, Place* w) {
  const uint32_t task = blockIdx.x * (kCopyThreads / 32) + (threadIdx.x >> 5), grp = lane / LPH;
  uint32_t t, strip;
  p.strips.divmod(task, &t, &strip);
  w->token = (t << p.log_tpw) + (grp >> p.log_hps);
  w->h = ((strip * U) << p.log_hps) + (grp & ((1u << p.log_hps) - 1));
  p.Q.divmod(w->token, &w->b, &w->q);
  return task < p.tasks && w->token < p.tokens;
}

template <typename T, int LPH, int U, bool E4M3>
__global__ void __launch_bounds__(kCopyThreads) write_kernel(const CopyParams p) {
  constexpr int NV = 2 * U;  // vectors of a lane: U keys, then U values
  pdl_wait();
  const int lane = threadIdx.x & 31, i = lane % LPH;
  Place w;
  const bool in = place<LPH, U>(p, lane, &w);
  const bool active = in && 8 * i < p.D;
  const uint32_t hps = 1u << p.log_hps;
  uint4 raw[NV];
  int64_t pos = -1;
  {
    const uint8_t* ks = p.k.row(w.b, w.q, w.h) + 16 * i;
    const uint8_t* vs = p.v.row(w.b, w.q, w.h) + 16 * i;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      raw[u] = raw[U + u] = make_uint4(0, 0, 0, 0);
      if (active && w.h + u * hps < p.H) {
        raw[u] = ld_stream(ks + (int64_t)(u * hps) * p.k.sh);
        raw[U + u] = ld_stream(vs + (int64_t)(u * hps) * p.v.sh);
      }
    }
  }
  if (in) pos = load_index(p.pos, w.token, p.pos_bytes);
  const int64_t cap = p.NB * (int64_t)p.bs.d;
  int64_t page = -1, off = 0;
  if (pos >= 0 && pos < cap) {
    const int64_t block = cap <= 0x7fffffff ? (int64_t)p.bs.div((uint32_t)pos) : pos / p.bs.d;
    off = pos - block * p.bs.d;
    page = load_index(p.page_table, w.b * p.NB + block, p.page_bytes);
  }
  const bool cell = page >= 0 && page < p.P;  // the same for all lanes of a vector

  // Largest magnitude of every vector. That of 16-bit floats is the largest of
  // their bits without the sign; a NaN is above infinity, which is above the rest.
  uint32_t mine = 0;
#pragma unroll
  for (int n = 0; n < NV; ++n) {
    const uint32_t a = __vmaxu2(__vmaxu2(raw[n].x & 0x7fff7fffu, raw[n].y & 0x7fff7fffu),
                                __vmaxu2(raw[n].z & 0x7fff7fffu, raw[n].w & 0x7fff7fffu));
    uint32_t m = max(a & 0xffffu, a >> 16);
#pragma unroll
    for (int o = 1; o < LPH; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (i % NV == n) mine = m;
  }
  // Lane n of the group takes vector n's scale: two IEEE divisions for NV vectors.
  const float amax = Half16<T>::unpack(mine).x;
  float scale = fmaxf(__fdiv_rn(amax, E4M3 ? 448.0f : 127.0f), kMinScale);
  float inv = __frcp_rn(scale);
  if (mine >= Half16<T>::kInf) {
    scale = __int_as_float(0x7fc00000);
    inv = 0.f;  // marks codes 0 (no finite vector has it: 3.39e38 / 127 < 2.7e36, whose inverse is a normal number)
  }
  if (cell && i < NV && w.h + (i % U) * hps < p.H) {
    const CacheSide& c = i < U ? p.kc : p.vc;
    c.scale[page * c.ssp + (w.h + (i % U) * hps) * c.ssh + off * c.sst] = scale;
  }
  uint8_t* const kd = p.kc.codes + page * p.kc.sp + w.h * p.kc.sh + off * p.kc.st + 8 * i;
  uint8_t* const vd = p.vc.codes + page * p.vc.sp + w.h * p.vc.sh + off * p.vc.st + 8 * i;
#pragma unroll
  for (int n = 0; n < NV; ++n) {
    const float f = __shfl_sync(0xffffffffu, inv, (lane & ~(LPH - 1)) + n);
    const f32x2 f2 = pair(f, f);
    const uint32_t x[4] = {raw[n].x, raw[n].y, raw[n].z, raw[n].w};
    float2 y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 t = Half16<T>::unpack(x[e]);
      y[e] = both(mul2(pair(t.x, t.y), f2));
    }
    uint2 codes;
    codes.x = E4M3 ? to_e4m3x4(y[0].x, y[0].y, y[1].x, y[1].y) : to_s8x4(y[0].x, y[0].y, y[1].x, y[1].y);
    codes.y = E4M3 ? to_e4m3x4(y[2].x, y[2].y, y[3].x, y[3].y) : to_s8x4(y[2].x, y[2].y, y[3].x, y[3].y);
    if (f == 0.f) codes = make_uint2(0, 0);
    const int u = n % U;
    if (active && cell && w.h + u * hps < p.H)
      *reinterpret_cast<uint2*>((n < U ? kd : vd) + (int64_t)(u * hps) * (n < U ? p.kc.sh : p.vc.sh)) = codes;
  }
}

template <typename T, int LPH, int U, bool E4M3>
__global__ void __launch_bounds__(kCopyThreads) read_kernel(const CopyParams p) {
  constexpr int NV = 2 * U;
  pdl_wait();
  const int lane = threadIdx.x & 31, i = lane % LPH;
  Place w;
  if (!place<LPH, U>(p, lane, &w) || 8 * i >= p.D) return;  // no lane needs another one's help
  const int64_t len = load_index(p.pos, w.b, p.pos_bytes);
  const uint32_t block = p.bs.div(w.q), off = w.q - block * p.bs.d;
  if (w.q >= len || block >= p.NB) return;
  const int64_t page = load_index(p.page_table, w.b * p.NB + block, p.page_bytes);
  const bool cell = page >= 0 && page < p.P;
  const uint32_t hps = 1u << p.log_hps;
  uint2 codes[NV];
  float scale[NV];
  {
    const uint8_t* ks = p.kc.codes + page * p.kc.sp + w.h * p.kc.sh + off * p.kc.st + 8 * i;
    const uint8_t* vs = p.vc.codes + page * p.vc.sp + w.h * p.vc.sh + off * p.vc.st + 8 * i;
    const float* kf = p.kc.scale + page * p.kc.ssp + w.h * p.kc.ssh + off * p.kc.sst;
    const float* vf = p.vc.scale + page * p.vc.ssp + w.h * p.vc.ssh + off * p.vc.sst;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      codes[u] = codes[U + u] = make_uint2(0, 0);
      scale[u] = scale[U + u] = 0.f;
      if (cell && w.h + u * hps < p.H) {
        codes[u] = ld_stream8(ks + (int64_t)(u * hps) * p.kc.sh);
        codes[U + u] = ld_stream8(vs + (int64_t)(u * hps) * p.vc.sh);
        scale[u] = kf[(int64_t)(u * hps) * p.kc.ssh];
        scale[U + u] = vf[(int64_t)(u * hps) * p.vc.ssh];
      }
    }
  }
  uint8_t* const kd = p.k.row(w.b, w.q, w.h) + 16 * i;
  uint8_t* const vd = p.v.row(w.b, w.q, w.h) + 16 * i;
#pragma unroll
  for (int n = 0; n < NV; ++n) {
    f32x2 f[4];
    decode4<E4M3>(codes[n].x, f[0], f[1]);
    decode4<E4M3>(codes[n].y, f[2], f[3]);
    const f32x2 s2 = pair(scale[n], scale[n]);
    uint32_t y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 t = both(mul2(f[e], s2));
      y[e] = Half16<T>::pack(t.x, t.y);
    }
    const int u = n % U;
    if (w.h + u * hps < p.H)
      *reinterpret_cast<uint4*>((n < U ? kd : vd) + (int64_t)(u * hps) * (n < U ? p.k.sh : p.v.sh)) =
          make_uint4(y[0], y[1], y[2], y[3]);
  }
}

}  // namespace kv
