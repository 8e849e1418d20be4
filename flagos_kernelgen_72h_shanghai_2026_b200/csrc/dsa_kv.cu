// dsa_kv.cu — host side of libdsa_kv.so (C ABI: include/dsa_kv.h): argument
// validation and launch planning of the rotation and of the cache's write and
// read. Device code: kv_rope_kernel.cuh, kv_copy_kernel.cuh. The attention's
// host side is dsa_kv_attn.cu.
#include <cuda_runtime.h>
#include <stdint.h>

#include "dsa_kv.h"
#include "kv_copy_kernel.cuh"
#include "kv_host.h"
#include "kv_rope_kernel.cuh"

namespace kv {

CacheSide side(void* codes, float* scale, const int64_t s[3], const int64_t ss[3]) {
  CacheSide c;
  c.codes = static_cast<uint8_t*>(codes);
  c.scale = scale;
  c.sp = s[0]; c.sh = s[1]; c.st = s[2];
  c.ssp = ss[0]; c.ssh = ss[1]; c.sst = ss[2];
  return c;
}

int lanes_of(int64_t D) { return D <= 64 ? 8 : D <= 128 ? 16 : 32; }

using RopeFn = void (*)(const RopeParams);
template <typename T, bool I, int U>
RopeFn rope_fn_u(int lanes) {
  return lanes == 8 ? rope_kernel<T, 8, U, I> : lanes == 16 ? rope_kernel<T, 16, U, I> : rope_kernel<T, 32, U, I>;
}
template <typename T, bool I>
RopeFn rope_fn(int lanes, int u) {
  return u == 2 ? rope_fn_u<T, I, 2>(lanes) : rope_fn_u<T, I, 4>(lanes);
}

using CopyFn = void (*)(const CopyParams);
template <typename T, bool E, int U>
CopyFn copy_fn_u(int lanes, bool write) {
  if (write)
    return lanes == 8 ? write_kernel<T, 8, U, E> : lanes == 16 ? write_kernel<T, 16, U, E> : write_kernel<T, 32, U, E>;
  return lanes == 8 ? read_kernel<T, 8, U, E> : lanes == 16 ? read_kernel<T, 16, U, E> : read_kernel<T, 32, U, E>;
}
template <typename T, bool E>
CopyFn copy_fn(int lanes, bool write, int u) {
  return u == 1 ? copy_fn_u<T, E, 1>(lanes, write) : u == 2 ? copy_fn_u<T, E, 2>(lanes, write) : copy_fn_u<T, E, 4>(lanes, write);
}

int rope(const dsa_kv_rope_args_t* a, void* stream) {
  if (!a) return DSA_KV_ERR_NULL_POINTER;
  if (a->struct_size != sizeof(*a)) return DSA_KV_ERR_BAD_ARGS_SIZE;
  const int ib = index_size(a->pos_dtype);
  if (!is_16bit(a->dtype) || !ib || !(is_16bit(a->gamma_dtype) || a->gamma_dtype == DSA_KV_FP32))
    return DSA_KV_ERR_BAD_DTYPE;
  if (a->B < 0 || a->Q < 0 || a->Hq < 0 || a->Hk < 0 || a->max_pos < 0 || (a->interleaved & ~1))
    return DSA_KV_ERR_BAD_SHAPE;
  if (a->D < 8 || a->D > 256 || a->D % 8 != 0 || a->rot < 0 || a->rot > a->D ||
      a->rot % (a->interleaved ? 8 : 16) != 0)
    return DSA_KV_ERR_BAD_HEAD_DIM;
  if (!fits(a->B, a->Q, a->Hq) || !fits(a->B, a->Q, a->Hk) || !fits(a->B, a->Q, a->Hq + a->Hk))
    return DSA_KV_ERR_UNSUPPORTED;
  if (a->B == 0 || a->Q == 0 || a->Hq + a->Hk == 0) return DSA_KV_OK;
  int st;
  if (a->Hq > 0) {
    if ((st = check_dense(a->q, a->B, a->Q, a->Hq, false)) != DSA_KV_OK) return st;
    if ((st = check_dense(a->q_out, a->B, a->Q, a->Hq, true)) != DSA_KV_OK) return st;
  }
  if (a->Hk > 0) {
    if ((st = check_dense(a->k, a->B, a->Q, a->Hk, false)) != DSA_KV_OK) return st;
    if ((st = check_dense(a->k_out, a->B, a->Q, a->Hk, true)) != DSA_KV_OK) return st;
  }
  if ((a->Hq > 0 && !a->q_gamma) || (a->Hk > 0 && !a->k_gamma) || !a->positions ||
      (a->rot > 0 && a->max_pos > 0 && !a->cos_sin))
    return DSA_KV_ERR_NULL_POINTER;
  if (!aligned(a->q_gamma, 16) || !aligned(a->k_gamma, 16) || !aligned(a->cos_sin, 16) ||
      !aligned(a->positions, ib))
    return DSA_KV_ERR_ALIGNMENT;

  int dev, sms;
  if (!bind_device(&dev) || !sm_count(dev, &sms)) return DSA_KV_ERR_CUDA;
  // Steps of two heads to a group of lanes where each then has a warp to itself on
  // one CTA per SM, else of four. Device time in us with two / four, 40 heads x
  // 128: 1 token 2.06 / 2.47, 32 tokens 2.47 / 2.77, 96 tokens 2.47 / 2.87, 128
  // tokens (160 CTAs) 2.98 / 2.88, 384 tokens 3.92 / 3.49, 8192 tokens 49 / 33.4 to 34.4.
  // Places of a step that heads leave empty are not looked at: 24 + 4 heads of 64 fill 28
  // of 48 with four (1665 tokens 5.3 us either way).
  const int lanes = lanes_of(a->D);
  int u = 2;
  int64_t steps_q, per_token;
  for (;; u = 4) {
    const int heads = 32 / lanes * u;  // of a step
    steps_q = ceil_div(a->Hq, heads);
    per_token = steps_q + ceil_div(a->Hk, heads);
    if (u == 4 || a->B * a->Q * per_token <= (int64_t)sms * kRopeWarps) break;
  }
  RopeParams p;
  p.q = dense(a->q);
  p.k = dense(a->k);
  p.q_out = dense(a->q_out);
  p.k_out = dense(a->k_out);
  p.q_gamma = a->q_gamma;
  p.k_gamma = a->k_gamma;
  p.cos_sin = a->cos_sin;
  p.positions = a->positions;
  p.max_pos = a->max_pos;
  p.tokens = (uint32_t)(a->B * a->Q);
  p.steps = (uint32_t)(a->B * a->Q * per_token);
  p.per_token.init((uint32_t)per_token);
  p.Q.init((uint32_t)a->Q);
  p.steps_q = (uint32_t)steps_q;
  p.Hq = (uint32_t)a->Hq;
  p.Hk = (uint32_t)a->Hk;
  p.D = (int32_t)a->D;
  p.rot = (int32_t)a->rot;
  p.gamma_dtype = a->gamma_dtype;
  p.pos_bytes = ib;
  p.eps = a->eps;
  p.inv_d = 1.0f / (float)a->D;
  const RopeFn fn = a->dtype == DSA_KV_BF16
                        ? (a->interleaved ? rope_fn<__nv_bfloat16, true>(lanes, u) : rope_fn<__nv_bfloat16, false>(lanes, u))
                        : (a->interleaved ? rope_fn<__half, true>(lanes, u) : rope_fn<__half, false>(lanes, u));
  // A warp for every step, as far as they are all resident at once.
  const int64_t most = (int64_t)sms * kRopeCtas, grid = ceil_div(p.steps, kRopeWarps);
  return launch(fn, grid < most ? grid : most, kRopeThreads, 0, 1, stream, p);
}

int copy(const dsa_kv_copy_args_t* a, void* stream, bool write) {
  if (!a) return DSA_KV_ERR_NULL_POINTER;
  if (a->struct_size != sizeof(*a)) return DSA_KV_ERR_BAD_ARGS_SIZE;
  const int ib = index_size(a->pos_dtype), pb = index_size(a->page_dtype);
  if (!is_16bit(a->dtype) || !ib || !pb) return DSA_KV_ERR_BAD_DTYPE;
  if (a->B < 0 || a->Q < 0 || a->NB < 0) return DSA_KV_ERR_BAD_SHAPE;
  int st = check_cache(a->cache, write ? kCacheWritten : kCacheRead);
  if (st != DSA_KV_OK) return st;
  const dsa_kv_cache_t& c = a->cache;
  if (!fits(a->B, a->Q, 2 * c.H) || a->NB > kMaxIndex) return DSA_KV_ERR_UNSUPPORTED;
  if (a->B == 0 || a->Q == 0 || a->NB == 0 || (write && c.P == 0)) return DSA_KV_OK;
  if ((st = check_dense(a->k, a->B, a->Q, c.H, !write)) != DSA_KV_OK) return st;
  if ((st = check_dense(a->v, a->B, a->Q, c.H, !write)) != DSA_KV_OK) return st;
  if (!a->page_table || !a->pos) return DSA_KV_ERR_NULL_POINTER;
  if (!aligned(a->page_table, pb) || !aligned(a->pos, ib)) return DSA_KV_ERR_ALIGNMENT;

  const int lanes = lanes_of(c.D);
  CopyParams p;
  p.k = dense(a->k);
  p.v = dense(a->v);
  p.kc = side(c.k_codes, c.k_scale, c.k_stride, c.k_scale_stride);
  p.vc = side(c.v_codes, c.v_scale, c.v_stride, c.v_scale_stride);
  p.page_table = a->page_table;
  p.pos = a->pos;
  p.P = c.P;
  // heads per step: what fills a warp, or all of them where they are fewer;
  // the rest of the warp then takes further tokens
  const int groups = 32 / lanes;
  int log_hps = 0;
  while ((1 << log_hps) < groups && (1 << log_hps) < c.H) ++log_hps;
  int log_tpw = 0;
  while ((1 << (log_hps + log_tpw)) < groups) ++log_tpw;
  const int64_t steps = ceil_div(c.H, 1 << log_hps);
  // Steps per lane, as many as there are up to 4. At 8 heads x 128 (us with
  // 1 / 2 / 4): write of 2 x 4096 tokens 13.0 / 11.0 / 11.0, read of 8 x up to
  // 8192 tokens 71.1 / 53.7 / 51.9; calls of 64 and of 333 tokens do not care.
  const int u = steps >= 4 ? 4 : steps >= 2 ? 2 : 1;
  const int64_t strips = ceil_div(steps, u), tokens = a->B * a->Q;
  p.tasks = (uint32_t)(ceil_div(tokens, 1 << log_tpw) * strips);
  p.tokens = (uint32_t)tokens;
  p.H = (uint32_t)c.H;
  p.log_hps = (uint32_t)log_hps;
  p.log_tpw = (uint32_t)log_tpw;
  p.strips.init((uint32_t)strips);
  p.Q.init((uint32_t)a->Q);
  p.bs.init((uint32_t)c.block_size);
  p.NB = a->NB;
  p.D = (int32_t)c.D;
  p.page_bytes = pb;
  p.pos_bytes = ib;
  const bool e = c.code_dtype == DSA_KV_E4M3;
  const CopyFn fn = a->dtype == DSA_KV_BF16
                        ? (e ? copy_fn<__nv_bfloat16, true>(lanes, write, u) : copy_fn<__nv_bfloat16, false>(lanes, write, u))
                        : (e ? copy_fn<__half, true>(lanes, write, u) : copy_fn<__half, false>(lanes, write, u));
  return launch(fn, ceil_div(p.tasks, kCopyThreads / 32), kCopyThreads, 0, 1, stream, p);
}

}  // namespace kv

extern "C" {

int dsa_kv_abi_version(void) { return DSA_KV_ABI_VERSION; }

const char* dsa_kv_strerror(int status) {
  switch (status) {
    case DSA_KV_OK: return "ok";
    case DSA_KV_ERR_NULL_POINTER: return "a required pointer is NULL";
    case DSA_KV_ERR_BAD_SHAPE: return "bad shape: a size or a stride below its least value";
    case DSA_KV_ERR_BAD_HEAD_DIM:
      return "head size or rotated part not supported (rotation: D <= 256, D % 8 == 0, rot <= D, rot % 16 == 0, "
             "interleaved rot % 8 == 0; cache: D <= 256, D % 16 == 0; attention: D 64, 128 or 256, block_size >= 8)";
    case DSA_KV_ERR_BAD_DTYPE:
      return "unsupported dtype (dense bf16/fp16, codes int8/e4m3, indices int32/int64, gamma bf16/fp16/fp32)";
    case DSA_KV_ERR_ALIGNMENT: return "misaligned pointer or stride (rows start on 16 bytes)";
    case DSA_KV_ERR_UNSUPPORTED: return "sizes beyond the 32-bit index range of the kernel";
    case DSA_KV_ERR_CUDA: return "a CUDA call failed";
    case DSA_KV_ERR_BAD_ARGS_SIZE:
      return "argument struct size mismatch (header and library differ) or reserved field not 0";
    case DSA_KV_ERR_DEVICE_TIMEOUT: return "a bounded device-side wait ran out";
    default: return "unknown dsa_kv status";
  }
}

int dsa_kv_rope_launch(const dsa_kv_rope_args_t* a, void* stream) { return kv::rope(a, stream); }
int dsa_kv_write_launch(const dsa_kv_copy_args_t* a, void* stream) { return kv::copy(a, stream, true); }
int dsa_kv_read_launch(const dsa_kv_copy_args_t* a, void* stream) { return kv::copy(a, stream, false); }

}  // extern "C"
