// dsa_kv_attn.cu — host side of dsa_kv_attn_launch (include/dsa_kv.h):
// validation, tensor maps and launch planning. Device code: kv_attn_kernel.cuh.
#include <atomic>

#include "kv_attn_kernel.cuh"
#include "kv_host.h"

namespace kv {

constexpr int kMaxDevices = 64;
constexpr int64_t kMaxBlockSize = 65536;

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                              const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                              CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// The driver's tensor-map encoder, looked up once (the library does not link libcuda).
EncodeFn encoder() {
  static std::atomic<void*> fn{nullptr};
  void* f = fn.load(std::memory_order_acquire);
  if (!f) {
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found) !=
            cudaSuccess ||
        found != cudaDriverEntryPointSuccess)
      return nullptr;
    fn.store(f, std::memory_order_release);
  }
  return reinterpret_cast<EncodeFn>(f);
}

// Map of the codes [P, H, block_size, D] as bytes: a box is `rows` tokens of
// one head and page, 128 bytes wide (64 where D = 64), swizzled over its
// width. Tokens behind the block read as zeros.
bool make_map(CUtensorMap* map, const dsa_kv_cache_t& c, void* codes, const int64_t stride[3], int rows) {
  EncodeFn encode = encoder();
  if (!encode) return false;
  const cuuint64_t dims[4] = {(cuuint64_t)c.D, (cuuint64_t)c.block_size, (cuuint64_t)c.H, (cuuint64_t)c.P};
  cuuint64_t strides[3] = {(cuuint64_t)stride[2], (cuuint64_t)stride[1], (cuuint64_t)stride[0]};
  for (int i = 0; i < 3; ++i)  // the stride of a dimension of one is never used
    if (dims[i + 1] == 1) strides[i] = (cuuint64_t)c.D;
  const cuuint32_t box[4] = {(cuuint32_t)(c.D == 64 ? 64 : 128), (cuuint32_t)rows, 1, 1}, step[4] = {1, 1, 1, 1};
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, codes, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                c.D == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

using AttnFn = void (*)(const AttnParams, const CUtensorMap, const CUtensorMap);
struct Variant {
  AttnFn fn;
  size_t smem;
};

// Ring slots per warp: as many as two CTAs per SM (D <= 128) or one have room for.
constexpr int slots_of(int D) { return D == 64 ? 6 : 3; }

template <typename T, bool E>
Variant variant_of(int64_t D) {
  switch (D) {
    case 64: return {attn_kernel<T, 64, E, slots_of(64)>, AttnSmem<64, slots_of(64)>::total};
    case 128: return {attn_kernel<T, 128, E, slots_of(128)>, AttnSmem<128, slots_of(128)>::total};
    default: return {attn_kernel<T, 256, E, slots_of(256)>, AttnSmem<256, slots_of(256)>::total};
  }
}

// Shared memory granted to each variant, per device.
std::atomic<bool> g_granted[kMaxDevices][12];

int attn(const dsa_kv_attn_args_t* a, void* stream) {
  if (!a) return DSA_KV_ERR_NULL_POINTER;
  if (a->struct_size != sizeof(*a)) return DSA_KV_ERR_BAD_ARGS_SIZE;
  const int bb = index_size(a->block_dtype), pb = index_size(a->page_dtype), ib = index_size(a->pos_dtype);
  if (!is_16bit(a->dtype) || !bb || !pb || !ib) return DSA_KV_ERR_BAD_DTYPE;
  if (a->B < 0 || a->Q < 0 || a->G < 1 || a->K < 0) return DSA_KV_ERR_BAD_SHAPE;
  int st = check_cache(a->cache, false);
  if (st != DSA_KV_OK) return st;
  const dsa_kv_cache_t& c = a->cache;
  if ((c.D != 64 && c.D != 128 && c.D != 256) || c.block_size < 8) return DSA_KV_ERR_BAD_HEAD_DIM;
  if (c.block_size > kMaxBlockSize || a->G > kMaxIndex) return DSA_KV_ERR_UNSUPPORTED;
  const int64_t MT = ceil_div(a->G, kRows);
  if (!fits(a->B, a->Q, c.H) || !fits(a->B * a->Q * c.H, MT, 1) || !fits(c.H, a->G, 1)) return DSA_KV_ERR_UNSUPPORTED;
  if (a->B == 0 || a->Q == 0) return DSA_KV_OK;
  if ((st = check_dense(a->q, a->B, a->Q, c.H * a->G, false)) != DSA_KV_OK) return st;
  if ((st = check_dense(a->out, a->B, a->Q, c.H * a->G, true)) != DSA_KV_OK) return st;
  if (!a->q_pos || !a->kv_lens || (a->K > 0 && (!a->blocks || !a->pages))) return DSA_KV_ERR_NULL_POINTER;
  if (!aligned(a->blocks, bb) || !aligned(a->pages, pb) || !aligned(a->q_pos, ib) || !aligned(a->kv_lens, ib) ||
      !aligned(a->lse, 4))
    return DSA_KV_ERR_ALIGNMENT;

  // Chunks: a block of more than 16 tokens is cut into pieces of 32, shorter
  // blocks share a chunk by two (9 to 16 tokens) or four (8).
  const int log_pieces = c.block_size > 16 ? 0 : c.block_size > 8 ? 1 : 2;
  const int64_t per_block = log_pieces ? 1 : ceil_div(c.block_size, kTok);
  const int64_t items = log_pieces ? ceil_div(a->K, 1 << log_pieces) : a->K * per_block;
  if (a->K > (1 << 30) || items > (1 << 30)) return DSA_KV_ERR_UNSUPPORTED;
  const int box_rows = (int)(c.block_size < (kTok >> log_pieces) ? c.block_size : (kTok >> log_pieces));

  AttnParams p;
  p.q = dense(a->q);
  p.out = dense(a->out);
  p.lse = a->lse;
  p.k_scale = c.k_scale;
  p.v_scale = c.v_scale;
  p.ksp = c.k_scale_stride[0]; p.ksh = c.k_scale_stride[1]; p.kst = c.k_scale_stride[2];
  p.vsp = c.v_scale_stride[0]; p.vsh = c.v_scale_stride[1]; p.vst = c.v_scale_stride[2];
  p.blocks = a->blocks;
  p.pages = a->pages;
  p.bsb = a->blocks_stride[0]; p.bsh = a->blocks_stride[1]; p.bsq = a->blocks_stride[2];
  p.psb = a->pages_stride[0]; p.psh = a->pages_stride[1]; p.psq = a->pages_stride[2];
  p.q_pos = a->q_pos;
  p.kv_lens = a->kv_lens;
  p.MT.init((uint32_t)MT);
  p.Q.init((uint32_t)a->Q);
  p.H.init((uint32_t)c.H);
  p.per_block.init((uint32_t)per_block);
  p.P = c.P;
  p.items = (uint32_t)items;
  p.G = (int32_t)a->G;
  p.K = (int32_t)a->K;
  p.bs = (int32_t)c.block_size;
  p.log_pieces = log_pieces;
  p.box_bytes = (uint32_t)(box_rows * (c.D == 64 ? 64 : 128));
  p.block_bytes = bb;
  p.page_bytes = pb;
  p.pos_bytes = ib;
  p.scale = a->softmax_scale * 1.44269504088896341f;
  CUtensorMap k_map = {}, v_map = {};
  if (c.P > 0 && (!make_map(&k_map, c, c.k_codes, c.k_stride, box_rows) ||
                  !make_map(&v_map, c, c.v_codes, c.v_stride, box_rows)))
    return DSA_KV_ERR_CUDA;

  const bool e = c.code_dtype == DSA_KV_E4M3, bf = a->dtype == DSA_KV_BF16;
  const Variant v = bf ? (e ? variant_of<__nv_bfloat16, true>(c.D) : variant_of<__nv_bfloat16, false>(c.D))
                       : (e ? variant_of<__half, true>(c.D) : variant_of<__half, false>(c.D));
  int dev;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return DSA_KV_ERR_CUDA;
  std::atomic<bool>& granted = g_granted[dev][(c.D / 128) * 4 + (e ? 2 : 0) + (bf ? 1 : 0)];
  if (!granted.load(std::memory_order_relaxed)) {
    if (cudaFuncSetAttribute(reinterpret_cast<const void*>(v.fn), cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (int)v.smem) != cudaSuccess)
      return DSA_KV_ERR_CUDA;
    granted.store(true, std::memory_order_relaxed);
  }
  return launch(v.fn, a->B * a->Q * c.H * MT, kAttnWarps * 32, v.smem, stream, p, k_map, v_map);
}

}  // namespace kv

extern "C" int dsa_kv_attn_launch(const dsa_kv_attn_args_t* a, void* stream) { return kv::attn(a, stream); }
