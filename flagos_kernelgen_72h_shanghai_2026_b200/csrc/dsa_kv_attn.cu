// dsa_kv_attn.cu — host side of dsa_kv_attn_launch (include/dsa_kv.h):
// validation, tensor maps and launch planning. Device code: kv_attn_kernel.cuh.
#include <atomic>

#include "kv_attn_kernel.cuh"
#include "kv_host.h"

namespace kv {

constexpr int64_t kMaxBlockSize = 65536;
constexpr size_t kSmemPerSm = 228 * 1024, kSmemReserved = 1024;  // of an SM; of it for each CTA, by the system

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                              const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                              CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// Map of the codes [P, H, block_size, D] as bytes: a box is `rows` tokens of
// one head and page, 128 bytes wide (64 where D = 64), swizzled over its
// width. Tokens behind the block read as zeros.
bool make_map(CUtensorMap* map, const dsa_kv_cache_t& c, void* codes, const int64_t stride[3], int rows) {
  static std::atomic<void*> entry{nullptr};
  const EncodeFn encode = reinterpret_cast<EncodeFn>(driver_entry(&entry, "cuTensorMapEncodeTiled"));
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
  size_t smem, more;  // shared memory of a CTA alone, and for each further CTA of its cluster
  int tok, ctas;      // tokens of a chunk, CTAs per SM
};
template <typename T, bool E, int D, int NB, int TOK, int CTAS>
Variant variant() {
  using L = AttnSmem<D, NB, TOK>;
  return Variant{attn_kernel<T, D, E, NB, TOK, CTAS>, L::total(1), L::total(2) - L::total(1), TOK, CTAS};
}
// Tokens of a chunk, and CTAs per SM that registers are laid out for. Measured
// (us, 2048 tokens to a row): chunks of 64 tokens against 32 with 16 heads at
// D = 128, 1024 rows: 83.0 against 85.0 (three CTAs of 32) and 100 (two): what a
// chunk costs besides its products weighs as much as the warps that hide it. CTAs
// with chunks of 64: three against two there 99.4 to 83.0 (spills); with 8 heads,
// 2048 rows, 107 to 122; at D = 64 with 8 heads three / four / five 73.6 / 67.0 /
// 68.4, with 16 heads two / three / four 112 / 94.8 / 98.1.
template <typename T, bool E>
Variant variant_of(int64_t D, int nb) {
  if (D == 64) return nb == 1 ? variant<T, E, 64, 1, 64, 4>() : variant<T, E, 64, 2, 64, 3>();
  if (D == 128) return nb == 1 ? variant<T, E, 128, 1, 64, 3>() : variant<T, E, 128, 2, 64, 2>();
  return nb == 1 ? variant<T, E, 256, 1, 32, 2>() : variant<T, E, 256, 2, 32, 2>();
}

// Shared memory granted to each variant, per device.
std::atomic<bool> g_granted[kMaxDevices][24];

// Clusters of 2^log_c CTAs that are resident at once with up to n of their CTAs
// on an SM: less than the SMs' number gives, as a cluster stays within one group
// of SMs. With shared memory for no more than n, it does not depend on the variant.
int64_t max_clusters(const Variant& v, int dev, int n, int log_c) {
  static std::atomic<int> known[kMaxDevices][8][4];  // plus one
  std::atomic<int>& have = known[dev][n - 1][log_c];
  int count = have.load(std::memory_order_relaxed) - 1;
  if (count >= 0) return count;
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = 1u << log_c;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(1u << log_c);
  cfg.blockDim = dim3(kAttnThreads);
  cfg.dynamicSmemBytes = kSmemPerSm / n - kSmemReserved;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  if (cudaOccupancyMaxActiveClusters(&count, reinterpret_cast<const void*>(v.fn), &cfg) != cudaSuccess) {
    (void)cudaGetLastError();
    return 0;  // no clusters then
  }
  have.store(count + 1, std::memory_order_relaxed);
  return count;
}

int attn(const dsa_kv_attn_args_t* a, int32_t* status, int32_t test_copies, void* stream) {
  if (!a) return DSA_KV_ERR_NULL_POINTER;
  if (a->struct_size != sizeof(*a)) return DSA_KV_ERR_BAD_ARGS_SIZE;
  const int bb = index_size(a->block_dtype), pb = index_size(a->page_dtype), ib = index_size(a->pos_dtype);
  if (!is_16bit(a->dtype) || !bb || !pb || !ib) return DSA_KV_ERR_BAD_DTYPE;
  if (a->B < 0 || a->Q < 0 || a->G < 1 || a->K < 0 || test_copies < 0 || test_copies == 1) return DSA_KV_ERR_BAD_SHAPE;
  int st = check_cache(a->cache, kCacheMapped);
  if (st != DSA_KV_OK) return st;
  const dsa_kv_cache_t& c = a->cache;
  if ((c.D != 64 && c.D != 128 && c.D != 256) || c.block_size < 8) return DSA_KV_ERR_BAD_HEAD_DIM;
  if (c.block_size > kMaxBlockSize || a->G > kMaxIndex) return DSA_KV_ERR_UNSUPPORTED;
  const int64_t n[3] = {c.P, c.H, c.block_size};
  for (int i = 0; i < 3; ++i)  // the kernel holds the scales' strides in 32 bits
    if (n[i] > 1 && (c.k_scale_stride[i] > kMaxIndex || c.v_scale_stride[i] > kMaxIndex)) return DSA_KV_ERR_UNSUPPORTED;
  const int nb = a->G <= 8 ? 1 : 2;
  const int64_t MT = ceil_div(a->G, 8 * nb);
  if (!fits(a->B, a->Q, c.H) || !fits(a->B * a->Q * c.H, MT, 1) || !fits(c.H, a->G, 1)) return DSA_KV_ERR_UNSUPPORTED;
  if (a->B == 0 || a->Q == 0) return DSA_KV_OK;
  if ((st = check_dense(a->q, a->B, a->Q, c.H * a->G, false)) != DSA_KV_OK) return st;
  if ((st = check_dense(a->out, a->B, a->Q, c.H * a->G, true)) != DSA_KV_OK) return st;
  if (!a->q_pos || !a->kv_lens || (a->K > 0 && (!a->blocks || !a->pages))) return DSA_KV_ERR_NULL_POINTER;
  if (!aligned(a->blocks, bb) || !aligned(a->pages, pb) || !aligned(a->q_pos, ib) || !aligned(a->kv_lens, ib) ||
      !aligned(a->lse, 4) || !aligned(status, 4))
    return DSA_KV_ERR_ALIGNMENT;

  const int64_t tiles = a->B * a->Q * c.H * MT;
  const bool e = c.code_dtype == DSA_KV_E4M3, bf = a->dtype == DSA_KV_BF16;
  const Variant v = bf ? (e ? variant_of<__nv_bfloat16, true>(c.D, nb) : variant_of<__nv_bfloat16, false>(c.D, nb))
                       : (e ? variant_of<__half, true>(c.D, nb) : variant_of<__half, false>(c.D, nb));

  // Chunks: a block of more than half a chunk is cut into chunks, shorter ones
  // share a chunk, at most 8 of them (block_size >= 8).
  int log_pieces = 0;
  while ((v.tok >> (log_pieces + 1)) >= c.block_size) ++log_pieces;
  const int piece = v.tok >> log_pieces;  // rows of a chunk for each block
  const int64_t per_block = ceil_div(c.block_size, piece);
  const int64_t items = log_pieces ? ceil_div(a->K, 1 << log_pieces) : a->K * per_block;
  if (a->K > (1 << 30) || items > (1 << 30)) return DSA_KV_ERR_UNSUPPORTED;
  const int box_rows = (int)(c.block_size < piece ? c.block_size : piece);

  int dev, sms;
  if (!bind_device(&dev) || !sm_count(dev, &sms)) return DSA_KV_ERR_CUDA;
  std::atomic<bool>& granted = g_granted[dev][(c.D / 128) * 8 + (nb - 1) * 4 + (e ? 2 : 0) + (bf ? 1 : 0)];
  if (!granted.load(std::memory_order_relaxed)) {
    if (cudaFuncSetAttribute(reinterpret_cast<const void*>(v.fn), cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (int)(kSmemPerSm - kSmemReserved)) != cudaSuccess)
      return DSA_KV_ERR_CUDA;
    granted.store(true, std::memory_order_relaxed);
  }
  // CTAs to a tile: what ends first. Of the tile's rounds (a chunk to each warp)
  // a cluster takes its share; joining 2, 4 or 8 CTAs takes as long as 1.5, 2 or
  // 2.5 rounds, and n CTAs on an SM make a round (n + 1) / 2 as long. A cluster is
  // taken only where all tiles' are resident at once. Measured (us with 1 / 2 / 4 /
  // 8 CTAs, 4 query heads, D = 128): 8 tiles of 8 chunks 6.3 / 6.8 / 7.3 / 7.3, of
  // 16 chunks 9.2 / 8.3 / 7.3 / 7.5, of 32 chunks 14.9 / 11.2 / 8.7 / 7.7; 64 tiles
  // of 32 chunks 16.0 / 12.4 / 11.4 / 18.5; 144 tiles of 16 chunks 12.2 / 13.0 /
  // 19.4 / 30.9. Over 738 cases of every head size the choice is 1.4 % off the best
  // in the mean and 29 % at worst (32 to 48 tiles of 32 blocks, 8 CTAs for 4); as many
  // CTAs as the SMs hold were 5.6 %, and up to 82 % where clusters did not fit the
  // groups of SMs that hold one together.
  int log_c = 0, per_sm = tiles <= (int64_t)sms * v.ctas ? (int)ceil_div(tiles, sms) : v.ctas;
  {
    const int join2[4] = {0, 3, 4, 5};  // twice the rounds of a join
    int64_t best = ceil_div(items, kAttnWarps) * (per_sm + 1);
    for (int l = 1; (1 << l) <= kMaxCluster && items > (int64_t)(kAttnWarps << (l - 1)); ++l) {
      int n = 1;
      while (n <= v.ctas && max_clusters(v, dev, n, l) < tiles) ++n;
      if (n > v.ctas) break;  // larger ones do not fit either
      const int64_t cost = ceil_div(items, kAttnWarps << l) * (n + 1) + join2[l];
      if (cost < best) {
        best = cost;
        log_c = l;
        per_sm = n;
      }
    }
  }
  const int cluster = 1 << log_c;

  // A grid of at most one wave spreads evenly over the SMs only if no more CTAs
  // than its share fit one, because the next launch's are placed wherever the
  // last ones of this leave room: shared memory is asked for until that is so
  // (256 tiles of 8 heads, 8192 tokens: 87.0 instead of 96.0 us call after call).
  const int64_t grid = tiles * cluster, resident = (int64_t)sms * v.ctas;
  const bool early = grid * 2 <= resident;
  size_t smem = v.smem + (cluster - 1) * v.more;
  if (!early && per_sm < v.ctas) {
    const size_t least = kSmemPerSm / (per_sm + 1) - kSmemReserved + 1;  // one CTA more does not fit
    if (smem < least) smem = least;
  }

  AttnParams p;
  p.q = dense(a->q);
  p.out = dense(a->out);
  p.lse = a->lse;
  p.k_scale = c.k_scale;
  p.v_scale = c.v_scale;
  p.ksp = (uint32_t)c.k_scale_stride[0]; p.ksh = (uint32_t)c.k_scale_stride[1]; p.kst = (uint32_t)c.k_scale_stride[2];
  p.vsp = (uint32_t)c.v_scale_stride[0]; p.vsh = (uint32_t)c.v_scale_stride[1]; p.vst = (uint32_t)c.v_scale_stride[2];
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
  p.cluster = (uint32_t)cluster;
  p.early = early;
  p.status = status;
  p.give_up = test_copies < 1 << 30 ? (uint32_t)test_copies : 0;
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

  return launch(v.fn, grid, kAttnThreads, smem, cluster, stream, p, k_map, v_map);
}

}  // namespace kv

extern "C" {

int dsa_kv_attn_launch(const dsa_kv_attn_args_t* a, void* stream) { return kv::attn(a, nullptr, 0, stream); }
int dsa_kv_attn_launch_status(const dsa_kv_attn_args_t* a, int32_t* status, int32_t test_copies, void* stream) {
  return kv::attn(a, status, test_copies, stream);
}

}  // extern "C"
