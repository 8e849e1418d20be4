// kv_attn_kernel.cuh — attention of query rows over selected blocks of the
// quantised paged cache (dsa_kv_attn_launch, include/dsa_kv.h).
//
// A row (b, h, q) has G query heads that share a key head and a selection. A
// CTA, or where there are few rows a cluster of up to 8 CTAs, works on 8 * NB
// of them (NB = 1 or 2). The row's selected tokens are cut into chunks of TOK
// = 32 or 64, dealt to the warps in turn; every warp runs the one-pass softmax on its own
// chunks and the partial results are joined at the end through the cluster's
// distributed shared memory: no workspace, no atomics, an order of summation
// that does not vary.
//
// Mathematics, per query head, tokens t with key codes k, value codes v and
// their scales ks, vs:
//     a_t = log2(e) * scale * ks_t * (q.k_t) + log2(vs_t)
//     o   = sum_t 2^(a_t - M) v_t,   l = sum_t 2^(a_t - M) / vs_t
//     out = o / l,   lse = ln 2 * (M + log2 l)
// with M the running maximum of a_t. The value scale sits in the exponent, so
// the weight of a token is at most 1 whatever the scales are, the products
// run on raw codes (exact in fp16), and the maximum bounds each term of o.
// It does not bound those of l, nor keep them near 1: where value scales differ
// by more than 2^126, 2^(a_t - M) may be zero in fp32 and 2^(a_t - M) / vs_t not. A
// warp that has met a scale above 2^32 (the least is 1e-12) takes the terms of l as
// 2^(a_t - M - log2(vs_t)) from then on, times 2^24 (a row's l lies between 2^-122
// and 2^85: a term 2^-28 of the least one still counts), and l is multiplied by
// powers of two that may themselves be too small in two steps, here and in the join.
// It does the same from a value scale on that is not finite: such a token enters a_t
// and l as if its scale were 1, and its weight in the second product is NaN.
//
// Precision: q is brought to fp16 by one power of two for all heads of a CTA, the
// largest value in [2^14, 2^15): bf16 values lose bits only 2^-28 below it. Where a
// head's largest value is more than 2^8 below the CTA's, every head has a power of its
// own, and all chunks go through the loop's second copy, which applies them.
// Weights are fp16 too, times 2^6: 2^-11 relative (the output's own half step
// is 2^-9 or 2^-12) down to 2^-20, with an absolute 2^-31 below. M lags behind
// the maximum by up to 8 (a weight is at most 2^14), so that o is rescaled
// only when the maximum really moves. Sums are fp32 throughout.
//
// Tensor-core tiles (m16n8k16): tokens, then values of D, are the 16 rows and
// query heads the 8 columns. Scores S = K q^T take 16 tokens x 8 heads at a
// time, outputs O^T = V^T P^T 16 values of D x 8 heads. With heads as rows
// instead, groups of up to 8 heads left half of every tile, and of the
// exponentials and the output's registers, empty.
//
// Data movement: a chunk's key rows and value rows come by one TMA box each, into
// two boxes of the warp's own, so that no CTA barrier is needed on the way: the
// keys' box is refilled as soon as the scores are done, the values' box after
// the second product. Scales follow by 4-byte asynchronous copies. (A third box
// a chunk ahead gained nothing, and took the third CTA's room. A producer warp
// that starts all copies of a CTA was slower, 109 for 98 us: a TMA instruction
// holds its warp for 85 cycles, and the rest of its work is one long chain.)
// Rows are 128 bytes (64 for D = 64), swizzled by the copy, which makes all
// fragment reads free of bank conflicts: a lane reads 32 contiguous bytes of two
// key rows of a tile for the products over D, whose order of summation is free
// to choose; value tiles come transposed, byte by byte, through ldmatrix. The
// weights change sides with movmatrix.
//
// Why mma.sync: a row has at most 16 heads to multiply a key with, the least
// tile of tcgen05 has 64 or 128 rows; with tokens as those rows fp16 operands would
// mean to write the codes back to shared memory widened. Its 8-bit kinds take the
// codes as they are copied, with queries and weights cut into 8-bit terms; that form
// has not been built.
//
// What bounds it: a decode batch is bound by HBM (32 rows x 8 key heads over 8192
// e4m3 tokens of D = 128: 87 to 88 us, 6.3 TB/s). Rows whose pages stay in L2 are bound
// by latency at 8 warps per SM (1024 rows x 16 heads x 2048 tokens, D = 128: 85.4 us):
// issue slots are 37 % and the tensor pipe 37 % busy; a chunk is a chain of wait, scores,
// maximum, exponentials, weights turned around, outputs, and 254 registers hold
// two CTAs. 32 tokens of 16 heads take an SM 379 cycles there at 1965 MHz in the mean, 274
// as the slope from 64 to 128 blocks; the tensor pipe needs 128 of them, the
// conversion of codes, on the half-rate integer pipe, 64. The mean holds the rows' start
// and join and the last wave: 1024 CTAs on 296 places are 3.46 waves, worth 13 %.
// The second copy of the loop (value scales above 2^32 or not finite, heads of
// unlike size) takes 24 % longer for values of that kind there, 8 % for such heads.
#pragma once

#include <cuda.h>
#include <type_traits>

#include "farq_kernel.cuh"
#include "kv_common.cuh"

namespace kv {

constexpr int kAttnWarps = 4;      // warps of a CTA
constexpr int kAttnThreads = 32 * kAttnWarps;
constexpr int kMaxCluster = 8;
constexpr float kLift = 6.0f;      // weights are 2^(a - M + kLift)
// The kernel holds M - kLift as it is rounded, and takes all differences from that: from
// 2^24 on kLift is below M's last place. It is moved where a maximum is at least the
// rounded (M - kLift) + kLift + kLag, so that no weight is above 2^14: a maximum that is
// larger than the sum is not smaller than the sum rounded. (Moved where M + kLag was
// exceeded, values 16 above an M of 2^26 stayed, and 2^(16 + kLift) is no fp16 number.)
constexpr float kLag = 8.0f;
constexpr float kWide = 4294967296.0f;  // value scales up to it: 1 / vs brings every term of l that counts back
constexpr float kSumLift = 24.0f;       // l is 2^kSumLift times its value from there on, and in the join
constexpr float kSumUp = 16777216.0f;   // 2^kSumLift
constexpr float kTwoSteps = -64.0f;     // powers of two below it are applied to l in two steps
constexpr uint64_t kAttnWaitNs = 2000000000ull;

struct AttnParams {
  Dense q, out;
  float* lse;  // may be null
  const float* k_scale;
  const float* v_scale;
  uint32_t ksp, ksh, kst, vsp, vsh, vst;  // scale strides (page, head, token)
  const void* blocks;
  const void* pages;
  int64_t bsb, bsh, bsq, psb, psh, psq;  // strides of blocks and pages (b, h, q)
  const void* q_pos;
  const void* kv_lens;
  FastDiv MT, Q, H;     // groups of 8 * NB query heads per row, rows
  FastDiv per_block;    // chunks of a block
  int64_t P;
  uint32_t items;       // chunks of a row
  int32_t G, K, bs;
  int32_t log_pieces;   // a chunk holds 2^log_pieces blocks, where they are short
  uint32_t box_bytes;   // bytes of one copied box
  int32_t block_bytes, page_bytes, pos_bytes;
  uint32_t cluster;     // CTAs that share a row's tokens
  bool early;           // the next launch fits beside this one
  int32_t* status;      // may be null
  uint32_t give_up;     // test only: copies after which a row's first warp takes its next wait as run out
  float scale;          // softmax_scale * log2(e)
};

// Shared-memory carve-up, identical on host and device.
template <int D, int NB, int TOK>
struct AttnSmem {
  static constexpr int W = kAttnWarps;
  static constexpr int R = 8 * NB;                // query heads
  static constexpr size_t box = (size_t)TOK * D;  // keys or values of a chunk
  static constexpr size_t ring = 0;
  static constexpr size_t region = 2 * box;       // of a warp: keys, values; at the end its partial result
  static_assert((size_t)R * D * 4 <= region, "the ring holds the partial result");
  static constexpr size_t tok = ring + W * region;                // [W][TOK] factors of a chunk's tokens
  static constexpr size_t scales = tok + (size_t)W * TOK * 16;    // [W][2][TOK]
  static constexpr size_t bars = scales + (size_t)W * 2 * TOK * 4;  // [W][2]
  // [W][2][R] maxima less kLift, and sums; until then the heads' own powers of two
  static constexpr size_t ml = bars + (size_t)W * 2 * 8;
  static constexpr size_t fin = ml + (size_t)W * 2 * R * 4;          // [R] 1 / l
  static constexpr bool q_in_smem = D >= 128 && NB == 2;             // where the output fills the registers
  static constexpr size_t qf = fin + R * 4;
  static constexpr size_t all = qf + (q_in_smem ? (size_t)(D / 16) * NB * 32 * 8 : 0);
  // [C * W][R] weights of the cluster's warps
  static constexpr size_t total(int cluster) { return all + (size_t)cluster * W * R * 4; }
};

__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int x, int tok, int head, int page,
                                         uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(map), "r"(x), "r"(tok), "r"(head), "r"(page), "r"(bar)
      : "memory");
}
// c += a * b for one m16n8k16 tile, fp16 operands, fp32 sums.
__device__ __forceinline__ void mma16816(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9},"
      " {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// c = a * b.
__device__ __forceinline__ void mma16816_first(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9},"
      " {%10, %10, %10, %10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
// Two 16 x 16 tiles of bytes, transposed: row addresses from lanes 0 to 15 and
// 16 to 31. Lane (g, c) gets rows 4c to 4c + 3 of column g (r[0], r[2]) and of
// column g + 8 (r[1], r[3]).
__device__ __forceinline__ void load_transposed(uint32_t r[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m16n16.x2.trans.shared.b8 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The transposed 8 x 8 tile of 16-bit values.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
// Four codes -> two pairs of fp16 values (bytes 0, 1 and bytes 2, 3).
// int8: the byte with its sign flipped, under the exponent of 1024, is the
// fp16 number 1024 + 128 + code; both steps are exact.
template <bool E4M3>
__device__ __forceinline__ void decode_pairs(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if (E4M3) {
    // one instruction each: the register's halves are named, not shifted
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
  } else {
    const uint32_t s = w ^ 0x80808080u, bias = 0x64806480u;
    const uint32_t a = __byte_perm(s, 0x64646464u, 0x4140), b = __byte_perm(s, 0x64646464u, 0x4342);
    const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&bias));
    const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&b), *reinterpret_cast<const __half2*>(&bias));
    lo = *reinterpret_cast<const uint32_t*>(&x);
    hi = *reinterpret_cast<const uint32_t*>(&y);
  }
}

// Address of another CTA's shared memory in the cluster, and loads from it.
__device__ __forceinline__ uint32_t mapa(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ float ld_cluster(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }

// Place of float4 `f4` of head `row` in a warp's partial result: the units of a
// head are permuted so that the lanes' writes spread over the banks.
template <int D>
__device__ __forceinline__ int part_index(int row, int f4) {
  return row * (D / 4) + (f4 ^ (((row >> 1) & 3) << 1));
}

template <typename T, int D, bool E4M3, int NB, int TOK, int CTAS>
__global__ void __launch_bounds__(kAttnThreads, CTAS)
    attn_kernel(const AttnParams p, const __grid_constant__ CUtensorMap k_map,
                const __grid_constant__ CUtensorMap v_map) {
  using L = AttnSmem<D, NB, TOK>;
  constexpr int W = kAttnWarps, R = L::R;
  constexpr int NH = D == 256 ? 2 : 1;    // boxes of at most 128 bytes' width per side
  constexpr int NU = D == 64 ? 1 : 2;     // 16-byte pieces of a key row per lane and box
  constexpr int NT = D / 16;              // 16-row tiles of the output
  constexpr int NS = TOK / 16;            // 16-row tiles of the scores
  constexpr int LT = TOK / 32;            // tokens of a lane, where each token has one: lane, lane + 32
  constexpr int LOG_TOK = TOK == 64 ? 6 : 5;
  constexpr int ROWB = D == 64 ? 64 : 128;
  constexpr bool QSMEM = L::q_in_smem;
  extern __shared__ __align__(1024) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const uint32_t C = p.cluster, rank = blockIdx.x & (C - 1), NW = C * W, wid = rank * W + warp;
  uint32_t r = blockIdx.x / C, mt, qi, h, b;
  p.MT.divmod(r, &r, &mt);
  p.Q.divmod(r, &r, &qi);
  p.H.divmod(r, &b, &h);
  const int head0 = (int)h * p.G + (int)mt * R;
  const int rows = min(R, p.G - (int)mt * R);

  const uint32_t base = farq::smem_u32(smem);
  uint8_t* const ring = smem + L::ring + warp * L::region;
  const uint32_t bars = base + (uint32_t)L::bars + warp * 2 * 8;
  float* const scales = reinterpret_cast<float*>(smem + L::scales) + warp * 2 * TOK;
  float4* const tok = reinterpret_cast<float4*>(smem + L::tok) + warp * TOK;
  if (lane == 0) {
    for (int s = 0; s < 2; ++s) farq::mbar_init(bars + 8 * s, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&k_map) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&v_map) : "memory");
  }
  __syncwarp();
  asm volatile("griddepcontrol.wait;" ::: "memory");
  // The next launch may come in: at once where it finds room beside this one,
  // else when this one's CTAs are about to end. Earlier, its waiting CTAs would
  // take the places that this grid's last CTAs need to spread evenly.
  if (p.early) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // Everything the first copies depend on is loaded at once: position and
  // length, the first 32 pieces of the selection, the queries.
  const int64_t pos = load_index(p.q_pos, (int64_t)b * p.Q.d + qi, p.pos_bytes);
  int64_t lim = load_index(p.kv_lens, b, p.pos_bytes);
  const int64_t brow = b * p.bsb + h * p.bsh + qi * p.bsq;
  const int64_t prow = b * p.psb + h * p.psh + qi * p.psq;
  const float* const k_scale = p.k_scale + (uint64_t)h * p.ksh;
  const float* const v_scale = p.v_scale + (uint64_t)h * p.vsh;

  // The warp looks its chunks up 32 pieces at a time (with lp = 0 a chunk is
  // one piece); a lane holds one: page, first token within the page, tokens
  // that count.
  const int lp = p.log_pieces, per = 1 << lp, pitch = TOK >> lp;
  uint32_t next_k = 0, active = 0, pieces = 0;  // chunks and pieces of this look-up that are left
  int pc_page = 0, pc_off = 0, pc_n = 0;
  int64_t ld_blk, ld_page;
  uint32_t ld_sub;
  auto fetch = [&] {  // the next 32 pieces' entries
    const uint32_t item = wid + (next_k + (lane >> lp)) * NW;
    next_k += 32 >> lp;
    uint32_t entry;
    ld_sub = 0;
    if (lp == 0)
      p.per_block.divmod(item, &entry, &ld_sub);
    else
      entry = (item << lp) + (lane & (per - 1));
    ld_blk = ld_page = -1;
    if (item < p.items && entry < (uint32_t)p.K) {
      ld_blk = load_index(p.blocks, brow + entry, p.block_bytes);
      ld_page = load_index(p.pages, prow + entry, p.page_bytes);
    }
  };
  auto look_up = [&] {
    pc_n = 0;
    if (ld_blk >= 0 && ld_blk < lim && ld_page >= 0 && ld_page < p.P) {
      const int64_t left = lim - (ld_blk * p.bs + (int64_t)ld_sub * TOK);
      const int most = min(TOK, p.bs - (int)ld_sub * TOK);
      pc_n = left <= 0 ? 0 : left < most ? (int)left : most;
      pc_page = (int)ld_page;
      pc_off = (int)ld_sub * TOK;
    }
    active = pieces = __ballot_sync(0xffffffffu, pc_n > 0);
    if (lp >= 1) active |= active >> 1;
    if (lp >= 2) active |= active >> 2;
    if (lp >= 3) active |= active >> 4;
    if (lp >= 1) active &= lp == 1 ? 0x55555555u : lp == 2 ? 0x11111111u : 0x01010101u;
  };
  // The chunk whose keys, and then values, are copied next: the piece that
  // this lane copies (lanes 0 to 2^lp - 1), its tokens and their scales.
  bool more = true;
  int cp_page = 0, cp_off = 0;
  bool copies = false;
  uint32_t cp_bytes = 0, cp_mask[LT];
  const float *cp_ks[LT], *cp_vs[LT];
  auto prepare = [&] {
    while (active == 0) {
      if (wid + next_k * NW >= p.items) {
        more = false;
        return;
      }
      fetch();
      look_up();
    }
    const int first = __ffs(active) - 1;
    active &= active - 1;
    if (lp == 0) {
      cp_page = __shfl_sync(0xffffffffu, pc_page, first);
      cp_off = __shfl_sync(0xffffffffu, pc_off, first);
      const int n = __shfl_sync(0xffffffffu, pc_n, first);
      cp_bytes = NH * p.box_bytes;
      copies = lane == 0;
      cp_ks[0] = k_scale + (uint64_t)(uint32_t)cp_page * p.ksp + (uint64_t)(uint32_t)(cp_off + lane) * p.kst;
      cp_vs[0] = v_scale + (uint64_t)(uint32_t)cp_page * p.vsp + (uint64_t)(uint32_t)(cp_off + lane) * p.vst;
      cp_mask[0] = n >= 32 ? 0xffffffffu : (1u << n) - 1;
      if (LT == 2) {
        cp_ks[LT - 1] = cp_ks[0] + (uint64_t)p.kst * 32;
        cp_vs[LT - 1] = cp_vs[0] + (uint64_t)p.vst * 32;
        cp_mask[LT - 1] = n >= 64 ? 0xffffffffu : n > 32 ? (1u << (n - 32)) - 1 : 0;
      }
      return;
    }
    const uint32_t here = (pieces >> first) & ((1u << per) - 1);
    cp_bytes = __popc(here) * NH * p.box_bytes;
    copies = lane < per && ((here >> lane) & 1);
#pragma unroll
    for (int t = 0; t < LT; ++t) {
      const int src = first + ((lane + 32 * t) >> (LOG_TOK - lp)), j = (lane + 32 * t) & (pitch - 1);
      const uint32_t page = __shfl_sync(0xffffffffu, pc_page, src);
      const uint32_t at = __shfl_sync(0xffffffffu, pc_off, src) + j;
      cp_mask[t] = __ballot_sync(0xffffffffu, j < __shfl_sync(0xffffffffu, pc_n, src));
      cp_ks[t] = k_scale + (uint64_t)page * p.ksp + (uint64_t)at * p.kst;
      cp_vs[t] = v_scale + (uint64_t)page * p.vsp + (uint64_t)at * p.vst;
    }
    cp_page = __shfl_sync(0xffffffffu, pc_page, first + lane);
    cp_off = __shfl_sync(0xffffffffu, pc_off, first + lane);
  };
  // Copies so far: the i-th fills box i % 2. Warps other than a row's first count
  // from 2^30, which p.give_up never is.
  uint32_t started = wid == 0 ? 0 : 1u << 30;
  auto copy = [&](const CUtensorMap* map, int s) {
    const uint32_t bar = bars + 8 * s;
    ++started;
    if (lane == 0) farq::mbar_arrive_expect_tx(bar, cp_bytes);
    if (lp != 0) __syncwarp();  // other lanes copy too
    if (copies) {
      const uint32_t dst = farq::smem_u32(ring) + s * (uint32_t)L::box + lane * pitch * ROWB;
#pragma unroll
      for (int hh = 0; hh < NH; ++hh) tma_load(dst + hh * TOK * 128, map, hh * 128, cp_off, h, cp_page, bar);
    }
  };
  // Scales of this lane's tokens; zeros, and no access, where there are none.
  auto copy_scales = [&] {
#pragma unroll
    for (int t = 0; t < LT; ++t) {
      const bool valid = (cp_mask[t] >> lane) & 1;
      const uint32_t dst = farq::smem_u32(scales + 32 * t + lane), bytes = valid ? 4 : 0;
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(valid ? cp_ks[t] : k_scale), "r"(bytes)
                   : "memory");
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst + TOK * 4), "l"(valid ? cp_vs[t] : v_scale),
                   "r"(bytes)
                   : "memory");
    }
  };
  float qs = 0.f;  // softmax_scale * log2(e) over the factor of the queries
  // Value scales above it take the wide form of the loop: all, where heads have powers of
  // their own (-1) or a wait is to be given up (the check is in that copy alone: in both
  // it cost 4 % of 1024 rows x 16 heads x 2048 tokens).
  float limit = p.give_up ? -2.f : kWide;
  // Factors of this lane's tokens: of their scores, the exponent and the
  // inverse of their value scales (in the wide form, what makes their weights NaN).
  // True if one of them has a scale above the limit, or one that is NaN.
  auto factors = [&](auto is_wide) {
    constexpr bool WIDE = decltype(is_wide)::value;
    bool above = false;
#pragma unroll
    for (int t = 0; t < LT; ++t) {
      const float ks = scales[32 * t + lane];
      float vs = scales[TOK + 32 * t + lane];
      vs = vs < kMinScale ? kMinScale : vs;
      above |= !(vs <= limit);
      const bool finite = vs <= 3.4028235e38f;
      tok[32 * t + lane] = WIDE ? make_float4(ks * qs, finite ? __log2f(vs) : 0.f, finite ? 0.f : vs - vs, 0.f)
                                : make_float4(ks * qs, __log2f(vs), rcp_approx(vs), 0.f);
    }
    return above;
  };
  // Rows that hold no token of the row: whatever lies there becomes zeros.
  auto clear = [&](uint8_t* box, const uint32_t (&mask)[LT]) {
    bool partial = false;
#pragma unroll
    for (int t = 0; t < LT; ++t) partial |= mask[t] != 0xffffffffu;
    if (!partial) return;
#pragma unroll
    for (int t = 0; t < LT; ++t)
      if (!((mask[t] >> lane) & 1)) {
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
          *reinterpret_cast<uint4*>(box + (i / 8) * TOK * 128 + (lane + 32 * t) * ROWB + (i % 8) * 16) =
              make_uint4(0, 0, 0, 0);
      }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
  };
  fetch();

  // Queries: lane (g, c) holds heads g, g + 8, values 32c + 16u + 4i .. + 3 of
  // each box (16c + 4i .. + 3 where D = 64), in the order of its key bytes.
  uint4 raw[NB][NH][NU * 2];
#pragma unroll
  for (int x = 0; x < NB; ++x) {
    const bool in = g + 8 * x < rows;
    const uint8_t* src = p.q.row(b, qi, head0 + (in ? g + 8 * x : 0)) + c * (NU * 32);
#pragma unroll
    for (int hh = 0; hh < NH; ++hh)
#pragma unroll
      for (int i = 0; i < NU * 2; ++i) raw[x][hh][i] = in ? ld_stream(src + hh * 256 + i * 16) : make_uint4(0, 0, 0, 0);
  }

  // Tokens t < lim count: the causal limit and the sequence's length.
  if (pos < lim) lim = pos + 1;
  if (pos < 0) lim = 0;
  lim = min(lim, (int64_t)1 << 40);  // so that no product overflows
  look_up();
  // The first chunk.
  uint32_t mask[LT];
#pragma unroll
  for (int t = 0; t < LT; ++t) mask[t] = 0;
  more = lim > 0;
  if (more) prepare();
  bool have = more;  // a chunk to work on
  if (have) {
    copy(&k_map, 0);
    copy_scales();
    copy(&v_map, 1);
#pragma unroll
    for (int t = 0; t < LT; ++t) mask[t] = cp_mask[t];
  }

  // In fp16, times the power of two that brings the CTA's largest finite value,
  // or each head's, into [2^14, 2^15).
  uint32_t qf[QSMEM ? 1 : D / 16][NB][2];
  {
    // The largest magnitude is the largest of the bits without the sign; one
    // that is not finite is left out, value by value.
    constexpr int MANTISSA = Half16<T>::kInf == 0x7f80u ? 7 : 10;  // bits
    uint32_t head[NB], all, low;  // largest of a lane's (then of a head's), of all; the least of those that are not 0
    auto ends = [&] {
      all = 0;
      low = 0xffffu;
#pragma unroll
      for (int x = 0; x < NB; ++x) {
        all = max(all, head[x]);
        low = min(low, head[x] - 1);
      }
      all = __reduce_max_sync(0xffffffffu, all);
      low = __reduce_min_sync(0xffffffffu, low) + 1;
    };
    auto largest = [&](auto all_finite) {
#pragma unroll
      for (int x = 0; x < NB; ++x) {
        uint32_t bits = 0;
#pragma unroll
        for (int hh = 0; hh < NH; ++hh)
#pragma unroll
          for (int i = 0; i < NU * 2; ++i) {
            const uint4& v = raw[x][hh][i];
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              uint32_t u = w[e] & 0x7fff7fffu;
              if (!decltype(all_finite)::value) {
                if ((u & 0xffffu) >= Half16<T>::kInf) u &= 0xffff0000u;
                if ((u >> 16) >= Half16<T>::kInf) u &= 0xffffu;
              }
              bits = __vmaxu2(bits, u);
            }
          }
        head[x] = max(bits & 0xffffu, bits >> 16);
      }
      ends();
    };
    auto exponent = [](uint32_t bits) {
      return max((int)(__float_as_uint(Half16<T>::unpack(bits).x) >> 23) - 127, -100);
    };
    auto power = [](int e) { return __uint_as_float((uint32_t)(e + 127) << 23); };
    auto convert = [&](const float (&up)[NB]) {
#pragma unroll
      for (int x = 0; x < NB; ++x)
#pragma unroll
        for (int hh = 0; hh < NH; ++hh)
#pragma unroll
          for (int i = 0; i < NU * 2; ++i) {
            float f[8];
            unpack8<T>(raw[x][hh][i], f);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int ks = (hh * NU * 2 + i) * 2 + e;
              const uint32_t b0 = Half16<__half>::pack(f[4 * e] * up[x], f[4 * e + 1] * up[x]);
              const uint32_t b1 = Half16<__half>::pack(f[4 * e + 2] * up[x], f[4 * e + 3] * up[x]);
              if (QSMEM) {
                if (warp == 0)
                  *reinterpret_cast<uint2*>(smem + L::qf + ((ks * NB + x) * 32 + lane) * 8) = make_uint2(b0, b1);
              } else {
                qf[QSMEM ? 0 : ks][x][0] = b0;
                qf[QSMEM ? 0 : ks][x][1] = b1;
              }
            }
          }
    };
    // More than 2^8 apart? Lanes first, and where they are, the heads, which four lanes hold.
    auto apart = [&] { return (all >> MANTISSA) > (low >> MANTISSA) + 8; };
    largest(std::true_type{});
    if (all >= Half16<T>::kInf || apart()) {
      largest(std::false_type{});
#pragma unroll
      for (int x = 0; x < NB; ++x)
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) head[x] = max(head[x], __shfl_xor_sync(0xffffffffu, head[x], o));
      ends();
    }
    float up[NB];
    if (apart()) {
      limit = -1.f;
      // A head's own power is 2^(14 - ex); its scores are taken times 2^(ex - least), at
      // most 2^96 (a score before the scales is below 2^32), and qs times the rest.
      const int least = max(exponent(all) - 96, 0);
#pragma unroll
      for (int x = 0; x < NB; ++x) {
        const int ex = exponent(head[x]);
        up[x] = power(14 - ex);
        if (c == 0) reinterpret_cast<float*>(smem + L::ml)[warp * 2 * R + g + 8 * x] = ldexpf(1.f, ex - least);
      }
      qs = p.scale * power(least - 14);
      convert(up);
    } else {
#pragma unroll
      for (int x = 0; x < NB; ++x) up[x] = all != 0 ? power(14 - exponent(all)) : 1.f;
      qs = p.scale / up[0];
      convert(up);
    }
    if (QSMEM) __syncthreads();
  }

  float o[NT][NB][4];
  float ref[NB][2];  // M - kLift of heads 2c, 2c + 1 (+ 8x)
  f32x2 l[NB], from[NB];  // sums of weights; -ref
#pragma unroll
  for (int x = 0; x < NB; ++x) {
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][x][e] = 0.f;
    ref[x][0] = ref[x][1] = -INFINITY;
    l[x] = 0;
    from[x] = 0;
  }
  bool failed = false;

  // Row r of a 16-row tile is token 4 (r / 2) + r % 2 for r < 8, two further for
  // r + 8: so the weights come out in the order of the transposed values, of
  // which a lane gets four tokens in a row.
  const int g0 = 4 * (g >> 1) + (g & 1);
  const int vr = lane & 15;  // this lane's row of a tile of values, and its 16-byte unit
  const uint32_t vaddr = farq::smem_u32(ring) + (uint32_t)L::box + vr * ROWB +
                         (((lane >> 4) ^ (D == 64 ? (vr >> 1) & 3 : vr & 7)) << 4);
  uint8_t* const kbox = ring;
  uint8_t* const vbox = ring + L::box;
  uint32_t parity = 0;
  // Works on chunks until none is left, or, where it is not `wide`, one holds a
  // value scale above the limit: then true, and the wide copy begins with that chunk
  // anew, its keys still in their box and the next chunk's addresses at hand. One
  // loop with both forms of the sums was 4 % slower (1024 rows x 16 heads x 2048 tokens).
  auto work = [&](auto is_wide) -> bool {
    constexpr bool WIDE = decltype(is_wide)::value;
    for (bool again = WIDE; have; parity ^= 1) {
      // this chunk's factors, the next chunk's addresses
      asm volatile("cp.async.wait_all;" ::: "memory");
      const bool above = factors(is_wide);
      if (more && !again) prepare();
      again = false;
      // a wait that runs out ends the loop before the next copy
      failed = (WIDE && started == p.give_up) || !farq::mbar_wait_bounded(bars, parity, kAttnWaitNs);
      clear(kbox, mask);

      // scores of tiles of 16 tokens
      float sc[NS][NB][4];
#pragma unroll
      for (int hh = 0; hh < NH; ++hh)
#pragma unroll
        for (int u = 0; u < NU; ++u) {
          uint4 kw[2 * NS];  // key rows, two of each tile
#pragma unroll
          for (int j = 0; j < 2 * NS; ++j) {
            const int row = 16 * (j >> 1) + 2 * (j & 1) + g0;
            const uint32_t at = D == 64 ? row * 64 + ((c ^ ((row >> 1) & 3)) << 4)
                                        : hh * TOK * 128 + row * 128 + (((2 * c + u) ^ (row & 7)) << 4);
            kw[j] = *reinterpret_cast<const uint4*>(kbox + at);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int ks = (hh * NU + u) * 4 + i;
            uint32_t bq[NB][2];
#pragma unroll
            for (int x = 0; x < NB; ++x) {
              if (QSMEM) {
                const uint2 v = *reinterpret_cast<const uint2*>(smem + L::qf + ((ks * NB + x) * 32 + lane) * 8);
                bq[x][0] = v.x;
                bq[x][1] = v.y;
              } else {
                bq[x][0] = qf[QSMEM ? 0 : ks][x][0];
                bq[x][1] = qf[QSMEM ? 0 : ks][x][1];
              }
            }
#pragma unroll
            for (int t = 0; t < NS; ++t) {
              const uint4 &lo = kw[2 * t], &hi = kw[2 * t + 1];
              uint32_t a[4];
              decode_pairs<E4M3>(i == 0 ? lo.x : i == 1 ? lo.y : i == 2 ? lo.z : lo.w, a[0], a[2]);
              decode_pairs<E4M3>(i == 0 ? hi.x : i == 1 ? hi.y : i == 2 ? hi.z : hi.w, a[1], a[3]);
#pragma unroll
              for (int x = 0; x < NB; ++x) {
                if (hh + u + i == 0)
                  mma16816_first(sc[t][x], a, bq[x][0], bq[x][1]);
                else
                  mma16816(sc[t][x], a, bq[x][0], bq[x][1]);
              }
            }
          }
        }
      __syncwarp();  // the keys and the scales are read, the factors written
      if (__any_sync(0xffffffffu, failed || (above && !WIDE))) return !__any_sync(0xffffffffu, failed);
      if (more) {
        copy(&k_map, 0);
        copy_scales();
      }

      // exponents of heads 2c, 2c + 1. M moves when a lane sees a value well above
      // it; until then nothing has to be exchanged between lanes.
      f32x2 a[2 * NS][NB];
      float inv[2 * NS], m[NB][2];
      bool partial = false;
#pragma unroll
      for (int t = 0; t < LT; ++t) partial |= mask[t] != 0xffffffffu;
      auto factor = [&](int j) { return tok[16 * (j >> 1) + 2 * (j & 1) + g0]; };
      if (WIDE) {  // the heads' own powers of two
#pragma unroll
        for (int x = 0; x < NB; ++x) {
          const float2 own = reinterpret_cast<const float2*>(smem + L::ml)[warp * R + c + 4 * x];
#pragma unroll
          for (int t = 0; t < NS; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[t][x][e] *= e & 1 ? own.y : own.x;
        }
      }
#pragma unroll
      for (int j = 0; j < 2 * NS; ++j) {
        const float4 f = factor(j);
        inv[j] = f.z;
#pragma unroll
        for (int x = 0; x < NB; ++x)
          a[j][x] =
              fma2(pair(sc[j >> 1][x][(j & 1) * 2], sc[j >> 1][x][(j & 1) * 2 + 1]), pair(f.x, f.x), pair(f.y, f.y));
      }
      if (partial) {
#pragma unroll
        for (int j = 0; j < 2 * NS; ++j)
#pragma unroll
          for (int x = 0; x < NB; ++x)
            if (!((mask[j / 4] >> (16 * ((j >> 1) & 1) + 2 * (j & 1) + g0)) & 1)) a[j][x] = pair(-INFINITY, -INFINITY);
      }
      bool moves = false;
#pragma unroll
      for (int x = 0; x < NB; ++x) {
        m[x][0] = m[x][1] = -INFINITY;
#pragma unroll
        for (int j = 0; j < 2 * NS; j += 2) {
          const float2 v = both(a[j][x]), w = both(a[j + 1][x]);
          m[x][0] = max3(m[x][0], v.x, w.x);
          m[x][1] = max3(m[x][1], v.y, w.y);
        }
        moves |= m[x][0] >= ref[x][0] + (kLift + kLag) || m[x][1] >= ref[x][1] + (kLift + kLag);
      }
      if (__any_sync(0xffffffffu, moves)) {
#pragma unroll
        for (int x = 0; x < NB; ++x) {
          float f[2], h[2];  // h: in the wide form, its root
#pragma unroll
          for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int y = 4; y <= 16; y <<= 1) m[x][e] = fmaxf(m[x][e], __shfl_xor_sync(0xffffffffu, m[x][e], y));
            const float top = fmaxf(ref[x][e], m[x][e] - kLift);
            f[e] = ref[x][e] == top ? 1.f : exp2_approx(ref[x][e] - top);
            if (WIDE) h[e] = ref[x][e] == top ? 1.f : exp2_approx(0.5f * (ref[x][e] - top));
            ref[x][e] = top;
          }
          l[x] = WIDE ? mul2(mul2(l[x], pair(h[0], h[1])), pair(h[0], h[1])) : mul2(l[x], pair(f[0], f[1]));
          from[x] = pair(ref[x][0] == -INFINITY ? 0.f : -ref[x][0], ref[x][1] == -INFINITY ? 0.f : -ref[x][1]);
#pragma unroll
          for (int i = 0; i < NT; ++i) {
            o[i][x][0] *= f[0];
            o[i][x][1] *= f[1];
            o[i][x][2] *= f[0];
            o[i][x][3] *= f[1];
          }
        }
      }
      // weights, as the columns of the second product: rows 2c, 2c + 1 of head g
      uint32_t pw[2 * NS][NB];
#pragma unroll
      for (int x = 0; x < NB; ++x)
#pragma unroll
        for (int j = 0; j < 2 * NS; ++j) {
          const float2 e = both(add2(a[j][x], from[x]));
          float w0 = exp2_approx(e.x), w1 = exp2_approx(e.y);
          if (WIDE) {
            const float4 f = factor(j);
            const float lv = f.y - kSumLift;
            l[x] = add2(l[x], pair(exp2_approx(e.x - lv), exp2_approx(e.y - lv)));
            w0 += f.z;  // 0 or NaN
            w1 += f.z;
          } else {
            l[x] = fma2(pair(w0, w1), pair(inv[j], inv[j]), l[x]);
          }
          pw[j][x] = transpose8x8(Half16<__half>::pack(w0, w1));
        }

      failed = (WIDE && started == p.give_up) || !farq::mbar_wait_bounded(bars + 8, parity, kAttnWaitNs);
      clear(vbox, mask);
      // values times weights: rows g and g + 8 of output tile y are values 16y + g and 16y + g + 8
#pragma unroll
      for (int t = 0; t < NS; ++t)
#pragma unroll
        for (int hh = 0; hh < NH; ++hh)
#pragma unroll
          for (int y = 0; y < NT / NH; y += 2) {
            uint32_t w[4];
            load_transposed(w, (vaddr + t * 16 * ROWB + hh * TOK * 128) ^ (y << 4));
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              uint32_t a[4];
              decode_pairs<E4M3>(w[2 * e], a[0], a[2]);
              decode_pairs<E4M3>(w[2 * e + 1], a[1], a[3]);
#pragma unroll
              for (int x = 0; x < NB; ++x) mma16816(o[hh * 8 + y + e][x], a, pw[2 * t][x], pw[2 * t + 1][x]);
            }
          }
      __syncwarp();  // the values and the factors are read
      if (__any_sync(0xffffffffu, failed)) return false;
      have = more;
      if (more) copy(&v_map, 1);
#pragma unroll
      for (int t = 0; t < LT; ++t) mask[t] = cp_mask[t];
    }
    return false;
  };
  const bool wide = work(std::false_type{});
  if (wide) {
#pragma unroll
    for (int x = 0; x < NB; ++x) {
      l[x] = mul2(l[x], pair(kSumUp, kSumUp));
      if (limit != -1.f && c == 0) reinterpret_cast<float*>(smem + L::ml)[warp * 2 * R + g + 8 * x] = 1.f;
    }
    __syncwarp();
    work(std::true_type{});
  }
  bool drained = true;
  if (__any_sync(0xffffffffu, failed)) {
    // A copy did not arrive: wait (bounded) for those in flight, at most the last two
    // of the two and more that were started; set the status and give NaN.
    for (uint32_t i = started - 2; i < started; ++i)
      drained &= farq::mbar_wait_bounded(bars + 8 * (i % 2), (i / 2) & 1, kAttnWaitNs);
    drained = __all_sync(0xffffffffu, drained);
    if (lane == 0 && p.status) atomicExch(p.status, (int)DSA_KV_ERR_DEVICE_TIMEOUT);
#pragma unroll
    for (int x = 0; x < NB; ++x) l[x] = pair(__int_as_float(0x7fc00000), __int_as_float(0x7fc00000));
  }
  asm volatile("cp.async.wait_all;" ::: "memory");

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // Partial results into the warp's own ring, whose copies are all done. Where one is
  // still out after the second wait, the ring stays as it is: the join makes NaN of it.
  float* const ml = reinterpret_cast<float*>(smem + L::ml);
  float* const part = reinterpret_cast<float*>(smem + L::ring + (size_t)warp * L::region);
#pragma unroll
  for (int x = 0; x < NB; ++x)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float sum = e ? both(l[x]).y : both(l[x]).x;
#pragma unroll
      for (int y = 4; y <= 16; y <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, y);
      const int row = 2 * c + e + 8 * x;
      if (g == 0) {
        // Tokens whose scores are all -inf are not the same as none.
        ml[warp * 2 * R + row] = ref[x][e] == -INFINITY && (started << 2) != 0 ? -3.4028235e38f : ref[x][e];
        ml[warp * 2 * R + R + row] = wide ? sum : sum * kSumUp;
      }
    }
  if (drained) {  // around all stores: asked row by row it cost 2 to 4 %
#pragma unroll
    for (int x = 0; x < NB; ++x)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = 2 * c + e + 8 * x;
#pragma unroll
        for (int y = 0; y < NT; ++y) {
          part[row * D + ((16 * y + g) ^ (c << 3))] = o[y][x][e];
          part[row * D + ((16 * y + 8 + g) ^ (c << 3))] = o[y][x][2 + e];
        }
      }
  }
  // Join. out = sum_n w_n o_n / sum_n w_n l_n over the warps, w_n = 2^(M_n - max).
  constexpr int LPR = kAttnThreads / R;  // lanes of a head: 16 or 8
  // total + w l, with w = 2^d
  auto add_sum = [](float total, float l, float w, float d) {
    const float h = exp2_approx(0.5f * d);
    return d < kTwoSteps ? fmaf(h * l, h, total) : fmaf(w, l, total);
  };
  auto finish = [&](float m, float total) { return m == -INFINITY && total == 0.f ? 0.f : 1.0f / total; };
  auto put_lse = [&](int row, float m, float total) {
    p.lse[((int64_t)b * p.Q.d + qi) * p.H.d * p.G + head0 + row] =
        total == 0.f ? -INFINITY : (m + log2f(total)) * 0.69314718055994531f;
  };
  auto store = [&](int row, int f4, const float4& acc, float f) {
    uint2 v;
    v.x = Half16<T>::pack(acc.x * f, acc.y * f);
    v.y = Half16<T>::pack(acc.z * f, acc.w * f);
    *reinterpret_cast<uint2*>(p.out.row(b, qi, head0 + row) + f4 * 8) = v;
  };
  if (C == 1) {
    // Every thread works the weights of its head out for itself: 0.4 us less than
    // weights by groups of lanes and a barrier.
    __syncthreads();
    const int row = threadIdx.x / LPR, sub = threadIdx.x % LPR;
    if (row >= rows) return;
    float w[W], m = -INFINITY, total = 0.f;
#pragma unroll
    for (int n = 0; n < W; ++n) {
      w[n] = ml[n * 2 * R + row];
      m = fmaxf(m, w[n]);
    }
    const float from_all = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int n = 0; n < W; ++n) {
      const float d = w[n] - from_all;
      w[n] = exp2_approx(d);
      total = add_sum(total, ml[n * 2 * R + R + row], w[n], d);
    }
    total *= 1.f / kSumUp;
    const float f = finish(m, total);
#pragma unroll
    for (int k = 0; k < D / 4 / LPR; ++k) {
      const int f4 = sub + k * LPR, at = part_index<D>(row, f4);
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int n = 0; n < W; ++n) {
        const float4 v = reinterpret_cast<const float4*>(smem + L::ring + n * L::region)[at];
        acc.x = fmaf(w[n], v.x, acc.x);
        acc.y = fmaf(w[n], v.y, acc.y);
        acc.z = fmaf(w[n], v.z, acc.z);
        acc.w = fmaf(w[n], v.w, acc.w);
      }
      store(row, f4, acc, f);
    }
    if (sub == 0 && p.lse) put_lse(row, m, total);
    return;
  }

  // Every CTA of the cluster works out the weights of all NW warps, a group of
  // lanes per head, and then its share of the output, as many lanes to four values
  // as there are to spare. (A thread per head and per four values took 2 us longer
  // with 32 warps: each walked through all of them.)
  cluster_arrive();
  cluster_wait();
  float* const all = reinterpret_cast<float*>(smem + L::all);
  float* const fin = reinterpret_cast<float*>(smem + L::fin);
  // Four values go to 2^log_lanes lanes. Where a lane has few partial results,
  // they are on their way while the weights are worked out (8 rows of 4 heads over
  // 2048 tokens, D = 128: 7.0 instead of 7.6 us; where several clusters share an SM it
  // costs more than it hides, 32 rows over 4096 tokens 12.6 instead of 12.1 us).
  constexpr int AHEAD = 8;
  const int units = rows * (D / 4), share = (units + (int)C - 1) >> (__ffs(C) - 1);
  int log_lanes = 0;
  while (log_lanes < 4 && (2u << log_lanes) <= NW && (share << (log_lanes + 1)) <= kAttnThreads) ++log_lanes;
  const uint32_t first_n = threadIdx.x & ((1u << log_lanes) - 1);
  const bool few = log_lanes > 0 && (NW >> log_lanes) <= AHEAD;
  float4 ahead[AHEAD];
  if (few) {
    const int at = (int)(threadIdx.x >> log_lanes), i = rank * share + at;
    const bool mine = at < share && i < units;
    const uint32_t off = base + (uint32_t)L::ring + (mine ? part_index<D>(i / (D / 4), i % (D / 4)) * 16 : 0);
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const uint32_t n = first_n + ((uint32_t)k << log_lanes);
      if (n < NW) ahead[k] = ld_cluster4(mapa(off + (n % W) * (uint32_t)L::region, n / W));
    }
  }
  {
    constexpr int MOST = kMaxCluster * W / LPR;
    const int row = threadIdx.x / LPR;
    const uint32_t sub = threadIdx.x % LPR;
    float top[MOST], sum[MOST], m = -INFINITY;
#pragma unroll
    for (int i = 0; i < MOST; ++i) {
      const uint32_t n = sub + i * LPR;
      top[i] = -INFINITY;
      sum[i] = 0.f;
      if (n < NW) {
        const uint32_t at = mapa(base + (uint32_t)L::ml + ((n % W) * 2 * R + row) * 4, n / W);
        top[i] = ld_cluster(at);
        sum[i] = ld_cluster(at + R * 4);
      }
      m = fmaxf(m, top[i]);
    }
#pragma unroll
    for (int y = 1; y < LPR; y <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, y));
    const float from_all = m == -INFINITY ? 0.f : m;
    float total = 0.f;
#pragma unroll
    for (int i = 0; i < MOST; ++i) {
      const uint32_t n = sub + i * LPR;
      const float d = top[i] - from_all, w = exp2_approx(d);
      total = add_sum(total, sum[i], w, d);
      if (n < NW) all[n * R + row] = w;
    }
#pragma unroll
    for (int y = 1; y < LPR; y <<= 1) total += __shfl_xor_sync(0xffffffffu, total, y);
    total *= 1.f / kSumUp;
    if (sub == 0) {
      fin[row] = finish(m, total);
      if (p.lse && rank == 0 && row < rows) put_lse(row, m, total);
    }
  }
  __syncthreads();
  for (int i0 = 0; i0 < share; i0 += kAttnThreads >> log_lanes) {
    const int at = i0 + (int)(threadIdx.x >> log_lanes), i = rank * share + at;
    const bool mine = at < share && i < units;
    const int row = mine ? i / (D / 4) : 0, f4 = mine ? i % (D / 4) : 0;
    const uint32_t off = base + (uint32_t)L::ring + part_index<D>(row, f4) * 16;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](uint32_t n, const float4& v) {
      const float w = all[n * R + row];
      acc.x = fmaf(w, v.x, acc.x);
      acc.y = fmaf(w, v.y, acc.y);
      acc.z = fmaf(w, v.z, acc.z);
      acc.w = fmaf(w, v.w, acc.w);
    };
    if (few) {
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        const uint32_t n = first_n + ((uint32_t)k << log_lanes);
        if (n < NW) add(n, ahead[k]);
      }
    } else {
#pragma unroll 4
      for (uint32_t n = first_n; n < NW; n += 1u << log_lanes)
        add(n, ld_cluster4(mapa(off + (n % W) * (uint32_t)L::region, n / W)));
    }
    // shared memory stays until every CTA has read it
    if (i0 + (kAttnThreads >> log_lanes) >= share) cluster_arrive();
    for (int y = 1; y < 1 << log_lanes; y <<= 1) {
      acc.x += __shfl_xor_sync(0xffffffffu, acc.x, y);
      acc.y += __shfl_xor_sync(0xffffffffu, acc.y, y);
      acc.z += __shfl_xor_sync(0xffffffffu, acc.z, y);
      acc.w += __shfl_xor_sync(0xffffffffu, acc.w, y);
    }
    if (mine && first_n == 0) store(row, f4, acc, fin[row]);
  }
  cluster_wait();
}

}  // namespace kv
