// kv_attn_kernel.cuh — attention of query rows over selected blocks of the
// quantised paged cache (dsa_kv_attn_launch, include/dsa_kv.h).
//
// A row (b, h, q) has G query heads that share a key head and a selection.
// Up to 16 of them are the rows of one m16n8k16 tensor-core tile, on which a
// CTA works. The row's selected tokens are cut into chunks of 32, dealt to the
// warps in turn; every warp runs the one-pass softmax on its own chunks and
// the partial results are joined at the end through shared memory.
//
// Mathematics, per query head, tokens t with key codes k, value codes v and
// their scales ks, vs:
//     a_t = log2(e) * scale * ks_t * (q.k_t) + log2(vs_t)
//     o   = sum_t 2^(a_t - M) v_t,   l = sum_t 2^(a_t - M) / vs_t
//     out = o / l,   lse = ln 2 * (M + log2 l)
// with M the running maximum of a_t. The value scale sits in the exponent, so
// the weight of a token is at most 1 whatever the scales are, the products
// run on raw codes (exact in fp16), and the maximum bounds each term of o.
//
// Precision: q is brought to fp16 by one power of two for the whole tile, its
// largest value in [2^14, 2^15): bf16 values lose bits only 2^-28 below it.
// Weights are fp16 too, times 2^6: 2^-11 relative (the output's own half step
// is 2^-9 or 2^-12) down to 2^-20, with an absolute 2^-31 below. M lags behind
// the maximum by up to 8 (a weight is at most 2^14), so that o is rescaled
// only when the maximum really moves. Sums are fp32 throughout.
//
// Data movement: a chunk's key rows and value rows come by one TMA copy each
// into a slot of the warp's own ring of S slots, so that no CTA barrier is
// needed on the way and S - 1 chunks per warp stay in flight. Rows are 128
// bytes (64 for D = 64), swizzled by the copy, which makes the 16-byte fragment
// reads free of bank conflicts: lane (g, c) of a warp reads 32 contiguous
// bytes of key row g for the products over D, whose order of summation is free
// to choose, and 16 bytes of value rows 2c, 2c+1, 2c+8, 2c+9 for the products
// over tokens, which are transposed pair by pair with byte permutes.
#pragma once

#include <cuda.h>

#include "farq_kernel.cuh"
#include "kv_common.cuh"

namespace kv {

constexpr int kTok = 32;           // tokens of a chunk
constexpr int kRows = 16;          // query heads of a tile
constexpr int kAttnWarps = 4;      // warps of a CTA
constexpr float kLift = 6.0f;      // weights are 2^(a - M + kLift)
constexpr float kLag = 8.0f;       // M is moved when a maximum exceeds it by more
constexpr uint64_t kAttnWaitNs = 2000000000ull;

struct AttnParams {
  Dense q, out;
  float* lse;  // may be null
  const float* k_scale;
  const float* v_scale;
  int64_t ksp, ksh, kst, vsp, vsh, vst;  // scale strides (page, head, token)
  const void* blocks;
  const void* pages;
  int64_t bsb, bsh, bsq, psb, psh, psq;  // strides of blocks and pages (b, h, q)
  const void* q_pos;
  const void* kv_lens;
  FastDiv MT, Q, H;     // tiles of 16 query heads per row, rows
  FastDiv per_block;    // chunks of a block
  int64_t P;
  uint32_t items;       // chunks of a row
  int32_t G, K, bs;
  int32_t log_pieces;   // a chunk holds 2^log_pieces blocks (blocks of at most 16 tokens)
  uint32_t box_bytes;   // bytes of one copied box
  int32_t block_bytes, page_bytes, pos_bytes;
  float scale;          // softmax_scale * log2(e)
};

// Shared-memory carve-up, identical on host and device.
template <int D, int S>
struct AttnSmem {
  static constexpr int W = kAttnWarps;
  static constexpr size_t side = (size_t)kTok * D;  // one side of a slot
  static constexpr size_t ring = 0;
  static constexpr size_t scales = ring + (size_t)W * S * 2 * side;
  static constexpr size_t tok = scales + (size_t)W * S * 2 * kTok * 4;
  static constexpr size_t flag = tok + (size_t)W * 3 * kTok * 4;
  static constexpr size_t bars = flag + (size_t)W * S * kTok * 4;
  static constexpr size_t ml = bars + (size_t)W * S * 8;        // [W][2][16] maxima and sums, then weights
  static constexpr size_t fin = ml + (size_t)W * 2 * kRows * 4;  // [16] 1 / l
  static constexpr size_t qf = fin + kRows * 4;
  static constexpr size_t total = qf + (D == 256 ? (size_t)(D / 16) * 32 * 16 : 0);
};

__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int x, int tok, int head, int page,
                                         uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(map), "r"(x), "r"(tok), "r"(head), "r"(page), "r"(bar)
      : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(a)
               : "memory");
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory");
  return v;
}
// c += a * b for one m16n8k16 tile, fp16 operands, fp32 sums.
__device__ __forceinline__ void mma16816(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9},"
      " {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Four codes -> two pairs of fp16 values (bytes 0, 1 and bytes 2, 3).
// int8: the byte with its sign flipped, under the exponent of 1024, is the
// fp16 number 1024 + 128 + code; both steps are exact.
template <bool E4M3>
__device__ __forceinline__ void decode_pairs(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if (E4M3) {
    lo = e4m3x2_to_half2((uint16_t)w);
    hi = e4m3x2_to_half2((uint16_t)(w >> 16));
  } else {
    const uint32_t s = w ^ 0x80808080u, bias = 0x64806480u;
    const uint32_t a = __byte_perm(s, 0x64646464u, 0x4140), b = __byte_perm(s, 0x64646464u, 0x4342);
    const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&bias));
    const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&b), *reinterpret_cast<const __half2*>(&bias));
    lo = *reinterpret_cast<const uint32_t*>(&x);
    hi = *reinterpret_cast<const uint32_t*>(&y);
  }
}

// Place of float4 `f4` of row `row` in a warp's partial result: the units of a
// row are permuted so that the writes of a quarter warp spread over the banks.
template <int D>
__device__ __forceinline__ int part_index(int row, int f4) {
  const int c = D == 64 ? (f4 >> 2) & 3 : (f4 >> 3) & 3;
  return row * (D / 4) + (f4 ^ ((c * 2 + (row & 1)) & 7));
}

template <typename T, int D, bool E4M3, int S>
__global__ void __launch_bounds__(kAttnWarps * 32)
    attn_kernel(const AttnParams p, const __grid_constant__ CUtensorMap k_map,
                const __grid_constant__ CUtensorMap v_map) {
  using L = AttnSmem<D, S>;
  constexpr int W = kAttnWarps;
  constexpr int NH = D == 256 ? 2 : 1;    // boxes of at most 128 bytes per side
  constexpr int NU = D == 64 ? 1 : 2;     // 16-byte pieces of a key row per lane and box
  constexpr int NT = D / 8;               // 8-wide column tiles of the output
  constexpr int ROWB = D == 64 ? 64 : 128;
  constexpr bool QSMEM = D == 256;        // q fragments in shared memory (registers hold the output)
  extern __shared__ __align__(1024) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  uint32_t r = blockIdx.x, mt, qi, h, b;
  p.MT.divmod(r, &r, &mt);
  p.Q.divmod(r, &r, &qi);
  p.H.divmod(r, &b, &h);
  const int head0 = (int)h * p.G + (int)mt * kRows;
  const int rows = min(kRows, p.G - (int)mt * kRows);

  const uint32_t base = farq::smem_u32(smem);
  const uint32_t slots = base + (uint32_t)L::ring + warp * (uint32_t)(S * 2 * L::side);
  const uint32_t bars = base + (uint32_t)L::bars + warp * S * 8;
  float* const scales = reinterpret_cast<float*>(smem + L::scales) + warp * S * 2 * kTok;
  float* const tok = reinterpret_cast<float*>(smem + L::tok) + warp * 3 * kTok;
  uint32_t* const flags = reinterpret_cast<uint32_t*>(smem + L::flag) + warp * S * kTok;
  if (lane == 0) {
    for (int s = 0; s < S; ++s) farq::mbar_init(bars + 8 * s, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  __syncwarp();
  pdl_wait();

  // Tokens t < lim count: the causal limit and the sequence's length.
  const int64_t pos = load_index(p.q_pos, (int64_t)b * p.Q.d + qi, p.pos_bytes);
  int64_t lim = load_index(p.kv_lens, b, p.pos_bytes);
  if (pos < lim) lim = pos + 1;
  if (pos < 0) lim = 0;
  lim = min(lim, (int64_t)1 << 40);  // so that no product below overflows
  const uint32_t items = lim > 0 ? p.items : 0;
  const uint32_t NW = W, wid = warp;
  const int64_t brow = b * p.bsb + h * p.bsh + qi * p.bsq;
  const int64_t prow = b * p.psb + h * p.psh + qi * p.psq;

  // The warp looks its chunks up 32 pieces at a time; a lane holds one piece:
  // page, first token within the page, valid tokens.
  const int lp = p.log_pieces, pitch = kTok >> lp;
  uint32_t next_k = 0, active = 0;
  int pc_page = 0, pc_off = 0, pc_n = 0;
  auto look_up = [&] {
    const uint32_t item = wid + (next_k + (lane >> lp)) * NW;
    next_k += 32 >> lp;
    uint32_t entry, sub = 0;
    if (lp == 0)
      p.per_block.divmod(item, &entry, &sub);
    else
      entry = (item << lp) + (lane & ((1 << lp) - 1));
    pc_n = 0;
    if (item < items && entry < (uint32_t)p.K) {
      const int64_t blk = load_index(p.blocks, brow + entry, p.block_bytes);
      const int64_t page = load_index(p.pages, prow + entry, p.page_bytes);
      if (blk >= 0 && blk < lim && page >= 0 && page < p.P) {
        const int64_t left = lim - (blk * p.bs + (int64_t)sub * kTok);
        const int most = min(kTok, p.bs - (int)sub * kTok);
        pc_n = left <= 0 ? 0 : left < most ? (int)left : most;
        pc_page = (int)page;
        pc_off = (int)sub * kTok;
      }
    }
    active = __ballot_sync(0xffffffffu, pc_n > 0);
    if (lp >= 1) active |= active >> 1;
    if (lp >= 2) active |= active >> 2;
    if (lp >= 1) active &= lp == 1 ? 0x55555555u : 0x11111111u;
  };
  // Starts the copies of the warp's next chunk into a slot; false when there is none.
  auto issue = [&](int s) -> bool {
    while (active == 0) {
      if (wid + next_k * NW >= items) return false;
      look_up();
    }
    const int first = __ffs(active) - 1;
    active &= active - 1;
    // scales, and whether the token counts, of this lane's token
    const int src = first + (lane >> (5 - lp)), j = lane & (pitch - 1);
    const int64_t page = __shfl_sync(0xffffffffu, pc_page, src);
    const int64_t at = __shfl_sync(0xffffffffu, pc_off, src) + j;
    const bool valid = j < __shfl_sync(0xffffffffu, pc_n, src);
    const float* ks = p.k_scale;
    const float* vs = p.v_scale;
    if (valid) {
      ks += page * p.ksp + h * p.ksh + at * p.kst;
      vs += page * p.vsp + h * p.vsh + at * p.vst;
    }
    const uint32_t sdst = farq::smem_u32(scales + s * 2 * kTok + lane), bytes = valid ? 4 : 0;
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(sdst), "l"(ks), "r"(bytes) : "memory");
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(sdst + kTok * 4), "l"(vs), "r"(bytes) : "memory");
    flags[s * kTok + lane] = valid;
    // one copy per piece and box, by the lane that holds the piece
    const int piece = lane - first;
    const bool copies = piece >= 0 && piece < (1 << lp) && pc_n > 0;
    const uint32_t n = __popc(__ballot_sync(0xffffffffu, copies));
    const uint32_t bar = bars + 8 * s;
    if (lane == first) farq::mbar_arrive_expect_tx(bar, n * 2 * NH * p.box_bytes);
    __syncwarp();
    if (copies) {
      const uint32_t dst = slots + s * (uint32_t)(2 * L::side) + piece * pitch * ROWB;
#pragma unroll
      for (int hh = 0; hh < NH; ++hh) {
        tma_load(dst + hh * kTok * 128, &k_map, hh * 128, pc_off, h, pc_page, bar);
        tma_load(dst + (uint32_t)L::side + hh * kTok * 128, &v_map, hh * 128, pc_off, h, pc_page, bar);
      }
    }
    return true;
  };

  uint32_t issued = 0;
  bool more = true;
#pragma unroll
  for (int s = 0; s < S; ++s) {
    if (more && (more = issue(s))) ++issued;
    asm volatile("cp.async.commit_group;" ::: "memory");
  }

  // The tile's q in fp16, as fragments of 16 values of D at a time: lane
  // (g, c) holds rows g and g + 8, values 32c + 16u + 4i .. + 3 of each box
  // (16c + 4i .. + 3 where D = 64), in the order of its key bytes.
  uint32_t qf[QSMEM ? 1 : D / 16][4];
  float qs;
  {
    uint4 raw[2][NH][NU * 2];
    float most = 0.f;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const bool in = g + 8 * x < rows;
      const uint8_t* src = p.q.row(b, qi, head0 + (in ? g + 8 * x : 0)) + c * (NU * 32);
#pragma unroll
      for (int hh = 0; hh < NH; ++hh)
#pragma unroll
        for (int i = 0; i < NU * 2; ++i) {
          raw[x][hh][i] = in ? ld_stream(src + hh * 256 + i * 16) : make_uint4(0, 0, 0, 0);
          float f[8];
          unpack8<T>(raw[x][hh][i], f);
#pragma unroll
          for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(f[e]) <= 3.4e38f ? fabsf(f[e]) : 0.f);
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    // the power of two that brings the largest finite value into [2^14, 2^15)
    const int ex = max((int)(__float_as_uint(most) >> 23) - 127, -100);
    const float up = most > 0.f ? __uint_as_float((uint32_t)(14 - ex + 127) << 23) : 1.f;
    qs = p.scale / up;
#pragma unroll
    for (int hh = 0; hh < NH; ++hh)
#pragma unroll
      for (int i = 0; i < NU * 2; ++i) {
        uint32_t w[2][4];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          float f[8];
          unpack8<T>(raw[x][hh][i], f);
#pragma unroll
          for (int e = 0; e < 4; ++e) w[x][e] = Half16<__half>::pack(f[2 * e] * up, f[2 * e + 1] * up);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int ks = (hh * NU * 2 + i) * 2 + e;
          const uint32_t a[4] = {w[0][2 * e], w[1][2 * e], w[0][2 * e + 1], w[1][2 * e + 1]};
          if (QSMEM) {
            if (warp == 0)
              *reinterpret_cast<uint4*>(smem + L::qf + (ks * 32 + lane) * 16) = make_uint4(a[0], a[1], a[2], a[3]);
          } else {
#pragma unroll
            for (int y = 0; y < 4; ++y) qf[QSMEM ? 0 : ks][y] = a[y];
          }
        }
      }
    if (QSMEM) __syncthreads();
  }

  float o[NT][4];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
  float M0 = -INFINITY, M1 = -INFINITY, l0 = 0.f, l1 = 0.f;
  bool failed = false;

  int s = 0;
  uint32_t parity = 0;
  for (uint32_t n = 0; n < issued; ++n) {
    const uint32_t kslot = slots + s * (uint32_t)(2 * L::side), vslot = kslot + (uint32_t)L::side;
    asm volatile("cp.async.wait_group %0;" ::"n"(S - 1) : "memory");
    // this lane's token: factor of its scores, exponent and inverse of its value scale
    const uint32_t valid = flags[s * kTok + lane];
    {
      const float ks = scales[s * 2 * kTok + lane];
      float vs = scales[s * 2 * kTok + kTok + lane];
      vs = vs < kMinScale ? kMinScale : vs;
      tok[lane] = ks * qs;
      tok[kTok + lane] = __log2f(vs);
      tok[2 * kTok + lane] = __frcp_rn(vs);
    }
    const uint32_t mask = __ballot_sync(0xffffffffu, valid != 0);
    if (!farq::mbar_wait_bounded(bars + 8 * s, parity, kAttnWaitNs)) failed = true;
    if (__any_sync(0xffffffffu, failed)) {
      failed = true;
      break;
    }
    if (mask != 0xffffffffu) {
      // rows that hold no token of the row: whatever lies there becomes zeros
      if (!valid) {
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          const uint32_t at = (i / 8) * kTok * 128 + lane * ROWB + (i % 8) * 16;
          asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(kslot + at), "r"(0) : "memory");
          asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(vslot + at), "r"(0) : "memory");
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      }
    }
    __syncwarp();

    // scores of 16 heads x 32 tokens
    float sc[4][4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) sc[j][e] = 0.f;
#pragma unroll
    for (int hh = 0; hh < NH; ++hh)
#pragma unroll
      for (int u = 0; u < NU; ++u) {
        uint4 kw[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t at = D == 64 ? (8 * j + g) * 64 + ((c ^ ((g >> 1) & 3)) << 4)
                                      : hh * kTok * 128 + (8 * j + g) * 128 + (((2 * c + u) ^ g) << 4);
          kw[j] = lds128(kslot + at);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int ks = (hh * NU + u) * 4 + i;
          uint32_t a[4];
          if (QSMEM) {
            const uint4 t = lds128(base + (uint32_t)L::qf + (ks * 32 + lane) * 16);
            a[0] = t.x; a[1] = t.y; a[2] = t.z; a[3] = t.w;
          } else {
#pragma unroll
            for (int y = 0; y < 4; ++y) a[y] = qf[QSMEM ? 0 : ks][y];
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t w = i == 0 ? kw[j].x : i == 1 ? kw[j].y : i == 2 ? kw[j].z : kw[j].w;
            uint32_t b0, b1;
            decode_pairs<E4M3>(w, b0, b1);
            mma16816(sc[j], a, b0, b1);
          }
        }
      }

    // weights; columns 2c, 2c + 1 of tile j are tokens 8j + 2c, 8j + 2c + 1
    float inv[4][2], m0 = -INFINITY, m1 = -INFINITY;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = *reinterpret_cast<const float2*>(tok + 8 * j + 2 * c);
      const float2 lv = *reinterpret_cast<const float2*>(tok + kTok + 8 * j + 2 * c);
      const float2 iv = *reinterpret_cast<const float2*>(tok + 2 * kTok + 8 * j + 2 * c);
      inv[j][0] = iv.x;
      inv[j][1] = iv.y;
      sc[j][0] = fmaf(sc[j][0], f.x, lv.x);
      sc[j][1] = fmaf(sc[j][1], f.y, lv.y);
      sc[j][2] = fmaf(sc[j][2], f.x, lv.x);
      sc[j][3] = fmaf(sc[j][3], f.y, lv.y);
      if (mask != 0xffffffffu) {
        const uint32_t bits = mask >> (8 * j + 2 * c);
        if (!(bits & 1)) sc[j][0] = sc[j][2] = -INFINITY;
        if (!(bits & 2)) sc[j][1] = sc[j][3] = -INFINITY;
      }
      m0 = fmaxf(m0, fmaxf(sc[j][0], sc[j][1]));
      m1 = fmaxf(m1, fmaxf(sc[j][2], sc[j][3]));
    }
#pragma unroll
    for (int x = 1; x <= 2; x <<= 1) {
      m0 = fmaxf(m0, __shfl_xor_sync(0xffffffffu, m0, x));
      m1 = fmaxf(m1, __shfl_xor_sync(0xffffffffu, m1, x));
    }
    if (__any_sync(0xffffffffu, m0 > M0 + kLag || m1 > M1 + kLag)) {
      const float n0 = fmaxf(M0, m0), n1 = fmaxf(M1, m1);
      const float f0 = M0 == n0 ? 1.f : exp2_approx(M0 - n0), f1 = M1 == n1 ? 1.f : exp2_approx(M1 - n1);
      M0 = n0;
      M1 = n1;
      l0 *= f0;
      l1 *= f1;
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        o[i][0] *= f0;
        o[i][1] *= f0;
        o[i][2] *= f1;
        o[i][3] *= f1;
      }
    }
    const float s0 = kLift - (M0 == -INFINITY ? 0.f : M0), s1 = kLift - (M1 == -INFINITY ? 0.f : M1);
    uint32_t pw[4][2];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float w0 = exp2_approx(sc[j][0] + s0), w1 = exp2_approx(sc[j][1] + s0);
      const float w2 = exp2_approx(sc[j][2] + s1), w3 = exp2_approx(sc[j][3] + s1);
      l0 = fmaf(w0, inv[j][0], fmaf(w1, inv[j][1], l0));
      l1 = fmaf(w2, inv[j][0], fmaf(w3, inv[j][1], l1));
      pw[j][0] = Half16<__half>::pack(w0, w1);
      pw[j][1] = Half16<__half>::pack(w2, w3);
    }

    // weights times values; column g of output tile x is value 16g + x of its box (8g + x where D = 64)
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const uint32_t a[4] = {pw[2 * t][0], pw[2 * t][1], pw[2 * t + 1][0], pw[2 * t + 1][1]};
#pragma unroll
      for (int hh = 0; hh < NH; ++hh) {
        constexpr int NWORD = D == 64 ? 2 : 4;
        uint32_t w[4][NWORD];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int row = 16 * t + 2 * c + (x & 1) + 8 * (x >> 1);
          if constexpr (D == 64) {
            const uint2 v = lds64(vslot + row * 64 + (((g >> 1) ^ c) << 4) + (g & 1) * 8);
            w[x][0] = v.x;
            w[x][1] = v.y;
          } else {
            const uint4 v = lds128(vslot + hh * kTok * 128 + row * 128 + ((g ^ (2 * c + (x & 1))) << 4));
            w[x][0] = v.x;
            w[x][1] = v.y;
            w[x][2] = v.z;
            w[x][3] = v.w;
          }
        }
#pragma unroll
        for (int i = 0; i < NWORD; ++i) {
          uint32_t b0[4], b1[4];
          decode_pairs<E4M3>(__byte_perm(w[0][i], w[1][i], 0x5140), b0[0], b0[1]);
          decode_pairs<E4M3>(__byte_perm(w[0][i], w[1][i], 0x7362), b0[2], b0[3]);
          decode_pairs<E4M3>(__byte_perm(w[2][i], w[3][i], 0x5140), b1[0], b1[1]);
          decode_pairs<E4M3>(__byte_perm(w[2][i], w[3][i], 0x7362), b1[2], b1[3]);
#pragma unroll
          for (int e = 0; e < 4; ++e) mma16816(o[hh * 16 + 4 * i + e], a, b0[e], b1[e]);
        }
      }
    }
    __syncwarp();  // the slot and the token factors are read
    if (more && (more = issue(s))) ++issued;
    asm volatile("cp.async.commit_group;" ::: "memory");
    if (++s == S) {
      s = 0;
      parity ^= 1;
    }
  }
  if (failed) {
    // A copy did not arrive: wait (bounded) for those in flight, give NaN.
    for (int t = 0; t < S; ++t) {
      (void)farq::mbar_wait_bounded(bars + 8 * s, parity, kAttnWaitNs);
      if (++s == S) {
        s = 0;
        parity ^= 1;
      }
    }
    l0 = l1 = __int_as_float(0x7fc00000);
  }
  asm volatile("cp.async.wait_all;" ::: "memory");

  // Partial results into the warp's own ring, whose copies are all done.
#pragma unroll
  for (int x = 1; x <= 2; x <<= 1) {
    l0 += __shfl_xor_sync(0xffffffffu, l0, x);
    l1 += __shfl_xor_sync(0xffffffffu, l1, x);
  }
  float4* const part = reinterpret_cast<float4*>(smem + L::ring + (size_t)warp * S * 2 * L::side);
  float* const ml = reinterpret_cast<float*>(smem + L::ml);
  if (c == 0) {
    float* const mine = ml + warp * 2 * kRows;
    mine[g] = M0;
    mine[g + 8] = M1;
    mine[kRows + g] = l0;
    mine[kRows + g + 8] = l1;
  }
#pragma unroll
  for (int x = 0; x < 2; ++x)
#pragma unroll
    for (int hh = 0; hh < NH; ++hh)
#pragma unroll
      for (int e = 0; e < 2; ++e) {  // columns 2c and 2c + 1
        constexpr int RUN = NT / NH;  // contiguous values of a column: 16, or 8 where D = 64
#pragma unroll
        for (int i = 0; i < RUN; i += 4) {
          const int f4 = (hh * 128 + (2 * c + e) * RUN + i) / 4, t = hh * 16 + i;
          part[part_index<D>(g + 8 * x, f4)] =
              make_float4(o[t][2 * x + e], o[t + 1][2 * x + e], o[t + 2][2 * x + e], o[t + 3][2 * x + e]);
        }
      }
  __syncthreads();

  // Join: maxima and sums of all warps first, then their outputs by weight.
  float* const fin = reinterpret_cast<float*>(smem + L::fin);
  if ((int)threadIdx.x < rows) {
    const int row = threadIdx.x;
    float m = -INFINITY, l = 0.f;
    for (uint32_t n = 0; n < NW; ++n) m = fmaxf(m, ml[n * 2 * kRows + row]);
    const float ms = m == -INFINITY ? 0.f : m;
    for (uint32_t n = 0; n < NW; ++n) {
      const float w = exp2_approx(ml[n * 2 * kRows + row] - ms);
      l = fmaf(w, ml[n * 2 * kRows + kRows + row], l);
      ml[n * 2 * kRows + row] = w;
    }
    fin[row] = l == 0.f ? 0.f : 1.0f / l;
    if (p.lse)
      p.lse[((int64_t)b * p.Q.d + qi) * p.H.d * p.G + head0 + row] =
          l == 0.f ? -INFINITY : (m - kLift + log2f(l)) * 0.69314718055994531f;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < rows * (D / 4); i += W * 32) {
    const int row = i / (D / 4), f4 = i % (D / 4);
    const uint32_t off = base + (uint32_t)L::ring + part_index<D>(row, f4) * 16;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (uint32_t n = 0; n < NW; ++n) {
      const uint4 v = lds128(off + n * (uint32_t)(S * 2 * L::side));
      const float w = ml[n * 2 * kRows + row];
      acc.x = fmaf(w, __uint_as_float(v.x), acc.x);
      acc.y = fmaf(w, __uint_as_float(v.y), acc.y);
      acc.z = fmaf(w, __uint_as_float(v.z), acc.z);
      acc.w = fmaf(w, __uint_as_float(v.w), acc.w);
    }
    const float f = fin[row];
    uint2 v;
    v.x = Half16<T>::pack(acc.x * f, acc.y * f);
    v.y = Half16<T>::pack(acc.z * f, acc.w * f);
    *reinterpret_cast<uint2*>(p.out.row(b, qi, head0 + row) + f4 * 8) = v;
  }
}

}  // namespace kv
