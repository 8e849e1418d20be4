/*
 * dsa_kv.h — C ABI of the B200 (sm_100a) operators around the quantised,
 * paged KV cache that dsa_topk.h selects blocks of (libdsa_kv.so).
 *
 * In the order in which a decoder layer runs them:
 *   dsa_kv_rope_launch    per-head RMSNorm of queries and keys and their
 *                         rotation by position, one pass
 *   dsa_kv_write_launch   keys and values of new tokens, quantised with one
 *                         scale per token and head, into their pages
 *   dsa_kv_read_launch    keys and values of whole sequences, back from their
 *                         pages as dense 16-bit tensors
 *   dsa_kv_attn_launch    attention of every query row over the blocks that
 *                         dsa_topk_page_table_transform selected for it
 * The reference project has none of them: its block selection ends with the
 * page ids, and the consumer of those ids is left to the caller.
 *
 * Memory contract: destination passing; every pointer is a device pointer the
 * caller owns. Nothing is allocated, no scratch memory is used, and two calls
 * share nothing but the tensors they are given. Every launch is asynchronous
 * on the given stream of the current device. Positions, block ids and page ids
 * are read on the device and checked there: one that is out of range is never
 * followed (what it gives instead is said at each entry point).
 */
#ifndef DSA_KV_H
#define DSA_KV_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define DSA_KV_ABI_VERSION 2

enum dsa_kv_dtype {
    DSA_KV_BF16 = 0,
    DSA_KV_FP16 = 1,
    DSA_KV_FP32 = 2,
    DSA_KV_INT8 = 3,
    DSA_KV_E4M3 = 4,
    DSA_KV_INT32 = 5,
    DSA_KV_INT64 = 6
};

enum dsa_kv_status {
    DSA_KV_OK = 0,
    DSA_KV_ERR_NULL_POINTER = 1,  /* a required pointer is NULL                    */
    DSA_KV_ERR_BAD_SHAPE = 2,     /* a size below its least value                  */
    DSA_KV_ERR_BAD_HEAD_DIM = 3,  /* head size or rotated part not supported       */
    DSA_KV_ERR_BAD_DTYPE = 4,     /* unsupported dtype                             */
    DSA_KV_ERR_ALIGNMENT = 5,     /* a pointer or a stride is not aligned          */
    DSA_KV_ERR_UNSUPPORTED = 6,   /* sizes beyond the kernel's index range         */
    DSA_KV_ERR_CUDA = 7,          /* a CUDA call failed                            */
    DSA_KV_ERR_BAD_ARGS_SIZE = 8, /* struct_size mismatch or reserved field not 0  */
    DSA_KV_ERR_DEVICE_TIMEOUT = 9 /* a bounded device wait ran out                 */
};

/* A dense tensor [B, Q, H, D] whose last dimension is contiguous. Strides in
 * elements. Rows start on 16 bytes: the pointer is 16-byte aligned and every
 * stride of a dimension larger than 1 is a multiple of 8 elements. */
typedef struct dsa_kv_dense {
    void*   ptr;
    int64_t stride_b, stride_q, stride_h;
} dsa_kv_dense_t;

/*
 * A paged cache: codes [P, H, block_size, D] (int8 or e4m3) and scales
 * [P, H, block_size] fp32, for keys and for values. Token t of a sequence is
 * at offset t % block_size of the page that page_table[b, t / block_size]
 * names. A vector x of D values is stored as
 *     scale = max(max|x| / QMAX, 1e-12),   code = rn(x * (1 / scale))
 * with QMAX = 448 (e4m3, saturating) or 127 (int8), every step in fp32 rounded
 * to nearest even, and stands for code * scale. Unlike the int8 activations of
 * farq.h, which truncate as the reference does, codes are rounded: that halves
 * the largest error of what is read back on every later step. A vector that
 * holds a NaN or an infinity gets the scale NaN and the codes 0, so that it
 * reads back as NaN.
 * Strides: codes in elements (bytes), scales in floats; D is contiguous, code
 * rows start on 16 bytes. A read and the attention take scales broadcast by
 * strides of 0 (one scale per head, or for all); the attention's strides are
 * below 2^40 (codes) and 2^31 (scales).
 */
typedef struct dsa_kv_cache {
    int32_t code_dtype;           /* INT8 | E4M3                                   */
    int32_t reserved0;            /* must be 0                                     */
    int64_t P, H, block_size, D;
    void*   k_codes;
    void*   v_codes;
    float*  k_scale;
    float*  v_scale;
    int64_t k_stride[3], v_stride[3];             /* page, head, token             */
    int64_t k_scale_stride[3], v_scale_stride[3]; /* page, head, token             */
} dsa_kv_cache_t;

/*
 * Per-head RMSNorm and rotation, for q [B, Q, Hq, D] and k [B, Q, Hk, D]:
 *     y = x * (1 / sqrt(mean(x^2) + eps)) * gamma
 *     (a, b) -> (a cos - b sin, b cos + a sin) over the rot pairs of y
 * in fp32, rounded once. Row p of cos_sin [max_pos, rot] holds rot/2 cosines,
 * then rot/2 sines. Pair i is (y[i], y[i + rot/2]), or (y[2i], y[2i+1]) where
 * interleaved is 1; values from rot on are only normalised.
 * positions [B, Q]: a negative one marks padding, whose output rows are left
 * as they are; one at max_pos or beyond has no angles, its rows become NaN.
 * q_out / k_out may be q / k themselves. Hk may be 0 (queries only).
 * D <= 256, D % 8 == 0; rot <= D, rot % 16 == 0 (interleaved: rot % 8 == 0).
 */
typedef struct dsa_kv_rope_args {
    uint32_t struct_size;         /* = sizeof(dsa_kv_rope_args_t)                  */
    int32_t  dtype;               /* BF16 | FP16: q, k, q_out, k_out               */
    int32_t  gamma_dtype;         /* BF16 | FP16 | FP32                            */
    int32_t  pos_dtype;           /* INT32 | INT64                                 */
    int32_t  interleaved;         /* 0 | 1                                         */
    float    eps;
    int64_t  B, Q, Hq, Hk, D, rot, max_pos;
    dsa_kv_dense_t q, k, q_out, k_out;
    const void*  q_gamma;         /* [D], 16-byte aligned                          */
    const void*  k_gamma;         /* [D], 16-byte aligned                          */
    const float* cos_sin;         /* [max_pos, rot], contiguous, 16-byte aligned   */
    const void*  positions;       /* [B, Q], contiguous                            */
} dsa_kv_rope_args_t;

/*
 * Quantised write of k, v [B, Q, H, D] at the positions q_pos [B, Q], and
 * dequantised read of the first min(kv_lens[b], S, NB * block_size) tokens of
 * every sequence b into k_out, v_out [B, S, H, D].
 * Write: a token whose position is negative (padding) or at least
 * NB * block_size, or whose page id is not in [0, P), writes nothing. Two
 * tokens of one call for the same cell: which of the two remains is not
 * specified, and it may be one's codes with the other's scale.
 * Read: rows behind a sequence's end are left as they are; a token whose page
 * id is not in [0, P) reads as zeros.
 * D <= 256, D % 16 == 0.
 */
typedef struct dsa_kv_copy_args {
    uint32_t struct_size;         /* = sizeof(dsa_kv_copy_args_t)                  */
    int32_t  dtype;               /* BF16 | FP16: the dense tensors                */
    int32_t  page_dtype;          /* INT32 | INT64: page_table                     */
    int32_t  pos_dtype;           /* INT32 | INT64: q_pos (write), kv_lens (read)  */
    int64_t  B, Q, NB;            /* Q: new tokens (write), S (read)               */
    dsa_kv_dense_t k, v;          /* inputs (write), outputs (read)                */
    dsa_kv_cache_t cache;
    const void* page_table;       /* [B, NB], contiguous                           */
    const void* pos;              /* q_pos [B, Q] (write), kv_lens [B] (read)      */
} dsa_kv_copy_args_t;

/*
 * Attention over selected blocks. q [B, Q, H * G, D]: query heads h * G to
 * h * G + G - 1 share key head h and its selection. blocks, pages [B, H, Q, K]
 * (as dsa_topk_launch writes them; the last dimension contiguous, strides in
 * elements): entry i of a row stands for the tokens
 *     t = blocks[i] * block_size + j,  0 <= j < block_size,
 *     t <= q_pos[b, q],  t < kv_lens[b]
 * whose keys and values lie in page pages[i]. An entry with a negative block
 * id, or a page id outside [0, P), stands for none; one that occurs twice
 * counts twice. No token lies at position 2^40 or beyond.
 *     out = sum_t softmax(scale * q.k_t) v_t,   lse = ln sum_t exp(scale * q.k_t)
 * A row without a token (and a padded one, q_pos < 0) has out = 0, lse = -inf.
 * One whose tokens all have the score -inf has out = NaN, lse = -inf.
 * Products are fp16 x codes with sums in fp32: queries are scaled by a power of two,
 * bf16 values more than 2^-20 below their head's largest may lose bits.
 * out may be q itself. A copy that has not arrived after two seconds ends its
 * row: the outputs become NaN, and dsa_kv_attn_launch_status says so.
 * v_scale is positive; one below 1e-12, the least that a write leaves, counts
 * as 1e-12. One that is NaN (a vector that held a NaN or an infinity) or infinite
 * makes out NaN in the rows that see its token; lse, which holds no values, is the
 * same as with any other scale.
 * D is 64, 128 or 256, block_size >= 8.
 */
typedef struct dsa_kv_attn_args {
    uint32_t struct_size;         /* = sizeof(dsa_kv_attn_args_t)                  */
    int32_t  dtype;               /* BF16 | FP16: q, out                           */
    int32_t  block_dtype;         /* INT32 | INT64: blocks                         */
    int32_t  page_dtype;          /* INT32 | INT64: pages                          */
    int32_t  pos_dtype;           /* INT32 | INT64: q_pos and kv_lens              */
    float    softmax_scale;
    int64_t  B, Q, G, K;
    dsa_kv_dense_t q, out;
    dsa_kv_cache_t cache;
    const void* blocks;
    const void* pages;
    int64_t  blocks_stride[3], pages_stride[3];   /* b, h, q                       */
    const void* q_pos;            /* [B, Q], contiguous                            */
    const void* kv_lens;          /* [B]                                           */
    float*   lse;                 /* [B, Q, H * G], contiguous; may be NULL        */
} dsa_kv_attn_args_t;

/* Each validates every argument before any device call and returns a
 * dsa_kv_status; on DSA_KV_OK the work is queued, not finished. */
int dsa_kv_rope_launch(const dsa_kv_rope_args_t* args, void* stream);
int dsa_kv_write_launch(const dsa_kv_copy_args_t* args, void* stream);
int dsa_kv_read_launch(const dsa_kv_copy_args_t* args, void* stream);
int dsa_kv_attn_launch(const dsa_kv_attn_args_t* args, void* stream);

/*
 * dsa_kv_attn_launch that tells a wait that ran out from NaN in the data: `status`,
 * a device int or NULL, is then set to DSA_KV_ERR_DEVICE_TIMEOUT (it is never
 * cleared). test_copies is 0, or, in tests of that path, a number of 2 and more:
 * the first warp of every row that has started so many copies (keys and values of
 * a chunk are one each) takes its next wait as run out, its copies in flight.
 */
int dsa_kv_attn_launch_status(const dsa_kv_attn_args_t* args, int32_t* status, int32_t test_copies, void* stream);

/* Static string for a dsa_kv_status (never NULL). */
const char* dsa_kv_strerror(int status);

/* DSA_KV_ABI_VERSION of the loaded library. */
int dsa_kv_abi_version(void);

#ifdef __cplusplus
}
#endif

#endif /* DSA_KV_H */
