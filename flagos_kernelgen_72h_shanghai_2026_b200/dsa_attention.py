"""Attention over the blocks that the block selection named.

``dsa_paged_attention`` is the consumer of ``dsa_topk_page_table_transform``'s
outputs: every query row attends to the tokens of its own selected blocks,
read from the quantised, paged cache that ``paged_kv_quant_write`` fills. One
sm_100a kernel in libdsa_kv.so (C ABI: include/dsa_kv.h); destination passing,
asynchronous on the current CUDA stream, no workspace.

Errors: ``TypeError`` for a non-CUDA tensor or a dtype the kernel does not
take, ``ValueError`` for shapes, strides and alignment, ``RuntimeError`` when a
CUDA call fails. There is no CPU fallback.
"""
from __future__ import annotations

import ctypes

import torch

from . import _kv_lib as L

_OP = "dsa_paged_attention"


def _selection(name, t, device, shape):
    L.check_tensor(name, t, device)
    L.check_shape(name, t, shape)
    if shape[3] > 1 and t.stride(3) != 1:
        raise ValueError(f"{name} must be contiguous along its last dimension")
    return L.dtype_code(name, t, L.INDEX_DTYPES)


def dsa_paged_attention(q: torch.Tensor, k_cache: torch.Tensor, k_scale: torch.Tensor,
                        v_cache: torch.Tensor, v_scale: torch.Tensor, blocks: torch.Tensor,
                        pages: torch.Tensor, q_pos: torch.Tensor, kv_lens: torch.Tensor,
                        out: torch.Tensor, lse: torch.Tensor | None, softmax_scale: float, *,
                        status: torch.Tensor | None = None, _test_copies: int = 0):
    """out = softmax(softmax_scale * q k^T) v over each row's selected tokens; returns ``(out, lse)``.

    q, out [B, Q, Hq, D] bf16 or fp16 (strided views whose rows start on 16
    bytes; out may be q itself); Hq is a multiple of the cache's H, query heads h * Hq/H and on
    share key head h and its selection. The cache as in ``kv_cache``: codes
    [P, H, block_size, D], scales [P, H, block_size], which may be broadcast
    (one scale per head, or for all). blocks, pages
    [B, H, Q, K] int32 or int64 (the last dimension contiguous; the others may
    be broadcast): entry i stands for the tokens t of block ``blocks[..., i]``,
    stored in page ``pages[..., i]``, with t <= q_pos[b, q] and t < kv_lens[b].
    An entry with a negative block id or a page id outside [0, P) stands for
    none, one that occurs twice counts twice. q_pos [B, Q] and kv_lens [B] as
    in the selection. ``lse`` [B, Q, Hq] fp32, or None, gets the natural
    logarithm of the softmax's denominator. A row without a token, and a
    padded one (negative position), has out = 0 and lse = -inf. A row that sees
    a value vector stored with a NaN or an infinity has out = NaN and the lse of
    its scores.

    Waits of the kernel are bounded: a row whose copies have not arrived after
    two seconds becomes NaN, and ``status``, an int32 tensor of one element if
    given, 9 (it is never cleared).

    D is 64, 128 or 256; block_size is 8 to 65536."""
    if L._fast is not None and status is None and not _test_copies:
        st = L._fast.kv_attn(q, k_cache, k_scale, v_cache, v_scale, blocks, pages, q_pos, kv_lens, out, lse,
                             softmax_scale)
        if st == 0:
            return out, lse
        if st > 0:
            L.raise_status(_OP, st)
    dev = L.check_tensor("q", q, None)
    a = L.AttnArgs()
    a.struct_size = ctypes.sizeof(a)
    a.dtype = L.dtype_code("q", q, L.HALF_DTYPES)
    a.cache = L.cache(k_cache, k_scale, v_cache, v_scale, dev)
    if q.dim() != 4:
        raise ValueError(f"q must be [B, Q, H, D], got {list(q.shape)}")
    B, Q, Hq, D = q.shape
    H = k_cache.shape[1]
    if D != k_cache.shape[3]:
        raise ValueError(f"q has head size {D}, the cache {k_cache.shape[3]}")
    if H == 0 or Hq == 0 or Hq % H != 0:
        raise ValueError(f"{Hq} query heads are not a multiple of the cache's {H} heads")
    a.q = L.dense("q", q, (B, Q, Hq, D), q.dtype, dev)
    a.out = L.dense("out", out, (B, Q, Hq, D), q.dtype, dev)
    L.check_tensor("blocks", blocks, dev)
    if blocks.dim() != 4:
        raise ValueError(f"blocks must be [B, H, Q, K], got {list(blocks.shape)}")
    K = blocks.shape[3]
    a.block_dtype = _selection("blocks", blocks, dev, (B, H, Q, K))
    a.page_dtype = _selection("pages", pages, dev, (B, H, Q, K))
    three = ctypes.c_int64 * 3
    a.blocks_stride = three(*blocks.stride()[:3])
    a.pages_stride = three(*pages.stride()[:3])
    for name, t, shape in (("q_pos", q_pos, (B, Q)), ("kv_lens", kv_lens, (B,))):
        L.check_tensor(name, t, dev)
        L.check_shape(name, t, shape)
        L.check_contiguous(name, t)
    a.pos_dtype = L.dtype_code("q_pos", q_pos, L.INDEX_DTYPES)
    if kv_lens.dtype != q_pos.dtype:
        raise TypeError(f"kv_lens must have q_pos's dtype {q_pos.dtype}, got {kv_lens.dtype}")
    if lse is not None:
        L.check_tensor("lse", lse, dev)
        L.check_shape("lse", lse, (B, Q, Hq))
        L.check_contiguous("lse", lse)
        if lse.dtype != torch.float32:
            raise TypeError(f"lse must be float32, got {lse.dtype}")
        a.lse = lse.data_ptr() or None
    if status is not None:
        L.check_tensor("status", status, dev)
        L.check_shape("status", status, (1,))
        if status.dtype != torch.int32:
            raise TypeError(f"status must be int32, got {status.dtype}")
    a.softmax_scale = float(softmax_scale)
    a.B, a.Q, a.G, a.K = B, Q, Hq // H, K
    a.blocks = blocks.data_ptr() or None
    a.pages = pages.data_ptr() or None
    a.q_pos = q_pos.data_ptr() or None
    a.kv_lens = kv_lens.data_ptr() or None
    L.launch(_OP, "dsa_kv_attn_launch_status", a, dev,
             status.data_ptr() if status is not None else None, _test_copies)
    return out, lse
