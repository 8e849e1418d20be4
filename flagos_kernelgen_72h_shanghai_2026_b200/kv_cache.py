"""The quantised, paged KV cache: writing new tokens, reading sequences back.

A cache is four tensors of the caller's: codes ``k_cache``, ``v_cache``
[P, H, block_size, D] (int8 or float8_e4m3fn) and fp32 scales ``k_scale``,
``v_scale`` [P, H, block_size], one for each token and head. They may be
strided views (a layer of a larger buffer, keys and values side by side, a
[P, block_size, H, D] buffer transposed) whose code rows start on 16 bytes.
Token t of sequence b is at offset ``t % block_size`` of page
``page_table[b, t // block_size]``; ``page_table`` and the positions are those
of ``dsa_topk_page_table_transform``.

A vector x is stored as ``scale = max(max|x| / QMAX, 1e-12)`` and
``code = round(x * (1 / scale))`` (QMAX 448 or 127, nearest even), and stands
for ``code * scale``. Codes are rounded, not truncated as the int8 activations
of ``fused_add_rmsnorm_group_quant``: the cache is read at every later step,
and rounding halves its largest error. A vector with a NaN or an infinity
reads back as NaN.

Errors: ``TypeError`` for a non-CUDA tensor or a dtype the kernels do not
take, ``ValueError`` for shapes, strides and alignment, ``RuntimeError`` when a
CUDA call fails. There is no CPU fallback. The device work is two sm_100a
kernels in libdsa_kv.so (C ABI: include/dsa_kv.h).
"""
from __future__ import annotations

import ctypes

import torch

from . import _kv_lib as L


def _args(k, v, names, k_cache, k_scale, v_cache, v_scale, page_table, pos, pos_name, pos_shape):
    dev = L.check_tensor(names[0], k, None)
    a = L.CopyArgs()
    a.struct_size = ctypes.sizeof(a)
    a.dtype = L.dtype_code(names[0], k, L.HALF_DTYPES)
    a.cache = L.cache(k_cache, k_scale, v_cache, v_scale, dev)
    if k.dim() != 4:
        raise ValueError(f"{names[0]} must be [B, Q, H, D], got {list(k.shape)}")
    B, Q = k.shape[:2]
    shape = (B, Q, k_cache.shape[1], k_cache.shape[3])
    a.k = L.dense(names[0], k, shape, k.dtype, dev)
    a.v = L.dense(names[1], v, shape, k.dtype, dev)
    L.check_tensor("page_table", page_table, dev)
    if page_table.dim() != 2 or page_table.shape[0] != B:
        raise ValueError(f"page_table must be [{B}, NB], got {list(page_table.shape)}")
    L.check_contiguous("page_table", page_table)
    a.page_dtype = L.dtype_code("page_table", page_table, L.INDEX_DTYPES)
    L.check_tensor(pos_name, pos, dev)
    L.check_shape(pos_name, pos, (B, Q) if pos_shape == 2 else (B,))
    L.check_contiguous(pos_name, pos)
    a.pos_dtype = L.dtype_code(pos_name, pos, L.INDEX_DTYPES)
    a.B, a.Q, a.NB = B, Q, page_table.shape[1]
    a.page_table = page_table.data_ptr() or None
    a.pos = pos.data_ptr() or None
    return a, dev


def paged_kv_quant_write(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor,
                         k_scale: torch.Tensor, v_cache: torch.Tensor, v_scale: torch.Tensor,
                         page_table: torch.Tensor, q_pos: torch.Tensor):
    """Quantise the new tokens' k, v [B, Q, H, D] (bf16 or fp16, rows on 16
    bytes) into the pages of their positions q_pos [B, Q]; returns
    ``(k_cache, k_scale, v_cache, v_scale)``.

    A token writes nothing if its position is negative (padding) or not below
    NB * block_size, or if its page id is not in [0, P). The tokens of a call
    have cells of their own: of two for the same cell, which remains is not
    specified, and it may be one's codes with the other's scale."""
    if L._fast is not None:
        st = L._fast.kv_copy(k, v, k_cache, k_scale, v_cache, v_scale, page_table, q_pos, True)
        if st == 0:
            return k_cache, k_scale, v_cache, v_scale
        if st > 0:
            L.raise_status("paged_kv_quant_write", st)
    a, dev = _args(k, v, ("k", "v"), k_cache, k_scale, v_cache, v_scale, page_table, q_pos,
                   "q_pos", 2)
    L.launch("paged_kv_quant_write", "dsa_kv_write_launch", a, dev)
    return k_cache, k_scale, v_cache, v_scale


def paged_kv_dequant_read(k_cache: torch.Tensor, k_scale: torch.Tensor, v_cache: torch.Tensor,
                          v_scale: torch.Tensor, page_table: torch.Tensor, kv_lens: torch.Tensor,
                          k_out: torch.Tensor, v_out: torch.Tensor):
    """Read the first min(kv_lens[b], S, NB * block_size) tokens of every
    sequence into k_out, v_out [B, S, H, D] (bf16 or fp16, rows on 16 bytes);
    returns both. Rows behind a sequence's end are left as they are; a token
    whose page id is not in [0, P) reads as zeros."""
    if L._fast is not None:
        st = L._fast.kv_copy(k_out, v_out, k_cache, k_scale, v_cache, v_scale, page_table, kv_lens, False)
        if st == 0:
            return k_out, v_out
        if st > 0:
            L.raise_status("paged_kv_dequant_read", st)
    a, dev = _args(k_out, v_out, ("k_out", "v_out"), k_cache, k_scale, v_cache, v_scale,
                   page_table, kv_lens, "kv_lens", 1)
    L.launch("paged_kv_dequant_read", "dsa_kv_read_launch", a, dev)
    return k_out, v_out
