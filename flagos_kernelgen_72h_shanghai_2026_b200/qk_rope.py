"""Per-head RMSNorm of queries and keys with the rotation by position.

``qk_rmsnorm_rope`` is the step between a decoder layer's query/key projection
and its attention: one sm_100a kernel in libdsa_kv.so (C ABI:
include/dsa_kv.h) reads every head once, normalises it, rotates it and writes
it. Destination passing, asynchronous on the current CUDA stream.

Errors: ``TypeError`` for a non-CUDA tensor or a dtype the kernel does not
take, ``ValueError`` for shapes, strides and alignment, ``RuntimeError`` when a
CUDA call fails. There is no CPU fallback.
"""
from __future__ import annotations

import ctypes

import torch

from . import _kv_lib as L

_OP = "qk_rmsnorm_rope"


def qk_rmsnorm_rope(q: torch.Tensor, k: torch.Tensor, q_gamma: torch.Tensor, k_gamma: torch.Tensor,
                    cos_sin: torch.Tensor, positions: torch.Tensor, q_out: torch.Tensor,
                    k_out: torch.Tensor, eps: float, *, interleaved: bool = False):
    """q_out, k_out = rotate(RMSNorm(q) * q_gamma), rotate(RMSNorm(k) * k_gamma); returns both.

    q [B, Q, Hq, D] and k [B, Q, Hk, D], bf16 or fp16, may be strided views
    (slices of a fused projection's output) whose rows start on 16 bytes;
    q_out and k_out likewise, and they may be q and k themselves. Gammas [D]
    bf16, fp16 or fp32. cos_sin [max_pos, rot] fp32 holds rot/2 cosines, then
    rot/2 sines of each position; the first rot of the D values are rotated,
    as pairs (i, i + rot/2), or (2i, 2i + 1) with ``interleaved``. positions
    [B, Q] int32 or int64: rows of a negative one (padding) are left as they
    are, rows of one at max_pos or beyond become NaN. The norm is over all D
    values, in fp32; outputs are rounded once.

    D % 8 == 0, D <= 256; rot % 16 == 0 (interleaved: rot % 8 == 0)."""
    if L._fast is not None:
        st = L._fast.kv_rope(q, k, q_gamma, k_gamma, cos_sin, positions, q_out, k_out, eps, interleaved)
        if st == 0:
            return q_out, k_out
        if st > 0:
            L.raise_status(_OP, st)
    dev = L.check_tensor("q", q, None)
    dt = L.dtype_code("q", q, L.HALF_DTYPES)
    if q.dim() != 4:
        raise ValueError(f"q must be [B, Q, H, D], got {list(q.shape)}")
    B, Q, Hq, D = q.shape
    L.check_tensor("k", k, dev)
    if k.dim() != 4:
        raise ValueError(f"k must be [B, Q, H, D], got {list(k.shape)}")
    Hk = k.shape[2]
    a = L.RopeArgs()
    a.struct_size = ctypes.sizeof(a)
    a.dtype = dt
    a.q = L.dense("q", q, (B, Q, Hq, D), q.dtype, dev)
    a.k = L.dense("k", k, (B, Q, Hk, D), q.dtype, dev)
    a.q_out = L.dense("q_out", q_out, (B, Q, Hq, D), q.dtype, dev)
    a.k_out = L.dense("k_out", k_out, (B, Q, Hk, D), q.dtype, dev)
    for name, t in (("q_gamma", q_gamma), ("k_gamma", k_gamma)):
        L.check_tensor(name, t, dev)
        L.check_shape(name, t, (D,))
        L.check_contiguous(name, t)
    a.gamma_dtype = L.dtype_code("q_gamma", q_gamma, L.GAMMA_DTYPES)
    if k_gamma.dtype != q_gamma.dtype:
        raise TypeError(f"k_gamma must have q_gamma's dtype {q_gamma.dtype}, got {k_gamma.dtype}")
    L.check_tensor("cos_sin", cos_sin, dev)
    if cos_sin.dtype != torch.float32:
        raise TypeError(f"cos_sin must be float32, got {cos_sin.dtype}")
    if cos_sin.dim() != 2:
        raise ValueError(f"cos_sin must be [max_pos, rot], got {list(cos_sin.shape)}")
    L.check_contiguous("cos_sin", cos_sin)
    L.check_tensor("positions", positions, dev)
    L.check_shape("positions", positions, (B, Q))
    L.check_contiguous("positions", positions)
    a.pos_dtype = L.dtype_code("positions", positions, L.INDEX_DTYPES)
    a.interleaved = 1 if interleaved else 0
    a.eps = float(eps)
    a.B, a.Q, a.Hq, a.Hk, a.D = B, Q, Hq, Hk, D
    a.max_pos, a.rot = cos_sin.shape
    a.q_gamma = q_gamma.data_ptr()
    a.k_gamma = k_gamma.data_ptr()
    a.cos_sin = cos_sin.data_ptr() or None
    a.positions = positions.data_ptr() or None
    L.launch(_OP, "dsa_kv_rope_launch", a, dev)
    return q_out, k_out
