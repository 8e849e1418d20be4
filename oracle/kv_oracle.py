"""Plain implementations in 64 bits of the operators around the paged KV cache
(TEST INFRASTRUCTURE: only tests/ and __graft_entry__.smoke() use this module;
the product path never imports it).

Everything is computed on the CPU in float64 from the operators' formulas
(include/dsa_kv.h), token by token where that says more than a batched form.
"""
from __future__ import annotations

import math

import torch

QMAX = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}
MIN_SCALE = 1e-12


def _rotate(x, gamma, cos_sin, positions, old, eps, interleaved):
    """(rotated heads, size of the terms that each output is the sum of)."""
    B, Q, H, D = x.shape
    rot = cos_sin.shape[1]
    half = rot // 2
    out, size = old.double().clone(), torch.zeros(B, Q, H, D, dtype=torch.float64)
    for b in range(B):
        for q in range(Q):
            pos = int(positions[b, q])
            if pos < 0:
                continue
            y = x[b, q].double()
            y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * gamma.double()
            if pos >= cos_sin.shape[0]:
                out[b, q] = math.nan
                continue
            o, m = y.clone(), y.abs()
            c, s = cos_sin[pos, :half].double(), cos_sin[pos, half:].double()
            i = torch.arange(half)
            ia, ib = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
            a, d = y[:, ia], y[:, ib]
            o[:, ia], o[:, ib] = a * c - d * s, d * c + a * s
            m[:, ia], m[:, ib] = (a * c).abs() + (d * s).abs(), (d * c).abs() + (a * s).abs()
            out[b, q], size[b, q] = o, m
    return out, size


def qk_rmsnorm_rope_ref(q, k, q_gamma, k_gamma, cos_sin, positions, q_old, k_old, eps, interleaved=False):
    """((q_out, its terms' size), (k_out, its terms' size)) in float64."""
    return (_rotate(q, q_gamma, cos_sin, positions, q_old, eps, interleaved),
            _rotate(k, k_gamma, cos_sin, positions, k_old, eps, interleaved))


def e4m3_round(v: torch.Tensor) -> torch.Tensor:
    """The e4m3 value nearest to each float64 (ties to the even code, saturating)."""
    a = v.abs().clamp(min=2.0 ** -6)
    step = torch.exp2(torch.floor(torch.log2(a)) - 3)
    return (torch.round(v / step) * step).clamp(-448.0, 448.0)


def quantise(x: torch.Tensor, code_dtype: torch.dtype):
    """(codes, scales) of the vectors x[..., D]. The format's definition rounds
    every step to fp32; each step is computed in float64 and rounded once
    (exact products; quotients of fp32 values are not doubly rounded, as
    53 >= 2 * 24 + 2)."""
    y = x.double()
    amax = y.abs().amax(-1)
    scale = (amax / QMAX[code_dtype]).float().double().clamp(min=float(torch.tensor(MIN_SCALE)))
    inv = (1.0 / scale).float().double()
    y = (y * inv[..., None]).float().double()
    bad = ~torch.isfinite(amax)
    y = torch.where(bad[..., None], 0.0, y)
    codes = e4m3_round(y).float() if code_dtype == torch.float8_e4m3fn else torch.round(y)
    return codes.to(code_dtype), torch.where(bad, math.nan, scale).float()


def paged_kv_quant_write_ref(k, v, k_cache, k_scale, v_cache, v_scale, page_table, q_pos):
    """The four cache tensors after the write (new tensors; codes as bytes)."""
    P, H, bs, D = k_cache.shape
    B, Q = q_pos.shape
    got = []
    for x, codes, scales in ((k, k_cache, k_scale), (v, v_cache, v_scale)):
        new_c, new_s = codes.view(torch.uint8).clone(), scales.clone()
        qc, qs = quantise(x, codes.dtype)
        qc = qc.view(torch.uint8)
        for b in range(B):
            for i in range(Q):
                pos = int(q_pos[b, i])
                if pos < 0 or pos >= page_table.shape[1] * bs:
                    continue
                page = int(page_table[b, pos // bs])
                if 0 <= page < P:
                    new_c[page, :, pos % bs] = qc[b, i]
                    new_s[page, :, pos % bs] = qs[b, i]
        got += [new_c, new_s]
    return tuple(got)


def paged_kv_dequant_read_ref(k_cache, k_scale, v_cache, v_scale, page_table, kv_lens, k_old, v_old):
    """(k_out, v_out) in float64; k_old, v_old are the outputs before the call."""
    P, H, bs, D = k_cache.shape
    B, S = k_old.shape[:2]
    got = []
    for codes, scales, old in ((k_cache, k_scale, k_old), (v_cache, v_scale, v_old)):
        out = old.double().clone()
        val = codes.float().double() * scales.double()[..., None]
        for b in range(B):
            for t in range(min(int(kv_lens[b]), S, page_table.shape[1] * bs)):
                page = int(page_table[b, t // bs])
                out[b, t] = val[page, :, t % bs] if 0 <= page < P else 0.0
        got.append(out)
    return tuple(got)


def dsa_paged_attention_ref(q, k_cache, k_scale, v_cache, v_scale, blocks, pages, q_pos, kv_lens, softmax_scale):
    """dict of float64 tensors: out [B, Q, Hq, D], lse [B, Q, Hq], and what error bounds are made of, per row and
    head: n, the number of tokens; score, the largest sum over D of the magnitudes of a score's terms; size [.., D],
    the weighted sum of the values' magnitudes; top, the largest weight times value scale."""
    P, H, bs, D = k_cache.shape
    B, Q, Hq, _ = q.shape
    G = Hq // H
    shape = (B, Q, Hq)
    r = {"out": torch.zeros(*shape, D, dtype=torch.float64), "lse": torch.full(shape, -math.inf, dtype=torch.float64),
         "size": torch.zeros(*shape, D, dtype=torch.float64), "n": torch.zeros(shape, dtype=torch.float64),
         "score": torch.zeros(shape, dtype=torch.float64), "top": torch.zeros(shape, dtype=torch.float64)}
    kc, vc = k_cache.float().double(), v_cache.float().double()
    for b in range(B):
        for i in range(Q):
            pos, n = int(q_pos[b, i]), int(kv_lens[b])
            lim = min(pos + 1, n) if pos >= 0 else 0
            for h in range(H):
                where = []
                for blk, page in zip(blocks[b, h, i].tolist(), pages[b, h, i].tolist()):
                    if blk >= 0 and 0 <= page < P:
                        where += [(page, j) for j in range(bs) if blk * bs + j < lim]
                if not where:
                    continue
                pg, off = torch.tensor(where).T
                ks, vs = k_scale[pg, h, off].double(), v_scale[pg, h, off].double()
                k, v = kc[pg, h, off] * ks[:, None], vc[pg, h, off] * vs[:, None]
                x = q[b, i, h * G:(h + 1) * G].double()
                s = x @ k.T * softmax_scale
                lse = torch.logsumexp(s, -1)
                p = torch.exp(s - lse[:, None])
                at = (b, i, slice(h * G, (h + 1) * G))
                r["out"][at], r["lse"][at], r["size"][at] = p @ v, lse, p @ v.abs()
                r["n"][at] = len(where)
                r["score"][at] = (x.abs() @ k.abs().T * abs(softmax_scale)).amax(-1)
                r["top"][at] = (p * vs).amax(-1)
    return r
