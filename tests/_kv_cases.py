"""Inputs of the paged-KV-cache tests, drawn on the CPU from a seed."""
import torch

from oracle.kv_oracle import quantise


def gen(seed):
    return torch.Generator().manual_seed(seed)


def angles(max_pos, rot, base=10000.0):
    half = rot // 2
    freq = base ** (-torch.arange(half, dtype=torch.float64) / max(half, 1))
    a = torch.arange(max_pos, dtype=torch.float64)[:, None] * freq
    return torch.cat([a.cos(), a.sin()], dim=1).float()


def random_cache(g, P, H, bs, D, code_dtype):
    """(codes, scales) of random vectors of unlike size."""
    x = torch.randn(P, H, bs, D, generator=g) * torch.exp(0.5 * torch.randn(P, H, bs, 1, generator=g))
    return quantise(x, code_dtype)


def caches(g, P, H, bs, D, code_dtype):
    return (*random_cache(g, P, H, bs, D, code_dtype), *random_cache(g, P, H, bs, D, code_dtype))


def page_table(g, B, NB, spare=2, dtype=torch.int32):
    """(table [B, NB] of distinct pages in no order, number of pages)."""
    P = B * NB + spare
    return torch.randperm(P, generator=g)[:B * NB].view(B, NB).to(dtype), P


def layout(t, how):
    """`t` [P, H, bs, ...] with the same values in another layout: "dense", "nhd" (tokens before heads),
    or "pair" (a slice of a buffer twice as wide in pages)."""
    if how == "nhd":
        return t.transpose(1, 2).contiguous().transpose(1, 2)
    if how == "pair":
        both = torch.stack([t.view(torch.uint8) if t.element_size() == 1 else t] * 2, dim=1)[:, 1]
        return both.view(t.dtype)
    return t
