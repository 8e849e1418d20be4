"""dsa_paged_attention on the GPU against the plain implementation in 64 bits
(oracle/kv_oracle.py), and the operators of a decoder layer run together.

Tolerances (u = 2^-24, half a step of fp32; magnitudes as the oracle gives
them, n tokens, D the head size):
  score    fp16 products are exact in fp32; a tile's sum of 16 products and its
           running value may lose two half steps of the largest term for each
           term: D/16 steps of 17 terms, at most (D + 16) * 2u * score; the
           factor, the exponent of the value scale and the running maximum add
           4u * (|a| <= score + 40) and 2^-21 for log2.
  weight   fp16: 2^-11 relative, at least 2^-31 of the largest weight; exp2
           2^-22; the score's error goes in twice (numerator, denominator).
  sums     over n tokens: n/16 steps of 17 terms as above.
  q        bf16 and fp16 values are exact down to 2^-28 of the tile's largest.
"""
import ctypes
import math
import subprocess
import sys
import threading
from pathlib import Path

import pytest
import torch

from oracle import kv_oracle as R
from oracle.dsa_topk_oracle import dsa_topk_page_table_transform_ref
from flagos_kernelgen_72h_shanghai_2026_b200 import (dsa_paged_attention, dsa_topk_page_table_transform,
                                                     paged_kv_dequant_read, paged_kv_quant_write, qk_rmsnorm_rope)
from _kv_cases import angles, caches, gen, layout, page_table

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
BF16, FP16 = torch.bfloat16, torch.float16
E4M3, INT8 = torch.float8_e4m3fn, torch.int8


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.fail("this test needs a CUDA device (run with -m 'not gpu' on CPU-only hosts)")
    from flagos_kernelgen_72h_shanghai_2026_b200._build import build_kv_lib
    build_kv_lib()
    return torch.device("cuda:0")


def bounds(r, D, qmax):
    score = (D + 16) * 2 * U * r["score"] + 4 * U * (r["score"] + 40) + 2.0 ** -21
    rel = 2.0 ** -11 + 2.0 ** -20 + 2 * score + (r["n"] / 16 + 2) * 17 * 2 * U
    # a weight below fp16's normal numbers is off by 2^-31 of the largest, times a code of at most qmax
    floor = r["n"] * 2.0 ** -31 * qmax * r["top"]
    out = rel[..., None] * r["size"] + floor[..., None]
    lse = score + 2.0 ** -20 + (r["n"] / 16 + 20) * U + 4 * U * r["lse"].abs().nan_to_num(posinf=0.0)
    return out, lse


def check(out, lse, r, D, qmax):
    tol_out, tol_lse = bounds(r, D, qmax)
    g, half = out.cpu().double(), torch.finfo(out.dtype).eps / 2
    assert torch.equal(g.isnan(), r["out"].isnan())
    tol = half * (r["out"].abs() + tol_out) + tol_out + (2.0 ** -25 if out.dtype == FP16 else 0.0)
    off = ((g - r["out"]).abs() - tol).nan_to_num(-1.0)
    assert float(off.max()) <= 0, f"out is off by {float(off.max()):.3g} more than allowed"
    if lse is not None:
        x = lse.cpu().double()
        empty = r["lse"] == -math.inf
        assert torch.equal(x == -math.inf, empty) and torch.equal(x.isnan(), r["lse"].isnan())
        off = ((x - r["lse"]).abs() - tol_lse)[~empty].nan_to_num(-1.0)
        assert off.numel() == 0 or float(off.max()) <= 0, f"lse is off by {float(off.max()):.3g} more than allowed"


def select(g, B, H, Q, K, NB, table, index=torch.int32):
    """Random selections of K of NB blocks (less where there are less), -1 behind them."""
    blocks = torch.full((B, H, Q, K), -1, dtype=torch.int64)
    n = min(K, NB)
    blocks[..., :n] = torch.rand(B, H, Q, NB, generator=g).argsort(-1)[..., :n]
    pages = table.long()[:, None, None].expand(B, H, Q, NB).gather(3, blocks.clamp(min=0))
    pages = torch.where(blocks >= 0, pages, -1)
    return blocks.to(index), pages.to(index)


def run(dev, q, c, blocks, pages, pos, lens, scale, how="dense", with_lse=True):
    cd = tuple(layout(t.to(dev), how) for t in c)
    qd = q.to(dev)
    out = torch.full_like(qd, 7.0)
    lse = torch.full(q.shape[:3], 7.0, device=dev) if with_lse else None
    got = dsa_paged_attention(qd, *cd, blocks.to(dev), pages.to(dev), pos.to(dev), lens.to(dev), out, lse, scale)
    assert got[0] is out and got[1] is lse
    torch.cuda.synchronize(dev)
    return out, lse


def case(dev, B, Q, H, G, D, bs, K, NB, dtype, code, seed, how="dense", index=torch.int32, full=False):
    g = gen(seed)
    table, P = page_table(g, B, NB)
    c = caches(g, P, H, bs, D, code)
    q = (2 * torch.randn(B, Q, H * G, D, generator=g)).to(dtype)
    blocks, pages = select(g, B, H, Q, K, NB, table, index)
    if full:
        lens = torch.full((B,), NB * bs)
    else:
        lens = torch.randint(1, NB * bs + 1, (B,), generator=g)
    pos = (lens[:, None] - Q + torch.arange(Q)).clamp(min=0)
    pos, lens = pos.to(index), lens.to(index)
    out, lse = run(dev, q, c, blocks, pages, pos, lens, D ** -0.5, how)
    check(out, lse, R.dsa_paged_attention_ref(q, *c, blocks, pages, pos, lens, D ** -0.5), D, R.QMAX[code])


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("code", [E4M3, INT8])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_types_and_head_sizes(dev, D, code, dtype):
    case(dev, 2, 2, 2, 4, D, 64, 5, 7, dtype, code, seed=D, full=True)


@pytest.mark.parametrize("bs", [8, 9, 10, 15, 16, 17, 24, 32, 33, 48, 64, 100, 128])
def test_block_sizes(dev, bs):
    case(dev, 2, 2, 2, 3, 128, bs, 6, 9, BF16, E4M3, seed=bs)
    case(dev, 1, 2, 1, 2, 64, bs, 40, 50, FP16, INT8, seed=bs + 1)


@pytest.mark.parametrize("bs", [200, 1000, 4096])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_long_blocks(dev, bs, D):
    case(dev, 2, 3, 1, 4, D, bs, 2, 3, BF16, E4M3, seed=bs + D)


@pytest.mark.parametrize("G", [1, 2, 7, 8, 9, 15, 16, 17, 32, 40])
def test_query_heads_per_key_head(dev, G):
    case(dev, 1, 2, 2, G, 128, 32, 4, 6, BF16, E4M3, seed=G)


@pytest.mark.parametrize("K,NB", [(1, 1), (1, 5), (3, 2), (33, 40), (128, 130), (300, 301)])
def test_selection_sizes(dev, K, NB):
    case(dev, 1, 1, 2, 4, 64, 16, K, NB, BF16, INT8, seed=K, full=True)
    case(dev, 2, 1, 1, 8, 128, 64, min(K, 40), min(NB, 60), FP16, E4M3, seed=K + 1)


@pytest.mark.parametrize("D,G", [(64, 4), (64, 16), (128, 4), (128, 16), (256, 4), (256, 16)])
def test_rows_shared_by_clusters(dev, D, G):
    """Numbers of rows and of blocks where the share of one, two, four and eight CTAs changes: too many rows for
    clusters to be resident, one chunk to a warp and less, uneven last rounds."""
    for B, K in ((1, 9), (1, 12), (1, 33), (37, 13), (37, 24), (76, 9), (149, 13)):
        case(dev, B, 1, 1, G, D, 64, K, K + 1, BF16, E4M3, seed=B + K)


@pytest.mark.parametrize("how", ["nhd", "pair"])
def test_cache_layouts(dev, how):
    case(dev, 2, 1, 3, 4, 128, 48, 4, 6, BF16, E4M3, seed=3, how=how)
    case(dev, 2, 1, 3, 4, 64, 16, 4, 6, BF16, INT8, seed=4, how=how)


def test_int64_indices(dev):
    case(dev, 2, 3, 2, 4, 128, 32, 5, 8, BF16, E4M3, seed=5, index=torch.int64)


def inputs(seed, B=2, Q=3, H=2, G=4, D=128, bs=32, K=6, NB=8, dtype=BF16, code=E4M3):
    g = gen(seed)
    table, P = page_table(g, B, NB)
    c = list(caches(g, P, H, bs, D, code))
    q = torch.randn(B, Q, H * G, D, generator=g).to(dtype)
    blocks, pages = select(g, B, H, Q, K, NB, table)
    lens = torch.full((B,), NB * bs, dtype=torch.int32)
    pos = (lens[:, None] - Q + torch.arange(Q)).int()
    return g, table, P, c, q, blocks, pages, pos, lens


def test_rows_without_tokens_and_bad_entries(dev):
    """Padded rows, empty caches, selections behind the row's position, ids and pages that do not exist."""
    _, _, P, c, q, blocks, pages, pos, lens = inputs(21)
    pos[0, 0] = -1                       # padding
    blocks[0, :, 1], pages[0, :, 1] = -1, -1  # nothing selected
    pos[0, 2] = 0                        # one token at most, if block 0 is selected
    blocks[0, 0, 2, 3] = 0
    blocks[0, 1, 2] = 5
    pages[1, 0, 0] = torch.tensor([P, P + 100, -5, 2 ** 31 - 1, -2 ** 31, 0])
    blocks[1, 0, 1, :3] = torch.tensor([-7, 2 ** 31 - 1, -2 ** 31])
    blocks[1, 1, 2] = blocks[1, 1, 2, 0]  # the same entry six times
    pages[1, 1, 2] = pages[1, 1, 2, 0]
    r = R.dsa_paged_attention_ref(q, *c, blocks, pages, pos, lens, 0.1)
    out, lse = run(dev, q, c, blocks, pages, pos, lens, 0.1)
    check(out, lse, r, 128, 448.0)
    assert (out[0, :2] == 0).all() and (lse[0, :2] == -math.inf).all()
    out2, none = run(dev, q, c, blocks, pages, pos, lens, 0.1, with_lse=False)
    assert none is None and torch.equal(out, out2)
    lens[1] = 0
    out, lse = run(dev, q, c, blocks, pages, pos, lens, 0.1)
    check(out, lse, R.dsa_paged_attention_ref(q, *c, blocks, pages, pos, lens, 0.1), 128, 448.0)
    # 64-bit ids and positions far beyond 32 bits
    blocks, pages, pos, lens = blocks.long(), pages.long(), pos.long(), lens.long()
    lens[1], pos[1, 0] = 2 ** 62, 2 ** 63 - 1
    blocks[1, 0, 2, 0], pages[1, 0, 2, 1] = 2 ** 40, 2 ** 33
    r = R.dsa_paged_attention_ref(q, *c, blocks, pages, pos, torch.tensor([int(lens[0]), 2 ** 40]), 0.1)
    out, lse = run(dev, q, c, blocks, pages, pos, lens, 0.1)
    # block 2^40 lies behind the most tokens that a sequence can have (2^40): an entry of no token
    check(out, lse, r, 128, 448.0)


@pytest.mark.parametrize("bs", [16, 24, 64])
def test_what_lies_behind_a_sequence_is_not_read(dev, bs):
    """NaN scales and NaN codes in the cells behind the last token, and in pages of nobody."""
    g, table, P, c, q, blocks, pages, pos, lens = inputs(22, bs=bs, Q=1)
    n = 4 * bs + 5
    lens[:], pos[:] = n, n - 1
    blocks = torch.arange(6).expand(2, 2, 1, 6).int()
    pages = table[:, None, None, :6].expand(2, 2, 1, 6)
    want = R.dsa_paged_attention_ref(q, *c, blocks, pages, pos, lens, 0.1)
    owned = torch.zeros(P, bs, dtype=torch.bool)
    for b in range(2):
        for t in range(n):
            owned[table[b, t // bs], t % bs] = True
    dirty = (~owned)[:, None].expand(P, 2, bs)
    for i in (0, 2):
        c[i] = c[i].view(torch.uint8).masked_fill(dirty[..., None], 0x7f).view(E4M3)
        c[i + 1] = c[i + 1].masked_fill(dirty, math.nan)
    out, lse = run(dev, q, c, blocks, pages, pos, lens, 0.1)
    check(out, lse, want, 128, 448.0)


def test_nan_and_infinite_tokens_reach_their_rows_alone(dev):
    _, table, P, c, q, blocks, pages, pos, lens = inputs(23)
    c[3][pages[0, 0, 0, 2], 0, 5] = math.nan     # a value that reads back as NaN
    c[1][pages[1, 1, 1, 0], 1, 31] = math.nan    # a key
    q = q.clone()
    q[0, 2, 5, 7] = math.nan
    q[1, 0, 0, 0] = math.inf
    out, lse = run(dev, q, c, blocks, pages, pos, lens, 0.1)
    r = R.dsa_paged_attention_ref(q, *c, blocks, pages, pos, lens, 0.1)
    bad = r["out"].isnan().any(-1)
    got = out.cpu().isnan()
    assert torch.equal(got.any(-1), bad)
    ok = {k: v[~bad] for k, v in r.items()}
    check(out.cpu()[~bad], None, ok, 128, 448.0)
    assert got[0, 2, 5].all() and got[1, 0, 0].all()


@pytest.mark.parametrize("code", [E4M3, INT8])
def test_scales_of_very_unlike_size(dev, code):
    """A first token with the largest score and next to no value, values up to 2^60 apart, and zero vectors."""
    g, table, P, c, q, blocks, pages, pos, lens = inputs(24, code=code)
    for i in (1, 3):
        c[i] = c[i] * torch.exp2(torch.randint(-30, 31, c[i].shape, generator=g).float() * (1 if i == 3 else 0.1))
    c[3][pages[0, 0, 0, 0], 0, 0] = R.MIN_SCALE
    c[2][pages[0, 0, 0, 0], 0, 0] = 0
    r = R.dsa_paged_attention_ref(q, *c, blocks, pages, pos, lens, 0.1)
    out, lse = run(dev, q, c, blocks, pages, pos, lens, 0.1)
    check(out, lse, r, 128, R.QMAX[code])


@pytest.mark.parametrize("scale_q", [1e-20, 1e4, 1e30])
def test_queries_of_any_size(dev, scale_q):
    _, _, _, c, q, blocks, pages, pos, lens = inputs(25)
    q = (q.float() * scale_q).to(BF16)
    s = 0.1 / scale_q
    out, lse = run(dev, q, c, blocks, pages, pos, lens, s)
    check(out, lse, R.dsa_paged_attention_ref(q, *c, blocks, pages, pos, lens, s), 128, 448.0)


def test_scores_far_apart_and_rising(dev):
    """Each block's scores lie well above those before it, so that the running maximum moves in every chunk."""
    _, table, P, c, q, blocks, pages, pos, lens = inputs(26, K=8, NB=8)
    blocks = torch.arange(8).expand(2, 2, 3, 8).int().contiguous()
    pages = table[:, None, None, :].expand(2, 2, 3, 8).contiguous()
    for b in range(2):
        for i in range(8):
            c[1][table[b, i]] *= 1.0 + 3 * i
    r = R.dsa_paged_attention_ref(q, *c, blocks, pages, pos, lens, 1.0)
    out, lse = run(dev, q, c, blocks, pages, pos, lens, 1.0)
    check(out, lse, r, 128, 448.0)
    r = R.dsa_paged_attention_ref(q, *c, blocks, pages, pos, lens, -1.0)
    out, lse = run(dev, q, c, blocks, pages, pos, lens, -1.0)
    check(out, lse, r, 128, 448.0)


def test_broadcast_selection_is_dense_attention(dev):
    """Every block selected by strides of 0: attention over the whole context."""
    _, table, P, c, q, blocks, pages, pos, lens = inputs(27, Q=5, bs=16, NB=11)
    lens[1], pos[1] = 100, torch.arange(95, 100).int()
    blocks = torch.arange(11, dtype=torch.int32).expand(2, 2, 5, 11)
    pages = table[:, None, None, :].expand(2, 2, 5, 11)
    r = R.dsa_paged_attention_ref(q, *c, blocks, pages, pos, lens, 0.1)
    cd = [t.to(dev) for t in c]
    bd = torch.arange(11, dtype=torch.int32, device=dev).expand(2, 2, 5, 11)
    pd = table.to(dev)[:, None, None, :].expand(2, 2, 5, 11)
    out, lse = torch.empty_like(q, device=dev), torch.empty(2, 5, 8, device=dev)
    dsa_paged_attention(q.to(dev), *cd, bd, pd, pos.to(dev), lens.to(dev), out, lse, 0.1)
    check(out, lse, r, 128, 448.0)


def test_broadcast_scales(dev):
    """One scale per head, and one for all keys, by strides of 0."""
    _, _, P, c, q, blocks, pages, pos, lens = inputs(44)
    c[1], c[3] = torch.tensor(0.01).expand(P, 2, 32), torch.tensor([0.02, 0.5])[:, None].expand(P, 2, 32)
    r = R.dsa_paged_attention_ref(q, *c, blocks, pages, pos, lens, 0.1)
    cd = [c[0].to(dev), torch.tensor(0.01, device=dev).expand(P, 2, 32), c[2].to(dev),
          torch.tensor([0.02, 0.5], device=dev)[:, None].expand(P, 2, 32)]
    out, lse = torch.empty_like(q, device=dev), torch.empty(q.shape[:3], device=dev)
    dsa_paged_attention(q.to(dev), *cd, *(t.to(dev) for t in (blocks, pages, pos, lens)), out, lse, 0.1)
    check(out, lse, r, 128, 448.0)


@pytest.mark.parametrize("B,Q,K", [(1, 1, 8), (8, 16, 8)])
def test_in_place(dev, B, Q, K):
    """The output over the queries, with clusters (few rows) and without."""
    _, _, _, c, q, blocks, pages, pos, lens = inputs(45, B=B, Q=Q, K=K, G=16)
    want, lse = run(dev, q, c, blocks, pages, pos, lens, 0.1)
    qd = q.to(dev)
    got = dsa_paged_attention(qd, *(t.to(dev) for t in (*c, blocks, pages, pos, lens)), qd, None, 0.1)
    assert got[0] is qd and torch.equal(qd, want)


_FIRST_IN_CAPTURE = """
import torch
from flagos_kernelgen_72h_shanghai_2026_b200 import *
dev = torch.device("cuda:0")
q = torch.randn(1, 2, 4, 64, device=dev).half()
k, v = torch.randn(1, 2, 2, 64, device=dev).half(), torch.randn(1, 2, 2, 64, device=dev).half()
gamma, pos = torch.ones(64, device=dev), torch.arange(2, dtype=torch.int32, device=dev)[None]
cs = torch.cat([torch.ones(8, 32), torch.zeros(8, 32)], 1).to(dev)
cache = (torch.zeros(3, 2, 16, 64, dtype=torch.int8, device=dev), torch.zeros(3, 2, 16, device=dev),
         torch.zeros(3, 2, 16, 64, dtype=torch.int8, device=dev), torch.zeros(3, 2, 16, device=dev))
table, lens = torch.tensor([[2, 0]], dtype=torch.int32, device=dev), torch.tensor([2], dtype=torch.int32, device=dev)
sel, pages = torch.zeros(1, 2, 2, 1, dtype=torch.int32, device=dev), torch.full((1, 2, 2, 1), 2, dtype=torch.int32, device=dev)
qo, ko, out, k2, v2 = (torch.zeros_like(t) for t in (q, k, q, k, v))
side = torch.cuda.Stream()
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g, stream=side):
    qk_rmsnorm_rope(q, k, gamma, gamma, cs, pos, qo, ko, 1e-6)
    paged_kv_quant_write(ko, v, *cache, table, pos)
    dsa_paged_attention(qo, *cache, sel, pages, pos, lens, out, None, 0.125)
    paged_kv_dequant_read(*cache, table, lens, k2, v2)
g.replay()
torch.cuda.synchronize()
n = q.float() / (q.float().square().mean(-1, keepdim=True) + 1e-6).sqrt()
assert (qo.float() - n).abs().max() < 0.01 and (k2 - ko).abs().max() < 0.03 and (v2 - v).abs().max() < 0.03
assert (out[0, 0].view(2, 2, 64) - v2[0, 0][:, None]).abs().max() < 0.01  # the first token sees itself alone
print("captured")
"""


def test_first_calls_of_a_process_in_a_capture(dev):
    """Nothing was launched, loaded or set up before the capture begins."""
    p = subprocess.run([sys.executable, "-c", _FIRST_IN_CAPTURE], capture_output=True, text=True, timeout=300,
                       cwd=Path(__file__).resolve().parent.parent)
    assert p.returncode == 0 and "captured" in p.stdout, p.stderr[-2000:]


def test_strided_queries_and_outputs(dev):
    _, _, _, c, q, blocks, pages, pos, lens = inputs(28)
    want, _ = run(dev, q, c, blocks, pages, pos, lens, 0.1)
    wide = torch.zeros(2, 3, 12, 128, dtype=BF16, device=dev)
    wide[:, :, 2:10] = q.to(dev)
    buf = torch.full((2, 3, 10, 128), 9.0, dtype=BF16, device=dev)
    dsa_paged_attention(wide[:, :, 2:10], *(t.to(dev) for t in c), blocks.to(dev), pages.to(dev), pos.to(dev),
                        lens.to(dev), buf[:, :, 1:9], None, 0.1)
    assert torch.equal(buf[:, :, 1:9], want) and (buf[:, :, [0, 9]] == 9).all()


def test_no_blocks_no_rows_no_pages(dev):
    _, _, _, c, q, blocks, pages, pos, lens = inputs(29)
    out, lse = run(dev, q, c, blocks[..., :0], pages[..., :0], pos, lens, 0.1)
    assert (out == 0).all() and (lse == -math.inf).all()
    out, lse = run(dev, q, [t[:0] for t in c], blocks, pages, pos, lens, 0.1)
    assert (out == 0).all() and (lse == -math.inf).all()
    run(dev, q[:, :0], c, blocks[:, :, :0], pages[:, :, :0], pos[:, :0], lens, 0.1)


def test_refusals(dev):
    _, _, _, c, q, blocks, pages, pos, lens = inputs(30)
    c = [t.to(dev) for t in c]
    q, blocks, pages, pos, lens = (t.to(dev) for t in (q, blocks, pages, pos, lens))
    out, lse = torch.empty_like(q), torch.empty(q.shape[:3], device=dev)

    def call(q=q, c=c, blocks=blocks, pages=pages, pos=pos, lens=lens, out=out, lse=lse):
        dsa_paged_attention(q, *c, blocks, pages, pos, lens, out, lse, 0.1)

    call()
    small = [t[:, :, :4] for t in c]
    odd = [t[..., :80] if t.dim() == 4 else t for t in c]
    for kw, err in ((dict(q=q.float()), TypeError), (dict(out=out.half()), TypeError), (dict(lse=lse.half()), TypeError),
                    (dict(blocks=blocks.float()), TypeError), (dict(lens=lens.long()), TypeError),
                    (dict(pages=pages.cpu()), TypeError), (dict(c=[c[0], c[1].double(), *c[2:]]), TypeError),
                    (dict(q=q[:, :, :7], out=out[:, :, :7], lse=lse[:, :, :7]), ValueError), (dict(pages=pages[..., :2]), ValueError),
                    (dict(blocks=blocks.transpose(2, 3).contiguous().transpose(2, 3)), ValueError),
                    (dict(lse=lse[:, :, :2]), ValueError), (dict(pos=pos[:, :2]), ValueError), (dict(c=small), ValueError),
                    (dict(q=q[..., :80], out=out[..., :80], c=odd), ValueError),
                    (dict(out=out[:, :, :1].expand_as(out)), ValueError)):
        with pytest.raises(err):
            call(**kw)


def test_results_do_not_depend_on_the_run(dev):
    g, table, P, c, q, blocks, pages, pos, lens = inputs(31, B=3, Q=4, K=8)
    first = run(dev, q, c, blocks, pages, pos, lens, 0.1)
    for _ in range(3):
        again = run(dev, q, c, blocks, pages, pos, lens, 0.1)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


# ------------------------------------------------------------ a layer's operators together
def layer(B, Q, Hq, H, D, bs, NB, K, code, seed):
    g = gen(seed)
    table, P = page_table(g, B, NB)
    c = caches(g, P, H, bs, D, code)
    qkv = torch.randn(B, Q, (Hq + 2 * H) * D, generator=g).to(BF16)
    gq, gk = (1 + 0.1 * torch.randn(D, generator=g) for _ in range(2))
    scores = torch.randn(B, H, Q, NB, generator=g)
    lens = torch.randint(Q + 1, NB * bs + 1, (B,), generator=g).int()
    pos = (lens[:, None] - Q + torch.arange(Q)).int()
    return table, c, qkv, gq, gk, angles(NB * bs, D), scores, lens, pos


def check_layer(dev, B, Q, Hq, H, D, bs, NB, K, code, graph):
    table, c, qkv, gq, gk, cs, scores, lens, pos = layer(B, Q, Hq, H, D, bs, NB, K, code, seed=B * Q + D)
    cd, (td, xd, gqd, gkd, csd, sd, ld, pd) = [t.to(dev) for t in c], (
        t.to(dev) for t in (table, qkv, gq, gk, cs, scores, lens, pos))
    q, k, v = (t.view(B, Q, -1, D) for t in xd.split([Hq * D, H * D, H * D], dim=-1))
    qo, ko = torch.empty(B, Q, Hq, D, dtype=BF16, device=dev), torch.empty(B, Q, H, D, dtype=BF16, device=dev)
    blocks = torch.empty(B, H, Q, K, dtype=torch.int32, device=dev)
    pages = torch.empty_like(blocks)
    out, lse = torch.empty_like(qo), torch.empty(B, Q, Hq, device=dev)
    full_k, full_v = (torch.zeros(B, NB * bs, H, D, dtype=BF16, device=dev) for _ in range(2))

    def step():
        qk_rmsnorm_rope(q, k, gqd, gkd, csd, pd, qo, ko, 1e-6)
        paged_kv_quant_write(ko, v, *cd, td, pd)
        dsa_topk_page_table_transform(sd, td, pd, ld, blocks, pages, bs, K)
        dsa_paged_attention(qo, *cd, blocks, pages, pd, ld, out, lse, D ** -0.5)
        paged_kv_dequant_read(*cd, td, ld, full_k, full_v)

    if graph:
        step()
        torch.cuda.synchronize(dev)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            step()
        for t, h in zip(cd, c):
            t.copy_(h)
        for t in (qo, ko, out, lse, full_k, full_v):
            t.zero_()
        gr.replay()
    else:
        step()
    torch.cuda.synchronize(dev)

    qc, kc, vc = (t.view(B, Q, -1, D) for t in qkv.split([Hq * D, H * D, H * D], dim=-1))
    (we, wsize), (ke, ksize) = R.qk_rmsnorm_rope_ref(qc, kc, gq, gk, cs, pos, qc, kc, 1e-6)
    for got, exact, size in ((qo, we, wsize), (ko, ke, ksize)):
        tol = 2.0 ** -8 * (exact.abs() + 14 * U * size) + 14 * U * size
        assert ((got.cpu().double() - exact).abs() <= tol).all()
    written = R.paged_kv_quant_write_ref(ko.cpu(), vc, *c, table, pos)
    for got, want in zip(cd, written):
        assert torch.equal(got.cpu().view(torch.uint8), want.view(torch.uint8))
    rb, rp = dsa_topk_page_table_transform_ref(scores, table, pos, lens, bs, K)
    assert (blocks.cpu().numpy() == rb).all() and (pages.cpu().numpy() == rp).all()
    now = (written[0].view(code), written[1], written[2].view(code), written[3])
    r = R.dsa_paged_attention_ref(qo.cpu(), *now, blocks.cpu(), pages.cpu(), pos, lens, D ** -0.5)
    check(out, lse, r, D, R.QMAX[code])
    zero = torch.zeros(B, NB * bs, H, D, dtype=BF16)
    for got, exact in zip((full_k, full_v), R.paged_kv_dequant_read_ref(*now, table, lens, zero, zero)):
        assert ((got.cpu().double() - exact).abs() <= (2.0 ** -8 + 3 * U) * exact.abs()).all()


@pytest.mark.parametrize("graph", [False, True], ids=["eager", "graph"])
@pytest.mark.parametrize("B,Q,Hq,H,D,bs,NB,K,code", [
    (1, 1, 8, 2, 128, 64, 8, 4, E4M3),
    (3, 1, 16, 2, 64, 16, 12, 6, INT8),
    (2, 9, 8, 4, 128, 32, 16, 5, E4M3),
], ids=str)
def test_a_layer_step(dev, B, Q, Hq, H, D, bs, NB, K, code, graph):
    check_layer(dev, B, Q, Hq, H, D, bs, NB, K, code, graph)


def test_calls_on_two_streams(dev):
    """Two calls at once on different streams, and a captured one replayed while an eager one runs."""
    a, b = inputs(41, B=4, Q=8, K=8), inputs(42, B=4, Q=8, K=8)
    want = [run(dev, x[4], x[3], *x[5:], 0.1) for x in (a, b)]
    args, outs = [], []
    for x in (a, b):
        args.append([t.to(dev) for t in (x[4], *x[3], *x[5:])])
        outs.append((torch.zeros_like(args[-1][0]), torch.zeros(x[4].shape[:3], device=dev)))
    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    torch.cuda.synchronize(dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=streams[0]):
        dsa_paged_attention(*args[0], *outs[0], 0.1)
    for _ in range(5):
        with torch.cuda.stream(streams[0]):
            graph.replay()
        with torch.cuda.stream(streams[1]):
            dsa_paged_attention(*args[1], *outs[1], 0.1)
    torch.cuda.synchronize(dev)
    for (o, l), (wo, wl) in zip(outs, want):
        assert torch.equal(o, wo) and torch.equal(l, wl)


def test_calls_from_other_threads(dev):
    """Threads that have made no CUDA call of their own, several at once, each on its own stream."""
    x = inputs(43, B=2, Q=4)
    want = run(dev, x[4], x[3], *x[5:], 0.1)
    args = [t.to(dev) for t in (x[4], *x[3], *x[5:])]
    outs = [(torch.zeros_like(args[0]), torch.zeros(x[4].shape[:3], device=dev)) for _ in range(4)]
    streams = [torch.cuda.Stream(dev) for _ in outs]
    torch.cuda.synchronize(dev)
    errors = []

    def work(o, stream):
        try:
            with torch.cuda.stream(stream):
                for _ in range(20):
                    dsa_paged_attention(*args, *o, 0.1)
        except Exception as e:
            errors.append(e)

    threads = [threading.Thread(target=work, args=a) for a in zip(outs, streams)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize(dev)
    assert not errors, errors
    for o, l in outs:
        assert torch.equal(o, want[0]) and torch.equal(l, want[1])


def test_a_first_call_from_a_thread_without_a_context(dev):
    """The C entry point called from a thread that has made no CUDA call at all."""
    from flagos_kernelgen_72h_shanghai_2026_b200 import _kv_lib as L
    q = torch.randn(1, 2, 4, 64, device=dev).to(BF16)
    gamma, cs = torch.ones(64, device=dev), angles(8, 64).to(dev)
    pos = torch.zeros(1, 2, dtype=torch.int32, device=dev)
    want, out = torch.empty_like(q), torch.zeros_like(q)
    k = torch.empty(1, 2, 0, 64, dtype=BF16, device=dev)
    qk_rmsnorm_rope(q, k, gamma, gamma, cs, pos, want, k, 1e-6)
    torch.cuda.synchronize(dev)
    a = L.RopeArgs(struct_size=ctypes.sizeof(L.RopeArgs), dtype=L.DTYPE_BF16, gamma_dtype=L.DTYPE_FP32,
                   pos_dtype=L.DTYPE_INT32, eps=1e-6, B=1, Q=2, Hq=4, Hk=0, D=64, rot=64, max_pos=8)
    a.q, a.q_out = L.Dense(q.data_ptr(), *q.stride()[:3]), L.Dense(out.data_ptr(), *out.stride()[:3])
    a.q_gamma = a.k_gamma = gamma.data_ptr()
    a.cos_sin, a.positions = cs.data_ptr(), pos.data_ptr()
    lib, got = L.load(), []
    t = threading.Thread(target=lambda: got.append(lib.dsa_kv_rope_launch(ctypes.byref(a), None)))
    t.start()
    t.join()
    torch.cuda.synchronize(dev)
    assert got == [L.OK] and torch.equal(out, want)


def test_a_long_row(dev):
    """One row over 8192 selected tokens of a large cache: the sums of the oracle, the bound on n/16 steps."""
    case(dev, 1, 1, 1, 8, 128, 64, 128, 140, BF16, E4M3, seed=50, full=True)


@pytest.mark.parametrize("code", [E4M3, INT8])
def test_offsets_beyond_32_bits(dev, code):
    """A cache of 9 GB, keys and values side by side, against a compact one of the pages in use; queries, new tokens
    and outputs with more than 4 GiB between their sequences. Same bits; the pages 2^32 bytes below stay as they were."""
    B, Q, Hq, H, D, bs, NB, K = 2, 256, 8, 8, 128, 64, 4, 3
    P, below = 70000, 2 ** 32 // (2 * H * bs * D)  # pages of 128 KiB
    g = gen(51)
    high = torch.tensor([[69999, 32768, 50000, 40001], [33000, 65535, 65000, 69000]])
    codes = torch.empty(P, 2, H, bs, D, dtype=torch.uint8, device=dev)
    scales = torch.empty(P, 2, H, bs, device=dev)
    codes[(high - below).to(dev)] = 17
    scales[(high - below).to(dev)] = 17.0
    big = (codes[:, 0].view(code), scales[:, 0], codes[:, 1].view(code), scales[:, 1])
    small = tuple(torch.zeros(B * NB, *t.shape[1:], dtype=t.dtype if t.dtype != code else torch.uint8, device=dev)
                  for t in big)
    small = tuple(t.view(code) if t.dtype == torch.uint8 else t for t in small)
    far = 2 ** 31 + 2 ** 20  # elements from one sequence to the next
    buf = torch.empty(far + 4 * Q * Hq * D, dtype=BF16, device=dev)

    def apart(n, t):  # the n-th tensor of such a buffer
        v = buf[n * Q * Hq * D:].as_strided((B, Q, Hq, D), (far, Hq * D, D, 1))
        return v if t is None else v.copy_(t)

    q, k, v = (torch.randn(B, Q, Hq, D, generator=g).to(BF16).to(dev) for _ in range(3))
    gamma, cs = torch.ones(D, device=dev), angles(NB * bs, D).to(dev)
    pos = torch.arange(Q).expand(B, Q).contiguous().int().to(dev)
    lens = torch.tensor([Q, Q - 5], dtype=torch.int32, device=dev)
    blocks = torch.rand(B, H, Q, NB, generator=g).argsort(-1)[..., :K].contiguous()
    got = []
    for cache, table, wide in ((big, high, True), (small, torch.arange(B * NB).view(B, NB), False)):
        pages = table[:, None, None].expand(B, H, Q, NB).gather(3, blocks).to(dev)
        a, b, c = (apart(n, t) if wide else t.clone() for n, t in enumerate((q, k, v)))
        out = apart(3, None) if wide else torch.empty_like(a)
        lse = torch.empty(B, Q, Hq, device=dev)
        kr, vr = (torch.zeros(B, NB * bs, H, D, dtype=BF16, device=dev) for _ in range(2))
        td = table.to(dev)
        qk_rmsnorm_rope(a, b, gamma, gamma, cs, pos, a, b, 1e-6)
        paged_kv_quant_write(b, c, *cache, td, pos)
        dsa_paged_attention(a, *cache, blocks.to(dev), pages, pos, lens, out, lse, D ** -0.5)
        paged_kv_dequant_read(*cache, td, lens, kr, vr)
        torch.cuda.synchronize(dev)
        got.append([t.cpu().clone() for t in (a, b, out, lse, kr, vr)])
    for x, y in zip(*got):
        assert torch.equal(x, y)
    assert got[0][2].abs().max() > 0 and not any(x.isnan().any() for x in got[0])
    assert (codes[(high - below).to(dev)] == 17).all() and (scales[(high - below).to(dev)] == 17.0).all()
