"""dsa_paged_attention at the ends of its inputs' ranges, against the plain
implementation in 64 bits (oracle/kv_oracle.py).

Tolerances: as in test_dsa_attention_gpu.py (u = 2^-24), with value scales
between 2^-40 and 2^128 instead of near 1:
  exponent log2 of a value scale is off by 2 of its last places, 4u * 128; the
           sums score + log2(vs), - maximum and - log2(vs) round three times, u
           * (|score| + 128) each; the maximum's own rounding cancels. Together
           with the score's factor at most 10u * (|score| + 128).
  sums     a rescaling of the denominator in two steps adds 2^-20; there is at
           most one for every 32 tokens, and one in the join.
  lse      the maximum and the logarithm of the sum may reach 128 + |lse| each and
           cancel: 4u * (|lse| + 256).
"""
import math
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from oracle import kv_oracle as R
from flagos_kernelgen_72h_shanghai_2026_b200 import dsa_paged_attention, paged_kv_quant_write
from test_dsa_attention_gpu import BF16, E4M3, FP16, INT8, U, dev, inputs, run  # noqa: F401

pytestmark = pytest.mark.gpu


def check(out, lse, r, D, qmax):
    score = (D + 16) * 2 * U * r["score"] + 10 * U * (r["score"] + 128) + 2.0 ** -21
    steps = (r["n"] / 32 + 2) * 2.0 ** -20
    rel = 2.0 ** -11 + 2.0 ** -20 + 2 * score + (r["n"] / 16 + 2) * 17 * 2 * U + steps
    floor = r["n"] * 2.0 ** -31 * qmax * r["top"]
    tol = rel[..., None] * r["size"] + floor[..., None]
    g, half = out.cpu().double(), torch.finfo(out.dtype).eps / 2
    assert torch.equal(g.isnan(), r["out"].isnan())
    off = ((g - r["out"]).abs() - half * (r["out"].abs() + tol) - tol).nan_to_num(-1.0)
    assert float(off.max()) <= 0, f"out is off by {float(off.max()):.3g} more than allowed"
    x, empty = lse.cpu().double(), r["lse"] == -math.inf
    assert torch.equal(x == -math.inf, empty) and torch.equal(x.isnan(), r["lse"].isnan())
    tol = score + 2.0 ** -20 + (r["n"] / 16 + 20) * U + 4 * U * (r["lse"].abs() + 256).nan_to_num(posinf=0.0) + steps
    off = ((x - r["lse"]).abs() - tol)[~empty].nan_to_num(-1.0)
    assert off.numel() == 0 or float(off.max()) <= 0, f"lse is off by {float(off.max()):.3g} more than allowed"


# B, Q, K, G, D, block_size: a CTA alone (rows enough), and clusters of two to eight
SHAPES = [(2, 3, 6, 4, 128, 32), (16, 4, 4, 16, 64, 64), (1, 1, 40, 4, 64, 64), (1, 1, 24, 16, 128, 64),
          (2, 2, 8, 16, 256, 32), (1, 1, 8, 1, 256, 64)]


# ------------------------------------------------------ value scales far apart
def test_one_huge_value_among_zeros(dev):
    """Written by the cache's own write: 31 value vectors of zeros (scale 1e-12) and one of 3e30, equal scores."""
    H, D, bs = 1, 64, 32
    k, v = torch.zeros(1, bs, H, D, dtype=BF16, device=dev), torch.zeros(1, bs, H, D, dtype=BF16, device=dev)
    v[0, 3] = 3e30
    cache = tuple(t.to(dev) for t in (torch.zeros(1, H, bs, D).to(E4M3), torch.zeros(1, H, bs),
                                      torch.zeros(1, H, bs, D).to(E4M3), torch.zeros(1, H, bs)))
    zero = torch.zeros(1, 1, dtype=torch.int32, device=dev)
    paged_kv_quant_write(k, v, *cache, zero, torch.arange(bs, dtype=torch.int32, device=dev)[None])
    q = torch.ones(1, 1, 1, D, dtype=BF16, device=dev)
    out, lse = torch.zeros_like(q), torch.zeros(1, 1, 1, device=dev)
    dsa_paged_attention(q, *cache, zero[None, None], zero[None, None], zero + bs - 1, zero[0] + bs, out, lse, 1.0)
    want = float(v[0, 3, 0, 0]) / bs
    # out: the code is exact (448), its scale rounded (u), the weight 2^-11 and the bound's 2^-14 of exponents
    assert abs(float(lse) - math.log(bs)) <= 4 * U * 260 + 2.0 ** -19
    assert ((out.double().cpu() - want).abs() <= want * (2.0 ** -8 + 2.0 ** -10)).all()


@pytest.mark.parametrize("how", ["spread", "rising", "falling", "first", "last"])
@pytest.mark.parametrize("code", [E4M3, INT8])
@pytest.mark.parametrize("B,Q,K,G,D,bs", SHAPES, ids=str)
def test_value_scales_far_apart(dev, B, Q, K, G, D, bs, code, how):
    """Value scales from the least (1e-12) to 2^118: in no order, with the position, at one token alone."""
    g, table, P, c, q, blocks, pages, pos, lens = inputs(60 + K, B=B, Q=Q, G=G, D=D, bs=bs, K=K, NB=K, code=code)
    blocks = torch.arange(K).expand(B, 2, Q, K).int().contiguous()
    pages = table[:, None, None, :].expand(B, 2, Q, K).contiguous()
    n = K * bs
    at = torch.arange(n).view(K, 1, bs)
    for b in range(B):
        if how == "spread":
            ex = torch.randint(-39, 119, (K, 2, bs), generator=g).float()
        elif how in ("rising", "falling"):
            ex = -39 + 157 * at.expand(K, 2, bs).float() / (n - 1)
            ex = ex if how == "rising" else ex.flip(0, 2)
        else:
            ex = torch.where(at == (0 if how == "first" else n - 1), 118.0, -40.0).expand(K, 2, bs)
        c[3][table[b].long()] = torch.exp2(ex).clamp(min=R.MIN_SCALE)
    r = R.dsa_paged_attention_ref(q, *c, blocks, pages, pos, lens, 0.1)
    out, lse = run(dev, q, c, blocks, pages, pos, lens, 0.1)
    check(out, lse, r, D, R.QMAX[code])


@pytest.mark.parametrize("code", [E4M3, INT8])
@pytest.mark.parametrize("B,Q,K,G,D,bs", SHAPES, ids=str)
def test_lse_holds_no_values(dev, B, Q, K, G, D, bs, code):
    """Value vectors with a NaN or an infinity, stored by the write with the scale NaN: out is NaN in the rows that see
    them, lse what the scores give. The same with a scale of infinity."""
    g, table, P, c, q, blocks, pages, pos, lens = inputs(70 + K, B=B, Q=Q, G=G, D=D, bs=bs, K=K, NB=K + 2, code=code)
    v = torch.randn(B, 3, 2, D, generator=g).to(BF16)
    v[0, 0, 0, 5], v[0, 1, 1, D - 1], v[-1, 2, 0] = math.nan, math.inf, -math.inf
    at = torch.tensor([[0, bs + 1, (K + 2) * bs - Q]]).expand(B, 3).int().contiguous()
    cd = tuple(t.to(dev) for t in c)
    paged_kv_quant_write(torch.zeros_like(v).to(dev), v.to(dev), *cd, table.to(dev), at.to(dev))
    c = [t.cpu() for t in cd]
    r = R.dsa_paged_attention_ref(q, *c, blocks, pages, pos, lens, 0.1)
    out, lse = run(dev, q, c, blocks, pages, pos, lens, 0.1)
    assert r["out"].isnan().any() and not r["lse"].isnan().any()
    assert torch.equal(out.cpu().isnan(), r["out"].isnan())
    r["out"], r["size"] = r["out"].nan_to_num(0.0), r["size"].nan_to_num(0.0)
    r["top"] = r["top"].nan_to_num(0.0)
    check(out.nan_to_num(0.0), lse, r, D, R.QMAX[code])
    c[3] = c[3].nan_to_num(math.inf)
    inf_out, inf_lse = run(dev, q, c, blocks, pages, pos, lens, 0.1)
    assert torch.equal(inf_out.isnan(), out.isnan()) and torch.equal(inf_lse, lse)


def test_all_values_without_a_scale(dev):
    """Every value scale NaN: no finite value scale to hold the maximum."""
    _, _, _, c, q, blocks, pages, pos, lens = inputs(71)
    c[3] = torch.full_like(c[3], math.nan)
    r = R.dsa_paged_attention_ref(q, *c, blocks, pages, pos, lens, 0.1)
    out, lse = run(dev, q, c, blocks, pages, pos, lens, 0.1)
    r["out"], r["size"], r["top"] = (torch.zeros_like(r[k]) for k in ("out", "size", "top"))
    assert out.isnan().all()
    check(torch.zeros_like(out), lse, r, 128, 448.0)


# ---------------------------------------------------------------- large scores
LN2 = 0.6931471805599453  # times log2(e) in fp32: 1


@pytest.mark.parametrize("above", [0, 1])
@pytest.mark.parametrize("e", [22, 23, 24, 25, 26, 27, 28])
def test_scores_a_few_places_apart(dev, e, above):
    """Scores of 2^e in units of ln 2, one to eight of their last places apart, the larger ones in a warp's second chunk.
    Every step up to the weights is exact, and these are powers of two: out is off by its own rounding, the sums' and
    the exponentials' (2^-20 at most); a weight below 2^-20 may go."""
    ulp = 2.0 ** (e - 23)
    B, Q, H, K, D, bs = 1, 128, 4, 8, 64, 64
    g, table, P, c, _, _, _, pos, lens = inputs(80, B=B, Q=Q, H=H, G=1, D=D, bs=bs, K=K, NB=K, code=INT8)
    blocks = torch.arange(K).expand(B, H, Q, K).int().contiguous()
    pages = table[:, None, None, :].expand(B, H, Q, K).contiguous()
    pos[:] = K * bs - 1
    q = torch.zeros(B, Q, H, D, dtype=BF16)
    q[..., 0], q[..., 1] = 2.0 ** (e - 6), ulp
    for delta in (1, 2, 4, 8):
        if delta * ulp > 64:
            continue
        kc, vc = torch.zeros(P, H, bs, D, dtype=torch.int8), torch.ones(P, H, bs, D, dtype=torch.int8)
        kc[..., 0], kc[..., 1] = 64, above
        high = table[0, 4:].long()
        kc[high, :, 9, 1] = above + delta
        vc[high, :, 9] = 3
        one = torch.ones(P, H, bs)
        out, _ = run(dev, q, (kc, one, vc, one), blocks, pages, pos, lens, LN2)
        w = 4 * 2.0 ** (delta * ulp)
        want = (K * bs - 4 + 3 * w) / (K * bs - 4 + w)
        assert abs(out.float() - want).max() <= want * (2.0 ** -8 + 2.0 ** -18) + 512 * 2.0 ** -20, (delta, want)


@pytest.mark.parametrize("B,Q,K,G,D,bs", SHAPES, ids=str)
def test_scores_of_minus_infinity(dev, B, Q, K, G, D, bs):
    """A query of -inf on keys that are all positive there: tokens, but no finite score. out is NaN and not the zeros of
    a row without tokens, lse is -inf for both; where some tokens have the code 0 there, the score is NaN."""
    _, _, _, c, q, blocks, pages, pos, lens = inputs(85 + G, B=B, Q=Q, G=G, D=D, bs=bs, K=K, NB=K + 1, code=INT8)
    c[0][..., 3] = c[0][..., 3].abs().clamp(min=1)
    c[0][c[1].argmax() % c[0].shape[0], :, 0, 3] = 0
    q[..., 0, 3] = -math.inf
    if Q > 1:
        pos[0, 1] = -1
    r = R.dsa_paged_attention_ref(q, *c, blocks, pages, pos, lens, 0.1)
    out, lse = run(dev, q, c, blocks, pages, pos, lens, 0.1)
    seen = (pos >= 0)[..., None].expand(r["lse"].shape)
    first = torch.arange(2 * G) == 0
    assert torch.equal(out.cpu().isnan(), r["out"].isnan())
    assert out.cpu()[seen & first].isnan().all() and (out.cpu()[~seen] == 0).all()
    assert torch.equal(lse.cpu() == -math.inf, r["lse"] == -math.inf)
    ok = {k: v[~first.expand(r["lse"].shape)] for k, v in r.items()}
    check(out.cpu()[~first.expand(r["lse"].shape)], lse.cpu()[~first.expand(r["lse"].shape)], ok, D, 127.0)


# ------------------------------------------------------- heads of unlike size
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("code", [E4M3, INT8])
@pytest.mark.parametrize("B,Q,K,G,D,bs", [*SHAPES, (1, 2, 5, 40, 64, 48)], ids=str)
def test_heads_of_unlike_size(dev, B, Q, K, G, D, bs, code, dtype):
    """Query heads up to 2^230 (fp16: 2^24) apart that share a key head: each has the scores of its own size, also beside
    heads of zeros and of values that are not finite."""
    _, table, P, c, q, blocks, pages, pos, lens = inputs(90 + G, B=B, Q=Q, G=G, D=D, bs=bs, K=K, NB=K + 1, code=code)
    most = 115 if dtype == BF16 else 12
    ex = torch.tensor([0, -9, most, -most, 3, -17, most - 5, 0, 9, -3])[torch.arange(2 * G) % 10]
    q = q.float() * torch.exp2(ex.float())[:, None]
    q[..., 5 % (2 * G), :] = 0
    if G > 2:
        q[0, 0, 1, 3], q[0, 0, G + 1, 7] = math.nan, math.inf
    q = q.to(dtype)
    r = R.dsa_paged_attention_ref(q, *c, blocks, pages, pos, lens, 0.1)
    out, lse = run(dev, q, c, blocks, pages, pos, lens, 0.1)
    bad = ~q.isfinite().all(-1)
    got_o, got_l = out.cpu(), lse.cpu()
    assert got_o[bad].isnan().all()
    ok = {k: v[~bad] for k, v in r.items()}
    check(got_o[~bad], got_l[~bad], ok, D, R.QMAX[code])


# ------------------------------------------------- captured, and two at a time
_FIRST_CLUSTER_IN_CAPTURE = """
import torch
from flagos_kernelgen_72h_shanghai_2026_b200 import *
dev = torch.device("cuda:0")
g = torch.Generator().manual_seed(3)
K, bs, D = 40, 64, 128
q = torch.randn(1, 1, 4, D, generator=g).half().to(dev)
kc = torch.randint(-127, 128, (K, 1, bs, D), generator=g).to(torch.int8)
vc = torch.randint(-127, 128, (K, 1, bs, D), generator=g).to(torch.int8)
cache = (kc.to(dev), torch.full((K, 1, bs), 0.01, device=dev), vc.to(dev), torch.full((K, 1, bs), 0.02, device=dev))
sel = torch.arange(K, dtype=torch.int32).view(1, 1, 1, K).to(dev)
pos, lens = torch.full((1, 1), K * bs - 1, dtype=torch.int32, device=dev), torch.full((1,), K * bs, dtype=torch.int32, device=dev)
out = torch.zeros_like(q)
side = torch.cuda.Stream()
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph, stream=side):
    dsa_paged_attention(q, *cache, sel, sel, pos, lens, out, None, 0.1)
graph.replay()
torch.cuda.synchronize()
k, v = kc.view(-1, D).double() * 0.01, vc.view(-1, D).double() * 0.02
want = torch.softmax(q.cpu().view(4, D).double() @ k.T * 0.1, -1) @ v
assert (out.cpu().view(4, D).double() - want).abs().max() < 0.01
print("captured")
"""


def test_the_first_call_of_a_process_in_a_capture_with_a_cluster(dev):
    """What a cluster's size is chosen from is asked of the device inside the capture. Values of up to 2.5 in an average
    of 2560: a wrong or missing part of the join shows in the second digit."""
    p = subprocess.run([sys.executable, "-c", _FIRST_CLUSTER_IN_CAPTURE], capture_output=True, text=True, timeout=300,
                       cwd=Path(__file__).resolve().parent.parent)
    assert p.returncode == 0 and "captured" in p.stdout, p.stderr[-2000:]


def test_rare_rows_in_graphs_on_two_streams(dev):
    """A graph of calls whose rows go through both forms of the loop, replayed while other calls run: same bits."""
    calls = []
    for n, (B, Q, K, G, D, bs) in enumerate(SHAPES):
        g, _, _, c, q, blocks, pages, pos, lens = inputs(120 + n, B=B, Q=Q, G=G, D=D, bs=bs, K=K, NB=K + 1)
        big = torch.rand(c[3].shape, generator=g) < 0.02
        c[3] = torch.where(big, 2.0 ** 90, c[3])
        q[0, 0, 0] *= 2.0 ** 20
        args = [t.to(dev) for t in (q, *c, blocks, pages, pos, lens)]
        want = run(dev, q, c, blocks, pages, pos, lens, 0.1)
        outs = [(torch.zeros_like(want[0]), torch.zeros_like(want[1])) for _ in range(2)]
        calls.append((args, want, outs))
    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    torch.cuda.synchronize(dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=streams[0]):
        for args, _, outs in calls:
            dsa_paged_attention(*args, *outs[0], 0.1)
    for _ in range(5):
        with torch.cuda.stream(streams[0]):
            graph.replay()
        with torch.cuda.stream(streams[1]):
            for args, _, outs in reversed(calls):
                dsa_paged_attention(*args, *outs[1], 0.1)
    torch.cuda.synchronize(dev)
    for _, want, outs in calls:
        for out, lse in outs:
            assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
