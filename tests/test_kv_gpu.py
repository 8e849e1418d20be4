"""The paged-KV-cache operators on the GPU: libdsa_kv.so against the plain
implementations in 64 bits (oracle/kv_oracle.py).

Tolerances. u = 2^-24 is half a step of fp32. A result rounded once to a
16-bit type T from a value v32 that is off by e from the exact v is off by at
most half(T) * (|v| + e) + e, half(T) = finfo(T).eps / 2; below the smallest
normal number of fp16 its half step is 2^-25.
"""
import pytest
import torch

from oracle import kv_oracle as R
from flagos_kernelgen_72h_shanghai_2026_b200 import (_kv_lib, dsa_paged_attention, paged_kv_dequant_read,
                                                     paged_kv_quant_write, qk_rmsnorm_rope)
from _kv_cases import angles, caches, gen, layout, page_table

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
E4M3, INT8 = torch.float8_e4m3fn, torch.int8


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.fail("this test needs a CUDA device (run with -m 'not gpu' on CPU-only hosts)")
    from flagos_kernelgen_72h_shanghai_2026_b200._build import build_kv_lib
    build_kv_lib()
    return torch.device("cuda:0")


def check_rounded(got, exact, err32, what):
    """`got` is `exact` rounded to got's type, from a 32-bit value off by at most err32."""
    g, half = got.cpu().double(), torch.finfo(got.dtype).eps / 2
    assert torch.equal(g.isnan(), exact.isnan()), what
    tol = half * (exact.abs() + err32) + err32 + (2.0 ** -25 if got.dtype == FP16 else 0.0)
    off = ((g - exact).abs() - tol).nan_to_num(-1.0)
    most = float(off.max()) if off.numel() else 0.0
    assert most <= 0, f"{what}: off by {most:.3g} more than allowed"


# ----------------------------------------------------------------------- rope
def rope_inputs(B, Q, Hq, Hk, D, dtype, gamma_dtype, seed, max_pos=300, fused=True):
    g = gen(seed)
    qkv = torch.randn(B, Q, (Hq + 2 * Hk) * D, generator=g).to(dtype)
    if fused:
        q, k = qkv[..., :Hq * D].view(B, Q, Hq, D), qkv[..., Hq * D:(Hq + Hk) * D].view(B, Q, Hk, D)
    else:
        q = qkv[..., :Hq * D].reshape(B, Q, Hq, D).clone()
        k = qkv[..., Hq * D:(Hq + Hk) * D].reshape(B, Q, Hk, D).clone()
    gq, gk = ((1 + 0.2 * torch.randn(D, generator=g)).to(gamma_dtype) for _ in range(2))
    pos = torch.randint(0, max_pos, (B, Q), generator=g)
    return q, k, gq, gk, pos


def check_rope(dev, q, k, gq, gk, cs, pos, eps=1e-6, interleaved=False, in_place=False):
    old_q, old_k = torch.full_like(q, 3.0), torch.full_like(k, -5.0)
    qd, kd = q.to(dev), k.to(dev)
    if in_place:
        old_q, old_k, qo, ko = q, k, qd, kd
    else:
        qo, ko = old_q.to(dev), old_k.to(dev)
    out = qk_rmsnorm_rope(qd, kd, gq.to(dev), gk.to(dev), cs.to(dev), pos.to(dev), qo, ko, eps, interleaved=interleaved)
    assert out[0] is qo and out[1] is ko
    torch.cuda.synchronize(dev)
    want = R.qk_rmsnorm_rope_ref(q, k, gq, gk, cs, pos, old_q, old_k, eps, interleaved)
    for got, (exact, size), what in zip(out, want, "qk"):
        # sum of squares: 4 products by fma into each of two sums, 6 sums across them and the lanes, all terms
        # positive: 10 u; times 1/D (rounded: u) plus eps by fma (u): 12 u; its root halves that: 6 u, rsqrt's 2 ulp
        # are at most 4 u: 10 u. gamma times cosine or sine u, times x u, the sum of the two products by fma u, times
        # the root u: 14 u of the terms.
        check_rounded(got, exact, 14 * U * size, what)


@pytest.mark.parametrize("B,Q,Hq,Hk,D,rot,dtype,gdt,inter", [
    (1, 1, 32, 8, 128, 128, BF16, BF16, False),
    (1, 1, 1, 1, 64, 64, FP16, FP32, True),
    (2, 7, 5, 3, 128, 64, FP16, FP16, False),
    (3, 5, 4, 2, 256, 256, BF16, FP32, False),
    (2, 3, 7, 1, 256, 64, FP16, BF16, True),
    (2, 9, 3, 1, 80, 32, BF16, BF16, False),
    (1, 33, 6, 2, 96, 96, FP16, FP32, False),
    (2, 4, 2, 2, 192, 192, BF16, BF16, True),
    (1, 5, 2, 1, 8, 8, FP16, FP32, True),
    (1, 5, 2, 1, 24, 16, BF16, FP32, False),
    (1, 6, 4, 0, 64, 32, BF16, FP32, False),
    (1, 6, 4, 4, 64, 0, BF16, FP32, False),
], ids=str)
def test_rope_against_64_bits(dev, B, Q, Hq, Hk, D, rot, dtype, gdt, inter):
    q, k, gq, gk, pos = rope_inputs(B, Q, Hq, Hk, D, dtype, gdt, seed=D + rot + Q)
    check_rope(dev, q, k, gq, gk, angles(300, rot), pos, interleaved=inter)


@pytest.mark.parametrize("inter", [False, True])
def test_rope_padding_far_positions_and_in_place(dev, inter):
    q, k, gq, gk, pos = rope_inputs(3, 6, 4, 2, 64, BF16, FP32, seed=5, fused=False)
    pos[0, 2:] = -1
    pos[2, 0], pos[1, 3], pos[1, 4] = 299, 300, 2 ** 31 - 1
    check_rope(dev, q, k, gq, gk, angles(300, 64), pos.int(), interleaved=inter)
    pos[1, 4] = 2 ** 40
    check_rope(dev, q, k, gq, gk, angles(300, 64), pos, interleaved=inter, in_place=True)


@pytest.mark.parametrize("B,Q,Hq,Hk,D,rot,dtype,gdt,inter", [
    (3, 700, 5, 1, 128, 128, BF16, BF16, False),
    (2, 1201, 9, 2, 64, 32, FP16, FP32, True),
    (1, 1500, 3, 3, 256, 256, BF16, FP32, False),
    (2, 611, 18, 0, 96, 64, FP16, FP16, False),
    (1, 1185, 2, 2, 192, 128, BF16, FP32, True),
    (37, 32, 1, 0, 128, 128, BF16, BF16, False),
], ids=str)
def test_rope_many_tokens(dev, B, Q, Hq, Hk, D, rot, dtype, gdt, inter):
    """More steps than warps: each walks over several, through padded tokens, ends of sequences and far positions."""
    q, k, gq, gk, pos = rope_inputs(B, Q, Hq, Hk, D, dtype, gdt, seed=B + Q)
    g = gen(Q)
    pos = torch.where(torch.rand(pos.shape, generator=g) < 0.1, -1, pos)
    pos[:, -3:] = -1
    pos[0, 5], pos[-1, 9] = 300, 2 ** 30
    check_rope(dev, q, k, gq, gk, angles(300, rot), pos, interleaved=inter)


def test_rope_zero_and_huge_heads(dev):
    q, k, gq, gk, pos = rope_inputs(1, 4, 2, 2, 128, BF16, FP32, seed=6)
    q = q.clone()
    q[0, 0, 0] = 0
    q[0, 1] *= 1e15
    q[0, 2] *= 1e-15
    check_rope(dev, q, k, gq, gk, angles(300, 128), pos, eps=1e-5)


def test_rope_strided_outputs_leave_the_rest(dev):
    """Queries and keys written into slices of one buffer: what lies between them stays."""
    q, k, gq, gk, pos = (t.to(dev) for t in rope_inputs(2, 5, 4, 2, 64, FP16, FP16, seed=7))
    cs = angles(300, 64).to(dev)
    buf = torch.full((2, 5, 10, 64), 9.0, dtype=FP16, device=dev)
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    qk_rmsnorm_rope(q, k, gq, gk, cs, pos, qo, ko, 1e-6)
    qk_rmsnorm_rope(q, k, gq, gk, cs, pos, buf[:, :, 1:5], buf[:, :, 6:8], 1e-6)
    assert torch.equal(buf[:, :, 1:5], qo) and torch.equal(buf[:, :, 6:8], ko)
    assert (buf[:, :, [0, 5, 8, 9]] == 9).all()


# ---------------------------------------------------------------------- cache
def same_bytes(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


def to_dev(ts, dev, how="dense"):
    return tuple(layout(t.to(dev), how) for t in ts)


@pytest.mark.parametrize("how", ["dense", "nhd", "pair"])
@pytest.mark.parametrize("B,Q,H,D,bs,NB,dtype,code", [
    (1, 1, 1, 64, 16, 2, BF16, E4M3),
    (3, 5, 8, 128, 64, 3, BF16, E4M3),
    (2, 37, 3, 64, 10, 7, FP16, INT8),
    (2, 9, 2, 256, 48, 2, FP16, E4M3),
    (1, 70, 5, 16, 1, 80, BF16, INT8),
    (4, 3, 1, 112, 7, 5, BF16, INT8),
    (2, 11, 2, 192, 32, 3, FP16, INT8),
], ids=str)
def test_write_is_exact(dev, B, Q, H, D, bs, NB, dtype, code, how):
    g = gen(B * Q + D)
    table, P = page_table(g, B, NB)
    c = caches(g, P, H, bs, D, code)
    kv = torch.randn(B, Q, 2 * H * D, generator=g).to(dtype)
    k, v = kv[..., :H * D].view(B, Q, H, D), kv[..., H * D:].view(B, Q, H, D)
    pos = torch.stack([torch.randperm(NB * bs, generator=g)[:Q] for _ in range(B)])
    cd = to_dev(c, dev, how)
    out = paged_kv_quant_write(k.to(dev), v.to(dev), *cd, table.to(dev), pos.to(dev))
    assert all(o is t for o, t in zip(out, cd))
    for got, want in zip(out, R.paged_kv_quant_write_ref(k, v, *c, table, pos)):
        assert same_bytes(got.cpu(), want)


@pytest.mark.parametrize("code", [E4M3, INT8])
def test_write_skips_what_has_no_cell(dev, code):
    """Padding, positions behind the table, pages that do not exist; rows of zeros, NaN and infinities."""
    g = gen(11)
    B, Q, H, D, bs, NB = 3, 8, 2, 64, 16, 4
    table, P = page_table(g, B, NB, dtype=torch.int64)
    table[1, 0], table[1, 1], table[1, 2] = -1, P, 2 ** 40
    c = caches(g, P, H, bs, D, code)
    k, v = (torch.randn(B, Q, H, D, generator=g).to(BF16) for _ in range(2))
    k[0, 0, 0], k[0, 1, 1, 3], k[0, 2, 0, 5], v[0, 3, 1, 63] = 0, float("nan"), float("inf"), -float("inf")
    v[2, 1], v[2, 2] = 1e-30, 3e38
    pos = torch.randperm(NB * bs, generator=g)[:Q].repeat(B, 1)
    pos[2, 4:] = torch.tensor([-1, NB * bs, 2 ** 40, -2 ** 40])
    cd = to_dev(c, dev)
    paged_kv_quant_write(k.to(dev), v.to(dev), *cd, table.to(dev), pos.to(dev))
    for got, want in zip(cd, R.paged_kv_quant_write_ref(k, v, *c, table, pos)):
        assert same_bytes(got.cpu().nan_to_num(-7.0) if got.dtype == FP32 else got.cpu(),
                          want.nan_to_num(-7.0) if want.dtype == FP32 else want)


@pytest.mark.parametrize("how", ["dense", "nhd", "pair"])
@pytest.mark.parametrize("B,S,H,D,bs,NB,dtype,code", [
    (1, 1, 1, 64, 16, 2, BF16, E4M3),
    (3, 100, 8, 128, 64, 2, BF16, E4M3),
    (2, 65, 3, 64, 10, 7, FP16, INT8),
    (2, 90, 2, 256, 48, 2, FP16, E4M3),
    (2, 50, 5, 16, 1, 40, BF16, INT8),
    (4, 30, 1, 112, 7, 5, FP16, INT8),
], ids=str)
def test_read_against_64_bits(dev, B, S, H, D, bs, NB, dtype, code, how):
    g = gen(S + D)
    table, P = page_table(g, B, NB)
    c = caches(g, P, H, bs, D, code)
    lens = torch.randint(0, S + 20, (B,), generator=g)
    lens[0] = S
    ko, vo = torch.full((B, S, H, D), 3.0, dtype=dtype), torch.full((B, S, H, D), -5.0, dtype=dtype)
    out = paged_kv_dequant_read(*to_dev(c, dev, how), table.to(dev), lens.to(dev), ko.to(dev), vo.to(dev))
    for got, exact in zip(out, R.paged_kv_dequant_read_ref(*c, table, lens, ko, vo)):
        check_rounded(got, exact, U * exact.abs(), "read")  # one product in fp32


def test_read_ends_bad_pages_and_nan(dev):
    g = gen(13)
    B, S, H, D, bs, NB = 4, 40, 2, 64, 16, 3
    table, P = page_table(g, B, NB)
    table[1, 1], table[1, 2] = -1, P
    c = list(caches(g, P, H, bs, D, INT8))
    c[1][table[0, 0], 1, 3] = float("nan")
    lens = torch.tensor([40, 48, 0, -3], dtype=torch.int32)
    ko, vo = torch.full((B, S, H, D), 3.0, dtype=FP16), torch.full((B, S, H, D), -5.0, dtype=FP16)
    out = paged_kv_dequant_read(*to_dev(c, dev), table.to(dev), lens.to(dev), ko.to(dev), vo.to(dev))
    for got, exact in zip(out, R.paged_kv_dequant_read_ref(*c, table, lens, ko, vo)):
        check_rounded(got, exact, U * exact.abs(), "read")
    assert out[0][0, 3, 1].isnan().all()


def test_a_cache_without_pages(dev):
    """No page exists: a write has no cell, a read gives zeros."""
    c = tuple(torch.empty(0, 2, 16, *d, dtype=t, device=dev) for d, t in (((64,), E4M3), ((), FP32)) * 2)
    k = torch.ones(1, 3, 2, 64, dtype=BF16, device=dev)
    table, pos = torch.zeros(1, 2, dtype=torch.int32, device=dev), torch.zeros(1, 3, dtype=torch.int32, device=dev)
    paged_kv_quant_write(k, k, *c, table, pos)
    ko, vo = torch.ones_like(k), torch.ones_like(k)
    paged_kv_dequant_read(*c, table, torch.tensor([2], device=dev), ko, vo)
    assert (ko[0, :2] == 0).all() and (vo[0, :2] == 0).all() and (ko[0, 2] == 1).all()


def test_refusals(dev):
    q = torch.zeros(1, 2, 4, 64, dtype=BF16, device=dev)
    k, gm = q[:, :, :2].contiguous(), torch.ones(64, device=dev)
    cs, pos = angles(8, 64).to(dev), torch.zeros(1, 2, dtype=torch.int32, device=dev)

    def rope(q=q, k=k, gq=gm, gk=gm, cs=cs, pos=pos, qo=None, ko=None, **kw):
        qk_rmsnorm_rope(q, k, gq, gk, cs, pos, torch.empty_like(q) if qo is None else qo,
                        torch.empty_like(k) if ko is None else ko, 1e-6, **kw)

    rope()
    for kw, err in ((dict(q=q.float()), TypeError), (dict(k=k.half()), TypeError), (dict(cs=cs.half()), TypeError),
                    (dict(pos=pos.float()), TypeError), (dict(gk=gm.half()), TypeError),
                    (dict(pos=pos.cpu()), TypeError), (dict(q=q[0]), ValueError), (dict(pos=pos[:, :1]), ValueError),
                    (dict(gq=gm[:32]), ValueError), (dict(qo=q[:, :, :3]), ValueError), (dict(cs=cs[:, ::2]), ValueError),
                    (dict(cs=cs[:, :24].contiguous()), ValueError), (dict(q=q[..., 4:36], qo=q[..., :32]), ValueError)):
        with pytest.raises(err):
            rope(**kw)

    c = tuple(t.to(dev) for t in caches(gen(1), 3, 2, 16, 64, E4M3))
    table, lens = torch.zeros(1, 2, dtype=torch.int32, device=dev), torch.ones(1, dtype=torch.int32, device=dev)

    def write(k=k, v=k, c=c, table=table, pos=pos):
        paged_kv_quant_write(k, v, *c, table, pos)

    write()
    for kw, err in ((dict(k=k.float()), TypeError), (dict(v=k.half()), TypeError), (dict(table=table.float()), TypeError),
                    (dict(c=(c[0], c[1].half(), *c[2:])), TypeError),
                    (dict(c=(c[0].view(torch.uint8), *c[1:])), TypeError),
                    (dict(c=(c[0], c[1], c[2].view(torch.int8), c[3])), TypeError),
                    (dict(v=k[:, :1]), ValueError), (dict(k=q, v=q), ValueError), (dict(table=table[0]), ValueError),
                    (dict(pos=pos[0]), ValueError), (dict(c=(c[0], c[1][:2], *c[2:])), ValueError),
                    (dict(c=(c[0][:, :1].expand(3, 2, 16, 64), *c[1:])), ValueError)):
        with pytest.raises(err):
            write(**kw)
    with pytest.raises(ValueError):
        paged_kv_dequant_read(*c, table, lens, k[:, :1].expand(1, 2, 2, 64), k)
    with pytest.raises(ValueError):
        paged_kv_dequant_read(*c, table, pos, k, k)


# ----------------------------------------------------------- streams and graphs
def test_write_and_read_on_a_side_stream_and_in_a_graph(dev):
    g = gen(17)
    B, Q, H, D, bs, NB = 2, 6, 4, 128, 16, 3
    table, P = page_table(g, B, NB)
    c = caches(g, P, H, bs, D, E4M3)
    k, v = (torch.randn(B, Q, H, D, generator=g).to(BF16) for _ in range(2))
    pos = torch.arange(Q).repeat(B, 1).int()
    lens = torch.full((B,), Q, dtype=torch.int32)
    want = R.paged_kv_dequant_read_ref(*(w if i % 2 else w.view(E4M3) for i, w in enumerate(
        R.paged_kv_quant_write_ref(k, v, *c, table, pos))), table, lens, k, v)
    cd = to_dev(c, dev)
    kd, vd, td, pd, ld = (t.to(dev) for t in (k, v, table, pos, lens))
    ko, vo = torch.zeros_like(kd), torch.zeros_like(vd)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))

    def both():
        paged_kv_quant_write(kd, vd, *cd, td, pd)
        paged_kv_dequant_read(*cd, td, ld, ko, vo)

    with torch.cuda.stream(side):
        both()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            both()
    for n in range(2):
        for t in (*cd, ko, vo):
            t.zero_()
        torch.cuda.synchronize(dev)
        graph.replay()
        torch.cuda.synchronize(dev)
        for got, exact in zip((ko, vo), want):
            check_rounded(got, exact, U * exact.abs(), f"replay {n}")


# ------------------------------------------------------------ C++ launch path
def test_both_launch_paths_give_the_same_bytes(dev):
    """The C++ launch path takes every one of these calls (strided inputs and parameters among them) and gives what
    the ctypes path gives."""
    from flagos_kernelgen_72h_shanghai_2026_b200._build import build_fast_ext
    build_fast_ext()
    fast = _kv_lib._fast
    assert fast is not None, "C++ launch path not loaded"
    g = gen(19)
    B, Q, Hq, H, D, bs, NB = 2, 3, 4, 2, 64, 16, 3
    table, P = page_table(g, B, NB)
    c = caches(g, P, H, bs, D, E4M3)
    q, k, gq, gk, _ = rope_inputs(B, Q, Hq, H, D, BF16, FP32, seed=20)
    lens = torch.tensor([40, 30], dtype=torch.int32)
    pos = (lens[:, None] - Q + torch.arange(Q)).int()
    cs, td, pd, ld, qd, kd = (t.to(dev) for t in (angles(48, D), table, pos, lens, q, k))
    params = tuple(torch.nn.Parameter(t.to(dev), requires_grad=False) for t in (gq, gk))
    blocks = torch.arange(NB, dtype=torch.int32, device=dev).expand(B, H, Q, NB)
    pages = td[:, None, None, :].expand(B, H, Q, NB)

    def layer():
        cd = to_dev(c, dev, "nhd")
        qo, ko = torch.empty(B, Q, Hq, D, dtype=BF16, device=dev), torch.empty(B, Q, H, D, dtype=BF16, device=dev)
        out, lse = torch.empty_like(qo), torch.empty(B, Q, Hq, device=dev)
        k2, v2 = (torch.zeros(B, 48, H, D, dtype=BF16, device=dev) for _ in range(2))
        qk_rmsnorm_rope(qd, kd, *params, cs, pd, qo, ko, 1e-6)
        paged_kv_quant_write(ko, kd, *cd, td, pd)
        dsa_paged_attention(qo, *cd, blocks, pages, pd, ld, out, lse, 0.1)
        paged_kv_dequant_read(*cd, td, ld, k2, v2)
        torch.cuda.synchronize(dev)
        return [t.cpu() for t in (qo, ko, *cd, out, lse, k2, v2)]

    class Counting:
        def __init__(self):
            self.ok = []

        def __getattr__(self, name):
            def call(*a):
                self.ok.append(getattr(fast, name)(*a))
                return self.ok[-1]
            return call

    counting = Counting()
    try:
        _kv_lib._fast = counting
        a = layer()
        _kv_lib._fast = None
        b = layer()
    finally:
        _kv_lib._fast = fast
    assert counting.ok == [0, 0, 0, 0]
    assert all(same_bytes(x, y) for x, y in zip(a, b))


def test_the_c_launch_path_declines_what_it_does_not_take(dev):
    from flagos_kernelgen_72h_shanghai_2026_b200._build import build_fast_ext
    build_fast_ext()
    k = torch.zeros(1, 2, 2, 64, dtype=BF16, device=dev)
    c = to_dev(caches(gen(1), 3, 2, 16, 64, E4M3), dev)
    table, pos = torch.zeros(1, 2, dtype=torch.int32, device=dev), torch.zeros(1, 2, dtype=torch.int32, device=dev)
    fast = _kv_lib._fast
    assert fast.kv_copy(k, k, *c, table, pos, True) == 0
    for bad in ((k.float(), k, *c, table, pos), (k.cpu(), k, *c, table, pos), (k, k[:, :1], *c, table, pos),
                (k, k, *c, table.float(), pos), (k, k, *c, table, pos[0]), (k, k, c[0], c[1], c[2].view(INT8), c[3], table, pos)):
        assert fast.kv_copy(*bad, True) == -1
    torch.cuda.synchronize(dev)
