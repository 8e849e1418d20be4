"""The paged-KV-cache operators without a GPU: libdsa_kv.so loads, exports what
include/dsa_kv.h declares and answers bad arguments with status codes before
any device work; the wrappers refuse what is no CUDA tensor; the oracle agrees
with independent statements of the formulas."""
import ctypes
import re
from pathlib import Path

import numpy as np
import pytest
import torch

import flagos_kernelgen_72h_shanghai_2026_b200 as pkg
from flagos_kernelgen_72h_shanghai_2026_b200 import _kv_lib as L
from flagos_kernelgen_72h_shanghai_2026_b200._build import KV_LIB_PATH, build_kv_lib
from oracle import kv_oracle as R
from _kv_cases import angles, caches, gen, page_table

HEADER = Path(__file__).resolve().parent.parent / "include" / "dsa_kv.h"


@pytest.fixture(scope="module")
def lib():
    build_kv_lib()
    return L.load()


def test_library_exports_every_declared_symbol(lib):
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    names = re.findall(r"^\s*(?:int|const char\*)\s+(dsa_kv_\w+)\s*\(", text, flags=re.M)
    assert {"dsa_kv_rope_launch", "dsa_kv_write_launch", "dsa_kv_read_launch", "dsa_kv_attn_launch",
            "dsa_kv_strerror", "dsa_kv_abi_version"} <= set(names)
    raw = ctypes.CDLL(str(KV_LIB_PATH))
    for name in names:
        assert hasattr(raw, name), f"{name} declared in dsa_kv.h but not exported"


def test_struct_layout(lib):
    assert ctypes.sizeof(L.Dense) == 4 * 8
    assert ctypes.sizeof(L.Cache) == 2 * 4 + 4 * 8 + 4 * 8 + 12 * 8
    assert ctypes.sizeof(L.RopeArgs) == 6 * 4 + 7 * 8 + 4 * 32 + 4 * 8
    assert ctypes.sizeof(L.CopyArgs) == 4 * 4 + 3 * 8 + 2 * 32 + ctypes.sizeof(L.Cache) + 2 * 8
    assert ctypes.sizeof(L.AttnArgs) == 6 * 4 + 4 * 8 + 2 * 32 + ctypes.sizeof(L.Cache) + 2 * 8 + 6 * 8 + 3 * 8
    assert lib.dsa_kv_abi_version() == L.ABI_VERSION
    for code in range(0, 9):
        assert lib.dsa_kv_strerror(code)
    assert b"unknown" in lib.dsa_kv_strerror(99)


def _set(a, kw):
    for key, v in kw.items():
        obj, *rest = key.split("__")
        if rest:
            sub = getattr(a, obj)
            if isinstance(v, tuple):
                v = (ctypes.c_int64 * 3)(*v)
            setattr(sub, rest[0], v)
        else:
            setattr(a, obj, v)
    return a


def _rope(**kw):
    a = L.RopeArgs(struct_size=ctypes.sizeof(L.RopeArgs), dtype=L.DTYPE_BF16, gamma_dtype=L.DTYPE_FP32,
                   pos_dtype=L.DTYPE_INT32, eps=1e-6, B=2, Q=3, Hq=8, Hk=2, D=128, rot=128, max_pos=64)
    for i, n in enumerate(("q", "k", "q_out", "k_out")):  # never dereferenced: every case fails validation
        h = 8 if n[0] == "q" else 2
        setattr(a, n, L.Dense(0x10000 * (i + 1), 3 * h * 128, h * 128, 128))
    a.q_gamma, a.k_gamma, a.cos_sin, a.positions = 0x100000, 0x110000, 0x120000, 0x130000
    return _set(a, kw)


def _copy(**kw):
    a = L.CopyArgs(struct_size=ctypes.sizeof(L.CopyArgs), dtype=L.DTYPE_BF16, page_dtype=L.DTYPE_INT32,
                   pos_dtype=L.DTYPE_INT32, B=2, Q=3, NB=4)
    three = ctypes.c_int64 * 3
    a.k, a.v = L.Dense(0x10000, 3 * 256, 256, 128), L.Dense(0x20000, 3 * 256, 256, 128)
    s, ss = three(2 * 16 * 128, 16 * 128, 128), three(32, 16, 1)
    a.cache = L.Cache(L.DTYPE_E4M3, 0, 9, 2, 16, 128, 0x30000, 0x40000, 0x50000, 0x60000, s, s, ss, ss)
    a.page_table, a.pos = 0x70000, 0x80000
    return _set(a, kw)


def _attn(**kw):
    a = L.AttnArgs(struct_size=ctypes.sizeof(L.AttnArgs), dtype=L.DTYPE_FP16, block_dtype=L.DTYPE_INT32,
                   page_dtype=L.DTYPE_INT64, pos_dtype=L.DTYPE_INT32, softmax_scale=0.1, B=2, Q=3, G=4, K=5)
    three = ctypes.c_int64 * 3
    a.q, a.out = L.Dense(0x10000, 3 * 1024, 1024, 128), L.Dense(0x20000, 3 * 1024, 1024, 128)
    a.cache = _copy().cache
    a.blocks, a.pages, a.q_pos, a.kv_lens, a.lse = 0x70000, 0x80000, 0x90000, 0xa0000, 0xb0000
    a.blocks_stride = a.pages_stride = three(30, 15, 5)
    return _set(a, kw)


@pytest.mark.parametrize("kw,code", [
    (dict(struct_size=8), L.ERR_BAD_ARGS_SIZE),
    (dict(cache__reserved0=1), L.ERR_BAD_ARGS_SIZE),
    (dict(dtype=L.DTYPE_E4M3), L.ERR_BAD_DTYPE),
    (dict(block_dtype=L.DTYPE_FP32), L.ERR_BAD_DTYPE),
    (dict(pos_dtype=9), L.ERR_BAD_DTYPE),
    (dict(G=0), L.ERR_BAD_SHAPE),
    (dict(K=-1), L.ERR_BAD_SHAPE),
    (dict(cache__D=96), L.ERR_BAD_HEAD_DIM),
    (dict(cache__block_size=7), L.ERR_BAD_HEAD_DIM),
    (dict(cache__block_size=65537), L.ERR_UNSUPPORTED),
    (dict(B=1 << 20, Q=1 << 10), L.ERR_UNSUPPORTED),
    (dict(K=1 << 31), L.ERR_UNSUPPORTED),
    (dict(K=1 << 29, cache__block_size=4096), L.ERR_UNSUPPORTED),
    (dict(blocks=0), L.ERR_NULL_POINTER),
    (dict(kv_lens=0), L.ERR_NULL_POINTER),
    (dict(q__ptr=0), L.ERR_NULL_POINTER),
    (dict(cache__k_scale=0), L.ERR_NULL_POINTER),
    (dict(q__ptr=0x10002), L.ERR_ALIGNMENT),
    (dict(out__stride_h=0), L.ERR_BAD_SHAPE),
    (dict(pages=0x80004), L.ERR_ALIGNMENT),
    (dict(lse=0xb0002), L.ERR_ALIGNMENT),
    (dict(cache__v_codes=0x40004), L.ERR_ALIGNMENT),
    (dict(cache__k_stride=(4096, 0, 128)), L.ERR_BAD_SHAPE),
    (dict(cache__v_stride=(1 << 40, 2048, 128)), L.ERR_UNSUPPORTED),
    (dict(cache__v_scale_stride=(1 << 31, 16, 1)), L.ERR_UNSUPPORTED),
    (dict(cache__k_scale_stride=(-16, 16, 1)), L.ERR_BAD_SHAPE),
])
def test_attention_validation_before_any_device_call(lib, kw, code):
    assert lib.dsa_kv_attn_launch(ctypes.byref(_attn(**kw)), None) == code


@pytest.mark.parametrize("kw,code", [
    (dict(struct_size=8), L.ERR_BAD_ARGS_SIZE),
    (dict(dtype=L.DTYPE_FP32), L.ERR_BAD_DTYPE),
    (dict(gamma_dtype=L.DTYPE_INT8), L.ERR_BAD_DTYPE),
    (dict(pos_dtype=L.DTYPE_FP32), L.ERR_BAD_DTYPE),
    (dict(B=-1), L.ERR_BAD_SHAPE),
    (dict(interleaved=2), L.ERR_BAD_SHAPE),
    (dict(D=260), L.ERR_BAD_HEAD_DIM),
    (dict(D=512), L.ERR_BAD_HEAD_DIM),
    (dict(D=124), L.ERR_BAD_HEAD_DIM),
    (dict(rot=136), L.ERR_BAD_HEAD_DIM),
    (dict(rot=24), L.ERR_BAD_HEAD_DIM),
    (dict(rot=12, interleaved=1), L.ERR_BAD_HEAD_DIM),
    (dict(B=1 << 20, Q=1 << 10, Hq=1 << 2), L.ERR_UNSUPPORTED),
    (dict(q_gamma=0), L.ERR_NULL_POINTER),
    (dict(positions=0), L.ERR_NULL_POINTER),
    (dict(cos_sin=0), L.ERR_NULL_POINTER),
    (dict(k_out__ptr=0), L.ERR_NULL_POINTER),
    (dict(q__ptr=0x10008), L.ERR_ALIGNMENT),
    (dict(q__stride_h=132), L.ERR_ALIGNMENT),
    (dict(q_out__stride_h=0), L.ERR_BAD_SHAPE),
    (dict(q__stride_q=-1024), L.ERR_BAD_SHAPE),
    (dict(k_gamma=0x110004), L.ERR_ALIGNMENT),
    (dict(pos_dtype=L.DTYPE_INT64, positions=0x130004), L.ERR_ALIGNMENT),
])
def test_rope_validation_before_any_device_call(lib, kw, code):
    assert lib.dsa_kv_rope_launch(ctypes.byref(_rope(**kw)), None) == code


@pytest.mark.parametrize("entry", ["dsa_kv_write_launch", "dsa_kv_read_launch"])
@pytest.mark.parametrize("kw,code", [
    (dict(struct_size=8), L.ERR_BAD_ARGS_SIZE),
    (dict(cache__reserved0=1), L.ERR_BAD_ARGS_SIZE),
    (dict(dtype=L.DTYPE_FP32), L.ERR_BAD_DTYPE),
    (dict(cache__code_dtype=L.DTYPE_BF16), L.ERR_BAD_DTYPE),
    (dict(page_dtype=L.DTYPE_FP32), L.ERR_BAD_DTYPE),
    (dict(Q=-1), L.ERR_BAD_SHAPE),
    (dict(cache__block_size=0), L.ERR_BAD_SHAPE),
    (dict(cache__D=8), L.ERR_BAD_HEAD_DIM),
    (dict(cache__D=120), L.ERR_BAD_HEAD_DIM),
    (dict(cache__D=272), L.ERR_BAD_HEAD_DIM),
    (dict(B=1 << 20, Q=1 << 12), L.ERR_UNSUPPORTED),
    (dict(NB=1 << 31), L.ERR_UNSUPPORTED),
    (dict(page_table=0), L.ERR_NULL_POINTER),
    (dict(cache__v_scale=0), L.ERR_NULL_POINTER),
    (dict(v__ptr=0), L.ERR_NULL_POINTER),
    (dict(cache__k_codes=0x30008), L.ERR_ALIGNMENT),
    (dict(cache__k_stride=(4096, 2048, 8)), L.ERR_ALIGNMENT),
    (dict(k__stride_h=4), L.ERR_ALIGNMENT),
    (dict(cache__v_scale_stride=(-1, 16, 1)), L.ERR_BAD_SHAPE),
    (dict(pos=0x80002), L.ERR_ALIGNMENT),
])
def test_copy_validation_before_any_device_call(lib, entry, kw, code):
    assert getattr(lib, entry)(ctypes.byref(_copy(**kw)), None) == code


def test_a_write_refuses_cells_on_one_another(lib):
    a = _copy(cache__k_stride=(4096, 0, 128))
    assert lib.dsa_kv_write_launch(ctypes.byref(a), None) == L.ERR_BAD_SHAPE


def test_null_arguments(lib):
    for name in L._LAUNCHES:
        assert getattr(lib, name)(None, None) == L.ERR_NULL_POINTER


def test_empty_calls_are_no_ops(lib):
    assert lib.dsa_kv_rope_launch(ctypes.byref(_rope(Q=0)), None) == L.OK
    assert lib.dsa_kv_rope_launch(ctypes.byref(_rope(Hq=0, Hk=0)), None) == L.OK
    for entry in (lib.dsa_kv_write_launch, lib.dsa_kv_read_launch):
        assert entry(ctypes.byref(_copy(B=0)), None) == L.OK
        assert entry(ctypes.byref(_copy(Q=0, k__ptr=0)), None) == L.OK
        assert entry(ctypes.byref(_copy(NB=0, page_table=0)), None) == L.OK
    assert lib.dsa_kv_write_launch(ctypes.byref(_copy(cache__P=0)), None) == L.OK
    assert lib.dsa_kv_attn_launch(ctypes.byref(_attn(B=0)), None) == L.OK
    assert lib.dsa_kv_attn_launch(ctypes.byref(_attn(Q=0, q__ptr=0)), None) == L.OK


def test_wrappers_refuse_cpu_tensors():
    q, k = torch.zeros(1, 2, 4, 64), torch.zeros(1, 2, 2, 64)
    pos = torch.zeros(1, 2, dtype=torch.int32)
    with pytest.raises(TypeError, match="CUDA"):
        pkg.qk_rmsnorm_rope(q, k, q[0, 0, 0], q[0, 0, 0], angles(4, 64), pos, q, k, 1e-6)
    c = caches(gen(0), 3, 2, 16, 64, torch.int8)
    table = torch.zeros(1, 2, dtype=torch.int32)
    with pytest.raises(TypeError, match="CUDA"):
        pkg.paged_kv_quant_write(k, k, *c, table, pos)
    with pytest.raises(TypeError, match="CUDA"):
        pkg.paged_kv_dequant_read(*c, table, pos[0, :1], k, k)
    sel = torch.zeros(1, 2, 2, 1, dtype=torch.int32)
    with pytest.raises(TypeError, match="CUDA"):
        pkg.dsa_paged_attention(q.half(), *c, sel, sel, pos, pos[0, :1], q.half(), None, 0.1)
    with pytest.raises(TypeError, match="torch.Tensor"):
        pkg.paged_kv_quant_write(None, k, *c, table, pos)


# ------------------------------------------------------------------- oracle
def test_oracle_rotation_keeps_lengths_and_differences():
    """The rotated norm has length sqrt(D) for gamma = 1, and the product of a rotated query and key depends on the
    difference of their positions alone."""
    g = gen(1)
    q, k = torch.randn(1, 1, 1, 64, generator=g), torch.randn(1, 1, 1, 64, generator=g)
    one, cs = torch.ones(64), angles(200, 64).double()
    for inter in (False, True):
        dots = []
        for a, b in ((7, 3), (104, 100), (4, 0)):
            (qo, _), _ = R.qk_rmsnorm_rope_ref(q, q, one, one, cs, torch.tensor([[a]]), q, q, 0.0, inter)
            (ko, _), _ = R.qk_rmsnorm_rope_ref(k, k, one, one, cs, torch.tensor([[b]]), k, k, 0.0, inter)
            assert abs(float(qo.norm()) - 8.0) < 1e-6
            dots.append(float((qo * ko).sum()))
        assert max(dots) - min(dots) < 1e-4


def test_oracle_quantise_against_the_casts():
    g = gen(2)
    x = torch.randn(50, 64, generator=g)
    x[3] = 0
    x[4, 5], x[5, 6] = float("nan"), float("inf")
    for dt in (torch.int8, torch.float8_e4m3fn):
        codes, scale = R.quantise(x, dt)
        s = (x.abs().amax(-1) / np.float32(R.QMAX[dt])).clamp(min=1e-12)
        y = x * (1.0 / s)[:, None]
        y[4:6] = 0
        want = y.to(dt) if dt == torch.float8_e4m3fn else torch.round(y).to(dt)
        assert torch.equal(codes.view(torch.uint8), want.view(torch.uint8))
        assert torch.equal(scale[:4], s[:4]) and scale[4:6].isnan().all() and torch.equal(scale[6:], s[6:])


def test_oracle_read_after_write_is_within_half_a_step():
    g = gen(3)
    for dt, step in ((torch.int8, 0.5 / 127), (torch.float8_e4m3fn, 2.0 ** -4)):
        c = caches(g, 6, 2, 16, 32, dt)
        table, _ = page_table(g, 1, 4)
        k, v = torch.randn(1, 40, 2, 32, generator=g), torch.randn(1, 40, 2, 32, generator=g)
        pos = torch.arange(40)[None]
        kc, ks, vc, vs = R.paged_kv_quant_write_ref(k, v, *c, table, pos)
        ko, vo = R.paged_kv_dequant_read_ref(kc.view(dt), ks, vc.view(dt), vs, table, torch.tensor([40]), k, v)
        for got, x in ((ko, k), (vo, v)):
            assert ((got - x).abs() <= step * x.abs().amax(-1, keepdim=True) * (1 + 1e-6)).all()


def test_oracle_attention_against_a_dense_softmax():
    """All blocks selected, one of them twice by mistake of nobody: the oracle against torch's softmax on the dense
    context, with the doubled block's tokens in it twice."""
    g = gen(4)
    B, Q, H, G, D, bs, NB = 2, 3, 2, 2, 16, 8, 4
    table, P = page_table(g, B, NB)
    c = caches(g, P, H, bs, D, torch.int8)
    q = torch.randn(B, Q, H * G, D, generator=g)
    lens = torch.tensor([29, 17])
    pos = lens[:, None] - Q + torch.arange(Q)
    order = torch.tensor([2, 0, 3, 1, 0])
    blocks = order.expand(B, H, Q, 5)
    pages = table.long()[:, order][:, None, None].expand(B, H, Q, 5)
    r = R.dsa_paged_attention_ref(q, *c, blocks, pages, pos, lens, 0.3)
    zero = torch.zeros(B, NB * bs, H, D)
    k, v = R.paged_kv_dequant_read_ref(*c, table, torch.full((B,), NB * bs), zero, zero)
    at = torch.arange(NB * bs)
    for b in range(B):
        for i in range(Q):
            for x in range(H * G):
                s = k[b, :, x // G] @ q[b, i, x].double() * 0.3 + torch.log((at < bs).double() + 1)
                s = s.masked_fill((at > pos[b, i]) | (at >= lens[b]), float("-inf"))
                want = torch.softmax(s, 0) @ v[b, :, x // G]
                assert torch.allclose(r["out"][b, i, x], want, atol=1e-12)
                assert abs(float(r["lse"][b, i, x] - torch.logsumexp(s, 0))) < 1e-12


def test_index_division_by_multiplication():
    """The kernels' division of n < 2^31 by a constant, restated, against Python's."""
    rng = np.random.default_rng(0)
    for d in [1, 2, 3, 5, 7, 10, 16, 48, 96, 255, 1000, 4097, (1 << 20) + 1, (1 << 30) - 1, (1 << 31) - 1]:
        shift = next(i for i in range(33) if (1 << i) >= d)
        mul = ((1 << 32) * ((1 << shift) - d)) // d + 1
        for n in {0, 1, d - 1, d, d + 1, (1 << 31) - 1, *rng.integers(0, 1 << 31, 200).tolist()}:
            if 0 <= n < 1 << 31:
                assert mul < 1 << 32 and (((n * mul) >> 32) + n) >> shift == n // d
