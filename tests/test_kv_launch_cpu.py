"""The launch paths of libdsa_kv.so without a GPU: the attention's entry with a
status, and which C++ launch path is taken."""
import ctypes

import pytest

from flagos_kernelgen_72h_shanghai_2026_b200 import _kv_lib as L
from flagos_kernelgen_72h_shanghai_2026_b200._build import build_kv_lib
from test_kv_cpu import _attn


@pytest.fixture(scope="module")
def lib():
    build_kv_lib()
    return L.load()


def test_the_entry_with_a_status_validates_like_the_other(lib):
    entry = lib.dsa_kv_attn_launch_status
    assert entry(None, None, 0, None) == L.ERR_NULL_POINTER
    assert entry(ctypes.byref(_attn(G=0)), None, 0, None) == L.ERR_BAD_SHAPE
    assert entry(ctypes.byref(_attn()), None, -1, None) == L.ERR_BAD_SHAPE
    assert entry(ctypes.byref(_attn()), None, 1, None) == L.ERR_BAD_SHAPE
    assert entry(ctypes.byref(_attn()), 0xb0002, 0, None) == L.ERR_ALIGNMENT
    assert entry(ctypes.byref(_attn(B=0)), 0xb0000, 2, None) == L.OK


def test_the_status_of_a_wait_has_a_name(lib):
    assert L.strerror(L.ERR_DEVICE_TIMEOUT) != L.strerror(99)
