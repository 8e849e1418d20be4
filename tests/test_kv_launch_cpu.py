"""The launch paths of libdsa_kv.so without a GPU: the attention's entry with a
status, and which C++ launch path is taken."""
import ctypes
import os
from types import SimpleNamespace

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


def test_an_extension_without_the_entry_points_is_not_taken():
    """One built before they were added has the other operators' alone; one of another version is no better."""
    old = SimpleNamespace(task01=print, task02=print)
    kv = dict(kv_rope=print, kv_copy=print, kv_attn=print)
    assert L.launch_path(None) is None and L.launch_path(old) is None
    assert L.launch_path(SimpleNamespace(**kv)) is None
    assert L.launch_path(SimpleNamespace(kv_abi_version=L.ABI_VERSION - 1, **kv)) is None
    assert L.launch_path(SimpleNamespace(kv_abi_version=L.ABI_VERSION, kv_rope=print, kv_copy=print)) is None
    now = SimpleNamespace(kv_abi_version=L.ABI_VERSION, **kv)
    assert L.launch_path(now) is now


def test_the_built_extension_is_taken():
    from flagos_kernelgen_72h_shanghai_2026_b200._build import build_fast_ext
    build_fast_ext()
    from flagos_kernelgen_72h_shanghai_2026_b200 import _farq_fast
    assert L.launch_path(_farq_fast) is _farq_fast and L._fast is _farq_fast


def test_the_extension_builds_where_a_library_is_not_there_yet(monkeypatch, tmp_path):
    """A tree built before libdsa_kv.so was added: the library is built, then linked."""
    from flagos_kernelgen_72h_shanghai_2026_b200 import _build as B
    lib, out, done = tmp_path / "libdsa_kv.so", tmp_path / "_farq_fast.so", []
    out.write_bytes(b"before")
    os.utime(out, (0, 0))

    def build(verbose=False):
        done.append("library")
        lib.write_bytes(b"")

    def run(cmd, verbose):
        done.append("link")
        (tmp_path / "_farq_fast.so.tmp").write_bytes(b"after")
        return ""

    for name, v in (("KV_LIB_PATH", lib), ("build_kv_lib", build), ("_run", run), ("fast_ext_path", lambda: out)):
        monkeypatch.setattr(B, name, v)
    assert B.build_fast_ext() == out
    assert done == ["library", "link"] and out.read_bytes() == b"after"
