"""CPU: what the paged cache's C entry points and operations refuse before anything is launched."""

from __future__ import annotations

import ctypes

import pytest
import torch

from tests.conftest import REPO

F32, F16, BF16 = 0, 1, 2
P, I64, I32, F = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_float


class Cache(ctypes.Structure):
    _fields_ = [(n, P) for n in ("k", "v", "table", "length", "refs", "free")] + [
        (n, I64) for n in ("layers", "pages", "kv_heads", "page", "dh", "rows", "width")] + [
        ("dtype", I32)]


class Attention(ctypes.Structure):
    _fields_ = [("cache", P), ("layer", I64), ("q", P), ("q_stride", I64), ("tokens", I64),
                ("heads", I64), ("n", I64), ("prefix", P), ("rows", P), ("offsets", P),
                ("mask", P), ("mask_rows", I64), ("words", I64), ("scale", F), ("out", P)]


BUF = ctypes.create_string_buffer(256)
AT = (ctypes.addressof(BUF) + 15) // 16 * 16


@pytest.fixture(scope="module")
def lib():
    lib = ctypes.CDLL(str(REPO / "cugo_amd" / "libcugo_hip.so"))
    lib.cugo_paged_append.argtypes = [P, I64, P, I64, P, I64, P, P, I64, P]
    lib.cugo_paged_branch.argtypes = [P, P, P, P, I64, P, P, I64, P]
    lib.cugo_paged_accept.argtypes = [P, P, P, P, I64, I64, I64, P, P, I64, P]
    lib.cugo_tree_attention.argtypes = [P, P, I64, P]
    for name in ("branch", "accept"):
        f = getattr(lib, f"cugo_paged_{name}_workspace")
        f.argtypes, f.restype = [P, I64], I64
    lib.cugo_tree_attention_workspace.argtypes = [P]
    lib.cugo_tree_attention_workspace.restype = I64
    return lib


def _cache(**over):
    x = dict(k=AT, v=AT, table=AT, length=AT, refs=AT, free=AT, layers=2, pages=9, kv_heads=2,
             page=16, dh=32, rows=3, width=4, dtype=BF16)
    return Cache(**{**x, **over})


BAD_CACHES = [(dict(k=None), -1), (dict(v=None), -1), (dict(table=None), -1),
              (dict(length=None), -1), (dict(refs=None), -1), (dict(free=None), -1),
              (dict(layers=0), -1), (dict(pages=0), -1), (dict(kv_heads=-1), -1),
              (dict(rows=0), -1), (dict(width=0), -1), (dict(dtype=3), -2), (dict(dh=16), -3),
              (dict(dh=96), -3), (dict(page=8), -3), (dict(page=48), -3), (dict(page=512), -3),
              (dict(k=AT + 8), -4), (dict(v=AT + 2), -4), (dict(pages=1 << 31), -1),
              (dict(width=1 << 27), -1), (dict(rows=1 << 32), -1), (dict(layers=5000), -1),
              (dict(kv_heads=5000), -1), (dict(pages=1 << 29, kv_heads=4096, layers=4096,
                                               dh=256, dtype=F32, page=256), -1)]


@pytest.mark.parametrize("over,code", BAD_CACHES)
def test_caches(lib, over, code):
    c = ctypes.byref(_cache(**over))
    assert lib.cugo_paged_append(c, 0, AT, 64, AT, 64, AT, None, 1, None) == code
    assert lib.cugo_paged_branch(c, AT, AT, AT, 1, AT, AT, 1 << 30, None) == code
    assert lib.cugo_paged_accept(c, AT, AT, AT, 1, 1, 1, AT, AT, 1 << 30, None) == code
    a = Attention(cache=ctypes.addressof(c._obj), q=AT, q_stride=64, tokens=1, heads=2, n=1, scale=1.0,
                  prefix=AT, out=AT)
    assert lib.cugo_tree_attention(ctypes.byref(a), AT, 1 << 30, None) == code
    assert lib.cugo_paged_branch_workspace(c, 4) == lib.cugo_paged_accept_workspace(c, 4) == 0


def test_no_cache(lib):
    assert lib.cugo_paged_append(None, 0, AT, 64, AT, 64, AT, None, 0, None) == -1
    assert lib.cugo_paged_branch(None, AT, AT, AT, 0, AT, AT, 1 << 30, None) == -1
    assert lib.cugo_paged_accept(None, AT, AT, AT, 1, 1, 0, AT, AT, 1 << 30, None) == -1
    assert lib.cugo_tree_attention(None, AT, 0, None) == -1
    assert lib.cugo_tree_attention_workspace(None) == 0
    a = Attention(q=AT, q_stride=64, tokens=1, heads=2, n=1, prefix=AT, out=AT)
    assert lib.cugo_tree_attention(ctypes.byref(a), AT, 0, None) == -1


def test_append(lib):
    c = ctypes.byref(_cache())

    def go(layer=0, k=AT, ks=64, v=AT, vs=64, pos=AT, n=1):
        return lib.cugo_paged_append(c, layer, k, ks, v, vs, pos, None, n, None)

    assert go(n=0) == 0
    for over in (dict(n=-1), dict(layer=-1), dict(layer=2), dict(ks=63), dict(vs=0), dict(k=None),
                 dict(v=None), dict(pos=None), dict(n=1 << 40)):
        assert go(**over) == -1, over
    for over in (dict(k=AT + 4), dict(v=AT + 8), dict(ks=68), dict(vs=65)):
        assert go(**over) == -4, over


def test_branch(lib):
    c = ctypes.byref(_cache())
    need = lib.cugo_paged_branch_workspace(c, 5)

    def go(dst=AT, src=AT, length=AT, n=5, ok=AT, at=AT, size=need):
        return lib.cugo_paged_branch(c, dst, src, length, n, ok, at, size, None)

    assert need > 0 and go(n=0) == 0
    for over in (dict(n=-1), dict(n=(1 << 23) + 1), dict(dst=None), dict(src=None),
                 dict(length=None), dict(ok=None), dict(at=None)):
        assert go(**over) == -1, over
    assert go(at=AT + 8) == -4
    assert go(size=need - 1) == -5


def test_accept(lib):
    c = ctypes.byref(_cache())
    need = lib.cugo_paged_accept_workspace(c, 5)

    def go(rows=AT, start=AT, keep=AT, stride=3, most=3, n=5, ok=AT, at=AT, size=need):
        return lib.cugo_paged_accept(c, rows, start, keep, stride, most, n, ok, at, size, None)

    assert need > 0 and go(n=0) == 0
    for over in (dict(n=-1), dict(n=(1 << 23) + 1), dict(most=-1), dict(most=1 << 31),
                 dict(stride=-3), dict(rows=None), dict(start=None), dict(keep=None),
                 dict(ok=None), dict(at=None)):
        assert go(**over) == -1, over
    assert go(at=AT + 8) == -4
    assert go(size=need - 1) == -5


def test_tree_attention(lib):
    cache = _cache()

    def go(**over):
        x = dict(cache=ctypes.addressof(cache), layer=1, q=AT, q_stride=128, tokens=6, heads=4, n=2,
                 prefix=AT, mask_rows=6, words=1, scale=1.0, out=AT)
        a = Attention(**{**x, **over})
        return lib.cugo_tree_attention(ctypes.byref(a), AT, 1 << 30, None)

    assert go(tokens=0) == go(tokens=0, n=0) == 0
    assert go(scale=0.0) == go(scale=float("nan")) == go(scale=float("inf")) == -1
    for over in (dict(layer=2), dict(layer=-1), dict(tokens=-1), dict(n=-1), dict(n=0),
                 dict(heads=0), dict(heads=3), dict(heads=1 << 17), dict(q_stride=127),
                 dict(tokens=1 << 24, offsets=AT), dict(n=1 << 24, offsets=AT), dict(tokens=7),
                 dict(q=None), dict(prefix=None), dict(out=None), dict(words=-1),
                 dict(words=1 << 17), dict(mask=AT, mask_rows=5),
                 dict(mask=AT, mask_rows=3, offsets=AT)):
        assert go(**over) == -1, over
    for over in (dict(q=AT + 8), dict(out=AT + 2), dict(q_stride=132)):
        assert go(**over) == -4, over


def _cpu_cache():
    from cugo_amd.paged_cache import PagedKVCache

    return PagedKVCache(1, 3, 2, 32, 9, 4, "cpu")


def test_operations_refuse_cpu_tensors():
    from cugo_amd import _cugo_torch50_hip as m
    from cugo_amd import paged_cache as pc

    c, i = _cpu_cache(), torch.zeros(2, dtype=torch.int64)
    x = torch.zeros(2, 2, 32, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA"):
        pc.append(m, c, 0, x, x, i)
    with pytest.raises(RuntimeError, match="CUDA"):
        pc.branch(m, c, i, i, i)
    with pytest.raises(RuntimeError, match="CUDA"):
        pc.accept(m, c, i, i, i[:, None])
    with pytest.raises(RuntimeError, match="CUDA"):
        pc.tree_attention(m, c, 0, x, i)


@pytest.mark.parametrize("scale", [2.5e38, -3.4e38])
def test_scales_that_are_infinite_in_base_2(lib, scale):
    cache = _cache()
    a = Attention(cache=ctypes.addressof(cache), layer=1, q=AT, q_stride=128, tokens=6, heads=4, n=2,
                  prefix=AT, scale=scale, out=AT)
    assert lib.cugo_tree_attention(ctypes.byref(a), AT, 1 << 30, None) == -1
    assert lib.cugo_tree_attention_workspace(ctypes.byref(a)) == 0


def test_append_with_answers(lib):
    f = lib.cugo_paged_append_ok
    f.argtypes = [P, I64, P, I64, P, I64, P, P, I64, P, P]
    c = ctypes.byref(_cache())
    for ok in (AT, None):
        assert f(c, 0, AT, 64, AT, 64, AT, None, 0, ok, None) == 0
        assert f(c, 2, AT, 64, AT, 64, AT, None, 1, ok, None) == -1
        assert f(c, 0, AT, 64, AT, 64, AT, None, -1, ok, None) == -1
        assert f(c, 0, AT + 8, 64, AT, 64, AT, None, 1, ok, None) == -4
        assert f(ctypes.byref(_cache(dh=48)), 0, AT, 64, AT, 64, AT, None, 1, ok, None) == -3
