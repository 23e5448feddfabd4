"""CPU: the paged cache's oracle against closed forms and against itself written densely, the tree's
masks, and the index arithmetic that the kernels share, built for the host."""

from __future__ import annotations

import os
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch

from cugo_amd.paged_cache import PagedKVCache, tree_mask
from oracle.paged_ref import dense_attention, of_cache, random_cache
from tests.conftest import REPO

HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")


def invariants(ref, pages_of_rows=None):
    """References are the rows that hold a page."""
    held = [0] * len(ref.refs)
    for r in range(ref.rows):
        for j in range(ref.held(ref.tokens(r))):
            held[ref.page_at(r, j)] += 1
    assert held == ref.refs


@pytest.mark.parametrize("seed", range(4))
def test_branch_keeps_tokens_and_counts(seed):
    """Random branches, cuts and growths: every row's tokens are what plain lists say, and the
    references add up."""
    rng = np.random.default_rng(seed)
    cache = random_cache(rng, [int(x) for x in rng.integers(0, 70, 9)], width=8, spare=40)
    ref = of_cache(cache)
    said = [_tokens(ref, r) for r in range(9)]
    for _ in range(30):
        n = int(rng.integers(1, 6))
        dst, src = rng.integers(-1, 10, n), rng.integers(-1, 10, n)
        want = rng.integers(-1, 130, n)
        before = [list(x) for x in said]
        ok = ref.branch(dst, src, want)
        invariants(ref)
        for d, s, w, done in zip(dst, src, want, ok):
            if done:
                said[d] = before[s][:w] + [None] * (w - len(before[s]))
            elif 0 <= d < 9 and list(dst).count(d) == 1 and d not in src and ref.length[d] == 0:
                said[d] = []
        for r in range(9):
            now = _tokens(ref, r)
            assert len(now) == len(said[r])
            assert all(b is None or np.array_equal(a, b) for a, b in zip(now, said[r]))


def _tokens(ref, r):
    return [ref.k[:, ref.page_at(r, t // ref.page), :, t % ref.page].copy()
            for t in range(ref.tokens(r))]


def test_accept_moves_a_path():
    rng = np.random.default_rng(5)
    ref = of_cache(random_cache(rng, [40, 20, 33], spare=0))
    old = [_tokens(ref, r) for r in range(3)]
    ok = ref.accept([2, 0], [30, 10], [[0, 2, -1, 1], [3, 9, 20, 29]])
    assert ok == [True, True] and ref.length == [14, 20, 32]
    want = {0: old[0][:10] + [old[0][t] for t in (13, 19, 30, 39)], 1: old[1],
            2: old[2][:30] + [old[2][30], old[2][32]]}
    for r in range(3):
        assert all(np.array_equal(a, b) for a, b in zip(_tokens(ref, r), want[r]))
    invariants(ref)
    assert ref.accept([0, 0, 3, -1, 1], [0, 0, 0, 0, 21], [[0]] * 5) == [False] * 5
    assert ref.accept([0], [10], [[1, 1]]) == [False] and ref.accept([0], [10], [[1, 4]]) == [False]
    assert ref.accept([0], [14], [[-1]]) == [True]


def test_accept_refuses_shared_pages():
    rng = np.random.default_rng(6)
    ref = of_cache(random_cache(rng, [40, 0], width=3, spare=3))
    assert ref.branch([1], [0], [40]) == [True]  # every page shared
    assert ref.accept([1], [20], [[1, 3]]) == [False]
    assert ref.accept([1], [20], [[0, 1]]) == [True] and ref.length == [40, 22]
    assert ref.branch([1], [1], [30]) == [True] and ref.accept([1], [22], [[1, 3]]) == [True]


def test_attention_one_key_and_equal_keys():
    rng = np.random.default_rng(7)
    cache = random_cache(rng, [5, 1], dtype=torch.float32, fill=0.0)
    ref = of_cache(cache)
    q = rng.standard_normal((2, 4, 32))
    out = ref.attention(0, q, [0, 0], rows=[1, 0])
    for t, r in ((0, 1), (1, 0)):
        for h in range(4):
            assert np.allclose(out[t, h], ref.v[0, ref.page_at(r, 0), h // 2, 0], atol=0, rtol=1e-15)
    mean = ref.attention(0, np.zeros((1, 4, 32)), [3], mask=[[2]], rows=[0])  # positions 0, 1, 2, 4
    v = ref.v[0, ref.page_at(0, 0)]
    assert np.allclose(mean[0, 1], v[0, [0, 1, 2, 4]].mean(0), atol=1e-15)
    assert not ref.attention(0, q, [0, 0], mask=[[0], [0]]).any()
    assert np.isnan(ref.attention(0, q, [0, 0], rows=[2, -1])).all()


@pytest.mark.parametrize("seed", range(6))
def test_dense_form_is_the_same(seed):
    rng = np.random.default_rng(seed)
    lengths = [int(x) for x in rng.integers(0, 90, 5)]
    cache = random_cache(rng, lengths, kv_heads=3, page=int(rng.choice([16, 32])),
                         dtype=torch.float32, fill=0.0)
    counts = rng.integers(0, 7, 4)
    offsets = np.concatenate([[1], 1 + counts.cumsum()])
    tokens = int(offsets[-1]) + 2
    q = torch.from_numpy(rng.standard_normal((tokens, 6, 32)))
    prefix, rows = torch.from_numpy(rng.integers(-3, 95, 4)), torch.from_numpy(rng.integers(0, 5, 4))
    mask = torch.from_numpy(rng.integers(-2**63, 2**63, (tokens, 2))) if seed % 2 else None
    got, _ = dense_attention(cache, 0, q.float(), prefix, mask, rows, torch.from_numpy(offsets))
    words = None if mask is None else mask.numpy().view(np.uint64)
    want = of_cache(cache).attention(0, q.float().numpy(), prefix.numpy(), words, rows.numpy(), offsets)
    assert np.allclose(got.numpy(), want, atol=1e-12)


def test_tree_masks():
    assert tree_mask([-1, 0, 0, 1, 3]).tolist() == [[1], [3], [5], [11], [27]]
    chain = tree_mask(range(-1, 129))
    assert chain.shape == (130, 3) and chain[129].tolist() == [-1, -1, 3]
    assert tree_mask([-1] * 64)[63].tolist() == [-2**63]
    assert tree_mask([]).shape == (0, 1)
    with pytest.raises(ValueError, match="parent"):
        tree_mask([0])


def test_a_new_cache_is_empty():
    for pages in (1, 63, 64, 65, 200):
        cache = PagedKVCache(1, 3, 2, 32, pages, 4, "cpu")
        assert torch.equal(cache.free, torch.from_numpy(of_cache(cache).free_words()))


def test_index_arithmetic_stays_inside(tmp_path):
    """The kernels' lookups of pages and slots, built for the host: for corrupt lengths and table
    entries too, every address lies in the pool, and segments cover each byte of a page once."""
    if not (Path(HIPCC).exists() or shutil.which("hipcc")):
        pytest.skip("hipcc is not installed")
    exe = tmp_path / "paged_check"
    subprocess.run([HIPCC, "-O1", "-std=c++17", f"-I{REPO / 'cugo_amd' / 'csrc'}",
                    str(REPO / "tests" / "paged_host_check.cpp"), "-o", str(exe)], check=True,
                   capture_output=True, timeout=300)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and "inside" in out.stdout, out.stdout + out.stderr
