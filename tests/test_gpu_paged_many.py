"""GPU: the paged cache's calls with many entries and long paths, bit for bit against the oracle: entries that
name a row twice among hundreds and thousands, kept tokens past 64 and past 256."""

from __future__ import annotations

import numpy as np
import pytest

from cugo_amd import paged_cache as pc
from oracle.paged_ref import of_cache, random_cache
from tests.conftest import announce
from tests.test_gpu_paged_cache import TYPES, i64, on_gpu, same

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [200, 257, 1025, 2049, 3000])
@pytest.mark.parametrize("spare", [50, 4000])
def test_branch_named_twice(ext, n, spare):
    """Rows that are another entry's dst or src, out of range, and too few pages, in calls of every size."""
    announce(f"paged branch of {n} entries, some named twice, {spare} pages")
    rng = np.random.default_rng(n + spare)
    rows = 2 * n
    lengths = [int(x) for x in rng.integers(0, 34, rows // 2)] + [0] * (rows - rows // 2)
    cache = on_gpu(random_cache(rng, lengths, kv_heads=1, width=3, spare=spare))
    ref = of_cache(cache)
    for turn in range(2):
        dst = rng.permutation(rows + 4)[:n] - 2
        twice = rng.integers(0, n, n // 20 + 2)
        dst[twice] = dst[rng.integers(0, n, len(twice))]
        src = np.where(rng.random(n) < 0.3, dst, rng.integers(-1, rows + 1, n))
        want = rng.integers(-1, 50, n)
        ok = pc.branch(ext, cache, i64(dst), i64(src), i64(want))
        assert ok.tolist() == ref.branch(dst, src, want)
        assert 0 < sum(ok.tolist()) < n
        same(cache, ref)


@pytest.mark.parametrize("n", [1, 40, 257, 1025, 3000])
@pytest.mark.parametrize("dtype,dh,layers", [("bf16", 32, 2), ("f32", 64, 1)])
def test_accept_of_many(ext, n, dtype, dh, layers):
    """Entries that name a row twice, paths that do not rise or go past the end, and shared pages."""
    announce(f"paged accept of {n} entries {dtype} dh {dh}")
    rng = np.random.default_rng(n + dh)
    rows = n + 30
    lengths = [int(x) for x in rng.integers(0, 60, rows)]
    cache = on_gpu(random_cache(rng, lengths, kv_heads=1, width=4, dh=dh, layers=layers, spare=40, dtype=TYPES[dtype]))
    if n > 1:  # the last rows share pages with the first
        k = min(10, n // 2)
        cut = rows - 1 - np.arange(k)
        assert pc.branch(ext, cache, i64(cut), i64(range(k)), i64(np.array(lengths)[:k])).all()
    ref = of_cache(cache)
    chosen = rng.permutation(rows + 2)[:n] - 1
    if n > 1:
        chosen[rng.integers(0, n, n // 30 + 1)] = chosen[0]
    have = np.array([ref.tokens(r) if 0 <= r < rows else 5 for r in chosen])
    start = np.array([rng.integers(0, h + 1) for h in have])
    most = 9
    keep = np.stack([np.sort(rng.permutation(20)[:most]) for _ in range(n)])
    keep[np.arange(most)[None] >= rng.integers(0, most + 1, n)[:, None]] = -1
    keep = np.where((start[:, None] + keep >= have[:, None]) & (rng.random((n, 1)) < 0.8), -1, keep)
    ok = pc.accept(ext, cache, i64(chosen), i64(start), i64(keep).view(n, most))
    assert ok.tolist() == ref.accept(chosen, start, keep)
    same(cache, ref)


@pytest.mark.parametrize("most", [64, 65, 128, 256, 257, 600])
@pytest.mark.parametrize("dtype,dh,page,kv_heads", [("bf16", 32, 16, 3), ("f32", 256, 64, 1), ("f16", 128, 256, 2)])
def test_long_paths(ext, most, dtype, dh, page, kv_heads):
    """As many kept tokens as there are columns, or fewer; some stay where they are; a path that fails
    only behind its first 64 or 256."""
    announce(f"paged accept of {most} tokens {dtype} dh {dh} page {page}")
    rng = np.random.default_rng(most + dh)
    total = 2 * most + 30
    width = -(-total // page)
    cache = on_gpu(random_cache(rng, [total] * 7, kv_heads=kv_heads, page=page, dh=dh, layers=2, width=width,
                                dtype=TYPES[dtype]))
    ref = of_cache(cache)
    start = rng.integers(0, 30, 7)
    keep = np.stack([np.sort(rng.permutation(total - 30)[:most]) for _ in range(7)])
    keep[1] = np.arange(most)  # all stay
    keep[2, :most // 2] = np.arange(most // 2)  # half do
    keep[2, most // 2:] = np.sort(rng.permutation(most)[:most - most // 2]) + most // 2
    keep[3, most - 1:] = -1
    keep[4, most // 3:] = -1
    keep[5, most - 1] = keep[5, most - 2]  # does not rise at its end
    keep[6, most - 1] = total  # past the end
    ok = pc.accept(ext, cache, i64(range(7)), i64(start), i64(keep).view(7, most))
    assert ok.tolist() == ref.accept(range(7), start, keep) == [True] * 5 + [False] * 2
    same(cache, ref)
