"""GPU: attention of drafted tokens for many sequences at once, against the definition in float64: waves of
games of which each wavefront takes an item (2,048 items or more), the search for a tile's sequence among
thousands, work shared out over up to 1,024 sequences; and how near the weights of few rows come."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from cugo_amd import paged_cache as pc
from oracle.paged_ref import dense_attention, random_cache
from tests.conftest import announce
from tests.test_gpu_paged_cache import TYPES, i64, on_gpu
from tests.test_gpu_tree_attention import queries, words_of

pytestmark = pytest.mark.gpu


def wave(rng, n, most, odd):
    """Ragged sequences, some of them empty: their counts, and offsets that begin past the first tokens."""
    counts = rng.integers(0, most + 1, n)
    counts[rng.random(n) < 0.2] = 0
    counts[-1] = most
    return counts, np.concatenate([[odd], odd + counts.cumsum()])


def check(got, cache, q, prefix, rows, offsets, mask, lost, before, twice=False):
    """Tokens of sequences are the definition's (NaN where the row is none), the others are as before."""
    safe = np.where(lost, 0, rows)
    want, bound = dense_attention(cache, 0, q, i64(prefix), mask, i64(safe), offsets, twice=twice)
    far = (got.double() - want).abs()
    token = np.full(q.shape[0], -1)
    for i in range(len(rows)):
        token[offsets[i]:offsets[i + 1]] = i
    missing = torch.from_numpy((token >= 0) & lost[token]).cuda()
    outside = torch.from_numpy(token < 0).cuda()
    assert got[missing].isnan().all()
    assert torch.equal(got[outside], before[outside])
    there = ~(missing | outside)
    bad = ~(far[there] <= bound[there])
    assert not bad.any(), (int(bad.sum()), float((far[there] / bound[there]).max()))


# sequences, drafts each, key heads, group, dh, table's width in pages of 16
WAVES = [(300, 16, 8, 1, 32, 8), (300, 5, 8, 4, 32, 8), (1100, 2, 4, 1, 64, 8), (300, 9, 8, 2, 64, 8),
         (300, 16, 8, 1, 128, 8), (300, 7, 8, 5, 128, 8), (300, 6, 8, 1, 256, 8),
         # fewer items: a workgroup each, or shared out
         (65, 9, 2, 1, 64, 8), (65, 9, 2, 1, 64, 300), (257, 6, 1, 2, 32, 300), (300, 9, 2, 2, 128, 300),
         (300, 3, 1, 1, 256, 300), (1024, 3, 1, 1, 64, 300), (1025, 3, 1, 1, 64, 300), (130, 40, 1, 2, 64, 300),
         (200, 70, 1, 2, 128, 300), (70, 70, 4, 1, 64, 8)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,most,kv_heads,group,dh,width", WAVES)
def test_waves(ext, dtype, n, most, kv_heads, group, dh, width):
    announce(f"tree attention of {n} sequences {dtype} {kv_heads} x {group} dh {dh} width {width}")
    rng = np.random.default_rng(n + most + dh)
    lengths = [int(x) for x in rng.integers(0, 100, 70)]
    lengths[:4] = [0, 1, 127, 128]
    if width > 8:
        lengths[4] = 1500
    cache = on_gpu(random_cache(rng, lengths, kv_heads=kv_heads, dh=dh, width=width, dtype=TYPES[dtype]))
    for masked in (True, False):
        odd = int(rng.integers(0, 9))
        counts, offsets = wave(rng, n, most, odd)
        rows = rng.integers(0, 70, n)
        lost = rng.random(n) < 0.03
        rows[lost] = rng.choice([-1, 70, 1 << 40], lost.sum())
        have = np.array(lengths)[np.where(lost, 0, rows)]
        prefix = np.where(rng.random(n) < 0.2, rng.integers(-5, 140, n), np.maximum(have - counts, 0))
        q = queries(rng, int(offsets[-1]) + 3, kv_heads * group, dh, TYPES[dtype])
        mask = words_of(rng, q.shape[0], 1 + int(rng.integers(0, 2))) if masked else None
        before = torch.full_like(q, 7.0)
        got = pc.tree_attention(ext, cache, 0, q, i64(prefix), mask=mask, rows=i64(rows), offsets=i64(offsets),
                                out=before.clone())
        check(got, cache, q, prefix, rows, offsets, mask, lost, before)


@pytest.mark.parametrize("masked", [True, False])
def test_more_sequences_than_two_turns_search(ext, masked):
    """4,100 sequences: 64 x 64 are not enough."""
    announce("tree attention of 4,100 sequences")
    rng = np.random.default_rng(4100)
    lengths = [int(x) for x in rng.integers(0, 40, 30)]
    cache = on_gpu(random_cache(rng, lengths, kv_heads=1, dh=32, width=4))
    n = 4100
    counts, offsets = wave(rng, n, 4, 1)
    rows, lost = rng.integers(0, 30, n), np.zeros(n, dtype=bool)
    prefix = np.maximum(np.array(lengths)[rows] - counts, 0)
    q = queries(rng, int(offsets[-1]), 1, 32, torch.bfloat16)
    mask = words_of(rng, q.shape[0], 1) if masked else None
    before = torch.full_like(q, 7.0)
    got = pc.tree_attention(ext, cache, 0, q, i64(prefix), mask=mask, rows=i64(rows), offsets=i64(offsets),
                            out=before.clone())
    check(got, cache, q, prefix, rows, offsets, mask, lost, before)


@pytest.mark.parametrize("each", [3, 16, 20])
def test_waves_of_one_size_and_tree(ext, each):
    """Without offsets, one tree for all: 512 games x 8 heads."""
    announce(f"tree attention of 512 sequences of {each}")
    rng = np.random.default_rng(each)
    lengths = [int(x) for x in rng.integers(each, 90, 40)]
    cache = on_gpu(random_cache(rng, lengths, kv_heads=8, dh=32, width=8))
    rows, lost = rng.integers(0, 40, 512), np.zeros(512, dtype=bool)
    prefix = np.array(lengths)[rows] - each
    q = queries(rng, 512 * each, 8, 32, torch.bfloat16)
    tree = pc.tree_mask([int(rng.integers(-1, j)) if j else -1 for j in range(each)], "cuda")
    got = pc.tree_attention(ext, cache, 0, q, i64(prefix), mask=tree, rows=i64(rows))
    check(got, cache, q, prefix, rows, np.arange(513) * each, tree.repeat(512, 1), lost, got)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("n,most,kv_heads,group,dh,width,length",
                         [(300, 16, 8, 1, 32, 8, 100), (300, 6, 8, 2, 64, 8, 60), (300, 8, 8, 1, 128, 8, 9),
                          (300, 4, 8, 1, 256, 8, 30), (20, 10, 2, 1, 64, 8, 40), (5, 10, 2, 1, 128, 1300, 20_000),
                          (3, 5, 1, 2, 32, 1300, 20_000)])
def test_weights_of_few_rows_are_two_numbers(ext, dtype, n, most, kv_heads, group, dh, width, length):
    """What little rounding is left there: half a step twice, not once."""
    announce(f"tree attention's weights {dtype} {n} sequences dh {dh} length {length}")
    rng = np.random.default_rng(n + dh + length)
    lengths = [int(x) for x in rng.integers(length // 2, length + 1, min(n, 40))]
    cache = on_gpu(random_cache(rng, lengths, kv_heads=kv_heads, dh=dh, width=width, dtype=TYPES[dtype]))
    counts, offsets = wave(rng, n, most, 0)
    rows, lost = rng.integers(0, len(lengths), n), np.zeros(n, dtype=bool)
    prefix = np.maximum(np.array(lengths)[rows] - counts, 0)
    q = queries(rng, int(offsets[-1]), kv_heads * group, dh, TYPES[dtype])
    got = pc.tree_attention(ext, cache, 0, q, i64(prefix), rows=i64(rows), offsets=i64(offsets))
    check(got, cache, q, prefix, rows, offsets, None, lost, got, twice=True)
