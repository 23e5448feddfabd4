"""GPU: infinite values and NaN in the attention of drafted tokens, wherever they lie: among the tokens that
all queries attend or among the drafts, in one tile or another, however the call is dealt out.  What attends
an infinite value is that infinity, two of different signs or NaN give NaN, and what does not attend
them is as without them."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from cugo_amd import paged_cache as pc
from oracle.paged_ref import dense_attention, random_cache
from tests.conftest import announce
from tests.test_gpu_paged_cache import TYPES, i64, on_gpu

pytestmark = pytest.mark.gpu

# lengths of rows, sequences, drafts each, heads a key head, table's width in pages of 16: the ways that
# calls are dealt out (a wavefront an item needs 2,048 of them)
DEALT = {"wavefront": ([150, 260, 33, 90], 1024, 3, 2, 32), "group": ([150, 260, 33], 3, 10, 2, 32),
         "shared": ([700, 260, 33], 3, 10, 2, 300), "one row": ([5000], 1, 1, 1, 320),
         "through LDS": ([400, 260, 140], 3, 40, 2, 32), "through LDS, shared": ([1500, 260, 140], 3, 40, 2, 300)}


def drafts_tree(rng, t):
    return [int(rng.integers(-1, j)) if j else -1 for j in range(t)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dh", [32, 64, 128, 256])
@pytest.mark.parametrize("dealt", DEALT)
def test_infinite_values(ext, dtype, dh, dealt):
    announce(f"tree attention of infinite values {dtype} dh {dh}, {dealt}")
    lengths, n, t, group, width = DEALT[dealt]
    rng = np.random.default_rng(dh + n + t)
    kv_heads = 2
    cache = on_gpu(random_cache(rng, lengths, kv_heads=kv_heads, dh=dh, page=16, width=width, dtype=TYPES[dtype]))
    rows = np.arange(n) % len(lengths)
    have = np.array(lengths)[rows]
    # equal queries for sequences of equal rows, so that the definition is worked out once a row
    q = torch.from_numpy(rng.standard_normal((len(lengths), t, kv_heads * group, dh))).to("cuda", TYPES[dtype])
    prefix, which = i64(have - t), i64(rows)
    tree = pc.tree_mask(drafts_tree(rng, t), "cuda")
    clean_k, clean_v = cache.k.clone(), cache.v.clone()
    few = len(lengths)

    def pages(row, at):
        return cache.table[row, at // 16].long(), at % 16

    for turn, kinds in enumerate((["inf"], ["-inf"], ["inf", "-inf"], ["nan"], ["inf", "inf"])):
        for where in ("early", "late", "drafts"):
            cache.k.copy_(clean_k)
            cache.v.copy_(clean_v)
            marked = torch.zeros(few, 2, max(lengths), dtype=torch.bool, device="cuda")  # up, down
            for r in range(few):
                for i, kind in enumerate(kinds):
                    low, high = {"early": (0, min(20, lengths[r] - t)), "late": (max(0, lengths[r] - t - 40), lengths[r] - t),
                                 "drafts": (lengths[r] - t, lengths[r])}[where]
                    at = int(rng.integers(low, high))
                    page, slot = pages(r, at)
                    cache.v[0, page, :, slot, ::3] = float(kind)
                    if marked[r, :, at].any():  # the other one is gone
                        marked[r, :, at] = False
                    marked[r, 0, at] = kind != "-inf"
                    marked[r, 1, at] = kind != "inf"
                    if turn == 4:  # of a weight near 0 beside the others
                        cache.k[0, page, :, slot] = 0.0
            got = pc.tree_attention(ext, cache, 0, q[rows].flatten(0, 1), prefix, mask=tree, rows=which)
            # the same everywhere else, within the definition's bound, from finite values
            finite = torch.where(cache.v.isfinite(), cache.v, 0.0)
            bad_v, cache.v = cache.v, finite
            want, bound = dense_attention(cache, 0, q.flatten(0, 1), i64(np.array(lengths) - t), tree)
            cache.v = bad_v
            got = got.view(n, t, kv_heads * group, dh)
            for r in range(few):
                mine = got[torch.from_numpy(rows == r).cuda()]
                assert torch.equal(mine, mine[:1].expand_as(mine)) or mine.isnan().any()
                y, far = want.view(few, t, -1, dh)[r], bound.view(few, t, -1, dh)[r]
                sees = torch.ones(t, max(lengths), dtype=torch.bool, device="cuda")
                at = torch.arange(max(lengths), device="cuda")
                b = (at - (lengths[r] - t)).clamp(0, 64 * tree.shape[1] - 1)
                sees &= (at < lengths[r] - t) | ((tree[:, b // 64] >> (b % 64)) & 1 == 1)
                sees &= at < lengths[r]
                up, down = ((sees & marked[r, k]).any(1) for k in (0, 1))
                for seq in mine[:3]:
                    seq = seq.double()
                    odd = torch.where(up & down, torch.nan, torch.where(up, torch.inf, -torch.inf))[:, None, None]
                    touched = (up | down)[:, None, None].expand(t, kv_heads * group, -1)
                    third = seq[..., ::3]
                    as_said = (third == odd) | (third.isnan() & odd.isnan())
                    near = (third - y[..., ::3]).abs() <= far[..., ::3]
                    assert torch.where(touched, as_said, near).all(), (kinds, where, r)
                    for rest in (1, 2):
                        assert ((seq[..., rest::3] - y[..., rest::3]).abs() <= far[..., rest::3]).all(), (kinds, where, r)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dh", [32, 64, 128, 256])
@pytest.mark.parametrize("dealt", DEALT)
def test_scores_of_minus_infinity(ext, dtype, dh, dealt):
    """Keys that some queries cannot score: of weight 0 for those, and zeros where all are."""
    announce(f"tree attention of scores of -inf {dtype} dh {dh}, {dealt}")
    lengths, n, t, group, width = DEALT[dealt]
    rng = np.random.default_rng(dh + n)
    cache = on_gpu(random_cache(rng, lengths, kv_heads=2, dh=dh, width=width, dtype=TYPES[dtype]))
    cache.k[0, :, :, :, 0] = -torch.inf
    cache.k[0, :, :, 1::3, 0] = 0.0
    few = len(lengths)
    q = torch.from_numpy(rng.standard_normal((few, t, 2 * group, dh))).to("cuda", TYPES[dtype])
    q[..., 0] = 1.0
    rows = np.arange(n) % few
    prefix = i64(np.array(lengths)[rows] - t)
    tree = pc.tree_mask(drafts_tree(rng, t), "cuda")
    for turn in range(2):
        got = pc.tree_attention(ext, cache, 0, q[rows].flatten(0, 1), prefix, mask=tree, rows=i64(rows))
        want, bound = dense_attention(cache, 0, q.flatten(0, 1), i64(np.array(lengths) - t), tree)
        far = (got.view(n, t, 2 * group, dh).double() - want.view(few, t, 2 * group, dh)[rows]).abs()
        assert (far <= bound.view(few, t, 2 * group, dh)[rows]).all()
        if turn == 0:
            assert want.abs().amax() > 0
            cache.k[0, :, :, :, 0] = -torch.inf
    assert not got.any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dh", [32, 64, 128, 256])
@pytest.mark.parametrize("dealt", DEALT)
@pytest.mark.parametrize("gap", [5.0, 30.0, 100.0])
def test_small_weights_of_infinities(ext, dtype, dh, dealt, gap):
    """An infinite value whose weight is e^-gap of another token's: an infinity all the same, before and
    behind that token."""
    announce(f"tree attention of infinite values of small weights {dtype} dh {dh}, {dealt}, {gap}")
    lengths, n, t, group, width = DEALT[dealt]
    tokens = lengths[0]
    cache = pc.PagedKVCache(1, 1, 1, dh, -(-tokens // 16), width, "cuda", page=16, dtype=TYPES[dtype])
    held = -(-tokens // 16)
    cache.table[0, :held] = torch.arange(held, dtype=torch.int32)
    cache.length.fill_(tokens)
    q = torch.zeros(n * t, 4 * group, dh, dtype=TYPES[dtype], device="cuda")
    q[..., 0] = 4.0
    for high, odd in ((0, tokens - t - 1), (tokens - t - 1, 0), (3, 70), (70, 3), (tokens - t - 1, tokens - t - 2)):
        cache.k.zero_()
        cache.v.fill_(1.0)
        cache.k[0, high // 16, 0, high % 16, 0] = 1.0
        cache.v[0, odd // 16, 0, odd % 16, 1::2] = torch.inf
        out = pc.tree_attention(ext, cache, 0, q, i64([tokens - t] * n), rows=i64([0] * n), scale=gap / 4)
        assert (out[..., 1::2] == torch.inf).all(), (high, odd)
        assert ((out[..., ::2].float() - 1).abs() <= 2 * torch.finfo(TYPES[dtype]).eps).all(), (high, odd)
