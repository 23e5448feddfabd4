"""GPU: attention of drafted tokens over the paged cache against the definition in float64
(oracle/paged_ref.py), each value within the bound that float32 sums and the types' roundings allow
(dense_attention works it out)."""

from __future__ import annotations

from types import SimpleNamespace

import numpy as np
import pytest
import torch

from cugo_amd import paged_cache as pc
from oracle.paged_ref import dense_attention, of_cache, random_cache
from tests.conftest import announce
from tests.test_gpu_paged_cache import TYPES, i64, on_gpu

pytestmark = pytest.mark.gpu


def close(got, cache, q, prefix, layer=0, **how):
    want, bound = dense_attention(cache, layer, q, prefix, **how)
    far = (got.double() - want).abs()
    bad = ~(far <= bound)
    assert not bad.any(), (int(bad.sum()), float((far / bound.clamp_min(1e-300)).max()))


def queries(rng, tokens, heads, dh, dtype):
    return torch.from_numpy(rng.standard_normal((tokens, heads, dh))).to("cuda", dtype)


def words_of(rng, tokens, words):
    """Random masks: sparse, dense, empty and full ones."""
    m = rng.integers(-2**63, 2**63, (tokens, words)) & rng.integers(-2**63, 2**63, (tokens, words))
    kind = rng.integers(0, 5, tokens)
    m[kind == 0] = 0
    m[kind == 1] = -1
    return torch.from_numpy(m).cuda()


GRID = [(dt, dh, page, kv, group) for dt in TYPES for dh, page, kv, group in
        ((32, 16, 8, 1), (32, 32, 2, 3), (64, 16, 3, 2), (64, 64, 1, 8), (128, 16, 2, 4),
         (128, 128, 1, 1), (256, 32, 2, 1), (256, 16, 1, 5), (128, 256, 4, 2))]


@pytest.mark.parametrize("dtype,dh,page,kv_heads,group", GRID)
def test_ragged_trees_and_chains(ext, dtype, dh, page, kv_heads, group):
    """Sequences with 0 to 40 queries over rows of 0 to 330 tokens, prefixes from below 0 to past
    the end; what no query may see is NaN."""
    announce(f"tree attention {dtype} dh {dh} page {page} heads {kv_heads} x {group}")
    rng = np.random.default_rng(dh + page + group)
    lengths = [0, 1, 15, 16, 17, 31, 32, 33, 64, 100, 250, 330, 5, 47]
    cache = on_gpu(random_cache(rng, lengths, layers=2, kv_heads=kv_heads, page=page, dh=dh,
                                dtype=TYPES[dtype]))
    for turn in range(3):
        n = 14 if turn else 9
        rows = rng.permutation(14)[:n]
        counts = rng.integers(0, 41, n) if turn else rng.integers(0, 3, n)
        counts[0], counts[-1] = 40, 0
        offsets = np.concatenate([[0], counts.cumsum()])
        have = np.array(lengths)[rows]
        prefix = np.where(rng.random(n) < 0.2, rng.integers(-5, 340, n), np.maximum(have - counts, 0))
        q = queries(rng, int(offsets[-1]), kv_heads * group, dh, TYPES[dtype])
        for words in (None, 1, 2):
            mask = None if words is None else words_of(rng, q.shape[0], words)
            how = dict(mask=mask, rows=i64(rows), offsets=i64(offsets))
            got = pc.tree_attention(ext, cache, 1, q, i64(prefix), **how)
            close(got, cache, q, i64(prefix), layer=1, **how)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("each", [1, 2, 5, 16, 17, 64, 130])
def test_sequences_of_one_size(ext, dtype, each):
    """Without offsets: as many queries each, and one tree for all."""
    announce(f"tree attention {dtype}, {each} queries each")
    rng = np.random.default_rng(each)
    lengths = [int(x) for x in rng.integers(each, each + 200, 11)]
    cache = on_gpu(random_cache(rng, lengths, kv_heads=4, dh=64, dtype=TYPES[dtype]))
    q = queries(rng, 11 * each, 8, 64, TYPES[dtype])
    prefix = i64(np.array(lengths) - each)
    close(pc.tree_attention(ext, cache, 0, q, prefix), cache, q, prefix)
    tree = pc.tree_mask([int(rng.integers(-1, j)) if j else -1 for j in range(each)], "cuda")
    close(pc.tree_attention(ext, cache, 0, q, prefix, mask=tree), cache, q, prefix, mask=tree)
    close(pc.tree_attention(ext, cache, 0, q, prefix, scale=0.5), cache, q, prefix, scale=0.5)


@pytest.mark.parametrize("dtype,kv_heads,group,dh,queries_each",
                         [("bf16", 1, 1, 128, 1), ("f16", 2, 8, 64, 3), ("f32", 1, 4, 128, 2),
                          ("bf16", 2, 4, 128, 70), ("f16", 1, 1, 256, 33), ("bf16", 8, 1, 32, 16)])
@pytest.mark.parametrize("sequences", [1, 3])
def test_long_rows(ext, dtype, kv_heads, group, dh, queries_each, sequences):
    """Rows of up to 20,000 tokens, few enough that they are split."""
    announce(f"tree attention over long rows {dtype} {kv_heads} x {group} dh {dh} n {sequences}")
    rng = np.random.default_rng(dh + queries_each)
    lengths = [20_001, 517, 9_999][:sequences]
    cache = on_gpu(random_cache(rng, lengths, kv_heads=kv_heads, page=64, dh=dh, dtype=TYPES[dtype]))
    q = queries(rng, sequences * queries_each, kv_heads * group, dh, TYPES[dtype]) * 2
    prefix = i64(np.array(lengths) - queries_each)
    mask = words_of(rng, q.shape[0], 2)
    close(pc.tree_attention(ext, cache, 0, q, prefix), cache, q, prefix)
    close(pc.tree_attention(ext, cache, 0, q, prefix, mask=mask), cache, q, prefix, mask=mask)


@pytest.mark.parametrize("dtype", TYPES)
def test_many_queries(ext, dtype):
    """A chunk of 300 tokens over 1,000 earlier ones, each over all before it."""
    announce(f"tree attention of a chunk {dtype}")
    rng = np.random.default_rng(9)
    cache = on_gpu(random_cache(rng, [1300, 307], kv_heads=2, page=32, dh=128, dtype=TYPES[dtype]))
    offsets, prefix = i64([0, 300, 601]), i64([1000, 6])
    q = queries(rng, 601, 6, 128, TYPES[dtype])
    close(pc.tree_attention(ext, cache, 0, q, prefix, offsets=offsets), cache, q, prefix, offsets=offsets)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dh", [32, 64, 128, 256])
def test_infinities_in_branches_not_taken(ext, dtype, dh):
    """A drafted token whose value is infinite or NaN shows in those that attend it only; a key of that
    kind too."""
    announce(f"tree attention beside infinite drafts {dtype} dh {dh}")
    rng = np.random.default_rng(10)
    cache = on_gpu(random_cache(rng, [60, 45], kv_heads=2, dh=dh, page=16, dtype=TYPES[dtype]))
    parents = [-1, 0, 0, 1, 2, 3, -1, 6, 7, 2]
    mask = pc.tree_mask(parents, "cuda")
    q = queries(rng, 20, 4, dh, TYPES[dtype])
    prefix = i64([50, 35])
    clean = pc.tree_attention(ext, cache, 0, q, prefix, mask=mask)
    for which, draft, value in (("v", 2, "inf"), ("v", 6, "nan"), ("k", 3, "nan"), ("v", 4, "-inf"),
                                ("k", 9, "inf")):
        bad = SimpleNamespace(**vars(cache))
        for name in ("k", "v"):
            setattr(bad, name, getattr(cache, name).clone())
        for row, start in ((0, 50), (1, 35)):
            t = start + draft
            page = int(cache.table[row, t // 16])
            getattr(bad, which)[0, page, :, t % 16, ::3] = float(value)
        got = pc.tree_attention(ext, bad, 0, q, prefix, mask=mask)
        sees = ((mask[:, 0] >> draft) & 1).bool().repeat(2)
        assert torch.equal(got[~sees], clean[~sees])
        if which == "v":  # in those that see it, only the elements that are infinite or NaN there
            assert torch.equal(got[sees][..., 1::3], clean[sees][..., 1::3])
            marked = got[sees][..., ::3].float()
            assert (marked.isnan() if value == "nan" else marked == float(value)).all()
        elif value == "nan":
            assert got[sees].isnan().all()


def test_what_is_not_there(ext):
    """Rows that do not exist, pages that do not, and tokens outside every sequence."""
    announce("tree attention without rows or pages")
    rng = np.random.default_rng(11)
    cache = on_gpu(random_cache(rng, [40, 20, 70], kv_heads=2, dh=32, width=6))
    q = queries(rng, 12, 2, 32, torch.bfloat16)
    out = torch.full_like(q, 7.0)
    offsets = i64([1, 3, 5, 8, 10])
    got = pc.tree_attention(ext, cache, 0, q, i64([40, 10, -4, 30]), rows=i64([0, 3, 1, -1]),
                            offsets=offsets, out=out)
    assert got.data_ptr() == out.data_ptr()
    assert (out[[0, 10, 11]] == 7).all() and out[3:5].isnan().all() and out[8:10].isnan().all()
    assert not out[[1, 2, 5, 6, 7]].isnan().any()
    cache.table[0, 1] = 1 << 30
    cache.table[2, 4] = -1
    got = pc.tree_attention(ext, cache, 0, q[:6], i64([16, 17, 64]), rows=i64([0, 0, 2]),
                            mask=torch.zeros(6, 1, dtype=torch.int64, device="cuda"))
    assert not got[:2].isnan().any() and got[2:4].isnan().all() and not got[4:].isnan().any()
    got = pc.tree_attention(ext, cache, 0, q[:1], i64([70]), rows=i64([2]))
    assert got.isnan().all()
    # a row's length past its table is the table's
    cache.length[1] = 1 << 40
    cache.table[1] = cache.table[1, 0]
    close(pc.tree_attention(ext, cache, 0, q[:2], i64([90]), rows=i64([1])), cache, q[:2], i64([90]),
          rows=i64([1]))
    assert pc.tree_attention(ext, cache, 0, q[:0], i64([])).shape == (0, 2, 32)
    nothing = torch.zeros(4, 0, dtype=torch.int64, device="cuda")
    close(pc.tree_attention(ext, cache, 0, q[:4], i64([0, 7]), mask=nothing, rows=i64([1, 1])), cache,
          q[:4], i64([0, 7]), mask=nothing, rows=i64([1, 1]))


@pytest.mark.parametrize("queries_each,width", [(3, 4), (40, 300), (3, 300)])
def test_offsets_outside_the_tokens(ext, queries_each, width):
    """Sequences that begin before the tokens or end past them have no queries, and the others are
    served, however the rows are dealt out; offsets that fall, which no caller may give, leave every
    token's place as it was or with some sequence's result."""
    announce(f"tree attention with offsets outside, {queries_each} queries, width {width}")
    rng = np.random.default_rng(16)
    cache = on_gpu(random_cache(rng, [60, 50, 64, 7], kv_heads=2, dh=64, width=width))
    each = queries_each
    tokens = 4 * each
    q = queries(rng, tokens, 8, 64, torch.bfloat16)
    prefix, rows = i64([40, 50, 10, 7]), i64([0, 1, 2, 3])
    for offsets, there in (([-50, 0, each, 2 * each, 9 * each], {1: 0, 2: each}),
                           ([-9, -8, -7, 1 << 40, 1 << 41], {}),
                           ([each, 2 * each, 2 * each, 4 * each, 4 * each], {0: each, 2: 2 * each})):
        out = torch.full_like(q, 7.0)
        pc.tree_attention(ext, cache, 0, q, prefix, rows=rows, offsets=i64(offsets), out=out)
        for i, first in there.items():
            last = offsets[i + 1]
            part = slice(first, last)
            close(out[part], cache, q[part], prefix[i:i + 1], rows=rows[i:i + 1])
            out[part] = 7.0
        assert (out == 7).all()
    for offsets in ([2 * each, 3 * each, 4 * each, each, each], [0, tokens, 0, tokens, 0],
                    [0, each, 0, 2 * each, 9 * each], [-50, 0, tokens, 0, tokens]):
        out = pc.tree_attention(ext, cache, 0, q, prefix, rows=rows, offsets=i64(offsets),
                                out=torch.full_like(q, 7.0))
        assert out.shape == q.shape


def test_negative_scale(ext):
    announce("tree attention with a negative scale")
    rng = np.random.default_rng(17)
    for dtype in TYPES.values():
        cache = on_gpu(random_cache(rng, [60, 50], kv_heads=2, dh=32, dtype=dtype))
        q = queries(rng, 6, 4, 32, dtype)
        got = pc.tree_attention(ext, cache, 0, q, i64([57, 47]), scale=-0.3)
        assert torch.equal(got, pc.tree_attention(ext, cache, 0, -q, i64([57, 47]), scale=0.3))


def test_strided_queries(ext):
    announce("tree attention of a packed projection's columns")
    rng = np.random.default_rng(12)
    cache = on_gpu(random_cache(rng, [30, 40], kv_heads=8, dh=32))
    packed = queries(rng, 10, 24, 32, torch.bfloat16).view(10, 768)
    q = packed[:, :256].reshape(10, 8, 32)
    assert not q.is_contiguous()
    prefix = i64([25, 35])
    a = pc.tree_attention(ext, cache, 0, q, prefix)
    assert torch.equal(a, pc.tree_attention(ext, cache, 0, q.contiguous(), prefix))
    odd = queries(rng, 10, 8, 33, torch.bfloat16)[..., 1:]
    close(pc.tree_attention(ext, cache, 0, odd, prefix), cache, odd.contiguous(), prefix)
    close(pc.tree_attention(ext, cache, 0, q.flip(1).transpose(0, 1).contiguous().transpose(0, 1), prefix),
          cache, q.flip(1).contiguous(), prefix)


def test_offsets_past_32_bits(ext):
    """Keys beyond 4 GiB of a layer's start."""
    announce("tree attention past 4 GiB")
    pages = 70_000
    k, v = (torch.zeros(1, pages, 8, 128, 32, dtype=torch.bfloat16, device="cuda") for _ in "kv")
    cache = pc.PagedKVCache(1, 2, 8, 32, pages, 4, "cuda")
    cache.k, cache.v = k, v
    cache.table[:, :3] = torch.tensor([[69_999, 0, 68_000], [67_000, 69_998, 3]], device="cuda")
    cache.length[:] = i64([300, 380])
    for p in (69_999, 0, 68_000, 67_000, 69_998, 3):
        k[0, p].normal_()
        v[0, p].normal_()
    rng = np.random.default_rng(13)
    q = queries(rng, 6, 8, 32, torch.bfloat16)
    close(pc.tree_attention(ext, cache, 0, q, i64([297, 377])), cache, q, i64([297, 377]))


def test_same_result_every_time_and_in_a_graph(ext):
    """Split and unsplit calls: bit for bit the same again, on another stream, and replayed with
    other work between."""
    announce("tree attention captured and replayed")
    rng = np.random.default_rng(14)
    for lengths, each in (([5000, 3000], 20), ([60] * 64, 9)):
        cache = on_gpu(random_cache(rng, lengths, kv_heads=2, dh=128, page=32))
        n = len(lengths)
        q = queries(rng, n * each, 8, 128, torch.bfloat16)
        other = queries(rng, n * each, 8, 128, torch.bfloat16)
        prefix = i64(np.array(lengths) - each)
        first, second = (pc.tree_attention(ext, cache, 0, x, prefix) for x in (q, other))
        assert torch.equal(first, pc.tree_attention(ext, cache, 0, q, prefix))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            again = pc.tree_attention(ext, cache, 0, q, prefix)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(first, again)
        given, given2 = q.clone(), other.clone()
        graphs, outs = [], []
        for x in (given, given2):  # two graphs, replayed in turn
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1]):
                outs.append(pc.tree_attention(ext, cache, 0, x, prefix))
        for turn in range(4):
            given.copy_(q if turn % 2 else other)
            graphs[0].replay()
            graphs[1].replay()
            eager = pc.tree_attention(ext, cache, 0, q, prefix)
            torch.cuda.synchronize()
            assert torch.equal(outs[0], first if turn % 2 else second)
            assert torch.equal(outs[1], second) and torch.equal(eager, first)


def test_refusals(ext):
    announce("tree attention refused")
    cache = pc.PagedKVCache(2, 3, 2, 32, 9, 4, "cuda")
    q = torch.zeros(6, 4, 32, dtype=torch.bfloat16, device="cuda")
    p = i64([0, 0])
    ok = torch.zeros(6, 1, dtype=torch.int64, device="cuda")
    for args, how in (((2, q, p), {}), ((-1, q, p), {}), ((0, q.float(), p), {}), ((0, q[0], p), {}),
                      ((0, q[:, :3], p), {}), ((0, q[..., :16], p), {}), ((0, q[:5], p), {}),
                      ((0, q, p.int()), {}), ((0, q, p.cpu()), {}), ((0, q.cpu(), p), {}),
                      ((0, q, p), dict(mask=ok.int())), ((0, q, p), dict(mask=ok[:4])),
                      ((0, q, p), dict(mask=ok[:, 0])), ((0, q, p), dict(mask=ok[:3], offsets=i64([0, 3, 6]))),
                      ((0, q, p), dict(mask=ok.cpu())), ((0, q, p), dict(rows=i64([0]))),
                      ((0, q, p), dict(offsets=i64([0, 6]))), ((0, q, p), dict(rows=p.int())),
                      ((0, q, p), dict(scale=0.0)), ((0, q, p), dict(scale=float("inf"))),
                      ((0, q, p), dict(scale=float("nan"))), ((0, q, p), dict(out=q[:5])), ((0, q, p), dict(out=q.float())), ((0, q, i64([])), {})):
        with pytest.raises(RuntimeError):
            pc.tree_attention(ext, cache, *args, **how)


def test_values_against_the_plain_loop(ext):
    """One small case against the oracle's loop over rows, queries and heads."""
    announce("tree attention against the loop")
    rng = np.random.default_rng(15)
    cache = random_cache(rng, [21, 50, 3], kv_heads=2, dh=32, dtype=torch.float32)
    q = rng.standard_normal((7, 4, 32)).astype(np.float32)
    mask = rng.integers(-2**63, 2**63, (7, 1))
    want = of_cache(cache).attention(0, q, [18, 44, 0], mask.view(np.uint64), [0, 1, 2], [0, 2, 6, 7])
    got = pc.tree_attention(ext, on_gpu(cache), 0, torch.from_numpy(q).cuda(), i64([18, 44, 0]),
                            mask=torch.from_numpy(mask).cuda(), offsets=i64([0, 2, 6, 7]))
    # float32 throughout: 50 tokens, scores below 8 of 32 products each
    assert np.abs(got.cpu().numpy() - want).max() <= 50 * 8 * 32 * 2.0**-24
