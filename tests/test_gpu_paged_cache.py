"""GPU: the paged cache's branch, append and accept, bit for bit against the oracle
(oracle/paged_ref.py): tokens, tables, lengths, references and free bits after every call."""

from __future__ import annotations

from types import SimpleNamespace

import numpy as np
import pytest
import torch

from cugo_amd import paged_cache as pc
from oracle.paged_ref import of_cache, random_cache
from tests.conftest import announce

pytestmark = pytest.mark.gpu
TENSORS = ("k", "v", "table", "length", "refs", "free")
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def on_gpu(cache):
    return SimpleNamespace(**{n: getattr(cache, n).cuda() for n in TENSORS})


def same(cache, ref):
    """Every tensor of the cache is what the oracle has (table entries past a row's pages too)."""
    assert cache.length.tolist() == ref.length
    assert cache.refs.tolist() == ref.refs
    assert np.array_equal(cache.table.cpu().numpy(), ref.table)
    assert np.array_equal(cache.free.cpu().numpy(), ref.free_words())
    assert np.array_equal(cache.k.double().cpu().numpy(), ref.k, equal_nan=True)
    assert np.array_equal(cache.v.double().cpu().numpy(), ref.v, equal_nan=True)


def i64(x):
    return torch.tensor([int(v) for v in np.ravel(x)], dtype=torch.int64, device="cuda")


SHAPES = [("bf16", 32, 16, 8, 4), ("f16", 64, 16, 3, 1), ("f32", 32, 32, 2, 2),
          ("bf16", 128, 64, 1, 3), ("f32", 256, 16, 1, 1), ("f16", 256, 128, 2, 2),
          ("bf16", 64, 256, 5, 1)]


@pytest.mark.parametrize("dtype,dh,page,kv_heads,layers", SHAPES)
@pytest.mark.parametrize("spare", [2, 40])
def test_random_calls(ext, dtype, dh, page, kv_heads, layers, spare):
    """Branches (copies, cuts, growths, frees; rows out of range, named twice; too few pages),
    appends and accepted paths in turn."""
    announce(f"paged calls {dtype} dh {dh} page {page} heads {kv_heads} x {layers} spare {spare}")
    rng = np.random.default_rng(dh + page + spare)
    rows, width = 12, 5
    cache = on_gpu(random_cache(rng, [int(x) for x in rng.integers(0, width * page, rows)],
                                layers=layers, kv_heads=kv_heads, page=page, dh=dh, width=width,
                                spare=spare, dtype=TYPES[dtype]))
    ref = of_cache(cache)
    for turn in range(12):
        n = int(rng.integers(1, 9))
        dst, src = rng.integers(-1, rows + 1, n), rng.integers(-1, rows + 1, n)
        if turn % 3 == 0:  # every entry its own row
            dst = rng.permutation(rows)[:n]
            src = np.where(rng.random(n) < 0.5, dst, src)
        want = rng.integers(-1, width * page + 2, n)
        want = np.where(rng.random(n) < 0.3, [ref.tokens(s) if 0 <= s < rows else 0 for s in src], want)
        ok = pc.branch(ext, cache, i64(dst), i64(src), i64(want))
        assert ok.tolist() == ref.branch(dst, src, want)
        same(cache, ref)
        # tokens at places of their own, some outside
        count = int(rng.integers(0, 30))
        places = rng.permutation((rows + 2) * (width * page + 2))[:count]
        at_row, pos = places // (width * page + 2) - 1, places % (width * page + 2) - 1
        new = [torch.from_numpy(rng.standard_normal((count, kv_heads, dh))).to(cache.k) for _ in "kv"]
        layer = int(rng.integers(0, layers))
        pc.append(ext, cache, layer, *new, i64(pos), i64(at_row))
        ref.append(layer, *(x.double().cpu().numpy() for x in new), pos, at_row)
        same(cache, ref)
        n = int(rng.integers(1, 7))
        chosen = rng.permutation(rows)[:n] if turn % 2 else rng.integers(-1, rows + 1, n)
        have = [ref.tokens(r) if 0 <= r < rows else 0 for r in chosen]
        start = np.array([rng.integers(max(0, h - 40), h + 1) for h in have])
        most = int(rng.integers(1, 30))
        keep = np.sort(rng.integers(0, 40, (n, most)), axis=1)
        if turn % 4 != 0:  # rising
            keep = np.stack([np.sort(rng.permutation(45)[:most]) for _ in range(n)])
        keep[np.arange(most)[None] >= rng.integers(0, most + 1, n)[:, None]] = -1
        keep = np.where((start[:, None] + keep >= np.array(have)[:, None]) & (rng.random((n, 1)) < 0.9),
                        -1, keep)
        ok = pc.accept(ext, cache, i64(chosen), i64(start), i64(keep).view(n, most))
        assert ok.tolist() == ref.accept(chosen, start, keep)
        same(cache, ref)


def test_many_entries_in_order(ext):
    """More entries than a workgroup has threads, and fewer pages than they need: the first ones get
    the lowest pages."""
    announce("paged branch of 3,000 entries")
    rng = np.random.default_rng(1)
    lengths = [int(x) for x in rng.integers(1, 40, 100)] + [0] * 3000
    cache = on_gpu(random_cache(rng, lengths, kv_heads=1, width=4, spare=4000))
    ref = of_cache(cache)
    dst = 100 + rng.permutation(3000)
    src, room = rng.integers(0, 100, 3000), rng.integers(0, 25, 3000)
    want = np.array(lengths)[src] + room
    ok = pc.branch(ext, cache, i64(dst), i64(src), i64(want))
    # the oracle's rule that no entry's row is another's, which holds here, is quadratic in them
    assert ok.tolist() == ref.branch(dst, src, want)
    assert 0 < sum(ok.tolist()) < 3000
    same(cache, ref)
    ok = pc.branch(ext, cache, i64(dst), i64(dst), i64(np.zeros(3000)))
    assert all(ok.tolist()) and ref.branch(dst, dst, np.zeros(3000)) == ok.tolist()
    same(cache, ref)


def test_pools_of_many_pages(ext):
    """Free bits over several words a lane, the last word part filled; pages used up to the last."""
    announce("paged branch over 70,001 pages")
    pages = 70_001
    cache = pc.PagedKVCache(1, 40, 1, 32, pages, 8000, "cuda", dtype=torch.float32)
    rng = np.random.default_rng(2)
    used = torch.from_numpy(rng.random(pages) < 0.9)
    used[-70:] = False
    cache.refs.copy_(used.int())
    bits = torch.zeros(cache.free.numel() * 64, dtype=torch.int64)
    bits[:pages] = ~used
    cache.free.copy_((bits.view(-1, 64) << torch.arange(64)).sum(1))
    ids = torch.nonzero(~used)[:, 0]
    take = [2500, ids.numel() - 2500 - 3, 7, 3, 1]  # the third does not fit, nor what is after it
    want = [16 * t for t in take]
    ok = pc.branch(ext, cache, i64(range(5)), i64(range(5)), i64(want))
    assert ok.tolist() == [True, True, False, False, False]
    assert torch.equal(cache.table[0, :2500].cpu().long(), ids[:2500])
    assert torch.equal(cache.table[1, :take[1]].cpu().long(), ids[2500:-3])
    left = cache.refs.cpu() == 0
    assert torch.equal(torch.nonzero(left)[:, 0], ids[-3:])
    ok = pc.branch(ext, cache, i64([2]), i64([2]), i64([48]))
    assert ok.item() and cache.table[2, :3].tolist() == ids[-3:].tolist() == [pages - 3, pages - 2, pages - 1]
    assert not cache.free.any()


def test_strided_tokens_rows_by_default(ext):
    """Keys and values as parts of a packed projection; token i to row i."""
    announce("paged append of a packed projection's columns")
    rng = np.random.default_rng(3)
    cache = on_gpu(random_cache(rng, [20] * 7, kv_heads=8, layers=2))
    ref = of_cache(cache)
    packed = torch.randn(7, 3 * 256, device="cuda").to(torch.bfloat16)
    q, k, v = (t.reshape(7, 8, 32) for t in packed.chunk(3, -1))
    assert not k.is_contiguous()
    pos = i64([0, 19, 20, 5, -1, 16, 15])
    pc.append(ext, cache, 1, k, v, pos)
    ref.append(1, k.double().cpu().numpy(), v.double().cpu().numpy(), pos.tolist(), range(7))
    same(cache, ref)
    odd = torch.randn(7, 3 * 256 + 1, device="cuda").to(torch.bfloat16)[:, 1:]  # not 16-byte aligned
    q, k, v = (t.reshape(7, 8, 32) for t in odd.chunk(3, -1))
    flipped = k.flip(1).transpose(1, 2).contiguous().transpose(1, 2)  # heads not one after another
    pc.append(ext, cache, 0, flipped, v, pos)
    ref.append(0, flipped.double().cpu().numpy(), v.double().cpu().numpy(), pos.tolist(), range(7))
    same(cache, ref)


def test_corrupt_entries_are_not_followed(ext):
    """Lengths and table entries that no call wrote: nothing outside the pool is touched, references
    of other pages stay."""
    announce("paged calls over corrupt tables")
    rng = np.random.default_rng(4)
    cache = on_gpu(random_cache(rng, [40, 33, 20, 0, 0, 7], width=4, spare=20, layers=2))
    cache.table[0, 1] = 1 << 30
    cache.table[1, 2] = -7
    cache.length[2] = 1 << 50
    cache.table[2] = torch.tensor([-1, 1 << 20, -2**31, 2**31 - 1], dtype=torch.int32)
    ref = of_cache(cache)
    for dst, src, want in (([3, 4], [0, 1], [45, 40]), ([3], [2], [64]), ([1, 2], [1, 2], [50, 10]),
                           ([0, 1, 2, 3, 4], [0, 1, 2, 3, 4], [0, 0, 0, 0, 0])):
        ok = pc.branch(ext, cache, i64(dst), i64(src), i64(want))
        assert ok.tolist() == ref.branch(dst, src, want)
        same(cache, ref)
    cache.table[5, 0] = 1 << 28
    ref = of_cache(cache)
    ok = pc.accept(ext, cache, i64([5]), i64([1]), i64([[2, 4]]).view(1, 2))
    assert ok.tolist() == ref.accept([5], [1], [[2, 4]]) == [False]
    new = torch.ones(1, 2, 32, device="cuda", dtype=torch.bfloat16)
    pc.append(ext, cache, 0, new, new, i64([3]), i64([5]))
    same(cache, ref)


def test_empty_calls(ext):
    announce("paged calls without entries")
    cache = pc.PagedKVCache(1, 2, 2, 32, 3, 2, "cuda")
    none = i64([])
    assert pc.branch(ext, cache, none, none, none).shape == (0,)
    assert pc.accept(ext, cache, none, none, none.view(0, 4)).shape == (0,)
    pc.append(ext, cache, 0, cache.k[0, :0, :, 0], cache.v[0, :0, :, 0], none, none)
    assert pc.branch(ext, cache, i64([1]), i64([1]), i64([20])).item()
    # nothing kept: the row ends at its start
    assert pc.accept(ext, cache, i64([1]), i64([4]), none.view(1, 0)).item()
    assert cache.length.tolist() == [0, 4] and cache.refs.tolist() == [1, 0, 0]
    same(cache, of_cache(cache))


def test_offsets_past_32_bits(ext):
    """Pages whose bytes lie beyond 4 GiB of a layer's start, and layers beyond that."""
    announce("paged copies past 4 GiB")
    pages, layers = 70_000, 2  # 65,536 bytes a page: 4.6 GB a layer
    shape = (layers, pages, 8, 128, 32)
    k, v = (torch.empty(shape, dtype=torch.bfloat16, device="cuda") for _ in "kv")
    cache = pc.PagedKVCache(1, 3, 8, 32, pages, 3, "cuda", page=16)
    cache.k, cache.v = k, v
    high = list(range(pages - 6, pages))
    cache.refs.fill_(1)
    cache.refs[high] = 0
    cache.free.zero_()
    for p in high:
        cache.free[p // 64] |= torch.tensor(1, dtype=torch.int64, device="cuda") << (p % 64)
    assert pc.branch(ext, cache, i64([0]), i64([0]), i64([200])).item()
    assert cache.table[0, :2].tolist() == high[:2]
    new = [torch.randn(200, 8, 32, device="cuda").to(torch.bfloat16) for _ in range(4)]
    for layer in (0, 1):
        pc.append(ext, cache, layer, new[2 * layer], new[2 * layer + 1], i64(range(200)), i64([0] * 200))
    assert pc.branch(ext, cache, i64([1]), i64([0]), i64([300])).item()
    assert cache.table[1].tolist() == [high[0], high[2], high[3]]
    assert pc.accept(ext, cache, i64([1]), i64([130]), i64([0, 10, 69]).view(1, 3)).item()
    for layer in (0, 1):
        for x, want in ((k, new[2 * layer]), (v, new[2 * layer + 1])):
            got = x[layer, [high[0], high[2]]].transpose(1, 2).reshape(256, 8, 32)
            assert torch.equal(got[:131], want[:131])
            assert torch.equal(got[131:133], want[[140, 199]])


def test_other_stream_and_graph(ext):
    """The calls on a stream of their own, and captured: every replay does what the eager call does."""
    announce("paged calls captured and replayed")
    rng = np.random.default_rng(6)
    lengths = [int(x) for x in rng.integers(1, 60, 8)] + [0] * 24
    host = random_cache(rng, lengths, kv_heads=8, layers=2, width=6, spare=200)
    eager, graphed = on_gpu(host), on_gpu(host)
    ref = of_cache(host)
    src = rng.integers(0, 8, 24)
    want = np.array(lengths)[src] + 7
    dst = 8 + rng.permutation(24)
    pos = (np.array(lengths)[src][:, None] + np.arange(7)).ravel()
    new = [torch.randn(24 * 7, 8, 32, device="cuda").to(torch.bfloat16) for _ in "kv"]
    keep = i64([[0, 2, 5, -1]] * 24).view(24, 4)
    args = [i64(dst), i64(src), i64(want), i64(np.array(lengths)[src]), i64(pos), i64(dst.repeat(7))]

    def round_of(cache):
        d, s, w, start, at, of = args
        a = pc.branch(ext, cache, d, s, w)
        pc.append(ext, cache, 1, *new, at, of)
        b = pc.accept(ext, cache, d, start, keep)
        return a, b

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        round_of(graphed)
    torch.cuda.current_stream().wait_stream(side)
    round_of(eager)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        oks = round_of(graphed)
    values = [x.double().cpu().numpy() for x in new]

    def by_oracle():
        a = ref.branch(dst, src, want)
        ref.append(1, *values, pos, dst.repeat(7))
        return a, ref.accept(dst, np.array(lengths)[src], keep.tolist())

    by_oracle()
    same(eager, ref)
    same(graphed, ref)
    for _ in range(4):
        for ok in oks:
            ok.zero_()
        graph.replay()
        seen = round_of(eager)
        torch.cuda.synchronize()
        wanted = by_oracle()
        for got, other, should in zip(oks, seen, wanted):
            assert got.tolist() == other.tolist() == should
        same(eager, ref)
        same(graphed, ref)


def test_refusals(ext):
    announce("paged calls refused")
    cache = pc.PagedKVCache(2, 3, 2, 32, 9, 4, "cuda")
    x = torch.zeros(4, 2, 32, dtype=torch.bfloat16, device="cuda")
    i = i64([0, 1, 2, 0])

    def changed(**over):
        return SimpleNamespace(**{**{n: getattr(cache, n) for n in TENSORS}, **over})

    for bad, match in ((dict(k=cache.k.double()), "v must be"), (dict(v=cache.v[:1]), "v must be"),
                       (dict(k=cache.k.double(), v=cache.v.double()), "float32, float16 or bfloat16"),
                       (dict(k=cache.k[..., :16].contiguous(), v=cache.v[..., :16].contiguous()), "dh"),
                       (dict(k=cache.k[:, :, :, :8].contiguous(), v=cache.v[:, :, :, :8].contiguous()), "page"),
                       (dict(k=cache.k[:, :, :, ::2], v=cache.v), "contiguous"),
                       (dict(table=cache.table.long()), "table"), (dict(table=cache.table.t()), "table"),
                       (dict(length=cache.length[:2]), "length"), (dict(refs=cache.refs[:8]), "refs"),
                       (dict(refs=cache.refs.long()), "refs"), (dict(free=cache.free.int()), "free"),
                       (dict(free=torch.zeros(2, dtype=torch.int64, device="cuda")), "free"),
                       (dict(table=cache.table.cpu()), "device|CUDA"), (dict(k=cache.k[:0], v=cache.v[:0]), "no pages")):
        with pytest.raises(RuntimeError, match=match):
            pc.branch(ext, changed(**bad), i, i, i)
    for bad in ((i.int(), i, i), (i[:3], i, i), (i, i, i[:, None]), (i.cpu(), i, i), (i, i[::2], i)):
        with pytest.raises(RuntimeError):
            pc.branch(ext, cache, *bad)
    for bad in ((2, x, x, i, i), (-1, x, x, i, i), (0, x.float(), x, i, i), (0, x, x[:3], i, i),
                (0, x[:, :1], x[:, :1], i, i), (0, x, x, i[:3], i), (0, x, x, i, i[:3]),
                (0, x, x, i.int(), i), (0, x.cpu(), x, i, i)):
        with pytest.raises(RuntimeError):
            pc.append(ext, cache, *bad)
    keep = i.view(4, 1)
    for bad in ((i, i, i), (i, i, keep.int()), (i, i, keep[:3]), (i[:3], i, keep), (i, i.int(), keep),
                (i, i, i64(range(16)).view(4, 4).t()), (i, i, keep.cpu())):
        with pytest.raises(RuntimeError):
            pc.accept(ext, cache, *bad)
