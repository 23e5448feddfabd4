"""GPU: what `append` says of tokens that it does not write, and how a row whose room others share gets room
of its own again."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from cugo_amd import paged_cache as pc
from cugo_amd.seq_selfplay import SeqPolicy
from oracle.paged_ref import of_cache, random_cache
from tests.conftest import announce
from tests.test_gpu_paged_cache import TYPES, i64, on_gpu, same
from tests.test_gpu_tree_step import paged_for

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,dh,kv_heads", [("bf16", 32, 8), ("f16", 64, 1), ("f32", 256, 5), ("bf16", 128, 40)])
def test_which_tokens_were_written(ext, dtype, dh, kv_heads):
    """Tokens of few and of many parts (several a workgroup; more than its threads)."""
    announce(f"paged append's answers {dtype} dh {dh} heads {kv_heads}")
    rng = np.random.default_rng(dh)
    cache = on_gpu(random_cache(rng, [40, 33, 0, 16, 64], kv_heads=kv_heads, dh=dh, layers=2, width=4, spare=9,
                                dtype=TYPES[dtype]))
    assert pc.branch(ext, cache, i64([2]), i64([0]), i64([35])).all()  # shares row 0's three pages
    cache.table[4, 3] = 1 << 29
    ref = of_cache(cache)
    at_row = [0, 0, 2, 2, 2, 1, 1, 3, 3, 3, -1, 5, 4, 4, 1 << 40, 1] + [1] * 10
    pos = [39, 20, 34, 35, 3, 32, 33, 15, 16, -1, 0, 0, 47, 48, 0, -(1 << 50)] + list(range(10))
    want = [False, False, False, False, False, True, False, True, False, False, False, False, True, False,
            False, False] + [True] * 10
    new = [torch.from_numpy(rng.standard_normal((len(pos), kv_heads, dh))).to(cache.k) for _ in "kv"]
    ok = pc.append(ext, cache, 1, *new, i64(pos), i64(at_row))
    ref.append(1, *(x.double().cpu().numpy() for x in new), pos, at_row)
    same(cache, ref)
    assert ok.dtype == torch.bool and ok.tolist() == want
    out = torch.zeros(len(pos), dtype=torch.bool, device="cuda")
    assert pc.append(ext, cache, 1, *new, i64(pos), i64(at_row), out=out).data_ptr() == out.data_ptr()
    assert out.tolist() == want
    same(cache, ref)
    for bad in (out[:-1], out.int(), out.cpu(), out[:, None]):
        with pytest.raises(RuntimeError):
            pc.append(ext, cache, 1, *new, i64(pos), i64(at_row), out=bad)


def test_room_that_a_child_shares(ext):
    """A row with room in the page that a child of its tokens shares: not written and said so; cut and
    grown again it has a page of its own, and the child keeps what it had."""
    announce("paged append into shared room")
    rng = np.random.default_rng(8)
    cache = on_gpu(random_cache(rng, [48, 0], kv_heads=2, width=4, spare=6, layers=1))
    assert pc.branch(ext, cache, i64([1]), i64([0]), i64([40])).all()
    new = [torch.randn(8, 2, 32, device="cuda").to(torch.bfloat16) for _ in "kv"]
    before = cache.k.clone(), cache.v.clone()
    room = i64(range(40, 48)), i64([0] * 8)
    assert not pc.append(ext, cache, 0, *new, *room).any()
    assert torch.equal(cache.k.nan_to_num(), before[0].nan_to_num())
    assert torch.equal(cache.v.nan_to_num(), before[1].nan_to_num())
    page = int(cache.table[1, 2])
    assert pc.branch(ext, cache, i64([0]), i64([0]), i64([40])).all()
    assert pc.branch(ext, cache, i64([0]), i64([0]), i64([48])).all()
    assert int(cache.table[0, 2]) != page == int(cache.table[1, 2])
    assert pc.append(ext, cache, 0, *new, *room).all()
    assert torch.equal(cache.k[0, page].nan_to_num(), before[0][0, page].nan_to_num())
    own = cache.k[0, cache.table[0, 2].long()]
    assert torch.equal(own[:, :8], before[0][0, page][:, :8])
    assert torch.equal(own[:, 8:], new[0].transpose(0, 1))


@torch.no_grad()
def test_step_says_which_had_a_place(ext):
    announce("tree step with drafts that have no place")
    torch.manual_seed(5)
    policy = SeqPolicy().to("cuda", torch.bfloat16).eval()
    cache = paged_for(policy, 3, 20)
    rows = i64([0, 1])
    assert pc.branch(ext, cache, rows, rows, i64([5, 20])).all()
    placed = torch.zeros(7, dtype=torch.bool, device="cuda")
    x = torch.randn(7, 256, device="cuda").to(torch.bfloat16)
    how = dict(rows=rows, offsets=i64([0, 5, 7]))
    at = i64([0, 1, 2, 3, 5, 19, 20]), i64([0] * 5 + [1] * 2)
    a = pc.tree_step(policy, ext, cache, x.clone(), i64([0, 19]), *at, placed=placed, **how)
    assert placed.tolist() == [True] * 4 + [False, True, False]
    assert torch.equal(a, pc.tree_step(policy, ext, cache, x.clone(), i64([0, 19]), *at, **how))
