"""GPU: the paged cache's operators as a search uses them: a policy's layers over trees of drafted
tokens (`tree_step`), rows branched from each other, paths accepted, against `cached_step` over a
dense cache that takes each path one token at a time."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from cugo_amd import paged_cache as pc
from cugo_amd.seq_decode import add_norm
from cugo_amd.seq_selfplay import SeqPolicy, policy_cache
from tests.conftest import announce
from tests.test_gpu_paged_cache import i64

pytestmark = pytest.mark.gpu

# Relative 2-norms.  float32: four layers, each at most 3 * 1,024 products and sums deep between
# norms, half a step (2^-24) each.  bfloat16: ten roundings of at most 2^-8 a layer (projections,
# attention's weights and outputs, two norms, two feed-forward layers, two sums).
TOLERANCE = {torch.float32: 4 * 3 * 1024 * 2.0**-24, torch.bfloat16: 4 * 10 * 2.0**-8}


def near(got, want):
    off = torch.linalg.vector_norm(got.double() - want.double()) / torch.linalg.vector_norm(want.double())
    assert off <= TOLERANCE[want.dtype], float(off)


def paged_for(policy, rows, pages, width=8, page=16):
    layers = policy.encoder.layers
    heads = layers[0].self_attn.num_heads
    d = policy.position.shape[1]
    return pc.PagedKVCache(len(layers), rows, heads, d // heads, pages, width, "cuda", page,
                           policy.event_in.weight.dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@torch.no_grad()
def test_rounds_of_a_search(ext, dtype):
    """Histories through the layers as chains; then rounds of: children branched, a tree of drafts in
    one pass, one path of it accepted.  Each draft's hidden state is what the dense cache gives when
    its path is appended token by token."""
    announce(f"rounds of a search {dtype}")
    torch.manual_seed(3)
    policy = SeqPolicy().to("cuda", dtype).eval()
    rng = np.random.default_rng(3)
    roots, children, d = 3, 7, 256
    cache = paged_for(policy, roots + children, 400)

    def tokens(n):
        return torch.randn(n, d, device="cuda").to(dtype)

    counts = [5, 16, 23]
    rows = i64(range(roots))
    prefix = i64([0] * roots)
    assert pc.branch(ext, cache, rows, rows, i64(counts)).all()
    history = [tokens(c) for c in counts]
    offsets = i64(np.concatenate([[0], np.cumsum(counts)]))
    which = np.repeat(np.arange(roots), counts)
    pos = i64(np.concatenate([np.arange(c) for c in counts]))
    pc.tree_step(policy, ext, cache, torch.cat(history), prefix, pos, i64(which), rows=rows,
                 offsets=offsets)
    paths = {r: list(history[r]) for r in range(roots)}
    for turn in range(3):
        src = rng.integers(0, roots, children)
        dst = roots + np.arange(children)
        parents = [-1, 0, 0, 1, 3, -1, 2, 5]
        t = len(parents)
        have = np.array([len(paths[s]) for s in src])
        assert pc.branch(ext, cache, i64(dst), i64(src), i64(have + t)).all()
        x = tokens(children * t)
        mask = pc.tree_mask(parents, "cuda")
        at = (have[:, None] + np.arange(t)).ravel()
        y, z = pc.tree_step(policy, ext, cache, x, i64(have), i64(at), i64(dst.repeat(t)), mask=mask,
                            rows=i64(dst), final_norm=policy.norm)
        near(z, add_norm(y.clone(), None, policy.norm)[1])
        # every draft's path, token by token over a dense cache
        lines, last = [], []
        for c in range(children):
            for j in range(t):
                line, k = [], j
                while k >= 0:
                    line.append(x[c * t + k])
                    k = parents[k]
                lines.append(paths[src[c]] + line[::-1])
        longest = max(map(len, lines))
        dense = policy_cache(policy, len(lines), "cuda", slots=longest + 1)
        dense.k, dense.v = dense.k.to(dtype), dense.v.to(dtype)
        for step in range(longest):
            now = torch.stack([line[min(step, len(line) - 1)] for line in lines])
            out = policy.cached_step(dense, now.clone())
            last.append(out)
            dense.length += 1
        want = torch.stack([last[len(line) - 1][i] for i, line in enumerate(lines)])
        near(y, want)
        # one child's path is taken over by its root; its other drafts are gone
        c = int(rng.integers(0, children))
        keep = i64([0, 1, 3, 4]).view(1, 4)
        assert pc.accept(ext, cache, i64(dst[c:c + 1]), i64(have[c:c + 1]), keep).all()
        root = int(src[c])
        paths[root] = paths[root] + [x[c * t + k] for k in (0, 1, 3, 4)]
        assert pc.branch(ext, cache, i64([root]), i64([dst[c]]), i64([len(paths[root])])).all()
    # a further token of each root by itself: the cache holds what the dense one would
    last = tokens(roots)
    have = np.array([len(paths[r]) for r in range(roots)])
    assert pc.branch(ext, cache, rows, rows, i64(have + 1)).all()
    y = pc.tree_step(policy, ext, cache, last.clone(), i64(have), i64(have), rows)
    longest = int(have.max()) + 1
    dense = policy_cache(policy, roots, "cuda", slots=longest + 1)
    dense.k, dense.v = dense.k.to(dtype), dense.v.to(dtype)
    outs = []
    for step in range(longest):
        now = torch.stack([(paths[r] + [last[r]])[min(step, have[r])] for r in range(roots)])
        outs.append(policy.cached_step(dense, now.clone()))
        dense.length += 1
    near(y, torch.stack([outs[have[r]][r] for r in range(roots)]))
    assert pc.branch(ext, cache, i64(range(roots + children)), i64(range(roots + children)),
                     i64([0] * (roots + children))).all()
    assert not cache.refs.any()
