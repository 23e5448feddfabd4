"""GPU: small softmax weights in the attention of drafted tokens.  One token's score lies far above all
others', whose values are all that the result is made of: a type's smallest numbers must not swallow
them, whichever way the call is dealt out."""

from __future__ import annotations

import math

import pytest
import torch

from cugo_amd import paged_cache as pc
from tests.conftest import announce
from tests.test_gpu_paged_cache import i64

pytestmark = pytest.mark.gpu

# sequences, queries each, heads a key head, tokens a row, table's width in pages of 128: a wavefront an
# item (2,048 of them at least), a workgroup an item, shared out; with more than 32 rows in few
# sequences the 16-bit types of dh 64 and more go through LDS
DEALT = {"wavefront": (2048, 1, 1, 4096, 32), "group": (3, 2, 4, 4096, 32), "shared": (1, 1, 1, 131_072, 1024),
         "shared, 3 rows": (3, 5, 1, 20_000, 400), "through LDS": (2, 48, 1, 1024, 8),
         "through LDS, shared": (1, 64, 2, 131_072, 1024)}


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dh", [32, 64, 128, 256])
@pytest.mark.parametrize("dealt", DEALT)
def test_many_small_weights(ext, dtype, dh, dealt):
    announce(f"tree attention of small weights {dtype} dh {dh}, {dealt}")
    n, each, group, tokens, width = DEALT[dealt]
    held = tokens // 128 + (tokens % 128 > 0)
    cache = pc.PagedKVCache(1, 1, 1, dh, held, width, "cuda", page=128, dtype=dtype)
    cache.table[0, :held] = torch.arange(held, dtype=torch.int32)
    cache.length.fill_(tokens)
    rows, prefix = i64([0] * n), i64([tokens - 1] * n)
    q = torch.zeros(n * each, group, dh, dtype=dtype, device="cuda")
    q[..., 0] = 4.0
    mask = torch.ones(n * each, 1, dtype=torch.int64, device="cuda")
    half = torch.finfo(dtype).eps / 2
    for first in (0, 70, tokens - 3):  # where the one lies
        cache.k.zero_()
        cache.k[0, first // 128, 0, first % 128, 0] = 1.0
        cache.v.fill_(64.0)
        cache.v[0, first // 128, 0, first % 128] = 0.0
        for gap in (9.0, 14.5, 17.0, 17.4, 19.0):  # natural logarithms of the weights' ratio
            out = pc.tree_attention(ext, cache, 0, q, prefix, rows=rows, mask=mask, scale=gap / 4)
            small = math.exp(-gap)
            want = 64 * (tokens - 1) * small / (1 + (tokens - 1) * small)
            # the output's rounding and the weights' (all of them the same way), float32's in a
            # score of 28 in base 2 and in sums of `tokens`; half of float16's smallest step, of weights
            # that are at least 2^7 at the top
            bound = want * (2 * half + 2 * 28 * 2.0**-24 + (tokens + 64) * 2.0**-24) + half * torch.finfo(dtype).smallest_normal
            if dtype == torch.float16:
                bound += 64 * (tokens - 1) * 2.0**-32
            far = (out.double() - want).abs().max().item()
            assert far <= bound, (first, gap, want, far, bound)
