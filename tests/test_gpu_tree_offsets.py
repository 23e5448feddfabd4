"""GPU: attention of drafted tokens whose offsets fall, which no caller may give: nothing outside the
call's tensors is read or written, and it ends."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from cugo_amd import paged_cache as pc
from tests.conftest import announce
from tests.test_gpu_paged_cache import i64

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,dh", [(torch.float16, 64), (torch.float32, 32)])
@pytest.mark.parametrize("group", [1, 8])
def test_more_work_than_is_counted(ext, dtype, dh, group):
    """400 sequences that claim all tokens in turn, over rows of 8 million: more tiles than 32 bits
    count.  Nobody is served."""
    announce(f"tree attention of falling offsets with too much work {dtype} dh {dh} x {group}")
    n, tokens = 400, 3200
    cache = pc.PagedKVCache(1, 3, 1, dh, 2, 1 << 15, "cuda", page=256, dtype=dtype)
    cache.table.zero_()
    cache.length.fill_(1 << 23)
    q = torch.ones(tokens, group, dh, dtype=dtype, device="cuda")
    offsets = i64(np.arange(n + 1) % 2 * tokens)
    rows, prefix = i64(np.arange(n) % 3), i64([1 << 23] * n)
    for fill in (0xff, 0x3f, 0x01):  # what the allocator's next block holds
        block = torch.full((64 << 20,), fill, dtype=torch.uint8, device="cuda")
        del block
        out = pc.tree_attention(ext, cache, 0, q, prefix, rows=rows, offsets=offsets,
                                out=torch.full_like(q, 7.0))
        assert (out == 7).all()
