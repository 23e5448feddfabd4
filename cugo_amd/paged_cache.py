"""A key/value cache in pages that rows share, and attention of drafted tokens over it.

The engine branches games (`clone_indexed`, `branch_indexed`); this is the sequence policy's
cache that branches with them.  The reference's cache (python/cugo_seq50.py:325-339) and
`seq_decode.KVCache` hold a run of slots for every row, so a child's history is copied whole
and its events are evaluated one at a time.  Here a row is a list of pages of a common pool:

  * `branch`: rows become copies of others, with room for more tokens.  Whole pages are shared; the
    page that will be written on is copied; the rows' old pages are given back.  With a row as its
    own source it grows, shrinks or (length 0) is freed;
  * `append`: new keys and values of one layer into their rows' pages;
  * `tree_attention`: the queries of drafted tokens over what their rows hold: the tokens before the
    drafts, and of the drafts those their mask names (their ancestors in a tree of events that may
    follow), or without a mask all earlier ones (a single new token, or a chunk of a sequence);
  * `accept`: of the drafts those on the accepted path move together, and the pages behind them are
    given back.

`tree_step` runs a policy's layers over drafted tokens with them, as `seq_decode.cached_step` does
over one token a row.  Everything is HIP kernels on the current stream without synchronising, and
can be captured in a HIP graph.  A cache is changed by one call at a time: calls on it from several
streams, and replays of graphs that hold them, have to be ordered by the caller.
"""

from __future__ import annotations

from typing import Sequence

import torch
from torch import nn

from .seq_decode import add_norm, attention_tail, linear


class PagedKVCache:
    """`rows` rows of up to `width` pages from a pool of `pages` pages of `page` tokens each.

    k and v [layers, pages, kv_heads, page, dh]; table int32 [rows, width] (a row's pages in order;
    entries past them mean nothing); length int64 [rows] (tokens that a row has pages for); refs
    int32 [pages] (rows that hold a page); free int64 [ceil(pages / 64)] (a bit for every page that
    none holds).  The functions below take any object with these tensors.  dh is 32, 64, 128 or
    256, page a power of two from 16 to 256, dtype bfloat16, float16 or float32."""

    def __init__(self, layers: int, rows: int, kv_heads: int, dh: int, pages: int, width: int,
                 device, page: int = 16, dtype: torch.dtype = torch.bfloat16) -> None:
        shape = (layers, pages, kv_heads, page, dh)
        self.k = torch.zeros(shape, dtype=dtype, device=device)
        self.v = torch.zeros(shape, dtype=dtype, device=device)
        self.table = torch.full((rows, width), -1, dtype=torch.int32, device=device)
        self.length = torch.zeros(rows, dtype=torch.int64, device=device)
        self.refs = torch.zeros(pages, dtype=torch.int32, device=device)
        self.free = torch.full(((pages + 63) // 64,), -1, dtype=torch.int64, device=device)
        if pages % 64:
            self.free[-1] = (1 << pages % 64) - 1


def _state(cache) -> tuple:
    return cache.k, cache.v, cache.table, cache.length, cache.refs, cache.free


def branch(ext, cache, dst: torch.Tensor, src: torch.Tensor, length: torch.Tensor) -> torch.Tensor:
    """Row dst[i] becomes the first min(cache.length[src[i]], length[i]) tokens of row src[i], with
    pages for length[i] (int64 [n] each); bool [n]: which entries were done.

    All entries see the rows as they are before the call.  Refused, and left as they are, are
    entries whose rows or length are out of range or whose dst is another entry's dst or src.  New
    pages are the lowest free ones, entry after entry; one that would need more than there are, with
    those before it, gets none (its dst is empty then; a row that is its own src stays).  After a
    call the positions from the kept tokens up to length[i] are the row's alone, to `append`
    into, until a row branched from it keeps tokens that end in one of their pages: cut a row to its
    tokens before (`accept`, or `branch` to itself), and grow it afterwards."""
    return ext.paged_branch(*_state(cache), dst, src, length)


def append(ext, cache, layer: int, k_new: torch.Tensor, v_new: torch.Tensor, pos: torch.Tensor,
           rows: torch.Tensor | None = None, *, out: torch.Tensor | None = None) -> torch.Tensor:
    """Token i's key and value (k_new and v_new [n, kv_heads, dh], any distance between tokens) to
    position pos[i] of row rows[i] (None: row i), int64 [n], in place; bool [n] (`out`, if given):
    which tokens were written.  Nothing is written outside a row's length or into a page that
    several rows hold (see `branch`).  No two tokens may have one place."""
    return ext.paged_append(*_state(cache), layer, k_new, v_new, pos, rows, out)


def accept(ext, cache, rows: torch.Tensor, start: torch.Tensor, keep: torch.Tensor) -> torch.Tensor:
    """Of the tokens of row rows[i] from position start[i] on, those at start[i] + keep[i, j] move to
    start[i] + j, in every layer, and the row ends behind them; bool [n]: which entries were done.

    rows and start int64 [n]; keep int64 [n, most], rising, ended by a negative entry (or the last
    one): a path through the drafted tokens.  Refused, and left as they are, are entries whose
    row or start is out of range, whose row is another entry's too, whose keep does not rise or goes past
    the length, or that would write into a page that several rows hold."""
    return ext.paged_accept(*_state(cache), rows, start, keep)


def tree_attention(ext, cache, layer: int, q: torch.Tensor, prefix: torch.Tensor, *,
                   mask: torch.Tensor | None = None, rows: torch.Tensor | None = None,
                   offsets: torch.Tensor | None = None, scale: float | None = None,
                   out: torch.Tensor | None = None) -> torch.Tensor:
    """softmax(q k^T scale) v over what each query attends: [tokens, heads, dh], q's dtype (the
    cache's; float32 sums).

    q [tokens, heads, dh] (any distance between tokens; heads a multiple of the cache's kv_heads,
    head h reads kv_head h // (heads // kv_heads)) holds the queries of n sequences one after
    another: sequence i's are offsets[i] ... offsets[i + 1] - 1 (int64 [n + 1], not falling; None: as
    many for each), its row rows[i] (int64 [n]; None: row i).  Query j of sequence i attends the positions
    below prefix[i] (int64 [n], taken into [0, length]) and from there on those whose bit is set in
    its mask, bit b for position prefix[i] + b, never past the row's length.  mask int64
    [tokens, words], bit b being bit b % 64 of word b // 64, or without offsets [tokens / n, words]
    for every sequence alike (`tree_mask`); None: the positions up to prefix[i] + j.

    A query that attends nothing, or only scores of -inf, gets zeros, one whose row does not exist
    NaN; tokens outside every sequence are left as they were in `out`.  scale None: dh ** -0.5.  No
    gradients."""
    return ext.tree_attention(*_state(cache), layer, q, prefix, mask, rows, offsets, scale, out)


def tree_mask(parents: Sequence[int], device=None) -> torch.Tensor:
    """`tree_attention`'s mask of one tree, int64 [tokens, words]: token j attends itself and its
    ancestors, parents[j] < j being its parent (negative: it follows the cached tokens)."""
    words = max(1, (len(parents) + 63) // 64)
    bits: list[int] = []
    for j, parent in enumerate(parents):
        if parent >= j:
            raise ValueError(f"token {j}'s parent {parent} must come before it")
        bits.append((bits[parent] if parent >= 0 else 0) | 1 << j)
    rows = [[(b >> 64 * w & (1 << 64) - 1) for w in range(words)] for b in bits]
    signed = [[x - (1 << 64) if x >> 63 else x for x in row] for row in rows]
    return torch.tensor(signed, dtype=torch.int64, device=device).reshape(len(parents), words)


def tree_step(model: nn.Module, ext, cache, x: torch.Tensor, prefix: torch.Tensor,
              pos: torch.Tensor, token_rows: torch.Tensor, *, mask: torch.Tensor | None = None,
              rows: torch.Tensor | None = None, offsets: torch.Tensor | None = None,
              final_norm: nn.Module | None = None, placed: torch.Tensor | None = None):
    """A policy's encoder layers over drafted tokens x [tokens, d] of n sequences: token t's key and
    value go to position pos[t] of row token_rows[t] at every layer, then the tokens attend
    (`tree_attention`'s prefix, mask, rows and offsets).  For modules laid out as
    `seq_decode.cached_step` takes them; the cache's rows need pages for the drafts (`branch`):
    `placed`, if given, bool [tokens], takes which tokens had a place (`append`); where one had none,
    those that attend it attend what is there.  Returns the final hidden states, and with
    final_norm (that, its norm)."""
    tokens, d = x.shape
    heads = cache.k.shape[2]
    layers = model.encoder.layers
    x, h = add_norm(x, None, layers[0].norm1)
    if placed is None:
        placed = torch.empty(tokens, dtype=torch.bool, device=x.device)
    for i, layer in enumerate(layers):
        sa = layer.self_attn
        q, k, v = (t.reshape(tokens, heads, d // heads)
                   for t in linear(h, sa.in_proj_weight, sa.in_proj_bias).chunk(3, -1))
        append(ext, cache, i, k, v, pos, token_rows, out=placed)
        a = tree_attention(ext, cache, i, q, prefix, mask=mask, rows=rows, offsets=offsets)
        last = i + 1 == len(layers)
        norm = final_norm if last else layers[i + 1].norm1
        out = attention_tail(layer, a.reshape(tokens, d), x, norm)
        x, h = out if norm is not None else (out, None)
    return x if final_norm is None else (x, h)
