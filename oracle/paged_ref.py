"""The paged cache's operators, plainly: rows as lists worked on one entry at a time, attention in
64 bits.  Test infrastructure for cugo_amd.paged_cache."""

from __future__ import annotations

import numpy as np


class PagedRef:
    """k and v: float64 [layers, pages, kv_heads, page, dh]; the rest as int64 arrays or lists."""

    def __init__(self, k, v, table, length, refs):
        self.k, self.v = np.array(k, dtype=np.float64), np.array(v, dtype=np.float64)
        self.table = np.array(table, dtype=np.int64)
        self.length = [int(x) for x in length]
        self.refs = [int(x) for x in refs]
        self.page = self.k.shape[3]
        self.rows, self.width = self.table.shape

    def tokens(self, row: int) -> int:
        return min(max(self.length[row], 0), self.width * self.page)

    def held(self, tokens: int) -> int:
        return -(-tokens // self.page)

    def page_at(self, row: int, index: int) -> int | None:
        p = int(self.table[row, index])
        return p if 0 <= p < len(self.refs) else None

    def free_words(self) -> np.ndarray:
        words = [0] * (-(-len(self.refs) // 64))
        for p, r in enumerate(self.refs):
            words[p // 64] |= (r == 0) << (p % 64)
        return np.array(words, dtype=np.uint64).view(np.int64)

    def _known(self, row: int) -> bool:
        return 0 <= row < self.rows

    def branch(self, dst, src, length) -> list[bool]:
        dst, src, length = [int(x) for x in dst], [int(x) for x in src], [int(x) for x in length]
        fine = []
        for i, (d, s, n) in enumerate(zip(dst, src, length)):
            others = [x for j in range(len(dst)) if j != i for x in (dst[j], src[j])]
            fine.append(self._known(d) and self._known(s) and 0 <= n <= self.width * self.page
                        and d not in others)
        for d, s, n, go in zip(dst, src, length, fine):
            if go:
                for j in range(self.held(n) if d == s else 0, self.held(self.tokens(d))):
                    if (p := self.page_at(d, j)) is not None:
                        self.refs[p] -= 1
        after = list(self.refs)
        empty = [p for p, r in enumerate(after) if r == 0]
        taken, ok, copies = 0, [], []
        for d, s, n, go in zip(dst, src, length, fine):
            if not go:
                ok.append(False)
                continue
            kept = min(self.tokens(s), n)
            whole, part = kept // self.page, kept % self.page
            copy = None
            if part and n == kept:
                whole += 1
            elif part:
                p = self.page_at(s, whole)
                if d == s and (p is None or after[p] <= 1):
                    whole += 1
                elif p is not None:
                    copy = p
            need = max(0, self.held(n) - whole)
            taken += need
            if need and taken > len(empty):
                ok.append(False)
                if d != s:
                    self.length[d] = 0
                continue
            new = empty[taken - need:taken]
            for p in new:
                self.refs[p] += 1
            for j in range(self.held(n)):
                if j >= whole:
                    self.table[d, j] = new[j - whole]
                elif d != s:
                    self.table[d, j] = self.table[s, j]
                    if (p := self.page_at(s, j)) is not None:
                        self.refs[p] += 1
            if copy is not None:
                copies.append((copy, new[0], part))
                if d == s:
                    self.refs[copy] -= 1
            self.length[d] = n
            ok.append(True)
        for a, b, part in copies:
            for x in (self.k, self.v):
                x[:, b, :, :part] = x[:, a, :, :part]
        return ok

    def append(self, layer, k_new, v_new, pos, rows) -> None:
        for i, (r, t) in enumerate(zip(rows, pos)):
            r, t = int(r), int(t)
            if not self._known(r) or not 0 <= t < self.tokens(r):
                continue
            p = self.page_at(r, t // self.page)
            if p is None or self.refs[p] != 1:
                continue
            self.k[layer, p, :, t % self.page] = k_new[i]
            self.v[layer, p, :, t % self.page] = v_new[i]

    def accept(self, rows, start, keep) -> list[bool]:
        rows, start = [int(x) for x in rows], [int(x) for x in start]
        ok, paths = [], []
        for r, s, path in zip(rows, start, keep):
            path = [int(x) for x in path]
            path = path[:next((j for j, x in enumerate(path) if x < 0), len(path))]
            fine = self._known(r) and rows.count(r) == 1
            fine = fine and 0 <= s <= self.tokens(r)
            fine = fine and all(a < b for a, b in zip(path, path[1:]))
            fine = fine and all(s + x < self.tokens(r) for x in path)
            if fine:
                for j, x in enumerate(path):
                    if x != j:
                        p = self.page_at(r, (s + j) // self.page)
                        fine = fine and p is not None and self.refs[p] == 1
            ok.append(fine)
            paths.append(path)
        for r, s, path, go in zip(rows, start, paths, ok):
            if not go:
                continue
            for j, x in enumerate(path):
                a = self.page_at(r, (s + x) // self.page)
                b = self.page_at(r, (s + j) // self.page)
                if x != j and a is not None:
                    for y in (self.k, self.v):
                        y[:, b, :, (s + j) % self.page] = y[:, a, :, (s + x) % self.page]
            for j in range(self.held(s + len(path)), self.held(self.tokens(r))):
                if (p := self.page_at(r, j)) is not None:
                    self.refs[p] -= 1
            self.length[r] = s + len(path)
        return ok

    def attention(self, layer, q, prefix, mask=None, rows=None, offsets=None, scale=None, out=None):
        """float64 [tokens, heads, dh]; tokens outside every sequence keep `out` (zeros)."""
        q = np.asarray(q, dtype=np.float64)
        tokens, heads, dh = q.shape
        group = heads // self.k.shape[2]
        n = len(prefix)
        scale = dh ** -0.5 if scale is None else scale
        out = np.zeros(q.shape) if out is None else np.array(out, dtype=np.float64)
        each = tokens // n if n else 0
        for i in range(n):
            first, end = ((i * each, (i + 1) * each) if offsets is None
                          else (int(offsets[i]), int(offsets[i + 1])))
            r = i if rows is None else int(rows[i])
            for t in range(first, end):
                if not self._known(r):
                    out[t] = np.nan
                    continue
                have = self.tokens(r)
                pre = min(max(int(prefix[i]), 0), have)
                seen = list(range(pre))
                if mask is None:
                    seen += [x for x in range(pre, min(pre + t - first + 1, have))]
                else:
                    words = mask[t if len(mask) == tokens else t - first]
                    for w, word in enumerate(words):
                        seen += [pre + 64 * w + b for b in range(64)
                                 if int(word) >> b & 1 and pre + 64 * w + b < have]
                if not seen:
                    out[t] = 0.0
                    continue
                pages = [self.page_at(r, x // self.page) for x in seen]
                if None in pages:
                    out[t] = np.nan
                    continue
                slots = [x % self.page for x in seen]
                for h in range(heads):
                    k = self.k[layer, pages, h // group, slots]
                    v = self.v[layer, pages, h // group, slots]
                    with np.errstate(invalid="ignore"):
                        s = k @ q[t, h] * scale
                        if s.max() == -np.inf:  # zeros
                            out[t, h] = 0.0
                            continue
                        e = np.exp(s - s.max())
                        out[t, h] = (e / e.sum()) @ v
        return out


def of_cache(cache) -> PagedRef:
    """The reference over a copy of a cache's tensors."""
    host = [t.double().cpu().numpy() for t in (cache.k, cache.v)]
    return PagedRef(*host, cache.table.cpu().numpy(), cache.length.tolist(), cache.refs.tolist())


def random_cache(rng, lengths, *, layers=1, kv_heads=2, page=16, dh=32, width=None, spare=3,
                 dtype=None, fill=float("nan")):
    """A cache on the CPU whose row r holds lengths[r] random tokens in pages anywhere in the pool;
    every slot that holds no token is `fill`."""
    from types import SimpleNamespace

    import torch

    rows = len(lengths)
    held = [-(-n // page) for n in lengths]
    width = max(1, *held) if width is None else width
    pages = sum(held) + spare
    place = rng.permutation(pages)
    table = np.full((rows, width), -1, dtype=np.int32)
    table[...] = rng.integers(-5, pages + 5, table.shape)  # entries past a row's pages mean nothing
    refs = np.zeros(pages, dtype=np.int32)
    k = np.full((2, layers, pages, kv_heads, page, dh), fill, dtype=np.float32)
    at = 0
    for r, n in enumerate(lengths):
        own = place[at:at + held[r]]
        at += held[r]
        table[r, :held[r]] = own
        refs[own] = 1
        for j, p in enumerate(own):
            have = min(page, n - j * page)
            k[:, :, p, :, :have] = rng.standard_normal((2, layers, kv_heads, have, dh))
    cache = SimpleNamespace(table=torch.from_numpy(table), refs=torch.from_numpy(refs),
                            length=torch.tensor([int(n) for n in lengths]))
    dtype = torch.bfloat16 if dtype is None else dtype
    cache.k, cache.v = (torch.from_numpy(x).to(dtype) for x in k)
    cache.free = torch.from_numpy(of_cache(cache).free_words())
    return cache


def dense_attention(cache, layer, q, prefix, mask=None, rows=None, offsets=None, scale=None, twice=False):
    """PagedRef.attention with torch in float64 on the tensors' device, for larger cases.  Returns the
    outputs, and for each how far one in `dtype` may be off when scores, softmax and sums are
    float32 and weights and outputs are rounded to the type (all bounds worked out below); `twice`:
    weights as the sum of two numbers of the type."""
    import torch

    tokens, heads, dh = q.shape
    page, kv_heads = cache.k.shape[3], cache.k.shape[2]
    group, n = heads // kv_heads, prefix.numel()
    scale = dh ** -0.5 if scale is None else scale
    out, bound = (torch.zeros(q.shape, dtype=torch.float64, device=q.device) for _ in range(2))
    half = torch.finfo(q.dtype).eps / 2
    single = 2.0**-24
    each = tokens // n if n else 0
    for i in range(n):
        first, end = (i * each, (i + 1) * each) if offsets is None else (int(offsets[i]), int(offsets[i + 1]))
        if end <= first:
            continue
        r = i if rows is None else int(rows[i])
        have = min(max(int(cache.length[r]), 0), cache.table.shape[1] * page)
        if have == 0:  # zeros, exactly
            continue
        pre = min(max(int(prefix[i]), 0), have)
        t = end - first
        at = torch.arange(have, device=q.device)
        j = torch.arange(t, device=q.device)
        if mask is None:
            seen = at <= pre + j[:, None]
        else:
            m = mask[first:end] if mask.shape[0] == tokens else mask
            b = (at - pre).clamp_min(0)
            inside = b < 64 * m.shape[1]
            word = m[:, (b // 64).clamp(max=max(0, m.shape[1] - 1))] if m.shape[1] else torch.zeros(t, have, dtype=torch.int64, device=q.device)
            seen = (at < pre) | (((word >> (b % 64)) & 1 == 1) & inside)
        held = cache.table[r, :-(-have // page)].long()
        k, v = (x[layer, held].transpose(0, 1).reshape(kv_heads, -1, dh)[:, :have].double()
                for x in (cache.k, cache.v))
        x = q[first:end].double().view(t, kv_heads, group, dh).permute(1, 2, 0, 3).reshape(kv_heads, group * t, dh)
        # masked places hold anything, NaN too: their keys are left out one way or the other
        s = (x @ k.mT).view(kv_heads, group, t, have) * scale
        s = s.masked_fill(~seen, -torch.inf)
        none = s.amax(3, keepdim=True) == -torch.inf  # nothing is attended, or only scores of -inf
        w = s.masked_fill(none, 0.0).softmax(3).masked_fill(~seen | none, 0.0)
        safe_v = torch.where(seen.any(0)[:, None], v, 0.0)
        y = (w.reshape(kv_heads, group * t, have) @ safe_v).view(kv_heads, group, t, dh)
        spread = (w.reshape(kv_heads, group * t, have) @ safe_v.abs()).view(kv_heads, group, t, dh)
        # a score's error: dh products and sums and the scaling, each half a step of the sum of
        # magnitudes; exp2 of a number of that size, a step of it and two of the result
        size = (x.abs() @ k.abs().mT).view(kv_heads, group, t, have) * scale
        size = size.masked_fill(~seen | (s == -torch.inf), 0.0).amax(3, keepdim=True)
        off = 2 * (dh + 8) * single * size + 4 * single
        # the weights' sum and the outputs' over `have` tokens, rescaled now and then; a weight
        # rounded to the type
        weight = 0.0 if q.dtype == torch.float32 else half * half if twice else half
        off = off + 2 * (have + 64) * single + weight
        far = half * y.abs() + 2 * off * spread + torch.finfo(q.dtype).smallest_normal
        if twice and q.dtype == torch.float16:  # half its smallest step, of weights of 2^7 at the top
            far = far + have * 2.0**-32 * safe_v.abs().amax(1)[:, None, None]
        out[first:end] = y.permute(2, 0, 1, 3).reshape(t, heads, dh)
        bound[first:end] = far.permute(2, 0, 1, 3).reshape(t, heads, dh)
    return out, bound
