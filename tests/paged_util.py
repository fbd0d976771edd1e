"""A paged cache with content, and the same content as 64-bit tensors per sequence."""
from __future__ import annotations

import torch

from moshi_b200.models import PagedBatch, PagedKVCache
from oracle import paged as oracle


class Content:
    """`lengths`: tokens in the cache of each sequence, in pages from anywhere; everything else in the cache is garbage (for e4m3 NaN)."""

    def __init__(self, lengths, kv_heads, dim, page, dtype, seed=0, spread=1.0, spare=2, capacity=None):
        g = torch.Generator().manual_seed(seed)
        self.kv_heads, self.dim, self.page, self.dtype, self.lengths = kv_heads, dim, page, dtype, list(lengths)
        room = [max(x, c) for x, c in zip(lengths, capacity or lengths)]
        counts = [-(-x // page) for x in room]
        self.pages, self.width = sum(counts) + spare, max(max(counts), 1)
        order = torch.randperm(self.pages, generator=g)
        self.table = torch.full((len(lengths), self.width), -1, dtype=torch.int32)      # never looked at behind a sequence's end
        at = 0
        for s, n in enumerate(counts):
            self.table[s, :n] = order[at:at + n].int()
            at += n
        qm = oracle.Q_MAX[dtype]
        self.codes, self.scales = [], []
        for size in (1.0, 0.5):
            c = oracle.nearest(torch.randn(self.pages, kv_heads, page, dim, generator=g, dtype=torch.float64) * (qm / 4), dtype)
            s = (size * 4 / qm * (0.5 + torch.rand(self.pages, kv_heads, generator=g)) * spread ** torch.randn(self.pages, kv_heads, generator=g)).float()
            self.codes.append(c)
            self.scales.append(s)

    def cache(self) -> PagedKVCache:
        """On the GPU; places that hold no token of a sequence get garbage."""
        used = torch.zeros(self.pages, self.page, dtype=torch.bool)
        for s, n in enumerate(self.lengths):
            for b in range(-(-n // self.page)):
                used[self.table[s, b], :min(n - b * self.page, self.page)] = True
        pools = []
        for c in self.codes:
            x = c.to(torch.int8) if self.dtype == "int8" else c.float().to(torch.float8_e4m3fn).view(torch.int8)
            x = torch.where(used[:, None, :, None], x, torch.full_like(x, -128 if self.dtype == "int8" else 127))
            pools.append((x if self.dtype == "int8" else x.view(torch.float8_e4m3fn)).cuda())
        free = ~used.any(1)
        scales = [torch.where(free[:, None], torch.full_like(s, float("nan")), s).cuda() for s in self.scales]
        return PagedKVCache.from_tensors(*pools, *scales)

    def tokens(self, s, side, n=None):
        """f64 [tokens, kv_heads, dim] of sequence s: keys (0) or values (1)."""
        n = self.lengths[s] if n is None else n
        page = self.table[s, :-(-n // self.page)].long()
        x = self.codes[side][page] * self.scales[side][page][..., None, None].double()
        return x.transpose(1, 2).reshape(-1, self.kv_heads, self.dim)[:n]

    def kvt(self, s):
        """Keys, values and the largest value that each token's scale can stand for."""
        page = self.table[s, :-(-self.lengths[s] // self.page)].long()
        top = (self.scales[1][page].double() * oracle.Q_MAX[self.dtype])[:, None].expand(-1, self.page, -1).reshape(-1, self.kv_heads)
        return self.tokens(s, 0), self.tokens(s, 1), top[:self.lengths[s]]


def batch_of(table, before, new, total=None, max_rows=None) -> PagedBatch:
    rows = [0]
    for n in new:
        rows.append(rows[-1] + n)
    as_i32 = lambda x: torch.as_tensor(x, dtype=torch.int32).cuda()      # noqa: E731
    return PagedBatch(as_i32(table), as_i32(before), as_i32(rows), rows[-1] if total is None else total, max(new) if max_rows is None else max_rows)
