"""Drafted trees and page pools in 64 bits, one thing after the other: who sees whom, rotation at positions of several axes, kept rows, forks and moves of pages."""
from __future__ import annotations

import math

import torch

from . import paged


def lines(parents: list[int]) -> list[list[int]]:
    """Of each token those that it sees: itself and the ones that it comes behind.  A parent that is not a token in front of it, nor -1, counts as -1."""
    out: list[list[int]] = []
    for i, p in enumerate(parents):
        out.append((out[p] if 0 <= p < i else []) + [i])
    return out


def depths(parents: list[int]) -> list[int]:
    return [len(x) - 1 for x in lines(parents)]


def visible(parents: list[int], before: int, window: int = 0, sinks: int = 0) -> torch.Tensor:
    """bool [rows, before + rows]."""
    n, d = len(parents), torch.tensor(depths(parents), dtype=torch.int64)
    seen = torch.zeros(n, before + n, dtype=torch.bool)
    seen[:, :before] = True
    for i, line in enumerate(lines(parents)):
        seen[i, [before + j for j in line]] = True
    key = torch.cat((torch.arange(before), before + d))
    return seen & (((before + d)[:, None] - key < window) | (key < sinks)) if window else seen


def attend(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, top: torch.Tensor, seen: torch.Tensor, scale: float) -> tuple[torch.Tensor, torch.Tensor]:
    """As ``paged.attend``, for any mask [rows, tokens]: the result, and how far from it weights in f16, 32-bit sums and a result in bf16 may be (derived there)."""
    rows, heads, _ = q.shape
    out, tol = torch.zeros_like(q), torch.zeros_like(q)
    for h in range(heads):
        kv = h * k.shape[1] // heads
        s = (q[:, h] @ k[:, kv].T * scale).masked_fill(~seen, -math.inf)
        size = (q[:, h].abs() @ k[:, kv].abs().T * scale).masked_fill(~seen, 0).amax(1, keepdim=True)
        w = torch.softmax(s, 1)
        out[:, h] = w @ v[:, kv]
        dropped = 2.0 ** -32 * k.shape[0] * (w * top[:, kv]).amax(1, keepdim=True)
        tol[:, h] = 2.0 ** -8 * out[:, h].abs() + (2.0 ** -11 + 2.0 ** -17 * (1 + size)) * (w @ v[:, kv].abs()) + dropped
    return out, tol


def rotated(x: torch.Tensor, positions: torch.Tensor, axes: list[int], rot_dims: int, base: float = 10000.0, pairing: str = "adjacent") -> torch.Tensor:
    """x f64 [rows, heads, dim], positions [axes, rows]: pair j is turned by positions[axes[j]]."""
    out = x.clone()
    for j, a in enumerate(axes):
        angle = positions[a].double() * base ** (-2 * j / rot_dims)
        cos, sin = angle.cos()[:, None], angle.sin()[:, None]
        i0, i1 = (2 * j, 2 * j + 1) if pairing == "adjacent" else (j, j + rot_dims // 2)
        out[..., i0], out[..., i1] = x[..., i0] * cos - x[..., i1] * sin, x[..., i0] * sin + x[..., i1] * cos
    return out


def keep(path: list[int], before: int, page_tokens: int, codes: list[torch.Tensor], scales: list[float], dtype: str):
    """One sequence, head and side: codes [blocks] of f64 [page_tokens, dim], scales [blocks] -> what they are afterwards, and of each kept row the value that it had, its block, its place and whether it came from
    another page.  Everything is read before anything is written."""
    new_codes, new_scales, rows = [c.clone() for c in codes], list(scales), []
    qm = paged.Q_MAX[dtype]
    for block in range(len(codes)):
        mine = [(before + i, before + a) for i, a in enumerate(path) if (before + i) // page_tokens == block]
        if not mine or all(a == b for a, b in mine):
            rows += [(codes[block][a % page_tokens] * scales[block], block, a % page_tokens, False) for a, _ in mine]
            continue
        older = max(0, before - block * page_tokens)
        far = [b for _, b in mine if b // page_tokens != block]
        s, doublings = scales[block], 0
        if far:
            top = max(float(codes[b // page_tokens][b % page_tokens].abs().max()) * scales[b // page_tokens] for b in far)
            if (older or len(far) < len(mine)) and s > 0:
                while s * qm < top:
                    s, doublings = 2 * s, doublings + 1
            else:
                s = max(top / qm, paged.SCALE_MIN) if top > 0 else 0.0
                new_codes[block][:older] = 0
        if scales[block] > 0 or not far:
            new_codes[block][:older] = paged.nearest(codes[block][:older] * 2.0 ** -doublings, dtype)
        for to, src in mine:
            b, slot = src // page_tokens, src % page_tokens
            value = codes[b][slot] * scales[b]
            if b == block:
                new = paged.nearest(codes[b][slot] * 2.0 ** -doublings, dtype) if scales[block] > 0 or not far else torch.zeros_like(codes[b][slot])
            else:
                new = paged.nearest(value / s, dtype) if s > 0 else torch.zeros_like(value)
            new_codes[block][to % page_tokens] = new
            rows.append((value, block, to % page_tokens, b != block))
        new_scales[block] = s
    return new_codes, new_scales, rows


class Pool:
    """A pool's tables with lists; the calls give the copies that the caches have to make, (from, to) in order."""

    def __init__(self, pages: int, page_tokens: int, sequences: int, width: int):
        self.page_tokens, self.width = page_tokens, width
        self.table: list[list[int]] = [[] for _ in range(sequences)]
        self.lengths, self.refs = [0] * sequences, [0] * pages

    def _blocks(self, tokens: int) -> int:
        return -(-tokens // self.page_tokens)

    def rearrange(self, source: list[int]) -> None:
        n = len(source)
        source = [s if -1 <= s < n else i for i, s in enumerate(source)]
        # one whose length is not one that its pages can have counts as empty
        table, lengths = self.table, [x if 0 <= x <= len(t) * self.page_tokens else 0 for x, t in zip(self.lengths, self.table)]
        self.table = [list(table[s][:self._blocks(lengths[s])]) if s >= 0 else [] for s in source]
        self.lengths = [lengths[s] if s >= 0 else 0 for s in source]
        self.refs = [0] * len(self.refs)
        for t in self.table:
            for p in t:
                self.refs[p] += 1

    def reserve(self, add: list[int]) -> list[tuple[int, int]] | None:
        """None: there are too few pages, and nothing has changed."""
        table, refs, moves = [list(t) for t in self.table], list(self.refs), []
        free = [p for p, r in enumerate(refs) if r == 0]
        for s, a in enumerate(add):
            n = self.lengths[s]
            if a <= 0 or n + a > self.width * self.page_tokens:
                continue
            block = n // self.page_tokens
            if self._blocks(n) < len(table[s]) and self.refs[table[s][self._blocks(n)]] > 1:      # shorter than it was, and not rearranged since: left out
                continue
            if n % self.page_tokens and refs[table[s][block]] > 1:
                if not free:
                    return None
                old, new = table[s][block], free.pop(0)
                refs[old], refs[new], table[s][block] = refs[old] - 1, 1, new
                moves.append((old, new))
            while len(table[s]) < self._blocks(n + a):
                if not free:
                    return None
                refs[free[0]] = 1
                table[s].append(free.pop(0))
        self.table, self.refs = table, refs
        return moves

    def compact(self) -> list[tuple[int, int]]:
        end = sum(r > 0 for r in self.refs)
        moves = list(zip([p for p in range(end, len(self.refs)) if self.refs[p] > 0], [p for p in range(end) if self.refs[p] == 0]))
        to = dict(moves)
        self.table = [[to.get(p, p) for p in t] for t in self.table]
        for a, b in moves:
            self.refs[b], self.refs[a] = self.refs[a], 0
        return moves
