"""Shared plumbing of the drafted-decoding tests: plain 64-bit oracles on the CPU."""
from __future__ import annotations

import math

import numpy as np
import torch


def ancestors(parents, nodes):
    """Per node the drafted nodes it sees: itself and its ancestors; a parent below -1 sees none."""
    seen = []
    for n in range(nodes):
        p = parents[n]
        if p < -1 or p >= n:
            seen.append([])
        else:
            line, a = [n], p
            while a >= 0 and seen[a]:
                line.append(a)
                a = parents[a]
            seen.append(sorted(line))
    return seen


def attention(query, keys, values, length, parents, nodes, group, scale):
    """One sequence: query [nodes][heads][D], keys / values [length + nodes][kv_heads][D], float64.
    Returns out, lse and the per-element weight sum_k p_k |v_k| that a rounding of p is relative to."""
    heads, dim = query.shape[1:]
    out = torch.zeros((nodes, heads, dim), dtype=torch.float64)
    size = torch.zeros_like(out)
    lse = torch.full((nodes, heads), -math.inf, dtype=torch.float64)
    for n, seen in enumerate(ancestors(parents, nodes)):
        at = list(range(length)) + [length + a for a in seen]
        if not at:
            continue
        for h in range(heads):
            k, v = keys[at, h // group], values[at, h // group]
            z = (k @ query[n, h]) * scale
            lse[n, h] = torch.logsumexp(z, 0)
            p = torch.softmax(z, 0)
            out[n, h] = p @ v
            size[n, h] = p @ v.abs()
    return out, lse, size


def verify(target, tokens, parents, coins, draw, draft, nodes):
    """One sequence in float64: (accepted path, next token)."""
    if nodes <= 0:
        return [], -1
    vocab = target.shape[1]
    path, node = [0], 0
    w, rejected, left = target[0].copy(), [], 1.0
    for n in range(1, nodes):
        if parents[n] != node:
            continue
        x = tokens[n]
        known = 0 <= x < vocab
        if draft is None:
            p = target[node, x] if known and x not in rejected else 0.0
            ok = coins[n] * left < p
        else:
            p = w[x] if known else 0.0
            ok = coins[n] * (draft[node, x] if known else 0.0) < p
        if ok:
            path.append(n)
            node, w, rejected, left = n, target[n].copy(), [], 1.0
        elif draft is None:
            rejected.append(x)
            left -= p
        else:
            r = w - draft[node]
            r = np.where(r > 0, r, np.where(r <= 0, 0.0, r))
            if math.isnan(r.sum()) or math.isinf(r.sum()):
                return path, -1
            if r.sum() > 0:
                w = r / r.sum()
    if draft is None:
        full = w.copy()
        for x in rejected:
            if 0 <= x < vocab:
                w[x] = 0.0
        w = full if w.sum() == 0 and rejected else w
    total = w.sum()
    if not (total > 0 and math.isfinite(total)):
        return path, -1
    above = np.nonzero(np.cumsum(w) > draw * total)[0]
    return path, int(above[0]) if len(above) else int(np.nonzero(w > 0)[0][-1])


class Book:
    """The page bookkeeping of include/tsac_cuda.h in lists; `rows` maps (page, slot) to a row's value."""

    def __init__(self, pages, page_size, sequences):
        self.size, self.refs = page_size, [0] * pages
        self.held = [[] for _ in range(sequences)]
        self.lengths = [0] * sequences
        self.rows = {}

    def reserve(self, entries):
        """entries: (sequence, positions).  False, and nothing changed, without enough free pages."""
        refs, held, copies, taken = list(self.refs), [list(h) for h in self.held], [], []
        free = [p for p, r in enumerate(self.refs) if r == 0]
        for s, more in entries:
            if more <= 0:
                continue
            first, last = self.lengths[s] // self.size, (self.lengths[s] + more - 1) // self.size
            for j in range(first, last + 1):
                if j < len(held[s]) and refs[held[s][j]] == 1:
                    continue
                if not free:
                    return False
                page = free.pop(0)
                taken.append(page)
                if j < len(held[s]):
                    copies.append((held[s][j], page))
                    refs[held[s][j]] -= 1
                    held[s][j] = page
                else:
                    held[s].append(page)
        for page in taken:
            refs[page] = 1
        old = dict(self.rows)
        for a, b in copies:
            for slot in range(self.size):
                if (a, slot) in old:
                    self.rows[(b, slot)] = old[(a, slot)]
        self.refs, self.held = refs, held
        return True

    def at(self, s, position):
        return self.held[s][position // self.size], position % self.size

    def append(self, s, values):
        for n, v in enumerate(values):
            self.rows[self.at(s, self.lengths[s] + n)] = v

    def keep(self, s, path, start=None):
        start = self.lengths[s] if start is None else start
        kept = [self.rows[self.at(s, start + n)] for n in path]
        for j, v in enumerate(kept):
            self.rows[self.at(s, start + j)] = v
        self.lengths[s] = start + len(path)

    def fork(self, parent, child):
        self.lengths[child] = self.lengths[parent]
        self.held[child] = list(self.held[parent][:-(-self.lengths[parent] // self.size)])
        for p in self.held[child]:
            self.refs[p] += 1

    def release(self, s, positions=0):
        stay = -(-positions // self.size)
        for p in self.held[s][stay:]:
            self.refs[p] -= 1
        self.held[s] = self.held[s][:stay]
        self.lengths[s] = min(self.lengths[s], positions)

    def compact(self):
        live = sum(r > 0 for r in self.refs)
        holes = [p for p in range(live) if self.refs[p] == 0]
        to = {p: p if p < live else holes.pop(0) for p, r in enumerate(self.refs) if r > 0}
        refs = [0] * len(self.refs)
        rows = {}
        for p, q in to.items():
            refs[q] = self.refs[p]
            rows.update({(q, slot): self.rows[(p, slot)] for slot in range(self.size) if (p, slot) in self.rows})
        self.refs, self.rows = refs, rows
        self.held = [[to[p] for p in h] for h in self.held]
        return live
