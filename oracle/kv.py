"""CPU restatement of the paged key/value cache's operators, in 64 bits and one entry at a time (test infrastructure).

`Pages` keeps the integer state and the pools as numpy arrays and applies free, fork, extend, compact and copy by their
definitions; `append` and `attention` compute rows in float64 from tensors."""
from __future__ import annotations

import numpy as np
import torch

MAX_LEN = 2**31 - 1


class Pages:
    def __init__(self, table, lens, refs, pools, page):
        self.table, self.lens, self.refs = table.copy(), lens.copy(), refs.copy()
        self.pools = [p.copy() for p in pools]              # [layers, pages, ...] each
        self.page = page

    def _held(self, s):
        if not 0 <= s < len(self.lens):
            return None
        return int(min(max(int(self.lens[s]), 0), self.table.shape[1] * self.page))

    def _pages(self, n):
        return -(-n // self.page)

    def _is_page(self, p):
        return 0 <= p < len(self.refs)

    def free(self, seqs):
        for s in seqs:
            n = self._held(s)
            if n is None:
                continue
            self.lens[s] = 0
            for j in range(self._pages(n)):
                p = self.table[s, j]
                self.table[s, j] = -1
                if self._is_page(p):
                    self.refs[p] -= 1

    def fork(self, parents, children):
        before, taken = self.lens.copy(), set()
        for par, ch in zip(parents, children):
            if not 0 <= ch < len(before) or before[ch] > 0 or not 0 <= par < len(before) or before[par] <= 0 or ch in taken:
                continue
            taken.add(ch)
            n = self._held(par)
            for j in range(self._pages(n)):
                p = self.table[par, j]
                self.table[ch, j] = p
                if self._is_page(p):
                    self.refs[p] += 1
            self.lens[ch] = n

    def extend(self, seqs, tokens):
        """Returns (copied, missing, refused)."""
        free = [p for p in range(len(self.refs)) if self.refs[p] == 0]
        table, lens, refs = self.table.copy(), self.lens.copy(), self.refs.copy()
        seen, copies, refused, need = set(), [], 0, 0
        for s, t in zip(seqs, tokens):
            n = self._held(s)
            if n is None or s in seen:
                continue
            seen.add(s)
            t = max(int(t), 0)
            if self._pages(n + t) > table.shape[1] or n + t > MAX_LEN:
                refused += 1
                continue
            had = self._pages(n)
            tail = self.table[s, had - 1] if t > 0 and n % self.page else -1
            if self._is_page(tail) and refs[tail] > 1:
                if need < len(free):
                    copies.append((tail, free[need]))
                    table[s, had - 1] = free[need]
                    refs[free[need]] = 1
                refs[tail] -= 1
                need += 1
            for j in range(had, self._pages(n + t)):
                if need < len(free):
                    table[s, j] = free[need]
                    refs[free[need]] = 1
                need += 1
            lens[s] = n + t
        if refused:
            return 0, 0, refused
        if need > len(free):
            return 0, min(need, len(refs) + 1) - len(free), 0
        self.table, self.lens, self.refs = table, lens, refs
        for a, b in copies:
            for pool in self.pools:
                pool[:, b] = pool[:, a]
        return len(copies), 0, 0

    def compact(self):
        """Returns (moved, live)."""
        live = int((self.refs > 0).sum())
        holes = [p for p in range(live) if self.refs[p] <= 0]
        movers = [p for p in range(live, len(self.refs)) if self.refs[p] > 0]
        to = dict(zip(movers, holes))
        for a, b in to.items():
            self.refs[b], self.refs[a] = self.refs[a], 0
            for pool in self.pools:
                pool[:, b] = pool[:, a]
        for s in range(len(self.lens)):
            for j in range(self._pages(self._held(s))):
                self.table[s, j] = to.get(int(self.table[s, j]), self.table[s, j])
        return len(movers), live

    def copy(self, src, dst):
        for a, b in zip(src, dst):
            if self._is_page(a) and self._is_page(b) and a != b:
                for pool in self.pools:
                    pool[:, b] = pool[:, a]


def gather(pool, row, n, page):
    """[positions, kv_heads, head_dim] of one layer's pool [pages, kv_heads, page, head_dim]; and which positions have a page."""
    ids = torch.as_tensor(row[: -(-n // page)]).long()
    there = (ids >= 0) & (ids < pool.shape[0])
    got = pool[ids.clamp(0, pool.shape[0] - 1).to(pool.device)].transpose(1, 2).reshape(-1, pool.shape[1], pool.shape[3])[:n]
    return got, there.repeat_interleave(page)[:n].to(pool.device)


def attention(q, k, v, table, lens, seqs, starts, scale):
    """(out, |v| averaged with the same weights, largest sum of |q||k| scale) in float64; rows of no sequence are NaN."""
    rows, heads, dim = q.shape
    out = torch.full((rows, heads, dim), float("nan"), dtype=torch.float64, device=q.device)
    size, big = out.clone(), 0.0
    group = heads // k.shape[1]
    for i, s in enumerate(seqs):
        a, b = starts[i], starts[i + 1]
        if not 0 <= s < len(lens) or b <= a:
            continue
        n, t = max(int(lens[s]), 0), b - a
        out[a:b] = size[a:b] = 0.0
        if n == 0:
            continue
        kk, there = gather(k, table[s], n, k.shape[2])
        vv, _ = gather(v, table[s], n, k.shape[2])
        pos = torch.arange(n, device=q.device)
        for j in range(t):
            see = there & (pos < n - t + j + 1)
            if not bool(see.any()):
                continue
            ks, vs = kk[see].double().repeat_interleave(group, 1), vv[see].double().repeat_interleave(group, 1)
            x = torch.einsum("hd,nhd->hn", q[a + j].double(), ks) * scale
            big = max(big, float((torch.einsum("hd,nhd->hn", q[a + j].double().abs(), ks.abs()) * abs(scale)).max()))
            w = torch.softmax(x, dim=-1)
            out[a + j] = torch.einsum("hn,nhd->hd", w, vs)
            size[a + j] = torch.einsum("hn,nhd->hd", w, vs.abs())
    return out, size, big


def append(qkv, q_heads, kv_heads, pos, q_weight, k_weight, eps, inv_freq, interleaved):
    """(queries, keys, values, and for queries and keys |a| + |b| of each turned pair) in float64 for rows at `pos`."""
    rows = qkv.shape[0]
    dim = qkv.shape[1] // (q_heads + 2 * kv_heads)
    x = qkv.double().view(rows, -1, dim)
    out = []
    for y, w in ((x[:, :q_heads], q_weight), (x[:, q_heads:q_heads + kv_heads], k_weight)):
        if w is not None:
            y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * w.double()
        z, both = y.clone(), y.abs()
        if inv_freq is not None:
            h = inv_freq.numel()
            angle = pos.double()[:, None] * inv_freq
            c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
            ia = torch.arange(h, device=y.device) * 2 if interleaved else torch.arange(h, device=y.device)
            ib = ia + 1 if interleaved else ia + h
            a, b = y[..., ia], y[..., ib]
            z[..., ia], z[..., ib] = a * c - b * s, b * c + a * s
            both[..., ia] = both[..., ib] = a.abs() + b.abs()
        out += [z, both]
    return out[0], out[2], x[:, q_heads + kv_heads:], out[1], out[3]
