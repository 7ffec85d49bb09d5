"""Plain implementations of the paged cache's operators, in 64 bits and one
step after another, that the tests compare the kernels with."""
import math

import numpy as np
import torch


class PlainCache:
    """The book-keeping of jasper_b200.paged.PagedCache on numpy arrays."""

    def __init__(self, cache):
        self.k, self.v = (t.detach().cpu().float().numpy().copy() for t in (cache.k, cache.v))
        self.table, self.lengths, self.refs = (t.cpu().numpy().copy()
                                               for t in (cache.table, cache.lengths, cache.refs))
        self.ps = cache.page_size
        self.status = 0

    def _pages(self, tokens):
        return -(-int(tokens) // self.ps)

    def _free(self):
        return [p for p in range(len(self.refs)) if self.refs[p] == 0]

    def _row(self, r):
        return 0 <= r < len(self.table)

    def extend(self, rows, tokens):
        free, upto, seen = self._free(), 0, set()
        for r, more in zip(rows, tokens):
            if not self._row(r) or r in seen or more < 0:
                self.status |= 2
                continue
            seen.add(r)
            have, want = self._pages(self.lengths[r]), self._pages(self.lengths[r] + more)
            if want > self.table.shape[1]:
                self.status |= 2
                continue
            need = want - have
            upto += need
            if need and upto > len(free):
                self.status |= 1
                continue
            for j in range(need):
                page = free[upto - need + j]
                self.table[r, have + j] = page
                self.refs[page] = 1
            self.lengths[r] += more

    def fork(self, parents, children):
        free, upto, seen = self._free(), 0, set()
        lengths = self.lengths.copy()
        for p, c in zip(parents, children):
            if not self._row(p) or not self._row(c) or c in seen or lengths[c] != 0:
                self.status |= 2
                if self._row(c):
                    seen.add(c)
                continue
            seen.add(c)
            n = int(lengths[p])
            whole, part = n // self.ps, n % self.ps
            last = int(self.table[p, whole]) if part else -1
            if last >= 0:
                upto += 1
                if upto > len(free):
                    self.status |= 1
                    continue
            for j in range(whole):
                self.table[c, j] = self.table[p, j]
                if self.table[p, j] >= 0:
                    self.refs[self.table[p, j]] += 1
            if part:
                self.table[c, whole] = -1
                if last >= 0:
                    page = free[upto - 1]
                    self.table[c, whole] = page
                    self.refs[page] = 1
                    for t in (self.k, self.v):
                        t[:, page, :part] = t[:, last, :part]
            self.lengths[c] = n

    def free(self, rows):
        for r in rows:
            if not self._row(r):
                self.status |= 2
                continue
            for page in self.table[r]:
                if page >= 0:
                    self.refs[page] -= 1
            self.table[r] = -1
            self.lengths[r] = 0

    def adopt(self, rows, pages, lengths=None):
        seen = set()
        for i, r in enumerate(rows):
            n = pages.shape[1] * self.ps if lengths is None else int(lengths[i])
            bad = not self._row(r) or r in seen or self.lengths[r] != 0 or n < 0
            if self._row(r):
                seen.add(r)
            if bad or self._pages(n) > pages.shape[1]:
                self.status |= 2
                continue
            for j in range(self._pages(n)):
                page = int(pages[i, j])
                if not 0 <= page < len(self.refs):
                    if page != -1:
                        self.status |= 4
                    page = -1
                else:
                    self.refs[page] += 1
                self.table[r, j] = page
            self.lengths[r] = n

    def compact(self):
        live = [p for p in range(len(self.refs)) if self.refs[p] > 0]
        holes = [p for p in range(len(live)) if self.refs[p] == 0]
        remap = np.full(len(self.refs), -1, np.int32)
        remap[live] = live
        for page, hole in zip([p for p in live if p >= len(live)], holes):
            remap[page] = hole
            for t in (self.k, self.v):
                t[:, hole] = t[:, page]
            self.refs[hole], self.refs[page] = self.refs[page], 0
        held = self.table >= 0
        self.table[held] = remap[self.table[held]]
        return remap

    def copy_pages(self, src, dst):
        for s, d in zip(src, dst):
            if not (0 <= s < len(self.refs) and 0 <= d < len(self.refs)):
                self.status |= 4
                continue
            for t in (self.k, self.v):
                t[:, d] = t[:, s]

    def check_against(self, cache):
        """The device cache equals this one, bit for bit."""
        for name in ("table", "lengths", "refs"):
            np.testing.assert_array_equal(getattr(cache, name).cpu().numpy(), getattr(self, name), err_msg=name)
        for name in ("k", "v"):
            np.testing.assert_array_equal(getattr(cache, name).detach().cpu().float().numpy(),
                                          getattr(self, name), err_msg=name)
        assert int(cache.status.item()) == self.status


def turned(x, positions, theta, rot, layout, scale=1.0, sign=1):
    """Rotary positions in 64 bits: x [tokens, heads, dim], positions int64."""
    x = x.detach().cpu().double()
    y = x.clone()
    half = rot // 2
    a, b = (slice(0, half), slice(half, rot)) if layout == "half" else (slice(0, rot, 2), slice(1, rot, 2))
    angle = sign * positions.cpu().double()[:, None, None] * torch.tensor(theta, dtype=torch.float64)
    c, s = scale * torch.cos(angle), scale * torch.sin(angle)
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    return y


def attention(q, k, v, pages, length, page_size, scale, window=0, mask=None):
    """One row's attention in 64 bits.  q [heads, dim]; k, v [pages,
    page_size, kv_heads, dim]; pages: the row's table.  Returns out, lse, the
    sum of p |v| and the largest scale * sum |q k| (for error bounds)."""
    heads, dim = q.shape
    kvh = k.shape[2]
    seen = [t for t in range(max(0, length - window) if window else 0, length)
            if pages[t // page_size] >= 0 and (mask is None or t >= len(mask) or mask[t])]
    out = torch.zeros(heads, dim, dtype=torch.float64)
    lse = torch.full((heads,), -math.inf, dtype=torch.float64)
    weight, reach = torch.zeros(heads, dim, dtype=torch.float64), 0.0
    if seen:
        t = torch.tensor(seen)
        page = torch.as_tensor(pages)[t // page_size].long()
        keys, values = k[page, t % page_size].double(), v[page, t % page_size].double()
        for h in range(heads):
            kh, vh = keys[:, h * kvh // heads], values[:, h * kvh // heads]
            s = scale * (kh @ q[h].double())
            p = torch.softmax(s, 0)
            out[h], lse[h] = p @ vh, torch.logsumexp(s, 0)
            weight[h] = p @ vh.abs()
            reach = max(reach, abs(scale) * float((kh.abs() @ q[h].double().abs()).max()))
    return out, lse, weight, reach
