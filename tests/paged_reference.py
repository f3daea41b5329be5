"""Plain 64-bit restatements of the paged cache's operators, on the CPU, and a host model of its page bookkeeping."""
import math

import torch


def rope_rows(x, pos, inv_freq, factor, interleaved):
    """x [T, heads, D] float64 at positions [T]."""
    r = 2 * inv_freq.numel()
    ang = pos.double()[:, None] * inv_freq.double()[None]
    c, s = (ang.cos() * factor)[:, None], (ang.sin() * factor)[:, None]
    y = x.clone()
    if interleaved:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        y[..., 0:r:2], y[..., 1:r:2] = a * c - b * s, b * c + a * s
    else:
        a, b = x[..., : r // 2], x[..., r // 2: r]
        y[..., : r // 2], y[..., r // 2: r] = a * c - b * s, b * c + a * s
    return y


def norm_rows(x, w, eps):
    return x if w is None else x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()


def attend(q, keys, values, seen, start, lens, causal, window, sinks, scale):
    """q [B, T, H, D]; keys / values: per row [KV, n, D] float64; seen: per row bool [n], keys that have a page."""
    B, T, H, D = q.shape
    out = torch.zeros(B, T, H, D, dtype=torch.float64)
    for b in range(B):
        k, v = keys[b].double(), values[b].double()
        group = H // k.shape[0]
        n = k.shape[1]
        j = torch.arange(n)
        for t in range(min(int(lens[b]), T)):
            p = int(start[b]) + t
            vis = seen[b] & (j < int(start[b]) + min(int(lens[b]), T))
            if causal:
                vis = vis & (j <= p)
            if window:
                vis = vis & ((p - j < window) | (j < sinks))
            idx = vis.nonzero()[:, 0]
            if not idx.numel():
                continue
            for h in range(H):
                s = (k[h // group, idx] @ q[b, t, h].double()) * scale
                out[b, t, h] = torch.softmax(s, 0) @ v[h // group, idx]
    return out


class HostPages:
    """The bookkeeping of PagedKVCache in Python lists: what each call must leave behind."""

    def __init__(self, batch, pages, page_size, row_pages):
        self.page, self.pages, self.row_pages = page_size, pages, row_pages
        self.table = [[-1] * row_pages for _ in range(batch)]
        self.length = [0] * batch
        self.refs = [0] * pages
        self.content = list(range(-pages, 0))  # an identity per page, to follow copies

    def _free(self):
        return [p for p in range(self.pages) if self.refs[p] == 0]

    def reserve(self, upto):
        B = len(self.table)
        cap = self.row_pages * self.page
        want = []
        held = [-1] * B
        for b in range(B):
            up = min(upto[b], cap)
            if up <= self.length[b]:
                continue
            held[b] = self.table[b][self.length[b] // self.page]
        for b in range(B):
            up = min(upto[b], cap)
            if up <= self.length[b]:
                continue
            first = self.length[b] // self.page
            p = held[b]
            if p >= 0 and self.refs[p] > 1:
                rank = sum(held[x] == p for x in range(b))
                if rank > 0 or self.refs[p] > held.count(p):
                    want.append((b, first, p))
            want += [(b, i, -1) for i in range(first, math.ceil(up / self.page)) if self.table[b][i] < 0]
        free = self._free()
        for (b, i, old), new in zip(want, free):
            if old >= 0:
                self.refs[old] -= 1
                self.content[new] = self.content[old]
            self.table[b][i] = new
            self.refs[new] = 1
        return len(want) <= len(free) and all(u <= cap for u in upto)

    def crop(self, to):
        for b, n in enumerate(to):
            self.length[b] = min(max(n, 0), self.length[b])
            for i in range(-(-self.length[b] // self.page), self.row_pages):
                if self.table[b][i] >= 0:
                    self.refs[self.table[b][i]] -= 1
                self.table[b][i] = -1

    def fork(self, src):
        old = [list(r) for r in self.table]
        length = list(self.length)
        for b, s in enumerate(src):
            if s == b or s < -1 or s >= len(src):
                continue
            n = length[s] if s >= 0 else 0
            new = [old[s][i] if i * self.page < n else -1 for i in range(self.row_pages)]
            for p in new:
                if p >= 0:
                    self.refs[p] += 1
            for p in old[b]:
                if p >= 0:
                    self.refs[p] -= 1
            self.table[b], self.length[b] = new, n

    def compact(self):
        used = sum(r > 0 for r in self.refs)
        move = dict(zip([p for p in range(used, self.pages) if self.refs[p] > 0],
                        [p for p in range(used) if self.refs[p] == 0]))
        for a, d in move.items():
            self.refs[d], self.refs[a] = self.refs[a], 0
            self.content[d] = self.content[a]
        self.table = [[move.get(p, p) for p in r] for r in self.table]
