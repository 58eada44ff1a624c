"""Plain restatements of the paged cache for the tests: the bookkeeping one page at a time, attention and rotary embedding in 64 bits."""
import math

import torch

D = 128


class Model:
    """Who holds what, and what the pages hold (`pool`, a CPU tensor with the same layout as the cache's)."""

    def __init__(self, pages, page, max_seqs, max_pages, pool):
        self.page, self.width = page, max_pages
        self.table = [[-1] * max_pages for _ in range(max_seqs)]
        self.lengths, self.refs, self.status = [0] * max_seqs, [0] * pages, 0
        self.pool = pool

    def need(self, tokens):
        return -(-tokens // self.page)

    def _free(self, but=()):
        return [p for p, r in enumerate(self.refs) if r == 0 and p not in but]

    def _drop(self, s):
        for p in self.table[s]:
            if p >= 0:
                self.refs[p] -= 1
        self.table[s], self.lengths[s] = [-1] * self.width, 0

    def _bad(self, slots):
        return len(set(slots)) < len(slots) or any(not 0 <= s < len(self.table) for s in slots)

    def reserve(self, slots, tokens, tps):
        pos = [-1] * (len(slots) * tps)
        if self._bad(slots) or min(tokens) < 0:
            self.status |= 4
            return pos
        if any(self.need(self.lengths[s] + t) > self.width for s, t in zip(slots, tokens)):
            self.status |= 2
            return pos
        want = [(s, k) for s, t in zip(slots, tokens) for k in range(self.need(self.lengths[s]), self.need(self.lengths[s] + t))]
        free = self._free()
        if len(free) < len(want):
            self.status |= 1
            return pos
        for (s, k), p in zip(want, free):
            self.table[s][k], self.refs[p] = p, 1
        for i, (s, t) in enumerate(zip(slots, tokens)):
            for j in range(min(t, tps)):
                pos[i * tps + j] = self.lengths[s] + j
            self.lengths[s] += t
        return pos

    def free(self, slots):
        if self._bad(slots):
            self.status |= 4
            return
        for s in slots:
            self._drop(s)

    def fork(self, src, dst, share=True):
        if self._bad(dst) or any(not 0 <= s < len(self.table) for s in src):
            self.status |= 4
            return
        was = ([list(r) for r in self.table], list(self.lengths), list(self.refs))
        old, length = was[0], was[1]
        pairs = [(a, b) for a, b in zip(src, dst) if a != b]
        full = {a: length[a] // self.page if share else 0 for a, _ in pairs}
        for _, b in pairs:
            self._drop(b)
        for a, b in pairs:
            for k in range(full[a]):
                self.table[b][k] = old[a][k]
                self.refs[old[a][k]] += 1
        want = [(a, b, k) for a, b in pairs for k in range(full[a], self.need(length[a]))]
        free = self._free(but={old[a][k] for a, _, k in want})
        if len(free) < len(want):
            self.table, self.lengths, self.refs = was
            self.status |= 1
            return
        before = self.pool.clone()
        for (a, b, k), p in zip(want, free):
            self.table[b][k], self.refs[p] = p, 1
            rows = min(self.page, length[a] - k * self.page)
            self.pool[:, :, p, :, :rows] = before[:, :, old[a][k], :, :rows]
        for a, b in pairs:
            self.lengths[b] = length[a]

    def compact(self):
        n = sum(r > 0 for r in self.refs)
        to = dict(zip([p for p in range(n, len(self.refs)) if self.refs[p] > 0], [p for p in range(n) if self.refs[p] == 0]))
        for a, b in to.items():
            self.pool[:, :, b] = self.pool[:, :, a]
            self.refs[b], self.refs[a] = self.refs[a], 0
        self.table = [[to.get(p, p) for p in row] for row in self.table]

    def common(self, slots):
        if len(slots) < 2:
            return 0
        k = 0
        while all(k < self.lengths[s] // self.page and self.table[s][k] == self.table[slots[0]][k] for s in slots):
            k += 1
        return k * self.page


def rope(x, positions, inv_freq):
    """x [tokens, heads, D] -> the same rotated, 64 bits."""
    ang = positions.double()[:, None, None] * inv_freq.double()
    a, b = x.double()[..., :D // 2], x.double()[..., D // 2:]
    return torch.cat((a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin()), -1)


def attention(cache, layer, q, positions, slots, n_heads, scale=None):
    """(output, sum of weights times |v|), 64 bits, [tokens, n_heads * D]."""
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    n_kv, T = cache.n_kv, q.shape[0]
    R, tps = n_heads // n_kv, T // len(slots)
    out = torch.zeros((T, n_heads, D), dtype=torch.float64, device=q.device)
    mag = torch.zeros_like(out)
    pos = positions.tolist()
    for i, s in enumerate(slots):
        keys = max(pos[i * tps:(i + 1) * tps]) + 1
        if keys <= 0:
            continue
        pages = cache.table[s, :-(-keys // cache.page_size)].long()
        k, v = (cache.pool[layer, w, pages].permute(1, 0, 2, 3).reshape(n_kv, -1, D)[:, :keys].double() for w in (0, 1))
        x = q[i * tps:(i + 1) * tps].double().view(tps, n_kv, R, D).permute(1, 2, 0, 3).reshape(n_kv, R * tps, D)
        lim = positions[i * tps:(i + 1) * tps].long().repeat(R)[None, :, None]
        sc = (x @ k.transpose(1, 2) * scale).masked_fill(torch.arange(keys, device=q.device) > lim, float("-inf"))
        p = torch.where(lim >= 0, torch.softmax(sc, -1), torch.zeros_like(sc))
        seen = torch.where(torch.arange(keys, device=q.device) > lim, torch.zeros_like(sc), torch.ones_like(sc)) > 0
        o, a = p @ torch.nan_to_num(v, 0.0, 0.0, 0.0), p @ torch.nan_to_num(v, 0.0, 0.0, 0.0).abs()
        if not torch.isfinite(v).all():                        # values that are not finite, for the rows that see them
            for kv, key, d in (~torch.isfinite(v)).nonzero().tolist():
                o[kv, seen[kv if seen.shape[0] > 1 else 0, :, key], d] += v[kv, key, d]
        back = lambda y: y.view(n_kv, R, tps, D).permute(2, 0, 1, 3).reshape(tps, n_heads, D)      # noqa: E731
        out[i * tps:(i + 1) * tps], mag[i * tps:(i + 1) * tps] = back(o), back(a)
    return out.view(T, -1), mag.view(T, -1)
