"""Plain 64-bit forms of the paged operators (numpy), for the tests."""
import math

import numpy as np


class Pages:
    """The bookkeeping of a paged cache: table, lens, refs and the pools (lists
    over layers of [n_pages, n_kv, page_size, hs] arrays), changed in place."""

    def __init__(self, n_pages, n_seqs, max_pages, page_size, pools=()):
        self.ps = page_size
        self.table = np.full((n_seqs, max_pages), -1, np.int64)
        self.lens = np.zeros(n_seqs, np.int64)
        self.refs = np.zeros(n_pages, np.int64)
        self.pools = list(pools)
        self.max_positions = max_pages * page_size

    def _pages(self, n):
        return -(-n // self.ps)

    def resize(self, seqs, lens):
        """Returns False (nothing changed) without enough free pages."""
        saved = self.table.copy(), self.lens.copy(), self.refs.copy()
        seen, entries, copies = set(), [], []
        for s, n in zip(seqs, lens):
            if s < 0 or s >= len(self.lens) or n < 0 or n > self.max_positions or s in seen:
                continue
            seen.add(s)
            entries.append((s, int(n)))
        for s, n in entries:
            for p in range(self._pages(n), self._pages(self.lens[s])):
                self.refs[self.table[s, p]] -= 1
                self.table[s, p] = -1
        order = []
        held = self.refs.copy()
        for s, n in entries:  # what each entry takes, in order
            old = int(self.lens[s])
            last = self.table[s, old // self.ps] if old % self.ps and n > old else -1
            copy = last >= 0 and held[last] > 1
            if copy:
                held[last] -= 1
            order.append((s, n, old, last if copy else -1))
        free = [p for p in range(len(self.refs)) if self.refs[p] == 0]
        need = sum(max(0, self._pages(n) - self._pages(old)) + (last >= 0) for s, n, old, last in order)
        if need > len(free):
            self.table[:], self.lens[:], self.refs[:] = saved
            return False
        for s, n, old, last in order:
            if last >= 0:
                p = free.pop(0)
                self.refs[last] -= 1
                self.refs[p] = 1
                self.table[s, old // self.ps] = p
                copies.append((last, p, old % self.ps))
            for c in range(self._pages(old), self._pages(n)):
                p = free.pop(0)
                self.refs[p] = 1
                self.table[s, c] = p
            self.lens[s] = n
        for a, b, rows in copies:
            for pool in self.pools:
                pool[b, :, :rows] = pool[a, :, :rows]
        return True

    def fork(self, src, dst):
        table, lens, seen = self.table.copy(), self.lens.copy(), set()
        for s, d in zip(src, dst):
            if s < 0 or d < 0 or s >= len(lens) or d >= len(lens) or d in seen:
                continue
            seen.add(d)
            for p in table[s][table[s] >= 0]:
                self.refs[p] += 1
            for p in table[d][table[d] >= 0]:
                self.refs[p] -= 1
            self.table[d], self.lens[d] = table[s], lens[s]

    def compact(self):
        n = int((self.refs > 0).sum())
        holes = [p for p in range(n) if self.refs[p] == 0]
        movers = [p for p in range(n, len(self.refs)) if self.refs[p] > 0]
        for a, b in zip(movers, holes):
            for pool in self.pools:
                pool[b] = pool[a]
            self.refs[b], self.refs[a] = self.refs[a], 0
            self.table[self.table == a] = b


def frequencies(rot, theta, scaling="none", factor=1.0, original_ctx=4096, beta_fast=32.0, beta_slow=1.0,
                freq_factors=None):
    """Radians per position of each pair, and the factor on cosine and sine."""
    f = np.array([theta ** (-2.0 * m / rot) for m in range(rot // 2)])
    if freq_factors is not None:
        f = f / np.asarray(freq_factors, np.float64)
    if scaling == "linear":
        return f / factor, 1.0
    if scaling == "yarn":
        edge = [rot * math.log(original_ctx / (r * 2 * math.pi)) / (2 * math.log(theta)) for r in (beta_fast, beta_slow)]
        low, high = max(math.floor(edge[0]), 0), min(math.ceil(edge[1]), rot - 1)
        part = np.clip((np.arange(rot // 2) - low) / max(high - low, 1e-3), 0, 1)
        return f / factor * part + f * (1 - part), 0.1 * math.log(max(factor, 1.0)) + 1.0
    return f, 1.0


def rotate(x, pos, f, g, layout):
    """x [rows, heads, hs] rotated at pos [rows]."""
    x = np.array(x, np.float64)
    r = 2 * len(f)
    one, two = (np.arange(r // 2), np.arange(r // 2) + r // 2) if layout == "half" else \
        (2 * np.arange(r // 2), 2 * np.arange(r // 2) + 1)
    a = np.asarray(pos, np.float64)[:, None, None] * f
    c, s = g * np.cos(a), g * np.sin(a)
    u, w = x[..., one], x[..., two]
    x[..., one], x[..., two] = u * c - w * s, u * s + w * c
    return x


def rms(x, w, eps):
    y = np.asarray(x, np.float64)
    y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps)
    return y if w is None else y * np.asarray(w, np.float64)


def visible(pos, window, sinks):
    t = np.arange(pos + 1)
    return t[(t > pos - window) | (t < sinks)] if window else t


def attend(q, k, v, pages, pos, scale, window, sinks):
    """One row: q [heads, hs]; k, v pools; returns (out, bound): bound is how far
    a computation with 32-bit sums may be off (see below)."""
    n_kv, ps, hs = k.shape[1:]
    q = np.asarray(q, np.float64).reshape(n_kv, -1, hs)
    t = visible(pos, window, sinks)
    if pos < 0 or not len(t):
        return np.zeros(q.shape).reshape(-1), np.zeros(q.shape).reshape(-1)
    kk = np.asarray(k[pages[t // ps], :, t % ps], np.float64)
    vv = np.asarray(v[pages[t // ps], :, t % ps], np.float64)
    x = scale * np.einsum("hgd,thd->hgt", q, kk)
    x0 = abs(scale) * np.einsum("hgd,thd->hgt", abs(q), abs(kk))
    p = np.exp(x - x.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    out = np.einsum("hgt,thd->hgd", p, vv)
    # A score is a sum of hs products in steps of 16 (each step rounds, at most 2^-23 of
    # the magnitudes summed), three parts, a factor and the exponential's argument:
    # |dx| <= (hs / 16 + 6) 2^-23 x0 + 2^-22.  Every weight is then off by at most dx, so
    # numerator and denominator by that much of sum p |v|; the sums over t add 2^-23 for
    # each of the tiles that a warp adds, the join of the warps and CTAs 2^-20 at most.
    dx = (hs / 16 + 6) * 2.0 ** -23 * x0.max(-1) + 2.0 ** -22
    mag = np.einsum("hgt,thd->hgd", p, abs(vv))
    bound = mag * (2 * dx[..., None] + (len(t) / 64 + 16) * 2.0 ** -23)
    return out.reshape(-1), bound.reshape(-1)


def beam(logits, scores, beams, finished=None, pad=0):
    """(scores, parents, tokens) by a full sort in 64 bits."""
    rows, vocab = logits.shape
    x = np.asarray(logits, np.float64).copy()
    x[np.isnan(x)] = -np.inf
    out_s, out_p, out_t = [], [], []
    for g in range(rows // beams):
        cand = []
        for b in range(g * beams, (g + 1) * beams):
            if finished is not None and finished[b]:
                cand.append((-float(scores[b]), b, pad))
                continue
            m = x[b].max()
            if m == -np.inf:
                continue
            lse = m + math.log(np.exp(x[b] - m).sum())
            best = np.argsort(-x[b], kind="stable")[:beams]
            cand += [(-(float(scores[b]) + (x[b, t] - lse)), b, int(t)) for t in best if x[b, t] > -np.inf]
        cand = [c for c in cand if c[0] < np.inf]
        cand.sort()
        cand = cand[:beams] + [(np.inf, -1, -1)] * (beams - len(cand[:beams]))
        out_s += [-c[0] for c in cand]
        out_p += [c[1] for c in cand]
        out_t += [c[2] for c in cand]
    return np.array(out_s), np.array(out_p), np.array(out_t)
