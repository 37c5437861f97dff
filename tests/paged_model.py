"""A cache in pages in plain Python and 64 bits: what the tests of the paged calls compare with."""
import numpy as np


def pages_of(rows, page_rows):
    return -(-rows // page_rows)


class Pages:
    """Lengths, table and stack of free pages, one entry and one page at a time."""

    def __init__(self, n_pages, page_rows, n_seqs, seq_pages):
        self.P, self.seq_pages = page_rows, seq_pages
        self.free = list(range(n_pages - 1, -1, -1))
        self.held = [[] for _ in range(n_seqs)]
        self.lens = [0] * n_seqs

    def map(self, entries, max_rows):
        """entries: [(sequence, change)].  The rows gained as (slot, position, sequence), or None where nothing was changed."""
        new = {}
        for s, d in entries:
            if not 0 <= s < len(self.lens) or s in new or self.lens[s] + d < 0 or self.lens[s] + d > self.seq_pages * self.P:
                return None
            new[s] = self.lens[s] + d
        need = sum(pages_of(n, self.P) - len(self.held[s]) for s, n in new.items())
        if need > len(self.free) or sum(max(0, d) for _, d in entries) > max_rows:
            return None
        for s, _ in reversed(entries):
            while len(self.held[s]) > pages_of(new[s], self.P):
                self.free.append(self.held[s].pop())
        rows = []
        for s, _ in entries:
            while len(self.held[s]) < pages_of(new[s], self.P):
                self.held[s].append(self.free.pop())
            rows += [(self.held[s][p // self.P] * self.P + p % self.P, p, s) for p in range(self.lens[s], new[s])]
            self.lens[s] = new[s]
        return rows


def turned(x, hd, positions, inv_freq, weight=None, bias=None, eps=1e-6):
    """[n, heads * hd] rows with bias, QK-norm and half-split rotation in 64 bits; the angle is the float32 product."""
    x = x.astype(np.float64)
    if bias is not None:
        x = x + bias
    x = x.reshape(len(x), -1, hd)
    if weight is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * weight
    angle = (positions.astype(np.float32)[:, None] * inv_freq).astype(np.float64)[:, None]
    a, b = x[..., :hd // 2], x[..., hd // 2:]
    return np.concatenate([a * np.cos(angle) - b * np.sin(angle), b * np.cos(angle) + a * np.sin(angle)], -1).reshape(len(x), -1)


def attended(q, k, v):
    """q [H, hd], k, v [KV, n, hd] in 64 bits: the output [H, hd], and how far a float32 computation of it may be off.

    With u = 2^-24: a score, a sum of hd products in any order and one scaling, is off by at most (hd + 2) u times the sum of
    their sizes, S of which the largest is taken; a weight then by a factor of exp(2 (hd + 2) u S) at most against the others and a
    few u of the exponential (its argument is rounded, too: another 2 u S); numerator and denominator are sums of n terms in any order, n u each,
    and the parts that a split over the keys leaves are scaled and added with a few u more."""
    H, hd = q.shape
    KV, n = k.shape[:2]
    q, k, v = (x.astype(np.float64) for x in (q, k, v))
    if n == 0:
        return np.zeros((H, hd)), np.zeros((H, hd))
    qg = q.reshape(KV, H // KV, hd)
    s = qg @ k.transpose(0, 2, 1) / np.sqrt(hd)
    w = np.exp(s - s.max(-1, keepdims=True))
    w /= w.sum(-1, keepdims=True)
    size = (np.abs(qg) @ np.abs(k).transpose(0, 2, 1) / np.sqrt(hd)).max(-1, keepdims=True)
    off = 2.0 ** -24 * (2 * (hd + 4) * size + 2 * n + 40) * (w @ np.abs(v))
    return (w @ v).reshape(H, hd), off.reshape(H, hd) + 1e-30
