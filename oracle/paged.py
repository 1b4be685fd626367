"""CPU oracle for rotary positions, the paged 4-bit cache and the attention over
it -- TEST INFRASTRUCTURE ONLY (tests/ alone imports it).

In float64 (numpy), from the definitions in include/fa_mi355x.h:

  rotate     -- pairs turned by position * frequency.
  stored     -- what 4 bits hold of a row: 32 columns to a power of two, each the
                nearest e2m1 number.
  PagedModel -- the values each slot of each page holds, by store / gather
                through a page table.
  attend     -- softmax attention of the newest queries, bottom-right causal,
                with the two sums that error bounds need.
"""
from __future__ import annotations

import numpy as np

E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
MAX_F16, MAX_BF16 = 65504.0, float(np.uint32(0x7F7F0000).view(np.float32))


def rotate(x, positions, frequencies, factor=1.0, interleaved=False, inverse=False):
    """x (B, S, heads, D) float64; positions (B, S) ints; frequencies (R/2)."""
    x = np.asarray(x, dtype=np.float64)
    R = 2 * len(frequencies)
    angle = np.asarray(positions, dtype=np.float64)[..., None] * np.asarray(frequencies)
    c = np.cos(angle)[:, :, None] * factor
    s = np.sin(angle)[:, :, None] * factor * (-1.0 if inverse else 1.0)
    y = x.copy()
    a, b = ((slice(0, R, 2), slice(1, R, 2)) if interleaved
            else (slice(0, R // 2), slice(R // 2, R)))
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    return y


def stored(x, fp16):
    """The values that the cache holds of x (.., D) float64."""
    x = np.asarray(x, dtype=np.float64)
    top = MAX_F16 if fp16 else MAX_BF16
    x = np.clip(np.where(np.isnan(x), 0.0, x), -top, top)
    b = x.reshape(*x.shape[:-1], -1, 32)
    big = np.abs(b).max(-1, keepdims=True)
    e = np.frexp(big)[1] - 3                  # floor(log2 big) - 2
    e = np.clip(np.where(big == 0, -126, e), -126, 13 if fp16 else 125)
    a = np.abs(np.ldexp(b, -e))
    # nearest of the grid; a tie goes to the even code
    d = np.abs(a[..., None] - E2M1)
    code = d.argmin(-1)
    nxt = np.minimum(code + 1, 7)
    tie = (np.take_along_axis(d, nxt[..., None], -1)[..., 0] == d.min(-1)) & (code % 2 == 1)
    code = np.where(tie, nxt, code)
    return np.ldexp(np.copysign(E2M1[code], b), e).reshape(x.shape)


class PagedModel:
    """Slots (pages, page_size, heads, D) of float64 keys and values, 0 at first."""

    def __init__(self, pages, page_size, heads, D, fp16):
        self.k = np.zeros((pages, page_size, heads, D))
        self.v = np.zeros((pages, page_size, heads, D))
        self.fp16 = fp16

    def slot(self, table, b, pos):
        """(page, slot) of a position, or None."""
        P = self.k.shape[1]
        if pos < 0 or pos // P >= table.shape[1]:
            return None
        page = int(table[b, pos // P])
        return (page, pos % P) if 0 <= page < self.k.shape[0] else None

    def store(self, k, v, table, start, counts=None):
        k, v = stored(k, self.fp16), stored(v, self.fp16)
        for b in range(k.shape[0]):
            n = k.shape[1] if counts is None else min(max(int(counts[b]), 0), k.shape[1])
            for i in range(n):
                at = self.slot(table, b, int(start[b]) + i)
                if at is not None:
                    self.k[at], self.v[at] = k[b, i], v[b, i]

    def gather(self, table, b, positions):
        """(k, v, held) of positions: (n, heads, D) and which slots exist."""
        heads, D = self.k.shape[2:]
        n = len(positions)
        k, v, held = np.zeros((n, heads, D)), np.zeros((n, heads, D)), np.zeros(n, dtype=bool)
        for i, p in enumerate(positions):
            at = self.slot(table, b, int(p))
            if at is not None:
                k[i], v[i], held[i] = self.k[at], self.v[at], True
        return k, v, held


def attend(q, model, table, lengths, counts=None, scale=None):
    """(out, lse, abs_out, abs_v, abs_s): q (B, Sq, H, D) float64.  abs_out =
    sum p |v|, abs_v = sum |v| over the keys seen (B, Sq, H, D), abs_s = the
    largest scale * sum |q k| of a row (B, H, Sq)."""
    q = np.asarray(q, dtype=np.float64)
    B, Sq, H, D = q.shape
    P, Hk = model.k.shape[1:3]
    G = H // Hk
    scale = D ** -0.5 if scale is None else scale
    out, abs_out, abs_v = (np.zeros((B, Sq, H, D)) for _ in range(3))
    lse, abs_s = np.full((B, H, Sq), np.inf), np.zeros((B, H, Sq))
    for b in range(B):
        n = Sq if counts is None else min(max(int(counts[b]), 0), Sq)
        keys = max(0, min(int(lengths[b]), table.shape[1] * P))
        k, v, held = model.gather(table, b, range(keys))
        for i in range(n):
            seen = held & (np.arange(keys) <= int(lengths[b]) - n + i)
            if not seen.any():
                continue
            ks, vs = k[seen].repeat(G, axis=1), v[seen].repeat(G, axis=1)
            s = np.einsum("hd,nhd->hn", q[b, i], ks) * scale
            top = s.max(-1, keepdims=True)
            p = np.exp(s - top)
            total = p.sum(-1, keepdims=True)
            p /= total
            out[b, i] = np.einsum("hn,nhd->hd", p, vs)
            abs_out[b, i] = np.einsum("hn,nhd->hd", p, np.abs(vs))
            abs_v[b, i] = np.abs(vs).sum(0)
            lse[b, :, i] = (top + np.log(total))[:, 0]
            abs_s[b, :, i] = (np.einsum("hd,nhd->hn", np.abs(q[b, i]), np.abs(ks))
                              * abs(scale)).max(-1)
    return out, lse, abs_out, abs_v, abs_s
