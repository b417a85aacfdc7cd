"""The 8-bit KV cache and the verification of drafts in 64 bits, written from their definitions with
plain loops over sequences: what the GPU tests compare with. Everything here runs on the CPU."""
from __future__ import annotations

import numpy as np

PAGE = 16


def e4m3_values() -> np.ndarray:
    """The 256 values by code: sign, 4 exponent bits (bias 7), 3 significand bits; 0x7F is NaN."""
    v = np.empty(256)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        x = m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        v[c] = np.nan if (c & 127) == 127 else (-x if c & 128 else x)
    return v


VALUES = e4m3_values()
POSITIVE = VALUES[:127]  # ascending, 0 .. 448
MIDDLES = (POSITIVE[1:] + POSITIVE[:-1]) / 2


def encode(x: np.ndarray) -> np.ndarray:
    """The codes of the nearest values, ties to the even code, past 448 clamped; NaN, inf: NaN."""
    x = np.asarray(x, np.float64)
    mag = np.where(np.isfinite(x), np.minimum(np.abs(x), 448.0), 0.0)
    low = np.searchsorted(MIDDLES, mag, side="left")  # ties stay below
    tie = (low < 126) & (mag == MIDDLES[np.minimum(low, 125)])
    code = low + (tie & (low % 2 == 1))
    code = np.where(np.isfinite(x), code, 127) | np.where(np.signbit(x), 128, 0)
    return code.astype(np.uint8)


def least_exponent(most: float) -> int:
    e = -15
    while e < 7 and most > 448.0 * 2.0 ** e:
        e += 1
    return e


class Cache:
    """One side (K or V) of a cache."""

    def __init__(self, num_pages, n_kv, dim, code=0x7F, scale=np.nan):
        self.codes = np.full((num_pages, n_kv, PAGE, dim), code, np.uint8)
        self.scale = np.full((num_pages, n_kv), scale, np.float32)

    def append(self, page, slot, x):
        """Writes x [rows, n_kv, dim] (64 bits) from `slot` of `page` on."""
        for h in range(x.shape[1]):
            mag = np.abs(x[:, h])
            most = mag[np.isfinite(mag)].max(initial=0.0)
            e = least_exponent(most)
            if slot > 0:
                old = int(np.log2(self.scale[page, h]))
                if e > old:
                    self.codes[page, h, :slot] = encode(
                        VALUES[self.codes[page, h, :slot]] * 2.0 ** (old - e))
                e = max(e, old)
            self.scale[page, h] = 2.0 ** e
            self.codes[page, h, slot:slot + x.shape[0]] = encode(x[:, h] * 2.0 ** -e)

    def rows(self, pages, positions):
        """[position, n_kv, dim] in 64 bits."""
        pg, slot = pages[positions // PAGE], positions % PAGE
        return VALUES[self.codes[pg, :, slot]] * self.scale[pg].astype(np.float64)[:, :, None]


def rotate(x, pos, inv_freq):
    """x [rows, heads, dim] at positions pos [rows], in 64 bits."""
    half = x.shape[-1] // 2
    a = pos[:, None].astype(np.float64) * inv_freq.astype(np.float64)
    c, s = np.cos(a)[:, None], np.sin(a)[:, None]
    x1, x2 = x[..., :half], x[..., half:]
    return np.concatenate([x1 * c - x2 * s, x2 * c + x1 * s], -1)


def spans(starts, lens, n_seqs):
    """(sequence, first row, end row, position of the first row) of every sequence."""
    for s in range(n_seqs):
        r0, r1 = (s, s + 1) if starts is None else (int(starts[s]), int(starts[s + 1]))
        yield s, r0, r1, int(lens[s]) - (r1 - r0)


def append(k, v, qkv, tables, starts, lens, inv_freq, n_heads, n_kv, dim):
    """Appends to the Caches k and v; returns q [rows, n_heads, dim] in 64 bits (NaN: a row of no
    sequence)."""
    n_rows, limit = qkv.shape[0], tables.shape[1] * PAGE
    x = qkv[:, :(n_heads + 2 * n_kv) * dim].astype(np.float64).reshape(n_rows, -1, dim)
    q = np.full((n_rows, n_heads, dim), np.nan)
    for s, r0, r1, first in spans(starts, lens, tables.shape[0]):
        pos = first + np.arange(r1 - r0)
        inside = (pos >= 0) & (pos < limit)
        with np.errstate(invalid="ignore"):
            turned = rotate(x[r0:r1, :n_heads + n_kv], pos, inv_freq)
        q[r0:r1] = np.where(inside[:, None, None], turned[:, :n_heads], 0.0)
        for page in sorted(set(pos[inside] // PAGE)):
            at = np.flatnonzero(inside & (pos // PAGE == page))
            slot = int(pos[at[0]] % PAGE)
            k.append(tables[s, page], slot, turned[at, n_heads:])
            v.append(tables[s, page], slot, x[r0 + at, n_heads + n_kv:])
    return q


def gather(cache, tables, starts, lens, n_rows):
    """[rows, n_kv, dim]; NaN-free zeros where a position is nowhere, +inf: a row of no sequence."""
    out = np.full((n_rows, cache.codes.shape[1], cache.codes.shape[3]), np.inf)
    for s, r0, r1, first in spans(starts, lens, tables.shape[0]):
        pos = first + np.arange(r1 - r0)
        inside = (pos >= 0) & (pos < tables.shape[1] * PAGE)
        out[r0:r1] = 0.0
        out[np.arange(r0, r1)[inside]] = cache.rows(tables[s], pos[inside])
    return out


def attention(q, k, v, tables, starts, lens):
    """(out, bound) [rows, heads, dim] in 64 bits. `bound` is what fp32 scores, weights and sums and
    one rounding to fp16 may be off by: a score s is a sum of dim products, off by at most dim 2^-24
    of sum |q_i k_i| / sqrt(dim), its distance to the maximum by that again and by 2^-22 of itself
    (scale, difference and exponent are each rounded); weights, and so Σ p v, by that relative to
    Σ p |v|, twice for the quotient, with 2^-20 for the exponentials and for sums of up to 2^16 terms
    taken in parts. A weight may enter Σ p v as two bf16, its first 8 bits cut off (what is left is
    below 2^-7 of it) and the rest rounded to 8 (2^-8 of the rest): 2^-15 of it."""
    n_rows, heads, dim = q.shape
    n_kv = k.codes.shape[1]
    out, bound = np.full(q.shape, np.inf), np.zeros(q.shape)
    q = q.astype(np.float64)
    for s, r0, r1, first in spans(starts, lens, tables.shape[0]):
        end = min(int(lens[s]), tables.shape[1] * PAGE)
        if end > 0:
            pos = np.arange(end)
            K, V = k.rows(tables[s], pos), v.rows(tables[s], pos)
        for r in range(r0, r1):
            see = min(first + (r - r0) + 1, end)
            for h in range(heads):
                if see <= 0:
                    out[r, h] = 0.0
                    continue
                g = h // (heads // n_kv)
                with np.errstate(invalid="ignore"):
                    a = K[:see, g] @ q[r, h] / np.sqrt(dim)
                    off = np.abs(K[:see, g]) @ np.abs(q[r, h]) / np.sqrt(dim) * dim * 2.0 ** -24
                    p = np.exp(a - a.max())
                    p /= p.sum()
                    out[r, h] = p @ V[:see, g]
                    rel = 2 * off + 2.0 ** -22 * np.abs(a - a.max())
                    rel = np.expm1(np.minimum(rel, 30.0)) + 2.0 ** -20
                    mean = (p * (rel + 2.0 ** -15)) @ np.abs(V[:see, g]) + (p * rel).sum() * (
                        p @ np.abs(V[:see, g]))
                bound[r, h] = mean + 2.0 ** -11 * np.abs(out[r, h]) + 2.0 ** -25
    return out, bound


def softmax(row, t):
    x = np.where(np.isnan(row), -np.inf, row.astype(np.float64))
    top = x.max()
    if top == -np.inf:
        return np.zeros_like(x)
    with np.errstate(invalid="ignore"):
        w = np.exp(np.where(x == top, 0.0, (x - top) / t))
    return w / w.sum()


def verify(logits, draft_logits, drafts, starts, temperature, accept_u, sample_u, n_seqs):
    """(n_accepted, tokens); tokens of rows of no sequence are -7."""
    n_rows, vocab = logits.shape
    accepted, tokens = np.zeros(n_seqs, np.int32), np.full(n_rows, -7, np.int32)
    for s, r0, r1, _ in spans(starts, np.zeros(n_seqs), n_seqs):
        t = 1.0 if temperature is None else float(temperature[s])
        tokens[r0:r1] = -1
        for r in range(r0, r1):
            row = np.where(np.isnan(logits[r]), -np.inf, logits[r].astype(np.float64))
            best = int(row.argmax()) if row.max() > -np.inf else -1
            d = int(drafts[r]) if r + 1 < r1 else -1
            inside = 0 <= d < vocab
            w = None
            if not t > 0:
                good = inside and d == best
            else:
                p = w = softmax(logits[r], t)
                if r + 1 < r1:
                    if draft_logits is not None:
                        q = softmax(draft_logits[r], t)
                    else:
                        q = np.zeros(vocab)
                        if inside:
                            q[d] = 1.0
                    good = inside and float(accept_u[r]) * q[d] < p[d]
                    w = np.maximum(p - q, 0.0)
                    w = w if w.sum() > 0 else p
            if r + 1 < r1 and good:
                tokens[r] = d
                continue
            accepted[s] = r - r0
            if w is None:
                tokens[r] = best
            elif w.sum() > 0:
                c = np.cumsum(w)
                at = np.searchsorted(c, float(sample_u[s]) * c[-1], side="right")
                tokens[r] = min(at, np.flatnonzero(w)[-1])
            break
    return accepted, tokens
