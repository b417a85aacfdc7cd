"""Adapters beside a shared projection, rotary positions and shared cache pages, written from their
definitions with plain loops, numbers in 64 bits: what the GPU tests compare with. All on the CPU."""
from __future__ import annotations

import numpy as np

HALF16, TINY16 = 2.0 ** -11, 2.0 ** -25  # fp16: half a step, relative and among subnormals


# ---------------------------------------------------------------------------------------------
# adapters
# ---------------------------------------------------------------------------------------------
def lora_add(x, a, b, ranks, scales, ids, starts, y, ends):
    """(result, bound): y [n_rows, out] in 64 bits with the adapters added, and what a result may be off by.

    h is a sum of `in` products of fp16 numbers, exact in fp32, added one behind the other: off by at most
    in 2^-24 of their magnitudes' sum, or twice that where an addition in a matrix instruction cuts instead of
    rounding. It is then held in two fp16 of 11 bits: off by 2^-22 of the largest |h| of the part, again
    doubled for both roundings. The outer sum of rank terms (two for each h) is off by (2 rank + 2) 2^-23 of
    its magnitudes; scale and y are multiplied and added in fp32, one 2^-24 each; fp16 rounds once."""
    out, bound = y.astype(np.float64), np.zeros(y.shape)
    x, a, b = (t.astype(np.float64) for t in (x, a, b))
    for s in range(len(ids)):
        r0, r1 = (s, s + 1) if starts is None else (int(starts[s]), int(starts[s + 1]))
        if not 0 <= ids[s] < a.shape[0] or r1 <= r0:
            continue
        A, rank = ids[s], a.shape[2] if ranks is None else min(int(ranks[ids[s]]), a.shape[2])
        if rank <= 0:
            continue
        scale, begin = 1.0 if scales is None else float(scales[A]), 0
        for p, end in enumerate(ends):
            w, v = a[A, p, :rank], b[A, begin:end, :rank]
            with np.errstate(all="ignore"):
                h = x[r0:r1] @ w.T
                add = h @ v.T
                size = np.abs(x[r0:r1]) @ np.abs(w).T
                off = size * x.shape[1] * 2.0 ** -23 + 2.0 ** -21 * np.abs(h).max(1, keepdims=True)
                off = off @ np.abs(v).T + (2 * rank + 2) * 2.0 ** -23 * (np.abs(h) @ np.abs(v).T)
                out[r0:r1, begin:end] += scale * add
                bound[r0:r1, begin:end] = abs(scale) * (off + 2.0 ** -22 * np.abs(add)) \
                    + 2.0 ** -23 * np.abs(y[r0:r1, begin:end].astype(np.float64))
            begin = end
    with np.errstate(all="ignore"):
        return out, bound + HALF16 * (np.abs(out) + bound) + TINY16


# ---------------------------------------------------------------------------------------------
# rotary positions
# ---------------------------------------------------------------------------------------------
def rotate(x, pos, inv_freq, table_ids, scales, rotary, pairs):
    """(result, bound) of x [rows, heads, dim] in 64 bits. Cosine and sine times the scale are rounded to
    fp32, so are the two products and their sum: 3 2^-24 of the products' magnitudes, and a fourth for what
    64 bits lose on the way; then fp16 rounds once."""
    n, half = x.shape[0], rotary // 2
    t = np.zeros(n, np.int64) if table_ids is None else table_ids.astype(np.int64)
    t = np.where((t >= 0) & (t < inv_freq.shape[0]), t, 0)
    angle = pos.astype(np.float64)[:, None] * inv_freq.astype(np.float64)[t]
    scale = 1.0 if scales is None else scales.astype(np.float64)[t][:, None]
    c, s = (np.cos(angle) * scale)[:, None], (np.sin(angle) * scale)[:, None]
    out, bound = x.astype(np.float64), np.zeros(x.shape)
    one = np.s_[..., 0:rotary:2] if pairs else np.s_[..., :half]
    two = np.s_[..., 1:rotary:2] if pairs else np.s_[..., half:rotary]
    x1, x2 = out[one].copy(), out[two].copy()
    out[one], out[two] = x1 * c - x2 * s, x2 * c + x1 * s
    off = 4 * 2.0 ** -24 * np.abs(scale if np.ndim(scale) == 0 else scale[:, None])
    bound[one] = bound[two] = off * (np.abs(x1) + np.abs(x2))
    bound[one] += HALF16 * (np.abs(out[one]) + bound[one]) + TINY16
    bound[two] += HALF16 * (np.abs(out[two]) + bound[two]) + TINY16
    return out, bound


# ---------------------------------------------------------------------------------------------
# pages
# ---------------------------------------------------------------------------------------------
def held(row, num_pages):
    pages = []
    for p in row:
        if not 0 <= p < num_pages:
            break
        pages.append(int(p))
    return pages


def fork(tables, lens, parents, reserve, refs, n_new, max_pages, page, num_pages):
    """(new_tables, new_lens, refs, copies, counts)."""
    before, refs = list(refs), [int(r) for r in refs]
    rows = [held(row, num_pages) for row in tables]
    for row in rows:
        for p in row:
            refs[p] -= 1
    new = np.full((n_new, max_pages), -1, np.int32)
    copies, new_lens, wanted, seen = np.full((n_new, 2), -1, np.int32), [], [], set()
    for c in range(n_new):
        p = int(parents[c])
        row = rows[p] if 0 <= p < len(rows) else []
        length = min(max(int(lens[p]), 0), len(row) * page) if row else 0
        new_lens.append(length)
        room = 0 if reserve is None else max(int(reserve[c]), 0)
        for j in range(min(max_pages, -(-(length + room) // page))):
            mine = row[j] if j < len(row) else -1
            if j < length // page or (mine >= 0 and p not in seen and before[mine] == 1):
                new[c, j] = mine
                refs[mine] += 1
            else:
                wanted.append((c, j, mine if j == length // page and length % page else -1))
        seen.add(p)
    copied = {mine for _, _, mine in wanted}
    free = [p for p in range(num_pages) if refs[p] == 0 and p not in copied]
    for (c, j, mine), to in zip(wanted, free):
        new[c, j], refs[to] = to, 1
        if mine >= 0:
            copies[c] = mine, to
    got = min(len(wanted), len(free))
    return (new, np.array(new_lens, np.int32), np.array(refs, np.int32), copies,
            np.array([got, len(wanted) - got], np.int32))


def compact(tables, refs):
    """(new_tables, new_refs, pairs, counts)."""
    live = [p for p in range(len(refs)) if refs[p] > 0]
    n = len(live)
    holes, movers = [p for p in range(n) if refs[p] <= 0], [p for p in live if p >= n]
    to = dict(zip(movers, holes))
    new = [int(refs[p]) if p < n else 0 for p in range(len(refs))]
    for p, hole in to.items():
        new[hole] = int(refs[p])
    tables = np.array([[to.get(int(p), int(p)) for p in row] for row in tables],
                      np.int32).reshape(tables.shape)
    return tables, np.array(new, np.int32), list(zip(movers, holes)), np.array([len(movers), n], np.int32)


def batch(rng, n, beams, max_len, page, max_pages, spare=0, tails=True):
    """A batch of n sequences in groups of up to `beams` that share whole pages: (tables, lens, refs,
    num_pages). Every sequence may hold a few pages behind its length."""
    tables, lens, wants, at = np.full((n, max_pages), -1, np.int64), np.zeros(n, np.int64), [], 0
    s = 0
    while s < n:
        k, length = min(int(rng.integers(1, beams + 1)), n - s), int(rng.integers(0, max_len + 1))
        whole = length // page
        tables[s:s + k, :whole] = at + np.arange(whole)
        at += whole
        for i in range(s, s + k):
            lens[i] = length
            more = int(length % page > 0) + (int(rng.integers(0, 3)) if tails else 0)
            more = min(more, max_pages - whole)
            tables[i, whole:whole + more] = at + np.arange(more)
            at += more
        s += k
    num_pages = max(1, at + spare)
    names = rng.permutation(num_pages)
    tables = np.where(tables >= 0, names[tables], -1)
    refs = np.bincount(tables[tables >= 0], minlength=num_pages)
    return tables.astype(np.int32), lens.astype(np.int32), refs.astype(np.int32), num_pages
