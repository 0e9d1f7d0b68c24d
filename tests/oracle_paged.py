"""A paged cache's operators and beam selection in plain numpy, in 64 bits, row by row."""
import math

import numpy as np


def rows_of(table, pages, page_size, seq, count):
    """(page, slot) of the first rows of a sequence; page -1 where the table names none."""
    got = []
    for r in range(count):
        p = int(table[seq, r // page_size]) if r // page_size < table.shape[1] else -1
        got.append((p if 0 <= p < pages else -1, r % page_size))
    return got


def rotate(x, cos, sin, rotary, neighbours):
    """x [heads, dim] by one row of the tables."""
    y = x.copy()
    half = rotary // 2
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if neighbours else (i, i + half)
        y[:, a] = x[:, a] * cos[i] - x[:, b] * sin[i]
        y[:, b] = x[:, b] * cos[i] + x[:, a] * sin[i]
    return y


def append(keys, values, table, lengths, starts, k, v, q=None, cos=None, sin=None, rotary=0, neighbours=False, positions=None):
    """keys, values [pages, heads, page, dim] of a layer are written in place; the rotated queries are returned (NaN where a token is not touched)."""
    pages, _, page, _ = keys.shape
    out = None if q is None else np.full(q.shape, np.nan)
    for s in range(len(lengths)):
        before = min(max(int(lengths[s]), 0), table.shape[1] * page)
        for t in range(starts[s], starts[s + 1]):
            row = before + t - starts[s]
            at = row if positions is None else int(positions[t])
            if rotary and not 0 <= at < len(cos):
                continue
            turn = (lambda x: rotate(x, cos[at], sin[at], rotary, neighbours)) if rotary else (lambda x: x)
            if q is not None:
                out[t] = turn(q[t])
            if row >= table.shape[1] * page:
                continue
            p = int(table[s, row // page])
            if 0 <= p < pages:
                keys[p, :, row % page] = turn(k[t])
                values[p, :, row % page] = v[t]
    return out


def sees(mask, causal_t, d):
    if mask is None:
        return d <= causal_t
    return d < 64 * len(mask) and (int(mask[d // 64]) >> (d % 64)) & 1 == 1


def attention(keys, values, table, lengths, starts, q, scale, mask=None):
    """(outputs, sum of weights times |value|, largest sum of |q k| of a row): the last two for bounds on rounding."""
    pages, nkv, page, dim = keys.shape
    tokens, heads, _ = q.shape
    per = heads // nkv
    out, mass, dot = np.zeros(q.shape), np.zeros(q.shape), np.zeros((tokens, heads))
    for s in range(len(lengths)):
        most = table.shape[1] * page
        before, new = min(max(int(lengths[s]), 0), most), starts[s + 1] - starts[s]
        end = min(before + new, most)
        where = rows_of(table, pages, page, s, end)
        there = np.array([p >= 0 for p, _ in where], dtype=bool)
        pick = [(max(p, 0), r) for p, r in where]
        kr = np.array([keys[p, :, r] for p, r in pick]).reshape(end, nkv, dim)
        vr = np.array([values[p, :, r] for p, r in pick]).reshape(end, nkv, dim)
        for t in range(starts[s], starts[s + 1]):
            m = None if mask is None else mask[t]
            vis = there.copy()
            for r in range(before, end):
                vis[r] = vis[r] and sees(m, t - starts[s], r - before)
            if not vis.any():
                continue
            for h in range(heads):
                kk, vv = kr[vis, h // per], vr[vis, h // per]
                x = kk @ q[t, h] * scale
                w = np.exp(x - x.max())
                w /= w.sum()
                out[t, h], mass[t, h] = w @ vv, w @ np.abs(vv)
                dot[t, h] = (np.abs(kk) @ np.abs(q[t, h])).max() * abs(scale)
    return out, mass, dot


def select(logits, scores, picks, done=None, end_token=-1):
    """[(value, beam, token)] of every group, best first, all candidates."""
    groups, beams, vocab = logits.shape
    got = []
    for g in range(groups):
        value = np.full((beams, vocab), -np.inf)
        for b in range(beams):
            if done is not None and done[g, b]:
                value[b, end_token] = scores[g, b]
                continue
            x = logits[g, b]
            top = x.max() if not np.isnan(x).any() else np.nan
            if not math.isfinite(top):
                continue
            value[b] = scores[g, b] + (x - (top + math.log(np.exp(x - top).sum())))
        flat = value.reshape(-1)
        order = np.argsort(-np.where(np.isnan(flat), -np.inf, flat), kind="stable")[:picks + 1]
        got.append([(flat[i], int(i) // vocab, int(i) % vocab) if flat[i] > -np.inf else (-np.inf, -1, -1) for i in order])
    return got


def keep(keys, values, table, lengths, accepted, counts):
    """keys, values [layers, pages, heads, page, dim] in place; the new lengths."""
    pages, page = keys.shape[1], keys.shape[3]
    most = table.shape[1] * page
    out = []
    for s in range(len(lengths)):
        before = min(max(int(lengths[s]), 0), most)
        n = min(max(int(counts[s]), 0), accepted.shape[1])
        where = rows_of(table, pages, page, s, most)
        old_k, old_v = keys.copy(), values.copy()
        for j in range(n):
            a = int(accepted[s, j])
            if a <= j or before + a >= most:
                continue
            (p, r), (pt, rt) = where[before + a], where[before + j]
            if p >= 0 and pt >= 0:
                keys[:, pt, :, rt] = old_k[:, p, :, r]
                values[:, pt, :, rt] = old_v[:, p, :, r]
        out.append(before + n)
    return np.array(out, dtype=np.int32)


def reorder(keys, values, table, lengths, parents, group):
    """keys, values in place; (new table, new lengths)."""
    page = keys.shape[3]
    new_table, new_len = table.copy(), np.array(lengths, dtype=np.int32)
    for g in range(0, len(lengths), group):
        par = [g + (int(p) if 0 <= p < group else i) for i, p in enumerate(parents[g:g + group])]
        free = [b for b in range(g, g + group) if b not in par]
        met = set()
        for i, p in enumerate(par):
            new_table[g + i], new_len[g + i] = table[p], lengths[p]
            last, rows = int(lengths[p]) // page, int(lengths[p]) % page
            if p in met:
                d = free.pop(0)
                old = int(lengths[d]) // page
                width = table.shape[1]
                for j in range(last, width):
                    new_table[g + i, j] = table[d, old + j - last] if old + j - last < width else -1
                if last < width and old < width:
                    to, src = int(table[d, old]), int(table[p, last])
                    for x in (keys, values):
                        x[:, to, :, :rows] = x[:, src, :, :rows]
            met.add(p)
    return new_table, new_len
