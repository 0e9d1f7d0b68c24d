"""More operators of a paged cache in plain numpy, in 64 bits, row by row: append with norms and axes, shared prefixes, sums of attention weights, eviction."""
import numpy as np

from tests.oracle_paged import rows_of, sees


def norm(x, w, eps):
    """x [heads, dim]"""
    return x if w is None else x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w


def turn(x, cos, sin, at, rotary, neighbours, axis):
    """x [heads, dim] with pair i turned by row at[axis[i]] of the tables; also the sum of the magnitudes that meet in every element."""
    y, mass = x.copy(), np.abs(x)
    half = rotary // 2
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if neighbours else (i, i + half)
        c, s = cos[at[axis[i]], i], sin[at[axis[i]], i]
        y[:, a] = x[:, a] * c - x[:, b] * s
        y[:, b] = x[:, b] * c + x[:, a] * s
        mass[:, a] = np.abs(x[:, a] * c) + np.abs(x[:, b] * s)
        mass[:, b] = np.abs(x[:, b] * c) + np.abs(x[:, a] * s)
    return y, mass


def append(keys, values, table, lengths, starts, k, v, q=None, cos=None, sin=None, rotary=0, neighbours=False, positions=None, q_norm=None, k_norm=None, eps=0.0, axis=None):
    """keys, values [pages, heads, page, dim] of a layer are written in place, positions [axes, tokens]. Returns the queries (NaN where a token is not
    touched) and the magnitudes that met in keys and queries (zero where nothing was computed)."""
    pages, _, page, _ = keys.shape
    out = None if q is None else np.full(q.shape, np.nan)
    mass_k, mass_q = np.zeros(keys.shape), None if q is None else np.zeros(q.shape)
    axis = [0] * (rotary // 2) if axis is None else axis
    for s in range(len(lengths)):
        before = min(max(int(lengths[s]), 0), table.shape[1] * page)
        for t in range(starts[s], starts[s + 1]):
            row = before + t - starts[s]
            at = [row] if positions is None else [int(p[t]) for p in positions]
            if rotary and not all(0 <= p < len(cos) for p in at):
                continue
            if q is not None:
                out[t], mass_q[t] = turn(norm(q[t], q_norm, eps), cos, sin, at, rotary, neighbours, axis)
            if row >= table.shape[1] * page:
                continue
            p = int(table[s, row // page])
            if 0 <= p < pages:
                keys[p, :, row % page], mass_k[p, :, row % page] = turn(norm(k[t], k_norm, eps), cos, sin, at, rotary, neighbours, axis)
                values[p, :, row % page] = v[t]
    return out, mass_k, mass_q


def attention(keys, values, table, lengths, starts, q, scale, mask=None, weights=None):
    """As tests/oracle_paged.py's attention; weights [sequences, kv heads, rows]: a copy with the softmax weights added comes back too."""
    pages, nkv, page, _ = keys.shape
    tokens, heads, _ = q.shape
    per = heads // nkv
    out, mass, dot = np.zeros(q.shape), np.zeros(q.shape), np.zeros((tokens, heads))
    sums = None if weights is None else weights.copy()
    for s in range(len(lengths)):
        most = table.shape[1] * page
        before, new = min(max(int(lengths[s]), 0), most), starts[s + 1] - starts[s]
        end = min(before + new, most)
        where = rows_of(table, pages, page, s, end)
        there = np.array([p >= 0 for p, _ in where], dtype=bool)
        pick = [(max(p, 0), r) for p, r in where]
        kr = np.array([keys[p, :, r] for p, r in pick]).reshape(end, nkv, -1)
        vr = np.array([values[p, :, r] for p, r in pick]).reshape(end, nkv, -1)
        wide = 0 if sums is None else min(end, sums.shape[2])
        if sums is not None and new > 0:
            sums[s, :, before:wide] = 0
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
                if sums is not None:
                    full = np.zeros(end)
                    full[vis] = w
                    sums[s, h // per, :wide] += full[:wide]
    return out, mass, dot, sums


def evict(keys, values, table, lengths, weights, weights_out, budget, recent):
    """keys, values [layers, pages, heads, page, dim] and weights_out in place; the new lengths."""
    layers, pages, heads, page, _ = keys.shape
    most = table.shape[1] * page
    heavy, out = budget - recent, []
    for s in range(len(lengths)):
        n = min(max(int(lengths[s]), 0), most)
        where = rows_of(table, pages, page, s, most)
        wide = weights.shape[3]
        out.append(min(n, budget))
        for layer in range(layers):
            for h in range(heads):
                w = weights[layer, s, h]
                if n <= budget:
                    weights_out[layer, s, h, :n] = w[:n]
                    continue
                rank = [-np.inf if r >= wide or np.isnan(w[r]) else w[r] for r in range(n - recent)]
                best = sorted(range(n - recent), key=lambda r: (-rank[r], r))[:heavy]
                holes, movers = sorted(set(range(heavy)) - set(best)), sorted(r for r in best if r >= heavy)
                moves = list(zip(movers, holes)) + [(n - recent + i, heavy + i) for i in range(recent)]
                source = list(range(heavy)) + [n - recent + i for i in range(recent)]
                for r, t in zip(movers, holes):
                    source[t] = r
                weights_out[layer, s, h, :budget] = w[source]
                old = [x[layer, :, h].copy() for x in (keys, values)]
                for r, t in moves:
                    (p, a), (pt, at) = where[r], where[t]
                    if p >= 0 and pt >= 0:
                        for x, o in zip((keys, values), old):
                            x[layer, pt, h, at] = o[p, a]
    return np.array(out, dtype=np.int32)
