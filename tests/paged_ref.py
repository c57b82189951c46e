"""The operators over ragged batches and paged caches from their definitions: numpy, in f64 and
whole numbers."""
import numpy as np

NONE = 0xFFFFFFFF


def block_tables(past, new, held, free, tables, block, rows):
    """starts, slots and positions of the live rows, held for the next step, tables."""
    past, new, held, free = ([int(v) for v in x] for x in (past, new, held, free))
    tables = np.array(tables, np.int64)
    B, taken, at, starts, slots, positions = len(past), held[-1], 0, [0], [], []
    for b in range(B):
        n = min(new[b], rows - at)
        while n and held[b] * block < past[b] + n and held[b] < tables.shape[1] and taken < len(free):
            tables[b, held[b]] = free[taken]
            held[b] += 1
            taken += 1
        for i in range(n):
            page, off = divmod(past[b] + i, block)
            slots.append((int(tables[b, page]) * block + off) % (1 << 32) if page < min(held[b], tables.shape[1]) else NONE)
            positions.append(past[b] + i)
        at += n
        starts.append(at)
    return starts, slots, positions, held[:-1] + [taken], tables


def paged_attention(q, kc, vc, tables, starts, past, scale, window):
    """(o, the mean of |value| under the weights) of every live row, f64; NaN elsewhere."""
    T, NH, HD = q.shape
    NB, NKV, BS, _ = kc.shape
    o, mag = np.full(q.shape, np.nan), np.full(q.shape, np.nan)
    for b in range(len(past)):
        for r in range(int(starts[b]), min(int(starts[b + 1]), T)):
            p = int(past[b]) + r - int(starts[b])
            j = np.arange(max(0, p + 1 - window) if window else 0, min(p + 1, tables.shape[1] * BS))
            page = tables[b][j // BS].astype(np.int64)
            j, page = j[page < NB], page[page < NB]
            for h in range(NH):
                if not len(j):
                    o[r, h], mag[r, h] = 0.0, 0.0
                    continue
                k, v = kc[page, h // (NH // NKV), j % BS], vc[page, h // (NH // NKV), j % BS]
                s = k @ q[r, h] * scale
                w = np.exp(s - s.max())
                w /= w.sum()
                o[r, h], mag[r, h] = w @ v, w @ np.abs(v)
    return o, mag


def verify(p, q, tokens, starts, u, draw):
    """(tokens of the live rows, accepted)."""
    out, accepted = [], []
    T = len(tokens)
    for b in range(len(draw)):
        r, e, n = min(int(starts[b]), T), min(int(starts[b + 1]), T), 0
        if r >= e:
            accepted.append(0)
            continue
        weight = None
        while r + 1 < e:
            x = int(tokens[r + 1])
            if x < p.shape[1] and float(u[r]) * (1.0 if q is None else q[r, x]) < p[r, x]:
                out.append(x)
                n, r = n + 1, r + 1
                continue
            if q is None:
                weight = p[r].copy()
                if x < p.shape[1]:
                    weight[x] = 0.0
            else:
                weight = p[r] - q[r]
            weight = np.where(weight > 0, weight, 0.0)
            if not weight.sum() > 0:
                weight = None
            break
        if weight is None:
            weight = np.where(p[r] > 0, p[r], 0.0)
        run = np.cumsum(weight)
        over = np.nonzero((run > float(draw[b]) * run[-1]) & (weight > 0))[0]
        out.append(int(over[0]) if len(over) else int(np.nonzero(weight)[0][-1]) if weight.any() else NONE)
        out += [NONE] * (e - r - 1)
        accepted.append(n)
    return out, accepted
