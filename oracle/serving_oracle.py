"""The operators of a quantised serving step on the CPU, from their definitions: page plans request by request, the cache's bits in the fp32
steps that define them (one rounding each), attention and 4-bit products in float64."""
import numpy as np
import torch

TOP = {'int8': np.float32(127), 'fp8': np.float32(448)}
FLOOR = np.float32(2.0**-100)


def plan(lens, new, ring, state, table, page, n_rows):
    """-> dict(lens, cu, slots, places, ring, state, table, status); the arguments stay as they are."""
    lens, ring, table = list(map(int, lens)), np.array(ring), np.array(table)
    head, count = map(int, state)
    n, blocks, wide = len(lens), len(ring), table.shape[1]
    pages = lambda t: -(-t // page)
    status, take, give, rows = 0, 0, 0, 0
    for length, add in zip(lens, map(int, new)):
        if length < 0:
            status |= 8
        held, room = max(length, 0), wide * page
        if held > room or (add > 0 and pages(held + add) > wide):
            status |= 1
        held, have = min(held, room), pages(min(held, room))
        take += max(min(pages(held + min(add, n_rows + 1)), wide) - have, 0) if add >= 0 else 0
        give += have if add < 0 else 0
        rows += min(max(add, 0), n_rows + 1)
    status |= 2 if take > max(count, 0) else 0
    status |= 4 if rows > n_rows else 0
    status |= 8 if count < 0 or not 0 <= head < blocks or max(count, 0) + give > blocks else 0
    out = dict(lens=lens, cu=[0] * (n + 1), slots=[-1] * n_rows, places=[-1] * n_rows, ring=ring, state=[head, count], table=table, status=status)
    if status:
        return out
    front, end, at = head, head + count, 0
    for b, add in enumerate(map(int, new)):
        out['cu'][b] = at
        have = pages(lens[b])
        if add < 0:
            for j in range(have):
                ring[end % blocks] = table[b, j]
                end += 1
            lens[b] = 0
            continue
        for j in range(have, pages(lens[b] + add)):
            table[b, j] = ring[front % blocks]
            front += 1
        for t in range(lens[b], lens[b] + add):
            slot = table[b, t // page] * page + t % page
            out['slots'][at], out['places'][at] = (int(slot) if 0 <= table[b, t // page] < blocks else -1), t
            at += 1
        lens[b] += add
    out['cu'][n], out['state'] = at, [front % blocks, end - front]
    return out


def rotate(x, cos_sin, pairs):
    """x fp32 [rows, heads, size], cos_sin [rows, rot / 2, 2]: every product, difference and sum rounded to x's type."""
    rot = 2 * cos_sin.shape[1]
    y = x.copy()
    c, s = cos_sin[:, None, :, 0], cos_sin[:, None, :, 1]
    i, j = (slice(0, rot, 2), slice(1, rot, 2)) if pairs else (slice(0, rot // 2), slice(rot // 2, rot))
    a, b = x[..., i], x[..., j]
    y[..., i], y[..., j] = a * c - b * s, b * c + a * s
    return y


def store(x, kind):
    """fp32 in units of the scale -> the 8-bit element, as the fp32 number that it is."""
    x = np.where(np.isnan(x), np.float32(0), x)
    if kind == 'int8':
        return np.clip(np.rint(x), -128, 127).astype(np.float32)
    return torch.from_numpy(np.ascontiguousarray(x)).to(torch.float8_e4m3fn).float().numpy()


def append(pool, scales, k, v, slots, page, kind, largest):
    """pool fp32 [blocks, 2, heads, page * size] (elements as numbers), scales fp32, k and v fp32 [rows, heads, size] as they enter: both changed
    in place.  `largest`: the largest finite value of the input's type."""
    blocks, _, heads, n = pool.shape
    size, rows, t = n // page, len(slots), 0
    while t < rows:
        s = int(slots[t])
        if not 0 <= s < blocks * page:
            t += 1
            continue
        block, off, end = s // page, s % page, t + 1
        while end < rows and int(slots[end]) == s + end - t and (s + end - t) // page == block:
            end += 1
        for which, x in ((0, k), (1, v)):
            x = np.clip(x[t:end], -np.float32(largest), np.float32(largest)).transpose(1, 0, 2)  # [heads, rows of the run, size]
            for h in range(heads):
                page_of = pool[block, which, h].reshape((page, size) if which == 0 else (size, page))
                at = page_of if which == 0 else page_of.T
                old = scales[block, which, h] if off else np.float32(0)
                with np.errstate(invalid='ignore'):
                    big = np.fmax(np.fmax.reduce(np.abs(x[h]), axis=None), FLOOR)
                new = max(old, np.float32(big / TOP[kind]))
                if off and new > old:
                    at[:off] = store(at[:off] * np.float32(old / new), kind)
                at[off:off + end - t] = store(x[h] / new, kind)
                scales[block, which, h] = new
        t = end


def attention(q, pool, scales, table, cu, lens, page, scale, window=0):
    """float64: q [rows, heads, size], pool [blocks, 2, kv_heads, page * size] as numbers -> (out, spread, worst): the result, sum_j p_j |v_j|, and the
    largest sum_d |q_d k_d| * scale of a visible key, of which an implementation's error is a small part.  Rows of no request are NaN."""
    rows, heads, size = q.shape
    kv = pool.shape[2]
    out, spread, worst = np.full(q.shape, np.nan), np.zeros(q.shape), np.zeros((rows, heads, 1))
    for b in range(len(lens)):
        n, length = int(cu[b + 1] - cu[b]), min(max(int(lens[b]), 0), table.shape[1] * page)
        for h in range(heads):
            j = h // (heads // kv)
            keys, vals, ok = np.zeros((length, size)), np.zeros((length, size)), np.zeros(length, bool)
            for i in range(-(-length // page)):
                block, m = int(table[b, i]), min(page, length - i * page)
                if 0 <= block < pool.shape[0]:
                    keys[i * page:i * page + m] = (pool[block, 0, j].astype(np.float64) * scales[block, 0, j]).reshape(page, size)[:m]
                    vals[i * page:i * page + m] = (pool[block, 1, j].astype(np.float64) * scales[block, 1, j]).reshape(size, page).T[:m]
                    ok[i * page:i * page + m] = True
            for i in range(n):
                r, place = int(cu[b]) + i, length - n + i
                see = ok & (np.arange(length) <= place) & (np.arange(length) > (place - window if window else -1))
                out[r, h] = 0
                if not see.any():
                    continue
                x = q[r, h].astype(np.float64)
                z = keys[see] @ x * scale
                p = np.exp(z - z.max())
                p /= p.sum()
                out[r, h], spread[r, h] = p @ vals[see], p @ np.abs(vals[see])
                worst[r, h] = (np.abs(keys[see]) @ np.abs(x)).max() * abs(scale)
    return out, spread, worst


def group_product(x, q, scales, group):
    """float64: -> (y, sum_k |x q s|, sum_k |x| s)."""
    w = np.repeat(scales.astype(np.float64), group, 1)[:, :q.shape[1]]
    x = x.astype(np.float64)
    return x @ (q * w).T, np.abs(x) @ np.abs(q * w).T, np.abs(x) @ w.T
