"""Plain statements of the batched cache's operators: integers and 64-bit floats, one request, tile and head after the other."""
import numpy as np

TILE, D, NONE = 16, 128, 0xFFFFFFFF
LOWEST, LARGEST = -15, 61440.0


def _decode_table():
    codes = np.arange(256)
    exp, man, sign = (codes >> 3) & 15, codes & 7, np.where(codes & 128, -1.0, 1.0)
    v = np.where(exp == 0, man * 2.0 ** -9, (8 + man) * 2.0 ** (exp - 10.0))
    v[(codes & 127) == 127] = np.nan
    return sign * v


E4M3 = _decode_table()
_POS = E4M3[:127]  # 0 .. 448 ascending, by code


def encode(x):
    """e4m3 codes of 64-bit values: nearest, ties to the even code, magnitudes above 448 as 448; NaN is 0x7f."""
    x = np.asarray(x, np.float64)
    a = np.minimum(np.abs(x), 448.0)
    a = np.where(np.isnan(x), 0.0, a)
    hi = np.searchsorted(_POS, a).clip(1, 126)
    lo = hi - 1
    dl, dh = a - _POS[lo], _POS[hi] - a
    code = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi).astype(np.uint8)
    return np.where(np.isnan(x), 0x7F, code | np.where(np.signbit(x), 0x80, 0)).astype(np.uint8)


def exponent(most):
    e = LOWEST
    while most > 448.0 * 2.0 ** e:
        e += 1
    return e


def append(x, slots, pool, exps):
    """x f16 [n, KV, 128] into pool u8 [blocks, KV, 16, 128] and exps i8 [blocks, KV], in place."""
    x = np.clip(x.astype(np.float64), -LARGEST, LARGEST)  # keeps NaN
    i, n = 0, len(slots)
    while i < n:
        if slots[i] == NONE:
            i += 1
            continue
        j = i + 1
        while j < n and slots[j] == slots[j - 1] + 1 and slots[j] % TILE:
            j += 1
        b, at = slots[i] // TILE, int(slots[i] % TILE)
        for h in range(x.shape[1]):
            a = np.abs(x[i:j, h])
            e = exponent(np.max(np.where(np.isnan(a), 0.0, a)))
            if at:
                old = int(exps[b, h])
                e = max(e, old)
                if e > old:
                    codes = pool[b, h, :at]
                    pool[b, h, :at] = np.where((codes & 127) == 127, codes, encode(E4M3[codes] * 2.0 ** (old - e)))
            pool[b, h, at:at + j - i] = encode(x[i:j, h] * 2.0 ** -e)
            exps[b, h] = e
        i = j


def plan(ctx, new, held, count, free, table, page, tokens):
    """What kv_block_tables answers, request by request; free and table are copied."""
    n, stride = table.shape
    free, table = free.copy(), table.copy()
    end, fits, need = 0, [], []
    for c, a in zip(ctx, new):
        end += int(a)
        need.append(-(-(int(c) + int(a)) // page))
        fits.append(need[-1] <= stride and end <= tokens)
    have = int(count)
    for r in range(n):
        if fits[r]:
            for j in range(need[r], int(held[r])):
                free[have] = table[r, j]
                have += 1
    left, taken, starts, lens, held_out = have, 0, [0], [], []
    refused = used = placed = 0
    slots, at = np.full(tokens, NONE, np.uint32), np.zeros(tokens, np.uint32)
    end = 0
    for r in range(n):
        want = max(need[r] - int(held[r]), 0) if fits[r] else 0
        taken += want
        ok = fits[r] and (want == 0 or taken <= have)
        if ok:
            for j in range(int(held[r]), need[r]):
                left -= 1
                table[r, j] = free[left]
            used += want
            placed += int(new[r])
        else:
            refused += 1
        lens.append(int(ctx[r]) + int(new[r]) if ok else 0)
        held_out.append(need[r] if ok else int(held[r]))
        for i in range(int(new[r])):
            if end + i < tokens:
                pos = int(ctx[r]) + i
                at[end + i] = pos
                if ok:
                    slots[end + i] = int(table[r, pos // page]) * page + pos % page
        end += int(new[r])
        starts.append(min(end, tokens))
    u = lambda v: np.asarray(v, np.uint32)  # noqa: E731
    return {"free": free, "table": table, "held_out": u(held_out), "free_out": u([left, refused, placed, used]), "starts": u(starts), "lens": u(lens),
            "slots": slots, "at": at}


def rows_of(table_row, n, page):
    t = np.arange(n)
    return table_row[t // page].astype(np.int64) * page + t % page


def attend(q, pool_k, exps_k, pool_v, exps_v, table, lens, starts, page, window, group, scale):
    """(out, bound): out in 64 bits, and how far an f16 result may be from it.

    Weights enter the second product in f16: each is off by at most 2^-11 of itself, or by 2^-25 of the largest where they are below f16's
    normal range (`tiny`; weights carry their tile's scale there, or not: the larger counts).  The result is rounded to f16: 2^-11 of itself.  Scores are sums of 128 exact products in f32,
    cut to 2^-23 of what they reach each time (`skew`), scaled with a rounding and raised by an exponential good to 2^-22; sums of weights and results add 2^-22 for each 16-token tile."""
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    for r in range(len(lens)):
        first, m, n = int(starts[r]), int(starts[r + 1] - starts[r]), int(lens[r])
        if m == 0 or n == 0:
            continue
        rows = rows_of(table[r], n, page)
        b, i = rows // TILE, rows % TILE
        pos = n - m + np.arange(m)[:, None]
        t = np.arange(n)[None, :]
        seen = (t <= pos) & ((t > pos - window) if window else True)
        for h in range(pool_k.shape[1]):
            k = E4M3[pool_k[b, h, i]] * 2.0 ** exps_k[b, h].astype(np.float64)[:, None]
            vq, ve = E4M3[pool_v[b, h, i]], 2.0 ** exps_v[b, h].astype(np.float64)
            v = vq * ve[:, None]
            for j in range(h * group, (h + 1) * group):
                x = q[first:first + m, j].astype(np.float64)
                s = np.where(seen, x @ k.T * scale, -np.inf)
                big = s.max(-1, keepdims=True)
                p = np.where(seen, np.exp(s - np.where(np.isfinite(big), big, 0.0)), 0.0)
                den = p.sum(-1, keepdims=True)
                live = den > 0
                den = np.where(live, den, 1.0)
                o = p @ v / den
                spread = p @ np.abs(v) / den
                reach = np.where(seen, np.abs(x) @ np.abs(k).T * scale, 0.0).max(-1, keepdims=True)
                skew = 128 * 2.0 ** -23 * reach + 2.0 ** -22 * (2 + n / TILE)
                tiny = 2.0 ** -25 * np.maximum((p * ve).max(-1, keepdims=True) * (seen @ np.abs(vq)), seen @ np.abs(v)) / den
                out[first:first + m, j] = np.where(live, o, 0.0)
                bound[first:first + m, j] = np.where(live, 2.0 ** -11 * (spread + np.abs(o)) * 1.01 + 2 * skew * spread + tiny + 2.0 ** -25, 0.0)
    return out, bound
