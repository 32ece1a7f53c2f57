"""Plain statements, in 64 bits, of what stands around the batched attention, each with how far its kernel may be from it.

The kernels compute in f32 (a rounding is off by at most U = 2^-24 of its result) and round once at the end: f16 by 2^-11 of the value or
2^-25 (half its grid near zero), bf16 by 2^-8, e4m3 by whatever ``blocks_ref.encode`` says of any value within the f32 error."""
import numpy as np

import blocks_ref as ref

U = 2.0 ** -24
REACH = np.float32(11.336)
D, TILE, NONE = ref.D, ref.TILE, ref.NONE


def f16_step(x):
    return 2.0 ** -11 * np.abs(x) + 2.0 ** -25


def frequencies(pairs, theta, dims, kind="plain", factor=1.0, trained=0.0, slow=1.0, fast=32.0):
    i = np.arange(pairs)
    f = theta ** (-2.0 * i / dims)
    turns = trained * f / (2 * np.pi)
    if kind == "plain":
        return f
    if kind == "linear":
        return f / factor
    if kind == "by_turns":
        keep = np.clip((turns - slow) / (fast - slow), 0, 1)
    else:
        at = [dims * np.log(trained / (t * 2 * np.pi)) / (2 * np.log(theta)) for t in (fast, slow)]
        lo, hi = max(np.floor(at[0]), 0.0), min(np.ceil(at[1]), dims - 1.0)
        keep = 1 - np.clip((i - lo) / (hi - lo), 0, 1) if hi > lo else np.where(i > lo, 0.0, 1.0)
    return keep * f + (1 - keep) * f / factor


def cos_sin(positions, freqs, magnitude):
    """Rows of cosines and sines from 80-bit angles (an f64 product of a position of 31 bits is off by 2^-22).  The kernel's angle is off by half a step of an f32 number of turns up to
    one half (2^-26), its sine and cosine by two units in the last place of 1, the product with the magnitude by one rounding."""
    turns = np.asarray(positions, np.longdouble)[:, None] * np.asarray(freqs, np.longdouble) / (2 * np.longdouble("3.14159265358979323846264338327950288"))
    a = ((turns - np.rint(turns)) * 2 * np.longdouble("3.14159265358979323846264338327950288")).astype(np.float64)
    m = float(np.float32(magnitude))
    return np.stack([m * np.cos(a), m * np.sin(a)], -1), m * (2 * np.pi * 2.0 ** -26 + 2 * 2.0 ** -23 + U) * 1.01


def pair_dims(head_dim, pairs, layout):
    i = np.arange(pairs)
    return (i, i + head_dim // 2) if layout == 0 else (i, i + pairs) if layout == 1 else (2 * i, 2 * i + 1)


def turn(x, rows, layout, rel=0.0):
    """x [tokens, heads, dims] (its values known to `rel` of them) turned by rows [tokens, pairs, 2] of f32: (out, f32 error)."""
    a, b = pair_dims(x.shape[-1], rows.shape[1], layout)
    c, s = (rows[:, None, :, j].astype(np.float64) for j in (0, 1))
    out, err = x.astype(np.float64).copy(), rel * np.abs(x)
    xa, xb = x[..., a].astype(np.float64), x[..., b].astype(np.float64)
    out[..., a], out[..., b] = xa * c - xb * s, xb * c + xa * s
    err[..., a] = (np.abs(xa * c) + np.abs(xb * s)) * (rel + 3 * U)  # two products and a sum
    err[..., b] = (np.abs(xb * c) + np.abs(xa * s)) * (rel + 3 * U)
    return out, err


def norm_weight(w, plus_one):
    w = np.asarray(w, np.float32)
    return (w + np.float32(1)) if plus_one else w


# A row of 128: 16 products summed a lane, then four sums; the mean, eps, a reciprocal root of two units: all that relative to the sum of squares counts half but the root.
NORM_REL = ((16 + 1 + 3 + 2) / 2 + 2 * 2 + 2 + 1) * U


def norm128(x, w):
    x = x.astype(np.float64)
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-6)
    return y if w is None else y * w.astype(np.float64)


def exponents(k_w, magnitude):
    """(e of keys, e of values) that the norms' bounds give."""
    most = np.max(np.abs(k_w)) * REACH * np.float32(magnitude)
    return ref.exponent(min(float(most), ref.LARGEST)), ref.exponent(float(REACH))


def append_normed(z, err, slots, pool, exps, least):
    """Values z [n, KV, 128] into a copy of the tiles: (lowest codes, highest codes, exponents): each code lies between the two, as values."""
    lo, hi, exps = pool.copy(), pool.copy(), exps.copy()
    i, n = 0, len(slots)
    while i < n:
        if slots[i] == NONE:
            i += 1
            continue
        j = i + 1
        while j < n and slots[j] == slots[j - 1] + 1 and slots[j] % TILE:
            j += 1
        b, at = slots[i] // TILE, int(slots[i] % TILE)
        for h in range(z.shape[1]):
            e = least
            if at:
                old = int(exps[b, h])
                e = max(least, old)
                if e > old:
                    codes = pool[b, h, :at]
                    again = np.where((codes & 127) == 127, codes, ref.encode(ref.E4M3[codes] * 2.0 ** (old - e)))
                    lo[b, h, :at], hi[b, h, :at] = again, again
            exps[b, h] = e
            v, d = z[i:j, h], err[i:j, h]
            cut = lambda x: np.clip(x, -ref.LARGEST, ref.LARGEST) * 2.0 ** -e  # noqa: E731
            lo[b, h, at:at + j - i], hi[b, h, at:at + j - i] = ref.encode(cut(v - d)), ref.encode(cut(v + d))
        i = j
    return lo, hi, exps


def between(codes, lo, hi):
    """Whether codes stand for values between those of lo and hi (a NaN only for a NaN)."""
    v, a, b = ref.E4M3[codes], ref.E4M3[lo], ref.E4M3[hi]
    return np.where(np.isnan(a), np.isnan(v), (v >= a) & (v <= b))


def block_norms(y, h, w_post, gate, w_pre, post, scale, eps):
    """gate: an array that broadcasts over [rows, hidden], or None.  (h', error, x, error), both errors before the final rounding.  A row's sum of squares takes at most 16 units a lane of
    eight products, ten butterfly steps; a mean, eps, a root of two units; weights 1 + w, their product, the gate's."""
    rel = ((128 + 10 + 3) / 2 + 4 + 4) * U
    h = h.astype(np.float64)
    if post == 2:
        out, err = h, np.zeros_like(h)
    else:
        n = y.astype(np.float64)
        if post:
            n = n / np.sqrt((n * n).mean(-1, keepdims=True) + eps) * w_post.astype(np.float64)
        if gate is not None:
            n = n * gate.astype(np.float64)
        out = (h + n) * scale
        err = (np.abs(n) * rel + (np.abs(h) + np.abs(n)) * 2 * U) * abs(scale)
    rms = np.sqrt((out * out).mean(-1, keepdims=True) + eps)
    x = out / rms * w_pre.astype(np.float64)
    off = np.sqrt((err * err).mean(-1, keepdims=True)) / rms  # of the root
    return out, err, x, err / rms * np.abs(w_pre) + np.abs(x) * (rel + off)


def read(pool, exps, table, first, starts, page, tokens):
    """f16 rows [tokens, KV, 128]; rows that no request has are NaN."""
    out = np.full((tokens,) + (pool.shape[1], D), np.nan, np.float64)
    for r in range(len(first)):
        t = np.arange(int(first[r]), int(first[r]) + int(starts[r + 1]) - int(starts[r]))
        rows = table[r, t // page].astype(np.int64) * page + t % page
        out[starts[r]:starts[r + 1]] = ref.E4M3[pool[rows // TILE, :, rows % TILE]] * 2.0 ** exps[rows // TILE].astype(np.float64)[:, :, None]
    return out
