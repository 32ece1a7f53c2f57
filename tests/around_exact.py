"""Statements of what stands around the batched attention that are independent of ``around_ref``: whole-number angles, complex rotations, bounds counted
from the kernels' own operations.

U = 2^-24 is what one rounding to f32 is off by, relative to its result."""
import numpy as np

import blocks_ref as ref

U = 2.0 ** -24
D = ref.D


# ---- keys of the pre-attention pass --------------------------------------------------------------------------------------------------
def pairs_of(pairs, layout, head_dim=D):
    return [((i, i + head_dim // 2), (i, i + pairs), (2 * i, 2 * i + 1))[layout] for i in range(pairs)]


def keys(k, w, rows, layout):
    """k [tokens, heads, 128] f16, w of 64 bits, rows [tokens, pairs, 2] f32: (keys before they are rounded, how far the kernel's f32 may be from them).
    A lane sums two times eight squares, their two sums, three steps over the row's lanes: 12 roundings of a sum of squares, its mean and eps one, which
    the root halves; the root itself 2 units in the last place (4 U), a weight 1 + w, its product with c or s, that with the value, a sum, the
    root's product: 16 in all on each product."""
    x = k.astype(np.float64)
    x = x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-6) * w
    out, size = x.copy(), np.abs(x)
    for i, (a, b) in enumerate(pairs_of(rows.shape[1], layout)):
        turn = rows[:, None, i, 0].astype(np.float64) + 1j * rows[:, None, i, 1].astype(np.float64)
        z = (x[..., a] + 1j * x[..., b]) * turn
        out[..., a], out[..., b] = z.real, z.imag
        size[..., a] = np.abs(x[..., a] * turn.real) + np.abs(x[..., b] * turn.imag)
        size[..., b] = np.abs(x[..., b] * turn.real) + np.abs(x[..., a] * turn.imag)
    return out, size * 16 * U


def key_exponent(w, magnitude, rot):
    """The least e >= -15 with 448 * 2^e at or above 11.336 max|w| times the rows' length, or times 1 where that is more and dims stay that do not turn."""
    reach = 11.336 * float(np.abs(w).max()) * (magnitude if rot == D else max(magnitude, 1.0))
    return max(-15, int(np.ceil(np.log2(min(reach, 61440.0) / 448.0)))) if reach else -15


# ---- angles --------------------------------------------------------------------------------------------------------------------------
BITS = 192


def _inverse_two_pi():
    """2^BITS / 2 pi in whole numbers: pi = 16 atan(1/5) - 4 atan(1/239)."""
    def atan_inverse(n):
        total, term, k = 0, (1 << (BITS + 80)) // n, 1
        while term:
            total += term // k if k % 4 == 1 else -(term // k)
            term //= n * n
            k += 2
        return total

    pi = 16 * atan_inverse(5) - 4 * atan_inverse(239)
    return (1 << (2 * BITS + 80)) // (2 * pi)


def cos_sin(positions, freqs, magnitude):
    """([tokens, pairs, 2], bounds): cosines and sines whose angles are whole numbers of 2^-192 turns, so that small sines keep their digits.
    The kernel's angle x, at most an eighth of a turn: its frequency is off by 2^-64 turns at most, times the position; it is cut below 2^-55 turns; converting it, a sum, the
    factor 2 pi 2^-32 (itself 0.47 U off) and that product are four roundings.  A sine of it: x by one fma, the series' rest (a tenth of it at most) by
    five more, cut off below 2.3e-9 of it (0.04 U), times the magnitude: 3 U of its value.  A cosine: half of the rest's 3.5 U times x^2 (0.62 at most) and an fma: 2.5 U, and the magnitude's."""
    inverse, one, m = _inverse_two_pi(), 1 << BITS, float(np.float32(magnitude))
    out, bound = np.empty((len(positions), len(freqs), 2)), np.empty((len(positions), len(freqs), 2))
    for j, f in enumerate(freqs):
        numerator, denominator = float(f).as_integer_ratio()
        step = numerator * inverse // denominator
        for i, p in enumerate(positions):
            turn = int(p) * step % one
            quarter = (turn + one // 8) * 4 // one
            x = 2 * np.pi * (float(turn - quarter * (one // 4)) / one)
            c, s = np.cos(x), np.sin(x)
            out[i, j] = [(c, s), (-s, c), (-c, -s), (s, -c)][quarter % 4]
            dx = abs(x) * 4.5 * U + 2 * np.pi * (abs(int(p)) * 2.0 ** -64 + 2.0 ** -55)
            off = (2.5 * U + U * c + abs(s) * dx, 3 * U * abs(s) + c * dx)
            bound[i, j] = off if quarter % 2 == 0 else off[::-1]
    return m * out, m * bound * 1.001


# ---- norms around a block --------------------------------------------------------------------------------------------------------------
INV_RMS = (24 + 1 + 5 + 2 + 4 + 3) / 2 + 4  # roundings of 1 / rms: see below


def block_norms(y, h, w_post, gate, w_pre, post, scale, eps):
    """(h', its error, x, its error), errors before the last rounding; weights as they multiply (1 + w added up), gate an array that broadcasts or None.
    A lane sums at most 24 squares one after the other (six units of eight values in two halves; eight units of four are 16), its halves, five steps over a warp, a
    row's warps in four groups of four (two and four), times 1 / hidden (rounded), plus eps: the root halves those 39 and is itself 2 units in the last
    place off.  y by its weight, gate and 1 / rms: four more.  h' takes two, x three."""
    h = h.astype(np.float64)
    out, err = h, np.zeros_like(h)
    if post != 2:
        n = y.astype(np.float64)
        if post == 1:
            n = n * (1 / np.sqrt(np.mean(n ** 2, -1, keepdims=True) + eps)) * w_post
        if gate is not None:
            n = gate * n
        out = scale * (h + n)
        err = abs(scale) * np.abs(n) * ((INV_RMS if post == 1 else 0) + 4) * U + 2 * U * np.abs(out)
    inverse = 1 / np.sqrt(np.mean(out ** 2, -1, keepdims=True) + eps)
    off = np.sqrt(np.mean(err ** 2, -1, keepdims=True)) * inverse
    x = out * inverse * w_pre
    return out, err * 1.001, x, (np.abs(x) * ((INV_RMS + 3) * U + off) + err * inverse * np.abs(w_pre)) * 1.001
