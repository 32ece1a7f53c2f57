"""GPU tests of the batched cache's attention against bounds that an output of zeros, or of another sign, misses.

``bound`` weighs what each key's score may be off by with that key's own weight, and counts f16 weights from the largest one that a row
has: they stand 2^7 above one where a row's maximum is found, so what f16's subnormal grid (2^-25, half a step) takes from a weight is at
most 2^-32 of the largest."""
import numpy as np
import pytest

import blocks_ref as ref
from test_gpu_blocks import Batch, D, SCALE, TILE, ctx  # noqa: F401

pytestmark = pytest.mark.gpu


def attend(b, window=0, scale=SCALE):
    """(out, bound) in 64 bits.  A score is off by 2^-23 of what its sum reaches for each of 128 products, by 2^-21 of itself, of the maximum
    and of the powers of two that are added to it (16 is more than those are in base e) for scaling, exponential and maximum; sums and rescaling by
    2^-21 for each tile of 16 keys; a weight by 2^-11 of itself or 2^-32 of the largest; the result by 2^-11 of itself or 2^-25."""
    out, bound = np.zeros(b.q.shape), np.zeros(b.q.shape)
    for r, n in enumerate(map(int, b.lens)):
        first, m = int(b.starts[r]), int(b.starts[r + 1] - b.starts[r])
        if m == 0 or n == 0:
            continue
        rows = ref.rows_of(b.table[r], n, b.page)
        blk, i = rows // TILE, rows % TILE
        pos, t = n - m + np.arange(m)[:, None], np.arange(n)[None, :]
        seen = (t <= pos) & ((t > pos - window) if window else True)
        for h in range(b.kv):
            k = ref.E4M3[b.kp[blk, h, i]] * 2.0 ** b.ke[blk, h].astype(np.float64)[:, None]
            vq, ve = ref.E4M3[b.vp[blk, h, i]], 2.0 ** b.ve[blk, h].astype(np.float64)
            v = vq * ve[:, None]
            for j in range(h * b.group, (h + 1) * b.group):
                x = b.q[first:first + m, j].astype(np.float64)
                s = np.where(seen, x @ k.T * scale, -np.inf)
                big = np.where(seen.any(-1, keepdims=True), s.max(-1, keepdims=True), 0.0)
                p = np.where(seen, np.exp(s - big), 0.0)
                live = p.sum(-1, keepdims=True) > 0
                den = np.where(live, p.sum(-1, keepdims=True), 1.0)
                o, spread = p @ v / den, p @ np.abs(v) / den
                off = 128 * 2.0 ** -23 * (np.abs(x) @ np.abs(k).T * scale) + 2.0 ** -21 * (np.abs(np.where(seen, s, 0.0)) + np.abs(big) + 16)
                off = p * np.expm1(off) + 2.0 ** -21 * (n / TILE) * p
                lost = 2.0 ** -11 * spread + 1.01 * 2.0 ** -32 * (p * ve).max(-1, keepdims=True) * (seen @ np.abs(vq)) / den
                d = (off @ np.abs(v) + off.sum(-1, keepdims=True) * np.abs(o)) / den + lost
                out[first:first + m, j] = np.where(live, o, 0.0)
                bound[first:first + m, j] = np.where(live, d + 2.0 ** -11 * (np.abs(o) + d) + 2.0 ** -25, 0.0)
    return out, bound


def run(ctx, b, window=0, scale=SCALE):  # noqa: F811
    (_, *rest), grid = b.call(window)
    ctx.dispatch_blocking(ctx.load_kernel("attn_blocks_e4m3_d128"), b.buffers(ctx), (scale, *rest), grid)
    return b.out.read().view(np.float16).reshape(b.q.shape).astype(np.float64)


def check(ctx, b, window=0, scale=SCALE, counts=None):  # noqa: F811
    """Within the bound, which on nearly all elements (of `counts`) excludes zero, and so any value of the other sign."""
    want, bound = attend(b, window, scale)
    n = int(b.starts[-1])
    told = (np.abs(want) > bound)[:n][..., counts if counts is not None else slice(None)]
    assert told.mean() > 0.9, f"the bound excludes zero on {told.mean()} of the elements"
    got = run(ctx, b, window, scale)[:n]
    assert np.isfinite(got).all()
    over = np.abs(got - want[:n]) - bound[:n]
    assert over.max() <= 0, f"{over.max()} beyond the bound at {np.unravel_index(over.argmax(), over.shape)}"


def _outliers(b, dims):
    """V's tiles at the least exponents, all values of one sign, but every fifth tile, which is 0 but for a few dims of the largest values."""
    for r, n in enumerate(map(int, b.lens)):
        rows = ref.rows_of(b.table[r], n, b.page)
        blocks = np.unique(rows // TILE)
        b.ve[blocks] = b.rng.integers(-15, -12, (len(blocks), b.kv))
        b.vp[rows // TILE, :, rows % TILE] = b.rng.integers(0x50, 0x7F, (n, b.kv, D))  # 8 to 448
        large = blocks[2::5]
        b.ve[large] = 3
        at = np.isin(rows // TILE, large)
        b.vp[rows[at] // TILE, :, rows[at] % TILE, dims:] = 0
    return b


@pytest.mark.parametrize("lens,new,kv,group", [
    ([9000, 300, 5000], [1, 1, 1], 16, 1), ([9000, 300, 5000], [1, 1, 1], 16, 4), ([9000, 300, 5000], [4, 1, 3], 16, 2),
    ([9000, 300, 5000], [8, 5, 1], 16, 2), ([9000, 40, 5000], [16, 9, 1], 16, 1), ([700, 333], [130, 70], 2, 2), ([700, 9000], [300, 40], 2, 1)])
def test_values_beside_tiles_of_much_larger_scale(ctx, lens, new, kv, group):  # noqa: F811
    """Dims in which the tiles of the largest scale hold nothing keep what the others hold: their weights are 2^-16 to 2^-18 of the largest."""
    check(ctx, _outliers(Batch(1, lens, new, kv, group, 32), 8))


def _nan_at(b, r, tokens, side, share):
    """NaNs of either sign in tokens of a request: in a share of V's dims, or in all of K's."""
    rows = ref.rows_of(b.table[r], int(b.lens[r]), b.page)[np.asarray(tokens)]
    pool = b.vp if side == "v" else b.kp
    at = b.rng.random((len(rows), b.kv, D)) < share
    codes = pool[rows // TILE, :, rows % TILE]
    pool[rows // TILE, :, rows % TILE] = np.where(at, b.rng.choice([0x7F, 0xFF], at.shape), codes)


@pytest.mark.parametrize("side", ["v", "k"])
@pytest.mark.parametrize("window", [0, 3, 40])
@pytest.mark.parametrize("lens,new,kv,group", [
    ([4, 50, 1037, 21], [4, 4, 2, 3], 3, 2), ([8, 50, 1037, 23], [8, 7, 8, 1], 2, 1), ([8, 50, 4037, 23], [8, 7, 8, 2], 3, 2), ([16, 50, 1037, 21], [16, 9, 13, 1], 2, 1),
    ([70, 100, 900, 65], [70, 33, 64, 1], 2, 1), ([300, 333, 1000, 64], [300, 129, 200, 3], 2, 2), ([5000, 200, 1300, 60], [300, 40, 31, 40], 2, 4)])
def test_nan_reaches_the_rows_that_see_it(ctx, lens, new, kv, group, window, side):  # noqa: F811
    """A NaN in a token's value is in the results of the rows that see that token, in its dims; one in a key in all dims of those rows.  The
    rows before it, and those whose window has passed it, are as they would be without."""
    b = Batch(7, lens, new, kv, group, 16, spare_rows=2)
    clean = b.kp.copy(), b.vp.copy()
    tokens = []
    for r, (n, m) in enumerate(zip(lens, new)):
        t = {n - 1, n - m, n - 1 - m // 2, max(0, n - m - 2), max(0, n - max(window, 1) - m // 3)} if r != 2 else {n - 1, max(0, n - m - window + 1)}
        tokens.append(sorted(t))
        _nan_at(b, r, tokens[r], side, 0.3 if side == "v" else 1.0)
    poisoned = b.vp if side == "v" else b.kp
    nan = np.zeros(b.q.shape, bool)
    for r, (n, m) in enumerate(zip(lens, new)):
        rows = ref.rows_of(b.table[r], n, b.page)[tokens[r]]
        pos, t = n - m + np.arange(m)[:, None], np.array(tokens[r])[None, :]
        seen = (t <= pos) & ((t > pos - window) if window else True)
        codes = (poisoned[rows // TILE, :, rows % TILE] & 127) == 127  # [token, kv, dim]
        hit = np.einsum("mt,thd->mhd", seen.astype(int), codes) > 0
        nan[int(b.starts[r]):int(b.starts[r]) + m] = np.repeat(hit, group, 1)
    got = run(ctx, b, window)
    n = int(b.starts[-1])
    (b.kp, b.vp), poison = clean, (b.kp, b.vp)
    want, bound = attend(b, window)
    wrong = np.isnan(got[:n]) != nan[:n]
    assert not wrong.any(), f"{wrong.sum()} of {wrong.size}, {nan[:n].sum()} are NaN; first at {np.argwhere(wrong)[0].tolist()}"
    assert (np.abs(got - want)[:n][~nan[:n]] <= bound[:n][~nan[:n]]).all()


@pytest.mark.parametrize("scale", [1.5e-45, 1e-43, 1e-38, 1e-20])
def test_scales_that_make_all_weights_equal(ctx, scale):  # noqa: F811
    for new in ([1, 3, 1], [8, 5, 1], [70, 200, 1]):
        b = Batch(3, [max(n, m) for n, m in zip([90, 200, 1000], new)], new, 2, 2, 16)
        b.ke[b.ke != 127] = -15
        scale = float(np.float32(scale))
        want, bound = attend(b, 40, scale)
        got = run(ctx, b, 40, scale)
        assert np.isfinite(got).all() and (np.abs(got - want) <= bound).all()
