"""GPU tests of the batched cache's attention and append against bounds that an output of zeros, or of another sign, misses.

``bound`` weighs what each key's score may be off by with that key's own weight, and counts f16 weights from the largest one that a row
has: they stand 2^7 above one where a row's maximum is found, so what f16's subnormal grid (2^-25, half a step) takes from a weight is at
most 2^-32 of the largest."""
import numpy as np
import pytest

import blocks_ref as ref
from test_gpu_blocks import Batch, D, SCALE, TILE, _pool, _run_append, ctx  # noqa: F401

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


def _peaked(b, q):
    """Scores of deviation 10 and more: few keys carry a row."""
    b.q = (b.q * np.float16(q)).astype(np.float16)
    return b


@pytest.mark.parametrize("lens,new,kv,group", [([500, 33, 2000], [1, 4, 1], 2, 2), ([500, 2000, 35], [16, 16, 1], 2, 1), ([500, 2000, 35], [8, 7, 1], 2, 2),
                                               ([500, 233, 3000], [130, 70, 300], 2, 2), ([500, 233], [130, 70], 2, 8)])
@pytest.mark.parametrize("window", [0, 100])
def test_peaked_softmaxes(ctx, lens, new, kv, group, window):  # noqa: F811
    check(ctx, _peaked(Batch(2, lens, new, kv, group, 32), 4), window)


@pytest.mark.parametrize("lens,new,kv,group", [([500, 33, 2000], [1, 4, 1], 2, 2), ([500, 2000, 35], [16, 16, 1], 2, 1), ([500, 2000, 35], [4, 4, 1], 2, 4),
                                               ([500, 233, 3000], [130, 70, 300], 2, 2), ([500, 233], [130, 70], 2, 8)])
def test_values_of_all_scales(ctx, lens, new, kv, group):  # noqa: F811
    """V's exponents anywhere between the ends of the format."""
    b = Batch(4, lens, new, kv, group, 32)
    real = b.ve != 127
    b.ve[real] = b.rng.integers(-15, 8, int(real.sum()))
    check(ctx, b)


def test_more_units_than_are_sorted(ctx):  # noqa: F811
    """Over 2048 units a head, over 1024 requests: units stand in the requests' order.  Requests of no token, of one, and refused ones between them."""
    rng = np.random.default_rng(21)
    requests = 2600
    new = rng.integers(9, 18, requests)
    new[rng.random(requests) < 0.1] = 1
    new[rng.random(requests) < 0.05] = 0
    new[[700, 1900]] = 300, 513  # several units each
    lens = np.maximum(new + rng.integers(0, 40, requests), 1)
    dead = set(np.flatnonzero(rng.random(requests) < 0.03).tolist()) - {700, 1900}
    assert sum(-(-int(m) // 256) for m in new if m > 8) > 2048
    check(ctx, Batch(21, lens, new, 3, 1, 16, spare_rows=3, dead=dead))


@pytest.mark.parametrize("many", [False, True])
def test_heads_whose_units_stand_together(ctx, many):  # noqa: F811
    """Prompts whose keys and values are more than 96 MiB: a head's units follow each other.  Every unit is cut, or most are whole items and more than
    are sorted."""
    kv = 16
    lens, new = [25700, 700, 40], [72, 1, 40]
    if many:
        rng = np.random.default_rng(22)
        new = np.concatenate([rng.integers(9, 12, 2100), new])
        lens = np.concatenate([new[:-3] + rng.integers(0, 20, 2100), lens])
    assert sum(int(n) // 1024 for n, m in zip(lens, new) if m > 8) * 1024 * kv * 2 * D > 96 << 20
    check(ctx, Batch(22, lens, new, kv, 1, 64, spare_rows=1, dead=(5, 9) if many else ()))


def test_append_of_nan_and_infinity_keeps_the_rest_of_the_tile(ctx):  # noqa: F811
    """Rows before the run are rounded again for the exponent that infinity calls for, rows behind it are left."""
    for kv, first, n in ((1, 4, 2), (3, 0, 5), (3, 9, 7), (2, 15, 1)):
        rng = np.random.default_rng(first)
        k, v = (rng.standard_normal((n, kv, D)).astype(np.float16) for _ in range(2))
        k[0, 0, :4] = [np.nan, np.inf, -np.inf, 65504]
        v[-1, -1, 5:8] = [-np.inf, -np.nan, 1]
        pools = [*_pool(1, 3, kv), *_pool(2, 3, kv)]
        for p in pools[::2]:
            p[1, 0, 0, 0] = 0x7F  # one that was there
        slots = np.arange(n) + TILE + first
        got = _run_append(ctx, k, v, slots, pools, kv)
        ref.append(k, slots, *pools[:2])
        ref.append(v, slots, *pools[2:])
        for g, w in zip(got, pools):
            if g.dtype == np.uint8:  # a NaN's sign is nobody's
                g, w = np.where((g & 127) == 127, 0x7F, g), np.where((w & 127) == 127, 0x7F, w)
            assert np.array_equal(g, w)
