"""GPU tests of what stands around the batched attention: angles, rotation, norms with the append, norms around a block, reading the cache
back, and all of them with the tables and the attention as a server runs them.

Results are held to bounds that ``around_ref`` derives from where the kernels round; placement, exponents and what is read back are exact.
What no token owns is poison and has to stay."""
import numpy as np
import pytest
import torch

import around_ref as around
import blocks_ref as ref
from cases import bind

pytestmark = pytest.mark.gpu
NONE, TILE, D = ref.NONE, ref.TILE, ref.D


@pytest.fixture(scope="module")
def ctx():
    import super_gemma_b200 as sg

    return sg.GpuContext(0)


def _u32(v):
    return np.asarray(v).astype(np.int64).astype(np.uint32)


def _within(got, want, bound, what=""):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    assert got.shape == want.shape, what
    assert np.array_equal(np.isnan(got), np.isnan(want)), f"{what}: NaN in other places"
    over = np.where(np.isnan(want), -1.0, np.abs(got - want) - bound)
    assert over.max(initial=-1) <= 0, f"{what}: {over.max()} beyond the bound at {np.unravel_index(over.argmax(), over.shape)}"


# ---- rows of cosines and sines -----------------------------------------------------------------------------------------------------
def _angles(ctx, freqs, positions, magnitude, spare=3):
    rot, n = 2 * len(freqs), len(positions)
    out = ctx.buffer_from_iter(np.full((n + spare) * rot, 7.5, np.float32))
    ctx.dispatch_blocking(ctx.load_kernel("rope_cos_sin"), bind(ctx.buffer_from_iter(freqs), ctx.buffer_from_iter(_u32(positions)), out), (rot, float(magnitude)), [n, 1, 1])
    got = out.read().reshape(n + spare, rot // 2, 2)
    assert (got[n:] == 7.5).all(), "rows behind the last token were written"
    return got[:n]


@pytest.mark.parametrize("rot", [16, 80, 128, 512, 1024])
@pytest.mark.parametrize("tokens", [1, 3, 64, 1000, 40011])
def test_angles(ctx, tokens, rot):
    if tokens * rot > 8_000_000:
        tokens = 8_000_000 // rot
    rng = np.random.default_rng(tokens + rot)
    for theta, far, magnitude in ((1e4, 131072, 1.0), (1e6, 1 << 31, 1.2079442)):
        positions = rng.integers(-far, far, tokens)
        positions[:4] = [far - 1, -far, 0, -1][:min(tokens, 4)]
        freqs = around.frequencies(rot // 2, theta, rot)
        want, bound = around.cos_sin(positions, freqs, magnitude)
        _within(_angles(ctx, freqs, positions, magnitude), want, bound, f"{theta} {far}")


def test_angles_of_frequencies_that_are_scaled(ctx):
    import super_gemma_b200 as sg

    freqs = sg.rope_frequencies(64, 1e4, kind="by_pairs", factor=16.0, trained=4096)
    positions = np.arange(60000, 66000)
    want, bound = around.cos_sin(positions, around.frequencies(64, 1e4, 128, "by_pairs", 16.0, 4096), 1.25)
    _within(_angles(ctx, freqs, positions, 1.25), want, bound + 2e-11 * 66000)  # the power's own rounding, times the position
    got = _angles(ctx, np.array([0.0, -0.5, np.inf, np.nan] + [1.0] * 4), [0, 3], 1.0)
    assert (got[:, 0] == [1, 0]).all() and np.isnan(got[1, 2:4]).all() and np.abs(got[1, 1] - [np.cos(1.5), -np.sin(1.5)]).max() < 4e-7


# ---- rotation ------------------------------------------------------------------------------------------------------------------------
def _rotate(ctx, q, k, rows, layout, gap=0, in_place=False, out_gap=0):
    """q, k [tokens, heads, dims] f16, `gap` values behind a token's heads (in one row with those of the other where it is not 0)."""
    n, d = q.shape[0], q.shape[2]
    heads = [q.shape[1], k.shape[1]]
    raw = [x.reshape(n, -1).view(np.uint16) for x in (q, k)]
    up = ctx.buffer_from_iter
    if gap:
        width = sum(heads) * d + gap
        whole = np.full((n, width), 0x3333, np.uint16)
        whole[:, :heads[0] * d], whole[:, heads[0] * d:sum(heads) * d] = raw
        wb = up(whole.reshape(-1))
        src, strides = [wb, wb.slice(heads[0] * d, n * width) if heads[1] else wb], [width, width]
    else:
        src, strides = [up(x.reshape(-1)) if x.size else up(np.zeros(8, np.uint16)) for x in raw], [0, 0]
    if in_place:
        dst, out_strides = src, strides
    else:
        out_strides = [h * d + out_gap for h in heads]
        dst = [up(np.full((n + 1) * max(8, s), 0x5555, np.uint16)) for s in out_strides]
    ctx.dispatch_blocking(ctx.load_kernel("rope_qk_f16"), bind(src[0], src[1], up(rows.reshape(-1)), dst[0], dst[1]),
                          (d, 2 * rows.shape[1], layout, *strides, *out_strides), [heads[0], heads[1], n])
    if in_place and gap:
        whole2 = wb.read().reshape(n, -1)
        assert (whole2[:, sum(heads) * d:] == 0x3333).all(), "values between the rows were written"
        got = [whole2[:, :heads[0] * d], whole2[:, heads[0] * d:sum(heads) * d]]
    elif in_place:
        got = [b.read()[:x.size].reshape(x.shape) for b, x in zip(dst, raw)]
    else:
        got = []
        for b, h, s in zip(dst, heads, out_strides):
            all_ = b.read()
            assert (all_[max(n * s, 0):] == 0x5555).all(), "rows behind the last token were written"
            rows_ = all_[:n * s].reshape(n, s)
            assert (rows_[:, h * d:] == 0x5555).all(), "values between the rows were written"
            got.append(rows_[:, :h * d])
    return [g.copy().view(np.float16).reshape(n, h, d) for g, h in zip(got, heads)]


HEADS = [(64, 64), (80, 80), (80, 32), (96, 48), (112, 112), (128, 128), (128, 64), (128, 16), (256, 256), (512, 128), (16, 16), (1024, 1024), (624, 304)]


@pytest.mark.parametrize("layout", [0, 1, 2])
@pytest.mark.parametrize("head_dim,rot", HEADS)
def test_rotation(ctx, head_dim, rot, layout):
    rng = np.random.default_rng(head_dim + rot + layout)
    for n, h, kv, gap, in_place, out_gap in ((1, 2, 1, 0, False, 0), (3, 5, 3, 24, True, 0), (67, 8, 2, 0, True, 0), (130, 7, 1, 8, False, 16), (5, 3, 0, 0, False, 8), (4, 3, 0, 8, True, 0)):
        q, k = ((rng.standard_normal((n, x, head_dim)) * 2.0 ** rng.integers(-18, 8, (n, x, 1))).astype(np.float16) for x in (h, kv))
        rows, _ = around.cos_sin(rng.integers(0, 100000, n), around.frequencies(rot // 2, 1e4, rot), 1.1)
        rows = rows.astype(np.float32)
        for name, x, got in zip("qk", (q, k), _rotate(ctx, q, k, rows, layout, gap, in_place, out_gap)):
            want, err = around.turn(x, rows, layout)
            still = np.setdiff1d(np.arange(head_dim), np.concatenate(around.pair_dims(head_dim, rot // 2, layout)))
            assert np.array_equal(got[..., still], x[..., still]), f"{name}: dims that do not turn, {(n, gap, in_place)}"
            _within(got, want, err + around.f16_step(want), f"{name} {(n, gap, in_place)}")


@pytest.mark.parametrize("tokens,heads,kv", [(9000, 8, 4), (30001, 2, 1), (257, 64, 64)])
def test_rotation_of_many_rows(ctx, tokens, heads, kv):
    rng = np.random.default_rng(tokens)
    q, k = (rng.standard_normal((tokens, x, 128)).astype(np.float16) for x in (heads, kv))
    rows = around.cos_sin(rng.integers(0, 100000, tokens), around.frequencies(64, 1e6, 128), 1.0)[0].astype(np.float32)
    for layout in (0, 2):
        for x, got in zip((q, k), _rotate(ctx, q, k, rows, layout, gap=8)):
            want, err = around.turn(x, rows, layout)
            _within(got, want, err + around.f16_step(want))


def test_rotation_of_infinities_and_nan(ctx):
    q = np.zeros((1, 1, 32), np.float16)
    q[0, 0, [0, 1, 18]] = [np.inf, np.nan, 65504]
    rows = np.zeros((1, 16, 2), np.float32)
    rows[..., 0] = 1.5
    got = _rotate(ctx, q, q, rows, 0)[0][0, 0]
    assert np.isinf(got[0]) and np.isnan(got[[1, 16, 17]]).all() and got[18] == np.inf and (np.delete(got, [0, 1, 16, 17, 18]) == 0).all()


def test_turning_back(ctx):
    """The rows of -p undo those of p."""
    rng = np.random.default_rng(4)
    q = rng.standard_normal((50, 4, 96)).astype(np.float16)
    p, freqs = rng.integers(0, 1 << 30, 50), around.frequencies(32, 1e4, 64)
    there, back = _angles(ctx, freqs, p, 1.0), _angles(ctx, freqs, -p, 1.0)
    once = _rotate(ctx, q, q, there, 1)[0]
    again = _rotate(ctx, once, once, back, 1)[0]
    pairs = np.hypot(q[..., :32].astype(np.float64), q[..., 32:64].astype(np.float64))
    _within(again, q, np.concatenate([pairs, pairs, np.zeros((50, 4, 32))], -1) * 2.0 ** -9 + 2.0 ** -23)  # two roundings to f16 of values no larger than the pair


def test_strides_beyond_32_bits(ctx):
    """Rows of 2^23 values: the last ones start beyond 2^32 bytes."""
    n, stride = 300, 1 << 23
    src = torch.zeros((n - 1) * stride + 256, dtype=torch.float16, device="cuda")
    x = torch.randn(n, 256, device="cuda").half()
    for t in range(n):
        src[t * stride:t * stride + 256] = x[t]
    torch.cuda.synchronize()
    rows = around.cos_sin(np.arange(n), around.frequencies(64, 1e4, 128), 1.0)[0].astype(np.float32)
    b = ctx.adopt(src.data_ptr(), src.numel() * 2, np.uint16, keep=src)
    out = [ctx.new_buffer(n * 128, np.uint16) for _ in range(2)]
    k = ctx.adopt(src.data_ptr() + 256, src.numel() * 2 - 256, np.uint16, keep=src)
    ctx.dispatch_blocking(ctx.load_kernel("rope_qk_f16"), bind(b, k, ctx.buffer_from_iter(rows.reshape(-1)), *out), (128, 128, 0, stride, stride, 0, 0), [1, 1, n])
    host = x.cpu().numpy()
    for i, o in enumerate(out):
        want, err = around.turn(host[:, None, 128 * i:128 * (i + 1)], rows, 0)
        _within(o.read().view(np.float16).reshape(n, 1, 128), want, err + around.f16_step(want))


# ---- norms, rotation and the append ----------------------------------------------------------------------------------------------------
def _pool(rng, blocks, kv, lo=-15, hi=9):
    codes = rng.integers(0, 256, (blocks, kv, TILE, D)).astype(np.uint8)
    return np.where((codes & 127) == 127, 0x11, codes).astype(np.uint8), rng.integers(lo, hi, (blocks, kv)).astype(np.int8)


class Step:
    """Packed tokens with their slots, weights and rows, over tiles that are all in use."""

    def __init__(self, seed, slots, heads, kv, blocks, rot=128, layout=0, plus_one=0, magnitude=1.0, packed=False, w_scale=1.0, exps=(-15, 9)):
        rng = np.random.default_rng(seed)
        n = len(slots)
        self.slots, self.heads, self.kv, self.blocks, self.n = np.asarray(slots, np.int64), heads, kv, blocks, n
        self.rot, self.layout, self.plus_one, self.magnitude, self.packed = rot, layout, plus_one, magnitude, packed
        self.q, self.k, self.v = ((rng.standard_normal((n, h, D)) * 2.0 ** rng.integers(-10, 10, (n, h, 1))).astype(np.float16) for h in (heads, kv, kv))
        self.q_w, self.k_w = ((w_scale * (1 - plus_one + 0.3 * rng.standard_normal(D))).astype(np.float32) for _ in range(2))
        self.rows = around.cos_sin(rng.integers(0, 100000, n), around.frequencies(rot // 2, 1e4, max(rot, 1)), magnitude)[0].astype(np.float32)
        self.pools = [*_pool(rng, blocks, kv, *exps), *_pool(rng, blocks, kv, *exps)]

    def buffers(self, ctx):
        up = ctx.buffer_from_iter
        if self.packed:
            gap = 8
            widths = [h * D for h in (self.heads, self.kv, self.kv)]
            whole = np.concatenate([x.reshape(self.n, -1).view(np.uint16) for x in (self.q, self.k, self.v)] + [np.full((self.n, gap), 0x7E00, np.uint16)], 1)
            self.whole = up(whole.reshape(-1))
            total = whole.size
            src = [self.whole, self.whole.slice(widths[0], total), self.whole.slice(widths[0] + widths[1], total)]
            self.strides = (sum(widths) + gap,) * 3
        else:
            src, self.strides = [up(x) for x in (self.q, self.k, self.v)], (0, 0, 0)
        self.q_out = up(np.full((self.n + 2) * self.heads * D, 0x5555, np.uint16))
        self.b = [up(p.reshape(-1)) for p in self.pools]
        rows = up(self.rows.reshape(-1)) if self.rot else up(np.zeros(4, np.float32))
        return bind(src[0], up(self.q_w), self.q_out, src[1], src[2], up(self.k_w), rows, up(_u32(self.slots)), *self.b)

    def call(self):
        return (self.rot, self.layout, self.plus_one, *self.strides, float(self.magnitude)), [self.heads, self.kv, self.n]

    def run(self, ctx):
        b = self.buffers(ctx)
        ctx.dispatch_blocking(ctx.load_kernel("qkv_norm_rope_append_blocks_e4m3_d128"), b, *self.call())
        self.check(what="run")
        return self

    def got(self):
        return [b.read().reshape(p.shape) for b, p in zip(self.b, self.pools)]

    def check(self, what=""):
        here = self.slots != NONE
        raw = self.q_out.read().reshape(self.n + 2, -1)
        assert (raw[:self.n][~here] == 0x5555).all() and (raw[self.n:] == 0x5555).all(), f"{what}: rows of tokens without a slot were written"
        q_w, k_w = (around.norm_weight(w, self.plus_one) for w in (self.q_w, self.k_w))
        want, err = around.turn(around.norm128(self.q, q_w), self.rows, self.layout, around.NORM_REL)
        _within(raw[:self.n][here].view(np.float16).reshape(-1, self.heads, D), want[here], (err + around.f16_step(want))[here], f"{what}: q")
        least = around.exponents(k_w, self.magnitude)
        z, err = around.turn(around.norm128(self.k, k_w), self.rows, self.layout, around.NORM_REL)
        y = around.norm128(self.v, None)
        got = self.got()
        for side, z, err, e, (pool, exps), (g, ge) in (("k", z, err, least[0], self.pools[:2], got[:2]), ("v", y, np.abs(y) * around.NORM_REL, least[1], self.pools[2:], got[2:])):
            lo, hi, we = around.append_normed(z, err, self.slots, pool, exps, e)
            assert np.array_equal(ge, we), f"{what}: exponents of {side}: {np.argwhere(ge != we)[:4].tolist()}"
            untouched = lo == hi
            ok = np.where(untouched, g == lo, around.between(g, lo, hi))
            assert ok.all(), f"{what}: {side} at {np.argwhere(~ok)[:4].tolist()}"


def _runs(seed, runs, blocks, pad):
    order = np.random.default_rng(seed).permutation(blocks)
    slots = [order[t // TILE] * TILE + t % TILE for t in (np.arange(first, first + n) for first, n in runs)]
    slots = np.concatenate(slots)
    return np.concatenate([[NONE], slots, [NONE] * 19]) if pad else slots


RUNS = [[(0, 1)], [(15, 1)], [(0, 16)], [(3, 13)], [(7, 60)], [(5, 3), (33, 1), (50, 30), (96, 16), (127, 1)], [(0, 200), (213, 11)]]


@pytest.mark.parametrize("heads,kv", [(1, 1), (6, 3), (32, 16), (5, 1), (16, 2)])
@pytest.mark.parametrize("runs", RUNS)
def test_pre_attention_matches_the_plain_statement(ctx, heads, kv, runs):
    for seed, more in enumerate(({}, {"layout": 2, "packed": True, "plus_one": 1}, {"rot": 64, "layout": 1, "magnitude": 1.3}, {"rot": 0}, {"rot": 48, "layout": 0, "packed": True})):
        Step(seed, _runs(seed, runs, 16, seed % 2), heads, kv, 16, **more).run(ctx)


@pytest.mark.parametrize("layout", [0, 1, 2])
@pytest.mark.parametrize("rot", [0, 16, 32, 48, 80, 112, 128])
def test_pre_attention_turns_part_of_the_head(ctx, rot, layout):
    Step(rot + layout, _runs(rot, [(5, 40)], 16, False), 4, 2, 16, rot=rot, layout=layout, plus_one=rot // 16 % 2).run(ctx)


@pytest.mark.parametrize("w_scale", [0.0, 1e-8, 1e-3, 30.0, 4000.0, 1e6])
def test_pre_attention_with_weights_of_all_sizes(ctx, w_scale):
    s = Step(int(np.log10(w_scale + 1e-9)) + 20, _runs(1, [(3, 9), (32, 20)], 8, False), 2, 2, 8, w_scale=w_scale)
    s.q_w[:] = 1.0  # (queries of such weights would not be f16 numbers)
    s.run(ctx)


@pytest.mark.parametrize("requests,heads,kv", [(5, 6, 3), (64, 32, 16), (700, 2, 2), (2500, 10, 5)])
def test_pre_attention_of_decode_steps(ctx, requests, heads, kv):
    """One token of each request, some with a draft of a few, at every place of a tile; a refused request now and then."""
    rng = np.random.default_rng(requests)
    run = np.where(rng.random(requests) < 0.1, rng.integers(2, 6, requests), 1)
    first, block = rng.integers(0, TILE, requests), rng.permutation(2 * requests)
    slots = np.concatenate([[block[2 * r + (first[r] + i) // TILE] * TILE + (first[r] + i) % TILE for i in range(run[r])] for r in range(requests)])
    slots[np.isin(np.repeat(np.arange(requests), run), np.arange(0, requests, 9))] = NONE
    for exps in ((-15, 9), (-6, -3)):
        Step(requests, slots, heads, kv, 2 * requests, exps=exps).run(ctx)


@pytest.mark.parametrize("tokens,heads,kv", [(1000, 4, 2), (4099, 2, 1), (3001, 16, 8)])
def test_pre_attention_of_prompts(ctx, tokens, heads, kv):
    blocks = tokens // TILE + 4
    Step(tokens, _runs(tokens, [(5, tokens)], blocks, True), heads, kv, blocks, packed=tokens == 4099, layout=tokens % 3).run(ctx)


@pytest.mark.parametrize("tokens,heads,kv", [(3, 130, 65), (2, 1500, 700), (2, 8192, 1024), (6000, 2, 1), (1500, 20, 5)])
def test_pre_attention_of_many_heads_and_of_few(ctx, tokens, heads, kv):
    """More rows a token than lanes share, and tokens enough that one group of lanes has all of a token's rows."""
    blocks = tokens // TILE + 3
    Step(tokens, _runs(tokens, [(15, tokens)], blocks, True), heads, kv, blocks, packed=heads != 20, layout=heads % 3, rot=(128, 96, 64)[heads % 3]).run(ctx)


def test_pre_attention_of_steps_with_room(ctx):
    """A step with room for many more tokens than it has: what is behind them is left, wherever the slots stand."""
    rng = np.random.default_rng(8)
    slots = np.full(3000, NONE, np.int64)
    slots[rng.choice(3000, 40, replace=False)] = rng.permutation(64)[:40] * TILE + rng.integers(0, TILE, 40)
    Step(8, slots, 4, 2, 64, packed=True).run(ctx)
    Step(8, np.full(70, NONE), 4, 2, 2).run(ctx)


def test_pre_attention_token_by_token(ctx):
    """A tile filled one token after another holds what one call for all of them writes, but for where it grew."""
    whole = Step(3, TILE + np.arange(TILE), 2, 2, 2).run(ctx)
    parts, pools = Step(3, TILE + np.arange(TILE), 2, 2, 2), None
    for t in range(TILE):
        one = Step(3, [TILE + t], 2, 2, 2)
        one.q, one.k, one.v, one.rows = (x[t:t + 1] for x in (parts.q, parts.k, parts.v, parts.rows))
        one.q_w, one.k_w = parts.q_w, parts.k_w
        one.pools = pools or parts.pools
        pools = one.run(ctx).got()
    assert all(np.array_equal(a, b) for a, b in zip(pools, whole.got()))


def test_pre_attention_with_nan_infinity_and_zeros(ctx):
    s = Step(9, [4, 5, 6, 7], 1, 1, 1)
    for x in (s.q, s.k, s.v):
        x[:] = 1
        x[0, 0, 3], x[1, 0, 3], x[2] = np.nan, np.inf, 0
    s.rows[:] = [1, 0]
    b = s.buffers(ctx)
    ctx.dispatch_blocking(ctx.load_kernel("qkv_norm_rope_append_blocks_e4m3_d128"), b, *s.call())
    q = s.q_out.read()[:4 * D].view(np.float16).reshape(4, D)
    kp, ke, vp, ve = s.got()
    for rows in (q, ref.E4M3[kp[0, 0, 4:8]], ref.E4M3[vp[0, 0, 4:8]]):
        assert np.isnan(rows[0]).all() and np.isnan(rows[1, 3]) and (np.delete(rows[1], [3, 67]) == 0).all() and (rows[2] == 0).all() and np.isfinite(rows[3]).all() and (rows[3] != 0).all()
    assert ve[0, 0] == max(-5, s.pools[3][0, 0])


def test_pre_attention_reports_slots_that_no_pool_has_or_no_order_allows(ctx):
    import super_gemma_b200 as sg

    for slots in ([0, 1, 64], [0, 5, 6], [3, 3, 17], [9, 8, 20], [1 << 31, 2, 3]):
        s = Step(1, slots, 2, 1, 4)
        b = s.buffers(ctx)
        with pytest.raises(sg.Bounds):
            ctx.dispatch_blocking(ctx.load_kernel("qkv_norm_rope_append_blocks_e4m3_d128"), b, *s.call())
        ctx.sync()
        got = s.got()
        used = {int(x) // TILE for x in slots}
        assert all(np.array_equal(g[i], p[i]) for g, p in zip(got, s.pools) for i in range(4) if i not in used), "another tile was written"
        assert (s.q_out.read().reshape(-1, 2 * D)[:3] != 0x5555).any(-1).all(), "a query is none of the cache's business"


def test_pre_attention_in_place(ctx):
    """q_out may be q."""
    s, t = (Step(5, _runs(5, [(2, 37)], 8, False), 3, 2, 8) for _ in range(2))
    s.run(ctx)
    b = t.buffers(ctx)
    b[2].buf = b[0].buf
    ctx.dispatch_blocking(ctx.load_kernel("qkv_norm_rope_append_blocks_e4m3_d128"), b, *t.call())
    assert np.array_equal(b[0].buf.read(), s.q_out.read()[:t.q.size]) and all(np.array_equal(x, y) for x, y in zip(s.got(), t.got()))


def test_pre_attention_and_read_beyond_32_bits(ctx):
    """A pool of more than 2^32 bytes a side: its last blocks are written, and read back."""
    kv, blocks = 16, (1 << 32) // (16 * 2048) + 70
    pools = [torch.zeros(blocks * kv * 2048, dtype=torch.uint8, device="cuda") for _ in range(2)]
    exps = [torch.zeros(blocks * kv, dtype=torch.int8, device="cuda") for _ in range(2)]
    torch.cuda.synchronize()
    first = (blocks - 64) // 4 * 64  # pages of 64
    slots = first + np.arange(150)
    s = Step(2, slots - first, 2, kv, 10)
    b = s.buffers(ctx)
    adopt = lambda t: ctx.adopt(t.data_ptr(), t.numel(), np.uint8, keep=t)  # noqa: E731
    big = [adopt(x) for x in (pools[0], exps[0], pools[1], exps[1])]
    for i, buf in enumerate(big):
        b[8 + i].buf = buf
    b[7].buf = ctx.buffer_from_iter(_u32(slots))
    k, push = ctx.load_kernel("qkv_norm_rope_append_blocks_e4m3_d128"), s.call()
    ctx.dispatch_blocking(k, b, *push)
    s.pools = [p * 0 for p in s.pools]
    block = first // TILE
    s.got = lambda: [t.view(blocks, -1)[block:block + 10].cpu().numpy().reshape(p.shape) for t, p in zip((pools[0], exps[0], pools[1], exps[1]), s.pools)]
    s.check("far")
    assert all(int(t.view(blocks, -1)[:block].any()) == 0 for t in pools)
    got = _read(ctx, big, np.array([[first // 64, first // 64 + 1, first // 64 + 2]]), [3], [0, 147], kv, 64, 147)
    kp, ke, vp, ve = s.got()
    table = np.array([[0, 1, 2]])
    for g, pool, e in zip(got, (kp, vp), (ke, ve)):
        padded = [np.concatenate([x, x[:2]]) for x in (pool, e)]
        assert np.array_equal(g.astype(np.float64), around.read(padded[0], padded[1], table, [3], [0, 147], 64, 147))


# ---- norms around a block ---------------------------------------------------------------------------------------------------------------
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
HALF_STEP = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": 2.0 ** -24}
TINY = {"f16": 2.0 ** -25, "bf16": 2.0 ** -134, "f32": 2.0 ** -150}


def _norms(ctx, kind, y, h, w_post, gate, w_pre, post, gates, plus_one=0, scale=1.0, eps=1e-6, in_place=False, spare=1):
    """Torch tensors on the device, [rows, hidden]; (h_out, x) with `spare` rows of poison behind them."""
    rows, hidden = h.shape
    h_out = torch.full((rows + spare, hidden), 3.0, dtype=h.dtype, device="cuda")
    x = torch.full((rows + spare, hidden), 3.0, dtype=torch.float16, device="cuda")
    if in_place:
        h_out[:rows], x[:rows] = h, y
        h, y = h_out, x
    torch.cuda.synchronize()
    adopt = lambda t: ctx.adopt(t.data_ptr(), t.numel() * t.element_size(), np.uint8, keep=t)  # noqa: E731
    b = {i: adopt(t) for i, t in enumerate((y, h, w_post, gate, w_pre, h_out, x))}
    if in_place:
        b[5], b[6] = b[1], b[0]
    ctx.dispatch_blocking(ctx.load_kernel("block_norms_" + kind), bind(*(b[i] for i in range(7))), (post, gates, plus_one, float(scale), float(eps)), [hidden, rows, 1])
    assert (h_out[rows:] == 3).all() and (x[rows:] == 3).all(), "rows behind the last were written"
    return h_out[:rows], x[:rows]


def _norms_case(seed, kind, rows, hidden, gates, spread=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    by = torch.exp2(torch.randint(-spread, spread + 1, (rows, 1), generator=gen, device="cuda").float())
    y, h = (normal(rows, hidden) * by).half(), (normal(rows, hidden) * 4 * by).to(TYPES[kind])
    w_post, w_pre = normal(hidden) * 0.3 + 1, normal(hidden) * 0.3 + 1
    return y, h, w_post, normal(max(1, (0, hidden, rows, 1)[gates])), w_pre


def _check_norms(got, y, h, w_post, gate, w_pre, kind, post, gates, plus_one, scale, eps, what):
    f = lambda t: t.float().cpu().numpy()  # noqa: E731
    g = {0: None, 1: f(gate)[:h.shape[1]], 2: f(gate)[:h.shape[0], None], 3: f(gate)[:1]}[gates]
    weight = lambda w: around.norm_weight(f(w), plus_one)  # noqa: E731
    want, err, x, x_err = around.block_norms(f(y), f(h), weight(w_post), g, weight(w_pre), post, float(np.float32(scale)), float(np.float32(eps)))
    if post == 2:
        assert (got[0] == 3).all(), "h_out was written"
    else:
        _within(f(got[0]), want, err + HALF_STEP[kind] * (np.abs(want) + err) + TINY[kind], f"{what}: h")
    _within(f(got[1]), x, x_err * 1.001 + around.f16_step(x), f"{what}: x")


SHAPES = [(1, 8), (5, 16), (3, 24), (130, 64), (1, 128), (33, 136), (7, 256), (200, 264), (2, 512), (9, 1000), (1, 1032), (65, 1096), (300, 2048), (3, 2056), (1, 5376), (64, 5376), (400, 5376),
          (11, 8192), (2, 8200), (3, 12296), (170, 16384), (1, 16384)]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("rows,hidden", SHAPES)
def test_norms(ctx, kind, rows, hidden):
    for n, (post, gates, plus_one, scale, in_place) in enumerate(((1, 0, 0, 1.0, False), (1, 1, 1, 0.75, True), (0, 2, 0, -1.5, False), (1, 3, 1, 1.0, False), (0, 0, 0, 0.5, True), (2, 0, 0, 1.0, False),
                                                                  (2, 0, 1, 1.0, False), (1, 2, 0, 0.25, True), (0, 1, 1, 2.0, False))):
        y, h, w_post, gate, w_pre = _norms_case(rows + hidden + n, kind, rows, hidden, gates)
        copies = y.clone(), h.clone()
        got = _norms(ctx, kind, y, h, w_post, gate, w_pre, post, gates, plus_one, scale, 1e-6, in_place)
        _check_norms(got, *copies, w_post, gate, w_pre, kind, post, gates, plus_one, scale, 1e-6, (post, gates, in_place))


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("rows,hidden", [(20000, 64), (40001, 8), (5003, 1096), (2500, 5376), (1200, 7168), (700, 16384)])
def test_norms_of_many_rows(ctx, kind, rows, hidden):
    for post, gates in ((1, 2), (0, 1)):
        case = _norms_case(rows, kind, rows, hidden, gates)
        got = _norms(ctx, kind, *case, post, gates, 0, 0.5, 1e-5)
        _check_norms(got, *case, kind, post, gates, 0, 0.5, 1e-5, (post, gates))


STREAMED = [("f16", 200_003, 72), ("bf16", 100_000, 136), ("f16", 13_001, 1096), ("bf16", 6500, 2048), ("f16", 2501, 5376), ("f32", 1700, 5376), ("bf16", 1600, 8192), ("f16", 800, 16384),
            ("f32", 1000, 10240), ("f32", 900, 10248), ("f32", 520, 16384), ("f32", 120_001, 72), ("f32", 32_011, 264)]


@pytest.mark.parametrize("kind,rows,hidden", STREAMED)
def test_norms_whose_rows_come_ahead(ctx, kind, rows, hidden):
    """From 80 MB on rows come ahead of their turn or ask late for their weights: 300 rows against the plain statement, all of them against calls of a few rows each."""
    assert rows * hidden * (4 + 2 * TYPES[kind].itemsize) >= 96 << 20
    some = torch.cat([torch.arange(100), torch.randint(0, rows, (100,), generator=torch.Generator().manual_seed(rows)), torch.arange(rows - 100, rows)]).cuda()
    for post, gates, plus_one, scale, in_place in ((1, 1, 1, 0.75, True), (0, 2, 0, -1.5, False), (1, 3, 0, 1.0, False), (2, 0, 1, 1.0, False), (0, 0, 0, 0.5, True)):
        y, h, w_post, gate, w_pre = _norms_case(rows + post, kind, rows, hidden, gates)
        y0, h0 = y.clone(), h.clone()
        got = _norms(ctx, kind, y, h, w_post, gate, w_pre, post, gates, plus_one, scale, 1e-6, in_place)
        rows_gate = gate[some] if gates == 2 else gate
        _check_norms([g[some] for g in got], y0[some], h0[some], w_post, rows_gate, w_pre, kind, post, gates, plus_one, scale, 1e-6, (post, gates, in_place))
        part = max(1, (70 << 20) // (hidden * (4 + 2 * h0.element_size())))
        for r in range(0, rows, part):
            few = _norms(ctx, kind, y0[r:r + part].clone(), h0[r:r + part].clone(), w_post, gate[r:r + part].clone() if gates == 2 else gate, w_pre, post, gates, plus_one, scale, 1e-6)
            for a, b, step in ((got[0][r:r + part], few[0], HALF_STEP[kind]), (got[1][r:r + part], few[1], 2.0 ** -11)):  # the order of a sum, a few units of 2^-24 of values below 32, and with it a rounding
                a, b = a.float(), b.float()
                assert ((a - b).abs() <= 2.02 * step * b.abs() + 1e-5).all(), f"rows from {r}, {(post, gates)}"


@pytest.mark.parametrize("kind", list(TYPES))
def test_norms_of_rows_of_all_sizes(ctx, kind):
    """Rows whose squares are near or below eps, zero rows, an eps of 0."""
    for eps in (1e-6, 0.0):
        case = _norms_case(5, kind, 60, 520, 0, spread=10)
        case[0][7], case[1][7] = (0, 0) if eps else (1, 0)
        case[0][8] = 0 if eps else 1
        got = _norms(ctx, kind, *case, 1, 0, 0, 1.0, eps)
        _check_norms(got, *case, kind, 1, 0, 0, 1.0, eps, eps)


def test_norms_keep_what_is_no_number_in_its_row(ctx):
    y, h, w_post, gate, w_pre = _norms_case(6, "f32", 4, 1000, 0)
    y[1, 500], h[2, 3] = float("nan"), float("inf")
    h_out, x = _norms(ctx, "f32", y, h, w_post, gate, w_pre, 1, 0)
    assert torch.isnan(h_out[1]).all() and torch.isnan(x[1]).all() and torch.isinf(h_out[2, 3]) and torch.isfinite(h_out[2, 4:]).all() and torch.isnan(x[2, 3]) and (x[2, 4:] == 0).all()
    assert torch.isfinite(h_out[[0, 3]]).all() and torch.isfinite(x[[0, 3]]).all()


def test_norms_beyond_32_bits(ctx):
    """2^32 bytes of h and more."""
    rows, hidden = 270_001, 4096
    h = torch.ones(rows, hidden, device="cuda")
    y = torch.zeros(rows, hidden, dtype=torch.float16, device="cuda")
    h[-1], y[-1] = 2.0, 3.0
    w = torch.ones(hidden, device="cuda")
    h_out, x = _norms(ctx, "f32", y, h, w, w, w, 0, 0, scale=2.0)
    assert (h_out[:-1] == 2).all() and (h_out[-1] == 10).all() and ((x.float() - 1).abs() <= 2.0 ** -10).all()


# ---- reading the cache back ----------------------------------------------------------------------------------------------------------------
def _read(ctx, pool_buffers, table, first, starts, kv, page, tokens):
    up = ctx.buffer_from_iter
    out = [up(np.full(tokens * kv * D, 0x7D7D, np.uint16)) for _ in range(2)]  # a NaN
    ctx.dispatch_blocking(ctx.load_kernel("kv_read_blocks_e4m3_d128"), bind(*pool_buffers, up(_u32(table).reshape(-1)), up(_u32(first)), up(_u32(starts)), *out),
                          (page, table.shape[1]), [kv, len(first), tokens])
    got = [b.read().reshape(tokens, kv, D) for b in out]
    assert all((g[starts[-1]:] == 0x7D7D).all() for g in got), "rows behind the last request were written"
    return [g.view(np.float16) for g in got]


@pytest.mark.parametrize("kv,page", [(1, 16), (3, 32), (16, 256), (5, 64), (8, 512)])
@pytest.mark.parametrize("requests,longest", [(1, 1), (1, 17), (1, 1000), (7, 60), (40, 300), (300, 20), (2100, 2)])
def test_reading_back(ctx, kv, page, requests, longest):
    rng = np.random.default_rng(requests + kv)
    n = rng.integers(0, longest + 1, requests)
    n[0] = longest
    first = rng.integers(0, 2 * page, requests) * (rng.random(requests) < 0.6)
    pages = np.maximum(-(-(first + n) // page), 1)
    order, stride = rng.permutation(int(pages.sum()) + 3), int(pages.max()) + 1
    table, at = np.full((requests, stride), NONE, np.int64), 0
    for r, m in enumerate(pages):
        table[r, :m] = order[at:at + m] if n[r] else NONE
        at += m
    blocks = len(order) * page // TILE
    pools = [*_pool(rng, blocks, kv), *_pool(rng, blocks, kv)]
    starts = np.concatenate([[0], np.cumsum(n)])
    got = _read(ctx, [ctx.buffer_from_iter(p.reshape(-1)) for p in pools], table, first, starts, kv, page, int(starts[-1]) + 5)
    for g, pool, exps in zip(got, pools[::2], pools[1::2]):
        want = around.read(pool, exps, table, first, starts, page, int(starts[-1]) + 5)
        with np.errstate(over="ignore"):
            assert np.array_equal(g[:starts[-1]], want[:starts[-1]].astype(np.float16))


def test_reading_exponents_that_no_append_writes(ctx):
    rng = np.random.default_rng(3)
    pools = [*_pool(rng, 256, 1), *_pool(rng, 256, 1)]
    pools[1][:, 0] = np.arange(-128, 128)
    pools[3][:, 0] = np.arange(-128, 128)[::-1]
    pools[0][130, 0, 3, 5] = 0x7F
    got = _read(ctx, [ctx.buffer_from_iter(p.reshape(-1)) for p in pools], np.arange(256)[None, :], [0], [0, 4096], 1, 16, 4096)
    for g, pool, exps in zip(got, pools[::2], pools[1::2]):
        want = around.read(pool, exps, np.arange(256)[None, :], [0], [0, 4096], 16, 4096)
        with np.errstate(over="ignore"):
            assert np.array_equal(g, want.astype(np.float16), equal_nan=True)


def test_reading_reports_pages_and_positions_that_are_not_there(ctx):
    import super_gemma_b200 as sg

    rng = np.random.default_rng(3)
    pools = [*_pool(rng, 8, 2), *_pool(rng, 8, 2)]
    b = [ctx.buffer_from_iter(p.reshape(-1)) for p in pools]
    for table, first in (([[0, 4]], [20]), ([[0, 0xFFFFFFFF]], [31]), ([[0, 1]], [64]), ([[0, 1]], [0xFFFFFFFF])):
        with pytest.raises(sg.Bounds):
            _read(ctx, b, np.array(table), first, [0, 30], 2, 32, 30)
        ctx.sync()
    up = ctx.buffer_from_iter  # starts that go back, or beyond the rows: rows of nobody are left, none is out of range
    out = [up(np.full(30 * 2 * D, 0x7D7D, np.uint16)) for _ in range(2)]
    for starts in ([0, 20, 10, 40], [25, 5, 5, 9], [7, 7, 7, 7]):
        ctx.dispatch_blocking(ctx.load_kernel("kv_read_blocks_e4m3_d128"), bind(*b, up(_u32([[0, 1], [2, 3], [1, 0]]).reshape(-1)), up(_u32([0, 0, 0])), up(_u32(starts)), *out),
                              (32, 2), [2, 3, 30])


# ---- all of it, as a server runs it -------------------------------------------------------------------------------------------------------
def test_steps_of_a_server(ctx):
    """Six steps of one layer for twelve requests that come, go on and end: a recorded graph of tables, angles, norms, the pre-attention pass, attention, the norms behind it,
    replayed with new lengths; a host copy follows every step.  The projections are the caller's: here the values themselves."""
    rng = np.random.default_rng(11)
    R, N, heads, kv, page, stride, pages = 12, 160, 4, 2, 32, 12, 80
    hidden = heads * D
    up, zeros = ctx.buffer_from_iter, lambda n, t=np.uint32: ctx.new_buffer(n, t)  # noqa: E731
    import super_gemma_b200 as sg

    freqs = sg.rope_frequencies(64, 1e4, kind="by_turns", factor=4.0, trained=256, slow=1.0, fast=8.0)
    magnitude = 1.1386294
    b = {"ctx": zeros(R), "new": zeros(R), "held": zeros(R), "count": up(_u32([pages, 0, 0, 0])), "free": up(_u32(rng.permutation(pages))), "table": zeros(R * stride), "starts": zeros(R + 1),
         "lens": zeros(R), "slots": zeros(N), "at": zeros(N), "freqs": up(freqs), "cos_sin": zeros(N * 128, np.float32), "h": zeros(N * hidden, np.float32),
         "y": zeros(N * hidden, np.uint16), "x": zeros(N * hidden, np.uint16), "q": zeros(N * heads * D, np.uint16), "k": zeros(N * kv * D, np.uint16), "v": zeros(N * kv * D, np.uint16),
         "kp": up(np.full(pages * page * kv * D, 0x7F, np.uint8)), "ke": up(np.full(pages * page // TILE * kv, 127, np.int8)),
         "vp": up(np.full(pages * page * kv * D, 0x7F, np.uint8)), "ve": up(np.full(pages * page // TILE * kv, 127, np.int8)), "out": zeros(N * heads * D, np.uint16),
         "x2": zeros(N * hidden, np.uint16), "one": up(np.ones(1, np.float32))}
    w = {n: (1 + 0.2 * rng.standard_normal(m)).astype(np.float32) for n, m in (("q_w", D), ("k_w", D), ("w_in", hidden), ("w_post", hidden), ("w_pre", hidden), ("gate", hidden))}
    b.update({n: up(v) for n, v in w.items()})
    b["work"] = ctx.new_buffer(ctx.attn_blocks_work_bytes(kv, heads // kv, R, N, 64), np.uint8)
    scale = float(np.float32(D ** -0.5))

    def layer(c):
        def run(kernel, names, push, grid):
            c.dispatch(c.load_kernel(kernel), bind(*(b[n] for n in names.split())), push, grid)

        run("kv_block_tables", "ctx new held count free table held count starts lens slots at", (page, stride), [R, N, 1])
        run("rope_cos_sin", "freqs at cos_sin", (128, magnitude), [N, 1, 1])
        run("block_norms_f32", "y h w_post one w_in h x", (2, 0, 0, 1.0, 1e-6), [hidden, N, 1])
        run("qkv_norm_rope_append_blocks_e4m3_d128", "x q_w q k v k_w cos_sin slots kp ke vp ve", (128, 0, 0, 0, 0, 0, magnitude), [heads, kv, N])
        run("attn_blocks_e4m3_d128", "q kp ke vp ve table lens starts out work", (scale, page, stride, 0, heads // kv, 64), [kv, R, N])
        run("block_norms_f32", "out h w_post gate w_pre h x2", (1, 1, 0, 0.5, 1e-6), [hidden, N, 1])

    graph = ctx.record_graph(layer)
    lens = np.zeros(R, np.int64)
    for step in range(6):
        new = np.where(lens == 0, rng.integers(0, 60, R) * (rng.random(R) < 0.5), rng.integers(1, 4, R))
        ended = (lens > 0) & (rng.random(R) < 0.15)
        lens[ended], new[ended] = 0, 0
        while new.sum() > N - 8:
            new[np.argmax(new)] //= 2
        n = int(new.sum())
        h = (rng.standard_normal((N, hidden)) * 3).astype(np.float32)
        k, v = (rng.standard_normal((N, kv, D)).astype(np.float16) for _ in range(2))
        before = {x: b[x].read() for x in ("kp", "ke", "vp", "ve")}
        b["ctx"].write(_u32(lens)), b["new"].write(_u32(new)), b["h"].write(h.reshape(-1)), b["k"].write(k.view(np.uint16).reshape(-1)), b["v"].write(v.view(np.uint16).reshape(-1))
        ctx.submit_blocking(graph)
        lens = lens + new
        starts, slots, at = b["starts"].read(), b["slots"].read().astype(np.int64), b["at"].read()
        assert starts[-1] == n and (slots[:n] != NONE).all() and (slots[n:] == NONE).all()
        rows, bound = around.cos_sin(at, freqs, magnitude)
        got_rows = b["cos_sin"].read().reshape(N, 64, 2)
        _within(got_rows, rows, bound, "angles")
        _, _, x, x_err = around.block_norms(None, h, None, None, w["w_in"], 2, 1.0, 1e-6)
        got_x = b["x"].read().view(np.float16).reshape(N, hidden)
        _within(got_x, x, x_err * 1.001 + around.f16_step(x), "x")
        s = Step(0, slots, heads, kv, pages * page // TILE)
        s.q, s.k, s.v, s.rows, s.magnitude, s.q_w, s.k_w = got_x.reshape(N, heads, D), k, v, got_rows, magnitude, w["q_w"], w["k_w"]
        shape = (pages * page // TILE, kv, TILE, D)
        s.pools = [before["kp"].reshape(shape), before["ke"].view(np.int8).reshape(shape[:2]), before["vp"].reshape(shape), before["ve"].view(np.int8).reshape(shape[:2])]
        s.b = [b[i] for i in ("kp", "ke", "vp", "ve")]
        got_q = b["q"].read().reshape(N, -1)
        s.q_out = type("Q", (), {"read": lambda self: np.concatenate([got_q[:n].reshape(-1), np.full((N + 2 - n) * heads * D, 0x5555, np.uint16)])})()
        s.check(f"step {step}")
        kp, ke, vp, ve = [g.view(p.dtype).reshape(p.shape) for g, p in zip(s.got(), s.pools)]
        table = b["table"].read().reshape(R, stride)
        want, bnd = ref.attend(got_q.view(np.float16).reshape(N, heads, D), kp, ke, vp, ve, table, lens, starts, page, 0, heads // kv, scale)
        out = b["out"].read().view(np.float16).reshape(N, heads, D)
        _within(out[:n], want[:n], bnd[:n], f"step {step}: attention")
        hw, err, x2, x2_err = around.block_norms(out.reshape(N, -1), h, w["w_post"], w["gate"], w["w_pre"], 1, 0.5, 1e-6)
        _within(b["h"].read().reshape(N, hidden)[:n], hw[:n], (err + 2.0 ** -24 * np.abs(hw))[:n], "h")
        _within(b["x2"].read().view(np.float16).reshape(N, hidden)[:n], x2[:n], (x2_err * 1.001 + around.f16_step(x2))[:n], "x2")
        total = int(lens.sum())
        back = _read(ctx, [b[i] for i in ("kp", "ke", "vp", "ve")], table, [0] * R, np.concatenate([[0], np.cumsum(lens)]), kv, page, total + 2)
        for g, pool, exps in zip(back, (kp, vp), (ke, ve)):
            assert np.array_equal(g[:total], around.read(pool, exps, table, [0] * R, np.concatenate([[0], np.cumsum(lens)]), page, total + 2)[:total])


def test_two_contexts_and_graphs_side_by_side(ctx):
    """Two streams, each replaying graphs of its own over its own tensors, and one graph twice: nothing is shared between dispatches."""
    import super_gemma_b200 as sg

    other = sg.GpuContext(0)
    steps = [[Step(i + 2 * c, _runs(i, [(3, 50 + 9 * i)], 8, i % 2), 4, 2, 8, layout=i) for i in range(2)] for c in range(2)]
    name = "qkv_norm_rope_append_blocks_e4m3_d128"
    graphs = []
    for c, mine in zip((ctx, other), steps):
        bound = [s.buffers(c) for s in mine]
        graphs.append([c.record_graph(lambda at, b=b, s=s: at.dispatch(at.load_kernel(name), b, *s.call())) for b, s in zip(bound, mine)])
    for _ in range(20):
        for c, g in zip((ctx, other), graphs):
            c.submit(g[0]), c.submit(g[1])
    ctx.sync(), other.sync()
    for mine in steps:
        for s in mine:
            # replayed twenty times, a tile that this call continues has long grown to its exponent
            grown = around.exponents(s.k_w, 1.0)
            for side, e in ((0, grown[0]), (2, grown[1])):
                lo, _, exps = around.append_normed(around.norm128(s.k, None) * 0, np.zeros(s.k.shape), s.slots, s.pools[side], s.pools[side + 1], e)
                keep = np.zeros(lo.shape[:1] + lo.shape[2:3], bool)
                keep[s.slots[s.slots != NONE] // TILE, s.slots[s.slots != NONE] % TILE] = True
                s.pools[side] = np.where(keep[:, None, :, None], s.pools[side], lo)
                s.pools[side + 1] = np.where(exps == s.pools[side + 1], s.pools[side + 1], exps)
            s.check("replayed")


def _one_of_each(ctx, seed):
    """A call of every operator over tensors of its own: (kernel, bindings, push, grid, the buffers it writes)."""
    rng = np.random.default_rng(seed)
    up = ctx.buffer_from_iter
    n, heads, kv, hidden = 90 + seed, 6, 3, 1096
    half = lambda *s: rng.standard_normal(s).astype(np.float16)  # noqa: E731
    fill = lambda k: up(np.full(k, 0x5555, np.uint16))  # noqa: E731
    freqs, positions = up(around.frequencies(64, 1e4, 128)), up(_u32(rng.integers(0, 1 << 20, n)))
    rows = up(np.zeros(n * 128, np.float32))
    q, k = up(half(n, heads, D)), up(half(n, kv, D))
    q_out, k_out = fill(n * heads * D), fill(n * kv * D)
    calls = [("rope_cos_sin", (freqs, positions, rows), (128, 1.25), [n, 1, 1], [rows]),
             ("rope_qk_f16", (q, k, rows, q_out, k_out), (D, 128, seed % 3, 0, 0, 0, 0), [heads, kv, n], [q_out, k_out])]
    for i, kind in enumerate(TYPES):
        h = rng.standard_normal((n, hidden)).astype(np.float32)
        h = up(h if kind == "f32" else h.astype(np.float16) if kind == "f16" else (h.view(np.uint32) >> 16).astype(np.uint16))
        h_out, x = ctx.new_buffer(h.nbytes, np.uint8), fill(n * hidden)
        w = [up(rng.standard_normal(hidden).astype(np.float32)) for _ in range(3)]
        calls.append(("block_norms_" + kind, (up(half(n, hidden)), h, w[0], w[1], w[2], h_out, x), (1, 1, i % 2, 0.5, 1e-6), [hidden, n, 1], [h_out, x]))
    s = Step(seed, _runs(seed, [(0, n)], 8, False), heads, kv, 8, exps=(-5, -4), magnitude=1.25)  # (tiles begin in it: nothing grows from replay to replay)
    b = s.buffers(ctx)
    b[6].buf = rows
    calls.append(("qkv_norm_rope_append_blocks_e4m3_d128", tuple(x.buf for x in b), *s.call(), [s.q_out, *s.b]))
    out = fill(n * kv * D), fill(n * kv * D)
    calls.append(("kv_read_blocks_e4m3_d128", (*s.b, up(_u32(np.random.default_rng(seed).permutation(8))), up(_u32([0])), up(_u32([0, n])), *out), (16, 8), [kv, 1, n], list(out)))
    return [(ctx.load_kernel(name), bind(*bufs), push, grid, written) for name, bufs, push, grid, written in calls]


def test_all_of_them_recorded_and_side_by_side(ctx):
    """Every operator twice in a recording with branches, replayed beside another context's: the bits of calls made one after the other."""
    import super_gemma_b200 as sg

    other = sg.GpuContext(0)
    sides = []
    for i, c in enumerate((ctx, other)):
        calls = _one_of_each(c, 2 * i) + _one_of_each(c, 2 * i + 1)
        for call in calls:
            c.dispatch_blocking(*call[:4])
        want = [[b.read() for b in call[4]] for call in calls]
        for call in calls[:2] + calls[7:9]:  # (not the cache: a tile's other rows are nobody's)
            for b in call[4]:
                b.zero()
        sides.append((c, calls, want, c.record_graph(lambda at, calls=calls: [at.dispatch(*call[:4]) for call in calls])))
    for _ in range(25):
        for c, _, _, graph in sides:
            c.submit(graph)
    for c, calls, want, _ in sides:
        c.sync()
        for n, (call, w) in enumerate(zip(calls, want)):
            for b, x in zip(call[4], w):
                assert np.array_equal(b.read(), x), f"{n}: {call[0].name}"
