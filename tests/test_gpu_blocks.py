"""GPU tests of the batched cache: block tables, append, attention, and the three together as a server runs them.

Placement and quantisation are exact.  Attention is held to the bound that ``blocks_ref.attend`` derives from where the kernel
rounds (weights and results to f16).  Whatever no request owns is poison: cache rows are NaN, exponents 127, table entries point nowhere."""
import numpy as np
import pytest

import blocks_ref as ref
from cases import bind

pytestmark = pytest.mark.gpu
NONE, TILE, D = ref.NONE, ref.TILE, ref.D
SCALE = float(np.float32(D ** -0.5))


@pytest.fixture(scope="module")
def ctx():
    import super_gemma_b200 as sg

    return sg.GpuContext(0)


def _u32(v):
    return np.asarray(v, np.uint32)


# ---- block tables ------------------------------------------------------------------------------------------------------------
def _plan_state(seed, requests, page, stride, tokens, free=None, busy=0.4, most_new=None):
    """Requests in every state: idle, decoding, prompts, ended, cut back (a draft was rejected), holding more than they need."""
    rng = np.random.default_rng(seed)
    ctx, new, held = (np.zeros(requests, np.int64) for _ in range(3))
    for r in range(requests):
        had = int(rng.integers(1, stride * page + 1))
        held[r] = -(-had // page)
        ctx[r], new[r] = had, 1
        if rng.random() < busy:
            kind = rng.integers(0, 5)
            if kind == 0:
                ctx[r] = new[r] = 0  # ended
            elif kind == 1:
                ctx[r], held[r], new[r] = 0, 0, rng.integers(0, (most_new or stride * page) + 1)  # a prompt, perhaps an empty one
            elif kind == 2:
                new[r] = 0  # idle
            elif kind == 3:
                ctx[r] = rng.integers(0, had + 1)  # cut back
            else:
                new[r] = rng.integers(2, 9)  # a draft, which may no longer fit its row
    spare = int(rng.integers(0, requests + 2)) if free is None else free
    pages = int(held.sum()) + spare
    order = rng.permutation(pages).astype(np.uint32)
    table, at = np.full((requests, stride), NONE, np.uint32), 0
    for r in range(requests):
        table[r, :held[r]] = order[at:at + held[r]]
        at += held[r]
    lst = np.full(pages + 3, 0xDEAD, np.uint32)
    lst[:spare] = order[at:]
    return ctx, new, held, spare, lst, table


def _run_plan(ctx, state, page, tokens, in_place=False):
    lens, new, held, count, lst, table = state
    requests, stride = table.shape
    up = ctx.buffer_from_iter
    b = {"ctx": up(_u32(lens)), "new": up(_u32(new)), "held": up(_u32(held)), "count": up(_u32([count, 0, 0, 0])), "free": up(lst), "table": up(table.reshape(-1))}
    for n, size in (("held_out", requests), ("free_out", 4), ("starts", requests + 1), ("lens", requests), ("slots", tokens), ("at", tokens)):
        b[n] = up(np.full(size, 0xABCD, np.uint32))
    if in_place:
        b["held_out"], b["free_out"] = b["held"], b["count"]
    names = "ctx new held count free table held_out free_out starts lens slots at".split()
    ctx.dispatch_blocking(ctx.load_kernel("kv_block_tables"), bind(*(b[n] for n in names)), (page, stride), [requests, tokens, 1])
    got = {n: b[n].read() for n in names[4:]}
    got["table"] = got["table"].reshape(table.shape)
    return got, b


@pytest.mark.parametrize("requests,page,stride,tokens,in_place", [
    (1, 16, 1, 1, False), (1, 256, 4, 1100, True), (3, 16, 5, 7, False), (33, 32, 9, 400, True), (64, 256, 4, 64, False), (64, 256, 4, 65, True), (1023, 16, 3, 9000, False),
    (1024, 64, 2, 20000, True), (1025, 16, 7, 30001, True), (3000, 512, 2, 5000, False),
    (4096, 16, 3, 4097, True), (4097, 16, 4, 9000, False), (9001, 64, 2, 20000, True)])
def test_block_tables_match_the_plain_statement(ctx, requests, page, stride, tokens, in_place):
    for seed in range(4):
        state = _plan_state(seed, requests, page, stride, tokens, busy=(0.0, 0.4, 0.9, 1.0)[seed], most_new=min(stride * page, 3 * tokens // requests + 1))
        want = ref.plan(*state[:3], *state[3:], page, tokens)
        got, _ = _run_plan(ctx, state, page, tokens, in_place)
        for name, w in want.items():
            assert np.array_equal(got[name], w), f"{name} of seed {seed}"


def test_block_tables_move_many_pages_of_one_request(ctx):
    page, stride = 16, 700
    held, table = np.array([699, 0, 1]), np.full((3, stride), NONE, np.uint32)
    table[0, :699], table[2, 0] = np.arange(699)[::-1], 5000
    state = (np.array([5, 0, 16]), np.array([1, 690 * 16 - 3, 1]), held, 40, np.arange(1000, 1800, dtype=np.uint32), table)
    want = ref.plan(*state, page, 12000)
    got, _ = _run_plan(ctx, state, page, 12000)
    assert want["free_out"][1] == 0 and all(np.array_equal(got[n], w) for n, w in want.items())


def test_block_tables_refuse_what_the_list_does_not_cover(ctx):
    """The second request wants more than there is: it and every later one that wants pages go without; those that want none go on."""
    table = np.full((4, 4), NONE, np.uint32)
    table[3, 0] = 9
    state = (np.array([0, 0, 0, 3]), np.array([16, 64, 16, 1]), np.array([0, 0, 0, 1]), 2, _u32([4, 7, 0, 0, 0]), table)
    got, _ = _run_plan(ctx, state, 16, 97)
    assert list(got["lens"]) == [16, 0, 0, 4] and list(got["free_out"]) == [1, 2, 17, 1] and got["table"][0, 0] == 7
    assert list(got["held_out"]) == [1, 0, 0, 1] and (got["slots"][16:96] == NONE).all() and got["slots"][96] == 9 * 16 + 3
    assert all(np.array_equal(got[n], w) for n, w in ref.plan(*state, 16, 97).items())


def test_block_tables_report_a_count_beyond_the_list(ctx):
    import super_gemma_b200 as sg

    table = np.full((1, 2), NONE, np.uint32)
    with pytest.raises(sg.Bounds):
        _run_plan(ctx, (np.array([0]), np.array([5]), np.array([0]), 9, _u32([3, 4]), table), 16, 5)
    ctx.sync()
    with pytest.raises(sg.Bounds):  # more pages held than the row has
        _run_plan(ctx, (np.array([0]), np.array([5]), np.array([3]), 2, _u32([3, 4, 0, 0, 0]), table), 16, 5)
    ctx.sync()


# ---- append ------------------------------------------------------------------------------------------------------------------
def _pool(seed, blocks, kv, poison=False):
    rng = np.random.default_rng(seed)
    if poison:
        return np.full((blocks, kv, TILE, D), 0x7F, np.uint8), np.full((blocks, kv), 127, np.int8)
    codes = rng.integers(0, 256, (blocks, kv, TILE, D)).astype(np.uint8)
    return np.where((codes & 127) == 127, 0x11, codes).astype(np.uint8), rng.integers(-15, 9, (blocks, kv)).astype(np.int8)


def _run_append(ctx, k, v, slots, pools, kv):
    up = ctx.buffer_from_iter
    b = [up(p.reshape(-1)) for p in pools]
    kb, vb, sb = up(k), up(v), up(_u32(slots))
    ctx.dispatch_blocking(ctx.load_kernel("kv_append_blocks_e4m3_d128"), bind(kb, vb, sb, *b), None, [kv, len(slots), 1])
    return [x.read().reshape(p.shape) for x, p in zip(b, pools)]


def _hard_values(rng, shape):
    """Normal values, whole scales of powers of two, zeros, f16's ends, ties."""
    x = rng.standard_normal(shape) * 2.0 ** rng.integers(-20, 12, shape[:2] + (1,))
    x = np.where(rng.random(shape) < 0.05, 0.0, x)
    x = np.where(rng.random(shape) < 0.02, rng.choice([65504.0, -65504.0, 61440.0, 2.0 ** -24, -2.0 ** -24, 6.0e-5, 1.75, 448.0, 449.0], shape), x)
    return x.astype(np.float16)


@pytest.mark.parametrize("kv", [1, 3, 16])
@pytest.mark.parametrize("runs", [[(0, 1)], [(15, 1)], [(0, 16)], [(3, 13)], [(7, 60)], [(5, 3), (33, 1), (50, 30), (96, 16), (127, 1)], [(0, 200), (213, 11)]])
def test_append_matches_the_plain_statement(ctx, kv, runs):
    blocks = 16
    for seed in range(3):
        rng = np.random.default_rng([seed, kv, len(runs)])
        slots, order = [], rng.permutation(blocks)  # physical blocks in any order, whole runs block by block
        for first, n in runs:
            t = np.arange(first, first + n)
            slots.append(order[t // TILE] * TILE + t % TILE)
        slots = np.concatenate(slots)
        if seed == 2:  # padding between and behind
            slots = np.concatenate([[NONE], slots, [NONE] * 19])
        k, v = _hard_values(rng, (len(slots), kv, D)), _hard_values(rng, (len(slots), kv, D))
        pools = [*_pool(seed, blocks, kv), *_pool(seed + 9, blocks, kv)]
        got = _run_append(ctx, k, v, slots, pools, kv)
        want = [p.copy() for p in pools]
        ref.append(k, slots, *want[:2])
        ref.append(v, slots, *want[2:])
        for name, g, w in zip(("k", "k exps", "v", "v exps"), got, want):
            assert np.array_equal(g, w), f"{name}, seed {seed}: {np.argwhere(g != w)[:4].tolist()}"


def test_append_token_by_token_and_large(ctx):
    """A tile filled one token at a time with growing values (its rows are rounded again each time), and a long prompt at once."""
    rng = np.random.default_rng(5)
    kv, pools = 2, [*_pool(1, 2, 2), *_pool(2, 2, 2)]
    want = [p.copy() for p in pools]
    for t in range(TILE):
        k, v = ((rng.standard_normal((1, kv, D)) * 2.0 ** (t - 8)).astype(np.float16) for _ in range(2))
        pools = _run_append(ctx, k, v, [TILE + t], pools, kv)
        ref.append(k, np.array([TILE + t]), *want[:2])
        ref.append(v, np.array([TILE + t]), *want[2:])
    assert all(np.array_equal(g, w) for g, w in zip(pools, want))
    n, kv = 5003, 5
    slots = np.arange(n) + 32 + 5
    k, v = (rng.standard_normal((n, kv, D)).astype(np.float16) for _ in range(2))
    pools = [*_pool(3, 340, kv), *_pool(4, 340, kv)]
    got = _run_append(ctx, k, v, slots, pools, kv)
    ref.append(k, slots, *pools[:2])
    ref.append(v, slots, *pools[2:])
    assert all(np.array_equal(g, w) for g, w in zip(got, pools))


@pytest.mark.parametrize("requests,kv", [(5, 3), (64, 16), (700, 2), (2500, 5)])
def test_append_of_decode_steps(ctx, requests, kv):
    """One token of each of few and many requests, some with a draft of a few, at every place of a tile, over tiles that have to grow and some that have not."""
    rng = np.random.default_rng(requests)
    run = np.where(rng.random(requests) < 0.1, rng.integers(2, 6, requests), 1)
    first = rng.integers(0, TILE, requests)
    block = rng.permutation(2 * requests)  # two blocks for each: a draft may go on in the second
    slots = np.concatenate([[block[2 * r + (first[r] + i) // TILE] * TILE + (first[r] + i) % TILE for i in range(run[r])] for r in range(requests)])
    if requests == 700:
        slots[np.isin(np.repeat(np.arange(requests), run), np.arange(0, requests, 9))] = NONE  # requests that were refused
    k, v = _hard_values(rng, (len(slots), kv, D)), _hard_values(rng, (len(slots), kv, D))
    pools = [*_pool(1, 2 * requests, kv), *_pool(2, 2 * requests, kv)]
    got = _run_append(ctx, k, v, slots, pools, kv)
    ref.append(k, slots, *pools[:2])
    ref.append(v, slots, *pools[2:])
    assert all(np.array_equal(g, w) for g, w in zip(got, pools))


def test_append_keeps_nan_and_cuts_infinity(ctx):
    k = np.ones((2, 1, D), np.float16)
    k[0, 0, :4] = [np.nan, np.inf, -np.inf, 65504]
    k[1, 0, 0] = np.nan
    got = _run_append(ctx, k, k, [4, 5], [*_pool(1, 1, 1), *_pool(2, 1, 1)], 1)
    for pool, exps in ((got[0], got[1]), (got[2], got[3])):
        v = ref.E4M3[pool[0, 0, 4:6]] * 2.0 ** exps[0, 0]
        assert exps[0, 0] == 8 and np.isnan(v[0, 0]) and list(v[0, 1:4]) == [61440, -61440, 61440] and (v[0, 4:] == 1).all() and np.isnan(v[1, 0])
    assert np.array_equal(got[0], got[2] * 0 + got[0])


def test_append_reports_slots_that_no_pool_has_or_no_order_allows(ctx):
    import super_gemma_b200 as sg

    x = np.ones((3, 1, D), np.float16)
    for slots in ([0, 1, 64], [0, 5, 6], [3, 3, 17], [9, 8, 20]):
        pools = [*_pool(1, 4, 1), *_pool(2, 4, 1)]
        with pytest.raises(sg.Bounds):
            _run_append(ctx, x, x, slots, pools, 1)
        ctx.sync()


# ---- attention -----------------------------------------------------------------------------------------------------------------
class Batch:
    """Requests over a poisoned cache: what their lengths say is real, nothing else."""

    def __init__(self, seed, lens, new, kv, group, page, spare_rows=0, dead=(), spread=1.0):
        rng = np.random.default_rng(seed)
        self.kv, self.group, self.page, self.rng = kv, group, page, rng
        self.lens = _u32([0 if r in dead else n for r, n in enumerate(lens)])
        self.starts = _u32(np.concatenate([[0], np.cumsum(new)]))
        self.tokens = int(self.starts[-1]) + spare_rows
        pages = [-(-int(n) // page) for n in self.lens]
        self.stride = max(1, max(pages))
        order = rng.permutation(sum(pages) + 2)
        self.table, at = np.full((len(lens), self.stride), NONE, np.uint32), 0
        blocks = len(order) * page // TILE
        (self.kp, self.ke), (self.vp, self.ve) = _pool(0, blocks, kv, True), _pool(0, blocks, kv, True)
        for r, n in enumerate(pages):
            self.table[r, :n] = order[at:at + n]
            at += n
            rows = ref.rows_of(self.table[r], int(self.lens[r]), page)
            for pool, exps, base in ((self.kp, self.ke, -7), (self.vp, self.ve, -8)):
                pool[rows // TILE, :, rows % TILE] = ref.encode((rng.standard_normal((len(rows), kv, D)) * 100).clip(-448, 448))
                b = np.unique(rows // TILE)
                lo, hi = (base, base + 4) if spread == 1.0 else (ref.LOWEST, 8)  # 448 * 2^7 is an f16 number, 448 * 2^8 none that an append writes
                exps[b] = rng.integers(lo, hi, (len(b), kv))
        self.q = (rng.standard_normal((max(1, self.tokens), kv * group, D)) * spread).astype(np.float16)
        self.max_q = max(1, max(int(x) for x in new))

    def buffers(self, ctx):
        up = ctx.buffer_from_iter
        self.out = up(np.full(self.q.size, 0x5555, np.uint16))
        work = ctx.attn_blocks_work_bytes(self.kv, self.group, len(self.lens), self.tokens, self.max_q)
        self.work = ctx.new_buffer(work, np.uint8)
        self.work.write(np.full(work, 0xFF, np.uint8))  # NaN
        return bind(up(self.q), up(self.kp.reshape(-1)), up(self.ke.reshape(-1)), up(self.vp.reshape(-1)), up(self.ve.reshape(-1)), up(self.table.reshape(-1)),
                    up(self.lens), up(self.starts), self.out, self.work)

    def call(self, window):
        return (SCALE, self.page, self.stride, window, self.group, self.max_q), [self.kv, len(self.lens), self.tokens]

    def check(self, raw, window, what=""):
        got = raw.view(np.float16).reshape(self.q.shape)
        want, bound = ref.attend(self.q, self.kp, self.ke, self.vp, self.ve, self.table, self.lens, self.starts, self.page, window, self.group, SCALE)
        n = int(self.starts[-1])
        assert (raw.reshape(self.q.shape)[n:] == 0x5555).all(), f"{what}: rows behind the last request were written"
        assert np.isfinite(got[:n]).all(), f"{what}: not finite at {np.argwhere(~np.isfinite(got[:n]))[:3].tolist()}"
        over = np.abs(got[:n].astype(np.float64) - want[:n]) - bound[:n]
        assert over.max(initial=-1) <= 0, f"{what}: {over.max()} beyond the bound at {np.unravel_index(over.argmax(), over.shape)}"

    def run(self, ctx, window=0, what=""):
        push, grid = self.call(window)
        ctx.dispatch_blocking(ctx.load_kernel("attn_blocks_e4m3_d128"), self.buffers(ctx), push, grid)
        raw = self.out.read()
        self.check(raw, window, what)
        return raw


@pytest.mark.parametrize("group", [1, 2, 4, 8])
@pytest.mark.parametrize("kv,page", [(1, 16), (3, 32), (16, 256)])
def test_decode_of_every_short_length(ctx, kv, page, group):
    lens = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 255, 256, 257, 300]
    Batch(kv + group, lens, [1] * len(lens), kv, group, page, spare_rows=3).run(ctx)


@pytest.mark.parametrize("n", [1, 16, 100, 1000, 5000, 20011])
def test_decode_of_one_request(ctx, n):
    Batch(n, [n], [1], 2, 2, 64).run(ctx)


@pytest.mark.parametrize("requests", [2, 7, 40, 150])
@pytest.mark.parametrize("seed", [1, 2])
def test_decode_of_ragged_batches(ctx, requests, seed):
    rng = np.random.default_rng(seed)
    lens = np.exp(rng.uniform(0, np.log(3000 if requests < 50 else 400), requests)).astype(int) + 1
    new = rng.integers(0, 2, requests)
    new[0] = 1
    Batch(seed, lens, new, 4, 2, 32, spare_rows=1).run(ctx)


@pytest.mark.parametrize("m,group", [(2, 1), (8, 1), (3, 2), (4, 2), (2, 4)])
def test_verify_is_causal_among_the_new_tokens(ctx, m, group):
    lens = [m, m + 1, 15, 16, 17, 50, 200, 1037]
    lens = [max(n, m) for n in lens]
    Batch(m * group, lens, [m, m, 1, m, 0, m, m - 1, m], 3, group, 16).run(ctx)


WIDE = [(9, 1), (16, 1), (17, 1), (32, 1), (5, 2), (8, 2), (9, 2), (16, 2), (3, 4), (4, 4), (5, 4), (8, 4), (2, 8), (3, 8), (4, 8)]


@pytest.mark.parametrize("window", [0, 40])
@pytest.mark.parametrize("m,group", WIDE)
def test_drafts_of_more_than_eight_rows(ctx, m, group, window):
    """Up to 32 rows, beside requests of fewer rows and of none; two requests that many warps share, two refused."""
    lens = [max(n, m) for n in (m, m + 1, 15, 16, 17, 50, 200, 1037, 5003, 64, 33)]
    Batch(m * group, lens, [m, m, 1, m, 0, m, m - 1, m, m, (m + 1) // 2, m], 3, group, 16, spare_rows=2, dead=(4, 10)).run(ctx, window)


@pytest.mark.parametrize("m,group", [(16, 1), (8, 4), (4, 8)])
def test_wide_drafts_over_one_head_and_large_scores(ctx, m, group):
    rng = np.random.default_rng(m)
    lens = rng.integers(m, 90, 70)
    lens[41] = 12000
    Batch(m, lens, rng.integers(0, m + 1, 70), 1, group, 16).run(ctx)
    Batch(m, [500, 2000, 35], [m, m, 1], 2, group, 32, spread=8.0).run(ctx)
    b = Batch(m, [3, 40, 9], [m, m, min(m, 9)], 2, group, 16)  # more queries than keys
    b.run(ctx)


@pytest.mark.parametrize("m,group", [(16, 1), (16, 2)])
def test_wide_drafts_again_give_the_same_bits(ctx, m, group):
    b = Batch(5, [4000, 17, 900, 333], [m, 1, m, m - 1], 4, group, 64)
    push, grid = b.call(0)
    k, bound = ctx.load_kernel("attn_blocks_e4m3_d128"), b.buffers(ctx)
    ctx.dispatch_blocking(k, bound, push, grid)
    first = b.out.read()
    b.check(first, 0)
    for _ in range(3):
        ctx.dispatch(k, bound, push, grid)
    ctx.sync()
    assert np.array_equal(b.out.read(), first)


@pytest.mark.parametrize("window", [1, 2, 16, 17, 100, 1024])
def test_window_over_few_and_many_queries(ctx, window):
    Batch(window, [1, 16, 40, 130, 1500, 3000], [1, 1, 4, 2, 1, 3], 2, 2, 32).run(ctx, window)
    Batch(window, [90, 16, 700, 1301], [90, 1, 130, 65], 2, 2, 32).run(ctx, window)


@pytest.mark.parametrize("new", [5, 16, 31, 63, 64, 65, 127, 128, 129, 200])
@pytest.mark.parametrize("group", [1, 2, 4, 8])
def test_prompts_of_odd_lengths(ctx, new, group):
    """Nothing cached before, a little, more than a tile of keys; beside them a request of one token and one of none."""
    Batch(new + group, [new, new + 1, new + 63, new + 64, new + 400, 77, 20], [new, new, new, new, new, 1, 0], 2, group, 16, spare_rows=2).run(ctx)


def test_prompts_of_every_length(ctx):
    for first in range(1, 140, 20):
        new = list(range(first, first + 20))
        Batch(first, [n + (7 * n) % 50 for n in new], new, 1, 2, 32).run(ctx, what=f"from {first}")


def test_one_chunk_over_a_long_context(ctx):
    Batch(3, [9000], [300], 2, 2, 256).run(ctx)
    Batch(4, [9001, 17], [67, 17], 3, 2, 64).run(ctx, 5000)


def test_mixed_prompts_and_single_tokens(ctx):
    rng = np.random.default_rng(9)
    new = [1, 300, 1, 1, 4, 129, 0, 1, 5, 64]
    lens = [int(n + rng.integers(0, 600)) for n in new]
    Batch(9, lens, new, 3, 2, 64, spare_rows=5).run(ctx)


def test_rows_that_see_nothing_are_zero(ctx):
    """Refused requests (length 0) with one query, a draft and a prompt; queries before the first key."""
    b = Batch(2, [40, 30, 200, 50, 5], [1, 4, 150, 1, 1], 2, 2, 16, dead=(0, 1, 2))
    b.run(ctx)
    b = Batch(3, [3, 40, 9], [4, 100, 9], 2, 2, 16)  # more queries than keys: the first of them stand before key 0
    raw = b.run(ctx).view(np.float16).reshape(b.q.shape)
    assert (raw[0] == 0).all() and (raw[4:64] == 0).all() and (raw[64:104] != 0).any(axis=(1, 2)).all()


def test_large_scores_and_scales(ctx):
    """Peaked softmaxes (queries of deviation 8) and tiles whose exponents lie 22 apart."""
    Batch(1, [500, 33, 2000], [1, 4, 1], 2, 2, 32, spread=8.0).run(ctx)
    Batch(2, [500, 233], [130, 70], 2, 2, 32, spread=8.0).run(ctx)


def test_reruns_and_neighbours_in_flight_give_the_same_bits(ctx):
    b = Batch(5, [4000, 17, 900, 333], [1, 1, 2, 200], 4, 2, 64)
    push, grid = b.call(0)
    k, bound = ctx.load_kernel("attn_blocks_e4m3_d128"), b.buffers(ctx)
    ctx.dispatch_blocking(k, bound, push, grid)
    first = b.out.read()
    b.check(first, 0)
    for _ in range(3):
        ctx.dispatch(k, bound, push, grid)
    ctx.sync()
    assert np.array_equal(b.out.read(), first)


def test_lengths_that_no_buffer_holds_are_reported(ctx):
    import super_gemma_b200 as sg

    k = ctx.load_kernel("attn_blocks_e4m3_d128")
    for change in ("lens", "starts", "order", "page", "queries"):
        b = Batch(6, [40, 50], [1, 2], 1, 1, 16)
        if change == "lens":
            b.lens[1] = 10 ** 9
        elif change == "starts":
            b.starts[2] = 10 ** 9
        elif change == "order":
            b.starts[1] = 7
        elif change == "page":
            b.table[1, 1] = 10 ** 6
        push, grid = b.call(0)
        if change == "queries":  # a request with more queries than the dispatch was told of
            b = Batch(6, [40, 50], [1, 9], 1, 1, 16)
            b.max_q = 1
            push, grid = b.call(0)
        with pytest.raises(sg.Bounds):
            ctx.dispatch_blocking(k, b.buffers(ctx), push, grid)
        ctx.sync()


def test_many_parts_of_one_request_among_many(ctx):
    """One kv head: every warp of the GPU has a stretch of it, and one long request's parts are merged by a CTA of few warps."""
    rng = np.random.default_rng(8)
    lens = rng.integers(1, 40, 400)
    lens[137] = 30000
    Batch(8, lens, np.ones(400, int), 1, 2, 16).run(ctx)
    Batch(9, lens[:300], rng.integers(0, 9, 300).clip(0, lens[:300]), 1, 1, 32).run(ctx)


@pytest.mark.parametrize("requests", [127, 128, 129, 513, 1100])
def test_more_requests_than_threads(ctx, requests):
    rng = np.random.default_rng(requests)
    lens = rng.integers(0, 50, requests)
    new = np.minimum(rng.integers(0, 4, requests), np.maximum(lens, 1))
    new[::37] = rng.integers(5, 30, len(new[::37]))
    Batch(requests, np.maximum(lens, new), new, 1, 4, 16, dead=set(range(5, requests, 50))).run(ctx)


@pytest.mark.parametrize("group", [1, 2, 4, 8])
def test_a_work_buffer_for_longer_drafts_does_for_shorter_ones(ctx, group):
    for kv in (1, 5, 16, 1024):
        sizes = [ctx.attn_blocks_work_bytes(kv, group, 20, 200, m) for m in range(1, 41)]
        assert sizes[0] > 0 and sizes == sorted(sizes)
    m = 16 // group
    b = Batch(group, [90, 40, 700], [m, 1, m], 2, group, 16)
    b.max_q = m + 30  # the prompts' kernel is launched too, and the drafts are its work
    b.run(ctx)


def test_offsets_beyond_32_bits(ctx):
    """Pools of more than 4 GiB each: tokens go into their last pages and are read from there."""
    import super_gemma_b200 as sg

    kv, page, keys = 16, 512, 700
    pages = (1 << 32) // (page * kv * D) + 3
    blocks = pages * page // TILE
    pools = [ctx.new_buffer(blocks * kv * TILE * D, np.uint8) for _ in range(2)]
    exps = [ctx.new_buffer(blocks * kv, np.int8) for _ in range(2)]
    assert pools[0].nbytes > 1 << 32
    table = _u32([[pages - 1, pages - 2, 0]])
    rng = np.random.default_rng(3)
    x = {n: rng.standard_normal((keys, kv * (2 if n == "q" else 1), D)).astype(np.float16) for n in "qkv"}
    slots = ref.rows_of(table[0], keys, page)
    assert slots.max() * kv * D > 1 << 32
    up = ctx.buffer_from_iter
    b = {n: up(x[n]) for n in "qkv"}
    ctx.dispatch_blocking(ctx.load_kernel("kv_append_blocks_e4m3_d128"), bind(b["k"], b["v"], up(_u32(slots)), pools[0], exps[0], pools[1], exps[1]), None, [kv, keys, 1])
    first = (pages - 2) * page // TILE  # the last two pages, as a pool of their own
    host = [np.zeros((2 * page // TILE, kv, TILE, D), np.uint8), np.zeros((2 * page // TILE, kv), np.int8)]
    host += [h.copy() for h in host]
    ref.append(x["k"], slots - first * TILE, *host[:2])
    ref.append(x["v"], slots - first * TILE, *host[2:])
    for p, e, hp, he in ((pools[0], exps[0], host[0], host[1]), (pools[1], exps[1], host[2], host[3])):
        assert np.array_equal(p.read(hp.size, first * kv * TILE * D).reshape(hp.shape), hp) and np.array_equal(e.read(he.size, first * kv).reshape(he.shape), he)
    for m in (1, 3, 300):
        q, out = up(x["q"][:m]), ctx.new_buffer(m * kv * 2 * D, np.uint16)
        work = ctx.new_buffer(ctx.attn_blocks_work_bytes(kv, 2, 1, m, m), np.uint8)
        ctx.dispatch_blocking(ctx.load_kernel("attn_blocks_e4m3_d128"),
                              bind(q, pools[0], exps[0], pools[1], exps[1], up(table.reshape(-1)), up(_u32([keys])), up(_u32([0, m])), out, work),
                              (SCALE, page, 3, 0, 2, m), [kv, 1, m])
        want, bound = ref.attend(x["q"][:m], *host, table - (pages - 2), [keys], [0, m], page, 0, 2, SCALE)
        got = out.read().view(np.float16).reshape(want.shape)
        assert (np.abs(got - want) <= bound).all(), m
    with pytest.raises(sg.Validation):  # a slice that is no whole number of heads' tiles is no pool
        ctx.dispatch(ctx.load_kernel("attn_blocks_e4m3_d128"), bind(q, pools[0].slice(0, 4096), exps[0], pools[1], exps[1], up(table.reshape(-1)), up(_u32([keys])),
                                                                    up(_u32([0, m])), out, work), (SCALE, page, 3, 0, 2, m), [kv, 1, m])


def test_contexts_side_by_side(ctx):
    """Two contexts, a stream and a work buffer each, with dispatches of both under way at a time, decode and prompts."""
    import super_gemma_b200 as sg

    other = sg.GpuContext(0)
    a, b = Batch(1, [3000, 50, 700], [1, 1, 300], 4, 2, 64), Batch(2, [900, 2000, 40], [200, 1, 40], 4, 2, 64)
    ba, bb = a.buffers(ctx), b.buffers(other)
    ka, kb = ctx.load_kernel("attn_blocks_e4m3_d128"), other.load_kernel("attn_blocks_e4m3_d128")
    for _ in range(20):
        ctx.dispatch(ka, ba, *a.call(0))
        other.dispatch(kb, bb, *b.call(0))
    ctx.sync()
    other.sync()
    a.check(a.out.read(), 0)
    b.check(b.out.read(), 0)


def test_graphs_that_share_a_work_buffer(ctx):
    """Two recorded dispatches over one work buffer, in one graph and in two, replayed in turn."""
    a, b = Batch(3, [1000, 50], [1, 100], 2, 2, 32), Batch(4, [600, 333], [90, 1], 2, 2, 32)
    ba, bb = a.buffers(ctx), b.buffers(ctx)
    work = a.work if a.work.nbytes >= b.work.nbytes else b.work
    ba[9].buf = bb[9].buf = work
    k = ctx.load_kernel("attn_blocks_e4m3_d128")
    ctx.dispatch(k, ba, *a.call(0))
    ctx.dispatch(k, bb, *b.call(0))
    ctx.sync()
    want = a.out.read(), b.out.read()
    a.check(want[0], 0)
    b.check(want[1], 0)

    def both(at):
        for _ in range(4):
            at.dispatch(k, ba, *a.call(0))
            at.dispatch(k, bb, *b.call(0))

    graphs = [ctx.record_graph(both), ctx.record_graph(lambda at: at.dispatch(k, ba, *a.call(0))), ctx.record_graph(lambda at: at.dispatch(k, bb, *b.call(0)))]
    a.out.zero()
    b.out.zero()
    for g in graphs + graphs[::-1]:
        ctx.submit(g)
    ctx.sync()
    assert np.array_equal(a.out.read(), want[0]) and np.array_equal(b.out.read(), want[1])


def test_work_of_a_larger_grid_serves_a_smaller_one(ctx):
    sizes = [ctx.attn_blocks_work_bytes(kv, 2, r, n, q) for kv, r, n, q in ((1, 1, 1, 1), (16, 1, 1, 1), (1000, 1, 1, 1), (1000, 64, 1, 1), (1000, 64, 64, 1), (1000, 64, 640, 10), (1000, 64, 6400, 100))]
    assert sizes == sorted(sizes) and sizes[0] > 0


# ---- together ------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("recorded", [False, True])
def test_a_server_plans_appends_and_attends(ctx, recorded):
    """Twelve steps of four requests over a pool that is too small for all: prompts, single tokens, a draft that is cut back, requests
    that end and make room.  All lengths and tables stay on the device; recorded, one graph serves every step."""
    page, stride, kv, group, requests, tokens, pages = 16, 12, 2, 2, 4, 96, 17
    rng = np.random.default_rng(11)
    up, new_u32 = ctx.buffer_from_iter, lambda n: ctx.new_buffer(n, np.uint32)
    b = {"ctx": new_u32(requests), "new": new_u32(requests), "held": new_u32(requests), "count": up(_u32([pages, 0, 0, 0])), "free": up(_u32(rng.permutation(pages))),
         "table": up(np.full(requests * stride, NONE, np.uint32)), "starts": new_u32(requests + 1), "lens": new_u32(requests), "slots": new_u32(tokens), "at": new_u32(tokens),
         "q": ctx.new_buffer(tokens * kv * group * D, np.uint16), "k": ctx.new_buffer(tokens * kv * D, np.uint16), "v": ctx.new_buffer(tokens * kv * D, np.uint16),
         "out": ctx.new_buffer(tokens * kv * group * D, np.uint16), "work": ctx.new_buffer(ctx.attn_blocks_work_bytes(kv, group, requests, tokens, tokens), np.uint8)}
    blocks = pages * page // TILE
    host = {s: _pool(0, blocks, kv, True) for s in "kv"}
    for s in "kv":
        b[s + "p"], b[s + "e"] = up(host[s][0].reshape(-1)), up(host[s][1].reshape(-1))

    def step(at):
        g = lambda names: bind(*(b[n] for n in names.split()))  # noqa: E731
        at.dispatch(at.load_kernel("kv_block_tables"), g("ctx new held count free table held count starts lens slots at"), (page, stride), [requests, tokens, 1])
        at.dispatch(at.load_kernel("kv_append_blocks_e4m3_d128"), g("k v slots kp ke vp ve"), None, [kv, tokens, 1])
        at.dispatch(at.load_kernel("attn_blocks_e4m3_d128"), g("q kp ke vp ve table lens starts out work"), (SCALE, page, stride, 0, group, tokens), [kv, requests, tokens])

    graph = ctx.record_graph(step) if recorded else None
    held, count, free, table = np.zeros(requests, np.uint32), pages, b["free"].read(), b["table"].read().reshape(requests, stride)
    have = np.zeros(requests, np.int64)
    refusals = 0
    script = [[40, 0, 17, 1], [1, 30, 1, 1], [1, 1, 60, 1], [4, 1, 1, 1], [-2, 1, 1, 1], [1, 80, 1, 0], [1, 1, -1000, 1], [1, 50, 1, 1], [-1000, 1, 1, 1], [90, 1, 1, 3], [1, 1, 1, 1], [1, 1, 1, 1]]
    for n, want in enumerate(script):
        new = np.array([max(w, 0) for w in want])
        have = np.maximum(have + np.array([min(w, 0) for w in want]), 0)  # cut back, or ended
        b["ctx"].write(_u32(have))
        b["new"].write(_u32(new))
        x = {s: rng.standard_normal((tokens, kv * (group if s == "q" else 1), D)).astype(np.float16) for s in "qkv"}
        for s in "qkv":
            b[s].write(x[s].view(np.uint16).reshape(-1))
        if recorded:
            ctx.submit_blocking(graph)
        else:
            step(ctx)
            ctx.sync()
        p = ref.plan(have, new, held, count, free, table, page, tokens)
        for name in ("free", "starts", "lens", "slots", "at"):
            assert np.array_equal(b[name].read(), p[name]), f"step {n}: {name}"
        assert np.array_equal(b["table"].read().reshape(table.shape), p["table"]) and np.array_equal(b["held"].read(), p["held_out"]) and np.array_equal(b["count"].read(), p["free_out"])
        held, count, free, table = p["held_out"], int(p["free_out"][0]), p["free"], p["table"]
        refusals += int(p["free_out"][1])
        for s in "kv":
            ref.append(x[s], p["slots"], *host[s])
            assert np.array_equal(b[s + "p"].read().reshape(host[s][0].shape), host[s][0]), f"step {n}: {s}"
            assert np.array_equal(b[s + "e"].read().reshape(host[s][1].shape), host[s][1]), f"step {n}: {s} exponents"
        want_out, bound = ref.attend(x["q"], *host["k"], *host["v"], table, p["lens"], p["starts"], page, 0, group, SCALE)
        got = b["out"].read().view(np.float16).reshape(x["q"].shape)[:int(p["starts"][-1])]
        assert np.isfinite(got).all() and (np.abs(got - want_out[:len(got)]) <= bound[:len(got)]).all(), f"step {n}: attention"
        have = np.where(p["lens"] > 0, p["lens"], have).astype(np.int64)
    assert refusals > 0
