"""GPU tests of the batched cache at the ends of what a dispatch takes: 65536 requests, a table row of 2097152 pages."""
import numpy as np
import pytest

import blocks_ref as ref
from cases import bind
from test_gpu_blocks import D, SCALE, TILE, _run_plan, _u32, ctx  # noqa: F401

pytestmark = pytest.mark.gpu
NONE = ref.NONE


@pytest.mark.parametrize("in_place", [False, True])
def test_block_tables_of_the_most_requests(ctx, in_place):  # noqa: F811
    rng = np.random.default_rng(1)
    n, page, stride, tokens = 65536, 16, 2, 70000
    lens, new = rng.integers(0, 31, n), np.where(rng.random(n) < 0.9, 1, rng.integers(0, 4, n))
    held = np.minimum(-(-lens // page) + (rng.random(n) < 0.1), stride)
    order = rng.permutation(int(held.sum()) + 3000).astype(np.uint32)
    table = np.full((n, stride), NONE, np.uint32)
    at = np.concatenate([[0], np.cumsum(held)])
    for j in range(stride):
        rows = held > j
        table[rows, j] = order[at[:-1][rows] + j]
    lst = np.full(len(order) + 1, 0xDEAD, np.uint32)
    lst[:3000] = order[at[-1]:]
    state = (lens, new, held, 3000, lst, table)
    want = ref.plan(*state, page, tokens)
    got, _ = _run_plan(ctx, state, page, tokens, in_place)
    assert want["free_out"][1] > 0
    for name, w in want.items():
        assert np.array_equal(got[name], w), name


def test_block_tables_of_the_longest_row(ctx):  # noqa: F811
    """A request takes all pages of a row but one in one step, and gives them back in the next."""
    page, stride = 16, 1 << 21
    pages = np.random.default_rng(2).permutation(stride + 5).astype(np.uint32)
    table = np.full((2, stride), NONE, np.uint32)
    state = [np.array([0, 0]), np.array([0, 3]), np.array([0, 0]), len(pages), pages, table]
    state[0][0] = (stride - 1) * page  # cached elsewhere so far: a table row is all that it lacks
    got, _ = _run_plan(ctx, tuple(state), page, 3)
    n = stride - 1
    assert np.array_equal(got["table"][0, :n], pages[::-1][:n]) and got["table"][0, n] == NONE and got["table"][1, 0] == pages[::-1][n]
    assert list(got["held_out"]) == [n, 1] and list(got["free_out"]) == [5, 0, 3, n + 1] and list(got["lens"]) == [n * page, 3]
    back = (np.array([0, 3]), np.array([0, 1]), got["held_out"], 5, got["free"], got["table"])
    again, _ = _run_plan(ctx, back, page, 3)
    assert list(again["held_out"]) == [0, 1] and list(again["free_out"]) == [5 + n, 0, 1, 0]
    assert np.array_equal(again["free"][5:5 + n], pages[::-1][:n]) and again["slots"][0] == int(pages[::-1][n]) * page + 3


@pytest.mark.parametrize("idle", [False, True])
@pytest.mark.parametrize("group,most", [(1, 1), (2, 4)])
def test_attention_of_the_most_requests(ctx, group, most, idle):  # noqa: F811
    """65536 requests of up to 16 keys, of one token or a draft each; or most of them without a token."""
    rng = np.random.default_rng(3)
    n = 65536
    new = rng.integers(1, most + 1, n)
    if idle:
        new[rng.random(n) < 0.99] = 0
    lens = np.maximum(rng.integers(1, TILE + 1, n), new)
    starts = np.concatenate([[0], np.cumsum(new)])
    table = rng.permutation(n)  # one page of one tile each
    codes = {s: rng.integers(0x20, 0x60, (n, TILE, D)) | rng.integers(0, 2, (n, TILE, D)) << 7 for s in "kv"}
    exps = {s: rng.integers(-4, 0, n) for s in "kv"}
    q = rng.standard_normal((int(starts[-1]), group, D)).astype(np.float16)
    up = ctx.buffer_from_iter
    out, work = up(np.full(q.size, 0x5555, np.uint16)), ctx.new_buffer(ctx.attn_blocks_work_bytes(1, group, n, len(q), most), np.uint8)
    ctx.dispatch_blocking(ctx.load_kernel("attn_blocks_e4m3_d128"),
                          bind(up(q), up(codes["k"].astype(np.uint8).reshape(-1)), up(exps["k"].astype(np.int8)), up(codes["v"].astype(np.uint8).reshape(-1)), up(exps["v"].astype(np.int8)),
                               up(_u32(table)), up(_u32(lens)), up(_u32(starts)), out, work), (SCALE, 16, 1, 0, group, most), [1, n, len(q)])
    got = out.read().view(np.float16).reshape(q.shape).astype(np.float64)
    owner = np.repeat(np.arange(n), new)
    pos = lens[owner] - new[owner] + np.arange(len(q)) - starts[owner]
    tile = table[owner]
    worst = 0.0
    for a in range(0, len(q), 8192):
        o = slice(a, a + 8192)
        k, v = (ref.E4M3[codes[s][tile[o]]] * 2.0 ** exps[s][tile[o]][:, None, None] for s in "kv")
        s = np.einsum("ngd,ntd->ngt", q[o].astype(np.float64), k) * SCALE
        s = np.where(np.arange(TILE) <= pos[o][:, None, None], s, -np.inf)
        p = np.exp(s - s.max(-1, keepdims=True))
        p /= p.sum(-1, keepdims=True)
        want, spread = np.einsum("ngt,ntd->ngd", p, v), np.einsum("ngt,ntd->ngd", p, np.abs(v))
        # weights and result in f16, 2^-11 each; scores: 128 products' sum in f32
        reach = (np.einsum("ngd,ntd->ngt", np.abs(q[o]).astype(np.float64), np.abs(k)) * SCALE).max(-1, keepdims=True)
        bound = 2.0 ** -11 * 1.01 * (spread + np.abs(want)) + 2 * spread * (128 * 2.0 ** -23 * reach + 2.0 ** -19) + 2.0 ** -25
        assert (np.abs(want) > bound).mean() > 0.9
        worst = max(worst, (np.abs(got[o] - want) / bound).max())
    assert worst <= 1, worst
