"""GPU tests of what stands around the batched attention at the ends of its documented ranges, and of a first call that is recorded."""
import os
import subprocess
import sys

import numpy as np
import pytest

import around_ref as around
import blocks_ref as ref
import test_gpu_around as base

pytestmark = pytest.mark.gpu
TILE, D = ref.TILE, ref.D


@pytest.fixture(scope="module")
def ctx():
    import super_gemma_b200 as sg

    return sg.GpuContext(0)


def _read_back(ctx, pools, table, first, lengths, page, kv):
    starts = np.concatenate([[0], np.cumsum(lengths)])
    got = base._read(ctx, [ctx.buffer_from_iter(p.reshape(-1)) for p in pools], table, first, starts, kv, page, int(starts[-1]) + 3)
    r = np.repeat(np.arange(len(lengths)), lengths)
    t = np.arange(starts[-1]) - starts[r] + np.asarray(first)[r]
    rows = table[r, t // page].astype(np.int64) * page + t % page
    for g, pool, exps in zip(got, pools[::2], pools[1::2]):
        want = ref.E4M3[pool[rows // TILE, :, rows % TILE]] * 2.0 ** exps[rows // TILE].astype(np.float64)[:, :, None]
        with np.errstate(over="ignore"):
            assert np.array_equal(g[:starts[-1]], want.astype(np.float16))


def test_reading_65536_requests(ctx):
    """Most of them empty, alone and many in a row; pages shared by many."""
    rng = np.random.default_rng(1)
    lengths = np.where(rng.random(65536) < 0.3, rng.integers(0, 4, 65536), 0)
    lengths[[0, 1, 65535]] = 0, 3, 2
    lengths[20000:30000] = 0
    _read_back(ctx, [*base._pool(rng, 64, 1), *base._pool(rng, 64, 1)], rng.integers(0, 64, (65536, 1)), rng.integers(0, 12, 65536), lengths, 16, 1)


def test_reading_1024_heads(ctx):
    rng = np.random.default_rng(2)
    _read_back(ctx, [*base._pool(rng, 5, 1024), *base._pool(rng, 5, 1024)], rng.permutation(5)[None, :].repeat(3, 0), [0, 30, 61], [20, 1, 18], 16, 1024)


@pytest.mark.parametrize("page", [1 << 16, 1 << 31])
def test_reading_a_page_larger_than_the_pool(ctx, page):
    rng = np.random.default_rng(3)
    _read_back(ctx, [*base._pool(rng, 9, 2), *base._pool(rng, 9, 2)], np.zeros((2, 1), np.int64), [0, 100], [70, 44], page, 2)


@pytest.mark.parametrize("layout", [0, 1, 2])
@pytest.mark.parametrize("tokens,heads,kv,head_dim,rot", [(3, 4096, 4096, 16, 16), (2, 4096, 1, 1024, 512), (70001, 1, 0, 16, 16), (1, 1, 4096, 48, 16)])
def test_rotation_of_the_most_heads(ctx, tokens, heads, kv, head_dim, rot, layout):
    rng = np.random.default_rng(tokens)
    q, k = (rng.standard_normal((tokens, h, head_dim)).astype(np.float16) for h in (heads, kv))
    rows = around.cos_sin(rng.integers(0, 100000, tokens), around.frequencies(rot // 2, 1e4, rot), 1.0)[0].astype(np.float32)
    for in_place in (False, True):
        for x, got in zip((q, k), base._rotate(ctx, q, k, rows, layout, in_place=in_place)):
            want, err = around.turn(x, rows, layout)
            base._within(got, want, err + around.f16_step(want))


@pytest.mark.parametrize("tokens,heads,kv", [(70_001, 1, 1), (33, 8192, 1), (33, 1, 1024)])
def test_pre_attention_at_the_ends_of_its_grid(ctx, tokens, heads, kv):
    base.Step(tokens, base._runs(tokens, [(9, tokens)], tokens // TILE + 2, True), heads, kv, tokens // TILE + 2, layout=kv % 3).run(ctx)


FIRST = """
import sys
sys.path[:0] = {path!r}
import numpy as np
import super_gemma_b200 as sg
from cases import bind
ctx, rng = sg.GpuContext(0), np.random.default_rng(1)
rows, hidden = 2001, 5376
up = ctx.buffer_from_iter
y, h = (up(rng.standard_normal(rows * hidden).astype(np.float16).view(np.uint16)) for _ in range(2))
w = up(rng.standard_normal(hidden).astype(np.float32))
out = [ctx.new_buffer(rows * hidden, np.uint16) for _ in range(4)]
call = lambda i: (ctx.load_kernel("block_norms_f16"), bind(y, h, w, w, w, out[i], out[i + 1]), (1, 1, 0, 0.5, 1e-6), [hidden, rows, 1])
graph = ctx.record_graph(lambda at: at.dispatch(*call(0)))
ctx.submit_blocking(graph)
ctx.dispatch_blocking(*call(2))
assert all(np.array_equal(out[i].read(), out[i + 2].read()) and out[i].read().any() for i in range(2))
print("recorded first")
"""


def test_a_first_call_that_is_recorded():
    """Rows that come ahead ask for their kernel's registers at the first call: in a new process, within a recording."""
    here = os.path.dirname(os.path.abspath(__file__))
    r = subprocess.run([sys.executable, "-c", FIRST.format(path=[os.path.dirname(here), here])], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "recorded first" in r.stdout, r.stdout + r.stderr
