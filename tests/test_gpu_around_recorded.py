"""GPU tests of recordings of what stands around the batched attention: every output is poison before every replay, and inputs change from replay to replay."""
import numpy as np
import pytest

import around_ref as around
import blocks_ref as ref
from cases import bind

pytestmark = pytest.mark.gpu
TILE, D, NONE = ref.TILE, ref.D, ref.NONE


@pytest.fixture(scope="module")
def ctx():
    import super_gemma_b200 as sg

    return sg.GpuContext(0)


class World:
    """A layer's calls over tensors of their own: angles feed the rotation and the pre-attention pass, a norm feeds its queries, its cache is read back, and the
    norms in the other two types stand beside them.  What a call writes is read by the next ones, so that a recording needs its edges."""

    def __init__(self, ctx, n, heads, kv, layout):
        self.ctx, self.n, self.heads, self.kv, self.hidden = ctx, n, heads, kv, heads * D
        self.blocks, self.b = n // TILE + 2, {}
        halves, floats = n * heads * D, n * heads * D
        for name, size, dtype in (("freqs", 64, np.float64), ("at", n, np.uint32), ("rows", n * 128, np.float32), ("q", n * heads * D, np.uint16), ("k", n * kv * D, np.uint16),
                                  ("v", n * kv * D, np.uint16), ("q_turned", n * heads * D, np.uint16), ("k_turned", n * kv * D, np.uint16), ("y", halves, np.uint16),
                                  ("h16", halves, np.uint16), ("hb", halves, np.uint16), ("h32", floats, np.float32), ("h16_out", halves, np.uint16), ("hb_out", halves, np.uint16),
                                  ("h32_out", floats, np.float32), ("x16", halves, np.uint16), ("xb", halves, np.uint16), ("x32", halves, np.uint16), ("w", self.hidden, np.float32),
                                  ("gate", n, np.float32), ("w128", D, np.float32), ("q_out", halves, np.uint16), ("slots", n, np.uint32), ("kp", self.blocks * kv * TILE * D, np.uint8),
                                  ("ke", self.blocks * kv, np.int8), ("vp", self.blocks * kv * TILE * D, np.uint8), ("ve", self.blocks * kv, np.int8), ("table", self.blocks, np.uint32),
                                  ("first", 1, np.uint32), ("starts", 2, np.uint32), ("k_read", n * kv * D, np.uint16), ("v_read", n * kv * D, np.uint16)):
            self.b[name] = ctx.new_buffer(size, dtype)
        self.written = "rows q_turned k_turned h16_out hb_out h32_out x16 xb x32 q_out kp ke vp ve k_read v_read".split()
        norms, half = (1, 2, 0, 0.5, 1e-6), [self.hidden, n, 1]
        self.calls = [("rope_cos_sin", "freqs at rows", (128, 1.25), [n, 1, 1]),
                      ("block_norms_f16", "y h16 w gate w h16_out x16", norms, half),
                      ("rope_qk_f16", "x16 k rows q_turned k_turned", (D, 128, layout, 0, 0, 0, 0), [heads, kv, n]),
                      ("block_norms_bf16", "x16 hb w gate w hb_out xb", norms, half),
                      ("qkv_norm_rope_append_blocks_e4m3_d128", "x16 w128 q_out k_turned v w128 rows slots kp ke vp ve", (128, layout, 0, 0, 0, 0, 1.25), [heads, kv, n]),
                      ("block_norms_f32", "q_out h32 w gate w h32_out x32", norms, half),
                      ("kv_read_blocks_e4m3_d128", "kp ke vp ve table first starts k_read v_read", (16, self.blocks), [kv, 1, n])]

    def fill(self, seed):
        """Inputs of a seed, and poison in whatever the calls write: NaN in rows and 16-bit tensors, codes and exponents of a used pool in the cache."""
        rng, n = np.random.default_rng(seed), self.n
        normal = lambda size: rng.standard_normal(size).astype(np.float32)  # noqa: E731
        for name, b in self.b.items():
            size = len(b)
            if name in ("kp", "vp"):
                b.write(rng.integers(0, 120, size).astype(np.uint8))
            elif name in ("ke", "ve"):
                b.write(rng.integers(-15, 0, size).astype(np.int8))
            elif name in self.written:
                b.write(np.full(size, np.nan, np.float32) if b.dtype == np.float32 else np.full(size, 0x7FFF, np.uint16))
            elif name in ("h32", "gate"):
                b.write(normal(size))
            elif name in ("w", "w128"):
                b.write(1 + 0.3 * normal(size))
            elif name == "hb":
                b.write((normal(size).view(np.uint32) >> 16).astype(np.uint16))
            elif b.dtype == np.uint16:
                b.write(normal(size).astype(np.float16).view(np.uint16))
        order, first = rng.permutation(self.blocks), int(rng.integers(1, TILE))
        at = first + np.arange(n)
        self.b["freqs"].write(around.frequencies(64, 1e4, 128) * (1 + seed % 7))
        self.b["at"].write(rng.integers(0, 1 << 20, n).astype(np.uint32))
        self.b["slots"].write((order[at // TILE] * TILE + at % TILE).astype(np.uint32))
        self.b["table"].write(order.astype(np.uint32))
        self.b["first"].write(np.array([first], np.uint32)), self.b["starts"].write(np.array([0, n], np.uint32))

    def run(self, at, blocking=False):
        for name, buffers, push, grid in self.calls:
            (at.dispatch_blocking if blocking else at.dispatch)(at.load_kernel(name), bind(*(self.b[x] for x in buffers.split())), push, grid)

    def got(self):
        return {name: self.b[name].read() for name in self.written}


@pytest.mark.parametrize("n,heads,kv", [(1, 4, 2), (90, 6, 3), (700, 8, 4)])
def test_replays_with_other_inputs(ctx, n, heads, kv):
    """Two contexts replay a recording each, side by side; a third tensor set takes the same calls one at a time."""
    import super_gemma_b200 as sg

    other = sg.GpuContext(0)
    worlds, alone = [World(c, n, heads, kv, 2 * i) for i, c in enumerate((ctx, other))], [World(ctx, n, heads, kv, 2 * i) for i in range(2)]
    graphs = [w.ctx.record_graph(w.run) for w in worlds]
    before = None
    for seed in range(6):
        for i in range(2):
            worlds[i].fill(10 * seed + i), alone[i].fill(10 * seed + i)
        ctx.sync(), other.sync()
        for w, g in zip(worlds, graphs):
            w.ctx.submit(g)
        for w in worlds:
            w.ctx.sync()
        for i in range(2):
            alone[i].run(ctx, blocking=True)
            got, want = worlds[i].got(), alone[i].got()
            for name in worlds[i].written:
                assert np.array_equal(got[name].view(np.uint8), want[name].view(np.uint8)), f"seed {seed}, context {i}: {name}"
            finite = [x.view(np.float16) for x in (want["x16"], want["q_turned"], want["q_out"], want["k_read"], want["v_read"], want["x32"], want["xb"])] + [want["rows"], want["h32_out"]]
            assert all(np.isfinite(x.astype(np.float32)).all() for x in finite), "poison was left"
        assert before is None or not np.array_equal(before, got["x32"]), "the inputs changed"
        before = got["x32"]
