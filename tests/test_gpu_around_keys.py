"""GPU tests of the keys that the pre-attention pass caches: no value is cut, whatever the rows' magnitude and however much of the head turns."""
import numpy as np
import pytest

import around_exact as exact
import blocks_ref as ref
from cases import bind

pytestmark = pytest.mark.gpu
TILE, D = ref.TILE, ref.D


@pytest.fixture(scope="module")
def ctx():
    import super_gemma_b200 as sg

    return sg.GpuContext(0)


@pytest.mark.parametrize("layout", [0, 1, 2])
@pytest.mark.parametrize("rot", [0, 64, 112, 128])
@pytest.mark.parametrize("magnitude", [0.03, 0.1, 0.25, 0.9, 1.0, 1.5])
def test_keys_fit_their_exponent(ctx, magnitude, rot, layout):
    """Rows whose energy is in one value, at each dim in turn, and spread ones, into tiles that begin with them: each key within half a step of e4m3 of its value."""
    rng = np.random.default_rng(rot + layout)
    n, kv, plus_one = 128 + 80, 2, layout % 2
    k = rng.standard_normal((n, kv, D))
    k[:128] = (np.eye(D) * rng.choice([-300.0, 0.5, 40.0], (D, 1)))[:, None]
    k = k.astype(np.float16)
    w = (1 - plus_one + 0.2 * rng.standard_normal(D)).astype(np.float32)
    weight = (w + np.float32(plus_one)).astype(np.float64)
    angles = rng.uniform(0, 7, (n, rot // 2))
    angles[:64] = 0.0
    rows = (magnitude * np.stack([np.cos(angles), np.sin(angles)], -1)).astype(np.float32)
    up = ctx.buffer_from_iter
    half = lambda x: up(np.ascontiguousarray(x).view(np.uint16).reshape(-1))  # noqa: E731
    blocks = n // TILE
    pools = [up(np.full(blocks * kv * TILE * D, 0x7F, np.uint8)) for _ in range(2)]
    exps = [up(np.full(blocks * kv, 127, np.int8)) for _ in range(2)]
    slots = (rng.permutation(blocks)[:, None] * TILE + np.arange(TILE)).reshape(-1)
    ctx.dispatch_blocking(ctx.load_kernel("qkv_norm_rope_append_blocks_e4m3_d128"),
                          bind(half(k), up(w), ctx.new_buffer(n * kv * D, np.uint16), half(k), half(k), up(w), up(rows.reshape(-1)) if rot else up(np.zeros(4, np.float32)),
                               up(slots.astype(np.uint32)), pools[0], exps[0], pools[1], exps[1]), (rot, layout, plus_one, 0, 0, 0, float(magnitude)), [kv, kv, n])
    want, err = exact.keys(k, weight, rows, layout)
    e = exact.key_exponent(weight, float(np.float32(magnitude)), rot)
    assert (np.abs(want) + err).max() <= 448 * 2.0 ** e, "the statement's own exponent holds them"
    got_e = exps[0].read().view(np.int8).reshape(blocks, kv)
    assert (got_e == e).all(), (e, np.unique(got_e))
    got = ref.E4M3[pools[0].read().reshape(blocks, kv, TILE, D)[slots // TILE, :, slots % TILE]] * 2.0 ** e
    off = np.abs(got - want) - err
    assert (off <= np.maximum(2.0 ** -4 * (np.abs(want) + err), 2.0 ** (e - 10))).all(), np.unravel_index(off.argmax(), off.shape)
