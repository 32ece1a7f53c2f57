"""GPU tests of the rows of cosines and sines against whole-number angles: bounds counted from the kernel's own roundings, in which a small sine keeps its digits."""
import numpy as np
import pytest

import around_exact as exact
import around_ref as around
from cases import bind

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    import super_gemma_b200 as sg

    return sg.GpuContext(0)


def _rows(ctx, positions, freqs, magnitude):
    n, pairs = len(positions), len(freqs)
    out = ctx.buffer_from_iter(np.full(n * pairs * 2, 7.5, np.float32))
    ctx.dispatch_blocking(ctx.load_kernel("rope_cos_sin"), bind(ctx.buffer_from_iter(np.asarray(freqs, np.float64)), ctx.buffer_from_iter(np.asarray(positions, np.int64).astype(np.uint32)), out),
                          (2 * pairs, float(magnitude)), [n, 1, 1])
    return out.read().reshape(n, pairs, 2)


def _check(got, want, bound, what):
    over = np.abs(got.astype(np.float64) - want) - bound
    assert (over <= 0).all(), f"{what}: {over.max()} beyond the bound at {np.unravel_index(over.argmax(), over.shape)}, {got.flat[over.argmax()]} for {want.flat[over.argmax()]}"


@pytest.mark.parametrize("theta", [1e4, 1e6, 1e7, 5e9])
@pytest.mark.parametrize("magnitude", [1.0, 0.3, 1.2079442])
def test_angles_near_and_far(ctx, theta, magnitude):
    positions = [0, 1, -1, 2, 3, 17, 4095, -4096, 131071, 1 << 20, 123456789, (1 << 31) - 1, -(1 << 31), *np.random.default_rng(int(theta)).integers(-(1 << 31), 1 << 31, 30)]
    freqs = around.frequencies(64, theta, 128)
    _check(_rows(ctx, positions, freqs, magnitude), *exact.cos_sin(positions, freqs, magnitude), f"{theta}")


def test_small_sines_keep_their_digits(ctx):
    """A slow pair in the first tokens: its sine is right to 8 roundings of itself, far below 2^-32 of a turn."""
    freqs = [1e7 ** (-126 / 128), 2.0 ** -24, 1e-9, 3e-12, -1e-10, 1.0, 0.5, -2.0]
    positions = [1, 2, -1, 5, 100]
    got, (want, bound) = _rows(ctx, positions, freqs, 1.0), exact.cos_sin(positions, freqs, 1.0)
    _check(got, want, bound, "small")
    at = np.array(positions)[:, None] * np.array(freqs)[:3]
    assert np.abs(got[:, :3, 1] / np.sin(at) - 1).max() <= 8 * exact.U


def test_angles_around_the_quarters(ctx):
    """Angles a few 2^-32 turns on either side of every eighth of a turn, where a quarter is chosen, and of every quarter, where sine or cosine is near 0."""
    freqs = [2 * np.pi * 2.0 ** -32, -2 * np.pi * 2.0 ** -32, 2 * np.pi * 2.0 ** -31, 1.0, 0.1, 0.01, 1e-3, 1e-4]
    positions = [s * (k * (1 << 29) + d) for k in range(4) for d in (-130, -2, -1, 0, 1, 2, 129) for s in (1, -1)]
    _check(_rows(ctx, positions, freqs, 1.0), *exact.cos_sin(positions, freqs, 1.0), "quarters")


@pytest.mark.parametrize("tokens,pairs", [(40000, 8), (20000, 40)])
def test_angles_of_many_tokens(ctx, tokens, pairs):
    """Eight tokens a thread: 200 of the rows against whole numbers, all of them against calls of a few."""
    rng = np.random.default_rng(tokens)
    positions, freqs = rng.integers(-(1 << 24), 1 << 24, tokens), around.frequencies(pairs, 1e6, 2 * pairs)
    got, some = _rows(ctx, positions, freqs, 1.1), rng.choice(tokens, 200, replace=False)
    _check(got[some], *exact.cos_sin(positions[some], freqs, 1.1), "some")
    for first in range(0, tokens, 997):
        assert np.array_equal(got[first:first + 997], _rows(ctx, positions[first:first + 997], freqs, 1.1)), first
