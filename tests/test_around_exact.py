"""CPU checks of the statements in ``around_exact``."""
import numpy as np
import pytest

import around_exact as exact
import blocks_ref as ref


@pytest.mark.parametrize("rot", [0, 16, 64, 128])
@pytest.mark.parametrize("magnitude", [0.03, 0.25, 0.9, 1.0, 1.5])
def test_key_exponents_hold_every_key(magnitude, rot):
    """Rows whose energy is in one value, at each dim, and spread ones: none is cut, and the exponent before would cut one."""
    rng = np.random.default_rng(rot)
    k = np.concatenate([np.eye(exact.D) * 100, rng.standard_normal((200, exact.D))]).astype(np.float16)[:, None]
    w = np.where(rng.random(exact.D) < 0.5, -1.25, 1.25)
    angles = rng.uniform(0, 7, (len(k), rot // 2))
    angles[:64] = 0.0
    rows = (magnitude * np.stack([np.cos(angles), np.sin(angles)], -1)).astype(np.float32)
    e = exact.key_exponent(w, magnitude, rot)
    for layout in range(3):
        z, err = exact.keys(k, w, rows, layout)
        assert (np.abs(z) + err).max() <= 448 * 2.0 ** e
        if rot or magnitude <= 1:
            assert np.abs(z).max() > 448 * 2.0 ** (e - 1) * 0.998  # 11.336 is 0.2 % above the square root of 128
        if rot:
            a, b = np.array(exact.pairs_of(rot // 2, layout)).T
            assert np.allclose(np.hypot(z[..., a], z[..., b]), magnitude * np.hypot(*(exact.keys(k, w, rows[:, :0], layout)[0][..., i] for i in (a, b))), rtol=1e-6)


def test_a_bound_without_the_dims_that_stay_would_cut_them():
    """Rows of length 0.25 over half the head: 448 * 2^e of their bound alone is 3.5, and normed values of 4.2 are ordinary."""
    rng = np.random.default_rng(1)
    k = rng.standard_normal((4096, 1, exact.D)).astype(np.float16)
    z, _ = exact.keys(k, np.ones(exact.D), np.zeros((4096, 32, 2), np.float32), 1)
    assert np.abs(z).max() > 448 * 2.0 ** exact.key_exponent(np.ones(exact.D), 0.25, exact.D) == 3.5
    assert ref.exponent(11.336) == exact.key_exponent(np.ones(exact.D), 0.25, 64) == exact.key_exponent(np.ones(exact.D), 0.25, 0) == -5


def test_whole_number_angles():
    """Against 64-bit angles where those are good, and against the sine's own series for the smallest."""
    freqs = [1.0, 0.3, -0.25, 1e6 ** (-126 / 128), 1e-12]
    at = np.array([0, 1, -1, 1000, -77])
    want, bound = exact.cos_sin(at, freqs, 1.25)
    a = at[:, None] * np.array(freqs)
    assert np.abs(want - 1.25 * np.stack([np.cos(a), np.sin(a)], -1)).max() < 1e-12 and bound.max() < 5e-7
    assert np.allclose(want[:, 4, 1], 1.25e-12 * at, rtol=1e-14, atol=0) and (bound[1, 3] <= [3.6e-7, 1.25e-6 * 8 * exact.U * 1.25]).all()


@pytest.mark.parametrize("post,gate,scale", [(1, None, 1.0), (1, 2.5, -0.5), (0, -1.0, 0.25), (2, None, 1.0)])
def test_norms_agree_with_the_other_statement(post, gate, scale):
    """Two statements written apart give the same values, and the bound counted here is the tighter one."""
    import around_ref as around

    rng = np.random.default_rng(post)
    y, h, w, v = (rng.standard_normal(s) for s in ((5, 48), (5, 48), (48,), (48,)))
    g = None if gate is None else np.full((5, 1), gate)
    here, there = exact.block_norms(y, h, w, g, v, post, scale, 1e-6), around.block_norms(y, h, w, g, v, post, scale, 1e-6)
    assert all(np.allclose(here[i], there[i], rtol=1e-13, atol=1e-13) for i in (0, 2))
    assert (here[3] <= there[3]).all() and (here[1] <= there[1] * 1.001).all()
