"""CPU checks of what stands around the batched attention: frequencies, the plain statements, what the launchers refuse before anything is launched."""
import os
import subprocess

import numpy as np
import pytest

import around_ref as around
import blocks_ref as ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def sg():
    from super_gemma_b200 import build

    build.build()
    import super_gemma_b200 as sg

    return sg


FREQUENCIES = [(64, 1e4, 128, {}), (8, 1e6, 16, {}), (64, 1e6, 512, {}), (512, 1e4, 1024, {}), (64, 1e4, 128, {"kind": "linear", "factor": 8.0}),
               (64, 5e5, 128, {"kind": "by_turns", "factor": 8.0, "trained": 8192, "slow": 1.0, "fast": 4.0}),
               (64, 1e4, 128, {"kind": "by_pairs", "factor": 32.0, "trained": 4096, "slow": 1.0, "fast": 32.0}),
               (20, 1.5, 40, {"kind": "by_pairs", "factor": 2.0, "trained": 4096, "slow": 3.0, "fast": 3.1}),
               (32, 1e4, 64, {"kind": "by_turns", "factor": 0.5, "trained": 100, "slow": 0.5, "fast": 40.0})]


@pytest.mark.parametrize("pairs,theta,dims,more", FREQUENCIES)
def test_frequencies(sg, pairs, theta, dims, more):
    got = sg.rope_frequencies(pairs, theta, dims=dims, **more)
    want = around.frequencies(pairs, theta, dims, **more)
    assert got.shape == (pairs,) and np.abs(got / want - 1).max() <= 32 * 2.0 ** -53 * np.log(theta) * 2  # a power: its exponent's rounding counts log(theta) times
    if not more:
        assert got[0] == 1.0 and (np.diff(got) < 0).all()
    else:
        plain = around.frequencies(pairs, theta, dims)
        slowest, fastest = sorted((1.0, 1.0 / more["factor"]))
        assert (got <= plain * fastest * (1 + 1e-12)).all() and (got >= plain * slowest * (1 - 1e-12)).all()


@pytest.mark.parametrize("change", [{"pairs": 0}, {"pairs": 513}, {"pairs": -1}, {"dims": 127}, {"theta": 1.0}, {"theta": 0.0}, {"theta": float("nan")}, {"theta": float("inf")},
                                    {"kind": "other"}, {"kind": "linear", "factor": 0.0}, {"kind": "linear", "factor": float("inf")}, {"kind": "by_turns"},
                                    {"kind": "by_turns", "trained": 4096, "slow": 4.0, "fast": 4.0}, {"kind": "by_pairs", "trained": 4096, "slow": 0.0},
                                    {"kind": "by_pairs", "trained": -1.0}])
def test_frequencies_that_are_refused(sg, change):
    call = {"pairs": 64, "theta": 1e4, "factor": 2.0, **change}
    with pytest.raises(sg.Validation):
        sg.rope_frequencies(call.pop("pairs"), call.pop("theta"), **call)


def test_frequencies_refuse_null(sg):
    import ctypes as C

    assert sg.lib().sgb_rope_frequencies(None, (C.c_double * 4)()) == sg.Validation.code
    assert sg.lib().sgb_rope_frequencies(C.byref(sg.gpu._RopeScaling(4, 8, 0, 0, 1e4, 1, 0, 1, 32)), None) == sg.Validation.code


def test_a_turn_keeps_lengths_and_turns_back():
    rng = np.random.default_rng(1)
    rows, _ = around.cos_sin([5, -5, 0], around.frequencies(8, 100.0, 16), 1.0)
    x = rng.standard_normal((3, 2, 32))
    for layout in range(3):
        out, _ = around.turn(x, rows, layout)
        back, _ = around.turn(out, rows * [1, -1], layout)
        assert np.allclose(back, x) and np.allclose((out ** 2).sum(-1), (x ** 2).sum(-1)) and np.array_equal(out[2], x[2])
        still = np.setdiff1d(np.arange(32), np.concatenate(around.pair_dims(32, 8, layout)))
        assert np.array_equal(out[..., still], x[..., still])


def test_a_norm_bounds_its_row():
    """The exponents hold every normed row: one whose energy is in a single value, and spread ones."""
    w = np.ones(D := 128, np.float32)
    x = np.zeros((3, D))
    x[0, 7], x[1] = 60000.0, np.random.default_rng(2).standard_normal(D)
    ek, ev = around.exponents(w * np.float32(3.0), 1.25)
    assert np.abs(around.norm128(x, w * 3)).max() * 1.25 <= 448 * 2.0 ** ek and np.abs(around.norm128(x, None)).max() <= 448 * 2.0 ** ev
    assert (ek, ev) == (-3, -5) and around.exponents(w * 0, 1.0)[0] == ref.LOWEST and around.exponents(w * np.float32(1e30), 1.0)[0] == 8


def test_a_loose_exponent_costs_no_digits():
    """Keys quantised with the bound's exponent are as near as with that of their largest value: both carry four significant bits."""
    rng = np.random.default_rng(3)
    w = (1 + 0.2 * rng.standard_normal(128)).astype(np.float32)
    z = around.norm128(rng.standard_normal((4096, 128)), w)
    loose, _ = around.exponents(w, 1.0)
    tight = ref.exponent(np.abs(z).max())
    off = [np.sqrt(((ref.E4M3[ref.encode(z * 2.0 ** -e)] * 2.0 ** e - z) ** 2).mean()) for e in (loose, tight)]
    assert loose >= tight + 1 and off[0] <= off[1] * 1.001


def test_calls_that_are_refused(tmp_path):
    from super_gemma_b200 import build

    lib, exe = build.build(), str(tmp_path / "refusals")
    cuda = os.path.join(os.path.dirname(os.path.dirname(build._nvcc())), "include")
    subprocess.run(["g++", "-std=c++17", "-I", cuda, "-I", os.path.join(ROOT, "super_gemma_b200", "csrc"), os.path.join(ROOT, "tests", "cpp", "around_refusals.cpp"),
                    lib, "-Wl,-rpath," + os.path.dirname(lib), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
