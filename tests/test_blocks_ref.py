"""CPU checks of the batched cache's plain statements, and of what the launchers refuse before anything is launched."""
import os
import subprocess

import numpy as np
import pytest

import blocks_ref as ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_codes_are_e4m3s():
    import torch

    codes = torch.arange(256, dtype=torch.uint8)
    want = codes.view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(ref.E4M3, want, equal_nan=True)
    x = np.random.default_rng(1).standard_normal(20000) * 2.0 ** np.random.default_rng(2).integers(-12, 9, 20000)
    x = np.concatenate([x.clip(-448, 448).astype(np.float32), [0.0, -0.0, 2.0 ** -10, 3 * 2.0 ** -10, 448, -448, 17, 19, 432]]).astype(np.float32)
    assert np.array_equal(ref.encode(x), torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy())


@pytest.mark.parametrize("most,e", [(0.0, -15), (448 * 2.0 ** -15, -15), (449 * 2.0 ** -15, -14), (448.0, 0), (448.5, 1), (61440.0, 8), (1.75, -8), (1.76, -7)])
def test_exponent_is_the_least(most, e):
    assert ref.exponent(most) == e


def test_every_cached_value_is_an_f16_number():
    for e in range(-15, 9):
        v = ref.E4M3[:127] * 2.0 ** e
        v = v[v <= ref.LARGEST]
        assert np.array_equal(v.astype(np.float16).astype(np.float64), v)


def test_growing_a_tile_rounds_its_tokens_again():
    pool, exps = np.zeros((1, 1, 16, 128), np.uint8), np.full((1, 1), 77, np.int8)
    x = np.zeros((2, 1, 128), np.float16)
    x[0, 0, :3] = [1.0, 1.0625, 0.001]
    x[1, 0, 0] = 1000.0
    ref.append(x[:1], np.array([0]), pool, exps)
    assert exps[0, 0] == -8 and list(ref.E4M3[pool[0, 0, 0, :3]] * 2.0 ** -8) == [1.0, 1.0, 2.0 ** -10]
    ref.append(x[1:], np.array([1]), pool, exps)
    assert exps[0, 0] == 2 and list(ref.E4M3[pool[0, 0, 0, :3]] * 4) == [1.0, 1.0, 0.0] and ref.E4M3[pool[0, 0, 1, 0]] * 4 == 1024.0


def test_plan_gives_back_before_it_takes():
    table = np.arange(12, dtype=np.uint32).reshape(3, 4)
    got = ref.plan([0, 30, 33], [0, 3, 0], [4, 2, 3], 0, np.zeros(8, np.uint32), table, 16, 5)
    assert list(got["held_out"]) == [0, 3, 3] and got["table"][1, 2] == 3 and list(got["free_out"]) == [3, 0, 3, 1]
    assert list(got["slots"]) == [5 * 16 + 14, 5 * 16 + 15, 3 * 16, ref.NONE, ref.NONE] and list(got["lens"]) == [0, 33, 33]


def test_launchers_refuse_before_they_launch(tmp_path):
    """Bad grids, sizes, pages and alignments come back as validation errors on a machine without a GPU: nothing was launched."""
    from super_gemma_b200 import build

    lib = build.build()
    exe = str(tmp_path / "refusals")
    cuda = os.path.join(os.path.dirname(os.path.dirname(build._nvcc())), "include")
    r = subprocess.run(["g++", "-std=c++17", "-I", cuda, "-I", os.path.join(ROOT, "super_gemma_b200", "csrc"), os.path.join(ROOT, "tests", "cpp", "blocks_refusals.cpp"),
                        lib, "-Wl,-rpath," + os.path.dirname(lib), "-o", exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
    assert r.stdout.strip().endswith("refused as they should be")
