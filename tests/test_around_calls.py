"""CPU checks of calls around the batched attention that nobody should make: what they are answered before anything is launched or written."""
import pytest


@pytest.fixture(scope="module")
def sg():
    from super_gemma_b200 import build

    build.build()
    import super_gemma_b200 as sg

    return sg


# Numbers whose lower 32 bits would be good ones among them: the array is as long as `pairs` says and the library writes as many numbers as its word says.
@pytest.mark.parametrize("change", [{"dims": -2}, {"dims": 2 ** 32}, {"dims": 2 ** 32 + 128}, {"dims": -2 ** 32 + 128}, {"pairs": 2 ** 32 + 64, "dims": 128}, {"pairs": -2 ** 32 + 64, "dims": 128},
                                    {"pairs": -2 ** 32 + 64}, {"pairs": 513, "dims": 2 ** 31}])
def test_frequencies_beyond_32_bits_are_refused(sg, monkeypatch, change):
    monkeypatch.setattr(sg.gpu, "lib", lambda: pytest.fail("the library was called"))
    call = {"pairs": 64, "theta": 1e4, **change}
    with pytest.raises(sg.Validation):
        sg.rope_frequencies(call.pop("pairs"), call.pop("theta"), **call)


def test_frequencies_at_the_limits(sg):
    assert sg.rope_frequencies(512, 1e4).shape == (512,) and sg.rope_frequencies(1, 1e4, dims=2 ** 32 - 1).tolist() == [1.0]


def test_groups_of_any_kind(sg):
    """Grids shorter or longer than three words, out of lists, tuples, arrays and iterators, reach the library as the same three words."""
    import struct

    import numpy as np

    ctx, seen = object.__new__(sg.GpuContext), []
    ctx._h = None  # (no context: nothing is called but the stand-in below)
    kernel = type("K", (), {"_h": None})()

    def dispatch(_ctx, _kernel, bindings, n, push, push_bytes, groups):
        seen.append(struct.unpack("3I", groups))
        return 0

    for want, words in (((5, 1, 1), [5]), ((5, 7, 1), [5, 7]), ((5, 7, 9), [5, 7, 9]), ((5, 7, 9), [5, 7, 9, 11])):
        for groups in (words, tuple(words), np.array(words), iter(words), (w for w in words)):
            ctx._dispatch(dispatch, kernel, [], None, groups)
            assert seen.pop() == want, (words, type(groups))


def test_overlaps_that_are_refused(sg, tmp_path):
    import os
    import subprocess

    from super_gemma_b200 import build

    root, lib, exe = os.path.dirname(os.path.dirname(os.path.abspath(__file__))), build.build(), str(tmp_path / "overlaps")
    cuda = os.path.join(os.path.dirname(os.path.dirname(build._nvcc())), "include")
    subprocess.run(["g++", "-std=c++17", "-I", cuda, "-I", os.path.join(root, "super_gemma_b200", "csrc"), os.path.join(root, "tests", "cpp", "around_overlaps.cpp"),
                    lib, "-Wl,-rpath," + os.path.dirname(lib), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
