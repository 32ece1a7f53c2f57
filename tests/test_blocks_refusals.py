"""CPU checks of what the batched cache's attention refuses, beside those of test_blocks_ref.py."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_scales_that_are_refused(tmp_path):
    from super_gemma_b200 import build

    lib, exe = build.build(), str(tmp_path / "scales")
    cuda = os.path.join(os.path.dirname(os.path.dirname(build._nvcc())), "include")
    subprocess.run(["g++", "-std=c++17", "-I", cuda, "-I", os.path.join(ROOT, "super_gemma_b200", "csrc"), os.path.join(ROOT, "tests", "cpp", "blocks_scales.cpp"),
                    lib, "-Wl,-rpath," + os.path.dirname(lib), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
