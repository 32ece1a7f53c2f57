"""CPU checks of what the batched cache's attention refuses, beside those of test_blocks_ref.py."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_scales_that_are_refused(tmp_path):
    from super_gemma_b200 import build

    lib, exe = build.build(), str(tmp_path / "scales")
    cuda = os.path.join(os.path.dirname(os.path.dirname(build._nvcc())), "include")
    subprocess.run(["g++", "-std=c++17", "-I", cuda, "-I", os.path.join(ROOT, "super_gemma_b200", "csrc"), os.path.join(ROOT, "tests", "cpp", "blocks_scales.cpp"),
                    lib, "-Wl,-rpath," + os.path.dirname(lib), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr


@pytest.mark.parametrize("kv,group,requests,tokens,most", [(0, 2, 3, 4, 1), (1025, 2, 3, 4, 1), (0xFFFFFFFF, 1, 1, 1, 1), (16, 0, 3, 4, 1), (16, 3, 3, 4, 1), (16, 5, 3, 4, 1), (16, 6, 3, 4, 1),
                                                           (16, 7, 3, 4, 1), (16, 9, 3, 4, 1), (16, 16, 3, 4, 1), (16, 2, 0, 4, 1), (16, 2, 65537, 70000, 1), (16, 2, 3, 0, 1), (16, 2, 3, 4, 0)])
def test_no_work_buffer_serves_what_the_dispatch_refuses(kv, group, requests, tokens, most):
    from super_gemma_b200 import build, gpu

    build.build()
    assert gpu.lib().sgb_attn_blocks_work_bytes(None, kv, group, requests, tokens, most) == 0
    assert gpu.lib().sgb_attn_blocks_work_bytes(None, 1024, 8, 65536, 70000, 1000) > 0
