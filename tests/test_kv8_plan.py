"""CPU: how a prefill call on the 8-bit KV cache is cut into tiles and parts
(csrc/kv8_plan.h), through the code the library runs, under the address and
undefined-behaviour sanitizers, against what the kernels index."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "apus-qwen3.6-35b-a3b_amd", "csrc")
CXX = "/opt/rocm/llvm/bin/clang++"


@pytest.fixture(scope="module")
def exe(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("plan") / "plan_drv")
    subprocess.run([CXX, "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined",
                    "-fno-sanitize-recover=undefined", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include",
                    "-I" + CSRC, os.path.join(ROOT, "tests", "kv8_plan", "plan_drv.cpp"), "-o", out],
                   check=True, capture_output=True)
    return out


@pytest.mark.parametrize("seed", [1, 2, 3])
def test_tiles_parts_and_slots(exe, seed):
    r = subprocess.run([exe, str(seed), "3000"], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout == "ok\n", (r.stdout, r.stderr[-2000:])
