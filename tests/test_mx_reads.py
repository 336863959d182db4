"""CPU: what the MXFP4 products read (csrc/mx_reads.h), through the code the
kernels run, under the address sanitizer: no read of scales leaves the rows,
whatever K and however it is shared out, and no tile is one of no rows."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "apus-qwen3.6-35b-a3b_amd", "csrc")
CXX = "/opt/rocm/llvm/bin/clang++"


def test_reads_stay_in_their_operands(tmp_path):
    exe = str(tmp_path / "reads_drv")
    subprocess.run([CXX, "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined",
                    "-fno-sanitize-recover=undefined", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include",
                    "-I" + CSRC, os.path.join(ROOT, "tests", "mx_reads", "reads_drv.cpp"), "-o", exe],
                   check=True, capture_output=True)
    r = subprocess.run([exe, "8192"], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout == "ok\n", (r.stdout, r.stderr[-2000:])
