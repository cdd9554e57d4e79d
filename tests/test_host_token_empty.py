"""Empty batches and buffers, without a GPU: the built library against the stand-in for the HIP runtime
(tests/host/token_empty_driver.cpp)."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIBDIR = os.path.join(ROOT, "aws_ofi_nccl_amd", "lib")


def test_buffers_of_nothing_may_be_null(tmp_path):
    if not shutil.which("g++"):
        pytest.skip("no host compiler")
    if not os.path.exists(os.path.join(LIBDIR, "libofi_amd_hotpath.so")):
        from aws_ofi_nccl_amd import build
        build.build_library()
    exe = os.path.join(tmp_path, "token_empty_driver")
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-D__HIP_PLATFORM_AMD__", "-I", "/opt/rocm/include", "-I", os.path.join(ROOT, "include"),
                    os.path.join(ROOT, "tests", "host", "token_empty_driver.cpp"), "-rdynamic", "-pthread", "-L", LIBDIR,
                    "-l:libofi_amd_hotpath.so", "-Wl,-rpath," + LIBDIR, "-Wl,-rpath,/opt/rocm/lib", "-Wl,--allow-shlib-undefined",
                    "-o", exe], check=True)
    proc = subprocess.run([exe], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=120)
    assert proc.returncode == 0 and "empty: ok" in proc.stdout, proc.stdout[-4000:]
