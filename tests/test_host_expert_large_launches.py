"""More tiles of the experts' products than one launch can have, without a GPU: the built library against the stand-in for the HIP runtime
(tests/host/expert_large_launch_driver.cpp)."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIBDIR = os.path.join(ROOT, "aws_ofi_nccl_amd", "lib")


@pytest.fixture(scope="module")
def driver(tmp_path_factory):
    if not shutil.which("g++"):
        pytest.skip("no host compiler")
    if not os.path.exists(os.path.join(LIBDIR, "libofi_amd_hotpath.so")):
        from aws_ofi_nccl_amd import build
        build.build_library()
    exe = os.path.join(tmp_path_factory.mktemp("launches"), "expert_large_launch_driver")
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-D__HIP_PLATFORM_AMD__", "-I", "/opt/rocm/include",
                    "-I", os.path.join(ROOT, "include"), os.path.join(ROOT, "tests", "host", "expert_large_launch_driver.cpp"),
                    "-rdynamic", "-pthread", "-L", LIBDIR, "-l:libofi_amd_hotpath.so", "-Wl,-rpath," + LIBDIR, "-Wl,-rpath,/opt/rocm/lib",
                    "-Wl,--allow-shlib-undefined", "-o", exe], check=True)
    return exe


@pytest.mark.parametrize("part", ["large", "refused"])
def test_launches(driver, part):
    proc = subprocess.run([driver, part], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=120)
    assert proc.returncode == 0 and part + ": ok" in proc.stdout, proc.stdout[-4000:]
