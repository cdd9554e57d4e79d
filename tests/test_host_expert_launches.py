"""What the experts' products launch and refuse, without a GPU: the built library against the stand-in for the HIP runtime
(tests/host/expert_launch_driver.cpp), from one row to the most that are taken."""
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
    exe = os.path.join(tmp_path_factory.mktemp("launches"), "expert_launch_driver")
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-D__HIP_PLATFORM_AMD__", "-I", "/opt/rocm/include",
                    "-I", os.path.join(ROOT, "include"), os.path.join(ROOT, "tests", "host", "expert_launch_driver.cpp"),
                    "-rdynamic", "-pthread", "-L", LIBDIR, "-l:libofi_amd_hotpath.so", "-Wl,-rpath," + LIBDIR, "-Wl,-rpath,/opt/rocm/lib",
                    "-Wl,--allow-shlib-undefined", "-o", exe], check=True)
    return exe


@pytest.mark.parametrize("part", ["spreads", "refusals"])
def test_launches(driver, part):
    proc = subprocess.run([driver, part], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=120)
    assert proc.returncode == 0 and part + ": ok" in proc.stdout, proc.stdout[-4000:]


def test_entry_points_fail_loudly_without_a_gpu(lib):
    import ctypes
    import errno
    import torch
    import aws_ofi_nccl_amd as m
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    p, enodev, bf16 = ctypes.c_void_p(64), -errno.ENODEV, m.BFLOAT16
    weight = p, 128, 128 * 128
    assert lib.ofi_amd_expert_gated(p, 128, None, 0, bf16, p, 1, 1, *weight, None, 64, 64, m.SILU, p, 128, bf16, None, 0, None, 0, 0, None, 0,
                                    None) == enodev
    assert lib.ofi_amd_expert_product(p, 128, None, 0, bf16, p, 1, 1, *weight, None, 64, 64, None, 0, 0, None, 0, p, 128, bf16, None, 0, None, 0, 0,
                                      None, 0, None) == enodev
    assert lib.ofi_amd_expert_hidden_grad(p, 128, bf16, p, 1, 1, *weight, 64, 64, 1, m.SILU, p, 256, bf16, None, 0, p, 256, None, 0, None) == enodev
    assert lib.ofi_amd_expert_rows_grad(p, 128, bf16, p, 1, 1, *weight, 64, 64, None, 0, p, 128, None) == enodev
    assert lib.ofi_amd_expert_weight_grad(p, 128, p, 128, bf16, p, 1, 1, 64, 64, None, *weight, bf16, None, None, None) == enodev
