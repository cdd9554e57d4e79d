"""What norms and token exchanges answer without a GPU: no silent CPU path, and the sizes of workspaces."""
import ctypes
import errno

import pytest

import aws_ofi_nccl_amd as m


def test_entry_points_fail_loudly_without_a_gpu(lib):
    import torch
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    p = ctypes.c_void_p(64)
    bf16, enodev = m.BFLOAT16, -errno.ENODEV
    assert lib.ofi_amd_rms_norm(p, 16, None, 0, p, bf16, 1, 8, bf16, 1e-6, p, 16, None, 0, None, 0, None, 0, 0, None, None) == enodev
    assert lib.ofi_amd_rms_norm_grad(p, 16, p, 16, p, p, bf16, 1, 8, bf16, None, 0, p, 16, None, None, 0, None) == enodev
    assert lib.ofi_amd_token_dispatch(p, m.INT32, 1, 1, 8, 1, p, p, None, None, 0, None, 0, 0, None, 0, None, 0, 0, p, 1 << 20,
                                      None) == enodev
    assert lib.ofi_amd_token_combine(p, 16, 1, p, None, 1, 1, 8, bf16, None, 0, p, 16, None) == enodev
    assert lib.ofi_amd_token_combine_grad(p, 16, p, 16, 1, p, None, 1, 1, 8, bf16, p, 16, p, None) == enodev


def test_workspaces_grow_with_their_calls_and_never_overflow(lib):
    assert lib.ofi_amd_rms_norm_grad_work_bytes(0, 100) == 0
    assert lib.ofi_amd_rms_norm_grad_work_bytes(1, 100) >= 400
    last = 0
    for rows in (1, 10, 1000, 100000, (1 << 31) - 1):
        need = lib.ofi_amd_rms_norm_grad_work_bytes(rows, 32768)
        assert last <= need <= 1024 * 32768 * 4
        last = need
    most = lib.ofi_amd_token_dispatch_work_bytes((1 << 31) - 1, 1, 1024)
    assert lib.ofi_amd_token_dispatch_work_bytes(40000, 8, 256) <= most < 1 << 40
