"""Norms and their gradients where a row starts between two words and is held by several wavefronts, in place and not: the bounds are those of
test_gpu_rms_norm.py."""
import pytest

from test_gpu_rms_norm import check_grad, check_norm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("in_place", [None, "x", "residual"])
@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("width", [263, 513, 1025, 1999, 2000, 8191, 8193, 16385, 32767])
@pytest.mark.parametrize("pad,shift", [(0, 0), (0, 1), (1, 0), (1, 1)])
def test_norms_in_place(lib, gpu, in_place, kind, width, pad, shift):
    check_norm(lib, 6, width, kind, 128, in_place=in_place, pad=pad, shift=shift, seed=width)


@pytest.mark.parametrize("in_place", ["x", "residual"])
@pytest.mark.parametrize("width", [513, 1999, 4097])
def test_many_norms_in_place(lib, gpu, in_place, width):
    """Beyond 2^19 chunks: two chunks a lane."""
    check_norm(lib, 9000 * 513 // width + 1100, width, "bf16", 0, in_place=in_place, train=False, seed=width)


@pytest.mark.parametrize("in_place", [None, "dout", "dsum"])
@pytest.mark.parametrize("width", [263, 513, 1999, 8191, 9001])
@pytest.mark.parametrize("rows", [6, 600])
@pytest.mark.parametrize("pad,shift", [(0, 1), (1, 0)])
def test_gradients_in_place(lib, gpu, in_place, width, rows, pad, shift):
    check_grad(lib, rows, width, "bf16", in_place=in_place, pad=pad, shift=shift, seed=width)
