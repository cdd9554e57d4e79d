"""ofi_amd_token_dispatch where the counts of its tiles are summed up by a launch of its own: beyond 128 tiles of 8192 pairs."""
import pytest

from test_gpu_token_dispatch import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pairs", [1 << 20, (1 << 20) + 1, 1100003, 2000000, 4194305])
@pytest.mark.parametrize("experts", [1, 15, 17, 1000, 1024])
def test_many_tiles(lib, gpu, pairs, experts):
    check(lib, pairs, 1, experts, seed=pairs + experts, wide=experts % 2 == 0, row_bytes=0, pairs=experts != 15)


def test_many_tiles_with_rows_scales_and_a_capacity(lib, gpu):
    check(lib, 150001, 8, 60, seed=1, row_bytes=16, scale_bytes=4, max_rows=1000003)
    check(lib, 150001, 8, 60, seed=2, row_bytes=16, skew=False)
