"""ofi_amd_token_dispatch into buffers with room for far more rows than the call has pairs."""
import pytest

from test_gpu_token_dispatch import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("most", [1 << 12, 1 << 16, (1 << 20) + 3, 5000001])
@pytest.mark.parametrize("tokens", [1, 5, 250, 600, 1025, 9000])
@pytest.mark.parametrize("row_bytes", [0, 16])
def test_rows_without_pairs(lib, gpu, tokens, most, row_bytes):
    check(lib, tokens, 2, 33, max_rows=most, row_bytes=row_bytes, scale_bytes=4 if row_bytes else 0, invalid=0.3, seed=tokens)
    check(lib, tokens, 2, 33, max_rows=most, row_bytes=row_bytes, invalid=1.0, seed=tokens)


def test_more_rows_than_the_workgroups_take_at_once(lib, gpu):
    for tokens in (3, 4000):
        check(lib, tokens, 1, 9, max_rows=100000007, row_bytes=0, seed=tokens)
