"""The experts' products in buffers with room for many more rows than there are: which variant runs goes by the room, what it computes by the rows,
and nothing of the room is touched."""
import pytest

from _experts import check_gated, check_hidden, check_product, check_rows, check_weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("counts", [[1], [0, 8, 0, 3], [0, 0], [70, 1, 0, 200]])
@pytest.mark.parametrize("spare", [600, 20000])
def test_room_for_many_more_rows(lib, gpu, counts, spare):
    check_gated(lib, counts, 264, 200, "bf16", "bf16", "e4m3", spare=spare)
    check_gated(lib, counts, 272, 2176, "e4m3", "e4m3", spare=spare)
    check_product(lib, counts, 136, 4104, "f16", a="gelu", residual=True, spare=spare)
    check_hidden(lib, counts, 136, 2056, "bf16", "e4m3", spare=spare)
    check_rows(lib, counts, 2056, 136, "f16", added=True, spare=spare)
    check_weights(lib, counts, 520, 264, "bf16", "f32", added=True, bias=True, spare=spare)
    check_hidden(lib, counts, 77, 130, "f16", "f16", False, "gelu", spare=spare)
    check_rows(lib, counts, 129, 63, "bf16", spare=spare)
    check_weights(lib, counts, 77, 130, "f16", "f16", bias=True, spare=spare)
