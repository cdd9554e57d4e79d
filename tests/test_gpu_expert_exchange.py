"""The layer of aws_ofi_nccl_amd.expert_exchange, forward and backward through the put path, against the formulas in 64 bits."""
import pytest

from aws_ofi_nccl_amd import expert_exchange

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("argv", [[], ["--tokens", "1", "--top-k", "2"], ["--tokens", "333", "--width", "520", "--experts", "10", "--ranks", "3"],
                                  ["--tokens", "2500", "--width", "256", "--experts", "6", "--ranks", "6", "--top-k", "6", "--inner", "64"]])
def test_layer(lib, gpu, argv, capsys):
    assert expert_exchange.main(argv) == 0, capsys.readouterr().out


def test_refuses_sizes_that_make_no_layer(capsys):
    for argv in (["--ranks", "9", "--experts", "8"], ["--top-k", "0"], ["--tokens", "0"]):
        with pytest.raises(SystemExit):
            expert_exchange.main(argv)
    capsys.readouterr()
