"""aws_ofi_nccl_amd.expert_exchange with gated experts of the library: forward, gradients of rows and of weights, over the put path."""
import pytest

from aws_ofi_nccl_amd import expert_exchange

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("argv", [[], ["--tokens", "77", "--width", "384", "--experts", "6", "--top-k", "3", "--ranks", "4", "--inner", "136"],
                                  ["--tokens", "9", "--width", "200", "--experts", "5", "--top-k", "2", "--ranks", "2", "--inner", "72"]])
@pytest.mark.parametrize("kept", ["8", "16"])
def test_gated_experts(gpu, capsys, argv, kept):
    assert expert_exchange.main(argv + ["--gated", kept]) == 0, capsys.readouterr().out


def test_checkpoints_have_8_or_16_bits(gpu):
    with pytest.raises(SystemExit):
        expert_exchange.main(["--gated", "4"])
