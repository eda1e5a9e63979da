"""What q4_operand takes as a bias, on the CPU."""
import pytest

from conftest import nmspmm

torch = pytest.importorskip("torch")


def test_a_bias_is_float32_or_refused():
    codes, meta = (torch.zeros(4096, dtype=torch.int32) for _ in range(2))
    good = nmspmm.q4_operand(codes, meta, None, 256, 64, bias=torch.zeros(64))
    assert good.bias
    for bad in (torch.zeros(64, dtype=torch.float64), torch.zeros(128, dtype=torch.bfloat16), torch.zeros(64, dtype=torch.int32),
                torch.zeros(128)[::2], torch.zeros(63)):
        with pytest.raises(ValueError):
            nmspmm.q4_operand(codes, meta, None, 256, 64, bias=bad)
