"""NMBlockStack's parameters, on the CPU."""
import importlib

import pytest

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("init", [0, 1, 0.5, True])
def test_gates_start_at_any_number(init):
    op = importlib.import_module("nm-spmm_amd.torch_op")
    stack = op.NMBlockStack([torch.nn.Identity(), torch.nn.Identity()], 8, gate=True, gate_init=init, device="cpu")
    assert len(stack.gate) == 2
    for g in stack.gate:
        assert g.dtype == torch.get_default_dtype() and g.requires_grad and bool((g == float(init)).all())
