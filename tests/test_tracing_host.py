"""Which calls the torch binding hands back to the dispatcher, on the CPU: None where someone else is to see the call; otherwise the
call itself, which refuses a CPU tensor."""
import importlib

import pytest

torch = pytest.importorskip("torch")
op = importlib.import_module("nm-spmm_amd.torch_op")


def handed_back(x, w=None):
    try:
        return op._binding().block_norm(x, None, None, None, 1.0, 0, None, None, 1, w, None, 1e-6, 0.0, None) is None
    except ValueError:
        return False


def during(transform, *args):
    seen = []
    transform(lambda v: (seen.append(handed_back(v)), v * 2)[1], *args)
    return seen


def test_ordinary_calls_are_taken():
    x = torch.randn((2, 8))
    assert not handed_back(x) and not handed_back(torch.nn.Parameter(x), torch.nn.Parameter(x[0]))
    assert not handed_back(torch.randn((2, 8), dtype=torch.complex64).conj().imag)
    with torch.inference_mode():
        assert not handed_back(torch.randn((2, 8)))
    with torch.no_grad(), torch.autocast("cpu"):
        assert not handed_back(x)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t):
        assert not handed_back(x)


def test_tracers_modes_transforms_and_wrappers_are_handed_back():
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx

    x = torch.randn((2, 8))
    assert all(during(lambda f: torch.jit.trace(f, x, check_trace=False)))
    assert all(during(lambda f: make_fx(f)(x)))
    assert all(during(lambda f: torch.func.vmap(f)(x)))
    assert all(during(lambda f: torch.func.grad(lambda v: f(v).sum())(x)))
    assert all(during(lambda f: torch.func.functionalize(f)(x)))
    assert all(during(lambda f: torch.func.jvp(f, (x,), (x,))))
    with FakeTensorMode(allow_non_fake_inputs=True) as mode:
        assert handed_back(x)
    assert handed_back(mode.from_tensor(x)) and handed_back(x, mode.from_tensor(x[0]))
