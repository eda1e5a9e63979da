"""The 4-bit layer and the block norm under tracers, dispatch modes and function transforms: what is recorded is the operator, not
the memory that its result lay in, and what a transform cannot do is refused."""
import importlib

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def op():
    return importlib.import_module("nm-spmm_amd.torch_op")


class Norms(torch.nn.Module):
    def __init__(self, gate, scale):
        super().__init__()
        self.pre, self.post = (torch.nn.Parameter(torch.rand(96, device="cuda") + 0.5) for _ in range(2))
        self.gate = gate
        self.scale = scale

    def forward(self, x, y):
        return op().block_norm(x, y, gate=self.gate, residual_scale=self.scale, post="layer", post_weight=self.post, pre="rms", pre_weight=self.pre)


def norms(kind):
    gate = {"none": None, "feature": torch.rand(96, device="cuda"), "sample": torch.rand((2, 1, 96), device="cuda"),
            "broadcast": torch.rand((1, 5, 96), device="cuda")}[kind]
    return Norms(gate, torch.rand(96, device="cuda") if kind == "sample" else 0.5)


def layer(n=1, m=1):
    return op().NMQuantLinear(torch.randn((64, 96), device="cuda"), n, m, bias=torch.randn(64, device="cuda"))


def inputs(k=2):
    return [torch.randn((2, 5, 96), device="cuda") for _ in range(k)]


@pytest.mark.parametrize("n,m", [(1, 1), (2, 8)])
def test_jit_trace_of_a_layer(n, m):
    lin = layer(n, m)
    x, other = inputs()
    traced = torch.jit.trace(lin, x)
    assert "nmspmm::quant_linear" in str(traced.inlined_graph)
    assert torch.equal(traced(x), lin(x)) and torch.equal(traced(other), lin(other))


@pytest.mark.parametrize("kind", ["none", "feature", "sample", "broadcast"])
@pytest.mark.parametrize("grad", [False, True])
def test_jit_trace_of_the_norms(kind, grad):
    module = norms(kind)
    with torch.set_grad_enabled(grad):
        traced = torch.jit.trace(module, tuple(inputs()))
        assert "nmspmm::block_norm" in str(traced.inlined_graph)
        given = inputs()
        for got, want in zip(traced(*given), module(*given)):
            assert torch.equal(got, want)


@pytest.mark.parametrize("kind", ["none", "feature"])
def test_a_trace_takes_other_numbers_of_rows(kind):
    module, lin = norms(kind), layer()
    traced, traced_lin = torch.jit.trace(module, tuple(inputs())), torch.jit.trace(lin, inputs()[0])
    for shape in ((2, 7, 96), (3, 10, 96), (1, 1, 96)):
        x, y = (torch.randn(shape, device="cuda", requires_grad=True) for _ in range(2))
        got, want = traced(x, y), module(x, y)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        leaves = [x, y, module.pre, module.post]
        for a, b in zip(*(torch.autograd.grad(r[0].square().sum() + r[1].square().sum(), leaves) for r in (got, want))):
            torch.testing.assert_close(a, b)
        assert torch.equal(traced_lin(x.detach()), lin(x.detach()))


def test_jit_trace_of_a_first_norm_and_a_stack():
    stack = op().NMBlockStack([torch.nn.Sequential(layer(), torch.nn.SiLU(), op().NMQuantLinear(torch.randn((96, 64), device="cuda")))], 96)
    x, other = inputs()
    with torch.no_grad():
        traced = torch.jit.trace(stack, x)
        for got, want in zip(traced(other), stack(other)):
            assert torch.equal(got, want)


@pytest.mark.parametrize("mode", ["real", "fake", "symbolic"])
def test_make_fx(mode):
    from torch.fx.experimental.proxy_tensor import make_fx

    lin, module = layer(), norms("sample")

    def run(x, y):
        return lin(x), *module(x, y)

    with torch.no_grad():
        graph = make_fx(run, tracing_mode=mode, _allow_non_fake_inputs=True)(*inputs())
        names = [str(n.target) for n in graph.graph.nodes]
        assert any("nmspmm.quant_linear" in n for n in names) and any("nmspmm.block_norm" in n for n in names)
        given = inputs()
        for got, want in zip(graph(*given), run(*given)):
            assert torch.equal(got, want)


def test_dispatch_modes_see_the_operators():
    from torch.utils._python_dispatch import TorchDispatchMode

    seen = []

    class Watch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    lin, module = layer(), norms("feature")
    x, y = inputs()
    want = (lin(x), *module(x, y))
    with Watch():
        got = (lin(x), *module(x, y))
    assert any("nmspmm.quant_linear" in s for s in seen) and any("nmspmm.block_norm" in s for s in seen)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def matches_or_raises(f, want):
    """A transform may have no rule for an operator; then it says so."""
    try:
        got = f()
    except (RuntimeError, NotImplementedError, ValueError):
        return
    got, want = (t if isinstance(t, tuple) else (t,) for t in (got, want))
    for a, b in zip(got, want):
        torch.testing.assert_close(a, b)


def test_function_transforms_match_or_are_refused():
    lin, module = layer(), norms("feature")
    x, y = inputs()
    with torch.no_grad():
        matches_or_raises(lambda: torch.func.vmap(lin)(x), lin(x))
        matches_or_raises(lambda: torch.func.vmap(module)(x, y), module(x, y))
        # the weight is what is mapped over, the rows are ordinary
        w = torch.rand((3, 96), device="cuda")
        norm = lambda v: op().block_norm(x, y, pre_weight=v)[1]  # noqa: E731
        matches_or_raises(lambda: torch.func.vmap(norm)(w), torch.stack([norm(v) for v in w]))

    def loss(a, b):
        return module(a, b)[1].square().sum()

    a = x.clone().requires_grad_(True)
    want, = torch.autograd.grad(loss(a, y), a)
    matches_or_raises(lambda: torch.func.grad(loss)(x, y), want)
    matches_or_raises(lambda: torch.func.grad(lambda v: lin(v).sum())(x), lin.dense_weight().sum(0).expand_as(x))
    matches_or_raises(lambda: torch.func.functionalize(lambda v: lin(v))(x), lin(x))


def test_subclasses_are_not_taken_for_missing_tensors():
    """A tensor that is a wrapper has no memory of its own: where it is a weight, it must count or be refused."""
    class Wrapper(torch.Tensor):
        @staticmethod
        def __new__(cls, inner):
            return torch.Tensor._make_wrapper_subclass(cls, inner.shape, dtype=inner.dtype, device=inner.device)

        def __init__(self, inner):
            self.inner = inner

        @classmethod
        def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
            bare = torch.utils._pytree.tree_map(lambda t: t.inner if isinstance(t, Wrapper) else t, (args, kwargs or {}))
            return func(*bare[0], **bare[1])

    x, y = inputs()
    w = torch.rand(96, device="cuda") + 0.5
    want = op().block_norm(x, y, pre_weight=w, gate=w)
    for at in ("pre_weight", "gate"):
        given = {"pre_weight": w, "gate": w, at: Wrapper(w)}
        matches_or_raises(lambda: op().block_norm(x, y, **given), want)
    lin = layer()
    matches_or_raises(lambda: lin(Wrapper(x)), lin(x))
    bias = lin.bias
    good = lin(x)
    lin._buffers["bias"] = Wrapper(bias)
    matches_or_raises(lambda: lin(x), good)
