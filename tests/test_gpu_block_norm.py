"""The norms around a block, forward and backward, against the formulas in 64 bits on the CPU.

Tolerances.  The oracle below computes each result together with its size: the same formula with every term's magnitude,
added.  A result is a chain of fp32 operations on terms of that size: at most 32 roundings for its products, sums and the
square root, and the sums over a row add 8 or 16 terms per thread, 6 steps in a wave and up to 16 waves: 64 roundings of
2^-24 cover both.  A sum over n rows adds n more (a walker's rows in turn, then the walkers).  Results of 16 bits are rounded once
more, by half a step (eps / 2 of the value), fp16 below its normal range by 2^-25."""
import importlib

import numpy as np
import pytest

from conftest import nmspmm

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
LEAVES = ("residual", "branch", "gate", "scale", "post_weight", "post_bias", "pre_weight", "pre_bias")
EPS = 1e-5


def op():
    return importlib.import_module("nm-spmm_amd.torch_op")


class V:
    """A value with its size."""

    def __init__(self, v, size=None):
        self.v, self.size = v, np.abs(v) if size is None else size

    def __add__(self, o):
        o = o if isinstance(o, V) else V(np.asarray(float(o)))
        return V(self.v + o.v, self.size + o.size)

    def __sub__(self, o):
        return V(self.v - o.v, self.size + o.size)

    def __mul__(self, o):
        o = o if isinstance(o, V) else V(np.asarray(float(o)))
        return V(self.v * o.v, self.size * o.size)

    def mean(self):
        return V(self.v.mean(-1, keepdims=True), self.size.mean(-1, keepdims=True))

    def sum(self, axes, keepdims=False):
        return V(self.v.sum(axes, keepdims=keepdims), self.size.sum(axes, keepdims=keepdims))


def standard(v, kind):
    if kind == "layer":
        v = v - v.mean()
    inv = 1.0 / np.sqrt((v.v * v.v).mean(-1, keepdims=True) + EPS)
    # the sum of squares is off by its own 2^-24s, relative to the squares of the terms' sizes
    spread = (v.size * v.size).mean(-1, keepdims=True) * inv * inv
    return V(v.v * inv, v.size * inv + np.abs(v.v * inv) * spread), V(inv, inv * (1 + spread))


def oracle(t, conf, grad_sum=None, grad_out=None):
    """{name: V} of sum, out and the gradients."""
    x = {k: None if v is None else V(v.detach().double().cpu().numpy()) for k, v in t.items()}
    off = conf["weight_offset"]

    def back(g, vn, inv, kind):
        d = g - vn * (g * vn).mean()
        if kind == "layer":
            d = d - g.mean()
        return d * inv

    def affine(v, w, b):
        if w is not None:
            v = v * (w + off)
        return v if b is None else v + b

    got = {}
    total = x["residual"]
    if x["branch"] is not None:
        yn, yinv = (x["branch"], None) if conf["post"] is None else standard(x["branch"], conf["post"])
        after = affine(yn, x["post_weight"], x["post_bias"])
        gated = after if x["gate"] is None else after * x["gate"]
        factor = x["scale"] if x["scale"] is not None else conf["factor"]
        total = total * factor + gated
    got["sum"] = total
    if conf["pre"] is not None:
        tn, tinv = standard(total, conf["pre"])
        got["out"] = affine(tn, x["pre_weight"], x["pre_bias"])
    if grad_sum is None and grad_out is None:
        return got
    rows = tuple(range(total.v.ndim - 1))
    zero = V(np.zeros_like(total.v))
    ds = zero if grad_sum is None else V(grad_sum.double().cpu().numpy())
    if grad_out is not None and conf["pre"] is not None:
        go = V(grad_out.double().cpu().numpy())
        got["d pre_weight"], got["d pre_bias"] = (go * tn).sum(rows), go.sum(rows)
        g = go if x["pre_weight"] is None else go * (x["pre_weight"] + off)
        ds = ds + back(g, tn, tinv, conf["pre"])
    else:
        got["d pre_weight"] = got["d pre_bias"] = V(np.zeros(total.v.shape[-1]))
    got["d residual"] = ds
    if x["branch"] is not None:
        got["d residual"] = ds * factor
        got["d scale"] = (ds * x["residual"]).sum(rows)
        da = ds
        if x["gate"] is not None:
            dg = ds * after
            axes = tuple(i for i in rows if x["gate"].v.ndim == 1 or (x["gate"].v.shape[i] == 1 and total.v.shape[i] != 1))
            got["d gate"] = dg.sum(axes, keepdims=x["gate"].v.ndim != 1) if axes else dg
            da = ds * x["gate"]
        got["d post_weight"], got["d post_bias"] = (da * yn).sum(rows), da.sum(rows)
        dy = da if x["post_weight"] is None else da * (x["post_weight"] + off)
        got["d branch"] = dy if conf["post"] is None else back(dy, yn, yinv, conf["post"])
    return got


def close(got, want, what, terms=0):
    g = got.detach().double().cpu().numpy().reshape(want.v.shape)
    bound = 2.0 ** -24 * (64 + terms) * want.size + 1e-42
    if got.dtype != torch.float32:
        bound = bound + torch.finfo(got.dtype).eps / 2 * (np.abs(want.v) + bound) + 2.0 ** -25
    err = np.abs(g - want.v)
    assert np.all(err <= bound), "%s: %g over its bound" % (what, float((err - bound).max()))


def make(seed, shape, dtype="fp32", residual="same", param="same", post="rms", pre="rms", gate="feature", scale="tensor", bias=None,
         branch=True, weights=True, weight_offset=0.0):
    g = torch.Generator().manual_seed(seed)
    D = shape[-1]
    dt = DTYPES[dtype]
    res = torch.float32 if residual == "fp32" else dt
    par = {"same": dt, "fp32": torch.float32, "bf16": torch.bfloat16}[param]

    def normal(*s):
        return torch.randn(s, generator=g, dtype=torch.float64)

    t = dict.fromkeys(LEAVES)
    t["residual"] = (2 * normal(*shape)).to(res)
    if branch:
        t["branch"] = (normal(*shape) + 0.3).to(dt)
        shapes = {"feature": (D,), "sample": (shape[0],) + (1,) * (len(shape) - 2) + (D,), "element": shape, "none": None}
        if shapes[gate]:
            t["gate"] = normal(*shapes[gate]).to(dt)
        if scale == "tensor":
            t["scale"] = (0.9 + 0.1 * normal(D)).to(par)
        if post and weights:
            t["post_weight"] = (1 - weight_offset + 0.2 * normal(D)).to(par)
        if post and (bias if bias is not None else post == "layer"):
            t["post_bias"] = (0.2 * normal(D)).to(par)
    if pre and weights:
        t["pre_weight"] = (1 - weight_offset + 0.2 * normal(D)).to(par)
    if pre and (bias if bias is not None else pre == "layer"):
        t["pre_bias"] = (0.2 * normal(D)).to(par)
    t = {k: None if v is None else v.cuda() for k, v in t.items()}
    conf = dict(post=post if branch else None, pre=pre, factor=0.875 if scale == "number" else 1.0, weight_offset=weight_offset)
    return t, conf, dt


def call(t, conf, dt):
    scale = t["scale"] if t["scale"] is not None else (conf["factor"] if t["branch"] is not None else 1.0)
    return op().block_norm(t["residual"], t["branch"], gate=t["gate"], residual_scale=scale, post=conf["post"],
                           post_weight=t["post_weight"], post_bias=t["post_bias"], pre=conf["pre"], pre_weight=t["pre_weight"],
                           pre_bias=t["pre_bias"], eps=EPS, weight_offset=conf["weight_offset"], dtype=dt)


def check_forward(t, conf, dt):
    total, out = call(t, conf, dt)
    want = oracle(t, conf)
    if t["branch"] is None:
        assert total is t["residual"]
    else:
        assert total.dtype == t["residual"].dtype
        close(total, want["sum"], "sum")
    if conf["pre"] is None:
        assert out is None
    else:
        assert out.dtype == dt
        close(out, want["out"], "out")


def check_backward(t, conf, dt, seed=5, grads=("sum", "out")):
    g = torch.Generator().manual_seed(seed)
    shape = t["residual"].shape
    gs = torch.randn(shape, generator=g).to(t["residual"].dtype).cuda() if "sum" in grads else None
    go = torch.randn(shape, generator=g).to(dt).cuda() if "out" in grads and conf["pre"] else None
    leaves = {k: v.detach().requires_grad_(True) for k, v in t.items() if v is not None}
    given = dict(t, **leaves)
    total, out = call(given, conf, dt)
    outputs = [(o, d) for o, d in ((total, gs), (out, go)) if d is not None]
    got = torch.autograd.grad([o for o, _ in outputs], list(leaves.values()), [d for _, d in outputs], allow_unused=True)
    want = oracle(t, conf, gs, go)
    rows = t["residual"].numel() // shape[-1]
    for (k, leaf), d in zip(leaves.items(), got):
        if d is None:
            assert not np.any(want["d " + k].v), k
            continue
        assert d.dtype == leaf.dtype and d.shape == leaf.shape
        close(d, want["d " + k], "d " + k, rows if k not in ("residual", "branch") else 0)
    return dict(zip(leaves, got))


SHAPES = [(1, 1), (1, 7), (3, 8), (1, 1, 64), (5, 3, 100), (2, 17, 256), (7, 511), (4, 5, 512), (3, 513), (2, 9, 1024), (33, 2049),
          (2, 3, 4096), (3, 5000), (2, 2, 8192), (3, 8200), (2, 16384), (2, 12345)]


@pytest.mark.parametrize("dtype,residual", [("fp32", "same"), ("bf16", "same"), ("bf16", "fp32"), ("fp16", "same"), ("fp16", "fp32")])
@pytest.mark.parametrize("shape", SHAPES)
def test_shapes_and_types(shape, dtype, residual):
    k = len(shape) + shape[-1]
    kinds = [("rms", "rms"), ("layer", "layer"), ("rms", "layer"), ("layer", "rms")][k % 4]
    made = make(k, shape, dtype, residual, ("same", "fp32", "bf16")[k % 3], *kinds, gate=("feature", "sample", "element")[k % 3])
    check_forward(*made)
    check_backward(*made)


@pytest.mark.parametrize("post", [None, "rms", "layer"])
@pytest.mark.parametrize("pre", [None, "rms", "layer"])
@pytest.mark.parametrize("gate", ["none", "feature", "sample", "element"])
@pytest.mark.parametrize("scale", ["none", "number", "tensor"])
def test_every_combination(post, pre, gate, scale):
    made = make(3, (3, 11, 136), "bf16", "fp32", "fp32", post, pre, gate, scale, weights=gate != "sample", weight_offset=float(gate == "element"))
    check_forward(*made)
    check_backward(*made)


@pytest.mark.parametrize("pre", ["rms", "layer"])
@pytest.mark.parametrize("dtype,residual", [("fp32", "same"), ("bf16", "same"), ("fp16", "fp32")])
@pytest.mark.parametrize("shape", [(1, 96), (40, 77), (2, 6, 2048)])
def test_first_norm_of_a_model(pre, dtype, residual, shape):
    made = make(4, shape, dtype, residual, "fp32", pre=pre, branch=False, bias=True)
    check_forward(*made)
    check_backward(*made)
    check_backward(*made, grads=("out",))
    check_backward(*made, grads=("sum",))


@pytest.mark.parametrize("grads", [("sum",), ("out",)])
def test_only_one_result_is_used(grads):
    check_backward(*make(6, (4, 9, 264), "bf16", post="layer", pre="rms", gate="sample"), grads=grads)


@pytest.mark.parametrize("samples,tokens,D", [(1, 3000, 128), (3, 700, 96), (500, 3, 64), (2, 2500, 520), (70, 40, 1000), (9, 1000, 16)])
@pytest.mark.parametrize("gate", ["sample", "feature", "element"])
def test_many_rows_are_cut_among_walkers(samples, tokens, D, gate):
    made = make(7, (samples, tokens, D), "fp32", post="layer", pre="layer", gate=gate)
    check_forward(*made)
    check_backward(*made)


def test_only_some_inputs_need_gradients():
    t, conf, dt = make(8, (6, 200), "fp32", gate="sample", post="layer", pre="layer")
    every = check_backward(t, conf, dt)
    gs, go = (torch.randn((6, 200), generator=torch.Generator().manual_seed(5)).cuda() for _ in range(2))
    for only in every:
        given = {k: v if v is None else v.detach().requires_grad_(k == only) for k, v in t.items()}
        total, out = call(given, conf, dt)
        g = torch.Generator().manual_seed(5)
        gs, go = torch.randn((6, 200), generator=g).cuda(), torch.randn((6, 200), generator=g).cuda()
        d, = torch.autograd.grad((total, out), (given[only],), (gs, go))
        assert torch.equal(d, every[only])


def test_gradients_agree_with_differences():
    """Along a random direction u of all inputs: sum(grad * u) against (f(x + h u) - f(x - h u)) / 2 h of the formula in 64 bits.
    The difference's own error is h^2 times a third derivative: below 1e-6 of it for h = 1e-4; the gradient's is 1e-5 of its size."""
    t, conf, dt = make(9, (3, 7, 130), "fp32", post="layer", pre="layer", gate="sample")
    grads = check_backward(t, conf, dt)
    g = torch.Generator().manual_seed(5)
    gs, go = torch.randn((3, 7, 130), generator=g).double(), torch.randn((3, 7, 130), generator=g).double()
    u = {k: torch.randn(v.shape, dtype=torch.float64) for k, v in t.items() if v is not None}

    def f(h):
        moved = {k: None if v is None else v.double().cpu() + h * u[k] for k, v in t.items()}
        w = oracle(moved, conf)
        return float((w["sum"].v * gs.numpy()).sum() + (w["out"].v * go.numpy()).sum())

    along = sum(float((grads[k].double().cpu() * u[k]).sum()) for k in u)
    size = sum(float((grads[k].double().cpu() * u[k]).abs().sum()) for k in u)
    assert abs(along - (f(1e-4) - f(-1e-4)) / 2e-4) <= 2e-5 * size


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_strided_rows_and_unaligned_memory(dtype):
    t, conf, dt = make(10, (4, 6, 128), dtype, gate="element", post="layer", pre="layer")
    want = call(t, conf, dt)
    for shift in (0, 1):
        apart = dict(t)
        for k in ("residual", "branch", "gate"):
            wide = torch.full((4, 6, 128 + 24), float("nan"), dtype=t[k].dtype, device="cuda")
            wide[:, :, shift:shift + 128] = t[k]
            apart[k] = wide[:, :, shift:shift + 128]
        for k in ("pre_weight", "post_bias", "scale"):
            long = torch.zeros(128 + shift, dtype=t[k].dtype, device="cuda")
            long[shift:] = t[k]
            apart[k] = long[shift:]
        got = call(apart, conf, dt)
        if shift == 0:
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        check_forward(apart, conf, dt)
        check_backward(apart, conf, dt)
    across = dict(t, residual=t["residual"].transpose(0, 1).contiguous().transpose(0, 1), branch=t["branch"].permute(2, 0, 1).contiguous().permute(1, 2, 0))
    got = call(across, conf, dt)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_gates_and_scales_that_broadcast():
    r, y = (torch.randn((3, 5, 64), device="cuda") for _ in range(2))
    for shape in ((64,), (1, 1, 64), (3, 1, 64), (3, 5, 64), (1, 5, 64), (5, 64), (3, 5, 1), (1,)):
        gate = torch.randn(shape, device="cuda", requires_grad=True)
        full = gate.detach().expand(3, 5, 64).contiguous().requires_grad_(True)
        a, b = op().block_norm(r, y, gate=gate), op().block_norm(r, y, gate=full)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        ga, = torch.autograd.grad(a[1].square().sum(), gate)
        gb, = torch.autograd.grad(b[1].square().sum(), full)
        # both are sums of the same up to 960 terms, in another order
        torch.testing.assert_close(ga, gb.sum_to_size(shape), rtol=1e-4, atol=1e-3)
    for scale in (torch.tensor(0.5, device="cuda"), torch.tensor([0.5], device="cuda"), torch.full((64,), 0.5, device="cuda")):
        scale.requires_grad_(True)
        a, b = op().block_norm(r, y, residual_scale=scale), op().block_norm(r, y, residual_scale=0.5)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        assert torch.autograd.grad(a[0].sum(), scale)[0].shape == scale.shape


def test_rows_that_are_constant_zero_large_or_not_finite():
    for kind in ("rms", "layer"):
        r = torch.zeros((5, 256), device="cuda")
        r[1], r[2], r[3, 7], r[4, 9] = 3.0, 1e15, float("inf"), float("nan")
        y = r.clone()
        total, out = op().block_norm(r, y, post=kind, pre=kind)
        assert torch.equal(total[0], r[0]) and torch.equal(out[0], r[0])
        assert bool(total[:3].isfinite().all()) and bool(out[:3].isfinite().all())
        if kind == "layer":
            assert bool((out[1] == 0).all())
        assert bool(out[3:].isnan().any(1).all())       # and no other row is touched by them


def test_sum_may_overwrite_the_residual_and_out_the_branch():
    t, conf, dt = make(11, (40, 512), "bf16", "same", "fp32", gate="sample")
    want = call(t, conf, dt)
    params = tuple(t[k] for k in ("gate", "scale", "post_weight", "post_bias", "pre_weight", "pre_bias"))
    r, y = t["residual"].clone(), t["branch"].clone()
    code = {torch.float32: nmspmm.F32, torch.bfloat16: nmspmm.BF16}
    packed = nmspmm.BLOCK_NORM.pack(40, 1, 512, 512, 512, 512, r.data_ptr(), y.data_ptr(), r.data_ptr(), y.data_ptr(), 0,
                                    *[0 if p is None else p.data_ptr() for p in params], *[0 if p is None else code[p.dtype] for p in params],
                                    512, code[dt], code[r.dtype], 1, 1, 1.0, EPS, 0.0)
    assert nmspmm.lib().nmspmm_block_norm_forward(packed, torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(r, want[0]) and torch.equal(y, want[1])


def test_empty_batches():
    for shape in ((0, 64), (3, 0, 64)):
        r = torch.zeros(shape, device="cuda", requires_grad=True)
        w = torch.ones(64, device="cuda", requires_grad=True)
        total, out = op().block_norm(r, r * 1, pre_weight=w, gate=w)
        assert total.shape == shape and out.shape == shape
        d = torch.autograd.grad(out.sum() + total.sum(), (r, w))
        assert d[0].shape == shape and not bool(d[1].any())


def test_repeats_and_streams_agree_bit_for_bit():
    made = make(12, (4, 300, 768), "bf16", gate="sample")
    want = check_backward(*made)
    for k in range(3):
        with torch.cuda.stream(torch.cuda.Stream()):
            torch.cuda.current_stream().wait_stream(torch.cuda.default_stream())
            got = check_backward(*made)
            torch.cuda.current_stream().synchronize()
        for name in want:
            assert torch.equal(got[name], want[name])


def test_graph_replays_forward_and_backward():
    t, conf, dt = make(13, (2, 64, 512), "bf16", gate="sample")
    leaves = {k: v.detach().clone().requires_grad_(True) for k, v in t.items() if v is not None}
    gs, go = torch.randn((2, 64, 512), device="cuda").bfloat16(), torch.randn((2, 64, 512), device="cuda").bfloat16()

    def step():
        total, out = call(dict(t, **leaves), conf, dt)
        return (total.detach(), out.detach(), *torch.autograd.grad((total, out), list(leaves.values()), (gs, go)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for k in range(4):
        with torch.no_grad():
            for v in leaves.values():
                v.copy_(torch.randn(v.shape, device="cuda") + 0.5)
        want = [x.detach().clone() for x in step()]
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, want):
            assert torch.equal(a, b)


def test_registered_operators_trace_and_match():
    t, conf, dt = make(14, (2, 9, 64), "fp32", gate="sample", post="layer", pre="layer")
    params = tuple(t[k] for k in LEAVES[2:])
    args = (t["residual"], t["branch"], *params, 1.0, 2, 2, EPS, 0.0, 9, dt, True)
    torch.library.opcheck(op()._block_norm_op, args)
    torch.library.opcheck(op()._block_norm_op, tuple(a.detach().requires_grad_(True) if isinstance(a, torch.Tensor) else a for a in args))

    block_norm = op().block_norm

    def f(residual, branch, gate, weight):
        total, out = block_norm(residual, branch, gate=gate, post="rms", pre_weight=weight)
        return total, out, block_norm(total, pre="layer")[1]

    given = [t["residual"], t["branch"], t["gate"], t["pre_weight"]]
    want = f(*given)
    got = torch.compile(f, fullgraph=True, backend="aot_eager")(*given)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    leaves = [v.detach().requires_grad_(True) for v in given]
    eager = torch.autograd.grad(sum(x.square().sum() for x in f(*leaves)), leaves)
    traced = torch.autograd.grad(sum(x.square().sum() for x in torch.compile(f, fullgraph=True, backend="aot_eager")(*leaves)), leaves)
    for a, b in zip(traced, eager):
        torch.testing.assert_close(a, b, rtol=1e-5, atol=1e-5)


def test_offsets_beyond_32_bits():
    """Rows whose elements lie beyond 4 GiB, forward and backward: the last are those of a small call."""
    rows, D = 290000, 8192
    r, y = (torch.zeros((rows, D), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    tail = [torch.randn((5, D), device="cuda").bfloat16() for _ in range(2)]
    r[-5:], y[-5:] = tail
    w = torch.randn(D, device="cuda")
    gs = torch.ones((5, D), dtype=torch.bfloat16, device="cuda")

    def f(a, b, d):
        a, b = a.detach().requires_grad_(True), b.detach().requires_grad_(True)
        total, out = op().block_norm(a, b, post="rms", post_weight=w, pre_weight=w)
        return (total.detach(), out.detach(), *torch.autograd.grad((total, out), (a, b), (d, d)))

    full = torch.zeros((rows, D), dtype=torch.bfloat16, device="cuda")
    full[-5:] = gs
    for got, want in zip(f(r, y, full), f(*tail, gs)):
        assert torch.equal(got[-5:], want) and not bool(got[:-5].any())


def test_refusals():
    r = torch.randn((4, 64), device="cuda")
    f = op().block_norm
    for args, kw in [((r.cpu(),), {}), ((r.double(),), {}), ((r.half(), r.bfloat16()), {}), ((r, r[:2]), {}), ((r, r.cpu()), {}),
                     ((r,), dict(pre=None)), ((r,), dict(gate=r[0])), ((r,), dict(post="rms")), ((r,), dict(residual_scale=2.0)),
                     ((r, r), dict(pre="batch")), ((r, r), dict(post_weight=r[0])), ((r, r), dict(pre=None, pre_bias=r[0])),
                     ((r, r), dict(pre_weight=r[0, :63])), ((r, r), dict(pre_weight=r[0].double())), ((r, r), dict(pre_weight=r[0].cpu())),
                     ((r, r), dict(eps=-1.0)), ((r, r), dict(eps=float("nan"))), ((r.half(),), dict(dtype=torch.bfloat16)),
                     ((torch.zeros((1, 16385), device="cuda"),), {}), ((torch.zeros((4, 0), device="cuda"),), {})]:
        with pytest.raises(ValueError):
            f(*args, **kw)
    with pytest.raises(RuntimeError):
        f(r, r, gate=torch.randn((3, 64), device="cuda"))      # does not broadcast
    x = r.clone().requires_grad_(True)
    d, = torch.autograd.grad(f(x, r)[1].sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(d.sum(), x)


def test_operators_refuse_what_does_not_fit():
    """The traced operators take each other's results by hand too: sizes are checked there as well."""
    r, w = torch.randn((4, 64), device="cuda"), torch.ones(64, device="cuda")
    ops = torch.ops.nmspmm
    conf = (1.0, 1, 1, EPS, 0.0, 4, torch.float32, True)
    total, out, stats = ops.block_norm(r, r, w, None, w, None, w, None, *conf)
    given = (r, r, w, None, w, None, w, None)
    needs = [t is not None for t in given]
    grads = ops.block_norm_backward(*given, stats, total, out, *conf, needs)
    assert [g.shape == t.shape if t is not None else g.numel() == 0 for g, t in zip(grads, given)] == [True] * 8
    for bad in (stats[:3], stats.double(), stats.cpu()):
        with pytest.raises((ValueError, NotImplementedError)):
            ops.block_norm_backward(*given, bad, total, out, *conf, needs)
    for d in (total[:3], total.bfloat16()):
        with pytest.raises(ValueError):
            ops.block_norm_backward(*given, stats, d, None, *conf, needs)
        with pytest.raises(ValueError):
            ops.block_norm_backward(*given, stats, None, d, *conf, needs)
    for kw in (dict(gate=w[:63]), dict(gate_rows=3), dict(post=3), dict(dtype=torch.float64)):
        a, c = list(given), list(conf)
        if "gate" in kw:
            a[2] = kw["gate"]
        else:
            c[dict(gate_rows=5, post=1, dtype=6)[next(iter(kw))]] = next(iter(kw.values()))
        with pytest.raises(ValueError):
            ops.block_norm(*a, *c)


def test_negated_views_and_tangents():
    """A view whose memory holds the negated values counts as what it stands for; forward-mode derivatives are refused."""
    z = torch.randn((5, 64), dtype=torch.complex64, device="cuda")
    r, w = z.conj().imag, torch.randn((64,), dtype=torch.complex64, device="cuda").conj().imag
    assert r.is_neg() and w.is_neg()
    got = op().block_norm(r, r, gate=w, post="rms", post_weight=w, pre_weight=w)
    plain, pw = -z.imag, w.resolve_neg()
    for a, b in zip(got, op().block_norm(plain, plain, gate=pw, post="rms", post_weight=pw, pre_weight=pw)):
        assert torch.equal(a, b)
    x = plain.clone().requires_grad_(True)
    total, out = op().block_norm(x, plain, pre_weight=pw)
    d1, = torch.autograd.grad((total, out), x, (r, r), retain_graph=True)
    d2, = torch.autograd.grad((total, out), x, (plain, plain))
    assert torch.equal(d1, d2)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(plain.contiguous(), torch.ones_like(plain))
        for args in ((dual,), (plain, dual)):
            with pytest.raises((ValueError, RuntimeError)):
                op().block_norm(*args)


def test_hooks_retained_graphs_and_checkpoints():
    """What autograd does around a node: saved tensors go through hooks, a graph is walked twice, a part is run again."""
    t, conf, dt = make(23, (6, 96), "bf16", "fp32", "fp32", gate="sample")
    leaves = [v.requires_grad_(True) for v in t.values() if v is not None]

    def run():
        total, out = call(t, conf, dt)
        return total.sum() + out.float().square().sum()

    want = torch.autograd.grad(run(), leaves)
    with torch.autograd.graph.save_on_cpu():
        loss = run()
    for _ in range(2):
        for a, b in zip(torch.autograd.grad(loss, leaves, retain_graph=True), want):
            assert torch.equal(a, b)
    again = torch.utils.checkpoint.checkpoint(run, use_reentrant=False)
    for a, b in zip(torch.autograd.grad(again, leaves), want):
        assert torch.equal(a, b)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(again, leaves)      # freed
    for k, leaf in enumerate(leaves):            # each gradient alone, as when the others are frozen
        assert torch.equal(torch.autograd.grad(run(), leaf)[0], want[k])


@pytest.mark.parametrize("norm", ["rms", "layer"])
def test_a_stack_of_compressed_blocks(norm):
    """Two blocks of 4-bit and of fp32 N:M-sparse layers between their norms, against the same run in 64 bits with the layers'
    dense weights; and the gradients of the norms' parameters and of x through a stack of differentiable blocks."""
    m = op()

    def mlp(kind, n, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        up, down = torch.randn((512, 128), generator=g, device="cuda") * 0.1, torch.randn((128, 512), generator=g, device="cuda") * 0.05
        return torch.nn.Sequential(kind(up, *n), torch.nn.GELU(), kind(down, *n))

    blocks = [mlp(m.NMQuantLinear, (1, 1), 1), mlp(m.NMSparseLinear, (2, 8), 2), mlp(m.NMQuantLinear, (2, 4), 3)]
    stack = m.NMBlockStack(blocks, 128, norm=norm, residual_scale=0.9, gate=True, gate_init=0.7)
    with torch.no_grad():
        for p in stack.parameters():
            p.add_(0.1 * torch.randn_like(p))
        for x in (torch.randn((1, 128), device="cuda"), torch.randn((2, 37, 128), device="cuda")):
            total, h = stack(x)

            def norm64(v, w, b):
                if norm == "layer":
                    v = v - v.mean(-1, keepdim=True)
                v = v / (v.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
                return v if b is None else v + b.double()

            s = x.double()
            for i, block in enumerate(blocks):
                z = norm64(s, stack.pre_weight[i], stack.pre_bias[i] if norm == "layer" else None)
                z = torch.nn.functional.gelu(z @ block[0].dense_weight().double().t()) @ block[2].dense_weight().double().t()
                s = 0.9 * s + stack.gate[i].double() * norm64(z, stack.post_weight[i], stack.post_bias[i] if norm == "layer" else None)
            # six products of up to 512 terms in fp32, each to about 1e-6 of its norm
            assert float((total.double() - s).norm() / s.norm()) < 2e-5
            want = norm64(s, stack.pre_weight[3], stack.pre_bias[3] if norm == "layer" else None)
            assert float((h.double() - want).norm() / want.norm()) < 2e-5
    dense = m.NMBlockStack([torch.nn.Linear(128, 128, device="cuda") for _ in range(2)], 128, norm=norm, gate=True)
    x = torch.randn((5, 128), device="cuda", requires_grad=True)
    total, h = dense(x)
    (total.square().sum() + h.sin().sum()).backward()
    assert x.grad is not None and all(p.grad is not None and bool(p.grad.isfinite().all()) for p in dense.parameters())
