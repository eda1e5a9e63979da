"""Measured passes of the operators for compressed linear layers in 4 bits and of the norms around a block.

Four operators:

* "linear": y = x W + b where W is an N:M-compressed (or dense) operand whose kept values are 4-bit
  codes with a scale and a zero point for each group of kept rows and column;
* "quantize": such an operand made from float32 values, and expanded back to the dense float32 matrix;
* "norm": the norm after a block, its gate, the scaled residual sum and the norm before the next block;
* "norm_train": the same with the gradients of everything that went in.

With `own` false every pass is elementary torch arithmetic; with `own` true it is the calls a program
makes of the package.
"""
import importlib
import math

import torch

own = False  # set from outside: False = plain torch arithmetic, True = the package's operators

_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_VECTOR = 32  # columns that share one index pattern


# ---- the cases -------------------------------------------------------------------------------------

def _linear(name, rows, K, N, dtype, n=1, m=1, group=128, zero=False, bias=False):
    return {"name": name, "op": "linear", "rows": rows, "K": K, "N": N, "dtype": dtype, "n": n, "m": m, "group": group,
            "zero": zero, "bias": bias}


def _norm(name, op, samples, tokens, features, dtype, residual="same", post="rms", pre="rms", gate="feature", scale="float",
          branch=True):
    return {"name": name, "op": op, "samples": samples, "tokens": tokens, "features": features, "dtype": dtype,
            "residual": residual, "post": post, "pre": pre, "gate": gate, "scale": scale, "branch": branch}


def listed():
    return [
        # one token through a square projection of a 4096-wide model, float32 like the library's other layers
        _linear("linear 1 row 4096x4096", 1, 4096, 4096, "fp32"),
        # one token through a 2:8 layer of 8192 features, zero points as imported checkpoints have them
        _linear("linear 1 row 8192x8192 2:8", 1, 8192, 8192, "fp32", 2, 8, 64, zero=True),
        # a small batch of sequences, one token each, through a down projection
        _linear("linear 8 rows 11008x4096 bf16", 8, 11008, 4096, "bf16", zero=True),
        # an uneven batch of decoding sequences through a 2:4 up projection
        _linear("linear 13 rows 4096x14336 2:4 bf16", 13, 4096, 14336, "bf16", 2, 4, 128, bias=True),
        # a prompt of 2000 tokens through an up projection
        _linear("linear 2000 rows 4096x11008 bf16", 2000, 4096, 11008, "bf16"),
        # a layer compressed when a model is loaded
        {"name": "quantize 4096x4096", "op": "quantize", "K": 4096, "N": 4096, "n": 1, "m": 1, "group": 128, "asymmetric": False},
        {"name": "quantize 11008x4096 2:8", "op": "quantize", "K": 11008, "N": 4096, "n": 2, "m": 8, "group": 32, "asymmetric": True},
        # between two blocks while one token is decoded; the residual stream in float32
        _norm("norm 1 token 4096 bf16", "norm", 1, 1, 4096, "bf16", "fp32"),
        # between two blocks of a prompt, with a gate for each sample
        _norm("norm 4x1024 tokens 8192 bf16", "norm", 4, 1024, 8192, "bf16", gate="sample", scale="tensor"),
        # an odd width and an odd count of rows, LayerNorms
        _norm("norm 3x357 tokens 2049 fp32", "norm", 3, 357, 2049, "fp32", post="layer", pre="layer", gate="element"),
        # training steps
        _norm("norm_train 2x2048 tokens 4096 bf16", "norm_train", 2, 2048, 4096, "bf16", scale="tensor"),
        _norm("norm_train 5x301 tokens 1536 fp32", "norm_train", 5, 301, 1536, "fp32", post="layer", pre="layer", gate="sample",
              scale="tensor"),
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], even over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["linear", "linear", "linear", "quantize", "norm", "norm_train"])
    if op in ("linear", "quantize"):
        n, m = rng.choice([(1, 1), (1, 1), (2, 4), (2, 8), (1, 8)])
        K, N = _spread(rng, 200, 14336), _spread(rng, 64, 14336)
        if m > 1:
            K, N = max(m, K // m * m), N // _VECTOR * _VECTOR
        group = rng.choice([32, 64, 128])
        if op == "quantize":
            return {"op": op, "K": K, "N": N, "n": n, "m": m, "group": group, "asymmetric": rng.random() < 0.5}
        rows = min(_spread(rng, 1, 2000), max(1, 2000 * 4096 * 11008 // (K * N)))
        c = _linear("", rows, K, N, rng.choice(["fp32", "bf16", "fp16"]), n, m, group, rng.random() < 0.5, rng.random() < 0.5)
    else:
        features = _spread(rng, 64, 8192)
        tokens = _spread(rng, 1, 2048)
        samples = min(_spread(rng, 1, 8), max(1, 2 * 2048 * 4096 // (features * tokens)))
        c = _norm("", op, samples, tokens, features, rng.choice(["fp32", "bf16", "fp16"]), rng.choice(["same", "fp32"]),
                  rng.choice(["rms", "layer", "none"]), rng.choice(["rms", "layer"]),
                  rng.choice(["none", "feature", "sample", "element"]), rng.choice(["none", "float", "tensor"]),
                  rng.random() < 0.9)
    del c["name"]
    return c


# ---- inputs ----------------------------------------------------------------------------------------

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _kept_rows(g, K, N, n, m):
    """int32 [K*n/m][N/32]: the ascending window-local rows that each 32-column vector keeps."""
    score = torch.rand((K // m, m, N // _VECTOR), generator=g, device="cuda")
    kept = score.topk(n, dim=1).indices.sort(dim=1).values
    return kept.reshape(K // m * n, N // _VECTOR).to(torch.int32)


def _linear_inputs(case, seed):
    g = _generator(seed)
    K, N, n, m, group = case["K"], case["N"], case["n"], case["m"], case["group"]
    W = K // m * n
    groups = -(-W // group)
    x = _normal(g, case["rows"], K) * (1.0 + 9.0 * (torch.rand((K,), generator=g, device="cuda") > 0.995))
    s = {"x": x.to(_TYPES[case["dtype"]])}
    # codes gather around the zero point; scales as checkpoints hold them, in 16 bits
    s["codes"] = torch.round(_normal(g, W, N) * 2.7 + 7.8).clamp_(0, 15).to(torch.uint8)
    s["scale"] = (0.004 * torch.exp(0.5 * _normal(g, groups, N))).to(torch.float16).to(torch.float32)
    s["zero"] = torch.randint(5, 11, (groups, N), generator=g, device="cuda").to(torch.uint8) if case["zero"] else None
    s["rows"] = _kept_rows(g, K, N, n, m) if m > 1 else None
    s["bias"] = _normal(g, N) if case["bias"] else None
    return s


def _quantize_inputs(case, seed):
    g = _generator(seed)
    K, N, n, m = case["K"], case["N"], case["n"], case["m"]
    values = 0.02 * _normal(g, K // m * n, N)
    values *= 1.0 + 4.0 * (torch.rand(values.shape, generator=g, device="cuda") > 0.999)
    values[:, N // 2:N // 2 + 3] = 0.0  # features that pruning emptied
    return {"values": values, "rows": _kept_rows(g, K, N, n, m) if m > 1 else None}


def _norm_inputs(case, seed):
    g = _generator(seed)
    B, T, D = case["samples"], case["tokens"], case["features"]
    dt = _TYPES[case["dtype"]]
    res = torch.float32 if case["residual"] == "fp32" else dt
    s = {"residual": (2.0 * _normal(g, B, T, D)).to(res), "branch": None, "gate": None, "scale": None, "post_weight": None,
         "post_bias": None, "pre_weight": (1.0 + 0.1 * _normal(g, D)).to(res),
         "pre_bias": (0.1 * _normal(g, D)).to(res) if case["pre"] == "layer" else None}
    if case["branch"]:
        s["branch"] = (0.7 * _normal(g, B, T, D) + 0.1).to(dt)
        shape = {"none": None, "feature": (D,), "sample": (B, 1, D), "element": (B, T, D)}[case["gate"]]
        s["gate"] = (0.5 * _normal(g, *shape)).to(dt) if shape else None
        if case["scale"] == "tensor":
            s["scale"] = (0.9 + 0.1 * _normal(g, D)).to(res)
        if case["post"] != "none":
            s["post_weight"] = (1.0 + 0.1 * _normal(g, D)).to(res)
            s["post_bias"] = (0.1 * _normal(g, D)).to(res) if case["post"] == "layer" else None
    if case["op"] == "norm_train":
        s["grad_sum"] = _normal(g, B, T, D).to(res)
        s["grad_out"] = _normal(g, B, T, D).to(dt)
        for k in _LEAVES:
            if s[k] is not None:
                s[k].requires_grad_(True)
    return s


_LEAVES = ("residual", "branch", "gate", "scale", "post_weight", "post_bias", "pre_weight", "pre_bias")
_EPS = 1e-6


def prepare(case, seed):
    s = {"linear": _linear_inputs, "quantize": _quantize_inputs}.get(case["op"], _norm_inputs)(case, seed)
    s["case"] = case
    if own:
        s["op"] = importlib.import_module("nm-spmm_amd.torch_op")
        if case["op"] == "linear":  # the weights of a layer are laid out once, when it is made
            s["layer"] = s["op"].NMQuantLinear.from_codes(s["codes"], s["scale"], s["zero"], case["K"], n=case["n"], m=case["m"],
                                                          rows=s["rows"], group=case["group"], bias=s["bias"])
    return s


# ---- plain forms -----------------------------------------------------------------------------------

def _expand(values, rows, K, n, m):
    """Compressed values [W][N] -> the dense matrix [K][N]."""
    if rows is None:
        return values
    W, N = values.shape
    first = torch.arange(W, device=values.device) // n * m
    at = (first[:, None] + rows).repeat_interleave(_VECTOR, dim=1)
    return torch.zeros((K, N), dtype=values.dtype, device=values.device).scatter_(0, at, values)


def _plain_linear(s):
    case = s["case"]
    W, group = s["codes"].shape[0], case["group"]
    zero = 8.0 if s["zero"] is None else s["zero"].float().repeat_interleave(group, dim=0)[:W]
    values = (s["codes"].float() - zero) * s["scale"].repeat_interleave(group, dim=0)[:W]
    y = s["x"].float() @ _expand(values, s["rows"], case["K"], case["n"], case["m"])
    if s["bias"] is not None:
        y = y + s["bias"]
    return y.to(s["x"].dtype)


def _plain_quantize(s):
    case = s["case"]
    v, group = s["values"], case["group"]
    W, N = v.shape
    groups = -(-W // group)
    w = torch.nn.functional.pad(v.double(), (0, 0, 0, groups * group - W)).reshape(groups, group, N)
    if case["asymmetric"]:
        low, high, steps = w.amin(1).clamp(max=0.0), w.amax(1).clamp(min=0.0), 15.0
        need = (high - low) / steps
    else:
        need = w.abs().amax(1) / 7.0
    # the scale: the smallest number of 20 significant bits that covers the group
    fraction, exponent = torch.frexp(need)
    scale = torch.ldexp(torch.ceil(torch.ldexp(fraction, torch.tensor(20, device=v.device))), exponent - 20)
    some = torch.where(scale > 0, scale, torch.ones_like(scale))
    zero = torch.round(-low / some).clamp(0, 15) if case["asymmetric"] else torch.full_like(scale, 8.0)
    code = (torch.round(w / some[:, None]) + zero[:, None]).clamp(0, 15)
    back = ((code - zero[:, None]) * scale[:, None]).reshape(groups * group, N)[:W].float()
    return _expand(back, s["rows"], case["K"], case["n"], case["m"])


def _plain_normed(v, kind, weight, bias):
    if kind == "none":
        return v
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    v = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + _EPS) * weight.float()
    return v if bias is None else v + bias.float()


def _factor(case):
    return 0.875 if case["scale"] == "float" else 1.0


def _plain_norm(s):
    case = s["case"]
    v = s["residual"].float()
    if s["branch"] is not None:
        y = _plain_normed(s["branch"].float(), case["post"], s["post_weight"], s["post_bias"])
        if s["gate"] is not None:
            y = y * s["gate"].float()
        v = v * (_factor(case) if s["scale"] is None else s["scale"].float()) + y
    h = _plain_normed(v, case["pre"], s["pre_weight"], s["pre_bias"])
    return v.to(s["residual"].dtype), h.to(_TYPES[case["dtype"]])


# ---- the package's operators -----------------------------------------------------------------------

def _own_quantize(s):
    case = s["case"]
    operand = s["op"].NMQuantOperand.quantize(s["values"], s["rows"], case["K"], n=case["n"], m=case["m"], group=case["group"],
                                              asymmetric=case["asymmetric"])
    return operand.dense()


def _own_norm(s):
    case = s["case"]
    if s["branch"] is None:  # the first norm of a model
        return s["op"].block_norm(s["residual"], pre=case["pre"], pre_weight=s["pre_weight"], pre_bias=s["pre_bias"], eps=_EPS,
                                  dtype=_TYPES[case["dtype"]])
    return s["op"].block_norm(s["residual"], s["branch"], gate=s["gate"],
                              residual_scale=_factor(case) if s["scale"] is None else s["scale"],
                              post=None if case["post"] == "none" else case["post"], post_weight=s["post_weight"], post_bias=s["post_bias"], pre=case["pre"],
                              pre_weight=s["pre_weight"], pre_bias=s["pre_bias"], eps=_EPS, dtype=_TYPES[case["dtype"]])


def run(state):
    op = state["case"]["op"]
    if op == "linear":
        return state["layer"](state["x"]) if own else _plain_linear(state)
    if op == "quantize":
        return _own_quantize(state) if own else _plain_quantize(state)
    total, out = _own_norm(state) if own else _plain_norm(state)
    if op == "norm":
        return {"sum": total, "out": out}
    leaves = {k: state[k] for k in _LEAVES if state[k] is not None}
    # (without a branch the sum is the residual itself: its gradient is added where the two meet)
    grads = torch.autograd.grad((total, out), list(leaves.values()), (state["grad_sum"], state["grad_out"]))
    return {"sum": total.detach(), "out": out.detach(), "grads": dict(zip(leaves, grads))}


# ---- what a pass cannot do without -----------------------------------------------------------------

def work(case):
    if case["op"] in ("linear", "quantize"):
        K, N, W = case["K"], case["N"], case["K"] // case["m"] * case["n"]
        groups = -(-W // case["group"])
        rows = W * N // _VECTOR if case["m"] > 1 else 0  # one byte would do for each
        if case["op"] == "quantize":
            return {"bytes": 4 * W * N + rows + 4 * K * N, "flops": 4 * W * N}
        size = 4 if case["dtype"] == "fp32" else 2
        operand = W * N / 2 + 4 * groups * N + rows
        return {"bytes": operand + size * case["rows"] * (K + N) + (4 * N if case["bias"] else 0),
                "flops": 2.0 * case["rows"] * W * N}
    B, T, D = case["samples"], case["tokens"], case["features"]
    size = 4 if case["dtype"] == "fp32" else 2
    res = 4 if case["residual"] == "fp32" else size
    n = B * T * D
    branch = 1 if case["branch"] else 0
    gate = branch * {"none": 0, "feature": D, "sample": B * D, "element": n}[case["gate"]]
    params = 6 * D
    forward = res * n * (1 + branch) + size * n * (1 + branch) + size * gate + res * params  # r, (sum), (branch), out, gate
    if case["op"] == "norm":
        return {"bytes": forward, "flops": 16 * n}
    back = res * n * 2 + size * n * (1 + branch) + size * gate + res * params                # their gradients
    return {"bytes": forward + back, "flops": 48 * n}


# ---- the definitions in 64 bits --------------------------------------------------------------------

def _exact_linear(case, seed):
    s = _linear_inputs(case, seed)
    W, N = s["codes"].shape
    x = s["x"].double()
    of_group = torch.div(torch.arange(W, device=x.device), case["group"], rounding_mode="floor")
    w = s["codes"].double()
    w -= 8 if s["zero"] is None else s["zero"].double()[of_group]
    w *= s["scale"].double()[of_group]
    if s["rows"] is None:
        y = torch.matmul(x, w)
    else:
        window = torch.div(torch.arange(W, device=x.device), case["n"], rounding_mode="floor") * case["m"]
        y = torch.empty((x.shape[0], N), dtype=torch.float64, device=x.device)
        for v in range(N // _VECTOR):
            columns = slice(v * _VECTOR, (v + 1) * _VECTOR)
            y[:, columns] = x[:, window + s["rows"][:, v]] @ w[:, columns]
    return y if s["bias"] is None else y + s["bias"].double()


def _exact_quantize(case, seed):
    s = _quantize_inputs(case, seed)
    v = s["values"].double()
    W, N = v.shape
    out = torch.empty_like(v)
    for begin in range(0, W, case["group"]):
        w = v[begin:begin + case["group"]]
        top, bottom = w.max(0).values, w.min(0).values
        if case["asymmetric"]:
            top, bottom = torch.relu(top), -torch.relu(-bottom)
            step = (top - bottom) / 15
        else:
            step = torch.maximum(top, -bottom) / 7
        unit = torch.exp2(torch.floor(torch.log2(step.clamp(min=1e-300))) - 19)
        step = torch.ceil(step / unit) * unit
        inverse_ok = step > 0
        q = torch.where(inverse_ok, w / step, torch.zeros_like(w))
        if case["asymmetric"]:
            z = torch.where(inverse_ok, -bottom / step, torch.zeros_like(step)).round()
            q = torch.minimum(torch.maximum(q.round(), -z), 15 - z)
        else:
            q = q.round()
        out[begin:begin + case["group"]] = q * step
    if s["rows"] is None:
        return out
    n, m = case["n"], case["m"]
    dense = torch.zeros((case["K"] // m, m, N // _VECTOR, _VECTOR), dtype=torch.float64, device=v.device)
    window = torch.arange(W, device=v.device)[:, None] // n
    vector = torch.arange(N // _VECTOR, device=v.device)[None, :]
    dense[window, s["rows"].long(), vector] = out.reshape(W, N // _VECTOR, _VECTOR)
    return dense.reshape(case["K"], N)


def _exact_norm(case, seed):
    s = {k: v.detach().double() if v is not None else None for k, v in _norm_inputs(case, seed).items()}
    D = case["features"]

    def standard(v, kind):  # (normalised values, 1 / deviation)
        if kind == "layer":
            v = v - v.sum(-1, keepdim=True) / D
        inv = 1.0 / torch.sqrt(v.pow(2).sum(-1, keepdim=True) / D + _EPS)
        return v * inv, inv

    def back(dn, v, inv, kind):  # gradient of the normalised values -> of what went in
        d = dn - v * ((dn * v).sum(-1, keepdim=True) / D)
        if kind == "layer":
            d = d - dn.sum(-1, keepdim=True) / D
        return d * inv

    r, y = s["residual"], s["branch"]
    factor = s["scale"] if s["scale"] is not None else _factor(case)
    total, gate = r, 1.0
    if y is not None:
        gate = s["gate"] if s["gate"] is not None else 1.0
        if case["post"] == "none":
            after = y
        else:
            yn, yinv = standard(y, case["post"])
            after = yn * s["post_weight"] + (s["post_bias"] if s["post_bias"] is not None else 0.0)
        total = r * factor + after * gate
    tn, tinv = standard(total, case["pre"])
    out = tn * s["pre_weight"] + (s["pre_bias"] if s["pre_bias"] is not None else 0.0)
    if case["op"] == "norm":
        return {"sum": total, "out": out}
    go = s["grad_out"]
    grads = {"pre_weight": (go * tn).sum((0, 1)), "pre_bias": go.sum((0, 1))}
    dt = s["grad_sum"] + back(go * s["pre_weight"], tn, tinv, case["pre"])
    grads["residual"] = dt
    if y is not None:
        grads["residual"] = dt * factor
        grads["scale"] = (dt * r).sum((0, 1))
        if s["gate"] is not None:
            dg = dt * after
            grads["gate"] = {"feature": lambda: dg.sum((0, 1)), "sample": lambda: dg.sum(1, keepdim=True),
                             "element": lambda: dg}[case["gate"]]()
        da = dt * gate
        if case["post"] == "none":
            grads["branch"] = da
        else:
            grads["post_weight"], grads["post_bias"] = (da * yn).sum((0, 1)), da.sum((0, 1))
            grads["branch"] = back(da * s["post_weight"], yn, yinv, case["post"])
    return {"sum": total, "out": out, "grads": {k: grads[k] for k in _LEAVES if s[k] is not None}}


def exact(case, seed):
    return {"linear": _exact_linear, "quantize": _exact_quantize}.get(case["op"], _exact_norm)(case, seed)
