"""A drop-in for torch.nn.Linear (inference) whose weight is N:M vector-sparse and whose forward
runs the library's kernels: dense weight -> compress -> widen / preprocess once at construction,
then one row-major multiplication per call.  PyTorch only supplies device memory and the stream.

The multiplication is registered with torch.library as the operator `nmspmm::sparse_linear`
(with a fake implementation that only derives the output's shape), so that tracing front ends
(torch.compile, torch.export) see one opaque node instead of a Python function they cannot follow.

The reference has no framework binding; its driver multiplies synthetic operands
(tests/test_nmspmm.cu:72-97).  The sequence of calls here is that driver's, on real weights.
"""
import importlib
import importlib.util
import os
from typing import List, Optional, Tuple

import torch

_nm = importlib.import_module(__name__.rsplit(".", 1)[0])

# (n, m) reduced to lowest terms -> (window, kept) the kernels run the pattern at
# (reference launchers, src/kernel_64x128_8x8.cu:264-289,584-602)
_GEOMETRY = {(1, 2): (32, 16), (3, 8): (32, 12), (1, 4): (64, 16), (1, 8): (64, 8)}


def _geometry(n, m):
    from math import gcd
    g = gcd(n, m)
    if (n // g, m // g) not in _GEOMETRY:
        raise ValueError("pattern %d:%d is not one of 1:2, 3:8, 1:4, 1:8 (or a multiple of them)" % (n, m))
    window, kept = _GEOMETRY[(n // g, m // g)]
    if window % m != 0:
        raise ValueError("pattern window %d does not divide the kernel window %d" % (m, window))
    return window, kept


_plans = {}  # (M, N, K, W, kept) -> (split, workspace floats): two library calls per shape, not per forward


@torch.library.custom_op("nmspmm::sparse_linear", mutates_args=(), device_types="cuda")
def sparse_linear(x: torch.Tensor, values: torch.Tensor, indices: torch.Tensor, column_info: Optional[torch.Tensor],
                  row_index: Optional[torch.Tensor], bias: Optional[torch.Tensor], window: int, kept: int, Ns: int,
                  flags: int) -> torch.Tensor:
    """x [..., K] row-major times the compressed weight (values [W, N], preprocessed indices,
    column_info for 64-row windows, optional row list) plus bias: [..., N].  The library's own
    choice of kernel and split; the workspace comes from torch's caching allocator."""
    W, N = values.shape
    K = x.shape[-1]
    x2 = x.reshape(-1, K).contiguous()
    M = x2.shape[0]
    y = torch.empty((M, N), dtype=torch.float32, device=x.device)
    if M > 0:
        key = (M, N, K, W, kept)
        if key not in _plans:
            split = _nm.suggest_split_k(M, N, W, kept)
            _plans[key] = (split, _nm.workspace_bytes_rowmajor(M, N, K, split) // 4)
        split, need = _plans[key]
        workspace = torch.empty(max(need, 4), dtype=torch.float32, device=x.device)
        _nm.spmm_rowmajor(x2, values, indices, column_info, y, M, N, K, W, window, kept, workspace, 32, Ns, split,
                          row_index, flags)
        if bias is not None:
            y += bias
    return y.reshape(*x.shape[:-1], N)


@sparse_linear.register_fake
def _sparse_linear_fake(x, values, indices, column_info, row_index, bias, window, kept, Ns, flags):
    return x.new_empty((*x.shape[:-1], values.shape[1]))


class NMSparseLinear(torch.nn.Module):
    """y = x @ prune(weight).T + bias with an n:m pattern shared by 32 adjacent output features.

    weight: float32 CUDA tensor [out_features, in_features]; in_features % window == 0 and
    out_features % 32 == 0.  Leading dimensions of x are flattened into rows; any row count runs on
    the matrix-core kernels (the copy of x the row-major entry point makes is padded to a row pitch
    of a multiple of four floats).  single_stream=True promises that all forwards of such modules
    are issued on one stream at a time; up to 64 rows they may then use more of the GPU when
    out_features is small (fewer than 256 groups of 32).
    """

    def __init__(self, weight, n, m, bias=None, single_stream=False):
        super().__init__()
        # single_stream: the caller issues every forward of every such module on one stream at a
        # time, which lets decode-sized calls cut their reductions across workgroups through the
        # library's device-resident scratch (nmspmm.h: NMSPMM_DECODE_SPLIT)
        self.flags = _nm.DECODE_SPLIT if single_stream else 0
        if weight.dtype != torch.float32 or not weight.is_cuda or weight.dim() != 2:
            raise ValueError("weight must be a 2-D float32 CUDA tensor")
        self.out_features, self.in_features = weight.shape
        self.n, self.m = n, m
        self.window, self.kept = _geometry(n, m)
        N, K = self.out_features, self.in_features
        if K % self.window != 0 or N % 32 != 0:
            raise ValueError("in_features must be a multiple of %d and out_features of 32" % self.window)
        self.Ns = 128 if N % 128 == 0 else 64 if N % 64 == 0 else 32
        self.W, self.Q = K // m * n, N // 32
        dense = weight.t().contiguous()                                   # K x N, row-major
        BT = torch.empty((self.W, N), dtype=torch.float32, device=weight.device)
        DT = torch.empty((self.W, self.Q), dtype=torch.int32, device=weight.device)
        _nm.compress_device(dense, K, N, n, m, BT, DT)
        D = torch.empty_like(DT)
        cinfo = None
        if self.window == 64:
            cinfo = torch.empty(_nm.column_info_ints(self.W, self.kept, self.window, N, self.Ns), dtype=torch.int32,
                                device=weight.device)
        got = _nm.preprocess_device(DT, n, m, self.W, self.Q, N, self.Ns, D, cinfo)
        assert got == (self.window, self.kept)
        # the row list: the index form the decode kernel (up to 64 rows) reads
        rows = torch.empty(_nm.row_index_ints(self.W, N), dtype=torch.int32, device=weight.device)
        _nm.row_index_device(D, cinfo, self.W, N, self.window, self.kept, self.Ns, rows)
        self.register_buffer("values", BT)
        self.register_buffer("indices", D.reshape(-1))
        self.register_buffer("column_info", cinfo)
        self.register_buffer("row_index", rows)
        self.register_buffer("bias", None if bias is None else bias.detach().to(torch.float32))

    def dense_weight(self):
        """The pruned weight as a dense [out_features, in_features] tensor (for checking)."""
        # undo the preprocessing by compressing the expansion instead of storing DT twice: the kept
        # values are in `values`, their rows are recovered from a multiplication with the identity
        eye = torch.eye(self.in_features, dtype=torch.float32, device=self.values.device)
        return self.forward(eye, add_bias=False).t().contiguous()

    def forward(self, x, add_bias=True):
        if x.dtype != torch.float32 or not x.is_cuda or x.shape[-1] != self.in_features:
            raise ValueError("x must be a float32 CUDA tensor whose last dimension is in_features")
        return sparse_linear(x, self.values, self.indices, self.column_info, self.row_index,
                             self.bias if add_bias else None, self.window, self.kept, self.Ns, self.flags)

    def extra_repr(self):
        return "in_features=%d, out_features=%d, pattern=%d:%d, bias=%s" % (
            self.in_features, self.out_features, self.n, self.m, self.bias is not None)


# ---- operands in 4 bits -----------------------------------------------------------------------------

_native = None


def _binding():
    """csrc/torch_binding.cpp, built beside the library; raises if it has not been (no silent fallback)."""
    global _native
    if _native is None:
        _nm.lib()
        path = os.path.join(os.path.dirname(_nm.LIB_PATH), "_torch_binding.so")
        if not os.path.exists(path):
            raise RuntimeError("_torch_binding.so is not built: run `make -C %s` (or __graft_entry__.build())" % _nm.CSRC_DIR)
        spec = importlib.util.spec_from_file_location(__name__.rsplit(".", 1)[0] + "._torch_binding", path)
        module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(module)
        module.set_error(_nm.NmSpmmError)
        _native = module
    return _native


def _guard(tensor):
    """Makes the tensor's device the current one (kernels are launched there)."""
    return torch.cuda.device(tensor.device)


def _floats(t):
    """float32, contiguous, and in memory what it stands for (a view of a complex tensor's conjugate may not be)."""
    return t.to(torch.float32).contiguous().resolve_neg()


class NMQuantOperand:
    """An operand B [K, N] in 4 bits (nmspmm.h: nmspmm_q4_operand): codes with a scale and a zero point
    per group of kept rows and column; n == m == 1 is a dense operand."""

    def __init__(self, K, N, n=1, m=1, group=128, device="cuda"):
        need = _nm.q4_codes_bytes(K, N, n, m)
        meta = _nm.q4_meta_bytes(K, N, n, m, group)
        if need == 0 or meta == 0:
            raise ValueError("no 4-bit operand of %d x %d with pattern %d:%d and groups of %d: n is 1, 2, 4 or 8 and m is 2 n, "
                             "4 n or 8 n with K %% m == 0 and N %% 32 == 0 (or n == m), group 32, 64 or 128" % (K, N, n, m, group))
        self.K, self.N, self.n, self.m, self.group = K, N, n, m, group
        self.codes = torch.empty(need // 4, dtype=torch.int32, device=device)
        self.scales = torch.empty(meta // 4, dtype=torch.int32, device=device)
        self.row_offsets = None
        if n != m:
            self.row_offsets = torch.empty(_nm.q4_row_offsets_bytes(K, N, n, m), dtype=torch.uint8, device=device)

    def _struct(self):
        return _nm.q4_operand(self.codes, self.scales, self.row_offsets, self.K, self.N, self.n, self.m, self.group)

    def _rows(self, rows, like):
        if self.n == self.m:
            if rows is not None:
                raise ValueError("rows belong to a pattern with n < m")
            return None
        if rows is None or rows.shape != (self.K // self.m * self.n, self.N // 32) or rows.device != like.device:
            raise ValueError("rows must be [K * n / m, N / 32] on the device of the values")
        return rows.to(torch.int32).contiguous()

    @classmethod
    def quantize(cls, values, rows, K, n=1, m=1, group=128, asymmetric=False):
        """From float values [K * n / m, N] and their window-local row numbers [K * n / m, N / 32] (None when n == m)."""
        if values.dim() != 2 or not values.is_cuda or not values.is_floating_point() or n < 1 or m < n or \
                values.shape[0] != _nm.q4_kept_rows(K, n, m):
            raise ValueError("values must be a 2-D floating CUDA tensor of K * n / m rows")
        operand = cls(K, values.shape[1], n, m, group, values.device)
        rows = operand._rows(rows, values)
        with _guard(values):
            _nm.q4_quantize_device(_floats(values), rows, operand._struct(),
                                   _nm.Q4_ASYMMETRIC if asymmetric else 0)
        return operand

    @classmethod
    def from_codes(cls, codes, scale, zero, K, n=1, m=1, rows=None, group=128):
        """From codes 0..15 [W, N] (W = K * n / m), scale and zero 0..15 [ceil(W / group), N]; zero None stands for 8.  Scales are
        kept to 20 significant bits, to the nearest: those that were 16-bit floats are exact, fp32 ones may change by 2^-20 of
        themselves.  Looks at all codes and zero points once (a synchronisation), except while a graph is captured."""
        if codes.dim() != 2 or not codes.is_cuda or codes.dtype != torch.uint8 or n < 1 or m < n or \
                codes.shape[0] != _nm.q4_kept_rows(K, n, m):
            raise ValueError("codes must be a 2-D uint8 CUDA tensor of K * n / m rows")
        operand = cls(K, codes.shape[1], n, m, group, codes.device)
        per_group = (-(-codes.shape[0] // group), codes.shape[1])
        if scale.shape != per_group or scale.device != codes.device or not scale.is_floating_point():
            raise ValueError("scale must be a floating tensor %s on the device of the codes" % (per_group,))
        if zero is not None and (zero.shape != per_group or zero.device != codes.device or zero.is_floating_point()):
            raise ValueError("zero must be a tensor %s of whole numbers 0..15 on the device of the codes" % (per_group,))
        rows = operand._rows(rows, codes)
        with _guard(codes):
            if not torch.cuda.is_current_stream_capturing():
                above = codes.max() > 15
                if zero is not None:
                    above = above | (zero.max() > 15) | (zero.min() < 0)
                if bool(above):
                    raise ValueError("codes and zero points must be 0..15")
            _nm.q4_pack_device(codes.contiguous(), _floats(scale),
                               None if zero is None else zero.to(torch.uint8).contiguous(), rows, operand._struct())
        return operand

    def dense(self):
        """The operand as a dense float32 tensor [K, N] (exact)."""
        out = torch.empty((self.K, self.N), dtype=torch.float32, device=self.codes.device)
        with _guard(out):
            _nm.q4_expand_device(self._struct(), out)
        return out


@torch.library.custom_op("nmspmm::quant_linear", mutates_args=(), device_types="cuda")
def quant_linear(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, row_offsets: Optional[torch.Tensor],
                 bias: Optional[torch.Tensor], K: int, N: int, n: int, m: int, group: int) -> torch.Tensor:
    """x [..., K] row-major times an operand in 4 bits (NMQuantOperand) plus a float32 bias: [..., N] of x's type."""
    return _binding().quant_linear(x, codes, scales, row_offsets, bias, K, N, n, m, group)


@quant_linear.register_fake
def _quant_linear_fake(x, codes, scales, row_offsets, bias, K, N, n, m, group):
    return x.new_empty((*x.shape[:-1], N))


class NMQuantLinear(torch.nn.Module):
    """y = x @ quantize(prune(weight)).T + bias: a linear layer whose kept weights are held in 4 bits.

    weight: floating CUDA tensor [out_features, in_features].  n < m prunes it as NMSparseLinear does (a
    pattern shared by 32 adjacent output features; n 1, 2, 4 or 8, m = 2 n, 4 n or 8 n, m of 4 to 32,
    in_features % m == 0, out_features % 32 == 0); n == m == 1 keeps all of it, at any size.  group: kept
    weights of an output feature that share a scale, 32, 64 or 128; asymmetric: and a zero point of their own.
    x is float32, bfloat16 or float16, the result has its type; sums are taken in float32.  For inference:
    there is no gradient.
    """

    def __init__(self, weight, n=1, m=1, group=128, asymmetric=False, bias=None):
        if weight.dim() != 2 or not weight.is_cuda or not weight.is_floating_point():
            raise ValueError("weight must be a 2-D floating CUDA tensor")
        N, K = weight.shape
        if n != m and (n < 1 or m < n or K % m != 0 or N % 32 != 0 or m not in (4, 8, 16, 32)):
            raise ValueError("pattern %d:%d needs m of 4, 8, 16 or 32, in_features a multiple of it and out_features of 32" % (n, m))
        values, rows = _floats(weight.detach().t()), None
        if n != m:
            dense, W = values, K // m * n
            values = torch.empty((W, N), dtype=torch.float32, device=weight.device)
            rows = torch.empty((W, N // 32), dtype=torch.int32, device=weight.device)
            with _guard(weight):
                _nm.compress_device(dense, K, N, n, m, values, rows)
        self._take(NMQuantOperand.quantize(values, rows, K, n, m, group, asymmetric), bias)

    @classmethod
    def from_codes(cls, codes, scale, zero, in_features, n=1, m=1, rows=None, group=128, bias=None):
        """The layer of weights that are in 4 bits already (NMQuantOperand.from_codes)."""
        layer = cls.__new__(cls)
        layer._take(NMQuantOperand.from_codes(codes, scale, zero, in_features, n, m, rows, group), bias)
        return layer

    def _take(self, operand, bias):
        super().__init__()
        self.in_features, self.out_features = operand.K, operand.N
        self.n, self.m, self.group = operand.n, operand.m, operand.group
        if bias is not None and (bias.shape != (operand.N,) or bias.device != operand.codes.device):
            raise ValueError("bias must have out_features elements on the weight's device")
        self.register_buffer("codes", operand.codes)
        self.register_buffer("scales", operand.scales)
        self.register_buffer("row_offsets", operand.row_offsets)
        self.register_buffer("bias", None if bias is None else _floats(bias.detach()))

    def _operand(self, add_bias=True):
        b = self._buffers
        bias = _floats(b["bias"]) if add_bias and b["bias"] is not None else None     # (.to() may have cast it)
        operand = _nm.q4_operand(b["codes"], b["scales"], b["row_offsets"], self.in_features, self.out_features, self.n, self.m, self.group, bias)
        operand.keeps = bias
        return operand

    def dense_weight(self):
        """The weight as a dense float32 [out_features, in_features] tensor."""
        out = torch.empty((self.in_features, self.out_features), dtype=torch.float32, device=self.codes.device)
        with _guard(out):
            _nm.q4_expand_device(self._operand(add_bias=False), out)
        return out.t().contiguous()

    def forward(self, x):
        b = self._buffers
        bias, codes = b["bias"], b["codes"]
        args = (x, codes, b["scales"], b["row_offsets"], bias, self.in_features, self.out_features, self.n, self.m, self.group)
        # eager inference goes straight to the binding; gradients, tracers, dispatch modes and function transforms (for which it
        # returns None) see the registered operator
        if not torch.compiler.is_compiling() and not (x.requires_grad and torch.is_grad_enabled()):
            y = _binding().quant_linear_direct(*args)
            if y is not None:
                return y
        return quant_linear(*args)

    def extra_repr(self):
        return "in_features=%d, out_features=%d, pattern=%d:%d, group=%d, bias=%s" % (
            self.in_features, self.out_features, self.n, self.m, self.group, self._buffers["bias"] is not None)


# ---- the norms around a block -----------------------------------------------------------------------

_NORMS = {None: _nm.NORM_NONE, "rms": _nm.NORM_RMS, "layer": _nm.NORM_LAYER}


# For tracing front ends: one node forward, one backward.  What is not wanted is an empty tensor.

@torch.library.custom_op("nmspmm::block_norm", mutates_args=(), device_types="cuda")
def _block_norm_op(residual: torch.Tensor, branch: Optional[torch.Tensor], gate: Optional[torch.Tensor], scale: Optional[torch.Tensor],
                   post_weight: Optional[torch.Tensor], post_bias: Optional[torch.Tensor], pre_weight: Optional[torch.Tensor],
                   pre_bias: Optional[torch.Tensor], factor: float, post: int, pre: int, eps: float, weight_offset: float,
                   gate_rows: int, dtype: torch.dtype, want_out: bool) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    total, out, stats = _binding().block_norm_forward([residual, branch, gate, scale, post_weight, post_bias, pre_weight, pre_bias], factor,
                                                      post, pre, eps, weight_offset, gate_rows, dtype, want_out)
    nothing = lambda: residual.new_empty(0)  # noqa: E731
    return nothing() if total is None else total, nothing() if out is None else out, stats


@_block_norm_op.register_fake
def _block_norm_fake(residual, branch, gate, scale, post_weight, post_bias, pre_weight, pre_bias, factor, post, pre, eps,
                     weight_offset, gate_rows, dtype, want_out):
    total = residual.new_empty(0 if branch is None else residual.shape)
    out = residual.new_empty(residual.shape, dtype=dtype) if want_out else residual.new_empty(0)
    return total, out, residual.new_empty((residual.numel() // residual.shape[-1], 4), dtype=torch.float32)


@torch.library.custom_op("nmspmm::block_norm_backward", mutates_args=(), device_types="cuda")
def _block_norm_backward_op(residual: torch.Tensor, branch: Optional[torch.Tensor], gate: Optional[torch.Tensor],
                            scale: Optional[torch.Tensor], post_weight: Optional[torch.Tensor], post_bias: Optional[torch.Tensor],
                            pre_weight: Optional[torch.Tensor], pre_bias: Optional[torch.Tensor], stats: torch.Tensor,
                            grad_sum: Optional[torch.Tensor], grad_out: Optional[torch.Tensor], factor: float, post: int, pre: int,
                            eps: float, weight_offset: float, gate_rows: int, dtype: torch.dtype, want_out: bool,
                            needs: List[bool]) -> List[torch.Tensor]:
    grads = _binding().block_norm_backward([residual, branch, gate, scale, post_weight, post_bias, pre_weight, pre_bias], stats, grad_sum,
                                           grad_out, factor, post, pre, eps, weight_offset, gate_rows, dtype, want_out, needs)
    return [residual.new_empty(0) if g is None else g for g in grads]


@_block_norm_backward_op.register_fake
def _block_norm_backward_fake(residual, branch, gate, scale, post_weight, post_bias, pre_weight, pre_bias, stats, grad_sum, grad_out,
                              factor, post, pre, eps, weight_offset, gate_rows, dtype, want_out, needs):
    given = (residual, branch, gate, scale, post_weight, post_bias, pre_weight, pre_bias)
    return [t.new_empty(t.shape) if need and t is not None else residual.new_empty(0) for t, need in zip(given, needs)]


def _block_norm_setup(ctx, inputs, output):
    ctx.save_for_backward(*inputs[:8], output[2])
    ctx.conf = inputs[8:]
    ctx.has_branch = inputs[1] is not None


def _block_norm_gradients(ctx, grad_sum, grad_out, grad_stats):
    *given, stats = ctx.saved_tensors
    needs = list(ctx.needs_input_grad[:8])
    if not ctx.has_branch:
        grad_sum = None
    if not ctx.conf[7]:
        grad_out = None
    if grad_sum is None and grad_out is None:
        return (None,) * 16
    grads = _block_norm_backward_op(*given, stats, grad_sum, grad_out, *ctx.conf, needs)
    return (*[g if need and t is not None else None for g, need, t in zip(grads, needs, given)], *([None] * 8))


_block_norm_op.register_autograd(_block_norm_gradients, setup_context=_block_norm_setup)


def _gate_rows(gate, shape):
    """(gate, consecutive rows that share one of its rows, 0 for all) for a gate that broadcasts against `shape`."""
    D = shape[-1]
    if gate.shape == (D,):
        return gate, 0
    if gate.dim() == len(shape) and gate.shape[-1] == D:
        lead, each = 0, 1
        while lead < len(shape) - 1 and gate.shape[lead] == shape[lead]:
            lead += 1
        for n in shape[lead:-1]:
            each *= n
        if all(n == 1 for n in gate.shape[lead:-1]):
            return gate, max(each, 1)
    return gate.expand(shape), 1


def block_norm(residual, branch=None, *, gate=None, residual_scale=1.0, post=None, post_weight=None, post_bias=None, pre="rms",
               pre_weight=None, pre_bias=None, eps=1e-6, weight_offset=0.0, dtype=None):
    """The norm after a block, its gate, the scaled residual sum and the norm before the next block, in one launch:

        after = post(branch) * post_weight + post_bias
        sum   = residual * residual_scale + after * gate
        out   = pre(sum) * pre_weight + pre_bias

    and returns (sum, out).  residual [..., D] and branch of its shape, D up to 16384; post and pre are "rms", "layer" or None; without
    a branch (the first norm of a model) sum is the residual; with pre None out is None.  gate broadcasts against
    branch ([D], [batch, 1, D], a whole [batch, tokens, D], ...); residual_scale is a number or a tensor [D] (or of one element); weights and
    biases are [D], weight_offset is added to the weights.  residual is float32 or of branch's type; `dtype` is out's type
    (branch's where there is one, else residual's unless given).  All arithmetic is float32.  Differentiable once with respect to every
    tensor; gradients repeat bit for bit.  (As with any torch operator, capture a backward pass into a graph only while no eager
    autograd graph over the same leaves is alive.)
    """
    if post not in _NORMS or pre not in _NORMS:
        raise ValueError('post and pre are "rms", "layer" or None')
    scale, factor = (residual_scale, 1.0) if isinstance(residual_scale, torch.Tensor) else (None, float(residual_scale))
    if not torch.compiler.is_compiling():
        made = _binding().block_norm(residual, branch, gate, scale, factor, _NORMS[post], post_weight, post_bias, _NORMS[pre], pre_weight,
                                     pre_bias, eps, weight_offset, dtype)
        if made is not None:        # (tracers, dispatch modes and function transforms see the registered operators)
            return made
    D = residual.shape[-1]
    if dtype is None:
        dtype = residual.dtype if branch is None else branch.dtype
    gate_rows = 0
    if gate is not None:
        gate, gate_rows = _gate_rows(gate, residual.shape)
    if scale is not None and scale.shape != (D,):
        scale = scale.reshape(-1).expand(D)
    total, out, _ = _block_norm_op(residual, branch, gate, scale, post_weight, post_bias, pre_weight, pre_bias, factor, _NORMS[post],
                                   _NORMS[pre], eps, weight_offset, gate_rows, dtype, pre is not None)
    return (residual if branch is None else total), (None if pre is None else out)


class NMBlockStack(torch.nn.Module):
    """Blocks of a model around one residual stream, with a norm before and after each of them.

    h = pre_0(x);  for every block i:  x = residual_scale * x + gate_i * post_i(block_i(h));  h = pre_{i+1}(x)
    and returns (x, h), h normed for what follows the last block.  Block i's post norm, gate and sum and block i+1's pre
    norm are one launch (block_norm).  blocks: modules [..., features] -> [..., features] (NMSparseLinear, NMQuantLinear or what is
    built of them); norm: "rms" or "layer"; gate: give each block a learned gate per feature, which starts at gate_init;
    dtype: the type of what the blocks take and return, x's own unless given (x may be float32 beside it).
    """

    def __init__(self, blocks, features, norm="rms", residual_scale=1.0, gate=False, gate_init=1.0, eps=1e-6, dtype=None, device="cuda"):
        super().__init__()
        if norm not in ("rms", "layer"):
            raise ValueError('norm is "rms" or "layer"')
        self.blocks = torch.nn.ModuleList(blocks)
        self.norm, self.residual_scale, self.eps, self.dtype = norm, residual_scale, eps, dtype
        count = len(self.blocks)

        def vectors(n, value):
            return torch.nn.ParameterList([torch.nn.Parameter(torch.full((features,), float(value), device=device)) for _ in range(n)])

        self.pre_weight, self.post_weight = vectors(count + 1, 1.0), vectors(count, 1.0)
        self.pre_bias = vectors(count + 1, 0.0) if norm == "layer" else None
        self.post_bias = vectors(count, 0.0) if norm == "layer" else None
        self.gate = vectors(count, gate_init) if gate else None

    def _pre(self, i):
        return dict(pre=self.norm, pre_weight=self.pre_weight[i], pre_bias=None if self.pre_bias is None else self.pre_bias[i], eps=self.eps)

    def forward(self, x):
        dtype = x.dtype if self.dtype is None else self.dtype
        _, h = block_norm(x, dtype=dtype, **self._pre(0))
        for i, block in enumerate(self.blocks):
            x, h = block_norm(x, block(h), gate=None if self.gate is None else self.gate[i], residual_scale=self.residual_scale,
                              post=self.norm, post_weight=self.post_weight[i],
                              post_bias=None if self.post_bias is None else self.post_bias[i], dtype=dtype, **self._pre(i + 1))
        return x, h
