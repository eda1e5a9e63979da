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
from typing import Optional

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

_TYPES = {torch.float32: _nm.F32, torch.bfloat16: _nm.BF16, torch.float16: _nm.F16}


def _on(device):
    """The stream that calls for tensors on this device go to (its current one), as an integer."""
    return torch.cuda.current_stream(device).cuda_stream


def _guard(tensor):
    """Makes the tensor's device the current one (kernels are launched there) where it is not."""
    return torch.cuda.device(tensor.device)


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
                values.shape[0] != K // m * n:
            raise ValueError("values must be a 2-D floating CUDA tensor of K * n / m rows")
        operand = cls(K, values.shape[1], n, m, group, values.device)
        rows = operand._rows(rows, values)
        with _guard(values):
            _nm.q4_quantize_device(values.to(torch.float32).contiguous(), rows, operand._struct(),
                                   _nm.Q4_ASYMMETRIC if asymmetric else 0)
        return operand

    @classmethod
    def from_codes(cls, codes, scale, zero, K, n=1, m=1, rows=None, group=128):
        """From codes 0..15 [W, N] (W = K * n / m), scale and zero [ceil(W / group), N]; zero None stands for 8."""
        if codes.dim() != 2 or not codes.is_cuda or codes.dtype != torch.uint8 or n < 1 or m < n or codes.shape[0] != K // m * n:
            raise ValueError("codes must be a 2-D uint8 CUDA tensor of K * n / m rows")
        operand = cls(K, codes.shape[1], n, m, group, codes.device)
        per_group = (-(-codes.shape[0] // group), codes.shape[1])
        if scale.shape != per_group or scale.device != codes.device or not scale.is_floating_point():
            raise ValueError("scale must be a floating tensor %s on the device of the codes" % (per_group,))
        if zero is not None and (zero.shape != per_group or zero.device != codes.device):
            raise ValueError("zero must be a tensor %s on the device of the codes" % (per_group,))
        rows = operand._rows(rows, codes)
        with _guard(codes):
            _nm.q4_pack_device(codes.contiguous(), scale.to(torch.float32).contiguous(),
                               None if zero is None else zero.to(torch.uint8).contiguous(), rows, operand._struct())
        return operand

    def dense(self):
        """The operand as a dense float32 tensor [K, N] (exact)."""
        out = torch.empty((self.K, self.N), dtype=torch.float32, device=self.codes.device)
        with _guard(out):
            _nm.q4_expand_device(self._struct(), out)
        return out


def _quant_linear(x, operand):
    """x [..., K] times the operand of the struct (its bias added): [..., N] of x's type."""
    K, N = operand.K, operand.N
    if x.shape[-1] != K or x.dtype not in _TYPES or not x.is_cuda:
        raise ValueError("x must be a float32, bfloat16 or float16 CUDA tensor whose last dimension is %d" % K)
    y = x.new_empty((*x.shape[:-1], N))
    M = y.numel() // N
    if M == 0:
        return y
    if x.dim() != 2:
        x = x.reshape(M, K)
    ldx = x.stride(0) if M > 1 else K
    if (K > 1 and x.stride(1) != 1) or ldx < K:
        x, ldx = x.contiguous(), K
    device = x.device
    if device.index != torch.cuda.current_device():
        with _guard(x):
            return _launch_quant_linear(x, ldx, y, N, M, operand, device)
    return _launch_quant_linear(x, ldx, y, N, M, operand, device)


def _launch_quant_linear(x, ldx, y, ldy, M, operand, device):
    status = _nm.lib().nmspmm_q4_linear(operand, x.data_ptr(), ldx, y.data_ptr(), ldy, M, _TYPES[x.dtype], _on(device))
    if status != _nm.OK:
        raise _nm.NmSpmmError("nmspmm_q4_linear", status)
    return y


@torch.library.custom_op("nmspmm::quant_linear", mutates_args=(), device_types="cuda")
def quant_linear(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, row_offsets: Optional[torch.Tensor],
                 bias: Optional[torch.Tensor], K: int, N: int, n: int, m: int, group: int) -> torch.Tensor:
    """x [..., K] row-major times an operand in 4 bits (NMQuantOperand) plus a float32 bias: [..., N] of x's type."""
    for t in (codes, scales, row_offsets, bias):
        if t is not None and (t.device != x.device or not t.is_contiguous()):
            raise ValueError("the operand's buffers and the bias must be contiguous and on the device of x")
    if bias is not None:
        bias = bias.to(torch.float32)
    return _quant_linear(x, _nm.q4_operand(codes, scales, row_offsets, K, N, n, m, group, bias))


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
        values, rows = weight.detach().t().to(torch.float32).contiguous(), None
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
        self.register_buffer("bias", None if bias is None else bias.detach().to(torch.float32).contiguous())

    def _operand(self):
        # the struct of device pointers is kept between calls and follows the buffers
        b = self._buffers
        codes, scales, rows, bias = b["codes"], b["scales"], b["row_offsets"], b["bias"]
        at = (codes.data_ptr(), scales.data_ptr(), None if rows is None else rows.data_ptr(), None if bias is None else bias.data_ptr())
        kept = self.__dict__.get("_struct")
        if kept is None or kept[0] != at:
            kept = (at, _nm.q4_operand(codes, scales, rows, self.in_features, self.out_features, self.n, self.m, self.group, bias))
            self.__dict__["_struct"] = kept
        return kept[1]

    def __getstate__(self):
        return {k: v for k, v in self.__dict__.items() if k != "_struct"}

    def dense_weight(self):
        """The weight as a dense float32 [out_features, in_features] tensor."""
        out = torch.empty((self.in_features, self.out_features), dtype=torch.float32, device=self.codes.device)
        with _guard(out):
            _nm.q4_expand_device(self._operand(), out)
        return out.t().contiguous()

    def forward(self, x):
        b = self._buffers
        bias, codes = b["bias"], b["codes"]
        # eager inference on the layer's device goes straight to the library; tracing, gradients and
        # layers that were cast go through the registered operator
        if type(x) is torch.Tensor and not torch.compiler.is_compiling() and x.device == codes.device and \
                (bias is None or bias.dtype is torch.float32) and not (x.requires_grad and torch.is_grad_enabled()):
            return _quant_linear(x, self._operand())
        return quant_linear(x, codes, b["scales"], b["row_offsets"], bias, self.in_features, self.out_features, self.n, self.m, self.group)

    def extra_repr(self):
        return "in_features=%d, out_features=%d, pattern=%d:%d, group=%d, bias=%s" % (
            self.in_features, self.out_features, self.n, self.m, self.group, self._buffers["bias"] is not None)
