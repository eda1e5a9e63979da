"""Operands in 4 bits on the GPU against 64-bit arithmetic on the CPU: packing, quantising and expanding are exact,
the product is within the rounding of its fp32 sums."""
import copy
import importlib
import math

import numpy as np
import pytest

from conftest import nmspmm

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def op():
    return importlib.import_module("nm-spmm_amd.torch_op")


def kept_rows(rng, K, N, n, m):
    if n == m:
        return None
    order = rng.random((K // m, m, N // 32)).argsort(axis=1)[:, :n]
    return np.sort(order, axis=1).reshape(K // m * n, N // 32).astype(np.int32)


def make(seed, K, N, n=1, m=1, group=128, zero=True):
    """codes, scale, zero, rows as numpy arrays, and the dense operand in 64 bits."""
    rng = np.random.default_rng(seed)
    W = K // m * n
    groups = -(-W // group)
    codes = rng.integers(0, 16, (W, N)).astype(np.uint8)
    scale = (0.01 * np.exp(rng.normal(size=(groups, N)))).astype(np.float16).astype(np.float32)
    z = rng.integers(0, 16, (groups, N)).astype(np.uint8) if zero else None
    rows = kept_rows(rng, K, N, n, m)
    of = np.arange(W) // group
    values = (codes.astype(np.float64) - (8 if z is None else z[of])) * scale[of].astype(np.float64)
    return codes, scale, z, rows, scatter(values, rows, K, n, m)


def scatter(values, rows, K, n, m):
    if rows is None:
        return values
    W, N = values.shape
    dense = np.zeros((K, N))
    at = (np.arange(W) // n * m)[:, None] + rows
    dense[np.repeat(at, 32, axis=1), np.arange(N)[None, :]] = values
    return dense


def cuda(a):
    return None if a is None else torch.from_numpy(np.ascontiguousarray(a)).cuda()


def layer_of(made, K, n=1, m=1, group=128, bias=None):
    codes, scale, z, rows, dense = made
    return op().NMQuantLinear.from_codes(cuda(codes), cuda(scale), cuda(z), K, n=n, m=m, rows=cuda(rows), group=group,
                                         bias=cuda(bias))


def check(y, x, made, group, bias=None, n=1, m=1):
    """fp32 sums: with u = 16 + code <= 31, a group's two sums add at most 128 terms each of magnitude 31 |x|, the groups,
    waves and pieces add at most W / 128 + 24 more; every addition rounds by 2^-24 of what it holds.  That is the bound on
    each element (times two for the two sums), to which the rounding to the result's type comes.  The errors of the
    roundings are independent: their 2-norm stays below 2^-24 * 31 * 2 / 4.6 (how much larger the two sums are than their
    difference) * sqrt(128), 1e-5 of the result's."""
    codes, scale, z, rows, dense = made
    xd = x.double().cpu().numpy()
    want = xd @ dense
    W = codes.shape[0]
    size = scatter(scale[np.arange(W) // group].astype(np.float64) * np.ones_like(codes, dtype=np.float64), rows,
                   dense.shape[0], n, m)
    bound = 2.0 ** -24 * (128 + W / 128 + 24) * 62.0 * (np.abs(xd) @ np.abs(size))
    if bias is not None:
        want = want + bias
        bound = bound + 2.0 ** -24 * np.abs(want)
    half = 0.0 if y.dtype == torch.float32 else torch.finfo(y.dtype).eps / 2
    tiny = 0.0 if y.dtype == torch.float32 else 2.0 ** -25      # half a step of fp16's subnormal numbers
    got = y.double().cpu().numpy()
    err = np.abs(got - want)
    assert np.all(err <= bound + (np.abs(want) + bound) * half + tiny), float(np.max(err - bound))
    norm = np.linalg.norm(want)
    assert np.linalg.norm(err) <= (1e-5 + half) * norm + tiny * math.sqrt(err.size)



def run(seed, M, K, N, dtype, n=1, m=1, group=128, zero=True, bias=False, layout="plain"):
    made = make(seed, K, N, n, m, group, zero)
    rng = np.random.default_rng(seed + 1)
    b = rng.normal(size=N).astype(np.float32) if bias else None
    layer = layer_of(made, K, n, m, group, b)
    x = torch.from_numpy(rng.normal(size=(M, K)).astype(np.float32)).to(DTYPES[dtype]).cuda()
    if layout == "rows apart":        # a view of a wider tensor, its rows 2-byte aligned only
        wide = torch.full((M, K + 5), float("nan"), dtype=x.dtype, device="cuda")
        wide[:, 3:3 + K] = x
        x = wide[:, 3:3 + K]
    elif layout == "transposed":
        x = x.t().contiguous().t()
    y = layer(x)
    assert y.shape == (M, N) and y.dtype == x.dtype
    check(y, x, made, group, b, n, m)
    return layer, x, y


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("M,K,N", [(1, 1, 1), (1, 7, 5), (1, 128, 16), (1, 129, 17), (1, 4096, 64), (2, 100, 33), (3, 257, 100),
                                   (4, 1000, 48), (5, 1024, 31), (8, 2056, 96), (15, 136, 40), (16, 640, 64), (17, 328, 16),
                                   (33, 1016, 80), (64, 512, 130), (65, 333, 66), (130, 264, 257), (300, 1160, 200)])
def test_dense_operand(dtype, M, K, N):
    run(M + K + N, M, K, N, dtype, group=(32, 64, 128)[(M + K) % 3], zero=K % 2 == 0, bias=N % 2 == 0)


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("n,m", [(1, 2), (2, 4), (4, 8), (8, 16), (1, 4), (2, 8), (8, 32), (1, 8), (4, 32), (8, 64)])
@pytest.mark.parametrize("M,windows,N", [(1, 1, 32), (1, 37, 96), (4, 16, 64), (5, 129, 32), (16, 33, 64), (21, 40, 32), (70, 19, 64),
                                         (150, 32, 128)])
def test_sparse_operand(dtype, n, m, M, windows, N):
    run(M + windows + m, M, windows * m, N, dtype, n, m, group=(32, 64, 128)[(M + n) % 3], zero=M % 2 == 0, bias=windows % 2 == 0)


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("layout", ["rows apart", "transposed"])
@pytest.mark.parametrize("M,K,N,n,m", [(1, 512, 64, 1, 1), (3, 264, 40, 1, 1), (19, 1024, 64, 1, 1), (130, 256, 96, 1, 1),
                                       (2, 256, 64, 2, 8), (70, 256, 64, 2, 4)])
def test_rows_of_x_with_strides(dtype, layout, M, K, N, n, m):
    run(M, M, K, N, dtype, n, m, layout=layout)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("n,m", [(1, 2), (2, 4), (4, 8), (8, 16)])
@pytest.mark.parametrize("M,K,N,group", [(5, 272, 96, 32), (8, 2064, 32, 128), (9, 16, 32, 64), (13, 784, 64, 128), (16, 1536, 64, 32),
                                         (11, 528, 8256, 64), (7, 528, 8256, 32)])
def test_aligned_rows_of_a_half_kept_operand(dtype, n, m, M, K, N, group):
    """Rows that are read whole and gathered afterwards: what lies behind them and what they hold in places that are not
    kept does not count, and the result is that of rows which cannot be read so."""
    layer, x, y = run(M + K, M, K, N, dtype, n, m, group)
    wide = torch.full((M, K + 8), float("nan"), dtype=x.dtype, device="cuda")
    wide[:, :K] = x
    assert torch.equal(layer(wide[:, :K]), y)
    odd = torch.full((M, K + 5), float("nan"), dtype=x.dtype, device="cuda")[:, 3:3 + K]
    odd.copy_(x)
    # the same products in the same order, whichever way the elements came
    assert torch.equal(layer(odd), y)
    first = layer.row_offsets.view(N // 32, -1)[0, :1].item()       # in the first 32 columns not kept: the first window's first other row
    lost = 1 if first == 0 else 0
    if n == 1:
        wide[:, lost] = float("inf")
        y2 = layer(wide[:, :K])
        assert torch.equal(y2[:, :32], y[:, :32])


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M,n,m", [(1, 1, 1), (4, 1, 1), (7, 1, 1), (13, 1, 1), (16, 1, 1), (6, 2, 8), (16, 2, 8), (14, 2, 4)])
def test_wide_operands(dtype, group, M, n, m):
    """Enough columns for every compute unit twice over."""
    run(M + group, M, 416, 8224, dtype, n, m, group)


def test_leading_dimensions_and_empty_batches():
    made = make(3, 256, 64)
    layer = layer_of(made, 256)
    x = torch.randn((2, 3, 5, 256), device="cuda")
    y = layer(x)
    assert y.shape == (2, 3, 5, 64) and torch.equal(y.reshape(30, 64), layer(x.reshape(30, 256)))
    assert layer(x[:, :0]).shape == (2, 0, 5, 64)
    # one row of a batch does not depend on how it is shaped, and an expanded x has rows zero elements apart
    assert torch.equal(layer(x[0, 0, 0]), layer(x[0, 0, 0].reshape(1, 256))[0])
    e = x[0, 0, 0].expand(4, 256)
    assert torch.equal(layer(e), layer(e.contiguous()))


@pytest.mark.parametrize("M", [1, 8, 40, 200])
def test_only_the_rows_and_columns_of_y_are_written(M):
    made = make(4, 320, 40)
    layer = layer_of(made, 320)
    x = torch.randn((M, 320), device="cuda", dtype=torch.bfloat16)
    y = torch.full((M + 2, 47), 7.0, device="cuda", dtype=torch.bfloat16)
    need = nmspmm.q4_workspace_bytes(M, 320, 40, 1, 1, nmspmm.BF16)
    assert (need == 0) == (M <= 8)
    space = torch.empty(need, dtype=torch.uint8, device="cuda") if need else None
    nmspmm.q4_linear(layer._operand(), x, y[1:], M, nmspmm.BF16, ldy=47, workspace=space)
    assert torch.equal(y[1:M + 1, :40], layer(x))
    assert bool((y[0] == 7).all()) and bool((y[M + 1] == 7).all()) and bool((y[1:M + 1, 40:] == 7).all())


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("M,n,m", [(1, 1, 1), (6, 1, 1), (80, 1, 1), (6, 2, 8), (80, 2, 8)])
def test_a_bad_row_of_x_stays_its_own(dtype, M, n, m):
    made = make(6, 256, 64, n, m)
    layer = layer_of(made, 256, n, m)
    x = torch.randn((M, 256), device="cuda").to(DTYPES[dtype])
    good = layer(x)
    bad = x.clone()
    bad[0] = float("inf")
    if M > 1:
        bad[M - 1] = float("nan")
    got = layer(bad)
    assert bool(got[0].isnan().all()) and bool(got[M - 1].isnan().all())
    assert torch.equal(got[1:M - 1], good[1:M - 1])


def test_padding_behind_x_is_not_read_into_the_result():
    """K = 136: the last block has 8 of its 128 rows; what lies behind each row of x is NaN."""
    for dtype in DTYPES.values():
        made = make(7, 136, 32)
        layer = layer_of(made, 136)
        wide = torch.full((5, 1024), float("nan"), device="cuda", dtype=dtype)
        wide[:, :136] = torch.randn((5, 136), device="cuda").to(dtype)
        check(layer(wide[:, :136]), wide[:, :136], made, 128)


def quantized(v, group, asymmetric):
    """(values that the codes stand for, scale, zero) by the rule of nmspmm.h, in exact arithmetic where it matters."""
    W, N = v.shape
    out = np.empty_like(v, dtype=np.float64)
    for b in range(0, W, group):
        w = v[b:b + group].astype(np.float64)
        if asymmetric:
            need = (np.maximum(w.max(0), 0) - np.minimum(w.min(0), 0)) / 15
        else:
            need = np.abs(w).max(0) / 7
        f, e = np.frexp(need)
        scale = np.ldexp(np.ceil(np.ldexp(f, 20)), e - 20)
        some = np.where(scale > 0, scale, 1.0)
        zero = np.clip(np.rint(-np.minimum(w.min(0), 0) / some), 0, 15) if asymmetric else 8.0
        out[b:b + group] = (np.clip(np.rint(w / some) + zero, 0, 15) - zero) * scale
    return out


@pytest.mark.parametrize("asymmetric", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("K,N,n,m", [(1, 1, 1, 1), (100, 17, 1, 1), (128, 64, 1, 1), (700, 130, 1, 1), (256, 64, 2, 4), (1000, 96, 2, 8),
                                     (264, 32, 1, 8), (640, 32, 8, 32), (64, 32, 8, 64), (14, 32, 1, 2)])
def test_quantise_and_expand_are_exact(K, N, n, m, group, asymmetric):
    rng = np.random.default_rng(K + N + group)
    W = K // m * n
    v = (0.02 * rng.normal(size=(W, N))).astype(np.float32)
    v[:, 0] = 0.0                                               # a column of zeros
    if N > 3:
        v[:, 1] = np.abs(v[:, 1])                               # of one sign
        v[:, 2] = rng.integers(-14, 15, W).astype(np.float32) * 0.5   # quotients on the border between two codes
        v[:, 3] = (v[:, 3] * 1e-38).astype(np.float32)          # subnormal numbers
        v[: W // 2, 3] = 0.0
    rows = kept_rows(rng, K, N, n, m)
    operand = op().NMQuantOperand.quantize(cuda(v), cuda(rows), K, n=n, m=m, group=group, asymmetric=asymmetric)
    want = scatter(quantized(v, group, asymmetric), rows, K, n, m)
    got = operand.dense().cpu().numpy()
    keep = np.ones(N, bool)
    if N > 3:
        keep[3] = False     # a scale of 20 bits need not exist below 2^-126: those are near, not equal
        assert np.max(np.abs(got[:, 3])) < 1e-38
    assert np.array_equal(got[:, keep], want[:, keep].astype(np.float32))


def test_values_next_to_a_border_go_to_the_nearer_code():
    """v = (k + 1/2) * scale exactly, and one step of fp32 above and below it."""
    base = np.float32(7 * 0.3)
    scale = quantized(np.array([[base]], np.float32), 32, False)[0, 0] / 7
    v = []
    for k in range(-7, 7):
        mid = np.float32((k + 0.5) * scale)
        v += [mid, np.nextafter(mid, np.float32(9)), np.nextafter(mid, np.float32(-9))]
    v = np.array([base] + v, np.float32)[:, None]
    got = op().NMQuantOperand.quantize(cuda(v), None, len(v), group=128).dense().cpu().numpy()
    assert np.array_equal(got, quantized(v, 128, False).astype(np.float32))


def test_codes_that_exist_already_come_back():
    for n, m in ((1, 1), (2, 8), (8, 64)):
        made = make(9, 512, 96, n, m, 64)
        operand = op().NMQuantOperand.from_codes(cuda(made[0]), cuda(made[1]), cuda(made[2]), 512, n=n, m=m, rows=cuda(made[3]), group=64)
        assert np.array_equal(operand.dense().cpu().numpy(), made[4].astype(np.float32))


@pytest.mark.parametrize("where", ["value", "scale"])
def test_what_is_not_finite_makes_its_group_nan(where):
    v = torch.randn((200, 20), device="cuda")
    if where == "value":
        v[70, 3], v[150, 5] = float("inf"), float("nan")
        d = op().NMQuantOperand.quantize(v, None, 200, group=64).dense()
    else:
        scale = torch.ones((4, 20), device="cuda")
        scale[1, 3], scale[2, 5] = float("inf"), float("nan")
        d = op().NMQuantOperand.from_codes(torch.full((200, 20), 3, dtype=torch.uint8, device="cuda"), scale, None, 200, group=64).dense()
    bad = d.isnan()
    want = torch.zeros_like(bad)
    want[64:128, 3] = True
    want[128:192, 5] = True
    assert torch.equal(bad, want)


@pytest.mark.parametrize("from_codes", [False, True])
def test_a_row_outside_its_window_counts_as_zero(from_codes):
    K, N, n, m = 256, 64, 2, 8
    made = make(10, K, N, n, m, 64)
    rows = made[3].copy()
    rows[5, 0], rows[17, 1], rows[63, 0] = -1, 8, 1 << 20
    values = torch.randn((64, N), device="cuda")
    if from_codes:
        operand = op().NMQuantOperand.from_codes(cuda(made[0]), cuda(made[1]), cuda(made[2]), K, n=n, m=m, rows=cuda(rows), group=64)
    else:
        operand = op().NMQuantOperand.quantize(values, cuda(rows), K, n=n, m=m, group=64, asymmetric=True)
        good = op().NMQuantOperand.quantize(values, cuda(made[3]), K, n=n, m=m, group=64, asymmetric=True)
    x = torch.eye(K, device="cuda")
    layer = op().NMQuantLinear.__new__(op().NMQuantLinear)
    layer._take(operand, None)
    got = layer(x).cpu().numpy()
    want = made[4].copy() if from_codes else good.dense().double().cpu().numpy()
    for r, v in ((5, 0), (17, 1), (63, 0)):
        want[r // n * m + made[3][r, v], v * 32:(v + 1) * 32] = 0.0
    # x is the identity: one term is not zero, its sum is exact
    assert np.array_equal(got, want.astype(np.float32))


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("n,m", [(1, 1), (2, 4), (2, 8), (1, 8)])
def test_layer_made_from_a_weight(dtype, n, m):
    w = torch.randn((96, 512), device="cuda") * 0.05
    b = torch.randn(96, device="cuda")
    layer = op().NMQuantLinear(w.to(DTYPES[dtype]), n, m, group=64, asymmetric=m == 8, bias=b)
    dense = layer.dense_weight()
    kept = w.to(DTYPES[dtype]).float()
    if n < m:       # the rows that compression keeps of the same weight
        pruned = op().NMSparseLinear(kept, n, m).dense_weight()
        assert not bool(((pruned == 0) & (dense != 0)).any())
        kept = pruned
    # half a step of a scale that covers the group: at most max|w| / 7 (1 + 2^-19) / 2, one step where a zero point was rounded too
    assert float((dense - kept).abs().max()) <= float(kept.abs().max()) / 7 * (1 + 2 ** -19) * (1.0 if m == 8 else 0.5) + 1e-7
    x = torch.randn((3, 512), device="cuda").to(DTYPES[dtype])
    want = x.double() @ dense.double().t() + b.double()
    got = layer(x).double()
    half = 0.0 if dtype == "fp32" else torch.finfo(DTYPES[dtype]).eps / 2
    assert float((got - want).norm()) <= (1e-5 + half) * float(want.norm())


def test_layer_survives_moves_copies_and_loading():
    w = torch.randn((64, 256), device="cuda")
    layer, other = op().NMQuantLinear(w, 2, 4, bias=torch.randn(64, device="cuda")), op().NMQuantLinear(-w, 2, 4, bias=torch.zeros(64, device="cuda"))
    x = torch.randn((2, 256), device="cuda")
    y = layer(x)
    twin = copy.deepcopy(layer)
    assert torch.equal(twin(x), y)
    other.load_state_dict(layer.state_dict())
    assert torch.equal(other(x), y)
    back = layer.cpu().cuda()
    assert torch.equal(back(x), y)
    half = copy.deepcopy(layer).to(torch.bfloat16)      # casts the bias only
    assert half(x.bfloat16()).dtype == torch.bfloat16


def test_registered_operator_traces_and_matches():
    layer = op().NMQuantLinear(torch.randn((64, 256), device="cuda"), bias=torch.randn(64, device="cuda"))
    x = torch.randn((5, 256), device="cuda")
    y = layer(x)
    assert torch.equal(torch.compile(layer, fullgraph=True, backend="aot_eager")(x), y)
    exported = torch.export.export(layer, (x,))
    assert sum("nmspmm.quant_linear" in str(n.target) for n in exported.graph.nodes if n.op == "call_function") == 1
    assert torch.equal(exported.module()(x), y)
    torch.library.opcheck(op().quant_linear, (x, layer.codes, layer.scales, None, layer.bias, 256, 64, 1, 1, 128))


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("M,n,m", [(1, 1, 1), (1, 2, 8), (12, 1, 1), (12, 2, 8), (24, 1, 1), (24, 2, 8), (150, 1, 1), (150, 2, 4)])
def test_graph_replays(M, n, m, dtype):
    made = make(12, 2048, 128, n, m)
    layer = layer_of(made, 2048, n, m)
    x = torch.randn((M, 2048), device="cuda", dtype=DTYPES[dtype])
    layer(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layer(x)
    for k in range(4):
        x.copy_(torch.randn((M, 2048), device="cuda"))
        want = layer(x)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)


def test_two_streams_and_repeats_agree_bit_for_bit():
    layers = [layer_of(make(s, 2048, 512, n, m), 2048, n, m) for s, n, m in ((20, 1, 1), (21, 2, 8))]
    xs = [torch.randn((M, 2048), device="cuda", dtype=t) for M, t in ((1, torch.float32), (7, torch.bfloat16), (100, torch.float16))]
    want = [layer(x) for layer in layers for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for k in range(6):
        for layer in layers:
            for x in xs:
                with torch.cuda.stream(streams[k % 2]):
                    got.append(layer(x))
    torch.cuda.synchronize()
    for k, y in enumerate(got):
        assert torch.equal(y, want[k % len(want)])


def test_offsets_beyond_32_bits():
    """x of more than 4 GiB: its last rows are multiplied like any others, the zeros before them give zeros.  Codes of more than 4 GiB (K 2^17, N 2^16 and a bit): the
    last columns are those of an operand that holds only them."""
    made = make(30, 8192, 96)
    layer = layer_of(made, 8192)
    M = 280000
    x = torch.zeros((M, 8192), dtype=torch.bfloat16, device="cuda")
    tail = torch.randn((70, 8192), device="cuda").bfloat16()
    x[-70:] = tail
    y = layer(x)
    assert not bool(y[:-70].any())
    check(y[-70:], tail, made, 128)
    del x, y
    K, N = 1 << 17, (1 << 16) + 64
    codes = torch.randint(0, 16, (K, N), dtype=torch.uint8, device="cuda")
    scale = torch.rand((K // 128, N), device="cuda").half().float()
    layer = op().NMQuantLinear.from_codes(codes, scale, None, K)
    small = op().NMQuantLinear.from_codes(codes[:, -128:].contiguous(), scale[:, -128:].contiguous(), None, K)
    del codes, scale
    for M, dtype in ((1, torch.float32), (3, torch.bfloat16), (100, torch.float16)):
        x = torch.randn((M, K), device="cuda").to(dtype)
        got, want = layer(x)[:, -128:].double(), small(x).double()
        # other waves and ranges of K may take the blocks: fp32 sums in another order, each below 1e-5 of its norm
        half = 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps
        assert float((got - want).norm()) <= (2e-5 + half) * float(want.norm())


def test_refusals():
    layer = layer_of(make(13, 256, 64), 256)
    x = torch.randn((2, 256), device="cuda")
    for bad in (x.double(), x[:, :255], x.cpu(), x.to(torch.int32)):
        with pytest.raises((ValueError, NotImplementedError)):
            layer(bad)
    w = torch.randn((64, 256), device="cuda")
    for args in ((w, 3, 8), (w, 2, 32), (w, 1, 2), (w[:48], 2, 4), (w[:, :250], 2, 4), (w, 1, 1, 16), (w.cpu(),), (w[0],), (w, 4, 2)):
        with pytest.raises(ValueError):
            op().NMQuantLinear(*args)
    with pytest.raises(ValueError):
        op().NMQuantLinear(w, bias=torch.zeros(63, device="cuda"))
    codes, scale, _, _, _ = make(1, 256, 64)
    with pytest.raises(ValueError):
        op().NMQuantOperand.from_codes(cuda(codes), cuda(scale)[:1], None, 256, group=128)
    with pytest.raises(ValueError):
        op().NMQuantOperand.from_codes(cuda(codes).int(), cuda(scale), None, 256)
    with pytest.raises(ValueError):
        op().NMQuantOperand.from_codes(cuda(codes), cuda(scale), cuda(scale), 256)       # a zero point that is no whole number
    with pytest.raises(ValueError):
        op().NMQuantOperand.from_codes(cuda(codes), cuda(scale), None, 512, n=1, m=2)     # no rows
    with pytest.raises(ValueError):
        op().NMQuantOperand.quantize(torch.randn((256, 64), device="cuda"), torch.zeros((256, 2), dtype=torch.int32, device="cuda"), 256)


def test_the_operator_refuses_buffers_that_are_not_the_operands():
    codes, scale, zero, rows, _ = make(2, 256, 64, 2, 4)
    o = op().NMQuantOperand.from_codes(cuda(codes), cuda(scale), cuda(zero), 256, 2, 4, cuda(rows))
    x = torch.randn((3, 256), device="cuda")
    good = [x, o.codes, o.scales, o.row_offsets, None, 256, 64, 2, 4, 128]
    f = torch.ops.nmspmm.quant_linear
    want = f(*good)
    assert torch.equal(f(*good[:4], torch.zeros(64, device="cuda", dtype=torch.bfloat16), *good[5:]), want)
    for at, bad in ((1, o.codes[:-1]), (1, o.codes[::2]), (2, o.scales[:-1]), (3, o.row_offsets[:-1]), (3, None), (4, x[0, :63]),
                    (4, x[:, :64]), (6, 96), (6, 0), (6, 1 << 40), (7, 3), (8, 5), (8, 1), (9, 48), (9, 0)):
        args = list(good)
        args[at] = bad
        with pytest.raises(ValueError):
            f(*args)


def test_too_many_rows_are_refused():
    o = op().NMQuantLinear.from_codes(torch.zeros((1, 1), dtype=torch.uint8, device="cuda"), torch.ones((1, 1), device="cuda"), None, 1)
    with pytest.raises(ValueError):
        o(torch.zeros(((1 << 24) + 1, 1), dtype=torch.float16, device="cuda"))


def test_negated_views_and_tangents():
    layer = layer_of(make(4, 256, 64), 256)
    z = torch.randn((3, 256), dtype=torch.complex64, device="cuda")
    x = z.conj().imag
    assert x.is_neg() and torch.equal(layer(x), layer(-z.imag))
    w = torch.randn((32, 64), dtype=torch.complex64, device="cuda").conj().imag
    assert torch.equal(op().NMQuantLinear(w).dense_weight(), op().NMQuantLinear(w.resolve_neg()).dense_weight())
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises((ValueError, RuntimeError)):
            layer(torch.autograd.forward_ad.make_dual(z.real.contiguous(), z.real.contiguous()))


def test_a_dense_operand_may_be_named_by_any_n_and_m():
    codes, scale, zero, _, _ = make(6, 300, 40)
    a, b, c = (op().NMQuantLinear.from_codes(cuda(codes), cuda(scale), cuda(zero), 300, n, n) for n in (1, 100, 7))
    x = torch.randn((2, 300), device="cuda")
    assert torch.equal(a(x), b(x)) and torch.equal(a(x), c(x))
    v = torch.randn((300, 40), device="cuda")
    assert torch.equal(op().NMQuantOperand.quantize(v, None, 300).dense(), op().NMQuantOperand.quantize(v, None, 300, 7, 7).dense())
    with pytest.raises(ValueError):     # all rows of a dense operand, not the 294 of whole windows
        op().NMQuantOperand.quantize(v[:294], None, 300, 7, 7)
    with pytest.raises(ValueError):
        op().NMQuantOperand.from_codes(cuda(codes)[:294], cuda(scale), cuda(zero), 300, 7, 7)
