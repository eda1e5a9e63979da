"""What the sums of the 4-bit product with a sparse operand may lose, element by element, in 64 bits: rows of x that the pattern
drops do not enter them."""
import numpy as np
import pytest

from test_gpu_q4 import DTYPES, layer_of, make, scatter

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def exact_terms_bound(x, dense, group, W):
    """Products of a piece of x (8 bits) and code - zero (4 bits) are exact in fp32.  A unit of at most 128 rows adds 3 * 128 of them,
    its scaling rounds once, the units and the ranges of K add W / 32 + 24 more: each addition is off by at most
    2^-23 (a matrix instruction may cut its inner sums off) of the magnitudes added so far, the pieces' being 1.02 of x's at most."""
    return 2.0 ** -23 * (3 * 128 + W / 32 + 24) * 1.02 * (np.abs(x) @ np.abs(dense))


def group_sums_bound(x, size, W):
    """Where zero points are taken off group sums (few rows): with u = 16 + code <= 31 a group's two sums add 128 terms of
    at most 31 |x| each, the groups, waves and pieces W / 128 + 24 more; each addition is within 2^-24 of what it holds."""
    return 2.0 ** -24 * (128 + W / 128 + 24) * 62.0 * (np.abs(x) @ np.abs(size))


def rounded(bound, want, dtype):
    half = 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
    tiny = 0.0 if dtype == torch.float32 else 2.0 ** -25
    return bound + (np.abs(want) + bound) * half + tiny


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("outlier", [1e3, 3e4])
@pytest.mark.parametrize("n,m,group", [(1, 8, 32), (2, 8, 128), (2, 4, 64), (4, 8, 128), (8, 64, 32), (1, 2, 128)])
@pytest.mark.parametrize("M", [17, 64, 150])
def test_dropped_rows_do_not_enter_the_sums(M, n, m, group, outlier, dtype):
    K, N = 16 * m if m > 16 else 512, 192
    made = make(M + m, K, N, n, m, group)
    codes, scale, z, rows, dense = made
    layer = layer_of(made, K, n, m, group)
    rng = np.random.default_rng(M)
    x = rng.normal(size=(M, K)).astype(np.float32)
    x[:, [5, K // 2 + 5]] *= outlier / 4        # (fp16's largest number is 65504)
    t = torch.from_numpy(x).to(DTYPES[dtype]).clamp(-6e4, 6e4).cuda()
    y = layer(t)
    xd, got = t.double().cpu().numpy(), y.double().cpu().numpy()
    want = xd @ dense
    err = np.abs(got - want)
    W = codes.shape[0]
    size = scatter(scale[np.arange(W) // group].astype(np.float64) * np.ones_like(codes, dtype=np.float64), rows, K, n, m)
    sums = group_sums_bound(xd, size, W)
    gathered = M <= 32 and (dtype != "fp32" or m > 2 * n or group == 128)
    bound = rounded(sums if gathered else exact_terms_bound(xd, dense, group, W), want, DTYPES[dtype])
    if dtype == "fp16":     # (a sum beyond its largest number)
        bound = np.where(np.abs(want) > 65000, np.inf, bound)
    assert np.all(~(err > bound)), float(np.nanmax(err / bound))
    # without the kept outliers: independent roundings of sums that grow like their result's norm, sqrt(3 * 128 + W / 32 + 24) of
    # 2^-23 each, 2.5e-6 of it; one more of the result's type
    if dtype == "fp32" and not gathered:
        vectors = [v for v in range(N // 32) if not np.any(dense[[5, K // 2 + 5], v * 32:v * 32 + 32])]
        for v in vectors:
            s = slice(v * 32, v * 32 + 32)
            assert np.linalg.norm(err[:, s]) <= 2.5e-6 * np.linalg.norm(want[:, s])
    # sixteen of the rows alone
    few = layer(t[:16].contiguous()).double().cpu().numpy()
    other = rounded(sums[:16], want[:16], DTYPES[dtype])
    apart = np.abs(few - got[:16])
    assert np.all(~(apart > bound[:16] + other)), float(np.nanmax(apart / (bound[:16] + other)))


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("n,m,group", [(1, 8, 32), (2, 8, 128), (2, 4, 64), (4, 8, 128), (8, 64, 32), (1, 2, 128)])
@pytest.mark.parametrize("M", [1, 5, 16, 17, 32, 33, 150])
def test_what_a_pattern_drops_changes_no_bit(M, n, m, group, dtype):
    K, N = 1024, 256
    made = make(M + m, K, N, n, m, group)
    rows = made[3].reshape(K // m, n, N // 32)
    layer = layer_of(made, K, n, m, group)
    x = torch.randn((M, K), device="cuda").to(DTYPES[dtype])
    window, column = next((w, c) for w in range(K // m) for c in range(m) if 0 < (rows[w] == c).any(0).sum() < N // 32)
    drops = ~(rows[window] == column).any(0)
    keep = torch.from_numpy(np.repeat(drops, 32)).cuda()
    y = layer(x)
    for value in (0.0, 6e4, -1e-3):
        x[:, window * m + column] = value
        assert torch.equal(layer(x)[:, keep], y[:, keep])


@pytest.mark.parametrize("outlier", [1e3, 1e5])
def test_an_outlier_that_one_vector_drops(outlier):
    """One column of x is large, and only some vectors keep it: the others' results do not know of it."""
    K, N, n, m = 512, 256, 2, 8
    made = make(5, K, N, n, m, 128)
    rows, dense = made[3], made[4]
    column = 8 * 3 + rows[6, 0]         # kept by the first vector
    drops = [v for v in range(N // 32) if column - 24 not in rows[6:8, v]]
    assert drops and 0 not in drops
    layer = layer_of(made, K, n, m)
    x = torch.randn((40, K), device="cuda")
    x[:, column] = outlier
    y, want = layer(x).double().cpu().numpy(), x.double().cpu().numpy() @ dense
    for v in drops:
        s = slice(v * 32, v * 32 + 32)
        assert np.linalg.norm(y[:, s] - want[:, s]) <= 2.5e-6 * np.linalg.norm(want[:, s])      # as above


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("n,m", [(2, 4), (1, 8)])
def test_sparse_rows_replay_in_a_graph_and_share_no_workspace(n, m, dtype):
    made = make(14, 1024, 160, n, m, 64)
    layer = layer_of(made, 1024, n, m, 64)
    xs = [torch.randn((M, 1024), device="cuda").to(DTYPES[dtype]) for M in (33, 90)]
    for x in xs:
        layer(x)
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in xs]
    ys = []
    for g, x in zip(graphs, xs):
        with torch.cuda.graph(g):
            ys.append(layer(x))
    for k in range(4):
        for x in xs:
            x.copy_(torch.randn(x.shape, device="cuda"))
        want = [layer(x) for x in xs]
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(ys, want))


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("n,m,windows", [(1, 8, 37), (2, 8, 37), (2, 4, 85), (4, 8, 43), (8, 64, 13), (1, 2, 39), (1, 4, 1), (8, 16, 5), (2, 4, 86)])
@pytest.mark.parametrize("M", [1, 4, 8, 13, 32, 40])
def test_what_fills_the_last_step_reads_no_dropped_row(M, n, m, windows, dtype):
    """W is no multiple of 32: the kept rows of the last step are filled up.  The first dense row of that step is dropped by some vectors."""
    K, N = windows * m, 256
    made = make(M + m, K, N, n, m, 32)
    rows = made[3].reshape(windows, n, N // 32)
    window = windows * n // 32 * 32 // n
    drops = ~(rows[window] == 0).any(0)
    assert drops.any()
    layer = layer_of(made, K, n, m, 32)
    keep = torch.from_numpy(np.repeat(drops, 32)).cuda()
    x = torch.randn((M, K), device="cuda").to(DTYPES[dtype])
    y = layer(x)
    for value in (0.0, 6e4, -777.0):
        x[:, window * m] = value
        assert torch.equal(layer(x)[:, keep], y[:, keep])


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("n,m", [(1, 1), (2, 4), (1, 8)])
@pytest.mark.parametrize("M", [2, 9, 20, 40, 1030])
def test_what_is_not_finite_shows_where_it_is_kept_and_in_its_row_alone(M, n, m, value, dtype):
    K, N = 256, 256
    made = make(M + m, K, N, n, m)
    layer = layer_of(made, K, n, m)
    x = torch.randn((M, K), device="cuda").to(DTYPES[dtype])
    y = layer(x)
    at = 3 if n == m else made[3][0, 0]         # of the first window, kept by the first vector
    x[1, at] = value
    got = layer(x)
    keeps = np.ones(N, bool) if n == m else np.repeat((made[3][:n] == at).any(0), 32)
    assert keeps.any() and not bool(got[1, torch.from_numpy(keeps).cuda()].isfinite().any())
    assert torch.equal(got[0], y[0]) and torch.equal(got[2:], y[2:])
