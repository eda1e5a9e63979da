"""fp32 activations of more rows than the few-row kernel takes: an fp32 product's accuracy."""
import numpy as np
import pytest

from test_gpu_q4 import layer_of, make
from test_gpu_q4_sums import exact_terms_bound

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M,K,N", [(20, 1024, 96), (40, 1000, 130), (70, 2048, 256), (150, 4096, 64), (600, 1024, 1024), (1100, 777, 130)])
def test_fp32_rows_are_as_exact_as_an_fp32_product(M, K, N, group):
    """Ordinary weights, some columns of x ten times the others: no further from the 64-bit result than an fp32 product is
    (fewer roundings: exact products, several of them to an addition)."""
    made = make(M + K, K, N, group=group)
    dense = made[4]
    layer = layer_of(made, K, group=group)
    rng = np.random.default_rng(K)
    x = torch.from_numpy((rng.normal(size=(M, K)) * np.where(rng.random(K) < 0.01, 10.0, 1.0)).astype(np.float32))
    want = x.double().numpy() @ dense
    plain = (x.cuda() @ torch.from_numpy(dense).float().cuda()).double().cpu().numpy()
    got = layer(x.cuda()).double().cpu().numpy()
    assert np.linalg.norm(got - want) <= np.linalg.norm(plain - want)


@pytest.mark.parametrize("M", [17, 64, 150, 1030])
@pytest.mark.parametrize("group", [32, 128])
def test_an_outlier_under_zero_weights_adds_nothing_in_fp32(M, group):
    """Rows of a dense operand whose codes are the zero point: what x holds there is multiplied by zero."""
    K, N = 700, 96
    made = make(M, K, N, group=group)
    codes, scale, z, rows, dense = made
    of = np.arange(K) // group
    for k in (3, 200, 699):
        codes[k] = z[of[k]]
        dense[k] = 0.0
    layer = layer_of(made, K, group=group)
    x = torch.randn((M, K), device="cuda")
    x[:, [3, 200, 699]] = 1e5
    xd = x.double().cpu().numpy()
    want, got = xd @ dense, layer(x).double().cpu().numpy()
    assert np.all(np.abs(got - want) <= exact_terms_bound(xd, dense, group, K))
    assert np.linalg.norm(got - want) <= 2.5e-6 * np.linalg.norm(want)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M,K,N", [(1001, 1, 1), (1030, 264, 257), (1025, 1016, 40), (1024, 130, 16)])
def test_many_rows_of_odd_sizes(M, K, N, group):
    """Rows that lie apart, an operand whose last block is not whole: each element within the bound, nothing else read."""
    made = make(M + N, K, N, group=group, zero=K % 2 == 0)
    layer = layer_of(made, K, group=group)
    wide = torch.full((M, K + 3), float("nan"), device="cuda")
    wide[:, 2:K + 2] = torch.randn((M, K), device="cuda")
    x = wide[:, 2:K + 2]
    xd = x.double().cpu().numpy()
    want, got = xd @ made[4], layer(x).double().cpu().numpy()
    assert np.all(np.abs(got - want) <= exact_terms_bound(xd, made[4], group, K))
    assert torch.equal(layer(x), layer(x.contiguous()))
