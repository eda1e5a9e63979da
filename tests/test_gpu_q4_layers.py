"""Ranges that end at the largest number, scales, codes that are none, layers that were cast, on the GPU."""
import copy

import numpy as np
import pytest

from conftest import nmspmm
from test_gpu_q4 import cuda, make, op, quantized

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("group", [32, 128])
def test_ranges_beyond_the_largest_number(group):
    """max - min is more than fp32 holds; the scale, a fifteenth of it, is not."""
    v = np.zeros((200, 5), np.float32)
    v[:, 0] = np.linspace(-3e38, 3e38, 200)
    v[:, 1] = np.where(np.arange(200) % 2, 3.4e38, -3.4e38)
    v[:, 2] = np.where(np.arange(200) % 3, np.finfo(np.float32).max, -np.finfo(np.float32).max)
    v[:, 3] = np.linspace(-3e38, 1e38, 200)
    v[:, 4] = np.linspace(0, 3.4e38, 200)
    for asymmetric in (False, True):
        got = op().NMQuantOperand.quantize(cuda(v), None, 200, group=group, asymmetric=asymmetric).dense().cpu().numpy()
        want = quantized(v, group, asymmetric)
        with np.errstate(over="ignore"):        # (a scale that covers the largest number may stand for more than it)
            assert np.array_equal(got, want.astype(np.float32))


def test_scales_are_kept_to_20_bits():
    """Nearest number of 20 significant bits; the largest numbers do not become infinite."""
    scale = np.array([[1.0, 1.0 + 2.0 ** -23, 1.0 + 3 * 2.0 ** -22, 0.1, -0.1, np.finfo(np.float32).max, 3.4e-39]], np.float32)
    codes = np.full((4, 7), 9, np.uint8)
    got = op().NMQuantOperand.from_codes(cuda(codes), cuda(scale), None, 4).dense().cpu().numpy()
    f, e = np.frexp(scale[0].astype(np.float64))
    want = np.ldexp(np.sign(f) * np.floor(np.ldexp(np.abs(f), 20) + 0.5), e - 20)
    assert np.array_equal(got[0, :5], want[:5].astype(np.float32))
    assert np.isfinite(got).all() and abs(got[0, 5] / scale[0, 5] - 1) <= 2.0 ** -19


def test_codes_and_zero_points_above_15_are_refused():
    codes, scale, zero, _, _ = make(3, 256, 64)
    for at in (0, 256 * 64 - 1):
        bad = codes.copy().reshape(-1)
        bad[at] = 16
        with pytest.raises(ValueError):
            op().NMQuantOperand.from_codes(cuda(bad.reshape(256, 64)), cuda(scale), cuda(zero), 256)
    for value in (16, -1, 256):
        bad = torch.from_numpy(zero.astype(np.int32)).cuda()
        bad[1, 3] = value
        with pytest.raises(ValueError):
            op().NMQuantLinear.from_codes(cuda(codes), cuda(scale), bad, 256)
    whole = torch.from_numpy(zero.astype(np.int64)).cuda()
    a, b = (op().NMQuantOperand.from_codes(cuda(codes), cuda(scale), z, 256).dense() for z in (whole, cuda(zero)))
    assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float64])
@pytest.mark.parametrize("n,m", [(1, 1), (2, 4)])
def test_a_cast_layer_still_shows_its_weight(dtype, n, m):
    w = torch.randn((64, 256), device="cuda")
    layer = op().NMQuantLinear(w, n, m, bias=torch.randn(64, device="cuda"))
    weight = layer.dense_weight()
    cast = copy.deepcopy(layer).to(dtype)
    assert cast.bias.dtype == dtype
    assert torch.equal(cast.dense_weight(), weight)
    # the struct names a float32 bias or none
    x, y = torch.randn((3, 256), device="cuda"), torch.empty((3, 64), device="cuda")
    operand = cast._operand()
    nmspmm.q4_linear(operand, x, y, 3, nmspmm.F32)
    assert torch.equal(y, cast(x))
    torch.testing.assert_close(y, x @ weight.t() + cast.bias.float(), rtol=1e-4, atol=1e-3)
