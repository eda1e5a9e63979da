"""CPU-only checks of the 4-bit entry points: buffer sizes and refusals, before anything touches a GPU."""
import ctypes

import pytest

from conftest import nmspmm

FAKE = ctypes.c_void_p(0x10000)


def operand(K=256, N=64, n=1, m=1, group=128, codes=0x10000, meta=0x10000, rows=0x10000, bias=None):
    return nmspmm.Q4Operand(codes, meta, rows, bias, K, N, n, m, group)


def test_buffer_sizes():
    # blocks of 128 kept rows x 16 columns, the columns filled up to 32
    assert nmspmm.q4_codes_bytes(4096, 4096) == 4096 * 4096 // 2
    assert nmspmm.q4_codes_bytes(1, 1) == 2 * 1024
    assert nmspmm.q4_codes_bytes(129, 33) == 4 * 2 * 1024
    assert nmspmm.q4_meta_bytes(4096, 4096, 1, 1, 128) == 4 * 32 * 4096
    assert nmspmm.q4_meta_bytes(4096, 4096, 2, 8, 32) == 4 * 32 * 4096
    assert nmspmm.q4_row_offsets_bytes(4096, 4096, 2, 8) == 1024 * 128
    assert nmspmm.q4_row_offsets_bytes(4096, 4096) == 0
    for bad in ((0, 64, 1, 1), (256, 0, 1, 1), (256, 64, 3, 8), (256, 64, 2, 32), (256, 64, 16, 32), (250, 64, 2, 4), (256, 48, 2, 4),
                (256, 64, 4, 2), (256, 64, 0, 4), (256, 64, -2, -4), ((1 << 22) + 1, 64, 1, 1), (64, (1 << 20) + 1, 1, 1)):
        assert nmspmm.q4_codes_bytes(*bad) == 0 and nmspmm.q4_meta_bytes(*bad) == 0 and nmspmm.q4_row_offsets_bytes(*bad) == 0
    for group in (0, 16, 48, 256, -32):
        assert nmspmm.q4_meta_bytes(256, 64, 1, 1, group) == 0


@pytest.mark.parametrize("op,status", [
    (dict(group=16), 3), (dict(n=3, m=8), 3), (dict(n=2, m=64), 3), (dict(n=0, m=0), 3), (dict(K=0), 2), (dict(N=-1), 2),
    (dict(K=250, n=2, m=4), 2), (dict(N=48, n=2, m=4), 2), (dict(codes=None), 1), (dict(meta=None), 1), (dict(n=2, m=4, rows=None), 1),
    (dict(codes=0x10004), 8), (dict(meta=0x10008), 8), (dict(n=2, m=4, rows=0x10001), 8), (dict(bias=0x10002), 8)])
def test_every_entry_point_refuses_a_bad_operand(op, status):
    L, o = nmspmm.lib(), operand(**op)
    assert L.nmspmm_q4_linear(o, FAKE, 1 << 20, FAKE, 1 << 20, 1, 0, None, 0, None) == status
    assert L.nmspmm_q4_quantize_device(FAKE, FAKE, o, 0, None) == status
    assert L.nmspmm_q4_pack_device(FAKE, FAKE, None, FAKE, o, None) == status
    assert L.nmspmm_q4_expand_device(o, FAKE, None) == status


def test_refusals_of_the_other_arguments():
    L, dense, sparse = nmspmm.lib(), operand(), operand(n=2, m=4)
    assert L.nmspmm_q4_linear(None, FAKE, 256, FAKE, 64, 1, 0, None, 0, None) == 1
    assert L.nmspmm_q4_linear(dense, None, 256, FAKE, 64, 1, 0, None, 0, None) == 1
    assert L.nmspmm_q4_linear(dense, FAKE, 256, None, 64, 1, 0, None, 0, None) == 1
    assert L.nmspmm_q4_linear(dense, None, 256, None, 64, 0, 0, None, 0, None) == 0      # no rows: nothing to do
    assert L.nmspmm_q4_linear(dense, FAKE, 255, FAKE, 64, 1, 0, None, 0, None) == 2
    assert L.nmspmm_q4_linear(dense, FAKE, 256, FAKE, 63, 1, 0, None, 0, None) == 2
    assert L.nmspmm_q4_linear(dense, FAKE, 256, FAKE, 64, -1, 0, None, 0, None) == 2
    assert L.nmspmm_q4_linear(dense, FAKE, 256, FAKE, 64, 1, 3, None, 0, None) == 3
    assert L.nmspmm_q4_linear(dense, ctypes.c_void_p(0x10002), 256, FAKE, 64, 1, 0, None, 0, None) == 8
    assert L.nmspmm_q4_linear(dense, ctypes.c_void_p(0x10001), 256, FAKE, 64, 1, 1, None, 0, None) == 8
    many = nmspmm.q4_workspace_bytes(65, 256, 64, 1, 1, 0)
    assert many > 0
    for rows in (1, 8):     # decoding takes no workspace
        assert nmspmm.q4_workspace_bytes(rows, 256, 64, 1, 1, 0) == 0 and nmspmm.q4_workspace_bytes(rows, 256, 64, 2, 4, 1) == 0
    for bad in ((0, 256, 64, 1, 1, 0), (-1, 256, 64, 1, 1, 0), (65, 256, 64, 1, 1, 3), (65, 0, 64, 1, 1, 0), (65, 256, 64, 3, 8, 0)):
        assert nmspmm.q4_workspace_bytes(*bad) == 0
    assert L.nmspmm_q4_linear(dense, FAKE, 256, FAKE, 64, 65, 0, None, 0, None) == 6
    assert L.nmspmm_q4_linear(dense, FAKE, 256, FAKE, 64, 65, 0, FAKE, many - 1, None) == 6
    assert L.nmspmm_q4_linear(dense, FAKE, 256, FAKE, 64, 65, 0, ctypes.c_void_p(0x10008), many, None) == 8
    assert L.nmspmm_q4_quantize_device(None, None, dense, 0, None) == 1
    assert L.nmspmm_q4_quantize_device(FAKE, None, sparse, 0, None) == 1
    assert L.nmspmm_q4_quantize_device(FAKE, None, dense, 2, None) == 2
    assert L.nmspmm_q4_pack_device(FAKE, None, None, None, dense, None) == 1
    assert L.nmspmm_q4_pack_device(None, FAKE, None, None, dense, None) == 1
    assert L.nmspmm_q4_expand_device(dense, None, None) == 1


def test_binding_checks_what_the_pointers_hold():
    torch = pytest.importorskip("torch")
    small, enough = torch.zeros(16, dtype=torch.int32), torch.zeros(4096, dtype=torch.int32)
    with pytest.raises(ValueError):
        nmspmm.q4_operand(small, enough, None, 256, 64)
    with pytest.raises(ValueError):
        nmspmm.q4_operand(enough, small, None, 256, 64)
    op = nmspmm.q4_operand(enough, enough, None, 256, 64)
    with pytest.raises(ValueError):
        nmspmm.q4_linear(op, torch.zeros(255), torch.zeros(64), 1, nmspmm.F32)
    with pytest.raises(ValueError):
        nmspmm.q4_linear(op, torch.zeros(256), torch.zeros(63), 1, nmspmm.F32)
    with pytest.raises(ValueError):
        nmspmm.q4_expand_device(op, torch.zeros(16))


def test_kept_rows():
    assert [nmspmm.q4_kept_rows(*a) for a in ((300, 1, 1), (300, 7, 7), (300, 2, 4), (64, 1, 8))] == [300, 300, 150, 8]
