"""CPU-only checks of the block norm's entry points: refusals with the documented status, before anything touches a GPU."""
import ctypes

import pytest

from conftest import nmspmm

AT = 0x10000
FIELDS = ("rows gate_rows ld_residual ld_branch ld_sum ld_out residual branch sum out stats gate scale post_weight post_bias pre_weight "
          "pre_bias gate_type scale_type post_weight_type post_bias_type pre_weight_type pre_bias_type features type residual_type post "
          "pre factor eps weight_offset").split()
GOOD = dict(rows=8, gate_rows=4, ld_residual=64, ld_branch=64, ld_sum=64, ld_out=64, residual=AT, branch=AT, sum=AT, out=AT, stats=AT,
            gate=AT, scale=AT, post_weight=AT, post_bias=AT, pre_weight=AT, pre_bias=AT, features=64, post=1, pre=2, eps=1e-6)
GRADS = "ld_sum ld_out ld_residual ld_branch sum out residual branch gate scale post_weight post_bias pre_weight pre_bias".split()


def packed(**kw):
    v = dict.fromkeys(FIELDS, 0)
    v.update(GOOD)
    v.update(kw)
    return nmspmm.BLOCK_NORM.pack(*[float(v[k]) if k in ("factor", "eps", "weight_offset") else v[k] for k in FIELDS])


def grads(**kw):
    v = dict.fromkeys(GRADS, 64)
    v.update({k: AT for k in GRADS[4:]})
    v.update(kw)
    return nmspmm.BLOCK_NORM_GRADS.pack(*[v[k] for k in GRADS])


@pytest.mark.parametrize("change,status", [
    (dict(type=3), 3), (dict(type=-1), 3), (dict(residual_type=1), 3), (dict(type=1, residual_type=2), 3), (dict(post=3), 3), (dict(pre=-1), 3),
    (dict(rows=-1), 2), (dict(rows=1 << 31), 2), (dict(features=0), 2), (dict(features=16385), 2), (dict(eps=-1.0), 2), (dict(eps=float("nan")), 2),
    (dict(gate_rows=0), 2), (dict(gate_rows=3), 2), (dict(ld_residual=63), 2), (dict(ld_branch=63), 2), (dict(ld_sum=0), 2), (dict(ld_out=-64), 2),
    (dict(branch=0), 3), (dict(branch=0, gate=0, scale=0, post_weight=0, post_bias=0), 3), (dict(post=0), 3), (dict(pre=0), 3), (dict(out=0), 3),
    (dict(residual=0), 1), (dict(sum=0), 1), (dict(branch=0, gate=0, scale=0, post_weight=0, post_bias=0, post=0, out=0, pre=0, pre_weight=0, pre_bias=0), 1),
    (dict(residual=AT + 2), 8), (dict(sum=AT + 1), 8), (dict(type=1, residual_type=1, branch=AT + 1), 8), (dict(out=AT + 2), 8), (dict(stats=AT + 8), 8),
    (dict(gate_type=5), 3), (dict(pre_bias_type=-1), 3), (dict(scale=AT + 2), 8), (dict(scale=AT + 1, scale_type=1), 8)])
def test_both_passes_refuse(change, status):
    L = nmspmm.lib()
    assert L.nmspmm_block_norm_forward(packed(**change), None) == status
    assert L.nmspmm_block_norm_backward(packed(**change), grads(), AT, 1 << 40, None) == status


def test_refusals_of_the_backward_pass():
    L = nmspmm.lib()
    need = L.nmspmm_block_norm_workspace_bytes(8, 4, 64)
    assert need > 0 and need % (64 * 4 * 6) == 0
    assert L.nmspmm_block_norm_forward(None, None) == 1
    assert L.nmspmm_block_norm_backward(None, grads(), AT, need, None) == 1
    assert L.nmspmm_block_norm_backward(packed(), None, AT, need, None) == 1
    assert L.nmspmm_block_norm_backward(packed(stats=0), grads(), AT, need, None) == 1
    assert L.nmspmm_block_norm_backward(packed(), grads(), 0, need, None) == 6
    assert L.nmspmm_block_norm_backward(packed(), grads(), AT, need - 1, None) == 6
    assert L.nmspmm_block_norm_backward(packed(), grads(), AT + 8, need, None) == 8
    assert L.nmspmm_block_norm_backward(packed(rows=0, gate_rows=1), grads(), AT, need, None) == 2
    for k in ("ld_sum", "ld_out", "ld_residual", "ld_branch"):
        assert L.nmspmm_block_norm_backward(packed(), grads(**{k: 63}), AT, need, None) == 2
    for k in ("gate", "scale", "post_weight", "post_bias", "pre_weight", "pre_bias"):
        assert L.nmspmm_block_norm_backward(packed(**{k: 0}), grads(), AT, 1 << 40, None) == 3     # a gradient of nothing
        assert L.nmspmm_block_norm_backward(packed(), grads(**{k: AT + 2}), AT, need, None) == 8
    assert L.nmspmm_block_norm_forward(packed(rows=0, gate_rows=1, residual=0, branch=0, sum=0, gate=0, scale=0, post=0, post_weight=0, post_bias=0), None) == 0
    for bad in ((0, 1, 64), (8, 3, 64), (8, 0, 64), (8, 8, 0), (8, 8, 16385), (1 << 31, 1, 64)):
        assert L.nmspmm_block_norm_workspace_bytes(*bad) == 0


def test_the_packed_structs_have_the_headers_size(tmp_path):
    import os
    import subprocess
    from conftest import ROOT
    src = tmp_path / "s.c"
    src.write_text('#include "nmspmm.h"\n#include <stdio.h>\nint main(void) { printf("%zu %zu %zu %zu\\n", sizeof(nmspmm_block_norm), '
                   'sizeof(nmspmm_block_norm_grads), offsetof(nmspmm_block_norm, factor), offsetof(nmspmm_block_norm, gate_type)); return 0; }\n')
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "s")], check=True)
    size = [int(v) for v in subprocess.run([str(tmp_path / "s")], check=True, capture_output=True, text=True).stdout.split()]
    assert size[:2] == [nmspmm.BLOCK_NORM.size, nmspmm.BLOCK_NORM_GRADS.size]
    assert size[2:] == [6 * 8 + 11 * 8 + 11 * 4, 6 * 8 + 11 * 8]
