"""Refusals of the many-class head and the 8-bit checkpoint operators that need no GPU."""
import ctypes

import pytest
import torch

import maxstyle_amd
from maxstyle_amd import ops
from maxstyle_amd._lib import lib


def test_cpu_tensors_are_refused():
    h, w, b, lab = torch.randn(1, 8, 4, 4), torch.randn(5, 8), torch.zeros(5), torch.zeros(1, 4, 4, dtype=torch.int64)
    for f in (ops.class_ce, ops.class_ce_fwd, maxstyle_amd.class_cross_entropy):
        with pytest.raises(RuntimeError, match="MI355X only"):
            f(h, w, b, lab)
    with pytest.raises(RuntimeError, match="MI355X only"):
        ops.act8_pack(h)
    with pytest.raises(RuntimeError, match="MI355X only"):
        ops.act8_unpack(h.to(torch.int8), torch.zeros(1, 8, 1))
    with pytest.raises(RuntimeError, match="MI355X only"):
        ops.act8_bn_act_bwd(h, h.to(torch.int8), torch.zeros(1, 8, 1), torch.zeros(8, 4), 0.2)
    with pytest.raises(ValueError, match="reduction"):
        maxstyle_amd.class_cross_entropy(h, w, b, lab, reduction="median")


def test_c_entries_refuse_before_any_launch():
    buf = ctypes.create_string_buffer(4096)
    p = ctypes.addressof(buf)
    assert lib.ms_class_ce_ws_bytes(0, 8, 5, 4, 0, 1) == 0 and lib.ms_class_ce_ws_bytes(1, 9000, 5, 4, 0, 1) == 0
    assert lib.ms_class_ce_ws_bytes(1, 8, (1 << 20) + 1, 4, 0, 1) == 0 and lib.ms_class_ce_ws_bytes(1, 8, 5, 4, 4, 1) == 0
    need = lib.ms_class_ce_ws_bytes(1, 8, 5, 4, 0, 1)
    assert need > 4096
    assert lib.ms_class_ce(p, p, p, p, p, p, p, p, 1, 8, 5, 4, 0, 1.0, 0, 0, p, 4096, 0) == -3          # workspace too small
    assert lib.ms_class_ce(p, p, p, p, 0, p, p, p, 1, 8, 5, 4, 0, 1.0, 0, 0, p, 1 << 40, 0) == -1       # no loss
    assert lib.ms_class_ce(0, p, p, p, p, p, p, p, 1, 8, 5, 4, 0, 1.0, 0, 0, p, 1 << 40, 0) == -1
    assert lib.ms_class_ce_fwd(p, p, p, p, 0, p, 1, 8, 5, 4, 0, p, 1 << 40, 0) == -1
    assert lib.ms_class_ce_bwd(p, p, p, p, 0, p, p, p, p, 1, 8, 5, 4, 0, p, 1 << 40, 0) == -1
    assert lib.ms_class_ce_bwd(p, p, p, p, p, p, 0, 0, 0, 1, 8, 5, 4, 0, p, 1 << 40, 0) == -1
    assert lib.ms_act8_pack(p, 0, p, p, 0, 1, 1, 0) == -1 and lib.ms_act8_pack(0, 0, p, p, 1, 1, 1, 0) == -1
    assert lib.ms_act8_pack(p, 0, p, p, 1 << 15, 1 << 15, 4096, 0) == -1
    assert lib.ms_act8_unpack(p, 0, 0, p, 1, 1, 1, 0) == -1
    assert lib.ms_act8_bwd_reduce(p, 0, p, p, 0, p, 0, p, 1, 1, 1, 0.2, 0) == -1
    assert lib.ms_act8_bn_act_bwd(p, 0, p, p, p, p, p, p, 1, 8, 4096, 0.2, p, 1, 0) == -3
    assert lib.ms_act8_bn_act_bwd(p, 0, p, p, p, 0, p, p, 1, 8, 64, 0.2, p, 4096, 0) == -1
    off = p + 8 - p % 16 if p % 16 <= 8 else p + 4            # a record that is not 16-byte aligned
    assert off % 16 and lib.ms_act8_pack(p, off, p, p, 1, 1, 1, 0) == -2 and lib.ms_act8_unpack(p, p, off, p, 1, 1, 1, 0) == -2
    assert lib.ms_act8_block() == ops.ACT8_BLOCK


def test_sizes_that_no_launch_holds_are_refused():
    buf = ctypes.create_string_buffer(4096)
    p = ctypes.addressof(buf) + 15 & ~15
    assert lib.ms_act8_pack(p, 0, p, p, 1 << 13, 1 << 13, 4, 0) == -1 and lib.ms_act8_unpack(p, p, 0, p, 1 << 13, 1 << 13, 4, 0) == -1
    assert lib.ms_act8_bwd_reduce(p, 0, p, p, p, p, 0, p, 1 << 13, 1 << 11, 4, 0.2, 0) == -1
    assert lib.ms_act8_bn_act_bwd(p, 0, p, p, p, p, p, p, 1 << 13, 1 << 11, 4, 0.2, p, 1 << 40, 0) == -1
    with pytest.raises(ValueError, match="2\\^31"):
        ops._act8_dims((1, 1, 1 << 16, 1 << 16), "act8_pack")
    assert lib.ms_class_ce_ws_bytes(1 << 15, 8, 5, (1 << 15) + 1, 0, 1) == 0


def test_logit_ce_refuses_before_any_launch():
    buf = ctypes.create_string_buffer(1 << 15)
    p = (ctypes.addressof(buf) + 15) & ~15
    n = lib.ms_logit_ce_ws_bytes()
    assert lib.ms_logit_ce(p, p, p, 0, 5, 4, 1.0, p, n, 0) == -1 and lib.ms_logit_ce(p, p, p, 1 << 15, 5, (1 << 15) + 1, 1.0, p, n, 0) == -1
    assert lib.ms_logit_ce(0, p, p, 1, 5, 4, 1.0, p, n, 0) == -1 and lib.ms_logit_ce(p, p, 0, 1, 5, 4, 1.0, p, n, 0) == -1
    assert lib.ms_logit_ce(p, p, p, 1, 5, 4, 1.0, p, n - 1, 0) == -3 and lib.ms_logit_ce(p, p, p, 1, 5, 4, 1.0, p + 4, n, 0) == -2
    with pytest.raises(RuntimeError, match="MI355X only"):
        ops.logit_ce(torch.randn(1, 5, 4, 4), torch.zeros(1, 4, 4, dtype=torch.int64))
