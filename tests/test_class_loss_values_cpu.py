"""Refusals and sizes of the class-list losses at the ends of their ranges."""
import ctypes as C

import pytest
import torch

from cerberusdet_amd import _lib as L
from cerberusdet_amd import ops
from test_class_loss_cpu import P, _desc, _tdesc


@pytest.mark.parametrize("tau,scale", [(1e-19, 1e-19), (1e-40, 0.0), (1e19, 1.0), (1e30, 1.0), (1.0, 2e38), (1.0, -3e38), (1e-3, 1e36), (1e-18, 1e21)])
def test_what_leaves_fp32_with_tau_or_scale_is_refused(tau, scale):
    """log2(e) / tau, scale log2(e) / tau and tau^2 beyond fp32 gave NaN or inf for every row."""
    lib, d = L.load(), _desc(tau=tau, scale=scale)
    assert lib.cdet_linear_distill_fwd(C.byref(d), P, P, 4, P, P, L.F32, P, P, P, None) == -1001
    assert lib.cdet_linear_distill_bwd(C.byref(d), P, P, 4, P, P, P, 1, P, 16, P, 16, P, None) == -1001
    assert b"tau" in lib.cdet_last_error()
    if tau == 1.0:
        assert lib.cdet_linear_ce_fwd(C.byref(d), P, P, P, P, P, P, None) == -1001
        assert lib.cdet_linear_ce_bwd(C.byref(d), P, P, P, P, P, 1, P, 16, P, 16, P, None) == -1001
    elif scale in (0.0, 1.0):
        assert lib.cdet_topk_distill(C.byref(_tdesc(tau=tau)), P, P, P, P, P, 2 * P, None) == -1001
        with pytest.raises(ValueError, match="GPU|tau"):
            ops.topk_distill(torch.zeros(4, 10), torch.zeros(4, 3, dtype=torch.int32), torch.zeros(4, 3), tau=tau)


@pytest.mark.parametrize("N", [200, 8192, 49152, 49153, 268800, 1 << 20, 1 << 24])
def test_workspace_of_many_rows(N):
    """dz of a piece: 192 MiB, or 4 KiB a row where 2048 classes take more; beside it (d = 8) less than 64 bytes a row and 8 MiB."""
    lib = L.load()
    for V in (300, 2048, 4500, 131072, 1 << 24):
        size = lib.cdet_linear_loss_ws_bytes(C.byref(_desc(N=N, V=V, d=8, x_ld=8, w_ld=8)), 1)
        rows = (N + 31) // 32 * 32
        assert 0 < size <= min(max(192 << 20, 4096 * rows), rows * 2 * ((V + 255) // 256 * 256)) + 64 * N + (8 << 20)


def test_gradients_over_their_inputs_are_refused():
    """topk_distill writes in place or beside the logits; a gradient that covers part of other pixels' logits is refused, as dx / dw in the place of x / w are."""
    lib, Z = L.load(), 1 << 20
    wide = dict(P=50, G=1, V=10, ld=64, grad_ld=64)
    over = [(_tdesc(**wide), Z + 4 * o) for o in (1, 9, -9, 55, 64, 64 * 49 + 9, 63, -64, -64 * 49)]
    over += [(_tdesc(**{**wide, "grad_ld": 65}), Z + 4 * 20), (_tdesc(P=1, V=100, ld=100, grad_ld=100), Z + 4 * 99), (_tdesc(P=1, V=100, ld=100, grad_ld=100), Z - 4 * 99),
             (_tdesc(**{**wide, "dtype": L.BF16, "grad_dtype": L.F32, "ld": 128, "grad_ld": 64}), Z + 2 * 8),
             (_tdesc(**{**wide, "dtype": L.BF16, "grad_dtype": L.F32, "ld": 128, "grad_ld": 64}), Z + 2 * 110), (_tdesc(P=50, V=10, ld=0, grad_ld=10), Z - 4 * 3)]
    for d, g in over:
        assert lib.cdet_topk_distill(C.byref(d), Z, P, P, P, P, g, None) == -1001, (d.ld, d.grad_ld, g - Z)
        assert b"overlaps" in lib.cdet_last_error()
    d = _desc()
    assert lib.cdet_linear_ce_bwd(C.byref(d), Z, P, P, P, P, 1, Z, 16, 2 * Z, 16, P, None) == -1001
    assert lib.cdet_linear_ce_bwd(C.byref(d), Z, P, P, P, P, 1, 2 * Z, 16, P, 16, P, None) == -1001
    assert lib.cdet_linear_distill_bwd(C.byref(d), Z, P, 3, P, P, P, 1, Z, 16, 2 * Z, 16, P, None) == -1001
