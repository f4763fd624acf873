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
