"""Refusals of the class-list losses: every bad argument is an error on the host, before anything reaches the GPU."""
import ctypes as C
import math

import pytest
import torch

from cerberusdet_amd import _lib as L
from cerberusdet_amd import ops


def _desc(**kw):
    d = L.LinearLossDesc()
    base = dict(N=4, V=10, d=16, dtype=L.BF16, x_ld=16, w_ld=16, scale=1.0, tau=1.0, offset=None, label64=1)
    for k, v in {**base, **kw}.items():
        setattr(d, k, v)
    return d


P = 4096  # a 16-byte aligned address that no kernel ever sees


@pytest.mark.parametrize("kw", [dict(dtype=L.F32), dict(d=0), dict(d=12), dict(d=65544), dict(V=0), dict(N=-1), dict(x_ld=20), dict(w_ld=8), dict(x_ld=1 << 22), dict(tau=0.0),
                                dict(tau=-1.0), dict(tau=2.0), dict(tau=math.nan), dict(scale=math.inf), dict(scale=math.nan), dict(w_ld=-16)])
def test_linear_ce_refuses(kw):
    lib, d = L.load(), _desc(**kw)
    assert lib.cdet_linear_ce_fwd(C.byref(d), P, P, P, P, P, P, None) == -1001
    assert lib.cdet_linear_ce_bwd(C.byref(d), P, P, P, P, P, 1, P, 16, P, 16, P, None) == -1001
    assert b"cdet_linear_ce_bwd" in lib.cdet_last_error()


def test_linear_refuses_pointers():
    lib, d = L.load(), _desc()
    assert lib.cdet_linear_ce_fwd(None, P, P, P, P, P, P, None) == -1001
    for bad in ((None, P, P, P, P, P), (P + 2, P, P, P, P, P), (P, None, P, P, P, P), (P, P + 8, P, P, P, P), (P, P, None, P, P, P), (P, P, P, None, P, P),
                (P, P, P, P, None, P), (P, P, P, P, P, None), (P, P, P, P, P, P + 4)):
        assert lib.cdet_linear_ce_fwd(C.byref(d), *bad, None) == -1001
    for dx, dxl, dw, dwl, st in ((P + 2, 16, P, 16, 1), (P, 8, P, 16, 1), (P, 17, P, 24, 1), (P, 16, P + 4, 16, 1), (P, 16, P, 20, 0), (P, 16, P, 16, 2)):
        assert lib.cdet_linear_ce_bwd(C.byref(d), P, P, P, P, P, st, dx, dxl, dw, dwl, P, None) == -1001
    for k in (0, 513, -1):
        assert lib.cdet_linear_distill_fwd(C.byref(d), P, P, k, P, P, L.F32, P, P, P, None) == -1001
        assert lib.cdet_linear_distill_bwd(C.byref(d), P, P, k, P, P, P, 1, P, 16, P, 16, P, None) == -1001
    assert lib.cdet_linear_distill_fwd(C.byref(d), P, P, 4, P, P, L.U8, P, P, P, None) == -1001
    assert lib.cdet_linear_distill_fwd(C.byref(d), P, P, 4, None, P, L.F32, P, P, P, None) == -1001
    assert lib.cdet_linear_loss_ws_bytes(None, 1) > 0
    n = [lib.cdet_linear_loss_ws_bytes(C.byref(_desc(N=a, V=b, d=c)), 1) for a, b, c in ((1, 1, 8), (4096, 65536, 640), (8192, 131072, 1024))]
    assert n[0] < 1 << 21 and n[2] < 1 << 30  # the logits in 16 bits alone would be 2 GiB


def test_no_rows_launch_nothing():
    lib, d = L.load(), _desc(N=0)
    assert lib.cdet_linear_ce_fwd(C.byref(d), None, P, None, None, None, None, None) == 0
    assert lib.cdet_linear_ce_bwd(C.byref(d), None, P, None, None, None, 0, P, 16, None, 16, None, None) == 0
    assert lib.cdet_linear_distill_fwd(C.byref(d), None, P, 3, None, None, L.F32, None, None, None, None) == 0
    assert lib.cdet_topk_distill(C.byref(_tdesc(P=0)), None, None, None, None, None, None, None) == 0


def _tdesc(**kw):
    d = L.TopkDistillDesc()
    base = dict(P=4, G=1, V=10, k=3, dtype=L.F32, val_dtype=L.F32, grad_dtype=L.F32, ld=10, grad_ld=10, tau=1.0, grad_scale=1.0)
    for k, v in {**base, **kw}.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("kw", [dict(dtype=L.U8), dict(val_dtype=L.U8), dict(grad_dtype=L.BF16), dict(G=0), dict(V=0), dict(P=-1), dict(k=0), dict(k=513), dict(tau=0.0),
                                dict(tau=math.nan), dict(ld=-1), dict(grad_ld=9), dict(P=1 << 30, G=4)])
def test_topk_distill_refuses(kw):
    lib, d = L.load(), _tdesc(**kw)
    assert lib.cdet_topk_distill(C.byref(d), P, P, P, P, P, 2 * P, None) == -1001
    assert b"cdet_topk_distill" in lib.cdet_last_error()


def test_topk_distill_refuses_pointers():
    lib = L.load()
    for d, args in ((_tdesc(), (None, P, P, P, P, P)), (_tdesc(), (P, None, P, P, P, P)), (_tdesc(), (P, P, None, P, P, P)), (_tdesc(), (P, P, P, P, None, P)),
                    (_tdesc(), (P + 2, P, P, P, P, 2 * P)), (_tdesc(), (P, P, P, P, P, 2 * P + 1)), (_tdesc(grad_ld=12), (P, P, P, P, P, P)),
                    (_tdesc(dtype=L.BF16), (P, P, P, P, P, P))):
        assert lib.cdet_topk_distill(C.byref(d), *args, None) == -1001


def test_wrappers_refuse_cpu_tensors_and_shapes():
    x, w, lab = torch.zeros(4, 16, dtype=torch.bfloat16), torch.zeros(10, 16, dtype=torch.bfloat16), torch.zeros(4, dtype=torch.int64)
    idx, val = torch.zeros(4, 3, dtype=torch.int32), torch.zeros(4, 3)
    for call in (lambda: ops.linear_ce_fwd(x, w, lab), lambda: ops.linear_distill_fwd(x, w, idx, val), lambda: ops.topk_distill(torch.zeros(4, 10), idx, val)):
        with pytest.raises(ValueError, match="GPU"):
            call()
    for a, b in ((x.float(), w.float()), (x, w.half()), (x[:, :8], w), (x[0], w)):
        with pytest.raises(ValueError):
            ops.linear_ce_fwd(a, b, lab)
    with pytest.raises(ValueError):
        ops.topk_distill(torch.zeros(10), idx, val)
    from cerberusdet_amd.utils import loss as UL

    with pytest.raises(ValueError):
        UL._reduced(torch.zeros(3), torch.ones(3, dtype=torch.bool), "average")
