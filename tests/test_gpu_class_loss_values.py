"""The class-list losses where their numbers end: NaN, infinities, far logits, masks, loss scales, the most rows. Tolerances are derived beside their use; none
of them grows with the logits' size."""
import math

import pytest
import torch

from test_gpu_class_loss import BF, DEV, F16, F32, _ops, _rand, ce_case, check_map, teacher

pytestmark = pytest.mark.gpu

# one length or more for every form of topk_distill: 4, 8, 16 lanes a row; a wave; 2, 4, 8, 16 waves; as stored, half and whole; in passes
FORMS = [16, 30, 60, 90, 128, 203, 700, 1500, 3001, 5000, 9001, 20003, 40000, 70001, 140000]


def distinct(N, V, k, seed):
    return teacher(N, V, k, seed, empty=False, dup=False)


@pytest.mark.parametrize("dtype", [F32, BF, F16])
@pytest.mark.parametrize("V", FORMS)
def test_nan_reaches_loss_and_gradient(V, dtype):
    """NaN in a row that takes part is NaN in its loss and where the formula puts it in its gradient -- a row of nothing but NaN, NaN among -inf, a teacher of
    nothing but NaN --, and reaches nothing from a row without a filled slot or without a class left. The other rows keep their bits."""
    k = 5
    z = (2 * _rand(11, V, seed=300)).to(dtype)
    idx, val = distinct(11, V, k, 301)
    loss0, dz0 = _ops().topk_distill(z, idx, val, tau=2.0)
    check_map((loss0, dz0), z, idx, val, 2.0, None)
    z[0] = math.nan
    z[1] = -math.inf
    z[1, V // 2] = math.nan
    z[2, V - 1] = math.nan
    val[3] = math.nan
    val[4], val[4, 1] = -math.inf, math.nan
    val[5, k - 1] = math.nan
    z[6], idx[6] = math.nan, -1
    z[7], val[7] = math.nan, -math.inf
    z[8], val[8] = -math.inf, math.nan
    for in_place in (False, True):
        own = z.clone()
        loss, dz = _ops().topk_distill(own, idx, val, tau=2.0, out=own if in_place else None)
        assert loss[:6].isnan().all() and dz[:3].isnan().all()
        for r in (3, 4, 5):
            named = torch.zeros(V, dtype=torch.bool, device=DEV)
            named[idx[r].long()] = True
            assert dz[r][named].isnan().all() and torch.equal(dz[r][~named], dz0[r][~named])
        assert torch.all(loss[6:9] == 0) and torch.all(dz[6:9] == 0)
        assert torch.equal(loss[9:], loss0[9:]) and torch.equal(dz[9:], dz0[9:])
    only, _ = _ops().topk_distill(z, idx, val, tau=2.0, want_grad=False)
    assert torch.equal(only.nan_to_num(-7.0), loss.nan_to_num(-7.0))


def test_nan_is_the_same_for_the_fused_projection():
    """linear_distill's rules for NaN are topk_distill's on the logits themselves."""
    x, w, _ = ce_case(6, 200, 32, BF, seed=310)
    idx, val = distinct(6, 200, 5, 311)
    x[0] = math.nan
    val[1] = math.nan
    val[2], val[2, 3] = -math.inf, math.nan
    x[3], val[3] = math.nan, -math.inf
    x[4], idx[4] = math.nan, -1
    fused, _ = _ops().linear_distill_fwd(x, w, idx, val)
    logits, _ = _ops().topk_distill(x.float() @ w.float().T, idx, val)
    for loss in (fused, logits):
        assert loss[:3].isnan().all() and torch.all(loss[3:5] == 0) and loss[5].isfinite()
