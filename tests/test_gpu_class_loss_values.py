"""The class-list losses where their numbers end: NaN, infinities, far logits, masks, loss scales, the most rows. Tolerances are derived beside their use; none
of them grows with the logits' size."""
import math

import pytest
import torch

from test_gpu_class_loss import BF, DEV, F16, F32, U, _ops, _rand, _randint, ce_case, check_grads, check_map, check_rows, loss_tol, map_reference, reference, run_ce, teacher

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


def check_far(got, z, idx, val, tau):
    """An exponent e = (z - max) log2(e) / tau takes four roundings of its own size, exp2 and log2 one or two; a sum of V terms adds up at most 48 + V / 1024 of
    them in a chain. Terms that count (p > 2^-150) have |e| < 150, and sum p |e| ln 2 <= ln V + 1: u (4 (ln V + 1) + V / 1024 + 64) of the sum, 700 u of one p."""
    loss, dz = got
    V, k = z.shape[-1], idx.shape[-1]
    wl, wd, mag = map_reference(z, idx, val, tau, None)
    logp = torch.log_softmax(z.double() / tau, -1).gather(-1, idx.long().clamp(0, V - 1))
    logp = torch.where(torch.isfinite(logp), logp, 0.0).abs().amax(-1)
    rel = U * (4 * (math.log(V) + 1) + V / 1024 + 64)
    # log p: four roundings of itself and the sum's; log q: the same of the teacher's logits, below 32; k products added up
    check_rows(loss, wl, tau * tau * 2 * (rel + U * (8 * logp + 8 * 32 + k + 32)))
    h = 0.0 if dz.dtype == F32 else torch.finfo(dz.dtype).eps / 2
    # exp2's results end at 2^-126 (below that the hardware gives 0): p is off by no more than that; and half a smallest step of the gradient's type
    tol = 1.01 * (h * wd.abs() + (rel + 700 * U) * mag + tau * 2.0 ** -126) + 2 * torch.finfo(dz.dtype).tiny * torch.finfo(dz.dtype).eps
    err = (dz.double() - wd).abs()
    assert torch.all(err <= tol), (err / tol).max().item()


FAR = [(F32, 1.0e5), (F32, -1.0e30), (F32, -3.3e38), (BF, 1.0e3), (BF, -1.0e5), (BF, -1.0e9), (BF, 1.0e30), (BF, -3.3e38), (F16, 1.0e3), (F16, -6.0e4)]


@pytest.mark.parametrize("dtype,base", FAR)
@pytest.mark.parametrize("V", FORMS)
def test_far_logits_cost_nothing(V, dtype, base):
    """Rows around one far value: loss and gradient are as exact as near 0, for neighbours of the type (tau of their distance) and for ties (tau = 1)."""
    k = 6
    step = 2.0 ** (math.floor(math.log2(abs(base))) - {F32: 23, BF: 7, F16: 10}[dtype])
    near = torch.tensor(base, dtype=dtype, device=DEV).double() + step * _randint(6, (7, V), 320)
    z = near.to(dtype)
    idx, val = distinct(7, V, k, 321)
    idx[1] = z[1].float().argmax().int()  # all slots on the largest
    z[2] = z[2, 0]
    z[3, 1::3] = -math.inf
    idx[3] = idx[3] // 3 * 3
    idx[4, 2:] = -1
    for tau in (1.0, step) if 2.0 ** -20 < step < 1e12 else (1.0,):
        v = val * tau  # (the teacher's distribution stays)
        check_far(_ops().topk_distill(z, idx, v, tau=tau), z, idx, v, tau)
        check_far(_ops().topk_distill(z, idx, v, tau=tau, grad_dtype=F32), z, idx, v, tau)


@pytest.mark.parametrize("dtype", [F32, BF, F16])
@pytest.mark.parametrize("V", FORMS)
def test_masks_of_the_lowest_value(V, dtype):
    """Classes masked with the type's lowest number: no probability beside others, all of it where nothing else is left; a teacher that names one has the loss
    that the formula gives, which is finite."""
    low = torch.finfo(dtype).min
    z = (2 * _rand(6, V, seed=330)).to(dtype)
    idx, val = distinct(6, V, 4, 331)
    z[0, ::2] = low
    idx[0] = idx[0] | 1
    z[1] = low
    z[2] = low
    z[2, 1::2] = -math.inf
    idx[2] = idx[2] // 2 * 2
    z[3, idx[3, 0].long()] = low
    val[3, 0] -= 12.0  # (tau^2 q 3.4e38 / tau stays in range)
    z[4] = torch.finfo(dtype).max
    for tau in (1.0, 2.0):
        got = _ops().topk_distill(z, idx, val, tau=tau)
        assert got[0].isfinite().all() and got[1].isfinite().all()
        check_far(got, z, idx, val, tau)


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("V", [60, 1500, 9001, 70001, 140000])
def test_gradient_of_16_bit_logits_under_a_loss_scale(V, dtype):
    """The gradient through autograd is rounded to the logits' type once, behind the incoming gradient: what a loss scale lifts into fp16's range is there."""
    from cerberusdet_amd.utils import loss as UL

    z = _rand(5, V, seed=340).to(dtype)
    idx, val = distinct(5, V, 7, 341)
    weight = torch.tensor([1.0, 0.5, -2.0, 0.0, 1.37], device=DEV) * 2.0 ** 13
    leaf = z.clone().requires_grad_()
    (UL.topk_distillation(leaf, idx, val, tau=2.0, reduction="none") * weight).sum().backward()
    wl, wd, mag = map_reference(z, idx, val, 2.0, weight)
    rel = U * (4 * (math.log(V) + 1) + V / 1024 + 64 + 64)  # check_far's; logits within 6 / tau of the maximum's 6: 4 roundings of an exponent below 9
    h = 0.0 if dtype == F32 else torch.finfo(dtype).eps / 2
    tol = 1.01 * (h * wd.abs() + rel * mag) + torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    err = (leaf.grad.double() - wd).abs()
    assert leaf.grad.dtype == dtype and torch.all(err <= tol), (err / tol).max().item()


@pytest.mark.parametrize("dtype,P,taped", [(BF, 1000, True), (F16, 1000, False), (F32, 1000, True), (F32, 300, False)])
def test_forward_holds_no_gradient_map(dtype, P, taped):
    """Long or 16-bit maps are read again by the backward, and a loss without one makes no gradient: neither keeps a map of the logits' size."""
    from cerberusdet_amd.utils import loss as UL

    z = _rand(P, 40000, seed=350, dtype=dtype).requires_grad_()
    idx, val = distinct(P, 40000, 4, 351)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    with torch.set_grad_enabled(taped):
        loss = UL.topk_distillation(z, idx, val)
    assert torch.cuda.max_memory_allocated() - before < z.numel()
    if not taped:
        return
    with torch.no_grad():
        z.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace"):  # (what the backward reads may not change: refused)
        loss.backward()


def test_topk_distillation_twice_through_one_graph():
    from cerberusdet_amd.utils import loss as UL

    z = _rand(50, 300, seed=360).requires_grad_()
    idx, val = teacher(50, 300, 6, 361)
    loss = UL.topk_distillation(z, idx, val, tau=1.5)
    a, = torch.autograd.grad(loss, z, retain_graph=True)
    b, = torch.autograd.grad(3 * loss, z)
    assert torch.allclose(3 * a, b, rtol=4 * 2.0 ** -23, atol=0)


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("N,V", [(1, 300), (70, 4000), (70, 20000), (2600, 3900), (300, 60000)])
def test_an_infinite_logit_beside_far_ones(N, V, dtype):
    """One class's logit overflows to +inf, another one far down the list is 300: the log-sum-exp is +inf (not NaN), and so is the loss of every other class."""
    d = 16
    x, w = torch.zeros(N, d, dtype=dtype, device=DEV), torch.zeros(V, d, dtype=dtype, device=DEV)
    x[:, 0] = 2.0
    off = 0.1 * _rand(V, seed=370)
    for a, b in ((1, V - 1), (V - 1, 1), (V // 2, 3)):
        w[:, 0] = 0
        w[a, 0] = 3.0
        o = off.clone()
        o[b] = 300.0
        labels = torch.full((N,), b, device=DEV)
        loss, lse = _ops().linear_ce_fwd(x, w, labels, offset=o, scale=1e38)
        assert torch.all(lse == math.inf) and torch.all(loss == math.inf)
        idx = torch.full((N, 2), b, dtype=torch.int32, device=DEV)
        idx[:, 1] = 7
        loss, saved = _ops().linear_distill_fwd(x, w, idx, torch.zeros(N, 2, device=DEV), offset=o, scale=1e38)
        assert torch.all(loss == math.inf)
        none = torch.full_like(idx, -1)
        loss, saved = _ops().linear_distill_fwd(x, w, none, torch.zeros(N, 2, device=DEV), offset=o, scale=1e38)
        assert torch.all(loss == 0) and torch.all(saved[:, 0] == math.inf)
    w[V // 2 + 5, 1] = math.nan  # NaN beside an infinite one stays NaN
    x[:, 1] = 1.0
    loss, lse = _ops().linear_ce_fwd(x, w, torch.full((N,), 1, device=DEV), offset=off, scale=1e38)
    assert lse.isnan().all() and loss.isnan().all()


def test_means_over_the_rows_that_take_part():
    """reduction="mean" divides by the rows that the kernels count: not by those whose filled slots hold nothing but -inf, or that have no class left."""
    from cerberusdet_amd.utils import loss as UL

    x, w, labels = ce_case(20, 50, 16, BF, seed=380)
    idx, val = distinct(20, 50, 4, 381)
    val[3] = -math.inf
    val[5, 1:] = -math.inf
    idx[7] = -1
    idx[9, :2] = -2
    val[9, 2:] = -math.inf
    part = torch.ones(20, dtype=torch.bool, device=DEV)
    part[[3, 7, 9]] = False
    xl = x.clone().requires_grad_()
    mean = UL.linear_distillation(xl, w, idx, val, tau=2.0)
    rows = UL.linear_distillation(x, w, idx, val, tau=2.0, reduction="none")
    assert torch.allclose(mean, rows[part].sum() / 17, rtol=1e-6) and torch.all(rows[~part] == 0)
    mean.backward()
    m = torch.full((1,), 1 / 17, device=DEV)
    check_grads(xl.grad, None, reference(x, w, idx=idx, val=val, tau=2.0, drow=m), x, tau=2.0)
    for z in (2 * _rand(20, 50, seed=382), 2 * _rand(20, 1000, seed=383), 2 * _rand(20, 3000, seed=384), 2 * _rand(20, 40000, seed=385), 2 * _rand(20, 80000, seed=386)):
        z[11] = -math.inf
        here = part.clone()
        here[11] = False
        val2 = val.clone()
        val2[12] = math.nan  # NaN takes part
        for v, n in ((val, 16), (val2, 16)):
            leaf = z.clone().requires_grad_()
            mean = UL.topk_distillation(leaf, idx, v, tau=2.0)
            rows = UL.topk_distillation(z, idx, v, tau=2.0, reduction="none")
            assert torch.all(rows[~here] == 0)
            if v is val:
                assert torch.allclose(mean, rows[here].sum() / n, rtol=1e-6)
                mean.backward()
                assert torch.allclose(leaf.grad * n, _ops().topk_distill(z, idx, v, tau=2.0)[1], rtol=1e-5, atol=1e-7)
            else:
                assert mean.isnan()
    two = 2 * _rand(6, 4, 16, seed=387)
    idx, val = teacher(24, 16, 3, 388)
    two[2, 1] = -math.inf
    idx, val = idx.view(6, 4, 3), val.view(6, 4, 3)
    val[4, 2] = -math.inf
    live = (((idx >= 0) & (idx < 16)) & (val > -math.inf)).any(-1)
    live[2, 1] = False
    rows = UL.topk_distillation(two, idx, val, reduction="none")
    assert torch.allclose(UL.topk_distillation(two, idx, val), rows.sum() / live.sum(), rtol=1e-6)
    none = UL.linear_cross_entropy(x, w, labels, offset=torch.full((50,), -math.inf, device=DEV))
    assert none == 0


@pytest.mark.parametrize("V", FORMS)
def test_rows_that_take_part_are_told(V):
    z = 2 * _rand(9, V, seed=395)
    idx, val = distinct(9, V, 3, 396)
    z[1] = -math.inf
    z[2] = math.nan
    idx[3] = -1
    val[4] = -math.inf
    val[5, 0] = math.nan
    part = torch.zeros(10, dtype=torch.bool, device=DEV)
    loss, _ = _ops().topk_distill(z, idx, val, part=part[:9], want_grad=False)
    assert part.tolist() == [True, False, True, False, False, True, True, True, True, False]
    for bad in (part, part[:9].int(), torch.zeros(18, dtype=torch.bool, device=DEV)[::2], torch.zeros(9, dtype=torch.bool)):
        with pytest.raises(ValueError):
            _ops().topk_distill(z, idx, val, part=bad)


@pytest.mark.parametrize("N", [9000, 300000])
def test_captured_means_of_many_rows(N):
    """The means of as many rows as a library's sum takes several workgroups for, captured and replayed on new numbers with eager work in between."""
    from cerberusdet_amd.utils import loss as UL

    V, k = 40, 3
    z, w, x = 2 * _rand(N, V, seed=400), _rand(V, 16, seed=401, dtype=BF), _rand(N, 16, seed=402, dtype=BF)
    idx, val = teacher(N, V, k, 403)
    labels = _randint(V, (N,), 404)

    def step(x, w, z, labels, idx, val):
        x, w, z = (t.detach().requires_grad_() for t in (x, w, z))
        total = UL.linear_cross_entropy(x, w, labels) + UL.linear_distillation(x, w, idx, val) + UL.topk_distillation(z, idx, val, tau=2.0)
        total = total + UL.topk_distillation(z, idx, val, reduction="sum") / N
        return [total.detach(), *torch.autograd.grad(total, (x, w, z))]

    data = (x, w, z, labels, idx, val)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*data)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(*data)
    for turn in range(6):
        x.copy_(_rand(N, 16, seed=410 + turn, dtype=BF))
        z.copy_(_rand(N, V, seed=420 + turn))
        labels.copy_(_randint(V + 9, (N,), 430 + turn) - 4)
        graph.replay()
        got = [o.clone() for o in outs]
        want = step(*data)
        _rand(N, 8, seed=440 + turn).sum()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b), turn


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("N,V,d", [(5, 70, 16), (100, 700, 64), (140, 2000, 64), (2600, 3900, 40)])
def test_offsets_of_the_lowest_value_leave_out(N, V, d, dtype):
    """A class masked with fp32's lowest number is left out like one of -inf, in every form: the same bits, whatever its weights hold."""
    ops = _ops()
    x, w, labels = ce_case(N, V, d, dtype, seed=390)
    idx, val = distinct(N, V, 6, 391)
    out = torch.zeros(V, dtype=torch.bool, device=DEV)
    out[::9] = True
    labels[1:] = torch.where(out[labels[1:]], -100, labels[1:])
    labels[0] = 9  # a left-out class beside others: loss +inf, the gradient reaches the others only
    idx[2:] = torch.where(out[idx[2:].long()], -1, idx[2:])
    idx[1, 0] = 18
    wb = w.clone()
    wb[out] = math.nan
    base = 0.1 * _rand(V, seed=392)
    got = []
    for low in (-math.inf, torch.finfo(F32).min, -3e38):
        off = torch.where(out, low, base)
        got.append(list(run_ce(x, wb, labels, offset=off)))
        for tau in (4.0, 0.5):
            kd, saved = ops.linear_distill_fwd(x, wb, idx, val, tau=tau, offset=off)
            got[-1] += [kd, *ops.linear_distill_bwd(x, wb, idx, saved, tau=tau, offset=off)]
    assert got[0][0][0] == math.inf and got[0][4][1] == math.inf and got[0][2].isfinite().all() and torch.all(got[0][3][out] == 0)
    for other in got[1:]:
        for a, b in zip(got[0], other):
            assert torch.equal(a, b)
    loss, lse, dx, dw = run_ce(x, w, labels, offset=torch.full((V,), torch.finfo(F32).min, device=DEV))
    assert torch.all(loss == 0) and torch.all(dx == 0) and torch.all(dw == 0)


# more rows than one launch of each form takes, and than a grid holds threads for
@pytest.mark.parametrize("P,V,dtype", [((1 << 28) + 3, 60, F32), ((1 << 26) + 1, 130, BF), ((1 << 22) + 1, 16400, BF), ((1 << 21) + 7, 70001, BF)])
def test_topk_distill_of_the_most_rows(P, V, dtype):
    """Rows that repeat one pattern (the logits by stride 0): every row's loss is its first occurrence's, to the bit."""
    z = (2 * _rand(1, V, seed=450)).to(dtype)
    idx = torch.arange(P, dtype=torch.int32, device=DEV).remainder_(4)[:, None]
    val = torch.zeros(P, 1, device=DEV)
    loss, _ = _ops().topk_distill(z.expand(P, V), idx, val, want_grad=False)
    wl = -torch.log_softmax(z[0].double(), 0)[:4]
    assert torch.all((loss[:4].double() - wl).abs() <= 2 * U * (4 * (math.log(V) + 1) + V / 1024 + 64 + 8 * wl))
    whole = P // 4 * 4
    assert torch.all(loss[:whole].view(-1, 4) == loss[:4]) and torch.equal(loss[whole:], loss[:P - whole])


def test_linear_distill_of_the_most_rows():
    """2^24 rows (one x by stride 0) of 17 slots: every row the same loss and dx; dw their sum."""
    ops = _ops()
    N, V, d, k = 1 << 24, 16, 8, 17
    x, w, _ = ce_case(1, V, d, BF, seed=460)
    idx, val = teacher(1, V, k, 461, empty=False)
    loss, saved = ops.linear_distill_fwd(x.expand(N, d), w, idx.expand(N, k), val.expand(N, k))
    assert torch.all(loss == loss[0]) and torch.all(saved[:, 0] == saved[0, 0])
    ref = reference(x, w, idx=idx, val=val)
    check_rows(loss[:1], ref["loss"], 2 * loss_tol(ref, d) + 64 * U * 16)
    dx, dw = ops.linear_distill_bwd(x.expand(N, d), w, idx.expand(N, k), saved, torch.full((1,), 2.0 ** -24, device=DEV))
    assert torch.all(dx == dx[0])
    one = torch.full((1,), 2.0 ** -24, device=DEV)
    check_grads(dx[:1], None, reference(x, w, idx=idx, val=val, drow=one), x)
    # 2^24 equal terms: at most 2^24 u = 1 of the sum in a chain, but the tiles' chains are shorter than 2^24 / 64 = 2^18: 2^-6, and dz's and dw's roundings
    want = reference(x, w, idx=idx, val=val)["dw"]
    mag = reference(x, w, idx=idx, val=val)["dz"].abs().T @ x.double().abs()
    assert torch.all((dw.double() - want).abs() <= mag * (2.0 ** -6 + 2.0 ** -7) + 2.0 ** -8 * want.abs())


@pytest.mark.parametrize("dtype,gdt", [(F32, F32), (BF, BF), (BF, F32)])
@pytest.mark.parametrize("V", [16, 203, 3001])
def test_gradient_beside_the_logits_in_one_map(V, dtype, gdt):
    """Logits and gradient as slices of one buffer: back to back a pixel, and one behind the other; a gradient shifted over the logits is refused."""
    ops, P, k = _ops(), 40, 5
    z = (2 * _rand(P, V, seed=470)).to(dtype)
    idx, val = distinct(P, V, k, 471)
    loss, dz = ops.topk_distill(z, idx, val, grad_dtype=gdt)
    wide = dtype.itemsize * ((V + 3) // 4 * 4)
    pitch = wide + gdt.itemsize * (V + 8)
    pitch += -pitch % 16
    raw = torch.zeros(P, pitch, dtype=torch.uint8, device=DEV)
    zs, gs = raw.view(dtype)[:, :V], raw[:, wide:].view(gdt)[:, 2:2 + V] if dtype == gdt else raw[:, wide + (-wide % 4):].view(gdt)[:, 2:2 + V]
    zs.copy_(z)
    got, out = ops.topk_distill(zs, idx, val, out=gs)
    assert torch.equal(got, loss) and torch.equal(gs, dz) and torch.equal(zs, z)
    if dtype == gdt:
        with pytest.raises(RuntimeError, match="overlaps"):
            ops.topk_distill(zs, idx, val, out=raw.view(dtype)[:, 1:1 + V])
        assert torch.equal(zs, z)


@pytest.mark.parametrize("dtype,V", [(BF, 900), (F16, 9001), (F32, 70000)])
def test_backward_from_the_logits_captured_and_on_two_streams(dtype, V):
    """The gradient that the backward makes, captured and replayed on new logits with eager work in between; forward and backward of two streams at once."""
    from cerberusdet_amd.utils import loss as UL

    P, k = (40000 if V < 1000 else 600), 4
    z = (2 * _rand(P, V, seed=480)).to(dtype)
    assert dtype != F32 or z.numel() > UL._AHEAD
    idx, val = teacher(P, V, k, 481)

    def step(z):
        leaf = z.detach().requires_grad_()
        loss = UL.topk_distillation(leaf, idx, val, tau=2.0)
        return [loss.detach(), *torch.autograd.grad(64.0 * loss, leaf)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(z)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(z)
    for turn in range(4):
        z.copy_(2 * _rand(P, V, seed=482 + turn))
        graph.replay()
        got = [o.clone() for o in outs]
        want = step(z)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), turn
    zs = [z, z.flip(1).contiguous()]
    want = [step(t) for t in zs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        got = []
        for s, t in zip(streams, zs):
            with torch.cuda.stream(s):
                got.append(step(t))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(p, q) for p, q in zip(a, b))
