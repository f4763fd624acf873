"""Losses over a long class list (csrc/class_loss.hip, csrc/topk_distill.hip) against their definitions in 64 bits.

Tolerances, derived (u = 2^-24 a rounding to fp32, h = half a step of the 16-bit type, relative):
  * a logit is a sum of d exact fp32 products (16-bit x 16-bit) in fp32: off by at most d u sum|x w|; scaling, offset, the log2 domain and the sums of
    exponentials add a few roundings of quantities below |z| + |lse| + log2 e * 32: loss_tol() counts 16 of them. lse moves by at most what the logits do.
  * dz is rounded once to 16 bits: h |dz|, and p is off by the factor exp(2 loss_tol) (fp16: the smallest step, relative to the largest row gradient, too).
  * dx / dw: those errors times |w| / |x|, n u for the fp32 sum over n terms, and the rounding of the result."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _ops():
    from cerberusdet_amd import ops

    return ops


def _rand(*shape, seed=0, dtype=F32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


def _randint(hi, shape, seed):
    return torch.randint(hi, shape, generator=torch.Generator().manual_seed(seed)).to(DEV)


def teacher(N, V, k, seed, empty=True, dup=True):
    idx = _randint(V, (N, k), seed).int()
    if not dup:
        idx = torch.stack([torch.randperm(V, generator=torch.Generator().manual_seed(seed + r))[:k] for r in range(N)]).int().to(DEV)
    if empty:
        idx[::3, k // 2:] = -1
        idx[::5] = -1
        idx[1::7, 0] = V  # behind the list: empty as well
    return idx, 3 * _rand(N, k, seed=seed + 1)


def reference(x, w, labels=None, idx=None, val=None, tau=1.0, offset=None, scale=1.0, drow=None):
    """Loss rows, dz, dx, dw in 64 bits, and the sums the tolerances need."""
    X, W = x.double(), w.double()
    z = scale * (X @ W.T) + (0 if offset is None else offset.double())
    out_cls = torch.zeros(w.shape[0], dtype=torch.bool, device=DEV) if offset is None else offset == -math.inf
    z = z.masked_fill(out_cls, -math.inf)
    V = w.shape[0]
    if idx is None:
        idx, q = labels.long()[:, None], torch.ones(len(labels), 1, dtype=torch.float64, device=DEV)
        q = q * ((idx >= 0) & (idx < V))
        logq = torch.zeros_like(q)
    else:
        idx = idx.long()
        ok = (idx >= 0) & (idx < V)
        t = (val.double() / tau).masked_fill(~ok, -math.inf)
        q = torch.softmax(t, 1).nan_to_num(0.0)
        logq = torch.where(q > 0, torch.log(q.clamp(min=1e-300)), 0.0)
    lse = torch.logsumexp(z / tau, 1)
    live = (q.sum(1) > 0) & (lse > -math.inf)
    at = idx.clamp(0, V - 1)
    logp = (z / tau).gather(1, at) - lse[:, None]
    loss = tau * tau * torch.where(q > 0, q * (logq - logp), 0.0).sum(1)
    loss = torch.where(live, loss, 0.0)
    g = torch.ones(len(x), dtype=torch.float64, device=DEV) if drow is None else drow.double().expand(len(x))
    p = torch.softmax(z / tau, 1)
    p[~live] = 0
    dz = p.clone().scatter_add_(1, at, -torch.where(live[:, None], q, 0.0)) * (g * tau * scale)[:, None]
    dz[~live] = 0
    dz[:, out_cls] = 0
    Xz = torch.where(live[:, None], X, 0.0)
    Wz = torch.where(out_cls[:, None], 0.0, W)
    mag = (X.abs() @ W.abs().T * abs(scale)).masked_fill(out_cls, 0.0).amax(1)
    if offset is not None:
        mag = mag + torch.where(out_cls, 0.0, offset.double().abs()).max()
    return dict(loss=loss, lse=torch.logsumexp(z, 1), live=live, dz=dz, p=p * (g * tau * scale).abs()[:, None], dx=dz @ Wz, dw=dz.T @ Xz, X=Xz, W=Wz, mag=mag / tau, g=g)


def loss_tol(ref, d):
    mag = torch.where(ref["live"], ref["mag"], 0.0).nan_to_num(0.0)
    return 2 * (d * U * mag + 16 * U * (2 * mag + 32 * 1.45))


def check_rows(got, want, tol):
    assert got.dtype == F32 and torch.equal(torch.isinf(got), torch.isinf(want)), "infinities"
    fin = torch.isfinite(want)
    err = (got.double() - want).abs()
    assert torch.all(err[fin] <= tol[fin]), (err[fin] / tol[fin]).max().item()


def check_grads(got_dx, got_dw, ref, x, scale=1.0, tau=1.0):
    h = torch.finfo(x.dtype).eps / 2
    tiny = torch.finfo(x.dtype).tiny * torch.finfo(x.dtype).eps  # smallest step of the type
    d, V, N = x.shape[1], ref["W"].shape[0], x.shape[0]
    dl = loss_tol(ref, d)
    gmax = torch.where(ref["live"], ref["g"].abs(), 0.0).max() * tau * abs(scale)
    edz = h * ref["dz"].abs() + ref["p"] * (2.2 * dl)[:, None] + gmax * 2 * tiny / (4096 if x.dtype == F16 else 1)
    edz = torch.where(ref["live"][:, None], edz, 0.0)
    for got, want, e, n, other in ((got_dx, ref["dx"], edz, V, ref["W"]), (got_dw, ref["dw"], edz.T, N, ref["X"])):
        if got is None:
            continue
        a = ref["dz"].abs() if got is got_dx else ref["dz"].abs().T
        tol = e @ other.abs() + (n + 8) * U * (a @ other.abs()) + 1.01 * h * want.abs() + tiny
        assert got.dtype == x.dtype and got.shape == want.shape
        err = (got.double() - want).abs()
        assert torch.all(err <= tol), (err / tol).max().item()


def run_ce(x, w, labels, offset=None, scale=1.0, drow=None, dx=True, dw=True):
    ops = _ops()
    loss, lse = ops.linear_ce_fwd(x, w, labels, offset=offset, scale=scale)
    return loss, lse, *ops.linear_ce_bwd(x, w, labels, lse, drow, offset=offset, scale=scale, want_dx=dx, want_dw=dw)


def ce_case(N, V, d, dtype, seed=0):
    return _rand(N, d, seed=seed, dtype=dtype), (_rand(V, d, seed=seed + 1) * (2 / math.sqrt(d))).to(dtype), _randint(V, (N,), seed + 2)


CE_SIZES = [(1, 1, 8), (1, 2, 8), (3, 5, 16), (1, 1000, 64), (64, 64, 64), (127, 129, 72), (130, 257, 104), (300, 1201, 320), (33, 9001, 264), (257, 128, 40),
            (2600, 3900, 40),   # 256 x 256 tiles
            (700, 21000, 24), (1100, 30000, 264),  # the same with classes cut into slices for dx
            (40000, 4500, 16),  # several pieces of the class list
            (9000, 300, 72), (5000, 130, 520)]  # rows cut into slices for dw


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("N,V,d", CE_SIZES)
def test_linear_ce(N, V, d, dtype):
    x, w, labels = ce_case(N, V, d, dtype)
    if N > 2:
        labels[::3] = -100
        labels[1] = V  # behind the list: left out as well
    drow = _rand(N, seed=9).abs() + 0.25
    loss, lse, dx, dw = run_ce(x, w, labels, drow=drow)
    ref = reference(x, w, labels, drow=drow)
    check_rows(loss, ref["loss"], loss_tol(ref, d))
    check_rows(lse, ref["lse"], 2 * (d * U * ref["mag"] + 16 * U * (2 * ref["mag"] + 46.4)))
    check_grads(dx, dw, ref, x)


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("N,V,d", [(5, 7, 8), (200, 700, 64), (2600, 3900, 40)])
def test_linear_ce_offset_scale_label_types(N, V, d, dtype):
    """Class offsets with left-out classes, a logit scale, int32 labels, one gradient for all rows, negative and zero row gradients."""
    x, w, labels = ce_case(N, V, d, dtype, seed=3)
    off = _rand(V, seed=4)
    off[::4] = -math.inf
    off[labels[2:]] = 0.5
    labels[0] = 4  # a left-out class: loss inf, the gradient reaches the others only
    off[4] = -math.inf
    drow = _rand(N, seed=5)
    drow[1] = 0
    loss, lse, dx, dw = run_ce(x, w, labels.int(), offset=off, scale=1.7, drow=drow)
    ref = reference(x, w, labels, offset=off, scale=1.7, drow=drow)
    assert loss[0].item() == math.inf
    check_rows(loss, ref["loss"], loss_tol(ref, d))
    check_grads(dx, dw, ref, x, scale=1.7)
    assert torch.all(dw[off == -math.inf] == 0)
    one = torch.tensor([0.125], device=DEV)
    _, _, dx1, dw1 = run_ce(x, w, labels, offset=off, scale=-0.4, drow=one)
    check_grads(dx1, dw1, reference(x, w, labels, offset=off, scale=-0.4, drow=one), x, scale=-0.4)


@pytest.mark.parametrize("dtype", [BF, F16])
def test_linear_ce_bad_values_in_left_out_places(dtype):
    """NaN and infinities in ignored rows of x and in left-out classes of w reach nothing."""
    x, w, labels = ce_case(150, 300, 64, dtype, seed=6)
    off = torch.zeros(300, device=DEV)
    off[::5] = -math.inf
    labels[labels % 5 == 0] += 1
    labels[::4] = -1
    clean = run_ce(x, w, labels, offset=off)
    xb, wb = x.clone(), w.clone()
    xb[::8], xb[4::8] = math.nan, math.inf
    wb[::10], wb[5::10] = math.nan, -math.inf
    bad = run_ce(xb, wb, labels, offset=off)
    live = labels >= 0
    for a, b in zip(clean, bad):
        if a.dim() == 1:
            assert torch.equal(a[live], b[live])
    assert torch.all(bad[0][~live] == 0)
    for a, b in zip(clean[2:], bad[2:]):
        assert torch.equal(a, b)
    assert torch.all(bad[2][~live] == 0) and torch.all(bad[3][::5] == 0)


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("N,V,d", [(2600, 3900, 40), (1100, 30000, 72), (40000, 4500, 16), (140, 2000, 64)])
def test_bad_values_in_left_out_places_of_every_tile(N, V, d, dtype):
    """The same over the large tile, slices and pieces of the class list, and for the distillation: same bits as with clean numbers there."""
    ops = _ops()
    x, w, labels = ce_case(N, V, d, dtype, seed=70)
    off = 0.1 * _rand(V, seed=71)
    off[::50] = -math.inf
    off[32:96] = -math.inf
    off[-1] = -math.inf
    out = off == -math.inf
    labels[out[labels]] = -1
    labels[::9] = -1
    idx, val = teacher(N, V, 10, 72, empty=False)
    idx[::9] = -1
    idx = torch.where(out[idx.long().clamp(min=0)], -1, idx).int()
    none = (idx < 0).all(1)
    xb, wb = x.clone(), w.clone()
    xb[(labels < 0) & none] = math.nan
    wb[out] = math.inf
    wb[out.nonzero()[::2, 0]] = math.nan
    for a, b in zip(run_ce(x, w, labels, offset=off)[2:], run_ce(xb, wb, labels, offset=off)[2:]):
        assert torch.equal(a, b)
    got = []
    for xs, ws in ((x, w), (xb, wb)):
        loss, saved = ops.linear_distill_fwd(xs, ws, idx, val, offset=off)
        got.append((loss, *ops.linear_distill_bwd(xs, ws, idx, saved, offset=off)))
    for a, b in zip(*got):
        assert torch.equal(a, b) and torch.all(torch.isfinite(a))
    ref = reference(x, w, labels, offset=off)
    check_grads(*run_ce(xb, wb, labels, offset=off)[2:], ref, x)


def test_linear_ce_nothing_left():
    """Every class left out, every row ignored, no rows at all: losses and gradients of 0."""
    x, w, labels = ce_case(9, 20, 16, BF)
    loss, lse, dx, dw = run_ce(x, w, labels, offset=torch.full((20,), -math.inf, device=DEV))
    assert torch.all(loss == 0) and torch.all(lse == -math.inf) and torch.all(dx == 0) and torch.all(dw == 0)
    loss, lse, dx, dw = run_ce(x, w, torch.full_like(labels, -100))
    assert torch.all(loss == 0) and torch.all(dx == 0) and torch.all(dw == 0)
    loss, lse, dx, dw = run_ce(x[:0], w, labels[:0])
    assert loss.shape == (0,) and dx.shape == (0, 16) and torch.all(dw == 0)


def test_linear_ce_far_logits():
    """Logits of +-10^3: the running maximum keeps the sums finite."""
    x, w, labels = ce_case(70, 400, 32, BF, seed=8)
    loss, lse, dx, dw = run_ce(x, w, labels, scale=300.0)
    ref = reference(x, w, labels, scale=300.0)
    check_rows(loss, ref["loss"], loss_tol(ref, 32))
    check_grads(dx, dw, ref, x, scale=300.0)


def test_linear_ce_strides_and_alignment():
    """Column slices of wider buffers, an odd pitch (copied), a repeated row, a misaligned start: same bits as contiguous inputs."""
    N, V, d = 100, 333, 48
    x, w, labels = ce_case(N, V, d, F16, seed=11)
    want = run_ce(x, w, labels)

    def within(t, pitch, lead):
        buf = torch.full((t.shape[0], pitch), math.nan, dtype=t.dtype, device=DEV)
        buf[:, lead:lead + t.shape[1]] = t
        return buf[:, lead:lead + t.shape[1]]

    for pitch, lead in ((64, 8), (51, 1), (56, 3)):
        for a, b in zip(want, run_ce(within(x, pitch, lead), within(w, pitch, lead), labels)):
            assert torch.equal(a, b)
    for a, b in zip(want, run_ce(x.T.contiguous().T, w.T.contiguous().T, labels)):
        assert torch.equal(a, b)
    rep = x[:1].expand(N, d)
    for a, b in zip(run_ce(rep.contiguous(), w, labels), run_ce(rep, w, labels)):
        assert torch.equal(a, b)


def test_linear_ce_parts_and_repeats():
    """dx alone, dw alone and both agree to the bit; so do two calls."""
    x, w, labels = ce_case(260, 1500, 80, BF, seed=12)
    a, b = run_ce(x, w, labels), run_ce(x, w, labels)
    for s, t in zip(a, b):
        assert torch.equal(s, t)
    assert torch.equal(run_ce(x, w, labels, dw=False)[2], a[2]) and run_ce(x, w, labels, dw=False)[3] is None
    assert torch.equal(run_ce(x, w, labels, dx=False)[3], a[3]) and run_ce(x, w, labels, dx=False)[2] is None


KD_SIZES = [(1, 1, 8, 1), (2, 9, 8, 3), (96, 365, 64, 16), (131, 1201, 72, 50), (5, 300, 16, 512), (2600, 3900, 40, 5), (40000, 4500, 16, 3)]


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("N,V,d,k", KD_SIZES)
def test_linear_distill(N, V, d, k, dtype):
    ops = _ops()
    x, w, _ = ce_case(N, V, d, dtype, seed=20)
    idx, val = teacher(N, V, k, 21, empty=N > 2)  # (drawn with repetition: classes are named twice)
    drow = _rand(N, seed=23).abs() + 0.25
    for tau, off in ((1.0, None), (2.5, _rand(V, seed=24))):
        loss, saved = ops.linear_distill_fwd(x, w, idx, val, tau=tau, offset=off, scale=1.3)
        dx, dw = ops.linear_distill_bwd(x, w, idx, saved, drow, tau=tau, offset=off, scale=1.3)
        ref = reference(x, w, idx=idx, val=val, tau=tau, offset=off, scale=1.3, drow=drow)
        # sum over slots of q times the error of log p and of log q (a teacher logit up to 16, a few roundings)
        check_rows(loss, ref["loss"], tau * tau * (2 * loss_tol(ref, d) + 64 * U * 16))
        check_grads(dx, dw, ref, x, scale=1.3, tau=tau)


FEW = [(1, 33, 8), (2, 32, 256), (31, 31, 264), (32, 97, 960), (32, 9001, 512), (33, 64, 608), (64, 700, 40), (60, 20000, 264), (65, 65, 320), (128, 1000, 256), (97, 12000, 304), (1, 40000, 520),
       (33, 70, 616), (70, 70, 328), (32, 70, 968),
       (16, 70, 1024), (16, 40, 1032), (17, 40, 960), (48, 70, 736), (48, 70, 744), (64, 70, 608), (64, 70, 616), (80, 70, 480), (80, 70, 488), (128, 70, 320)]  # as much as its LDS holds, and more


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("N,V,d", FEW)
def test_few_rows(N, V, d, dtype):
    """The ends of the backward of few rows, with every kind of row and class: ignored rows and left-out classes that hold NaN, negative and zero gradients."""
    ops = _ops()
    x, w, labels = ce_case(N, V, d, dtype, seed=60)
    off = _rand(V, seed=61)
    drow = _rand(N, seed=62)
    xb, wb = x.clone(), w.clone()
    if N > 2:
        labels[::5] = -1
        xb[::5] = math.nan
        drow[1] = 0
    if V > 32:
        off[::7] = -math.inf
        wb[::7] = math.inf
        off[labels[labels >= 0]] = 0.25
    wb = torch.where((off == -math.inf)[:, None], wb, w)
    loss, lse, dx, dw = run_ce(xb, wb, labels, offset=off, scale=0.8, drow=drow)
    ref = reference(x, w, labels, offset=off, scale=0.8, drow=drow)
    check_rows(loss, ref["loss"], loss_tol(ref, d))
    check_grads(dx, dw, ref, x, scale=0.8)
    again = run_ce(xb, wb, labels, offset=off, scale=0.8, drow=drow)
    assert torch.equal(dx, again[2]) and torch.equal(dw, again[3])
    assert torch.equal(run_ce(xb, wb, labels, offset=off, scale=0.8, drow=drow, dw=False)[2], dx)
    assert torch.equal(run_ce(xb, wb, labels, offset=off, scale=0.8, drow=drow, dx=False)[3], dw)
    k = min(V, 11)
    idx, val = teacher(N, V, k, 63, empty=N > 2)
    loss, saved = ops.linear_distill_fwd(x, w, idx, val, tau=2.0)
    dx, dw = ops.linear_distill_bwd(x, w, idx, saved, drow, tau=2.0)
    ref = reference(x, w, idx=idx, val=val, tau=2.0, drow=drow)
    check_rows(loss, ref["loss"], 4 * (2 * loss_tol(ref, d) + 64 * U * 16))
    check_grads(dx, dw, ref, x, tau=2.0)


@pytest.mark.parametrize("N,k", [(8, 512), (9, 512), (128, 32), (128, 33)])
def test_few_rows_slots(N, k):
    """As many slots as the few rows' kernel takes, and one row or slot more."""
    ops = _ops()
    x, w, _ = ce_case(N, 900, 64, BF, seed=65)
    idx, val = teacher(N, 900, k, 66)
    loss, saved = ops.linear_distill_fwd(x, w, idx, val, tau=1.5)
    ref = reference(x, w, idx=idx, val=val, tau=1.5)
    check_rows(loss, ref["loss"], 2.25 * (2 * loss_tol(ref, 64) + 64 * U * 16))
    check_grads(*ops.linear_distill_bwd(x, w, idx, saved, tau=1.5), ref, x, tau=1.5)


def test_linear_distill_types_and_infinities():
    """16-bit teacher logits; -inf in a slot counts as nothing; a slot at a left-out class is loss inf; NaN in rows without a teacher reaches nothing."""
    ops = _ops()
    x, w, _ = ce_case(40, 90, 32, BF, seed=30)
    idx, val = teacher(40, 90, 6, 31, empty=False, dup=False)
    idx[3] = -1
    val[5, 2:] = -math.inf
    val[6] = -math.inf
    xb = x.clone()
    xb[3], xb[6] = math.nan, math.inf
    for vt in (val.to(BF), val.to(F16), val):
        loss, saved = ops.linear_distill_fwd(xb, w, idx, vt, tau=1.5)
        dx, dw = ops.linear_distill_bwd(xb, w, idx, saved, tau=1.5)
        ref = reference(x, w, idx=idx, val=vt, tau=1.5)
        check_rows(loss, ref["loss"], 2.25 * (2 * loss_tol(ref, 32) + 64 * U * 16))
        assert loss[3] == 0 and loss[6] == 0
        check_grads(dx, dw, ref, x, tau=1.5)
    off = torch.zeros(90, device=DEV)
    off[idx[0, 0].long()] = -math.inf
    loss, saved = ops.linear_distill_fwd(x, w, idx[:1].expand(40, 6), val[:1].expand(40, 6), offset=off)
    assert torch.all(loss == math.inf)


def test_ce_is_distillation_from_one_class():
    """k = 1 is the cross entropy of that class."""
    ops = _ops()
    x, w, labels = ce_case(60, 200, 64, BF, seed=33)
    loss, lse = ops.linear_ce_fwd(x, w, labels)
    kd, _ = ops.linear_distill_fwd(x, w, labels.int()[:, None], torch.zeros(60, 1, device=DEV))
    ref = reference(x, w, labels)
    assert torch.all((loss - kd).abs().double() <= 2 * loss_tol(ref, 64))


def map_reference(z, idx, val, tau, drow):
    z, V = z.double(), z.shape[-1]
    idx = idx.long()
    ok = (idx >= 0) & (idx < V)
    q = torch.softmax((val.double() / tau).masked_fill(~ok, -math.inf), -1).nan_to_num(0.0)
    live = (q.sum(-1) > 0) & (z.amax(-1) > -math.inf)
    q = q * live[..., None]
    lp = torch.log_softmax(z / tau, -1)
    at = idx.clamp(0, V - 1)
    logq = torch.where(q > 0, torch.log(q.clamp(min=1e-300)), 0.0)
    loss = tau * tau * torch.where(q > 0, q * (logq - lp.gather(-1, at)), 0.0).sum(-1)
    g = (torch.ones_like(loss) if drow is None else drow.double().expand(loss.shape)) * tau
    p = torch.where(live[..., None], lp.exp(), 0.0)
    dz = p.clone().scatter_add_(-1, at, -q) * g[..., None]
    return loss, dz, (p + p.clone().zero_().scatter_add_(-1, at, q)) * g.abs()[..., None]


def check_map(got, z, idx, val, tau, drow):
    loss, dz = got
    wl, wd, mag = map_reference(z, idx, val, tau, drow)
    V = z.shape[-1]
    zm = torch.where(torch.isfinite(z), z.abs(), 0).double().amax(-1) / tau
    # exponent (z - max) c: two roundings of it, exp2 / log2 to two; the sum of V terms in a tree over 16 per thread and lanes: 48 roundings at most
    rel = U * (8 * zm + 64)
    check_rows(loss, wl, tau * tau * 2 * (rel + U * 16 * (zm + 40)))
    h = 0.0 if dz.dtype == F32 else torch.finfo(dz.dtype).eps / 2
    tiny = torch.finfo(dz.dtype).tiny * torch.finfo(dz.dtype).eps
    tol = 1.01 * (h * wd.abs() + (rel[..., None] + 64 * U) * mag) + 2 * tiny
    err = (dz.double() - wd).abs()
    assert torch.all(err <= tol), (err / tol).max().item()


MAP_SIZES = [(1, 1, 1, 1), (1, 1, 2, 2), (7, 1, 16, 16), (300, 4, 16, 9), (70, 1, 17, 5), (65, 1, 3, 17), (90, 1, 74, 74), (40, 2, 128, 33), (40, 1, 129, 128), (33, 4, 16, 16), (50, 4, 13, 5), (20, 1, 64, 64), (20, 1, 65, 64), (9, 1, 64, 65), (40, 1, 80, 10),
             (13, 1, 1203, 32), (6, 2, 2048, 100), (5, 1, 2049, 40), (3, 1, 8191, 512), (3, 1, 8193, 7), (2, 1, 16385, 33), (2, 1, 32768, 64), (2, 1, 32769, 64), (2, 1, 65537, 64), (2, 1, 100003, 30), (2, 1, 131073, 9)]


@pytest.mark.parametrize("dtype,gdt", [(F32, F32), (BF, BF), (F16, F16), (BF, F32), (F16, F32)])
@pytest.mark.parametrize("P,G,V,k", MAP_SIZES)
def test_topk_distill(P, G, V, k, dtype, gdt):
    z = (2.5 * _rand(P, G, V, seed=40)).to(dtype)
    idx, val = teacher(P * G, V, k, 41, empty=P > 2)
    idx, val = idx.view(P, G, k), val.view(P, G, k)
    drow = _rand(P, G, seed=42) + 1.5
    got = _ops().topk_distill(z, idx, val, tau=2.0, drow=drow, grad_dtype=gdt)
    assert got[1].dtype == gdt and got[1].shape == z.shape
    check_map(got, z, idx, val, 2.0, drow)
    if G == 1:
        two = _ops().topk_distill(z[:, 0], idx[:, 0], val[:, 0], tau=2.0, drow=drow[:, 0], grad_dtype=gdt)
        assert torch.equal(two[0], got[0][:, 0]) and torch.equal(two[1], got[1][:, 0])


# both numbers of slots a lane of every narrow form, tails inside a lane's classes and slots, rows that do not fill a workgroup
NARROW = [(129, 3, 16, 4), (65, 2, 10, 3), (90, 1, 4, 16), (90, 1, 32, 8), (67, 1, 31, 9), (70, 1, 6, 29), (70, 1, 64, 16), (33, 2, 50, 17), (70, 1, 96, 16), (35, 1, 95, 17), (31, 1, 12, 90),
          (70, 1, 128, 16), (33, 1, 97, 128), (17, 1, 127, 99)]


@pytest.mark.parametrize("dtype,vdt", [(F32, F32), (BF, F32), (BF, BF), (F16, F16), (F32, BF)])
@pytest.mark.parametrize("P,G,V,k", NARROW)
def test_topk_distill_narrow_rows(P, G, V, k, dtype, vdt):
    z = (2.5 * _rand(P, G, V, seed=43)).to(dtype)
    for dup in (True, False):
        if not dup and k > V:
            continue
        idx, val = teacher(P * G, V, k, 44, dup=dup)
        idx, val = idx.view(P, G, k), val.view(P, G, k).to(vdt)
        check_map(_ops().topk_distill(z, idx, val, tau=1.5), z, idx, val, 1.5, None)


@pytest.mark.parametrize("dtype", [F32, BF, F16])
@pytest.mark.parametrize("V", [130, 133, 255, 503, 511, 512, 513, 519, 1017, 1024, 1026, 1033, 2041, 2046, 2047])
def test_topk_distill_row_tails(V, dtype):
    """What is left of a row behind its last whole 16 bytes, and the ends of the forms by length."""
    z = (2.5 * _rand(9, V, seed=45)).to(dtype)
    idx, val = teacher(9, V, 70, 46)
    idx[:, 5] = V - 1
    idx[1, 6:9] = V - 2
    got = _ops().topk_distill(z, idx, val, tau=1.5)
    check_map(got, z, idx, val, 1.5, None)
    same = torch.cat([z, z], 1)  # in place, every row at another alignment
    part = same[:, V:]
    loss, _ = _ops().topk_distill(part, idx, val, tau=1.5, out=part)
    assert torch.equal(loss, got[0]) and torch.equal(part, got[1]) and torch.equal(same[:, :V], z)


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("V,k", [(700, 9), (2051, 9), (3001, 33), (4097, 30), (9001, 30), (20003, 7), (33001, 9), (65535, 30), (65541, 31), (100001, 6), (131079, 5)])
def test_topk_distill_odd_values_of_every_type(V, k, dtype):
    """Rows that hold NaN and have no teacher, rows of nothing but -inf, -inf in the tail, one class in every slot, over all forms by length."""
    z = (2 * _rand(7, V, seed=54)).to(dtype)
    idx, val = teacher(7, V, k, 55, empty=False)
    idx[0] = V - 1
    idx[1, 1:4] = V - 2
    z[2, -5:] = -math.inf
    idx[2] = torch.where(idx[2] >= V - 5, 0, idx[2])
    z[3] = -math.inf
    idx[4] = -1
    z[4] = math.nan
    idx[5, 1:] = -1
    got = _ops().topk_distill(z, idx, val, tau=1.0)
    assert torch.all(got[0][3:5] == 0) and torch.all(got[1][3:5] == 0)
    zr = z.clone()
    zr[4] = 0
    check_map(got, zr, idx, val, 1.0, None)
    same = z.clone()
    loss, _ = _ops().topk_distill(same, idx, val, tau=1.0, out=same)
    assert torch.equal(loss, got[0]) and torch.equal(same, got[1])
    only, none = _ops().topk_distill(z, idx, val, tau=1.0, want_grad=False)
    assert none is None and torch.equal(only, got[0])


@pytest.mark.parametrize("P,V,k", [(9, 100, 300), (5, 1, 200), (6, 2048, 512), (3, 2040, 511)])
def test_topk_distill_more_slots_than_classes_and_the_most(P, V, k):
    z = 2.5 * _rand(P, V, seed=47)
    idx, val = teacher(P, V, k, 48)
    check_map(_ops().topk_distill(z, idx, val, tau=2.0), z, idx, val, 2.0, None)
    check_map(_ops().topk_distill(z.bfloat16(), idx, val, tau=2.0), z.bfloat16(), idx, val, 2.0, None)


@pytest.mark.parametrize("V,k", [(16, 4), (30, 8), (64, 16), (80, 10), (90, 80), (128, 16)])
def test_topk_distill_narrow_odd_values(V, k):
    test_topk_distill_odd_values(V, k)


@pytest.mark.parametrize("V,k", [(16, 12), (30, 12), (40, 12), (100, 70), (1000, 20), (1000, 100), (5000, 20), (9000, 20), (40000, 20), (140000, 20)])
def test_topk_distill_odd_values(V, k):
    """The same class in many slots, -inf logits, rows of nothing but -inf, rows without a teacher that hold NaN, far logits."""
    z = 2 * _rand(12, V, seed=50)
    idx, val = teacher(12, V, k, 51, empty=False, dup=False)
    idx[0, :] = 3
    idx[1, ::2] = idx[1, 0].item()
    z[2, ::2] = -math.inf
    idx[2] = idx[2] | 1
    z[3] = -math.inf
    idx[4] = -1
    z[4] = math.nan
    z[5] *= 400
    z[6, idx[6, 0].long()] = -math.inf  # the student rules out what the teacher names: loss inf, the gradient stays finite
    got = _ops().topk_distill(z, idx, val, tau=1.0)
    assert got[0][3] == 0 and got[0][4] == 0 and torch.all(got[1][3:5] == 0) and got[0][6] == math.inf
    zr = z.clone()
    zr[4] = 0
    check_map(got, zr, idx, val, 1.0, None)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("G,V,lead,tail", [(4, 16, 0, 80), (1, 80, 64, 0), (1, 77, 3, 5), (1, 3001, 65, 6)])
def test_topk_distill_on_a_slice_of_a_map(G, V, lead, tail, dtype):
    """Channels of an NHWC map read in place, the gradient written into a slice of another map (and into the map itself), the neighbours untouched."""
    ops = _ops()
    P, k = 60, 8
    full = (2 * _rand(P, lead + G * V + tail, seed=60)).to(dtype)
    idx, val = teacher(P * G, V, k, 61)
    idx, val = idx.view(P, G, k), val.view(P, G, k)

    def part(t):
        return t[:, lead:lead + G * V].unflatten(1, (G, V))

    want = ops.topk_distill(part(full).contiguous(), idx, val, tau=2.0)
    got = ops.topk_distill(part(full), idx, val, tau=2.0)
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
    grad = torch.full((P, lead + G * V + tail + 9), 7.0, dtype=dtype, device=DEV)
    loss, out = ops.topk_distill(part(full), idx, val, tau=2.0, out=part(grad))
    assert torch.equal(part(grad), want[1]) and out.data_ptr() == part(grad).data_ptr()
    grad[:, lead:lead + G * V] = 7.0
    assert torch.all(grad == 7.0)
    same = full.clone()
    loss, _ = ops.topk_distill(part(same), idx, val, tau=2.0, out=part(same))
    assert torch.equal(loss, want[0]) and torch.equal(part(same), want[1])
    same[:, lead:lead + G * V] = full[:, lead:lead + G * V]
    assert torch.equal(same, full)
    only, none = ops.topk_distill(part(full), idx, val, tau=2.0, want_grad=False)
    assert none is None and torch.equal(only, want[0])


def test_no_rows():
    ops = _ops()
    loss, dz = ops.topk_distill(torch.empty(0, 50, device=DEV), torch.empty(0, 4, dtype=torch.int32, device=DEV), torch.empty(0, 4, device=DEV))
    assert loss.shape == (0,) and dz.shape == (0, 50)
    w = _rand(30, 16, dtype=BF)
    loss, saved = ops.linear_distill_fwd(w[:0], w, torch.empty(0, 4, dtype=torch.int32, device=DEV), torch.empty(0, 4, device=DEV))
    dx, dw = ops.linear_distill_bwd(w[:0], w, torch.empty(0, 4, dtype=torch.int32, device=DEV), saved)
    assert loss.shape == (0,) and dx.shape == (0, 16) and torch.all(dw == 0)


def test_gradients_against_differences():
    """dx and dw of the fused losses, and dlogits, against central differences of the 64-bit loss along random directions. The difference's own error is
    (step^2 / 6) of a third derivative (below 1e-5 here); the kernels' is that of a 16-bit gradient, h sqrt(n) of sum |g_i u_i| at random signs -- 4 h of the
    2-norms' product is asserted."""
    from cerberusdet_amd.utils import loss as UL

    x, w, labels = ce_case(24, 60, 32, BF, seed=70)
    idx, val = teacher(24, 60, 8, 71)
    drow = _rand(24, seed=72).abs()
    cases = [("ce", lambda X, W: reference(X, W, labels)["loss"], lambda X, W: UL.linear_cross_entropy(X, W, labels, reduction="none")),
             ("kd", lambda X, W: reference(X, W, idx=idx, val=val, tau=2.0)["loss"], lambda X, W: UL.linear_distillation(X, W, idx, val, tau=2.0, reduction="none"))]
    for name, exact, fused in cases:
        xl, wl = x.clone().requires_grad_(), w.clone().requires_grad_()
        (fused(xl, wl) * drow).sum().backward()
        for leaf, seed in ((xl, 73), (wl, 74)):
            u = _rand(*leaf.shape, seed=seed).double()
            step = 1e-4

            def at(s):
                X = x.double() + (s * u if leaf is xl else 0)
                W = w.double() + (s * u if leaf is wl else 0)
                return (exact(X, W) * drow.double()).sum()

            num = (at(step) - at(-step)) / (2 * step)
            ana = (leaf.grad.double() * u).sum()
            assert abs(num - ana) <= 4 * (2.0 ** -8) * leaf.grad.double().norm() + 1e-4, (name, num, ana)
    z = _rand(24, 60, seed=75).requires_grad_()
    (UL.topk_distillation(z, idx, val, tau=2.0, reduction="none") * drow).sum().backward()
    u = _rand(24, 60, seed=76).double()

    def mat(s):
        return (map_reference(z.detach().double() + s * u, idx, val, 2.0, None)[0] * drow.double()).sum()

    assert abs((mat(1e-4) - mat(-1e-4)) / 2e-4 - (z.grad.double() * u).sum()) <= 1e-4


def test_streams_and_captured_graphs():
    """Calls on another stream, and forward + backward captured in two graphs that are replayed in turn with eager work between, give the eager result."""
    ops = _ops()
    data = []
    for s in (80, 90):
        x, w, labels = ce_case(150, 700, 64, BF, seed=s)
        idx, val = teacher(150, 700, 12, s + 5)
        z = 2 * _rand(40, 700, seed=s + 7)
        data.append((x, w, labels, idx, val, z))

    def all_of(x, w, labels, idx, val, z):
        loss, lse = ops.linear_ce_fwd(x, w, labels)
        kd, saved = ops.linear_distill_fwd(x, w, idx, val, tau=2.0)
        return [loss, lse, *ops.linear_ce_bwd(x, w, labels, lse), kd, *ops.linear_distill_bwd(x, w, idx, saved, tau=2.0), *ops.topk_distill(z, idx[:40], val[:40])]

    want = [all_of(*d) for d in data]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = all_of(*data[0])
    side.synchronize()
    for a, b in zip(want[0], got):
        assert torch.equal(a, b)
    graphs = []
    for d in data:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = all_of(*d)
        graphs.append((g, outs))
    for _ in range(3):
        for (g, outs), ref in zip(graphs, want):
            for o in outs:
                o.fill_(5)
            g.replay()
            eager = all_of(*data[0])
            torch.cuda.synchronize()
            for a, b in zip(ref, outs):
                assert torch.equal(a, b)
            for a, b in zip(want[0], eager):
                assert torch.equal(a, b)


def test_captured_training_step():
    """The differentiable losses with their means and a backward pass, captured once and replayed with new data in the same buffers: each replay is the eager
    step on that data. (The leaves' gradients are taken with autograd.grad; no eager graph of the same leaves lives during the capture.)"""
    from cerberusdet_amd.utils import loss as UL

    N, V, d, k = 5000, 700, 64, 10
    x, w, labels = ce_case(N, V, d, BF, seed=120)
    idx, val = teacher(N, V, k, 121)
    z = 2 * _rand(N, 50, seed=122)
    zi, zv = teacher(N, 50, k, 123)

    def step(x, w, z, labels, idx, val, zi, zv):
        x, w, z = (t.detach().requires_grad_() for t in (x, w, z))
        total = UL.linear_cross_entropy(x, w, labels) + 0.5 * UL.linear_distillation(x, w, idx, val, tau=2.0) + UL.topk_distillation(z, zi, zv, tau=2.0)
        return [total.detach(), *torch.autograd.grad(total, (x, w, z))]

    data = (x, w, z, labels, idx, val, zi, zv)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*data)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(*data)
    for turn in range(4):
        x.copy_(_rand(N, d, seed=130 + turn, dtype=BF))
        z.copy_(_rand(N, 50, seed=140 + turn))
        labels.copy_(_randint(V, (N,), 150 + turn))
        for o in outs:
            o.fill_(3)
        graph.replay()
        got = [o.clone() for o in outs]
        want = step(*data)
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b), turn


def test_two_threads_two_streams():
    """Calls of different sizes from two host threads on streams of their own."""
    import threading

    cases = [ce_case(n, v, d, BF, seed=160 + n) for n, v, d in ((300, 2000, 64), (1100, 30000, 264))]
    want = [run_ce(*c) for c in cases]
    torch.cuda.synchronize()
    got, streams = [None, None], [torch.cuda.Stream(), torch.cuda.Stream()]

    def work(i):
        with torch.cuda.stream(streams[i]):
            for _ in range(10):
                got[i] = run_ce(*cases[i])
        streams[i].synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for a, b in zip(want, got):
        for s, t in zip(a, b):
            assert torch.equal(s, t)


def test_gradients_leave_pitch_tails_alone():
    """Through the C interface: dx and dw with pitches above d; what lies behind a row stays."""
    import ctypes as C

    from cerberusdet_amd import _lib as L

    ops, N, V, d = _ops(), 200, 700, 64
    x, w, labels = ce_case(N, V, d, BF, seed=170)
    loss, lse, dx, dw = run_ce(x, w, labels)
    lib = L.load()
    desc = L.LinearLossDesc(N, V, d, L.BF16, d, d, 1.0, 1.0, None, 1)
    bx, bw = torch.full((N, d + 24), 9.0, dtype=BF, device=DEV), torch.full((V, d + 8), 9.0, dtype=BF, device=DEV)
    ws = torch.empty(lib.cdet_linear_loss_ws_bytes(C.byref(desc), 1), dtype=torch.uint8, device=DEV).fill_(255)  # (contents do not matter)
    L.check(lib.cdet_linear_ce_bwd(C.byref(desc), x.data_ptr(), w.data_ptr(), labels.data_ptr(), lse.data_ptr(), None, 0, bx.data_ptr(), d + 24, bw.data_ptr(), d + 8,
                                   ws.data_ptr(), ops.stream()))
    assert torch.equal(bx[:, :d], dx) and torch.equal(bw[:, :d], dw) and torch.all(bx[:, d:] == 9) and torch.all(bw[:, d:] == 9)


def test_offsets_beyond_32_bits():
    """Rows more than 2^31 elements apart from the first: x and w with the largest pitch, logits of 2.6e9 elements."""
    ops, ld = _ops(), (1 << 22) - 8
    x, w, labels = ce_case(700, 600, 64, BF, seed=180)
    want = run_ce(x, w, labels)
    big = torch.empty(700, ld, dtype=BF, device=DEV)
    big[:, :64], big[:600, 128:192] = x, w
    for a, b in zip(want, run_ce(big[:, :64], big[:600, 128:192], labels)):
        assert torch.equal(a, b)
    del big
    P, V = 40000, 65536
    z = torch.empty(P, V, dtype=BF, device=DEV)
    z[:] = _rand(1, V, seed=181).to(BF)
    z[P - 3:] = _rand(3, V, seed=182).to(BF)
    idx, val = teacher(P, V, 4, 183)
    loss, dz = ops.topk_distill(z, idx, val)
    few = ops.topk_distill(z[P - 3:].clone(), idx[P - 3:], val[P - 3:])
    assert torch.equal(loss[P - 3:], few[0]) and torch.equal(dz[P - 3:], few[1])


def test_few_rows_far_and_pitched():
    """Rows of x and w more than 2^31 elements from the first; dx and dw with pitches above d and a workspace full of ones: what lies behind a row stays."""
    import ctypes as C

    from cerberusdet_amd import _lib as L

    ops, ld, N, V, d = _ops(), (1 << 22) - 8, 100, 600, 64
    x, w, labels = ce_case(N, V, d, BF, seed=190)
    loss, lse, dx, dw = run_ce(x, w, labels)
    big = torch.empty(V, ld, dtype=BF, device=DEV)
    big[:N, :d], big[:, 128:128 + d] = x, w
    for a, b in zip((loss, lse, dx, dw), run_ce(big[:N, :d], big[:, 128:128 + d], labels)):
        assert torch.equal(a, b)
    del big
    lib = L.load()
    desc = L.LinearLossDesc(N, V, d, L.BF16, d, d, 1.0, 1.0, None, 1)
    bx, bw = torch.full((N, d + 24), 9.0, dtype=BF, device=DEV), torch.full((V, d + 8), 9.0, dtype=BF, device=DEV)
    size = lib.cdet_linear_loss_ws_bytes(C.byref(desc), 1)
    ws = torch.empty(size + 512, dtype=torch.uint8, device=DEV).fill_(255)
    L.check(lib.cdet_linear_ce_bwd(C.byref(desc), x.data_ptr(), w.data_ptr(), labels.data_ptr(), lse.data_ptr(), None, 0, bx.data_ptr(), d + 24, bw.data_ptr(), d + 8,
                                   ws.data_ptr(), ops.stream()))
    assert torch.equal(bx[:, :d], dx) and torch.equal(bw[:, :d], dw) and torch.all(bx[:, d:] == 9) and torch.all(bw[:, d:] == 9) and torch.all(ws[size:] == 255)


@pytest.mark.parametrize("N,V,d,k", [(1, 5000, 264, 9), (37, 900, 320, 20), (100, 700, 64, 5)])
def test_few_rows_captured(N, V, d, k):
    """Losses and gradients of few rows captured and replayed on new numbers, eager calls of other sizes in between; and on two streams at once."""
    ops = _ops()
    x, w, labels = ce_case(N, V, d, BF, seed=200)
    idx, val = teacher(N, V, k, 201, empty=False)

    def step(x, w):
        loss, lse = ops.linear_ce_fwd(x, w, labels)
        kd, saved = ops.linear_distill_fwd(x, w, idx, val, tau=2.0)
        return [loss, lse, *ops.linear_ce_bwd(x, w, labels, lse), kd, *ops.linear_distill_bwd(x, w, idx, saved, tau=2.0)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x, w)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(x, w)
    for turn in range(4):
        x.copy_(_rand(N, d, seed=210 + turn, dtype=BF))
        run_ce(*ce_case(33 + turn, 77, 40, BF, seed=220))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, step(x, w)):
            assert torch.equal(a, b), turn
    y = _rand(N, d, seed=230, dtype=BF)
    want = step(x, w), step(y, w)
    torch.cuda.synchronize()
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        outs = []
        for s, inp in zip(streams, (x, y)):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                outs.append(step(inp, w))
        torch.cuda.synchronize()
        for a, b in zip(want, outs):
            assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_used_together():
    """A student classifier learns from labels and from a teacher's top logits in one backward; the fused distillation is that of its own logits."""
    from cerberusdet_amd.utils import loss as UL

    ops = _ops()
    N, V, d, k = 200, 900, 64, 20
    x, w, labels = ce_case(N, V, d, BF, seed=100)
    xt, wt = _rand(N, d, seed=101, dtype=BF), _rand(V, d, seed=102, dtype=BF)
    val, idx = (xt.float() @ wt.float().T).topk(k, dim=1)
    xl, wl = x.clone().requires_grad_(), w.clone().requires_grad_()
    total = UL.linear_cross_entropy(xl, wl, labels) + 0.5 * UL.linear_distillation(xl, wl, idx.int(), val, tau=2.0)
    total.backward()
    m = torch.full((1,), 1 / N, device=DEV)
    rc, rk = reference(x, w, labels, drow=m), reference(x, w, idx=idx, val=val, tau=2.0, drow=0.5 * m)
    assert abs(total.item() - rc["loss"].mean().item() - 0.5 * rk["loss"].mean().item()) < 1e-4
    # two 16-bit gradients, rounded and added in 16 bits: half a step each, and the errors of their dz (as much again)
    for got, key in ((xl.grad, "dx"), (wl.grad, "dw")):
        want = rc[key] + rk[key]
        assert (got.double() - want).norm() <= 2.0 ** -8 * 2 * (rc[key].norm() + rk[key].norm())
    z = x.double() @ w.double().T
    on_logits, _ = ops.topk_distill(z.float(), idx.int(), val, tau=2.0)
    fused, _ = ops.linear_distill_fwd(x, w, idx.int(), val, tau=2.0)
    assert torch.all((on_logits - fused).abs().double() <= 4 * (2 * loss_tol(rk, d) + 64 * U * 16) * 2)


def test_head_distillation_of_a_model():
    """The Detect head's own maps: box bins and class logits of a model's output against a teacher's, and the gradient that reaches the maps."""
    import copy
    import sys

    from util import load_golden

    from cerberusdet_amd.models import CerberusDet
    from cerberusdet_amd.utils.loss import HeadDistillation

    _, meta = load_golden("model_tiny2")
    m = CerberusDet(meta["tasks"], meta["nc"], cfg=copy.deepcopy(meta["cfg"]), verbose=False)
    m.sequential_split(meta["cfg"]["cerber"], "cpu")
    m = m.to(DEV).train()
    task = meta["tasks"][0]
    nc = m.get_head(task).nc
    img = torch.rand(2, 3, 64, 64, generator=torch.Generator().manual_seed(3)).to(DEV)
    feats = [f.detach().clone().requires_grad_() for f in m(img, task)]
    teach = [f.detach() + _rand(*f.shape, seed=5 + i) for i, f in enumerate(feats)]
    scalar, items = HeadDistillation(m, k=2, tau=2.0, box=0.5, cls=2.0)(feats, teach, task)
    scalar.backward()
    box = cls = 0.0
    px = sum(f.shape[0] * f.shape[2] * f.shape[3] for f in feats)
    leaves = [f.detach().double().requires_grad_() for f in feats]
    for f, t in zip(leaves, teach):
        fr, tr = f.permute(0, 2, 3, 1).reshape(-1, 64 + nc), t.double().permute(0, 2, 3, 1).reshape(-1, 64 + nc)
        q = torch.softmax(tr[:, :64].view(-1, 4, 16) / 2, -1)
        box = box + 4 * (q * (q.log() - torch.log_softmax(fr[:, :64].view(-1, 4, 16) / 2, -1))).sum()
        val, idx = tr[:, 64:].topk(min(2, nc), dim=1)
        q = torch.softmax(val / 2, -1)
        cls = cls + 4 * (q * (q.log() - torch.log_softmax(fr[:, 64:] / 2, -1).gather(1, idx))).sum()
    want = 0.5 * box / (4 * px) + 2 * cls / px
    want.backward()
    assert abs(scalar.item() - want.item()) <= 1e-5 * abs(want.item())
    assert torch.allclose(items.double().cpu(), torch.stack([box / (4 * px), cls / px]).detach().cpu(), rtol=1e-5)
    for f, l in zip(feats, leaves):
        assert (f.grad.double() - l.grad).abs().max() <= 1e-5 * l.grad.abs().max()
