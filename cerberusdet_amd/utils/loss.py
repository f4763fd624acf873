"""`Loss` with the reference's interface (ai-forever/CerberusDet cerberusdet/utils/loss.py:48-181):
`Loss(model, task_ids)`; `loss(preds, batch, task) -> (scalar, items[4])` where scalar = 2*bs*(box+cls+dfl) [sic,
loss.py:179-181]. The whole computation -- anchors, DFL decode, task-aligned assignment, BCE, CIoU, DFL and the gradient
w.r.t. the head maps -- is one call into csrc/det_loss.hip; autograd sees a single node."""
from __future__ import annotations

import math

import torch

from .torch_utils import get_hyperparameter


def pad_targets(batch, batch_size, imgsz_hw, device, n_max=None, dropped=None):
    """Loss.preprocess (reference loss.py:111-124) as ONE kernel (csrc/det_loss.hip, cdet_pad_targets):
    labels [n] -> gt [bs, n_max, 5] (cls, x1, y1, x2, y2 in pixels), zero rows = padding, file order kept inside an image.
    n_max=None: sized from the batch like the reference (`counts.max()`, loss.py:117 -- one host sync). With n_max given there is
    no sync; a label that does not fit is dropped and counted in `dropped` (device int32[1]) -- the trainer checks it at its
    once-per-iteration sync, so an undersized n_max fails loudly instead of corrupting targets."""
    import ctypes as C

    from .. import _lib as L
    from ..ops import ptr, stream

    device = torch.device(device)
    if device.type != "cuda":
        raise RuntimeError("cerberusdet_amd.pad_targets runs on the MI355X only (there is no CPU path)")
    bi = batch["batch_idx"].to(device=device, dtype=torch.float32).reshape(-1).contiguous()
    n = bi.numel()
    if n_max is None:
        n_max = int(torch.bincount(bi.long(), minlength=batch_size).max()) if n else 0
    n_max = max(int(n_max), 1)
    cls = batch["cls"].to(device=device, dtype=torch.float32).reshape(-1).contiguous()
    box = batch["bboxes"].to(device=device, dtype=torch.float32).reshape(-1, 4).contiguous()
    out = torch.empty(batch_size, n_max, 5, device=device)
    h, w = imgsz_hw
    lib = L.load()
    L.check(lib.cdet_pad_targets(ptr(bi), ptr(cls), ptr(box), n, batch_size, n_max, float(w), float(h), ptr(out), ptr(dropped), stream()),
            "cdet_pad_targets")
    return out


class _DetLossFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gt, nc, gains, strides, f0, f1, f2):
        from .. import ops

        feats = [f.permute(0, 2, 3, 1).contiguous().float() for f in (f0, f1, f2)]  # NHWC fp32 (no-op for plan buffers' layout)
        loss5, dfe, _ = ops.det_loss(feats, gt, nc, gains, strides, grad_scale=1.0, grad_dtype=torch.float32)
        ctx.dfe = dfe
        return loss5[4].clone(), loss5[:4].clone()

    @staticmethod
    def backward(ctx, g_scalar, g_items):
        grads = [d.permute(0, 3, 1, 2) * g_scalar for d in ctx.dfe]
        return None, None, None, None, grads[0], grads[1], grads[2]


class Loss:
    def __init__(self, model, task_ids):
        h = model.hyp
        self.device = next(model.parameters()).device
        self.stride, self.reg_max = None, None
        self.nc, self.no, self.loss_weights = {}, {}, {}
        for task_idx, task in enumerate(task_ids):
            self.loss_weights[task] = dict(box=get_hyperparameter(h, "box", task_idx, task), dfl=get_hyperparameter(h, "dfl", task_idx, task),
                                           cls=get_hyperparameter(h, "cls", task_idx, task))
        for task_name in model.heads:
            head = model.get_head(task_name)
            self.nc[task_name], self.no[task_name] = head.nc, head.no
            assert self.reg_max in (None, head.reg_max)
            self.reg_max = head.reg_max
            assert self.stride is None or torch.equal(self.stride, head.stride)
            self.stride = head.stride
        self.use_dfl = self.reg_max > 1

    def __call__(self, preds, batch, task):
        feats = preds[1] if isinstance(preds, tuple) else preds
        bs = feats[0].shape[0]
        imgsz = (feats[0].shape[2] * float(self.stride[0]), feats[0].shape[3] * float(self.stride[0]))
        gt = pad_targets(batch, bs, imgsz, feats[0].device)
        scalar, items = _DetLossFn.apply(gt, self.nc[task], self.loss_weights[task], [float(s) for s in self.stride], *feats)
        return scalar, items.detach()


# ---- losses over a long class list and from a teacher (csrc/class_loss.hip, csrc/topk_distill.hip) -----------------------------------------------------
def _reduced(rows, counted, reduction):
    if reduction == "none":
        return rows
    if reduction == "sum":
        return rows.sum()
    if reduction == "mean":  # over the rows that take part
        return rows.sum() / counted.sum().clamp(min=1)
    raise ValueError(f"reduction must be 'none', 'sum' or 'mean', got {reduction!r}")


class _LinearCeFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, labels, offset, scale):
        from .. import ops

        loss, lse = ops.linear_ce_fwd(x, w, labels, offset=offset, scale=scale)
        ctx.save_for_backward(x, w, labels, offset, lse)
        ctx.scale = scale
        ctx.mark_non_differentiable(lse)
        return loss, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g, _):
        from .. import ops

        x, w, labels, offset, lse = ctx.saved_tensors
        dx, dw = ops.linear_ce_bwd(x, w, labels, lse, g.float(), offset=offset, scale=ctx.scale, want_dx=ctx.needs_input_grad[0], want_dw=ctx.needs_input_grad[1])
        return dx, dw, None, None, None


class _LinearDistillFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, idx, val, tau, offset, scale):
        from .. import ops

        loss, saved = ops.linear_distill_fwd(x, w, idx, val, tau=tau, offset=offset, scale=scale)
        ctx.save_for_backward(x, w, idx, offset, saved)
        ctx.tau, ctx.scale = tau, scale
        ctx.mark_non_differentiable(saved)
        return loss, saved

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g, _):
        from .. import ops

        x, w, idx, offset, saved = ctx.saved_tensors
        dx, dw = ops.linear_distill_bwd(x, w, idx, saved, g.float(), tau=ctx.tau, offset=offset, scale=ctx.scale, want_dx=ctx.needs_input_grad[0],
                                        want_dw=ctx.needs_input_grad[1])
        return dx, dw, None, None, None, None, None


# fp32 logits of a map whose gradient is made in the forward (forward and backward of 67200 x 250: 142 us, 180 the other way, of x 500 152 and 179, of x 700 196
# and 181, of x 1203 299 and 269; 4096 x 131072 bf16, always in the backward, 775 us, ahead 1658)
_AHEAD = 1 << 25


class _TopkDistillFn(torch.autograd.Function):
    """The gradient is made in the backward, from the logits: rounded once, behind the incoming gradient -- a 16-bit one made ahead has lost what a loss scale
    lifts into fp16's range -- and never kept or multiplied as a map. Small fp32 maps, bound by the host, have it made in the forward's one call and multiplied."""

    @staticmethod
    def forward(ctx, logits, idx, val, tau, ahead, part):
        from .. import ops

        ctx.tau = tau
        loss, ctx.dz = ops.topk_distill(logits, idx, val, tau=tau, want_grad=ahead, part=part)
        if not ahead:
            ctx.save_for_backward(logits, idx, val)
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        if ctx.dz is not None:
            return ctx.dz * g[..., None], None, None, None, None, None
        from .. import ops

        logits, idx, val = ctx.saved_tensors
        return ops.topk_distill(logits, idx, val, tau=ctx.tau, drow=g.float())[1], None, None, None, None, None


def linear_cross_entropy(x, w, labels, offset=None, scale=1.0, reduction="mean"):
    """Cross entropy of a linear classifier over a long class list, differentiable in x [N, d] and w [V, d] (bf16 / fp16); the N x V logits are never in
    memory. Labels outside of 0 .. V-1 leave their row out; "mean" is over the rows that take part. See ops.linear_ce_fwd."""
    loss, lse = _LinearCeFn.apply(x, w, labels, offset, float(scale))
    return _reduced(loss, (labels.clamp(0, w.shape[0] - 1) == labels) & (lse != -math.inf), reduction)


def linear_distillation(x, w, idx, val, tau=1.0, offset=None, scale=1.0, reduction="mean"):
    """Distillation of that classifier from a teacher's top k logits (idx [N, k] int32, val [N, k]), differentiable in x and w. See ops.linear_distill_fwd."""
    loss, saved = _LinearDistillFn.apply(x, w, idx, val, float(tau), offset, float(scale))
    return _reduced(loss, saved[:, 0] != math.inf, reduction)  # (the forward's mark of a row that takes no part)


def topk_distillation(logits, idx, val, tau=1.0, reduction="mean"):
    """Distillation of logits [P, V] or [P, G, V] in memory from a teacher's top k, differentiable in the logits, which the backward reads again. See
    ops.topk_distill."""
    ahead = logits.dtype == torch.float32 and logits.numel() <= _AHEAD and logits.requires_grad and torch.is_grad_enabled()
    part = torch.empty(logits.shape[:-1], dtype=torch.bool, device=logits.device) if reduction == "mean" else None
    loss = _TopkDistillFn.apply(logits, idx, val, float(tau), ahead, part)
    return _reduced(loss, part, reduction)


class HeadDistillation:
    """Distillation of a task's Detect head from a teacher's head maps of the same strides: `HeadDistillation(model, k, tau)(preds, teacher_preds, task)` ->
    (scalar, items[2]), items = (box, cls). Box: the four reg_max-bin distributions of every pixel against the teacher's; cls: the class logits against the
    teacher's k largest. Both are means over the pixels of all maps (box: and their four distributions), weighted by `box` and `cls`. preds: three NCHW maps
    as Loss takes them (the model's NHWC buffers are read in place)."""

    def __init__(self, model, k=16, tau=2.0, box=1.0, cls=1.0):
        self.k, self.tau, self.box, self.cls = int(k), float(tau), float(box), float(cls)
        self.reg_max = {t: model.get_head(t).reg_max for t in model.heads}
        self.nc = {t: model.get_head(t).nc for t in model.heads}

    def __call__(self, preds, teacher_preds, task):
        feats = preds[1] if isinstance(preds, tuple) else preds
        teach = teacher_preds[1] if isinstance(teacher_preds, tuple) else teacher_preds
        R, nc, items = self.reg_max[task], self.nc[task], []
        for part in (0, 1):
            total, count = 0.0, 0
            for f, t in zip(feats, teach):
                if f.shape != t.shape:
                    raise ValueError(f"student and teacher maps differ: {tuple(f.shape)} and {tuple(t.shape)}")
                fr, tr = (m.permute(0, 2, 3, 1) for m in (f, t.detach()))  # NHWC
                n = fr.shape[0] * fr.shape[1] * fr.shape[2]
                if part == 0:
                    z, tz = (m[..., :4 * R].reshape(n, 4 * R).unflatten(1, (4, R)) for m in (fr, tr))
                else:
                    z, tz = (m[..., 4 * R:4 * R + nc].reshape(n, nc) for m in (fr, tr))
                val, idx = tz.topk(R if part == 0 else min(self.k, nc), dim=-1)
                total = total + topk_distillation(z, idx.int(), val, self.tau, reduction="sum")
                count += idx[..., 0].numel()
            items.append(total / count)
        return self.box * items[0] + self.cls * items[1], torch.stack(items).detach()
