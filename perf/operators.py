"""What is measured of the losses over a large class list: the linear class projection fused with softmax cross entropy, the same projection fused
with distillation from a teacher's top logits, and that distillation on logits that are in memory already (the head's own maps).

Shapes: N rows (anchors or regions that were assigned an object), d features each, V classes, k teacher logits a row."""
import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}

#: rows x classes x features of the largest listed case; a drawn case stays below it
_MOST = 8192 * 131072 * 1024


def listed():
    return [
        # -- linear_ce: class projection + softmax cross entropy, logits never in memory ------------------------------------------------------
        # one region scored against a list of class embeddings: a query, where latency counts
        {"name": "ce-score-1x32768x512", "op": "ce", "N": 1, "V": 32768, "d": 512, "dtype": "bf16", "grad": False, "offset": False, "ignored": 0.0},
        # every anchor of one 640-pixel image against a long class list, validation (no gradient); d is the class branch's width in the x-large head
        {"name": "ce-score-8400x1203x320", "op": "ce", "N": 8400, "V": 1203, "d": 320, "dtype": "f16", "grad": False, "offset": True, "ignored": 0.0},
        # a training step on the assigned anchors of a small batch: odd sizes, class priors and left-out classes, ignored rows, fp16 with a loss scale
        {"name": "ce-train-997x1201x320", "op": "ce", "N": 997, "V": 1201, "d": 320, "dtype": "f16", "grad": True, "offset": True, "ignored": 0.1},
        # an ordinary training step over an open class list
        {"name": "ce-train-2048x20000x512", "op": "ce", "N": 2048, "V": 20000, "d": 512, "dtype": "bf16", "grad": True, "offset": False, "ignored": 0.05},
        # the largest: a batch of 32 images' assigned anchors over a vocabulary; the logits alone would be 4.3 GB in 32 bits
        {"name": "ce-train-8192x131072x1024", "op": "ce", "N": 8192, "V": 131072, "d": 1024, "dtype": "bf16", "grad": True, "offset": False, "ignored": 0.05},
        # -- linear_distill: the same projection against a teacher's top k -------------------------------------------------------------------
        # a small task head, few anchors
        {"name": "kd-train-96x365x320", "op": "kd", "N": 96, "V": 365, "d": 320, "k": 16, "dtype": "f16", "grad": True, "offset": False, "empty": 0.1, "tau": 2.0},
        # ragged everything; some of the teacher's slots are empty
        {"name": "kd-train-1021x32003x512", "op": "kd", "N": 1021, "V": 32003, "d": 512, "k": 50, "dtype": "bf16", "grad": True, "offset": True, "empty": 0.1, "tau": 2.0},
        # a batch's assigned anchors over a vocabulary
        {"name": "kd-train-4096x65536x640", "op": "kd", "N": 4096, "V": 65536, "d": 640, "k": 64, "dtype": "bf16", "grad": True, "offset": False, "empty": 0.0, "tau": 1.0},
        # -- topk_distill: logits in memory, loss and gradient in one call --------------------------------------------------------------------
        # one image's coarsest map, class logits of the head as it stores them (64 box bins | classes, one pixel after the other)
        {"name": "map-400x80", "op": "map", "N": 400, "V": 80, "k": 10, "groups": 1, "before": 64, "dtype": "f32", "empty": 0.1, "tau": 2.0},
        # the box bins of a batch of 32: four distributions of 16 bins a pixel, the teacher's whole distribution (k = 16)
        {"name": "map-268800x4x16", "op": "map", "N": 268800, "V": 16, "k": 16, "groups": 4, "before": 0, "after": 80, "dtype": "f32", "empty": 0.0, "tau": 4.0},
        # class logits of a batch of 8 over a long class list
        {"name": "map-67200x1203", "op": "map", "N": 67200, "V": 1203, "k": 32, "groups": 1, "before": 64, "after": 5, "dtype": "f32", "empty": 0.1, "tau": 2.0},
        # rows over a vocabulary, 16-bit
        {"name": "map-4096x131072", "op": "map", "N": 4096, "V": 131072, "k": 64, "groups": 1, "before": 0, "dtype": "bf16", "empty": 0.0, "tau": 1.0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("ce", "kd", "map"))
    if op == "map":
        groups = rng.choice((1, 1, 4))
        V = _log(rng, 16, 131072 if groups == 1 else 64)
        N = min(_log(rng, 1, 268800), max(1, 4096 * 131072 // (2 * V * groups)))
        return {"op": op, "N": N, "V": V, "k": min(V, _log(rng, 1, 128)), "groups": groups, "before": rng.choice((0, 3, 64)), "after": rng.choice((0, 5, 80)),
                "dtype": rng.choice(("f32", "bf16", "f16")), "empty": rng.choice((0.0, 0.1)), "tau": rng.choice((1.0, 2.0, 4.0))}
    d = 8 * _log(rng, 8, 128)
    V = _log(rng, 64, 131072)
    N = min(_log(rng, 1, 8192), max(1, _MOST // (V * d)))
    case = {"op": op, "N": N, "V": V, "d": d, "dtype": rng.choice(("bf16", "f16")), "grad": rng.random() < 0.75, "offset": rng.random() < 0.5}
    if op == "ce":
        return {**case, "ignored": rng.choice((0.0, 0.1))}
    return {**case, "k": min(V, _log(rng, 1, 128)), "empty": rng.choice((0.0, 0.1)), "tau": rng.choice((1.0, 2.0))}


def _teacher(gen, rows, V, k, empty):
    """A teacher's top k of every row: distinct classes, falling logits; of `empty` of the rows the last slots hold none (index -1), of some all."""
    first = torch.randint(V, (rows, 1), generator=gen, device="cuda")
    idx = (first + torch.randperm(V, generator=gen, device="cuda")[:k]) % V
    val = (3 * torch.randn(rows, k, generator=gen, device="cuda") + 4).sort(dim=1, descending=True).values
    if empty:
        kept = torch.where(torch.rand(rows, 1, generator=gen, device="cuda") < empty, torch.randint(k + 1, (rows, 1), generator=gen, device="cuda"), k)
        idx = torch.where(torch.arange(k, device="cuda") < kept, idx, -1)
    return idx.int(), val


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    N, V, dt = case["N"], case["V"], _DT[case["dtype"]]
    s = dict(case)
    if case["op"] == "map":
        G, lead, k = case["groups"], case["before"], case["k"]
        ld = lead + G * V + case.get("after", 0)
        full = torch.randn(N, ld, generator=gen, device="cuda", dtype=torch.float32 if dt == torch.float32 else dt).mul_(2.5)
        s["logits"] = full[:, lead:lead + G * V].unflatten(1, (G, V)) if G > 1 else full[:, lead:lead + V]
        idx, val = _teacher(gen, N * G, V, k, case["empty"])
        s["idx"], s["val"] = (idx.view(N, G, k), val.view(N, G, k)) if G > 1 else (idx, val)
        s["drow"] = torch.rand(N * G, generator=gen, device="cuda").add_(0.5).view(s["idx"].shape[:-1])  # per-row weights: the assignment's scores
        return s
    d = case["d"]
    w = torch.randn(V, d, generator=gen, device="cuda").mul_(2 / math.sqrt(d))
    label = torch.randint(V, (N,), generator=gen, device="cuda")
    # a model that has learned something: the features lean towards their class
    s["x"] = (torch.randn(N, d, generator=gen, device="cuda") + 3 * torch.nn.functional.normalize(w[label], dim=1)).to(dt)
    s["w"] = w.to(dt)
    s["off"] = None
    if case["offset"]:  # class priors, and one class in 50 that this data set does not annotate
        off = torch.randn(V, generator=gen, device="cuda")
        off[torch.rand(V, generator=gen, device="cuda") < 0.02] = -math.inf
        off[label] = off[label].clamp(min=-3.0)
        s["off"] = off
    if case["op"] == "ce":
        s["label"] = torch.where(torch.rand(N, generator=gen, device="cuda") < case["ignored"], -100, label)
    else:
        s["idx"], s["val"] = _teacher(gen, N, V, case["k"], case["empty"])
        if s["off"] is not None:
            s["off"] = s["off"].clamp(min=-3.0)
    # gradient of the mean loss, times the loss scale that fp16 training runs with
    s["drow"] = torch.full((N,), (1024.0 if dt == torch.float16 else 1.0) / N, device="cuda")
    return s


def _soft_teacher(idx, val, tau):
    """q [.., k] over the slots that hold a class, log q with zeros where q is zero, and which rows hold any."""
    t = torch.where(idx >= 0, val.float() / tau, -math.inf)
    some = (idx >= 0).any(-1)
    t = torch.where(some[..., None], t, 0.0)
    logq = torch.log_softmax(t, -1)
    q = torch.where(idx >= 0, logq.exp(), 0.0)
    return q, torch.where(q > 0, logq, 0.0), some


def _plain_linear(s):
    x, w = s["x"].float(), s["w"].float()
    tau = s.get("tau", 1.0)
    z = x @ w.T
    if s["off"] is not None:
        z += s["off"]
    if tau != 1.0:
        z /= tau
    lse = torch.logsumexp(z, 1)
    if s["op"] == "ce":
        some = s["label"] >= 0
        at, q = s["label"].clamp(min=0)[:, None], some.float()[:, None]
        loss = torch.where(some, lse - z.gather(1, at)[:, 0], 0.0)
        out = {"loss": loss, "lse": lse}
    else:
        q, logq, some = _soft_teacher(s["idx"], s["val"], tau)
        at = s["idx"].clamp(min=0).long()
        out = {"loss": tau * tau * (q * (logq - z.gather(1, at) + lse[:, None])).sum(1)}
    if not s["grad"]:
        return out
    g = torch.where(some, s["drow"] * tau, 0.0)[:, None]
    dz = z.sub_(lse[:, None]).exp_().mul_(g).scatter_add_(1, at, -q * g)
    return {**out, "dx": (dz @ w).to(s["x"].dtype), "dw": (dz.T @ x).to(s["w"].dtype)}


def _plain_map(s):
    tau = s["tau"]
    z = s["logits"].float() / tau
    lse = torch.logsumexp(z, -1, keepdim=True)
    q, logq, some = _soft_teacher(s["idx"], s["val"], tau)
    at = s["idx"].clamp(min=0).long()
    loss = tau * tau * (q * (logq - z.gather(-1, at) + lse)).sum(-1)
    g = torch.where(some, s["drow"] * tau, 0.0)[..., None]
    dz = (z - lse).exp_().mul_(g).scatter_add_(-1, at, -q * g)
    return {"loss": loss, "dlogits": dz.to(s["logits"].dtype)}


def _own_pass(s):
    from cerberusdet_amd import ops

    if s["op"] == "ce":
        loss, lse = ops.linear_ce_fwd(s["x"], s["w"], s["label"], offset=s["off"])
        out = {"loss": loss, "lse": lse}
        if s["grad"]:
            out["dx"], out["dw"] = ops.linear_ce_bwd(s["x"], s["w"], s["label"], lse, s["drow"], offset=s["off"])
        return out
    if s["op"] == "kd":
        loss, saved = ops.linear_distill_fwd(s["x"], s["w"], s["idx"], s["val"], tau=s["tau"], offset=s["off"])
        out = {"loss": loss}
        if s["grad"]:
            out["dx"], out["dw"] = ops.linear_distill_bwd(s["x"], s["w"], s["idx"], saved, s["drow"], tau=s["tau"], offset=s["off"])
        return out
    loss, dlogits = ops.topk_distill(s["logits"], s["idx"], s["val"], tau=s["tau"], drow=s["drow"])
    return {"loss": loss, "dlogits": dlogits}


def run(state):
    if own:
        return _own_pass(state)
    return _plain_map(state) if state["op"] == "map" else _plain_linear(state)


def work(case):
    N, V = case["N"], case["V"]
    e = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "map":
        rows = N * case["groups"]
        # logits read, gradient written, the teacher's indexes and logits, row weights and losses; an exp, a subtraction and two products a logit
        return {"bytes": rows * (2 * V * e + 8 * case["k"] + 8), "flops": 5 * rows * V}
    d = case["d"]
    targets = N * 8 if case["op"] == "ce" else N * case["k"] * 8
    once = (N + V) * d * e
    return {"bytes": once * (2 if case["grad"] else 1) + targets + 12 * N + (4 * V if case["offset"] else 0), "flops": 2 * N * V * d * (3 if case["grad"] else 1)}


def exact(case, seed):
    """The definitions, in 64 bits, with the gradients that differentiation of the loss gives."""
    s = prepare(case, seed)
    tau = case.get("tau", 1.0)
    if case["op"] == "map":
        leaf = s["logits"].double().detach().requires_grad_()
        z = leaf
    else:
        x, w = s["x"].double().requires_grad_(), s["w"].double().requires_grad_()
        z = torch.matmul(x, w.t())
        if s["off"] is not None:
            z = z + s["off"].double()
    logp = torch.nn.functional.log_softmax(z / tau, dim=-1)
    if case["op"] == "ce":
        rows = torch.nn.functional.nll_loss(logp, s["label"], ignore_index=-100, reduction="none")
    else:
        held = s["idx"].ge(0)
        teacher = torch.exp(s["val"].double() / tau - (s["val"].double() / tau).amax(-1, keepdim=True)) * held
        teacher = teacher / teacher.sum(-1, keepdim=True).clamp_min(1e-300)
        cross = torch.special.xlogy(teacher, teacher) - teacher * logp.gather(-1, s["idx"].long() * held)
        rows = cross.sum(-1) * tau ** 2
    with torch.no_grad():
        out = {"loss": rows.detach()}
        if case["op"] == "ce":
            out["lse"] = torch.logsumexp(z, dim=1)
    if case["op"] == "map":
        rows.mul(s["drow"].double()).sum().backward()
        out["dlogits"] = leaf.grad
    elif case["grad"]:
        rows.mul(s["drow"].double()).sum().backward()
        out["dx"], out["dw"] = x.grad, w.grad
    return out
