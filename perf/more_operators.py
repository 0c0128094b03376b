"""The operators that learn from another model's logits and answer with a model's own, measured through the framework's public entry points.

  distill    losses.distill_loss: divergence from a teacher's top logits and what it gave the other classes, loss and gradient of the logits
  top        functional.top_logits: the k largest logits of each row in order, their classes, and the log-sum of the others
  constrain  functional.constrain_logits: penalties for classes chosen before, biases and masks of classes, forward and backward

`listed()` names twelve cases, `draw()` gives more of the same ranges: one row up to tens of thousands, 2 classes up to a large
vocabulary, fp32, bf16 and fp16, contiguous and padded rows.
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}


def listed():
    return [
        # one batch of a ten-class image classifier learns from the three best classes of another: launches are all there is
        {"name": "distill_classes_512x10", "op": "distill", "rows": 512, "classes": 10, "pad": 0, "k": 3, "rest": True, "dtype": "fp32", "teacher": "fp32", "ignored": 0.0,
         "temperature": 2.0},
        # a thousand classes, soft targets at a high temperature
        {"name": "distill_images_8192x1000", "op": "distill", "rows": 8192, "classes": 1000, "pad": 0, "k": 16, "rest": True, "dtype": "fp32", "teacher": "fp32", "ignored": 0.0,
         "temperature": 4.0},
        # tokens of an odd vocabulary in rows padded to whole blocks, prompts ignored, the teacher's list taken for all it knows
        {"name": "distill_padded_2000x50001", "op": "distill", "rows": 2000, "classes": 50001, "pad": 47, "k": 20, "rest": False, "dtype": "fp16", "teacher": "fp16",
         "ignored": 0.1, "temperature": 1.0},
        # a batch of answers over a large vocabulary: the largest of all
        {"name": "distill_tokens_4096x131072", "op": "distill", "rows": 4096, "classes": 131072, "pad": 0, "k": 64, "rest": True, "dtype": "bf16", "teacher": "fp32",
         "ignored": 0.1, "temperature": 1.0},
        # the five best classes of an image classifier
        {"name": "top_classes_512x200", "op": "top", "rows": 512, "classes": 200, "pad": 0, "k": 5, "dtype": "fp32", "masked": 0.0, "temperature": 1.0},
        # one token of a served model: a single long row has to fill the card
        {"name": "top_scored_1x131072", "op": "top", "rows": 1, "classes": 131072, "pad": 0, "k": 50, "dtype": "bf16", "masked": 0.0, "temperature": 0.7},
        # a batch that is served under masks, an odd vocabulary in padded rows
        {"name": "top_served_300x50001", "op": "top", "rows": 300, "classes": 50001, "pad": 47, "k": 200, "dtype": "fp16", "masked": 0.3, "temperature": 1.0},
        # a teacher's lists for a batch of answers
        {"name": "top_teacher_4096x131072", "op": "top", "rows": 4096, "classes": 131072, "pad": 0, "k": 64, "dtype": "bf16", "masked": 0.0, "temperature": 1.0},
        # one token is answered under a grammar, after five hundred others
        {"name": "constrain_step_1x131072", "op": "constrain", "rows": 1, "classes": 131072, "pad": 0, "history": 500, "penalties": "numbers", "bias": "none", "allowed": "bits",
         "dtype": "bf16", "train": False},
        # a batch is answered, each answer with penalties of its own, a bias of its own and a long past
        {"name": "constrain_served_256x50001", "op": "constrain", "rows": 256, "classes": 50001, "pad": 47, "history": 4000, "penalties": "rows", "bias": "rows",
         "allowed": "bits", "dtype": "fp16", "train": False},
        # a small policy learns under a mask of its actions
        {"name": "constrain_actions_4096x1000", "op": "constrain", "rows": 4096, "classes": 1000, "pad": 0, "history": 0, "penalties": "none", "bias": "shared",
         "allowed": "flags", "dtype": "fp32", "train": True},
        # a large batch learns under a grammar, with the penalties that its answers were drawn with
        {"name": "constrain_tokens_4096x65536", "op": "constrain", "rows": 4096, "classes": 65536, "pad": 0, "history": 1024, "penalties": "numbers", "bias": "none",
         "allowed": "bits", "dtype": "bf16", "train": True},
    ]


MOST_LOGITS = 4096 * 131072 // 2    # of a drawn case: below the largest listed ones


def _log_uniform(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("distill", "top", "constrain"))
    dtype = rng.choice(("fp32", "bf16", "fp16"))
    classes = _log_uniform(rng, 2, 131072)
    rows = _log_uniform(rng, 1, max(1, min(32768, MOST_LOGITS // classes)))
    case = {"op": op, "rows": rows, "classes": classes, "pad": rng.choice((0, 0, 1, 47)), "dtype": dtype}
    if op == "distill":
        return dict(case, k=_log_uniform(rng, 1, min(256, classes)), rest=rng.random() < 0.6, teacher=rng.choice(("fp32", dtype)), ignored=rng.choice((0.0, 0.1, 0.5)),
                    temperature=rng.choice((0.5, 1.0, 2.0, 4.0)))
    if op == "top":
        return dict(case, k=_log_uniform(rng, 1, min(256, classes)), masked=rng.choice((0.0, 0.0, 0.3)), temperature=rng.choice((0.7, 1.0, 2.0)))
    penalties = rng.choice(("none", "numbers", "rows"))
    return dict(case, history=_log_uniform(rng, 1, 8192) if penalties != "none" else 0, penalties=penalties, bias=rng.choice(("none", "shared", "rows")),
                allowed=rng.choice(("none", "flags", "bits")), train=rng.random() < 0.5)


# ---- inputs ----------------------------------------------------------------------------------------------------------

REPETITION, PRESENCE, FREQUENCY = 1.2, 0.4, 0.1


def _rows_at_once(classes):
    return max(1, (1 << 26) // classes)


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _logits(g, rows, classes, pad, dtype, also=None):
    """Rows of logits with a spread as trained heads have it, a few classes raised in each; also(first row, logits in fp32) is called with each part."""
    out = torch.empty(rows, classes + pad, device="cuda", dtype=dtype)
    for r in range(0, rows, _rows_at_once(classes + pad)):
        part = out[r:r + _rows_at_once(classes + pad)]
        z = torch.randn(part.shape, generator=g, device="cuda") * 2.5
        raised = torch.randint(0, classes, (z.size(0), 3), generator=g, device="cuda")
        z.scatter_add_(1, raised, 6.0 * torch.rand(raised.shape, generator=g, device="cuda"))
        part.copy_(z)
        if also:
            also(r, part[:, :classes].float())
    return out[:, :classes]


LOSS_SCALE = {"fp32": 1.0, "bf16": 1.0, "fp16": 4096.0}     # fp16 trains with a scaled loss: gradients of a mean would lie below its normal range


def _prepare_distill(case, seed):
    g, dtype = _generator(seed), DTYPES[case["dtype"]]
    rows, classes, k, t = case["rows"], case["classes"], case["k"], case["temperature"]
    values = torch.empty(rows, k, device="cuda", dtype=DTYPES[case["teacher"]])
    chosen = torch.empty(rows, k, device="cuda", dtype=torch.int32)
    rest = torch.empty(rows, device="cuda")

    def teach(r, z):    # another model that mostly agrees
        z = z + 1.2 * torch.randn(z.shape, generator=g, device="cuda")
        top = z.topk(k, dim=1)
        values[r:r + z.size(0)] = top.values
        chosen[r:r + z.size(0)] = top.indices
        rest[r:r + z.size(0)] = torch.logsumexp(z.scatter(1, top.indices, -math.inf) / t, 1)

    logits = _logits(g, rows, classes, case["pad"], dtype, teach)
    if case["ignored"] > 0.0:
        chosen[torch.rand(rows, generator=g, device="cuda") < case["ignored"]] = -1
    return {"case": case, "logits": logits.requires_grad_(), "values": values, "chosen": chosen, "rest": rest if case["rest"] else None}


def _prepare_top(case, seed):
    g = _generator(seed)
    logits = _logits(g, case["rows"], case["classes"], case["pad"], DTYPES[case["dtype"]])
    if case["masked"] > 0.0:    # a grammar has left few classes of some rows
        for r in (torch.rand(case["rows"], generator=g, device="cuda") < case["masked"]).nonzero().view(-1).split(256):
            left = torch.rand(r.numel(), case["classes"], generator=g, device="cuda") * case["classes"] < 30.0
            logits[r] = logits[r].masked_fill(~left, -math.inf)
    return {"case": case, "logits": logits}


def _prepare_constrain(case, seed):
    g, rows, classes = _generator(seed), case["rows"], case["classes"]
    rand = lambda *size: torch.rand(*size, generator=g, device="cuda")
    state = {"case": case, "logits": _logits(g, rows, classes, case["pad"], DTYPES[case["dtype"]]).requires_grad_(case["train"])}
    if case["train"]:
        grad = torch.empty(rows, classes, device="cuda", dtype=DTYPES[case["dtype"]])
        for part in grad.split(_rows_at_once(classes)):
            part.copy_(torch.randn(part.shape, generator=g, device="cuda"))
        state["grad"] = grad
    if case["history"]:     # few classes often, many rarely; buffers of one length, each filled to its own
        state["history"] = (rand(rows, case["history"]).pow_(3) * classes).to(torch.int32).clamp_(max=classes - 1)
        state["lengths"] = torch.randint(case["history"] // 2, case["history"] + 1, (rows,), generator=g, device="cuda", dtype=torch.int32)
    if case["penalties"] == "rows":
        state["repetition"], state["presence"], state["frequency"] = 1.0 + 0.5 * rand(rows), 0.5 * rand(rows), 0.2 * rand(rows)
    elif case["penalties"] == "numbers":
        state["repetition"], state["presence"], state["frequency"] = REPETITION, PRESENCE, FREQUENCY
    if case["bias"] != "none":
        state["bias"] = torch.randn((rows, classes) if case["bias"] == "rows" else (classes,), generator=g, device="cuda")
    if case["allowed"] == "flags":
        state["allowed"] = rand(rows, classes) < 0.6
    elif case["allowed"] == "bits":     # half of the rows may choose anything, the others a class in eight
        words = lambda: torch.randint(-2 ** 31, 2 ** 31, (rows, (classes + 31) // 32), generator=g, device="cuda").to(torch.int32)
        few = words() & words() & words()
        state["allowed"] = torch.where(rand(rows, 1) < 0.5, -1, few)
    return state


def prepare(case, seed):
    return {"distill": _prepare_distill, "top": _prepare_top, "constrain": _prepare_constrain}[case["op"]](case, seed)


# ---- one pass ----------------------------------------------------------------------------------------------------------


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    from sortnet_amd import functional as F
    from sortnet_amd import losses
    case, logits = state["case"], state["logits"]
    if case["op"] == "distill":
        loss, divergences = losses.distill_loss(logits, state["values"], state["chosen"], state["rest"], temperature=case["temperature"],
                                                weight=LOSS_SCALE[case["dtype"]])
        return (loss.detach(), divergences, *torch.autograd.grad(loss, logits))
    if case["op"] == "top":
        return F.top_logits(logits, case["k"], temperature=case["temperature"])
    given = {name: state[name] for name in ("history", "lengths", "repetition", "presence", "frequency", "bias", "allowed") if name in state}
    if not case["train"]:
        with torch.no_grad():
            return (F.constrain_logits(logits, **given),)
    out = F.constrain_logits(logits, **given)
    return (out.detach(), *torch.autograd.grad(out, logits, state["grad"]))


def _plain_distill(state):
    case = state["case"]
    logits, chosen, t = state["logits"].detach(), state["chosen"].long(), case["temperature"]
    rows, classes = logits.shape
    there = chosen >= 0
    at = chosen.clamp(min=0)
    nothing = torch.full((rows, 1), -math.inf, device="cuda", dtype=torch.float64)
    # the teacher's outcomes: its entries and, as one more, all other classes; there are few, in 64 bits
    a = torch.cat((torch.where(there, state["values"].double() / t, -math.inf), nothing if state["rest"] is None else state["rest"].double().view(-1, 1)), 1)
    most = a.amax(1, keepdim=True)
    counted = there.any(1, keepdim=True) & (most > -math.inf)
    weight = (a - most.clamp(min=-1e300)).exp()
    q = weight / weight.sum(1, keepdim=True)
    log_q = q.log()
    # the student's: the others' sum over the row, in 32 bits
    z = logits.float() / t
    listed_ones = torch.zeros(rows, classes + 1, device="cuda", dtype=torch.bool).scatter_(1, torch.where(there, chosen, classes), True)[:, :classes]
    u = z.gather(1, at).double().masked_fill_(~there, -math.inf)
    z.masked_fill_(listed_ones, -math.inf)
    top = z.amax(1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    z.sub_(top).exp_()
    total = z.sum(1, keepdim=True).double()
    u = torch.cat((u, total.log() + top.double()), 1)
    high = u.amax(1, keepdim=True).clamp(min=-1e300)
    log_p = u - high - (u - high).exp().sum(1, keepdim=True).log()
    each = torch.where(q > 0, q * (log_q - log_p), 0.0).sum(1)
    divergences = torch.where(counted.view(-1), each, 0.0)
    scale = LOSS_SCALE[case["dtype"]] * t / counted.sum().clamp(min=1).double()
    slope = torch.where(counted, (log_p.exp() - q) * scale, 0.0)
    z.mul_(torch.where(total > 0, slope[:, -1:] / total, 0.0).float())
    z.masked_fill_(~counted, 0.0)
    z.scatter_add_(1, at, torch.where(there, slope[:, :-1], 0.0).float())
    return (scale * t * divergences.sum()).float(), divergences.float(), z.to(logits.dtype)


def _plain_top(state):
    case, z = state["case"], state["logits"]
    rows, classes = z.shape
    bits = (z.float() + 0.0).view(torch.int32)
    order = bits ^ ((bits >> 31) & 0x7fffffff)      # whole numbers in the order of the values
    del bits
    key = (order.long() << 32) | torch.arange(classes - 1, -1, -1, device="cuda")
    del order
    chosen = classes - 1 - (key.topk(case["k"], dim=1).values & 0xffffffff)
    others = (z.float() / case["temperature"]).scatter_(1, chosen, -math.inf)
    top = others.amax(1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    rest = others.sub_(top).exp_().sum(1).double().log() + top.view(-1).double()
    return z.gather(1, chosen), chosen.to(torch.int32), rest.float()


def _allowed_flags(allowed, classes):
    if allowed.dtype == torch.bool:
        return allowed
    return ((allowed.unsqueeze(-1) >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1).bool().flatten(1)[:, :classes]


def _of_rows(value, dtype=torch.float32):
    return value.to(dtype).view(-1, 1) if isinstance(value, torch.Tensor) else value


def _plain_constrain(state):
    case, logits = state["case"], state["logits"].detach()
    rows, classes = logits.shape
    z = logits.float()
    slope = None
    if case["history"]:
        live = torch.arange(case["history"], device="cuda") < state["lengths"].view(-1, 1)
        count = torch.zeros(rows, classes, device="cuda").scatter_add_(1, state["history"].long(), live.float())
        seen = count > 0
        rep = _of_rows(state["repetition"])
        if case["train"]:
            slope = torch.where(seen, torch.where(z > 0, 1.0 / rep, rep), 1.0)
        z = torch.where(seen, torch.where(z > 0, z / rep, z * rep) - _of_rows(state["frequency"]) * count - _of_rows(state["presence"]), z)
    if case["bias"] != "none":
        z = z + state["bias"]
    flags = _allowed_flags(state["allowed"], classes) if case["allowed"] != "none" else None
    out = (z if flags is None else torch.where(flags, z, -math.inf)).to(logits.dtype)
    if not case["train"]:
        return (out,)
    grad = state["grad"].float()
    if slope is not None:
        grad = grad * slope
    return out, (grad if flags is None else torch.where(flags, grad, 0.0)).to(logits.dtype)


def _run_plain(state):
    return {"distill": _plain_distill, "top": _plain_top, "constrain": _plain_constrain}[state["case"]["op"]](state)


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------


def work(case):
    size, rows, classes = BYTES[case["dtype"]], case["rows"], case["classes"]
    logits = rows * classes
    if case["op"] == "distill":
        kept = rows * (1.0 - case["ignored"])
        return {"bytes": int(kept * classes * size + logits * size + rows * (case["k"] * (4 + BYTES[case["teacher"]]) + 4 * case["rest"] + 4)), "flops": int(8 * kept * classes)}
    if case["op"] == "top":
        return {"bytes": logits * size + rows * (case["k"] * (size + 4) + 4), "flops": 4 * logits}
    per_logit = 2 * size + {"none": 0, "flags": 1, "bits": 0.125}[case["allowed"]] + (4 if case["bias"] == "rows" else 0) + (2 * size if case["train"] else 0)
    small = rows * 3 * case["history"] + (4 * classes if case["bias"] == "shared" else 0) + (12 * rows if case["penalties"] == "rows" else 0)
    return {"bytes": int(logits * per_logit) + small, "flops": (2 if case["train"] else 1) * 2 * logits}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------------


def _exact_distill(state):
    case, t = state["case"], state["case"]["temperature"]
    logits, classes = state["logits"].detach(), state["case"]["classes"]
    counted = (state["chosen"] >= 0).any(1)     # (prepare() gives every such row something finite)
    count, scale = max(1, int(counted.sum())), LOSS_SCALE[case["dtype"]]
    divergences = torch.zeros(case["rows"], device="cuda", dtype=torch.float64)
    grad = torch.zeros(logits.shape, device="cuda", dtype=torch.float64)
    for r in counted.nonzero().view(-1).split(_rows_at_once(classes)):
        z, at = logits[r].double() / t, state["chosen"][r].long()
        mine = torch.log_softmax(z, 1)
        others = torch.ones_like(z, dtype=torch.bool)
        others[torch.arange(r.numel(), device="cuda").view(-1, 1), at] = False
        mine_other = torch.logsumexp(mine.masked_fill(~others, -math.inf), 1, keepdim=True)
        theirs = state["values"][r].double() / t
        if state["rest"] is not None:
            theirs = torch.cat((theirs, state["rest"][r].double().view(-1, 1)), 1)
        theirs = torch.log_softmax(theirs, 1)
        outcomes = torch.cat((mine.gather(1, at), mine_other), 1)[:, :theirs.size(1)]
        share = theirs.exp()
        divergences[r] = torch.where(share > 0, share * (theirs - outcomes), 0.0).sum(1)
        g = mine.exp()
        if state["rest"] is not None:
            within = (mine - mine_other).masked_fill(~others, -math.inf).exp().nan_to_num(0.0)
            g = torch.where(others, within * (mine_other.exp() - share[:, -1:]), g)
        g.scatter_add_(1, at, -share[:, :at.size(1)])
        grad[r] = g * (scale * t / count)
    return scale * t * t * divergences.sum() / count, divergences, grad


def _exact_top(state):
    case, z = state["case"], state["logits"]
    values, chosen, rests = [], [], []
    for part in z.split(max(1, _rows_at_once(case["classes"]) // 4)):
        s = part.double().sort(dim=1, descending=True, stable=True)
        values.append(s.values[:, :case["k"]])
        chosen.append(s.indices[:, :case["k"]].to(torch.int32))
        others = s.values[:, case["k"]:] / case["temperature"]
        rests.append(torch.logsumexp(others, 1) if others.size(1) else torch.full_like(s.values[:, 0], -math.inf))
    return torch.cat(values), torch.cat(chosen), torch.cat(rests)


def _exact_constrain(state):
    case, logits = state["case"], state["logits"].detach()
    rows, classes = logits.shape
    out = torch.empty(rows, classes, device="cuda", dtype=torch.float64)
    grad = torch.empty_like(out) if case["train"] else None
    step = _rows_at_once(classes)
    for r in range(0, rows, step):
        z = logits[r:r + step].double()
        n = z.size(0)
        y, g = z.clone(), state["grad"][r:r + step].double() if case["train"] else None
        if case["history"]:
            past, lengths = state["history"][r:r + step].long(), state["lengths"][r:r + step].long()
            row = torch.arange(n, device="cuda").view(-1, 1).expand_as(past)
            keep = torch.arange(past.size(1), device="cuda").view(1, -1) < lengths.view(-1, 1)
            counts = torch.bincount((row * classes + past)[keep], minlength=n * classes).view(n, classes)
            rep, pres, freq = (v[r:r + step].double().view(-1, 1).expand_as(z) if isinstance(v, torch.Tensor) else torch.full_like(z, v)
                               for v in (state[name] for name in ("repetition", "presence", "frequency")))
            past, factor = counts > 0, torch.where(z > 0, 1.0 / rep, rep)
            y[past] = (z * factor - freq * counts - pres)[past]
            if g is not None:
                g[past] = (g * factor)[past]
        if case["bias"] != "none":
            y += state["bias"][r:r + step] if case["bias"] == "rows" else state["bias"]
        if case["allowed"] != "none":
            allowed = state["allowed"][r:r + step]
            if case["allowed"] == "bits":
                column = torch.arange(classes, device="cuda")
                allowed = (allowed[:, column // 32].long() >> (column % 32)) & 1 == 1
            y.masked_fill_(~allowed, -math.inf)
            if g is not None:
                g.masked_fill_(~allowed, 0.0)
        out[r:r + step] = y
        if g is not None:
            grad[r:r + step] = g
    return (out,) if grad is None else (out, grad)


def exact(case, seed):
    return {"distill": _exact_distill, "top": _exact_top, "constrain": _exact_constrain}[case["op"]](prepare(case, seed))
