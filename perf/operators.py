"""The operators that train a head's logits, measured through the framework's public entry points.

  label       losses.label_log_probs: log probability of the label of each row of logits, and its gradient
  preference  losses.preference_loss: paired answers, chosen against rejected, loss and gradient of the logits
  policy      losses.policy_loss: clipped policy loss with a KL term, loss and gradient of the logits
  dropout     functional.dropout / bound_dropout: dropout from the counter generator, forward and backward

`listed()` names twelve cases, `draw()` gives more of the same ranges: one row up to tens of thousands, 2 classes up to a large
vocabulary, fp32, bf16 and fp16, contiguous and padded rows.
"""
import math

import numpy as np
import torch

own = False

IGNORE = -100
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}


def listed():
    return [
        # one batch of a ten-class image classifier, forward and backward: launches are all there is
        {"name": "label_classes_512x10", "op": "label", "rows": 512, "classes": 10, "pad": 0, "dtype": "fp32", "ignored": 0.0, "train": True},
        # one token of a served model is scored: a single long row has to fill the card
        {"name": "label_scored_1x131072", "op": "label", "rows": 1, "classes": 131072, "pad": 0, "dtype": "bf16", "ignored": 0.0, "train": False},
        # tokens of an odd vocabulary in rows padded to whole blocks, a tenth of them prompt
        {"name": "label_padded_2000x50001", "op": "label", "rows": 2000, "classes": 50001, "pad": 47, "dtype": "fp16", "ignored": 0.1, "train": True},
        # answers of one label each, 200 classes: preferences over the predictions of an image classifier
        {"name": "preference_classes_256x200", "op": "preference", "pairs": 128, "tokens": 1, "packed": False, "classes": 200, "dtype": "fp32", "ignored": 0.0, "smoothing": 0.1},
        # answers of uneven length, packed one behind the other, with their prompts ignored
        {"name": "preference_packed_24x32000", "op": "preference", "pairs": 24, "tokens": 150, "packed": True, "classes": 32000, "dtype": "bf16", "ignored": 0.3, "smoothing": 0.0},
        # a padded batch of pairs over a large vocabulary
        {"name": "preference_padded_8x256x65536", "op": "preference", "pairs": 8, "tokens": 256, "packed": False, "classes": 65536, "dtype": "bf16", "ignored": 0.2, "smoothing": 0.0},
        # a small policy over ten actions
        {"name": "policy_actions_256x10", "op": "policy", "answers": 256, "tokens": 1, "classes": 10, "dtype": "fp32", "ignored": 0.0, "kl": 0.0, "shared": False},
        # a batch of states and a thousand actions, with the KL term
        {"name": "policy_actions_4096x1000", "op": "policy", "answers": 4096, "tokens": 1, "classes": 1000, "dtype": "fp32", "ignored": 0.0, "kl": 0.05, "shared": False},
        # answers sampled from a large vocabulary, one advantage per answer: the largest of all
        {"name": "policy_tokens_8x512x131072", "op": "policy", "answers": 8, "tokens": 512, "classes": 131072, "dtype": "bf16", "ignored": 0.1, "kl": 0.02, "shared": True},
        # values, lower and upper bounds of a dense head of 512 features under one mask
        {"name": "dropout_box_512x512", "op": "dropout", "rows": 512, "features": 512, "box": True, "dtype": "fp32", "q": 0.9},
        # an odd size in half precision
        {"name": "dropout_odd_1001x2047", "op": "dropout", "rows": 1001, "features": 2047, "box": False, "dtype": "fp16", "q": 0.5},
        # long rows of activations
        {"name": "dropout_long_8192x16384", "op": "dropout", "rows": 8192, "features": 16384, "box": False, "dtype": "bf16", "q": 0.85},
    ]


MOST_LOGITS = 4096 * 131072 // 2    # of a drawn case: below the largest listed one


def _log_uniform(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("label", "preference", "policy", "dropout"))
    dtype = rng.choice(("fp32", "bf16", "fp16"))
    if op == "dropout":
        features = _log_uniform(rng, 1, 16384)
        rows = _log_uniform(rng, 1, min(65536, max(2, (1 << 26) // features)))
        return {"op": op, "rows": rows, "features": features, "box": rng.random() < 0.4, "dtype": dtype, "q": round(rng.uniform(0.05, 0.98), 3)}
    classes = _log_uniform(rng, 2, 131072)
    most = max(2, min(32768, MOST_LOGITS // classes))
    ignored = rng.choice((0.0, 0.1, 0.5))
    if op == "label":
        return {"op": op, "rows": _log_uniform(rng, 1, most), "classes": classes, "pad": rng.choice((0, 0, 1, 47)), "dtype": dtype, "ignored": ignored,
                "train": rng.random() < 0.7}
    if op == "preference":
        tokens = _log_uniform(rng, 1, max(1, min(1024, most // 2)))
        return {"op": op, "pairs": _log_uniform(rng, 1, max(1, min(256, most // (2 * tokens)))), "tokens": tokens, "packed": rng.random() < 0.5,
                "classes": classes, "dtype": dtype, "ignored": ignored, "smoothing": rng.choice((0.0, 0.1))}
    tokens = _log_uniform(rng, 1, min(2048, most))
    return {"op": op, "answers": _log_uniform(rng, 1, max(1, min(4096, most // tokens))), "tokens": tokens, "classes": classes, "dtype": dtype,
            "ignored": ignored, "kl": rng.choice((0.0, 0.02, 0.1)), "shared": rng.random() < 0.5}


# ---- inputs ----------------------------------------------------------------------------------------------------------

BETA, CLIP_LOW, CLIP_HIGH = 0.1, 0.2, 0.28


def _rows_at_once(classes):
    return max(1, (1 << 26) // classes)


def _logits(g, labels, rows, classes, pad, dtype):
    """Rows of logits with a spread as trained heads have it, the label's own raised in most rows."""
    out = torch.empty(rows, classes + pad, device="cuda", dtype=dtype)
    for r in range(0, rows, _rows_at_once(classes + pad)):
        part = out[r:r + _rows_at_once(classes + pad)]
        z = torch.randn(part.shape, generator=g, device="cuda") * 2.5
        at = labels[r:r + part.size(0)].clamp(min=0).view(-1, 1)
        z.scatter_add_(1, at, 6.0 * (torch.rand(at.shape, generator=g, device="cuda") < 0.8).float())
        part.copy_(z)
    return out[:, :classes]


def _model_log_probs(logits, labels):
    """What a program has kept of another model's pass: log probabilities of the labels, in fp32."""
    parts = []
    for r in range(0, logits.size(0), _rows_at_once(logits.size(1))):
        z = logits[r:r + _rows_at_once(logits.size(1))].float()
        at = labels[r:r + z.size(0)].clamp(min=0).view(-1, 1)
        parts.append(torch.log_softmax(z, 1).gather(1, at).squeeze(1))
    return torch.cat(parts)


def _labels(g, rows, classes, ignored):
    labels = torch.randint(0, classes, (rows,), generator=g, device="cuda")
    if ignored > 0.0:
        labels[torch.rand(rows, generator=g, device="cuda") < ignored] = IGNORE
    return labels


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, dtype = case["op"], DTYPES[case["dtype"]]
    randn = lambda *size: torch.randn(*size, generator=g, device="cuda")
    if op == "dropout":
        size = (case["rows"], case["features"])
        count = 3 if case["box"] else 1
        x = [randn(*size) for _ in range(count)]
        if case["box"]:     # values between their bounds
            x = [x[0], x[0] - x[1].abs() * 0.1, x[0] + x[2].abs() * 0.1]
        return {"case": case, "x": [t.to(dtype).requires_grad_() for t in x], "grad": [randn(*size).to(dtype) for _ in range(count)],
                "seed": seed * 2654435761 % (1 << 32)}
    classes = case["classes"]
    if op == "label":
        labels = _labels(g, case["rows"], classes, case["ignored"])
        logits = _logits(g, labels, case["rows"], classes, case["pad"], dtype)
        return {"case": case, "logits": logits.requires_grad_(case["train"]), "labels": labels, "grad": randn(case["rows"])}
    if op == "preference":
        answers, tokens = 2 * case["pairs"], case["tokens"]
        state = {"case": case}
        if case["packed"]:
            lengths = torch.randint(0, tokens + 1, (answers,), generator=g, device="cuda")
            lengths[0] = tokens
            rows = _most_rows(case) + 3         # the buffer's size is fixed; the last answers are cut, or rows stand behind them
            state["offsets"] = torch.zeros(answers + 1, device="cuda", dtype=torch.int32)
            state["offsets"][1:] = lengths.cumsum(0).clamp(max=rows - 3)
            shape = (rows,)
        else:
            shape = (answers, tokens)
            rows = answers * tokens
        labels = _labels(g, rows, classes, case["ignored"])
        logits = _logits(g, labels, rows, classes, 0, dtype)
        ref = _model_log_probs(logits, labels) + 0.3 * randn(rows)
        state.update(logits=logits.view(*shape, classes).requires_grad_(), labels=labels.view(shape), ref=ref.view(shape))
        return state
    shape = (case["answers"], case["tokens"])
    rows = shape[0] * shape[1]
    labels = _labels(g, rows, classes, case["ignored"])
    logits = _logits(g, labels, rows, classes, 0, dtype)
    now = _model_log_probs(logits, labels)
    moved = 0.2 * randn(rows)
    for border in (math.log(1 - CLIP_LOW), math.log(1 + CLIP_HIGH)):    # the loss has no derivative on the clip's borders
        moved = torch.where((moved - border).abs() < 1e-3, moved + 3e-3, moved)
    advantages = randn(shape[0], 1) if case["shared"] else randn(*shape)
    return {"case": case, "logits": logits.view(*shape, classes).requires_grad_(), "labels": labels.view(shape), "old": (now - moved).view(shape),
            "ref": (now + 0.3 * randn(rows)).view(shape) if case["kl"] else None, "advantages": advantages.expand(shape)}


# ---- one pass ----------------------------------------------------------------------------------------------------------


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    from sortnet_amd import functional as F
    from sortnet_amd import losses
    case = state["case"]
    op = case["op"]
    if op == "label":
        logits = state["logits"]
        if not case["train"]:
            with torch.no_grad():
                return (losses.label_log_probs(logits, state["labels"]),)
        values = losses.label_log_probs(logits, state["labels"])
        return (values.detach(), *torch.autograd.grad(values, logits, state["grad"]))
    if op == "preference":
        loss, rewards = losses.preference_loss(state["logits"], state["labels"], state["ref"], offsets=state.get("offsets"), beta=BETA,
                                               label_smoothing=case["smoothing"])
        return (loss.detach(), rewards, *torch.autograd.grad(loss, state["logits"]))
    if op == "policy":
        loss, stats = losses.policy_loss(state["logits"], state["labels"], state["old"], state["advantages"], ref_log_probs=state["ref"],
                                         clip=CLIP_LOW, clip_high=CLIP_HIGH, kl_coef=case["kl"])
        return (loss.detach(), stats, *torch.autograd.grad(loss, state["logits"]))
    if case["box"]:
        outs = F.bound_dropout(*state["x"], case["q"], state["seed"])
    else:
        outs = [F.dropout(state["x"][0], case["q"], state["seed"])]
    return (*[y.detach() for y in outs], *torch.autograd.grad(outs, state["x"], state["grad"]))


def _plain_rows(logits, labels):
    """Row statistics in 32 bits: the logits, the largest, the sum of exponentials and the label's log probability (0 where ignored)."""
    z = logits.detach().float()
    top = z.amax(1, keepdim=True)
    total = (z - top).exp().sum(1, keepdim=True)
    kept = labels != IGNORE
    at = torch.where(kept, labels, 0).view(-1, 1)
    values = (z.gather(1, at) - top - total.log()).squeeze(1)
    return z, top, total, kept, at, torch.where(kept, values, 0.0)


def _plain_gradient(z, top, total, at, weight, dtype):
    """weight (1[v = label] - softmax), the weight being 0 where a row is ignored."""
    grad = (z - top).exp() * (-weight.view(-1, 1) / total)
    grad.scatter_add_(1, at, weight.view(-1, 1))
    return grad.to(dtype)


def _answer_of_row(state, rows):
    """The answer that each row belongs to, one past the last for the rows behind it."""
    if "offsets" not in state:
        return torch.arange(rows, device="cuda") // state["case"]["tokens"]
    return (torch.arange(rows, device="cuda").view(-1, 1) >= state["offsets"][1:].view(1, -1)).sum(1)


def _plain_dropout_words(size, seed):
    """A 32-bit word for each pair of neighbouring values, in 64-bit whole numbers."""
    word = 0xffffffff

    def mix(h):
        h = h ^ (h >> 16)
        h = (h * 0x21f0aaad) & word
        h = h ^ (h >> 15)
        h = (h * 0x735a2d97) & word
        return h ^ (h >> 15)

    pair = torch.arange((size + 1) // 2, device="cuda")
    row, col = (pair >> 15) & word, pair & 0x7fff
    key = mix(((seed ^ (5 * 0x9e3779b9 & word)) + row) & word)
    other = mix(((seed ^ (6 * 0x9e3779b9 & word)) + row) & word)
    return mix(mix((key + (col + 1) * 0x85ebca6b) & word) ^ other)


def _run_plain(state):
    case = state["case"]
    op = case["op"]
    if op == "dropout":
        limit = int(math.floor(case["q"] * 65536 + 0.5))
        size = state["x"][0].numel()
        words = _plain_dropout_words(size, state["seed"])
        keep = (torch.stack((words & 0xffff, words >> 16), 1).view(-1)[:size] < limit).view(state["x"][0].shape)
        scale = 65536.0 / limit if limit else 0.0
        return tuple(torch.where(keep, t.detach().float() * scale, 0.0).to(t.dtype) for t in (*state["x"], *state["grad"]))
    logits, labels = state["logits"], state["labels"].reshape(-1)
    flat = logits.detach().view(-1, logits.size(-1)) if logits.is_contiguous() else logits.detach()
    rows, dtype = flat.size(0), logits.dtype
    z, top, total, kept, at, values = _plain_rows(flat, labels)
    if op == "label":
        if not case["train"]:
            return (values,)
        return values, _plain_gradient(z, top, total, at, torch.where(kept, state["grad"], 0.0), dtype)
    if op == "preference":
        pairs, smoothing = case["pairs"], case["smoothing"]
        answer = _answer_of_row(state, rows)
        ratios = torch.where(kept, values - state["ref"].reshape(-1), 0.0).double()
        sums = torch.zeros(2 * pairs + 1, device="cuda", dtype=torch.float64).index_add_(0, answer, ratios)[:-1]
        rewards = BETA * sums
        x = rewards[:pairs] - rewards[pairs:]
        log_sigmoid = lambda t: t.clamp(max=0.0) - (1.0 + (-t.abs()).exp()).log()
        loss = -((1.0 - smoothing) * log_sigmoid(x) + smoothing * log_sigmoid(-x)).sum() / pairs
        slope = -BETA / pairs * ((1.0 - smoothing) / (1.0 + x.exp()) - smoothing / (1.0 + (-x).exp()))
        of_answer = torch.cat((slope, -slope, slope.new_zeros(1))).float()
        weight = torch.where(kept, of_answer[answer], 0.0)
        return loss.float(), rewards.float(), _plain_gradient(z, top, total, at, weight, dtype).view(logits.shape)
    advantages, kl = state["advantages"].reshape(-1), case["kl"]
    count = kept.sum().clamp(min=1)
    ratio = torch.where(kept, values - state["old"].reshape(-1), 0.0).exp()
    free, bounded = ratio * advantages, ratio.clamp(1.0 - CLIP_LOW, 1.0 + CLIP_HIGH) * advantages
    clipped = kept & (bounded < free)
    surrogate = torch.where(kept, -torch.minimum(free, bounded), 0.0).double().sum() / count
    slope = torch.where(clipped, 0.0, -free)
    divergence = torch.zeros((), device="cuda", dtype=torch.float64)
    if kl:
        apart = torch.where(kept, state["ref"].reshape(-1) - values, 0.0)
        grown = apart.exp()
        divergence = (grown - apart - 1.0).double().sum() / count
        slope = slope + kl * (1.0 - grown)
    weight = torch.where(kept, slope / count, 0.0)
    stats = torch.stack((surrogate, divergence, clipped.sum() / count.double())).float()
    return (surrogate + kl * divergence).float(), stats, _plain_gradient(z, top, total, at, weight, dtype).view(logits.shape)


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------


def _most_rows(case):
    """Rows of a case; of packed answers as many as there are on average."""
    if case["op"] == "label":
        return case["rows"]
    if case["op"] == "policy":
        return case["answers"] * case["tokens"]
    return case["pairs"] * case["tokens"] if case["packed"] else 2 * case["pairs"] * case["tokens"]


def work(case):
    size = BYTES[case["dtype"]]
    if case["op"] == "dropout":
        values = case["rows"] * case["features"] * (3 if case["box"] else 1)
        return {"bytes": 4 * values * size, "flops": 2 * values}
    rows = _most_rows(case)
    logits = rows * case["classes"]
    if case["op"] == "label" and not case["train"]:
        return {"bytes": logits * size + rows * 12, "flops": 4 * logits}
    small = {"label": 16, "preference": 12, "policy": 16 + (4 if case.get("kl") else 0)}[case["op"]]
    return {"bytes": 2 * logits * size + rows * small, "flops": 8 * logits}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------------


def _exact_values(logits, labels):
    parts = []
    for r in range(0, logits.size(0), _rows_at_once(logits.size(1))):
        z = logits[r:r + _rows_at_once(logits.size(1))].detach().double()
        label = labels[r:r + z.size(0)]
        value = z.gather(1, label.clamp(min=0).view(-1, 1)).squeeze(1) - torch.logsumexp(z, 1)
        parts.append(value.masked_fill(label == IGNORE, 0.0))
    return torch.cat(parts)


def _exact_gradient(logits, labels, weight):
    grad = torch.empty(logits.shape, device="cuda", dtype=torch.float64)
    for r in range(0, logits.size(0), _rows_at_once(logits.size(1))):
        part = grad[r:r + _rows_at_once(logits.size(1))]
        torch.softmax(logits[r:r + part.size(0)].detach().double(), 1, out=part)
        label = labels[r:r + part.size(0)].clamp(min=0)
        part[torch.arange(part.size(0), device="cuda"), label] -= 1.0
        part *= -weight[r:r + part.size(0)].view(-1, 1)
    return grad


def _exact_keep(size, seed, q):
    """Which values stay, in numpy's own 32-bit arithmetic."""
    def scramble(v):
        v = v ^ (v >> np.uint32(16))
        v = v * np.uint32(0x21f0aaad)
        v = v ^ (v >> np.uint32(15))
        v = v * np.uint32(0x735a2d97)
        return v ^ (v >> np.uint32(15))

    limit = math.floor(q * 65536 + 0.5)
    keep = np.empty(size, dtype=bool)
    for row in range((size + 65535) // 65536):
        first, second = (scramble(np.array([seed ^ (stream * 0x9e3779b9 & 0xffffffff)], dtype=np.uint32) + np.uint32(row)) for stream in (5, 6))
        step = np.arange(1, 32769, dtype=np.uint32) * np.uint32(0x85ebca6b)
        words = scramble(scramble(step + first) ^ second)
        fields = words.astype("<u4").view("<u2")
        part = keep[row * 65536:(row + 1) * 65536]
        part[:] = fields[:part.size] < limit
    return keep, limit


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "dropout":
        keep, limit = _exact_keep(case["rows"] * case["features"], state["seed"], case["q"])
        mask = torch.from_numpy(keep).cuda().view(case["rows"], case["features"])
        scale = 65536.0 / limit if limit else 0.0
        return tuple((t.detach().double() * scale).masked_fill(~mask, 0.0) for t in (*state["x"], *state["grad"]))
    logits, labels = state["logits"], state["labels"].reshape(-1)
    flat = logits.detach() if logits.dim() == 2 else logits.detach().flatten(0, 1)
    values = _exact_values(flat, labels)
    if op == "label":
        if not case["train"]:
            return (values,)
        weight = state["grad"].double().masked_fill(labels == IGNORE, 0.0)
        return values, _exact_gradient(flat, labels, weight)
    live = (labels != IGNORE).double()
    if op == "preference":
        pairs, smoothing = case["pairs"], case["smoothing"]
        ends = state["offsets"].tolist() if "offsets" in state else [a * case["tokens"] for a in range(2 * pairs + 1)]
        ratios = (values - state["ref"].reshape(-1).double()) * live
        rewards = BETA * torch.stack([ratios[a:b].sum() for a, b in zip(ends[:-1], ends[1:])])
        margin = rewards[:pairs] - rewards[pairs:]
        soft = torch.nn.functional.softplus
        loss = ((1 - smoothing) * soft(-margin) + smoothing * soft(margin)).mean()
        slope = (torch.sigmoid(margin) - (1 - smoothing)) * BETA / pairs
        weight = torch.zeros_like(values)
        for a in range(2 * pairs):
            weight[ends[a]:ends[a + 1]] = slope[a] if a < pairs else -slope[a - pairs]
        return loss, rewards, _exact_gradient(flat, labels, weight * live).view(logits.shape)
    advantages, kl = state["advantages"].reshape(-1).double(), case["kl"]
    count = live.sum().clamp(min=1.0)
    ratio = torch.exp((values - state["old"].reshape(-1).double()) * live)
    low, high = torch.tensor(1.0 - CLIP_LOW, dtype=torch.float64), torch.tensor(1.0 + CLIP_HIGH, dtype=torch.float64)
    outside = ((advantages > 0) & (ratio > high)) | ((advantages < 0) & (ratio < low))
    held = torch.where(advantages > 0, torch.clamp(ratio, max=float(high)), torch.clamp(ratio, min=float(low)))
    surrogate = -(held * advantages * live).sum() / count
    weight = torch.where(outside, 0.0, -ratio * advantages)
    divergence = torch.zeros_like(surrogate)
    if kl:
        apart = (state["ref"].reshape(-1).double() - values) * live
        divergence = (torch.expm1(apart) - apart).sum() / count
        weight = weight - kl * torch.expm1(apart)
    stats = torch.stack((surrogate, divergence, (outside.double() * live).sum() / count))
    return surrogate + kl * divergence, stats, _exact_gradient(flat, labels, weight * live / count).view(logits.shape)
