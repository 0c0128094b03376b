"""Log probabilities of labels, preference loss and policy loss against their definitions in 64 bits.

Tolerances, with u = 2^-24, half a step of fp32.  A row's sum is added up by at least 64 work-items where it has more than 64 vectors, so a partial
sum takes n = classes / 64 + 64 steps at most, each of them, the exponential and its argument off by a few u: relative error of the sum
2 (n + 64) u.  A log probability z - top - log(sum) is off by that and by u times its size, twice; the softmax at distance d = z - top by
that and 1.5 |d| u + 8 u.  Stored results are off by half a step of their type and, below its normal range, of its smallest number."""
import math

import pytest
import torch

from sortnet_amd import losses

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
IGNORE = -100
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
SMALLEST = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -24}    # (numbers below fp32's normal range may be 0)
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def sum_error(classes):
    return 2 * (classes / 64 + 128) * U


def make(rows, classes, dtype, seed, ignored=0.2, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    z = (torch.randn(rows, classes, generator=g) * spread).to(dtype)
    labels = torch.randint(0, classes, (rows,), generator=g)
    labels[torch.rand(rows, generator=g) < ignored] = IGNORE
    return z.cuda(), labels.cuda(), g


def exact_rows(z, labels):
    """Log probabilities and softmax in 64 bits, and how far a kernel may be off in the first."""
    z = z.detach().double()
    lse = torch.logsumexp(z, 1, keepdim=True)
    kept = (labels != IGNORE).view(-1, 1)
    lp = (z.gather(1, labels.clamp(min=0).view(-1, 1)) - lse).masked_fill(~kept, 0.0).squeeze(1)
    return lp, (z - lse).exp(), kept, sum_error(z.size(1)) + 4 * U * (lp.abs() + math.log(max(2, z.size(1))))


def close(got, want, tol, what):
    err = (got.double() - want).abs()
    assert not torch.isnan(err).any(), what
    worst = (err - tol).max().item() if err.numel() else -1.0
    assert worst <= 0.0, "%s: %g over the tolerance, error %g" % (what, worst, err.max().item())


def check_gradient(grad, z, labels, weight, weight_error, what):
    """grad against weight (1[v = label] - softmax); weight_error: how far the kernel's weight may be off."""
    zd = z.detach().double()
    _, p, kept, _ = exact_rows(z, labels)
    weight = weight.view(-1, 1) * kept
    hot = torch.zeros_like(p).scatter_(1, labels.clamp(min=0).view(-1, 1), 1.0)
    want = weight * (hot - p)
    far = zd.amax(1, keepdim=True) - zd
    off = p * (sum_error(z.size(1)) + (1.5 * far + 8) * U)
    tol = weight.abs() * (off + 4 * U * hot) + weight_error.view(-1, 1) * (hot - p).abs() * 1.01
    tol = tol + (want.abs() + tol) * HALF_STEP[z.dtype] + SMALLEST[z.dtype]
    close(grad, want, tol, what)
    assert (grad[labels == IGNORE] == 0).all(), what


SHAPES = [(1, 1), (3, 1), (5, 2), (9, 3), (512, 10), (77, 33), (7, 257), (300, 1000), (64, 2048), (13, 2049), (9, 4096), (5, 4097), (3, 16385), (1, 50001), (700, 8200), (2, 131072), (40, 20000), (33, 60001), (2100, 8200), (70, 131072), (13, 100), (21, 200), (6, 15), (31, 60)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows, classes", SHAPES)
def test_log_probs_and_gradient(rows, classes, dtype):
    z, labels, g = make(rows, classes, dtype, rows * 131 + classes)
    z.requires_grad_()
    up = torch.randn(rows, generator=g).cuda()
    lp = losses.label_log_probs(z, labels)
    assert lp.dtype == torch.float32 and lp.shape == labels.shape
    want, _, _, tol = exact_rows(z, labels)
    close(lp.detach(), want, tol, "log probs")
    grad, = torch.autograd.grad(lp, z, up)
    assert grad.dtype == dtype and grad.shape == z.shape
    check_gradient(grad, z, labels, up.double(), torch.zeros_like(up).double(), "gradient")
    with torch.no_grad():
        assert torch.equal(losses.label_log_probs(z, labels.int()), lp)


@pytest.mark.parametrize("classes", [10, 1000, 9001])
def test_rows_with_strides(classes):
    """Padded vocabularies, parts of a batch, expanded and transposed tensors: the results of a contiguous copy."""
    g = torch.Generator().manual_seed(classes)
    base = torch.randn(6, 9, classes + 3, generator=g).to(torch.bfloat16).cuda()
    labels = torch.randint(0, classes, (6, 9), generator=g).cuda()
    views = [base[:, :, 1:classes + 1], base[:, :-1, :classes], base[::2, 1::3, 2:classes + 2], base[:1, :1, :classes].expand(6, 9, classes),
             base[..., :classes].transpose(0, 1), base[0, :, :classes], base[..., :classes].reshape(3, 2, 9, classes)]
    for view in views:
        t = labels.reshape(-1)[:view[..., 0].numel()].view(view.shape[:-1])
        leaf, flat = view.detach().requires_grad_(), view.detach().contiguous().view(-1, classes).requires_grad_()
        got, want = losses.label_log_probs(leaf, t), losses.label_log_probs(flat, t.reshape(-1))
        assert torch.equal(got.reshape(-1), want)
        up = torch.randn(want.shape, generator=g).cuda()
        a, = torch.autograd.grad(got, leaf, up.view(got.shape))
        b, = torch.autograd.grad(want, flat, up)
        assert a.shape == view.shape and torch.equal(a.reshape(-1, classes), b)
    wide = torch.randn(classes, 5, generator=g).cuda().t().requires_grad_()     # classes that are not neighbours
    t = labels.reshape(-1)[:5]
    assert torch.equal(losses.label_log_probs(wide, t), losses.label_log_probs(wide.contiguous(), t))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("classes", [5, 700, 5000, 70000])
def test_masked_classes(classes, dtype):
    """Classes masked by -inf or the type's lowest value, at the start, in the middle and all but one."""
    z, labels, g = make(8, classes, dtype, classes, ignored=0.0)
    lowest = torch.finfo(dtype).min
    z[0, :classes // 2] = -math.inf
    z[1, classes // 2:] = lowest
    z[2] = -math.inf
    z[2, classes // 3] = 1.5
    z[3] = lowest                        # all alike: uniform
    z[4, 1:] = -math.inf
    labels[0], labels[1], labels[2], labels[3], labels[4] = classes - 1, 0, classes // 3, 1, 0
    z.requires_grad_()
    lp = losses.label_log_probs(z, labels)
    want = torch.log_softmax(z.detach().double(), 1).gather(1, labels.view(-1, 1)).squeeze(1)
    close(lp.detach(), want, sum_error(classes) + 4 * U * (want.abs() + math.log(classes)), "log probs")
    assert lp[2] == 0 and lp[4] == 0
    grad, = torch.autograd.grad(lp.sum(), z)
    p = torch.softmax(z.detach().double(), 1)
    want = torch.zeros_like(p).scatter_(1, labels.view(-1, 1), 1.0) - p
    far = (z.detach().double().amax(1, keepdim=True) - z.detach().double()).clamp(max=200.0)
    tol = p * (sum_error(classes) + (1.5 * far + 8) * U) + 4 * U
    close(grad, want, tol + (want.abs() + tol) * HALF_STEP[dtype] + SMALLEST[dtype], "gradient")
    assert (grad[0, :classes // 2] == 0).all() and (grad[2] == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("rows, classes", [(7, 5), (7, 700), (7, 5000), (7, 70000), (3000, 9000), (1100, 8800)])
def test_values_of_any_size(rows, classes, dtype):
    """Rows whose largest value lies near the ends of the type's range, on both sides of 1e38, with values next to it, and large offsets: log
    probabilities and gradients as in 64 bits.  (Softmax at distance d: see the head of this file; the products with an offset of z are exact.)"""
    z, labels, g = make(rows, classes, dtype, classes, ignored=0.0)
    big = torch.tensor([3.3e38, 1.01e38, 0.99e38, -0.99e38, -1.01e38, -3.3e38, 1e4], device="cuda")
    for k, b in enumerate(big.tolist()):
        for r in (k, rows - 1 - k) if rows > 100 else (k,):
            if k < 6:
                z[r] = -torch.finfo(dtype).max if k > 2 else 0.0
                z[r, classes // 2:] = b
                z[r, -1] = b * 0.5 if b > 0 else b * 1.02
                labels[r] = classes // 2
            else:
                z[r] = (z[r].float() + 1e4).to(dtype)
    z.requires_grad_()
    exact = torch.log_softmax(z.detach().double(), 1)
    want = exact.gather(1, labels.view(-1, 1)).squeeze(1)
    lp = losses.label_log_probs(z, labels)
    close(lp.detach(), want, sum_error(classes) + 4 * U * (want.abs() + math.log(classes)), "log probs")
    p = exact.exp()
    hot = torch.zeros_like(p).scatter_(1, labels.view(-1, 1), 1.0)
    far = (-exact).clamp(max=200.0)
    off = p * (sum_error(classes) + (1.5 * far + 8) * U) + 4 * U * hot
    tol = off + (hot - p).abs() * HALF_STEP[dtype] + off * HALF_STEP[dtype] + SMALLEST[dtype]
    close(torch.autograd.grad(lp, z, torch.ones_like(lp))[0], hot - p, tol, "gradient")
    one = torch.ones(rows, device="cuda")
    loss, _ = losses.policy_loss(z, labels, lp.detach(), -one)       # ratio 1: the same gradient over the rows
    got, = torch.autograd.grad(loss, z)
    close(got.double() * rows, hot - p, tol + 8 * U + (hot - p).abs() * (HALF_STEP[dtype] + 8 * U) + SMALLEST[dtype] * rows, "gradient of the policy")


@pytest.mark.parametrize("classes", [6, 3000 + 7, 40000])
def test_rows_without_values(classes):
    """Ignored rows hold anything; rows of -inf alone, with +inf or NaN, and labels that name no class give NaN, and touch no other row."""
    z, labels, g = make(9, classes, torch.float32, 3, ignored=0.0)
    clean = losses.label_log_probs(z, labels)
    for r, v in ((0, math.nan), (1, math.inf), (2, -math.inf)):
        z[r] = v
        labels[r] = IGNORE
    z[3, 1], z[4, classes - 1], z[5] = math.nan, math.inf, -math.inf
    labels[6], labels[7] = classes, -1
    z.requires_grad_()
    lp = losses.label_log_probs(z, labels)
    assert (lp[:3] == 0).all() and torch.isnan(lp[3:8]).all() and lp[8] == clean[8]
    grad, = torch.autograd.grad(lp, z, torch.ones_like(lp))
    assert (grad[:3] == 0).all() and torch.isnan(grad[6:8]).all() and torch.isnan(grad[3]).all() and torch.isfinite(grad[8]).all()
    assert torch.isnan(torch.log_softmax(z.detach()[3:6], 1)).any(1).all()      # as torch has it


def test_other_ignore_index_and_empty_batches():
    z, labels, _ = make(6, 11, torch.float32, 1, ignored=0.0)
    labels[2] = 4
    lp = losses.label_log_probs(z, labels, ignore_index=4)
    assert (lp[labels == 4] == 0).all() and (lp[labels != 4] != 0).all()
    none = z[:0].detach().requires_grad_()
    out = losses.label_log_probs(none, labels[:0])
    assert out.shape == (0,) and torch.autograd.grad(out.sum(), none)[0].shape == (0, 11)
    all_ignored = torch.full_like(labels, IGNORE)
    zr = z.detach().requires_grad_()
    loss, stats = losses.policy_loss(zr, all_ignored, torch.zeros(6, device="cuda"), torch.ones(6, device="cuda"))
    assert loss == 0 and (stats == 0).all() and (torch.autograd.grad(loss, zr)[0] == 0).all()
    loss, rewards = losses.preference_loss(zr, all_ignored, torch.zeros(6, device="cuda"))
    assert abs(loss.item() - math.log(2)) <= 2 * U and (rewards == 0).all() and (torch.autograd.grad(loss, zr)[0] == 0).all()


# ---- preferences ----------------------------------------------------------------------------------------------------

def exact_preference(z, labels, ref, ends, beta, smoothing):
    lp, _, kept, tol = exact_rows(z, labels)
    kept = kept.squeeze(1)
    ratio = torch.where(kept, lp - ref.double(), 0.0)
    off = torch.where(kept, tol + U * ratio.abs(), 0.0)
    sums = torch.stack([ratio[a:b].sum() for a, b in zip(ends[:-1], ends[1:])])
    offs = torch.stack([off[a:b].sum() for a, b in zip(ends[:-1], ends[1:])])
    pairs = (len(ends) - 1) // 2
    rewards, reward_off = beta * sums, beta * offs + U * beta * sums.abs()
    x = rewards[:pairs] - rewards[pairs:]
    x_off = reward_off[:pairs] + reward_off[pairs:]
    sp = torch.nn.functional.softplus
    each = (1 - smoothing) * sp(-x) + (smoothing * sp(x) if smoothing else 0.0)
    slope = (torch.sigmoid(x) - (1 - smoothing)) * beta / pairs
    weight, weight_off = torch.zeros_like(lp), torch.zeros_like(lp)
    for k in range(2 * pairs):
        i = k % pairs
        weight[ends[k]:ends[k + 1]] = slope[i] if k < pairs else -slope[i]
        weight_off[ends[k]:ends[k + 1]] = beta / pairs * x_off[i] / 4 + 2 * U * slope[i].abs()     # |sigma'| <= 1/4
    loss = each.mean()
    return loss, x_off.mean() + U * loss, rewards, reward_off, weight * kept, weight_off * kept


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("pairs, tokens, classes, smoothing", [(1, 1, 2, 0.0), (3, 1, 10, 0.1), (128, 1, 200, 0.1), (5, 7, 33, 0.0), (2, 300, 1000, 0.2), (1, 65, 9000, 0.0), (1100, 1, 3, 0.0)])
def test_preference_of_padded_answers(pairs, tokens, classes, smoothing, dtype):
    rows = 2 * pairs * tokens
    z, labels, g = make(rows, classes, dtype, rows + classes, ignored=0.3 if tokens > 1 else 0.0)
    ref = exact_rows(z, labels)[0].float() + 0.3 * torch.randn(rows, generator=g).cuda()
    ref[labels == IGNORE] = math.nan
    ends = [tokens * k for k in range(2 * pairs + 1)]
    want = exact_preference(z, labels, ref, ends, 0.3, smoothing)
    shape = (2 * pairs, tokens) if tokens > 1 else (2 * pairs,)
    leaf = z.view(*shape, classes).requires_grad_()
    loss, rewards = losses.preference_loss(leaf, labels.view(shape), ref.view(shape), beta=0.3, label_smoothing=smoothing)
    assert loss.shape == () and not rewards.requires_grad
    close(loss.detach(), want[0], want[1], "loss")
    close(rewards, want[2], want[3], "rewards")
    grad, = torch.autograd.grad(loss, leaf)
    check_gradient(grad.view(rows, classes), z, labels, want[4], want[5], "gradient")
    loss2, rewards2 = losses.preference_loss(leaf.detach(), labels.view(shape), ref.view(shape), beta=0.3, label_smoothing=smoothing)
    assert torch.equal(loss, loss2) and torch.equal(rewards, rewards2)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("bits", [torch.int32, torch.int64], ids=str)
@pytest.mark.parametrize("classes", [7, 5000])
def test_preference_of_packed_answers(classes, bits, dtype):
    """Answers of no row, of one and of many; rows behind the last answer hold NaN and get zeros."""
    lengths = [0, 1, 3, 200, 2, 0, 70, 64]
    ends = [0]
    for n in lengths:
        ends.append(ends[-1] + n)
    rows = ends[-1] + 5
    z, labels, g = make(rows, classes, dtype, classes + 1)
    labels[ends[2]:ends[3]] = IGNORE        # an answer with nothing kept
    labels[-1] = IGNORE
    ref = exact_rows(z, labels)[0].float() + 0.3 * torch.randn(rows, generator=g).cuda()
    want = exact_preference(z, labels, ref, ends, 0.1, 0.0)
    z[ends[-1]:] = math.nan
    z.requires_grad_()
    loss, rewards = losses.preference_loss(z, labels, ref, offsets=torch.tensor(ends, dtype=bits, device="cuda"))
    close(loss.detach(), want[0], want[1], "loss")
    close(rewards, want[2], want[3], "rewards")
    grad, = torch.autograd.grad(loss, z, torch.tensor(2.5, device="cuda"))
    assert (grad[ends[-1]:] == 0).all()
    n = ends[-1]
    check_gradient(grad[:n], z[:n], labels[:n], 2.5 * want[4][:n], 2.5 * want[5][:n] + 4 * U * want[4][:n].abs(), "gradient")


def test_preference_far_apart():
    """Margins so large that one side of the logarithm vanishes."""
    z, labels, _ = make(4, 5, torch.float32, 2, ignored=0.0)
    lp = losses.label_log_probs(z, labels)
    for shift in (80.0, 4000.0):
        ref = lp.clone()
        ref[0] -= shift
        ref[1] += shift
        loss, rewards = losses.preference_loss(z.requires_grad_(), labels, ref, beta=1.0)
        assert abs(loss.item() - shift / 2) <= 1e-5 * shift and torch.isfinite(torch.autograd.grad(loss, z)[0]).all()


# ---- policies -------------------------------------------------------------------------------------------------------

def exact_policy(z, labels, old, adv, ref, low, high, kl):
    lp, _, kept, tol = exact_rows(z, labels)
    kept = kept.squeeze(1)
    n = max(1, int(kept.sum()))
    zero = torch.zeros_like(lp)
    d = torch.where(kept, lp - old.double(), zero)
    adv = torch.where(kept, adv.double(), zero)
    ratio = d.exp()
    ratio_off = ratio * (tol + U * (d.abs() + 8))
    free, bounded = ratio * adv, ratio.clamp(1 - low, 1 + high) * adv
    clipped = bounded < free
    term = -torch.minimum(free, bounded)
    slope, slope_off = torch.where(clipped, zero, -free), torch.where(clipped, zero, ratio_off * adv.abs())
    term_off = ratio_off * adv.abs() + 4 * U * term.abs()
    div, div_off = zero, zero
    if kl:
        apart = torch.where(kept, ref.double() - lp, zero)
        div = torch.expm1(apart) - apart
        grown_off = apart.exp() * (tol + U * (apart.abs() + 8))
        div_off = grown_off + tol + 4 * U * (div.abs() + apart.abs())
        slope, slope_off = slope - kl * torch.expm1(apart), slope_off + kl * grown_off + 4 * U * kl * (apart.exp() + 1)
    stats = torch.stack((term.sum() / n, div.sum() / n, clipped.double().sum() / n))
    off = torch.stack((term_off.sum() / n, div_off.sum() / n, zero.sum()))
    return (stats[0] + kl * stats[1], off[0] + kl * off[1] + U * (stats[0] + kl * stats[1]).abs(), stats, off + U * stats.abs(),
            slope / n, slope_off / n + 6 * U * slope.abs() / n)


def away_from_borders(moved, low, high):
    """The loss has a kink where the ratio is 1 - low or 1 + high."""
    for border in (math.log(1 - low) if low < 1 else -1e9, math.log(1 + high)):
        moved = torch.where((moved - border).abs() < 2e-3, moved + 5e-3, moved)
    return moved


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("answers, tokens, classes, kl, shared", [(1, 1, 2, 0.0, False), (256, 1, 10, 0.0, False), (3, 50, 33, 0.1, True), (40, 3, 1000, 0.05, False), (5, 9, 4500, 0.1, True),
                                                                 (1, 3, 70001, 0.02, True), (5000, 1, 4, 0.3, False)])
def test_policy(answers, tokens, classes, kl, shared, dtype):
    rows, low, high = answers * tokens, 0.2, 0.28
    z, labels, g = make(rows, classes, dtype, rows + classes, ignored=0.2)
    lp = exact_rows(z, labels)[0].float()
    old = lp - away_from_borders(0.25 * torch.randn(rows, generator=g).cuda(), low, high)
    ref = lp + 0.3 * torch.randn(rows, generator=g).cuda()
    adv = torch.randn(answers, 1 if shared else tokens, generator=g).cuda().expand(answers, tokens)
    old[labels == IGNORE] = math.nan
    ref[labels == IGNORE] = math.inf
    want = exact_policy(z, labels, old, adv.reshape(-1), ref, low, high, kl)
    leaf = z.view(answers, tokens, classes).requires_grad_()
    shape = (answers, tokens)
    args = (labels.view(shape), old.view(shape), adv)
    kw = dict(ref_log_probs=ref.view(shape) if kl else None, clip=low, clip_high=high, kl_coef=kl)
    loss, stats = losses.policy_loss(leaf, *args, **kw)
    assert loss.shape == () and stats.shape == (3,) and not stats.requires_grad
    close(loss.detach(), want[0], want[1], "loss")
    close(stats, want[2], want[3], "stats")
    grad, = torch.autograd.grad(loss, leaf)
    check_gradient(grad.view(rows, classes), z, labels, want[4], want[5], "gradient")
    quiet = losses.policy_loss(leaf.detach(), *args, **kw)
    assert torch.equal(quiet[0], loss) and torch.equal(quiet[1], stats)


@pytest.mark.parametrize("answers, tokens, classes, kl, dtype", [(40000, 1, 230, 0.1, torch.float32), (2000, 42, 203, 0.0, torch.float16), (1030, 1, 9001, 0.05, torch.float32),
                                                                (60, 20, 16500, 0.1, torch.bfloat16), (1 << 20, 1, 9, 0.0, torch.float32), (1 << 22, 1, 5, 0.1, torch.bfloat16)])
def test_policy_of_many_rows(answers, tokens, classes, kl, dtype):
    """Logits of 32 MiB and more, whose gradient is made with the loss: alone, scaled, kept for a second backward, and in a replayed graph."""
    rows, low, high = answers * tokens, 0.2, 0.28
    assert rows * classes * torch.finfo(dtype).bits // 8 >= 32 << 20
    z, labels, g = make(rows, classes, dtype, rows + classes, ignored=0.2)
    lp = exact_rows(z, labels)[0].float()
    old = lp - away_from_borders(0.25 * torch.randn(rows, generator=g).cuda(), low, high)
    ref = lp + 0.3 * torch.randn(rows, generator=g).cuda()
    adv = torch.randn(answers, 1, generator=g).cuda().expand(answers, tokens)
    want = exact_policy(z, labels, old, adv.reshape(-1), ref, low, high, kl)
    shape = (answers, tokens)
    leaf = z.view(*shape, classes).requires_grad_()
    call = lambda t: losses.policy_loss(t, labels.view(shape), old.view(shape), adv, ref_log_probs=ref.view(shape) if kl else None, clip=low, clip_high=high, kl_coef=kl)
    loss, stats = call(leaf)
    close(loss.detach(), want[0], want[1], "loss")
    close(stats, want[2], want[3], "stats")
    check = lambda got, by: check_gradient(got.view(rows, classes), z, labels, by * want[4], abs(by) * (want[5] + 4 * U * want[4].abs()), "gradient")
    first, = torch.autograd.grad(loss, leaf, retain_graph=True)
    check(first, 1.0)
    whole = first.clone()
    first.zero_()                           # the caller's own
    second, = torch.autograd.grad(loss, leaf, torch.tensor(-0.375, device="cuda"), retain_graph=True)
    check(second, -0.375)
    second.zero_()
    third, = torch.autograd.grad(loss, leaf)
    assert torch.equal(third, whole)
    loss, _ = call(leaf)
    scaled, = torch.autograd.grad(0.3 * loss, leaf)
    check(scaled, float(torch.tensor(0.3)))
    loss, _ = call(leaf)
    loss.backward()
    assert torch.equal(leaf.grad, whole)
    nothing, = torch.autograd.grad(call(leaf)[0], leaf, torch.zeros((), device="cuda"))
    assert (nothing == 0).all()
    if classes > 5:
        static, other = leaf.detach().clone().requires_grad_(), leaf.detach().flip(1 if tokens > 1 else 0).contiguous()
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            torch.autograd.grad(call(static)[0], static)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            outs = call(static)
            made, = torch.autograd.grad(outs[0], static)
        for data in (other, leaf.detach(), other):
            with torch.no_grad():
                static.copy_(data)
            fresh = data.clone().requires_grad_()
            eager = call(fresh)
            eager_grad, = torch.autograd.grad(eager[0], fresh)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(outs[0], eager[0]) and torch.equal(outs[1], eager[1]) and torch.equal(made, eager_grad)


@pytest.mark.parametrize("forward_captured", [False, True])
def test_policy_backward_in_a_graph_of_its_own(forward_captured):
    """A backward captured apart from its forward, which made the gradient: run several times for one forward, with another upstream gradient
    each time and after the caller has overwritten what it got."""
    rows, classes = 40000, 230
    z, labels, g = make(rows, classes, torch.float32, 77, ignored=0.2)
    assert rows * classes * 4 >= 32 << 20
    old = exact_rows(z, labels)[0].float() - 0.1
    adv = torch.randn(rows, generator=g).cuda()
    call = lambda t: losses.policy_loss(t, labels, old, adv)[0]
    static, up = z.clone().requires_grad_(), torch.ones((), device="cuda")
    stream, pool = torch.cuda.Stream(), torch.cuda.graph_pool_handle()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        torch.autograd.grad(call(static), static, up)
        loss = None if forward_captured else call(static)
    torch.cuda.synchronize()
    first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    if forward_captured:
        with torch.cuda.graph(first, stream=stream, pool=pool):
            loss = call(static)
    with torch.cuda.graph(second, stream=stream, pool=pool):
        made, = torch.autograd.grad(loss, static, up)
    if forward_captured:
        first.replay()
    fresh = z.clone().requires_grad_()
    eager = call(fresh)
    for factor in (1.0, -0.5, 1.0, 1.0):
        up.fill_(factor)
        second.replay()
        torch.cuda.synchronize()
        assert torch.equal(made, torch.autograd.grad(eager, fresh, torch.full((), factor, device="cuda"), retain_graph=True)[0]), factor
        made.zero_()


def test_policy_clips_and_defaults():
    """Each side of the clip with either sign of the advantage; clip_high defaults to clip; a clip of 1 and 0."""
    z, labels, _ = make(6, 5, torch.float32, 4, ignored=0.0)
    z.requires_grad_()
    lp = losses.label_log_probs(z, labels).detach()
    moved = torch.tensor([0.5, 0.5, -0.5, -0.5, 0.01, 0.01], device="cuda")
    adv = torch.tensor([1.0, -1.0, 1.0, -1.0, 1.0, -1.0], device="cuda")
    for low, high in ((0.2, None), (0.2, 0.3), (1.0, 0.0), (0.0, 1.0)):
        loss, stats = losses.policy_loss(z, labels, lp - moved, adv, clip=low, clip_high=high)
        want = exact_policy(z, labels, lp - moved, adv, None, low, low if high is None else high, 0.0)
        close(loss.detach(), want[0], want[1], "loss")
        close(stats, want[2], want[3], "stats")
        check_gradient(torch.autograd.grad(loss, z)[0], z, labels, want[4], want[5], "gradient")


# ---- in use ------------------------------------------------------------------------------------------------------------

def test_gradients_against_differences():
    """Central differences of the kernels' own losses along random directions u, |u_v| <= 1, step h = 1/32.  Along u a log probability has a slope
    of at most 2, a second derivative (a variance) of at most 1 and a third one (a third central moment) of at most 2.  Weights
    of 0.5 on four rows: third derivative at most 4.  Preference, two pairs, beta = 0.5: first three derivatives of the margin at most 2, 1 and 2,
    of the logistic loss 1, 1/4 and 0.1: 2 + 3 * 2 / 4 + 0.8 < 5.  Policy: exp(d) (2 + 3 * 2 + 8) < 20 for ratios up to 1.2, 0.2 (1.5 * 16 + 2) < 6
    for the divergence (ratios up to 1.5): 26.  The difference is off by h^2 / 6 of that, and by 1e-5 / h for values that are off by 1e-5."""
    z, labels, g = make(4, 9, torch.float32, 8, ignored=0.0, spread=1.0)
    lp = losses.label_log_probs(z, labels)
    up = torch.tensor([0.5, -0.5, 0.5, -0.5], device="cuda")
    ref = lp + torch.tensor([0.3, -0.2, 0.1, 0.4], device="cuda")
    old = lp - torch.tensor([0.1, -0.1, 0.6, -0.6], device="cuda")
    adv = torch.tensor([1.0, -1.0, 1.0, -1.0], device="cuda")     # the last two are far outside the clip: constant
    h = 1 / 32
    for f, tol in ((lambda t: (losses.label_log_probs(t, labels) * up).sum(), 4 * h * h / 6 + 1e-5 / h),
                   (lambda t: losses.preference_loss(t, labels, ref, beta=0.5, label_smoothing=0.1)[0], 5 * h * h / 6 + 1e-5 / h),
                   (lambda t: losses.policy_loss(t, labels, old, adv, ref_log_probs=ref, kl_coef=0.2)[0], 26 * h * h / 6 + 1e-5 / h)):
        leaf = z.detach().requires_grad_()
        grad, = torch.autograd.grad(f(leaf), leaf)
        for _ in range(4):
            u = (torch.rand(z.shape, generator=g) * 2 - 1).cuda()
            with torch.no_grad():
                diff = (f(z + h * u).double() - f(z - h * u).double()) / (2 * h)
            assert abs((grad.double() * u).sum().item() - diff.item()) <= tol


@pytest.mark.parametrize("classes", [10, 6000, 80000])
def test_captured_training_step_replays(classes):
    """Two graphs with their own inputs, replayed in turn and on two streams at once, each against its eager result."""
    graphs = []
    for k in range(2):
        z, labels, g = make(6, classes, torch.bfloat16, 10 + k)
        lp = exact_rows(z, labels)[0].float()
        old, ref, adv = lp - 0.1, lp + 0.2, torch.randn(6, generator=g).cuda()
        static = z.clone().requires_grad_()

        def step(leaf, labels=labels, ref=ref, old=old, adv=adv):    # (a graph reads them where they are: they have to live)
            values = losses.label_log_probs(leaf, labels)
            loss, rewards = losses.preference_loss(leaf, labels, ref)
            second, stats = losses.policy_loss(leaf, labels, old, adv, ref_log_probs=ref, kl_coef=0.1)
            grad, = torch.autograd.grad(values.sum() + loss + second, leaf)
            return [values.detach(), loss.detach(), rewards, second.detach(), stats, grad]

        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            step(static)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            outs = step(static)
        graphs.append((graph, static, outs, step, stream))
    for replay in range(4):
        wants = []
        for graph, static, outs, step, stream in graphs:
            with torch.no_grad():
                static.copy_((torch.randn(static.shape, generator=torch.Generator().manual_seed(replay)) * 2).to(static.dtype))
            wants.append(step(static.detach().clone().requires_grad_()))
        torch.cuda.synchronize()
        if replay % 2:
            for graph, _, _, _, stream in graphs:
                with torch.cuda.stream(stream):
                    graph.replay()
        else:
            for graph, *_ in graphs:
                graph.replay()
        torch.cuda.synchronize()
        for (_, _, outs, _, _), want in zip(graphs, wants):
            for a, b in zip(outs, want):
                assert torch.equal(a, b)


def test_other_streams_and_repeats():
    """Work on a stream of the caller's; the same bits each time."""
    z, labels, g = make(300, 5001, torch.float16, 5)
    z.requires_grad_()
    up = torch.randn(300, generator=g).cuda()
    lp = losses.label_log_probs(z, labels)
    grad, = torch.autograd.grad(lp, z, up)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            again = losses.label_log_probs(z, labels)
            g2, = torch.autograd.grad(again, z, up)
            assert torch.equal(again, lp) and torch.equal(g2, grad)
    torch.cuda.current_stream().wait_stream(side)


def test_what_is_refused():
    z, labels, _ = make(4, 3, torch.float32, 1, ignored=0.0)
    r = torch.zeros(4, device="cuda")
    for bad in (lambda: losses.label_log_probs(z.double(), labels), lambda: losses.label_log_probs(z, labels.float()), lambda: losses.label_log_probs(z, labels[:3]),
                lambda: losses.label_log_probs(z[0], labels[0]), lambda: losses.label_log_probs(z, labels.cpu()), lambda: losses.label_log_probs(z[:, :0], labels),
                lambda: losses.preference_loss(z, labels, r[:3]), lambda: losses.preference_loss(z, labels, r.double()), lambda: losses.preference_loss(z[:3], labels[:3], r[:3]),
                lambda: losses.preference_loss(z[:0], labels[:0], r[:0]), lambda: losses.preference_loss(z, labels, r, label_smoothing=0.5),
                lambda: losses.preference_loss(z, labels, r, offsets=torch.tensor([0, 2], device="cuda")), lambda: losses.preference_loss(z, labels, r, offsets=torch.tensor([0, 2, 4])),
                lambda: losses.preference_loss(z, labels, r, offsets=torch.tensor([0.0, 2, 4], device="cuda")),
                lambda: losses.preference_loss(z.view(2, 2, 3), labels.view(2, 2), r.view(2, 2), offsets=torch.tensor([0, 2, 4], device="cuda")),
                lambda: losses.preference_loss(z, labels, r.clone().requires_grad_()), lambda: losses.policy_loss(z, labels, r, r.clone().requires_grad_()),
                lambda: losses.policy_loss(z, labels, r, r.view(4, 1)), lambda: losses.policy_loss(z, labels, r, r, kl_coef=0.1), lambda: losses.policy_loss(z, labels, r, r, clip=1.5),
                lambda: losses.policy_loss(z[:0], labels[:0], r[:0], r[:0]), lambda: losses.policy_loss(z, labels, r.to(torch.bfloat16), r)):
        with pytest.raises(RuntimeError):
            bad()
    leaf = z.clone().requires_grad_()
    lp = losses.label_log_probs(leaf, labels)
    with torch.no_grad():
        leaf.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(lp.sum(), leaf)


@pytest.mark.parametrize("rows, classes, dtype", [(1100, 131072, torch.bfloat16), (4400, 16389, torch.float32)])
def test_logits_larger_than_the_caches(rows, classes, dtype):
    """More than 256 MiB of logits: some rows are read past the caches, with each of the losses."""
    assert rows * classes * torch.finfo(dtype).bits // 8 > 256 << 20
    z, labels, g = make(rows, classes, dtype, 77, ignored=0.1)
    z.requires_grad_()
    up = torch.randn(rows, generator=g).cuda()
    lp = losses.label_log_probs(z, labels)
    want, _, _, tol = exact_rows(z, labels)
    close(lp.detach(), want, tol, "log probs")
    check_gradient(torch.autograd.grad(lp, z, up)[0], z, labels, up.double(), torch.zeros_like(up).double(), "gradient")
    ref = want.float() + 0.3 * torch.randn(rows, generator=g).cuda()
    pw = exact_preference(z, labels, ref, [0, rows // 3, rows // 2, rows // 2 + 7, rows - 2], 0.1, 0.0)
    loss, rewards = losses.preference_loss(z, labels, ref, offsets=torch.tensor([0, rows // 3, rows // 2, rows // 2 + 7, rows - 2], device="cuda"))
    close(loss.detach(), pw[0], pw[1], "loss")
    close(rewards, pw[2], pw[3], "rewards")
    check_gradient(torch.autograd.grad(loss, z)[0], z, labels, pw[4], pw[5], "gradient")
    old = want.float() - away_from_borders(0.25 * torch.randn(rows, generator=g).cuda(), 0.2, 0.2)
    pol = exact_policy(z, labels, old, up, ref, 0.2, 0.2, 0.1)
    loss, stats = losses.policy_loss(z, labels, old, up, ref_log_probs=ref, kl_coef=0.1)
    close(loss.detach(), pol[0], pol[1], "loss")
    close(stats, pol[2], pol[3], "stats")
    check_gradient(torch.autograd.grad(loss, z)[0], z, labels, pol[4], pol[5], "gradient")


def test_two_threads_and_a_first_call_under_capture():
    """Calls of two host threads on one stream give what each gives alone; a graph needs no call before it."""
    import threading
    data = [make(64, 5000 + 100 * k, torch.float32, 30 + k, ignored=0.0) for k in range(2)]
    wants = []
    for z, labels, _ in data:
        leaf = z.clone().requires_grad_()
        loss, rewards = losses.preference_loss(leaf, labels, torch.zeros(64, device="cuda"))
        wants.append((loss.detach(), rewards, torch.autograd.grad(loss, leaf)[0]))
    wrong = []

    def work(k):
        z, labels, _ = data[k]
        for _ in range(20):
            leaf = z.clone().requires_grad_()
            loss, rewards = losses.preference_loss(leaf, labels, torch.zeros(64, device="cuda"))
            got = (loss.detach(), rewards, torch.autograd.grad(loss, leaf)[0])
            if not all(torch.equal(a, b) for a, b in zip(got, wants[k])):
                wrong.append(k)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
    z, labels, _ = make(5, 90001, torch.float16, 9)
    zero = torch.zeros(5, device="cuda")
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        outs = [losses.label_log_probs(z, labels), *losses.policy_loss(z, labels, zero, zero)]
    eager = [losses.label_log_probs(z, labels), *losses.policy_loss(z, labels, zero, zero)]
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, eager))


def test_transforms_are_refused():
    z, labels, _ = make(4, 3, torch.float32, 1, ignored=0.0)
    r = torch.zeros(4, device="cuda")
    with torch.autograd.forward_ad.dual_level():
        dual, dual_r = torch.autograd.forward_ad.make_dual(z, torch.ones_like(z)), torch.autograd.forward_ad.make_dual(r, torch.ones_like(r))
        for bad in (lambda: losses.label_log_probs(dual, labels), lambda: losses.preference_loss(dual, labels, r), lambda: losses.preference_loss(z, labels, dual_r),
                    lambda: losses.policy_loss(z, labels, dual_r, r), lambda: losses.policy_loss(z, labels, r, dual_r), lambda: losses.policy_loss(z, labels, r, r, ref_log_probs=dual_r)):
            with pytest.raises(NotImplementedError):
                bad()


def test_rows_beyond_32_bit_offsets():
    """The last row of a tensor of more than 2^32 elements."""
    classes, rows = 1 << 20, (1 << 12) + 1
    z = torch.empty(rows, classes, device="cuda", dtype=torch.bfloat16)
    z[-1] = torch.linspace(-2, 2, classes, device="cuda").to(torch.bfloat16)
    z[0] = 0.0
    labels = torch.full((rows,), IGNORE, device="cuda")
    labels[-1], labels[0] = classes - 3, 5
    z.requires_grad_()
    lp = losses.label_log_probs(z, labels)
    want, _, _, tol = exact_rows(z[-1:], labels[-1:])
    close(lp[-1:].detach(), want, tol, "last row")
    assert abs(lp[0].item() + math.log(classes)) <= sum_error(classes) + 4 * U * 28
    grad, = torch.autograd.grad(lp.sum(), z)
    check_gradient(grad[-1:], z[-1:], labels[-1:], torch.ones(1, device="cuda", dtype=torch.float64), torch.zeros(1, device="cuda", dtype=torch.float64), "gradient")
    assert (grad[1:3] == 0).all() and (grad[-2] == 0).all()


def test_second_derivatives_are_refused():
    """A gradient under create_graph is the gradient; whatever asks for its derivative raises, and what does not, does not."""
    z, labels, g = make(8, 30, torch.float32, 3)
    ref, adv = exact_rows(z, labels)[0].float() + 0.1, torch.randn(8, generator=g).cuda()
    up = torch.randn(8, generator=g).cuda().requires_grad_()
    leaf = z.requires_grad_()
    wide = (torch.randn(30, 8, generator=g).cuda().requires_grad_(), lambda t: t.t())       # logits that are copied
    for start, view in ((leaf, lambda t: t), (leaf, lambda t: torch.tanh(t) * 3), wide):
        for call in (lambda t: (losses.label_log_probs(t, labels) * up).sum(), lambda t: losses.preference_loss(t, labels, ref)[0],
                     lambda t: losses.policy_loss(t, labels, ref, adv, ref_log_probs=ref, kl_coef=0.1)[0]):
            plain, = torch.autograd.grad(call(view(start)), start)
            loss = call(view(start))
            grad, = torch.autograd.grad(loss, start, create_graph=True)
            assert torch.equal(grad, plain) and grad.requires_grad
            with pytest.raises(RuntimeError, match="differentiated once"):
                torch.autograd.grad(grad.pow(2).sum(), start, retain_graph=True)
            with pytest.raises(RuntimeError, match="differentiated once"):
                (loss + grad.pow(2).sum()).backward(retain_graph=True)
            again, = torch.autograd.grad(loss + grad.detach().sum(), start)
            assert torch.equal(again, plain)
    loss = (losses.label_log_probs(leaf, labels) * up).sum()
    grad, = torch.autograd.grad(loss, leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiated once"):
        torch.autograd.grad(grad.sum(), up)
    empty = z[:0].detach().requires_grad_()
    grad, = torch.autograd.grad(losses.label_log_probs(empty, labels[:0]).sum(), empty, create_graph=True)
    assert grad.shape == (0, 30)


def test_second_derivatives_of_a_gradient_made_with_the_loss():
    """The same where the policy's forward made the gradient (32 MiB of logits and more)."""
    rows, classes = 40000, 230
    z, labels, g = make(rows, classes, torch.float32, 78)
    old, adv = exact_rows(z, labels)[0].float(), torch.randn(rows, generator=g).cuda()
    z.requires_grad_()
    plain, = torch.autograd.grad(losses.policy_loss(z, labels, old, adv)[0], z)
    for retain in (True, False):
        loss = losses.policy_loss(z, labels, old, adv)[0]
        grad, = torch.autograd.grad(loss, z, create_graph=True, retain_graph=retain)
        assert torch.equal(grad, plain)
        with pytest.raises(RuntimeError, match="differentiated once"):
            torch.autograd.grad(grad.sum(), z)


@pytest.mark.parametrize("bits", [torch.int32, torch.int64], ids=str)
@pytest.mark.parametrize("classes", [7, 5000, 40001])
def test_preference_of_packed_answers_in_half_precision(classes, bits):
    test_preference_of_packed_answers(classes, bits, torch.float16)


def test_policy_scaled_by_its_inputs():
    """A positive factor, a power of two, on advantages and kl_coef is one on the loss: the same bits, its sizes and the gradient made with the loss included."""
    for rows, classes in ((64, 30), (40000, 230)):
        z, labels, g = make(rows, classes, torch.float32, 11)
        lp = exact_rows(z, labels)[0].float()
        old, ref, adv = lp - 0.2 * torch.randn(rows, generator=g).cuda(), lp + 0.2, torch.randn(rows, generator=g).cuda()
        z.requires_grad_()
        loss, _ = losses.policy_loss(z, labels, old, adv, ref_log_probs=ref, kl_coef=0.5)
        scaled, _ = losses.policy_loss(z, labels, old, 8 * adv, ref_log_probs=ref, kl_coef=4.0)
        assert torch.equal(8 * loss, scaled)
        assert torch.equal(torch.autograd.grad(8 * loss, z)[0], torch.autograd.grad(scaled, z)[0])
