"""How close log probabilities and what is summed of them come to 64 bits, with u = 2^-24, half a step of fp32.

Sums over rows show what the errors of the rows have in common.  An exponential at distance v is off by a rounding of v log2(e), uniform within |v| u
and to either side, and by the error of the hardware's exp2, at most 2 u (one step) and of one side by 0.06 u on average (measured); 0.25 u are allowed
for that.  Rows here have a peak p = log(C / 32) +- 1 in one class, the label, and the others' values uniform in -4 .. 0: all but a ninth
of a sum comes of thousands of terms at |v| of 3 to 10, whose roundings, of 3.2 u at most (standard deviation), leave 0.04 u in the mean over them.
A log probability between -4 and 0 is stored within 2 u, uniform: 1.2 u, so the mean over R rows has 0.05 u for R = 600."""
import math

import pytest
import torch

from sortnet_amd import losses

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
IGNORE = -100
TYPES = [torch.float32, torch.bfloat16, torch.float16]
# which of them are read by part of a wavefront, by a workgroup that holds them, by one that does not, and in parts
FORMS = {"short": (2048, 1000), "held": (600, 9000), "whole": (2048, 32000), "parts": (600, 40000)}


def peaked(rows, classes, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    z = (torch.rand(rows, classes, generator=g, device="cuda") * -4).to(dtype)
    labels = torch.randint(0, classes, (rows,), generator=g, device="cuda")
    peak = round(math.log(classes / 32) * 16) / 16 - 1 + torch.arange(rows, device="cuda") % 32 / 16
    z[torch.arange(rows, device="cuda"), labels] = peak.to(dtype)
    return z, labels


def exact_values(z, labels):
    parts = []
    for r in range(0, z.size(0), 256):
        d = z[r:r + 256].double()
        parts.append(d.gather(1, labels[r:r + 256].clamp(min=0).view(-1, 1)).squeeze(1) - torch.logsumexp(d, 1))
    return torch.cat(parts)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("form", FORMS)
def test_mean_of_log_probs(form, dtype):
    """0.25 u and six standard deviations of 0.07 u."""
    z, labels = peaked(*FORMS[form], dtype, 5)
    off = losses.label_log_probs(z, labels).double() - exact_values(z, labels)
    assert abs(off.mean().item()) <= (0.25 + 6 * 0.07) * U


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_rewards_of_long_answers(dtype):
    """Answers of 1024 tokens over 32000 classes: beta times 1024 errors with a mean of 0.25 u at most and a standard deviation of 1.2 u."""
    z, labels = peaked(4 * 1024, 32000, dtype, 6)
    want = exact_values(z, labels)
    ref = want.float() + 0.3 * torch.randn(want.shape, generator=torch.Generator(device="cuda").manual_seed(7), device="cuda")
    _, rewards = losses.preference_loss(z.view(4, 1024, -1), labels.view(4, 1024), ref.view(4, 1024), beta=0.1)
    exact = 0.1 * (want - ref.double()).view(4, 1024).sum(1)
    assert ((rewards.double() - exact).abs() <= 0.1 * (1024 * 0.25 + 6 * math.sqrt(1024) * 1.2) * U + U * exact.abs()).all()


@pytest.mark.parametrize("rows", [1, 40])
def test_divergence_of_near_policies(rows):
    """exp(a) - 1 - a of reference and policy, a from 1e-6 to 20 of either sign.  Rows of one class that can be chosen have the log probability 0, so a is the
    reference's: below 1/2 the power series rounds a, its square, eight steps of which the last two count, and the result: 8 u.  Beyond, expm1 is off by
    2 u of its value, and its argument, rounded already, by nothing; that is 2 u (1 - exp(-1/2)) / (exp(-1/2) - 1/2) = 7.4 u of the result at -1/2 and 8.8 u
    at 1/2, less further out; and 2 u for the results, stored twice."""
    z = torch.full((rows, 5), -math.inf, device="cuda")
    z[:, 3] = 1.25
    labels = torch.full((rows,), 3, device="cuda")
    zero, one = torch.zeros(rows, device="cuda"), torch.ones(rows, device="cuda")
    for size in (1e-6, 1e-5, 1e-4, 1e-3, 1e-2, 0.1, 0.3, 0.4999, 0.5, 0.5001, 0.7, 1.0, 3.0, 20.0):
        for a in (size, -size):
            ref = torch.full((rows,), a, device="cuda")
            d = ref[0].double().item()
            exact = d * d / 2 * (1 + d / 3 * (1 + d / 4 * (1 + d / 5))) if size < 0.005 else math.expm1(d) - d
            z.requires_grad_()
            loss, stats = losses.policy_loss(z, labels, zero, zero, ref_log_probs=ref, kl_coef=1.0)
            assert abs(stats[1].item() - exact) <= 11 * U * exact and abs(loss.item() - exact) <= 11 * U * exact, a


# ---- every class counts, once ------------------------------------------------------------------------------------------
# Rows of -30 with a 0 in one class, its place going over the row, and -1 in the label: a class that is left out or read twice changes log
# probability and gradient by tenths.  The -1 is scaled once or not at all: off by 6 u of its part, exp(-1) / (1 + exp(-1)) = 0.27; sums of up
# to 32 values lose 5 u, the result 2 u: 9 u, and the probabilities in the gradient as much and 6 u for their own products.

def places(classes, vec):
    """Starts and ends of vectors and parts, the row's ends, and some others."""
    at = {0, 1, vec - 1, vec, classes // 2, classes - 1, classes - 2, classes // vec * vec - 1, classes // vec * vec, classes // vec * vec - vec}
    for k in range(256 * vec, classes, 256 * vec):
        at |= {k - 1, k}
    at |= set(range(17, classes, classes // 20 + 1))
    return sorted(p for p in at if 0 <= p < classes)


def spiked(spike, classes, dtype):
    z = torch.full((len(spike), classes), -30.0, device="cuda", dtype=dtype)
    row, spike = torch.arange(len(spike), device="cuda"), torch.tensor(spike, device="cuda")
    labels = (spike + classes // 3 + 1) % classes
    z[row, labels] = -1.0
    z[row, spike] = 0.0
    total = 1 + math.exp(-1) + (classes - 2) * math.exp(-30)
    slope = torch.full((len(spike), classes), -math.exp(-30) / total, device="cuda", dtype=torch.float64)
    slope[row, labels], slope[row, spike] = 1 - math.exp(-1) / total, -1 / total
    return z.requires_grad_(), labels, -1 - math.log(total), slope


def close(grad, want, dtype, by=1.0):
    half, smallest = torch.finfo(dtype).eps / 2, {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -24}[dtype]
    assert ((grad.double() - want).abs() <= want.abs() * half + 15 * U * by * (1 + half) + smallest).all()


def check_places(rows, classes, dtype, at):
    for first in range(0, len(at), rows):
        spike = (at[first:first + rows] * rows)[:rows]
        z, labels, value, slope = spiked(spike, classes, dtype)
        lp = losses.label_log_probs(z, labels)
        assert ((lp.double() - value).abs() <= 9 * U).all()
        close(torch.autograd.grad(lp, z, torch.ones_like(lp))[0], slope, dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("classes", [2, 3, 4, 7, 8, 9, 15, 17, 33, 63, 65, 100, 257, 511, 1003, 2047, 4095])
def test_every_class_of_short_rows(classes, dtype):
    check_places(classes, classes, dtype, list(range(classes)))


# rows held by 256 and by 512 work-items (16 bits; fp32 in parts), read by 256, read in parts, one row in parts
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows, classes", [(600, 9001), (300, 50001), (720, 9001), (720, 50003), (20, 131071), (1, 16403), (1, 131071)])
def test_classes_of_long_rows(rows, classes, dtype):
    at = places(classes, 4 if dtype == torch.float32 else 8)
    check_places(rows, classes, dtype, at if rows > 1 else at[:8] + at[8:-8:9] + at[-8:])


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows, classes", [(70000, 257), (17000, 1003), (600, 30001), (600, 60001), (520, 131071)])
def test_classes_of_rows_whose_gradient_is_made_with_the_loss(rows, classes, dtype):
    """The policy loss at ratio 1 and an advantage of -1: the same gradients over the number of rows."""
    if dtype == torch.float32 and classes > 65536:
        classes = 65535         # the longest row that a workgroup holds
    assert rows * classes * dtype.itemsize >= 32 << 20
    at = places(classes, 4 if dtype == torch.float32 else 8) if classes > 4096 else list(range(classes))
    z, labels, value, slope = spiked((at * rows)[:rows], classes, dtype)
    one = torch.ones(rows, device="cuda")
    loss, stats = losses.policy_loss(z, labels, value * one, -one)
    grad, = torch.autograd.grad(loss, z)
    assert abs(loss.item() - 1) <= 16 * U and abs(stats[0].item() - 1) <= 16 * U
    close(grad, slope / rows, dtype, 2 / rows)


# ---- rows of any values -------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("spread", [1.0, 4.0])
@pytest.mark.parametrize("rows, classes", [(300, 10), (200, 33), (100, 1003), (70, 4095), (600, 9001), (300, 50001), (720, 9001), (720, 20003), (20, 131071), (1, 131071)])
def test_each_log_prob(rows, classes, spread, dtype):
    """Each row within what its own values allow: a term at distance v is off by 2 |v| u (the difference, the product) and 2 u (exp2), and by 2 u each time that
    its sum is scaled, to each maximum of a work-item's share, which has at most classes / 4096 + 20 steps with the joins (the distances add up to v); sums
    of up to 32 values lose 5 u; the logarithm is off by 2e-9 and the result by half a step, 2^-24 of its size."""
    g = torch.Generator(device="cuda").manual_seed(rows + classes)
    z = (torch.randn(rows, classes, generator=g, device="cuda") * spread).to(dtype)
    labels = torch.randint(0, classes, (rows,), generator=g, device="cuda")
    scaled = 0 if classes <= 2048 else classes / 4096 + 20
    for first in range(0, rows, 100):
        d = z[first:first + 100].double()
        top = d.amax(1, keepdim=True)
        p = torch.softmax(d, 1)
        tol = (2 * (p * (top - d)).sum(1) + 7 + 2 * scaled) * U
        want = exact_values(z[first:first + 100], labels[first:first + 100])
        got = losses.label_log_probs(z, labels)[first:first + 100]
        assert ((got.double() - want).abs() <= tol + U * want.abs() + 2e-9).all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("classes", [1000, 9000, 131072])
def test_logarithms_and_their_differences(classes, dtype):
    """Rows of n equal values and -inf, whose sum is n exactly: log prob - ref = -log n - ref, with a reference a few steps away, within the 2e-9 of the
    logarithm, 4 steps of 64 bits at log n < 12, and half a step of the result; the reward, beta = 1, is that of one row, and a log prob is -log n stored."""
    rows = 800
    g = torch.Generator().manual_seed(classes)
    n = torch.cat((torch.arange(1, 201), torch.randint(1, classes + 1, (rows - 200,), generator=g))).cuda()
    z = torch.full((rows, classes), 2.5, device="cuda", dtype=dtype)
    z.masked_fill_(torch.arange(classes, device="cuda") >= n.view(-1, 1), -math.inf)
    labels = (torch.rand(rows, device="cuda") * n).long().clamp(max=n - 1)
    want = -n.double().log()
    ref = (want + 1e-6 * torch.randn(rows, generator=g).cuda()).float()
    lp = losses.label_log_probs(z, labels)
    assert ((lp.double() - want).abs() <= 2.1e-9 + U * want.abs()).all()
    _, rewards = losses.preference_loss(z, labels, ref, beta=1.0)
    exact = want - ref.double()
    assert ((rewards.double() - exact).abs() <= 2.1e-9 + 2 * U * exact.abs()).all()
