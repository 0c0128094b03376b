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
