"""Distillation from a teacher's top logits against its definition in 64 bits.

Tolerances, with u = 2^-24, half a step of fp32.  The sum S over the other classes is off by at most delta = 2 (classes / 64 + 128) u of itself: a partial sum
takes classes / 64 + 64 steps at most, each of them, the exponential and its argument off by a few u.  What is done per outcome is in 64 bits, so log p is off by
delta, a divergence by 2 delta (the weights of what is off sum to 2 at most) and its rounding, u of it.  The gradient of an entry, w (p - q) with w = weight T / count, is
off by w p delta and four roundings; that of another class at distance d from the largest one, w (p_r - q_r) s with s its share of S, by w p_r delta s and
by (delta + (4 d / T + 8) u) of itself.  Stored results are off by half a step of their type and, below its normal range, by half its smallest number."""
import math

import pytest
import torch

from sortnet_amd import losses

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
SMALLEST = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}    # (numbers below fp32's normal range may be 0)


def sum_error(classes):
    return 2 * (classes / 64 + 128) * U


def make(rows, classes, k, dtype, seed, temperature=1.0, ignored=0.2, spread=2.5, teacher=torch.float32):
    """Logits, the entries and rest of a teacher that mostly agrees; some rows without entries."""
    g = torch.Generator().manual_seed(seed)
    z = (torch.randn(rows, classes, generator=g) * spread).to(dtype)
    t = z.float() + torch.randn(rows, classes, generator=g)
    top = t.topk(k, dim=1)
    rest = torch.logsumexp(t.scatter(1, top.indices, -math.inf) / temperature, 1)
    chosen = top.indices.clone()
    chosen[torch.rand(rows, generator=g) < ignored] = -1
    return z.cuda(), top.values.to(teacher).cuda(), chosen.cuda(), rest.cuda(), g


def exact(z, values, chosen, rest, temperature, weight):
    """loss, divergences, gradient and how far a kernel may be off in each; row by row in 64 bits on the CPU."""
    rows, classes = z.shape
    delta, dtype = sum_error(classes), z.dtype
    z, values, chosen = z.detach().double().cpu() / temperature, values.double().cpu() / temperature, chosen.cpu().long()
    rest = torch.full((rows,), -math.inf, dtype=torch.float64) if rest is None else rest.double().cpu()
    there = chosen >= 0
    teacher = torch.cat((values.masked_fill(~there, -math.inf), rest.view(-1, 1)), 1)
    counted = there.any(1) & ~(teacher == -math.inf).all(1)
    count = max(1, int(counted.sum()))
    w = weight * temperature / count
    D, D_off = torch.zeros(rows, dtype=torch.float64), torch.zeros(rows, dtype=torch.float64)
    grad, off = torch.zeros_like(z), torch.zeros_like(z)
    for r in counted.nonzero().view(-1).tolist():
        q = torch.softmax(teacher[r], 0)
        share = torch.zeros(classes, dtype=torch.float64)       # of q, by class
        listed = torch.zeros(classes, dtype=torch.bool)
        for j in there[r].nonzero().view(-1).tolist():
            share[chosen[r, j]] += q[j]
            listed[chosen[r, j]] = True
        log_p = torch.log_softmax(z[r], 0)
        log_pr = torch.logsumexp(log_p.masked_fill(listed, -math.inf), 0)
        mine = torch.cat((log_p[chosen[r].clamp(min=0)], log_pr.view(1)))
        live = q > 0
        D[r] = (q[live] * (q[live].log() - mine[live])).sum()
        D_off[r] = 2 * delta + U * D[r].abs() + 1e-12 * mine[live].abs().sum()
        p, pr = log_p.exp(), log_pr.exp()
        grad[r] = torch.where(listed, w * (p - share), 0.0)
        off[r] = torch.where(listed, abs(w) * (delta * p + 5 * U * (p - share).abs()), 0.0)
        if not listed.all() and log_pr > -math.inf:
            s = (log_p - log_pr).exp().masked_fill(listed, 0.0)
            far = (z[r][~listed].max() - z[r]).clamp(min=0, max=800)
            grad[r] += w * (pr - q[-1]) * s
            off[r] += abs(w) * s * (delta * pr + (pr - q[-1]).abs() * (delta + (4 * far + 8) * U))
    off = off + (grad.abs() + off) * torch.finfo(dtype).eps / 2 + SMALLEST[dtype]
    loss = weight * temperature ** 2 * D.sum() / count
    loss_off = abs(weight) * temperature ** 2 * D_off.sum() / count + 3 * U * loss.abs()
    return (loss, loss_off), (D, D_off), (grad, off), counted


def close(got, want, what):
    want, off = want
    got = got.detach().double().cpu()
    finite = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), finite), what
    worst = ((got - want).abs() - off)[finite]
    assert worst.numel() == 0 or worst.max() <= 0, "%s: %g over the tolerance" % (what, worst.max())


def check(z, values, chosen, rest, temperature=1.0, weight=1.0, up=None):
    leaf = z.detach().requires_grad_()
    loss, divergences = losses.distill_loss(leaf, values, chosen, rest, temperature=temperature, weight=weight)
    assert loss.shape == () and loss.dtype == torch.float32 and divergences.dtype == torch.float32 and divergences.shape == z.shape[:-1] and not divergences.requires_grad
    scale = 1.0 if up is None else up
    grad, = torch.autograd.grad(loss, leaf, None if up is None else torch.tensor(up, device="cuda"))
    want_loss, want_d, _, counted = exact(z, values, chosen, rest, temperature, weight)
    close(loss, want_loss, "loss")
    close(divergences, want_d, "divergences")
    want_grad = exact(z, values, chosen, rest, temperature, weight * scale)[2]
    assert grad.dtype == z.dtype and grad.shape == z.shape
    close(grad, want_grad, "gradient")
    assert (grad[~counted.cuda()] == 0).all() and (divergences[~counted.cuda()] == 0).all()
    with torch.no_grad():
        again = losses.distill_loss(z, values, chosen, rest, temperature=temperature, weight=weight)
    assert torch.equal(again[0], loss) and torch.equal(again[1], divergences)
    return loss, divergences, grad


SHAPES = [(1, 1, 1), (3, 2, 1), (5, 2, 2), (512, 10, 3), (77, 33, 7), (7, 257, 200), (300, 1000, 16), (64, 2048, 20), (13, 2049, 5), (9, 4097, 256), (3, 16385, 64), (2, 32769, 9),
          (1, 70001, 256), (33, 20001, 3), (2000, 40, 2)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows, classes, k", SHAPES)
def test_loss_and_gradient(rows, classes, k, dtype):
    z, values, chosen, rest, _ = make(rows, classes, k, dtype, rows * 3 + classes, 2.0)
    check(z, values, chosen, rest, 2.0, weight=64.0)
    check(z, values, chosen.int(), None, 1.0, weight=-3.0, up=16.0)


@pytest.mark.parametrize("rows, classes, k, dtype", [(17001, 1003, 3, torch.bfloat16), (5200, 4100, 3, torch.float16), (1400, 8003, 40, torch.float32), (720, 30001, 256, torch.bfloat16),
                                                     (512, 131072, 5, torch.bfloat16), (2100, 33001, 20, torch.float32), (70003, 2005, 2, torch.bfloat16)])
def test_gradient_with_the_loss(rows, classes, k, dtype):
    """Large batches, for most of which the gradient is made with the loss: some rows against the definition, all of them against the loss."""
    z, values, chosen, rest, g = make(rows, classes, k, dtype, classes)
    leaf = z.requires_grad_()
    loss, divergences = losses.distill_loss(leaf, values, chosen, rest, temperature=0.8, weight=64.0)
    grad, = torch.autograd.grad(loss, leaf, retain_graph=True)
    counted = (chosen >= 0).any(1)
    some = torch.cat((torch.tensor([0, 1, rows - 1]), torch.randint(0, rows, (30,), generator=g))).cuda()
    share = int(counted[some].sum()) / int(counted.sum())
    _, want_d, want_grad, _ = exact(z[some], values[some], chosen[some], rest[some], 0.8, 64.0 * share)
    close(divergences[some], want_d, "divergences")
    close(grad[some], want_grad, "gradient")
    assert (grad[~counted] == 0).all() and (divergences[~counted] == 0).all()
    # (a mean of numbers of fp32 in 64 bits and two products: rounded once at the end)
    want = 64.0 * 0.8 ** 2 * divergences.double().sum() / counted.sum()
    assert abs(loss.double() - want) <= 2 * U * want.abs()
    twice, = torch.autograd.grad(loss, leaf, torch.tensor(-2.0, device="cuda"))
    _, _, want_grad, _ = exact(z[some], values[some], chosen[some], rest[some], 0.8, -128.0 * share)
    close(twice[some], want_grad, "gradient")


def test_more_workgroups_than_a_launch_has():
    rows = (1 << 26) + 70
    z = torch.randn(1 << 12, 12, device="cuda").half().repeat((1 << 14) + 1, 1)[:rows].requires_grad_()
    chosen = torch.full((rows, 1), 3, device="cuda", dtype=torch.int32)
    values = torch.zeros(rows, 1, device="cuda")
    loss, divergences = losses.distill_loss(z, values, chosen, weight=float(rows))
    grad, = torch.autograd.grad(loss, z)
    assert torch.equal(divergences[:1 << 12], divergences[1 << 25:(1 << 25) + (1 << 12)]) and torch.equal(grad[:1 << 12], grad[1 << 25:(1 << 25) + (1 << 12)])
    assert torch.equal(divergences[-70:], divergences[:70]) and torch.equal(grad[-70:], grad[:70])
    want = -torch.log_softmax(z[:1 << 12].detach().double(), 1)[:, 3]       # (q is 1 for the only entry)
    assert ((divergences[:1 << 12] - want).abs() <= 2 * sum_error(12) + U * want.abs()).all()


@pytest.mark.parametrize("temperature", [0.1, 0.5, 1.0, 3.0, 100.0])
@pytest.mark.parametrize("teacher", TYPES, ids=str)
def test_temperatures_and_types_of_the_teacher(teacher, temperature):
    z, values, chosen, rest, _ = make(20, 700, 10, torch.bfloat16, 5, temperature, teacher=teacher)
    check(z, values, chosen, rest, temperature)


@pytest.mark.parametrize("classes", [6, 900, 20000])
def test_lists_of_different_lengths_and_repeats(classes):
    """Entries of -1 anywhere, classes that stand in several entries, values of -inf, rests of -inf; the same class in all entries."""
    z, values, chosen, rest, g = make(12, classes, 5, torch.float32, classes, ignored=0.0)
    chosen[0, 1:] = -1
    chosen[1, 0] = -7
    chosen[2, 3] = chosen[2, 0]
    chosen[3] = chosen[3, 2].clone()
    chosen[4, 4] = chosen[4, 1]
    chosen[4, 3] = chosen[4, 1]
    values[5, 1:] = -math.inf
    values[6] = -math.inf
    values[7] = -math.inf
    rest[7] = rest[8] = -math.inf
    values[9, 0] = 60.0
    rest[10] = 50.0
    check(z, values, chosen, rest)
    check(z, values, chosen, None, 1.5, up=0.25)


def test_teacher_and_student_alike():
    """Divergences near 0 and what the student gives the others however little it is: rows whose entries hold all but 1e-30 of it."""
    z, values, chosen, rest, _ = make(8, 3000, 4, torch.float32, 1, ignored=0.0)
    values = z.gather(1, chosen)
    rest = torch.logsumexp(z.double().scatter(1, chosen, -math.inf), 1).float()
    loss, divergences, _ = check(z, values, chosen, rest)
    assert divergences.abs().max() <= 2 * sum_error(3000)
    z[:, 7:] -= 70.0
    chosen = torch.arange(4, device="cuda").expand(8, 4).contiguous()
    z[:, 4:7] = -60.0
    values = z.gather(1, chosen)
    check(z, values, chosen, rest - 70.0)
    far = z.clone()
    far[:, 4:] -= 3000.0            # below the smallest exponential
    check(far, values, chosen, rest - 70.0)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("classes", [5, 700, 20000])
def test_masked_classes(classes, dtype):
    """The student's -inf and its type's lowest value: among the others, among the entries, all of the others."""
    z, values, chosen, rest, _ = make(6, classes, 2, dtype, classes, ignored=0.0)
    z[0, classes // 2:] = -math.inf
    z[1, :classes // 2] = torch.finfo(dtype).min
    chosen[0], chosen[1] = torch.tensor([0, 1]), torch.tensor([classes - 1, classes - 2])
    z[2] = torch.finfo(dtype).min
    z[3, 2:] = -math.inf            # nothing is left for the others, and the teacher gives them nothing
    chosen[3] = torch.tensor([0, 1])
    rest[3] = -math.inf
    check(z, values, chosen, rest)
    z[4, 2:] = -math.inf            # the teacher gives classes what the student cannot
    chosen[4] = torch.tensor([1, 0])
    z[5, 1] = -math.inf
    chosen[5] = torch.tensor([1, 2])
    leaf = z.detach().requires_grad_()
    loss, divergences = losses.distill_loss(leaf, values, chosen, rest)
    assert loss == math.inf and divergences[4] == math.inf and divergences[5] == math.inf and torch.isfinite(divergences[1:4]).all()
    assert (divergences[0] == math.inf) == (classes == 5)       # (of five classes the mask takes all three that are in no entry)
    grad, = torch.autograd.grad(loss, leaf)
    assert torch.isfinite(grad).all() and (grad[4, 2:] == 0).all() and grad[5, 1] < 0


@pytest.mark.parametrize("classes", [7, 900, 20000])
def test_rows_without_values(classes):
    """Rows that do not count hold anything; NaN, infinities and classes past the end give NaN in their row alone."""
    z, values, chosen, rest, _ = make(9, classes, 3, torch.float32, 3, ignored=0.0)
    clean = losses.distill_loss(z, values, chosen, rest)[1]
    z[0], z[1] = math.nan, math.inf
    chosen[0] = -1
    rest[0] = math.nan
    values[1], rest[1] = -math.inf, -math.inf
    chosen[2, 1] = classes
    z[3, (chosen[3, 0] + 1) % classes] = math.nan
    values[4, 2] = math.nan
    rest[5] = math.nan
    z[6] = -math.inf
    z[7, chosen[7, 1]] = math.inf
    z.requires_grad_()
    loss, divergences = losses.distill_loss(z, values, chosen, rest)
    assert torch.isnan(loss) and (divergences[:2] == 0).all() and torch.isnan(divergences[2:8]).all() and divergences[8] == clean[8]
    grad, = torch.autograd.grad(loss, z)
    assert (grad[:2] == 0).all() and torch.isnan(grad[2:6]).all() and torch.isnan(grad[7]).any() and torch.isfinite(grad[8]).all()
    nothing = torch.full_like(chosen, -1)
    loss, divergences = losses.distill_loss(z, values, nothing, rest)
    assert loss == 0 and (divergences == 0).all() and (torch.autograd.grad(loss, z)[0] == 0).all()


@pytest.mark.parametrize("classes", [10, 1000, 20001])
def test_strides(classes):
    g = torch.Generator().manual_seed(classes)
    base = torch.randn(6, 9, classes + 3, generator=g).to(torch.bfloat16).cuda()
    t = torch.randn(6, 9, classes, generator=g).cuda().topk(4)
    rest = torch.randn(6, 9, generator=g).cuda()
    for z in (base[:, :, 1:classes + 1], base[..., :classes], base.transpose(0, 1)[..., 2:classes + 2].transpose(0, 1), base[:1, :1, :classes].expand(6, 9, classes)):
        flat = z.detach().reshape(54, classes).contiguous().requires_grad_()
        want = losses.distill_loss(flat, t.values.view(54, 4), t.indices.view(54, 4), rest.view(54), temperature=2.0)
        leaf = z.detach().requires_grad_()
        wide_values, wide_classes = torch.stack((t.values, t.values), -1)[..., 0], torch.stack((t.indices, t.indices), -1)[..., 1]
        got = losses.distill_loss(leaf, wide_values, wide_classes, rest.t().contiguous().t(), temperature=2.0)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1].view(54), want[1])
        assert torch.equal(torch.autograd.grad(got[0], leaf)[0].reshape(54, classes), torch.autograd.grad(want[0], flat)[0])
    four = base[..., :classes].reshape(3, 2, 9, classes)
    got = losses.distill_loss(four, t.values.view(3, 2, 9, 4), t.indices.view(3, 2, 9, 4), rest.view(3, 2, 9))
    assert torch.equal(got[1].view(6, 9), losses.distill_loss(base[..., :classes], t.values, t.indices, rest)[1])


def test_gradient_by_differences():
    z, values, chosen, rest, _ = make(2, 9, 3, torch.float32, 4, ignored=0.0)
    leaf = z.clone().requires_grad_()
    loss = lambda t: losses.distill_loss(t, values, chosen, rest)[0].double().item()
    grad, = torch.autograd.grad(losses.distill_loss(leaf, values, chosen, rest)[0], leaf)
    step = 2.0 ** -6
    # central differences are off by the third derivative, at most 1 for a softmax's logarithm, times step^2 / 6, and by the rounding of two losses below 8
    off = step ** 2 / 6 + 2 * (sum_error(9) * 2 + 8 * U) / step / 2
    for i in range(2):
        for j in range(9):
            move = torch.zeros_like(z)
            move[i, j] = step
            assert abs((loss(z + move) - loss(z - move)) / (2 * step) - grad[i, j].item()) <= off


def test_second_derivatives_and_transforms_are_refused():
    z, values, chosen, rest, _ = make(3, 9, 2, torch.float32, 4, ignored=0.0)
    leaf = z.clone().requires_grad_()
    grad, = torch.autograd.grad(losses.distill_loss(leaf, values, chosen, rest)[0], leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiated once"):
        torch.autograd.grad(grad.sum(), leaf)
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level():
        for args in ((fwd.make_dual(z, z), values, chosen, rest), (z, fwd.make_dual(values, values), chosen, rest), (z, values, chosen, fwd.make_dual(rest, rest))):
            with pytest.raises(NotImplementedError, match="forward mode"):
                losses.distill_loss(*args)


def test_refusals():
    z, values, chosen, rest, _ = make(4, 9, 3, torch.float32, 4)
    for match, call in [
            ("classes", lambda: losses.distill_loss(z[0], values[0], chosen[0])), ("top_values must have the sizes", lambda: losses.distill_loss(z, values[:2], chosen[:2])),
            ("top_classes must have the sizes of top_values", lambda: losses.distill_loss(z, values, chosen[:, :2])), ("top_classes must have dtype", lambda: losses.distill_loss(z, values, values)),
            ("top_values must have dtype", lambda: losses.distill_loss(z, values.double(), chosen)), ("top_rest must have dtype", lambda: losses.distill_loss(z, values, chosen, rest.half())),
            ("top_rest must have the sizes", lambda: losses.distill_loss(z, values, chosen, rest.view(4, 1))), ("top_rest must be a CUDA", lambda: losses.distill_loss(z, values, chosen, rest.cpu())),
            ("top_values must not require", lambda: losses.distill_loss(z, values.clone().requires_grad_(), chosen)),
            ("top_rest must not require", lambda: losses.distill_loss(z, values, chosen, rest.clone().requires_grad_())), ("k=0", lambda: losses.distill_loss(z, values[:, :0], chosen[:, :0])),
            ("k=257", lambda: losses.distill_loss(z, values[:, :1].expand(4, 257), chosen[:, :1].expand(4, 257))), ("temperature=0", lambda: losses.distill_loss(z, values, chosen, temperature=0)),
            ("temperature=nan", lambda: losses.distill_loss(z, values, chosen, temperature=math.nan)), ("weight=inf", lambda: losses.distill_loss(z, values, chosen, weight=math.inf)),
            ("rows=0", lambda: losses.distill_loss(z[:0], values[:0], chosen[:0]))]:
        with pytest.raises(RuntimeError, match=match):
            call()


@pytest.mark.parametrize("rows, classes", [(40, 10), (5, 20001), (700, 50001)])
def test_captured_and_on_other_streams(rows, classes):
    """A graph reads logits, lists and the upstream gradient in each replay; eager calls run beside it on another stream."""
    z, values, chosen, rest, g = make(rows, classes, 3, torch.bfloat16, 3)
    leaf, up = z.clone().requires_grad_(), torch.ones((), device="cuda")

    def step():
        loss, divergences = losses.distill_loss(leaf, values, chosen, rest, temperature=2.0)
        return loss.detach(), divergences, torch.autograd.grad(loss, leaf, up)[0]

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    side = torch.cuda.Stream()
    for n in range(4):
        up.fill_([1.0, 3.0, 1.0, 0.5][n])
        chosen.copy_(torch.stack([torch.randperm(classes, generator=g)[:3] for _ in range(rows)]))
        chosen[n] = -1
        with torch.no_grad():
            leaf.add_(torch.randn(rows, classes, generator=g).cuda().to(leaf.dtype))
        graph.replay()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            want = step()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), n


def _save_on_cpu_and_back(t):
    """A saved tensor as a hook that keeps it on the host hands it back: as large, contiguous."""
    return torch.empty(t.shape, dtype=t.dtype, device="cuda").copy_(t)


def _turned(t):
    """The same with another order of its last two dimensions in memory."""
    return t.transpose(-1, -2).contiguous().transpose(-1, -2) if t.dim() > 1 else t


@pytest.mark.parametrize("unpack", [_save_on_cpu_and_back, _turned])
@pytest.mark.parametrize("rows, classes", [(40, 10), (7, 9001), (3, 140001)])
def test_saved_tensors_that_come_back_laid_out_otherwise(rows, classes, unpack):
    """Hooks may hand back what a call saved with other strides than it had: the gradients of all losses on logits read it as it lies then."""
    z, values, chosen, rest, g = make(rows, classes, 3, torch.bfloat16, 8, ignored=0.0)
    leaf = z.requires_grad_()
    labels = torch.randint(0, classes, (rows,), generator=g).cuda()
    runs = [lambda: losses.distill_loss(leaf, values, chosen, rest, temperature=2.0)[0],
            lambda: losses.label_log_probs(leaf, labels).sum(),
            lambda: losses.policy_loss(leaf, labels, torch.full((rows,), -3.0, device="cuda"), torch.ones(rows, device="cuda"))[0]]
    for run in runs:
        want, = torch.autograd.grad(run(), leaf)
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
            out = run()
        got, = torch.autograd.grad(out, leaf)
        assert torch.equal(got, want)


@pytest.mark.parametrize("classes", [6, 900, 20000, 140001])
def test_entries_of_one_class(classes):
    """A class of several entries is one class of the student's and takes the sum of their q in the gradient; the divergence is a sum over the entries, each with its own
    q log q.  It lies below that of a list in which they are one entry by the sum of q_j log(q / q_j), which the logits do not change."""
    g = torch.Generator().manual_seed(classes)
    z = torch.randn(1, classes, generator=g).cuda().requires_grad_()
    twice = losses.distill_loss(z, torch.zeros(1, 2, device="cuda"), torch.full((1, 2), 3, device="cuda"))
    once = losses.distill_loss(z, torch.zeros(1, 1, device="cuda"), torch.full((1, 1), 3, device="cuda"))
    off = 4 * sum_error(classes) + 2 * U * once[1].item()
    assert abs((once[1] - twice[1]).item() - math.log(2.0)) <= off      # (q = 1/2 twice)
    a, b = (torch.autograd.grad(loss, z)[0] for loss, _ in (twice, once))
    assert ((a - b).abs() <= 2 * U * a.abs() + 2.0 ** -126).all()       # (1/2 + 1/2 is 1 in 64 bits; one rounding each)
    sure = torch.full((1, classes), -200.0, device="cuda")
    sure[0, 3] = 200.0
    assert abs(losses.distill_loss(sure, torch.zeros(1, 2, device="cuda"), torch.full((1, 2), 3, device="cuda"))[1].item() + math.log(2.0)) <= 2 * U


@pytest.mark.parametrize("rows, classes, k, dtype", [(540, 65537, 7, torch.float32), (600, 65536, 7, torch.float32), (520, 131073, 256, torch.bfloat16), (515, 140007, 20, torch.float16)])
def test_batches_of_rows_that_no_workgroup_holds(rows, classes, k, dtype):
    """Large batches on both sides of the longest row that a workgroup holds, 16384 vectors of 16 bytes: beyond it rows are read in parts and the gradient is made by itself."""
    test_gradient_with_the_loss(rows, classes, k, dtype)
