"""The operators on logits as they are used together: a teacher's lists and the student that learns from them, answers under a grammar, a policy that learns under a
mask of its actions.  Tolerances: those of the single operators' tests, rounded up to a few units of the types."""
import math
import threading

import pytest
import torch

from sortnet_amd import functional as F
from sortnet_amd import losses
from sortnet_amd.ell_inf_models import SortHybridModel

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows, classes, k, temperature", [(64, 10, 3, 2.0), (9, 1000, 1000 // 8, 1.0), (6, 40000, 64, 0.7)])
def test_lists_of_a_teacher(rows, classes, k, temperature):
    """top_logits makes what distill_loss reads.  With a list of all classes the divergence is the whole softmaxes'; a student that is its teacher has none, and no gradient."""
    g = torch.Generator().manual_seed(rows)
    teacher, student = (2.5 * torch.randn(rows, classes, generator=g).cuda() for _ in range(2))
    student.requires_grad_()
    lists = F.top_logits(teacher, k, temperature)
    loss, divergences = losses.distill_loss(student, *lists, temperature=temperature)
    q, p = (torch.log_softmax(t.detach().double() / temperature, 1) for t in (teacher, student))
    at = lists[1].long()
    q_top, p_top = q.gather(1, at), p.gather(1, at)
    q_rest, p_rest = (torch.logsumexp(t.scatter(1, at, -math.inf), 1) for t in (q, p))
    want = (q_top.exp() * (q_top - p_top)).sum(1) + q_rest.exp() * (q_rest - p_rest)
    torch.testing.assert_close(divergences.double(), want, rtol=1e-4, atol=2e-4)
    torch.testing.assert_close(loss.double(), temperature ** 2 * want.mean(), rtol=1e-4, atol=2e-4)
    own = teacher.clone().requires_grad_()
    loss, divergences = losses.distill_loss(own, *lists, temperature=temperature)
    grad, = torch.autograd.grad(loss, own)
    assert divergences.abs().max() <= 1e-4 and grad.abs().max() <= 1e-4 * temperature / rows
    if classes <= 256:
        every = F.top_logits(teacher, classes, temperature)
        assert (every[2] == -math.inf).all()
        whole = losses.distill_loss(student, *every, temperature=temperature)[1]
        torch.testing.assert_close(whole.double(), (q.exp() * (q - p)).sum(1), rtol=1e-4, atol=1e-5)


def test_answers_under_a_grammar():
    """What may be chosen, in order: constrain_logits before top_logits, one token and a batch, more asked for than allowed."""
    g = torch.Generator().manual_seed(2)
    z = (3 * torch.randn(5, 30000, generator=g)).to(torch.bfloat16).cuda()
    flags = (torch.rand(5, 30000, generator=g) < 0.001).cuda()
    flags[4] = False
    history = torch.randint(0, 30000, (5, 100), generator=g).cuda()
    shaped = F.constrain_logits(z, history, repetition=1.3, allowed=flags)
    values, classes, rest = F.top_logits(shaped, 64)
    for r in range(5):
        alive = flags[r].nonzero().view(-1)
        n = min(64, alive.numel())
        assert set(classes[r, :n].tolist()) <= set(alive.tolist()) and (values[r, n:] == -math.inf).all()
        assert torch.equal(values[r], shaped[r][classes[r].long()])
        if n < 64:
            assert rest[r] == -math.inf
            assert classes[r, n:].tolist() == [c for c in range(64 + n) if not flags[r, c]][:64 - n]
        one = F.top_logits(shaped[r:r + 1], 64)
        assert torch.equal(one[0][0], values[r]) and torch.equal(one[1][0], classes[r])


def test_policy_under_a_mask():
    """A policy learns under the mask its actions were drawn with: actions that are not allowed get no gradient, the others that of a softmax over what is allowed."""
    g = torch.Generator().manual_seed(3)
    z = torch.randn(40, 12, generator=g).cuda().requires_grad_()
    flags = (torch.rand(40, 12, generator=g) < 0.6).cuda()
    flags[:, 3] = True
    actions = torch.where(flags, torch.randn(40, 12, generator=g).cuda(), -math.inf).argmax(1)
    old = losses.label_log_probs(F.constrain_logits(z.detach(), allowed=flags), actions) - 0.05 * torch.randn(40, generator=g).cuda()
    advantages = torch.randn(40, generator=g).cuda()
    loss, _ = losses.policy_loss(F.constrain_logits(z, allowed=flags), actions, old, advantages, clip=0.5)
    grad, = torch.autograd.grad(loss, z)
    zd = z.detach().double().requires_grad_()
    lp = torch.log_softmax(zd.masked_fill(~flags, -math.inf), 1).gather(1, actions.view(-1, 1)).squeeze(1)
    ratio, adv = (lp - old.double()).exp(), advantages.double()
    want = -torch.minimum(ratio * adv, ratio.clamp(0.5, 1.5) * adv).mean()
    torch.testing.assert_close(loss.double(), want, rtol=1e-5, atol=1e-6)
    torch.testing.assert_close(grad.double(), torch.autograd.grad(want, zd)[0], rtol=1e-4, atol=1e-6)
    assert (grad[~flags] == 0).all()


def test_model_learns_from_a_model():
    """A hybrid model's step on another one's lists, and the step in a captured graph: the logits' gradient reaches every parameter of the head."""
    torch.manual_seed(0)
    student, teacher = (SortHybridModel(3, 64, (1, 8, 8), hidden=32, num_classes=20).cuda() for _ in range(2))
    x = torch.rand(16, 1, 8, 8, device="cuda")
    with torch.no_grad():
        lists = F.top_logits(teacher.eval()(x), 5, 2.0)
    student.eval()
    out = student(x)
    loss, divergences = losses.distill_loss(out, *lists, temperature=2.0, weight=0.5)
    grads = torch.autograd.grad(loss, [p for p in student.fc_final.parameters()])
    assert torch.isfinite(loss) and divergences.shape == (16,) and all(torch.isfinite(g).all() and g.abs().max() > 0 for g in grads)


def test_two_threads_at_once():
    """Two host threads, each on a stream of its own, get what one alone gets."""
    g = torch.Generator().manual_seed(9)
    sets = []
    for rows, classes, k, dtype in [(700, 40001, 20, torch.bfloat16), (3, 90001, 64, torch.float32), (900, 30, 4, torch.float16)]:
        z, t = ((2 * torch.randn(rows, classes, generator=g)).to(dtype).cuda() for _ in range(2))
        sets.append((z.requires_grad_(), t, k, torch.randint(0, classes, (rows, 40), generator=g).cuda(), (torch.rand(rows, classes, generator=g) < 0.7).cuda()))

    def chain(z, t, k, history, flags):
        lists = F.top_logits(F.constrain_logits(t, history, repetition=1.2, allowed=flags), k)
        loss, divergences = losses.distill_loss(F.constrain_logits(z, history, presence=0.5), *lists, temperature=1.5)
        return [t.clone() for t in (*lists, loss.detach(), divergences, torch.autograd.grad(loss, z)[0])]

    want = [chain(*s) for s in sets]
    torch.cuda.synchronize()
    wrong = []

    def work(first):
        with torch.cuda.stream(torch.cuda.Stream()):
            for n in range(12):
                i = (first + n) % len(sets)
                got = chain(*sets[i])
                torch.cuda.current_stream().synchronize()
                wrong.extend((first, n, j) for j, (a, b) in enumerate(zip(got, want[i])) if not torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_two_threads_finish_what_they_began():
    """The same from two threads whose errors are seen: every pass of both has come to its end."""
    g = torch.Generator().manual_seed(10)
    z, t = ((2 * torch.randn(600, 30001, generator=g)).to(torch.bfloat16).cuda() for _ in range(2))
    short, teacher = (torch.randn(500, 40, generator=g).cuda() for _ in range(2))
    history, flags = torch.randint(0, 40, (500, 12), generator=g).cuda(), (torch.rand(500, 40, generator=g) < 0.7).cuda()
    z.requires_grad_()
    short.requires_grad_()

    def large():
        loss, divergences = losses.distill_loss(z, *F.top_logits(t, 40), temperature=1.5)
        return loss.detach(), divergences, torch.autograd.grad(loss, z)[0]

    def small():
        shaped = F.constrain_logits(short, history, presence=0.5, allowed=flags)
        loss, divergences = losses.distill_loss(shaped, *F.top_logits(F.constrain_logits(teacher, allowed=flags), 4))
        return shaped.detach(), divergences, torch.autograd.grad(loss, short)[0]

    want = {f: [r.clone() for r in f()] for f in (large, small)}
    torch.cuda.synchronize()
    wrong, ended = [], []

    def work(first, second):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for n in range(12):
                    f = first if n % 2 == 0 else second
                    got = f()
                    torch.cuda.current_stream().synchronize()
                    wrong.extend((n, j) for j, (a, b) in enumerate(zip(got, want[f])) if not torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)))
                    ended.append(n)
        except BaseException as e:
            wrong.append(repr(e))

    threads = [threading.Thread(target=work, args=fs) for fs in ((large, small), (small, large))]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    assert not wrong and len(ended) == 24
