"""Penalties, biases and masks of logits against their definition in 64 bits.

Tolerances, with u = 2^-24, half a step of fp32: the penalised value is a quotient or product with a number that is rounded to fp32 (2 u), two
differences and a sum, each off by u of its size, which is at most the sum of the sizes of what went in: 6 u of that sum.  A gradient is one product or
quotient: 2 u.  Stored results are off by half a step of their type, and below its normal range by half its smallest number."""
import math

import pytest
import torch

from sortnet_amd import functional as F

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
SMALLEST = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}    # (numbers below fp32's normal range may be 0)


def words_of(flags):
    """bool (..., classes) as int32 (..., words)"""
    classes = flags.size(-1)
    bits = torch.nn.functional.pad(flags, (0, -classes % 32)).view(*flags.shape[:-1], -1, 32).long()
    words = (bits << torch.arange(32, device=flags.device)).sum(-1)
    return (words - ((words >> 31) << 32)).to(torch.int32)


def exact(z, history=None, lengths=None, repetition=1.0, presence=0.0, frequency=0.0, bias=None, flags=None, grad=None):
    """(result, its tolerance, gradient, its tolerance) of contiguous rows, in 64 bits on the CPU, class by class."""
    rows, classes = z.shape
    dtype, z = z.dtype, z.detach().double().cpu()
    of_row = lambda v: v.double().cpu().view(-1, 1) if isinstance(v, torch.Tensor) else torch.full((rows, 1), float(v), dtype=torch.float64)
    rep, pres, freq = of_row(repetition), of_row(presence), of_row(frequency)
    count = torch.zeros(rows, classes, dtype=torch.float64)
    if history is not None:
        for r, past in enumerate(history.cpu().tolist()):
            for token in past[:None if lengths is None else max(0, int(lengths[r]))]:
                if 0 <= token < classes:
                    count[r, token] += 1
    seen = count > 0
    factor = torch.where(seen, torch.where(z > 0, 1 / rep, rep), 1.0)
    y = torch.where(seen, z * factor - freq * count - pres, z)
    sizes = (z * factor).abs() + (freq * count).abs() + seen * pres.abs()
    if bias is not None:
        y = y + bias.double().cpu()
        sizes = sizes + bias.double().cpu().abs()
    tol = 6 * U * sizes if history is not None or bias is not None else torch.zeros_like(z)
    g = g_tol = None
    if grad is not None:
        g = grad.double().cpu() * factor
        g_tol = 2 * U * g.abs() * seen
    if flags is not None:
        y = y.masked_fill(~flags.cpu(), -math.inf)
        if g is not None:
            g = g.masked_fill(~flags.cpu(), 0.0)
    half = torch.finfo(dtype).eps / 2
    tol = tol + (y.abs() + tol) * half + SMALLEST[dtype]
    if g is not None:
        g_tol = g_tol + (g.abs() + g_tol) * half + SMALLEST[dtype]
    return y, tol, g, g_tol


def close(got, want, tol, what):
    got = got.detach().double().cpu()
    finite = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), finite) and torch.equal(got[~finite], want[~finite]), what
    worst = ((got - want).abs() - tol)[finite]
    assert worst.numel() == 0 or worst.max() <= 0, "%s: %g over the tolerance" % (what, worst.max())


def make(rows, classes, dtype, seed, places=0):
    g = torch.Generator().manual_seed(seed)
    z = (3 * torch.randn(rows, classes, generator=g)).to(dtype).cuda()
    history = torch.randint(0, max(1, min(classes, 2 * places)), (rows, places), generator=g).cuda() if places else None
    return z, history, g


def check(z, flags=None, bits=False, grad_seed=5, **given):
    """Forward and backward on z against the definition; returns the result."""
    g = torch.Generator().manual_seed(grad_seed)
    up = torch.randn(z.shape, generator=g).to(z.dtype).cuda()
    allowed = None if flags is None else words_of(flags) if bits else flags
    leaf = z.detach().requires_grad_()
    out = F.constrain_logits(leaf, allowed=allowed, **given)
    assert out.dtype == z.dtype and out.shape == z.shape and out.is_contiguous()
    got, = torch.autograd.grad(out, leaf, up)
    y, tol, want, g_tol = exact(z, flags=flags, grad=up, **given)
    close(out, y, tol, "result")
    close(got, want, g_tol, "gradient")
    with torch.no_grad():
        assert torch.equal(F.constrain_logits(z, allowed=allowed, **given), out)
    return out


SHAPES = [(1, 1, 1), (5, 2, 3), (3, 7, 1), (300, 10, 4), (40, 33, 7), (7, 257, 100), (3, 1000, 2000), (2, 2049, 5), (5, 8191, 300), (3, 8193, 257), (2, 20001, 1000), (1, 70003, 4000)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows, classes, places", SHAPES)
def test_everything_at_once(rows, classes, places, dtype):
    z, history, g = make(rows, classes, dtype, rows * 7 + classes, places)
    lengths = torch.randint(0, places + 1, (rows,), generator=g).cuda()
    flags = (torch.rand(rows, classes, generator=g) < 0.7).cuda()
    numbers = [t.cuda() for t in (0.7 + torch.rand(rows, generator=g), torch.randn(rows, generator=g), 0.3 * torch.randn(rows, generator=g))]
    bias = torch.randn(rows, classes, generator=g).cuda()
    check(z, flags, history=history, lengths=lengths, repetition=numbers[0], presence=numbers[1], frequency=numbers[2], bias=bias)
    check(z, flags, True, history=history.int(), lengths=lengths.int(), repetition=1.3, presence=0.25, frequency=0.5, bias=bias[0])


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows, classes", [(9, 5), (3, 700), (2, 9001)])
def test_one_thing_at_a_time(rows, classes, dtype):
    z, history, g = make(rows, classes, dtype, classes, 20)
    flags = (torch.rand(rows, classes, generator=g) < 0.5).cuda()
    check(z, history=history, repetition=1.5)
    check(z, history=history, presence=0.5)
    check(z, history=history, frequency=-0.25)
    check(z, bias=torch.randn(classes, generator=g).cuda())
    check(z, flags)
    check(z, flags, True)
    assert torch.equal(check(z), z) and torch.equal(check(z, history=history), z) and torch.equal(check(z, history=history[:, :0], repetition=2.0), z)
    assert torch.equal(check(z, flags[0].expand(rows, classes)), F.constrain_logits(z, allowed=flags[0]))
    assert torch.equal(check(z, flags[0].expand(rows, classes)), F.constrain_logits(z, allowed=words_of(flags[0])))


def test_rows_with_nothing_allowed_and_odd_values():
    """Rows that may choose nothing are -inf with a gradient of zeros, whatever they hold; infinities and NaN pass through the others."""
    z = torch.tensor([[1.0, -2.0, 3.0], [math.nan, math.inf, -math.inf], [math.nan, math.inf, -math.inf], [0.0, -0.0, 1.0]], device="cuda", requires_grad=True)
    flags = torch.tensor([[False] * 3, [False] * 3, [True] * 3, [True] * 3], device="cuda")
    history = torch.tensor([[0, 1, 2]] * 4, device="cuda")
    for allowed in (flags, words_of(flags)):
        out = F.constrain_logits(z, history, repetition=2.0, presence=1.0, allowed=allowed)
        assert (out[:2] == -math.inf).all() and torch.isnan(out[2, 0]) and out[2, 1] == math.inf and out[2, 2] == -math.inf
        assert out[3].tolist() == [-1.0, -1.0, -0.5]
        grad, = torch.autograd.grad(out, z, torch.full_like(out, 3.0))
        assert (grad[:2] == 0).all() and grad[2, 1] == 1.5 and grad[2, 2] == 6.0 and grad[3].tolist() == [6.0, 6.0, 1.5]


def test_places_that_hold_no_class():
    """A padding of any negative number, classes past the end, lengths past the ends and 64-bit numbers whose low half names a class."""
    z = torch.randn(4, 9, device="cuda")
    history = torch.tensor([[3, -1, 3, 9], [-100, 1 << 32, (1 << 32) + 2, -(1 << 32) + 2], [8, 8, 8, 8], [0, 1, 2, 3]], device="cuda")
    lengths = torch.tensor([4, 4, 100, -3], device="cuda")
    out = F.constrain_logits(z, history, lengths, frequency=1.0)
    want = z.clone()
    want[0, 3] -= 2
    want[2, 8] -= 4
    assert torch.equal(out, want)
    many = torch.full((1, 100000), 5, device="cuda", dtype=torch.int32)     # one class, often
    out = F.constrain_logits(z[:1], many, frequency=1e-3, presence=-1.0)
    close(out, z[:1].double().cpu() - torch.nn.functional.one_hot(torch.tensor([5]), 9) * (100 - 1), torch.full((1, 9), 6 * U * 110, dtype=torch.float64), "often")


@pytest.mark.parametrize("places, classes", [(65535, 7), (65536, 7), (65540, 5000), (70001, 9001), (131073, 30000)])
def test_long_histories(places, classes):
    """Histories of more places than 16 bits count: one class all along, then another."""
    history = torch.full((2, places), 3, device="cuda", dtype=torch.int32)
    history[1, 5:] = classes - 1
    history[1, -1] = 0
    z = torch.randn(2, classes, device="cuda")
    for past in (history, history.long()):
        check(z, history=past, repetition=1.25, frequency=2.0 ** -10, presence=1.0)


@pytest.mark.parametrize("classes", [10, 500, 9001])
def test_strides(classes):
    """Padded vocabularies, parts and transposes of batches, expanded histories and masks: the results of contiguous copies."""
    g = torch.Generator().manual_seed(classes)
    base = torch.randn(6, 5, classes + 5, generator=g).to(torch.bfloat16).cuda()
    past = torch.randint(-1, classes, (6, 40), generator=g).cuda()
    flags = (torch.rand(6, 5, classes + 3, generator=g) < 0.5).cuda()
    bias = torch.randn(5, classes + 2, generator=g).cuda()
    words = words_of(flags[..., :classes])
    wide = torch.nn.functional.pad(words, (0, 2))
    for z in (base[..., 3:classes + 3], base[..., :classes], base.transpose(0, 1)[..., 1:classes + 1].transpose(0, 1)):
        history, of_rows = past.view(6, 1, 40)[..., 5:37].expand(6, 5, 32), bias[:, 1:classes + 1].expand(6, 5, classes)
        flat = F.constrain_logits(z.reshape(-1, classes).contiguous(), history.reshape(30, 32).contiguous(), repetition=1.2, bias=of_rows.reshape(30, classes).contiguous(),
                                  allowed=flags[..., :classes].reshape(30, classes).contiguous())
        for allowed in (flags[..., :classes], words, wide[..., :words.size(-1)]):
            leaf = z.detach().requires_grad_()
            out = F.constrain_logits(leaf, history, repetition=1.2, bias=of_rows, allowed=allowed)
            assert out.shape == z.shape and torch.equal(out.view(30, classes), flat)
            up = torch.randn(out.shape, generator=g).to(out.dtype).cuda()
            grad, = torch.autograd.grad(out, leaf, up.transpose(0, 1).contiguous().transpose(0, 1))
            want = exact(z.reshape(30, classes), history.reshape(30, 32), repetition=1.2, flags=flags[..., :classes].reshape(30, classes), grad=up.view(30, classes))
            close(grad.reshape(30, classes), want[2], want[3], "gradient")
    four = base[..., :classes].reshape(3, 2, 5, classes)
    out = F.constrain_logits(four, past.view(3, 2, 1, 40).expand(3, 2, 5, 40), presence=1.0, allowed=flags[..., :classes].reshape(3, 2, 5, classes))
    assert torch.equal(out.view(30, classes), F.constrain_logits(base[..., :classes].reshape(30, classes), past.view(6, 1, 40).expand(6, 5, 40).reshape(30, 40), presence=1.0,
                                                                 allowed=flags[..., :classes].reshape(30, classes)))
    turned = torch.randn(classes, 7, generator=g).cuda().t()
    assert torch.equal(F.constrain_logits(turned, allowed=turned > 0), torch.where(turned > 0, turned, -math.inf))


def test_gradients_by_differences_and_twice():
    g = torch.Generator().manual_seed(1)
    z = torch.randn(3, 12, generator=g).cuda()
    z = torch.where(z.abs() < 0.05, 0.1, z)
    history = torch.randint(0, 12, (3, 6), generator=g).cuda()
    flags = (torch.rand(3, 12, generator=g) < 0.7).cuda()
    leaf = z.clone().requires_grad_()
    run = lambda t: F.constrain_logits(t, history, repetition=1.5, presence=0.5, frequency=0.25, allowed=flags)
    up = torch.randn(3, 12, generator=g).cuda().requires_grad_()
    grad, = torch.autograd.grad(run(leaf), leaf, up, create_graph=True)
    assert grad.requires_grad
    step = 2.0 ** -6        # the map is linear on both sides of 0: differences are exact but for rounding
    for i in range(3):
        for j in range(12):
            if not flags[i, j]:
                assert grad[i, j] == 0
                continue
            move = torch.zeros_like(z)
            move[i, j] = step
            slope = ((run(z + move) - run(z - move))[i, j].double() / (2 * step)).item()
            assert abs(slope * up[i, j].item() - grad[i, j].item()) <= 16 * U * 4 / step * abs(up[i, j].item())
    again, = torch.autograd.grad(grad, up, torch.ones_like(grad))
    # g / r is rounded once, 1 / r and its product with g once each: they are at most 3 u apart (u^2 aside)
    assert ((again * up - grad).abs() <= 4 * U * grad.abs()).all()
    plain = z.clone().requires_grad_()
    bias = torch.randn(12, generator=g).cuda()
    assert torch.equal(torch.autograd.grad(F.constrain_logits(plain, bias=bias), plain, up)[0], up.detach())


def test_changed_inputs_before_the_backward():
    z = torch.randn(2, 5, device="cuda", requires_grad=True)
    history = torch.zeros(2, 3, device="cuda", dtype=torch.int64)
    out = F.constrain_logits(z, history, presence=1.0)
    history[0, 0] = 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


def test_logits_changed_after_a_mask():
    """Under a mask alone the gradient does not depend on the logits: they are not kept, and may be changed."""
    z = torch.randn(2, 3, 40, device="cuda")
    flags = torch.rand(2, 3, 40, device="cuda") < 0.5
    leaf = z.clone().requires_grad_()
    logits = leaf * 1.0
    out = F.constrain_logits(logits, allowed=flags)
    with torch.no_grad():
        logits.zero_()
    up = torch.randn_like(z)
    assert torch.equal(torch.autograd.grad(out, leaf, up)[0], up * flags)
    out = F.constrain_logits(logits, torch.zeros(2, 3, 1, device="cuda", dtype=torch.int64), repetition=2.0)
    with torch.no_grad():
        logits.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out, leaf, up)


def test_empty_batches():
    z = torch.empty(0, 7, device="cuda", requires_grad=True)
    out = F.constrain_logits(z, torch.empty(0, 3, device="cuda", dtype=torch.int64), repetition=2.0, allowed=torch.ones(7, device="cuda", dtype=torch.bool))
    assert out.shape == (0, 7) and torch.autograd.grad(out.sum(), z)[0].shape == (0, 7)


@pytest.mark.parametrize("kind", [torch.int64, torch.int32], ids=str)
def test_histories_of_no_places(kind):
    """The first step of an answer: nothing was chosen yet, with and without lengths."""
    z, _, g = make(3, 700, torch.bfloat16, 3, 5)
    flags = (torch.rand(3, 700, generator=g) < 0.5).cuda()
    none, lengths = torch.empty(3, 0, device="cuda", dtype=kind), torch.zeros(3, device="cuda", dtype=kind)
    leaf, up = z.clone().requires_grad_(), torch.ones_like(z)
    for given in (None, lengths):
        out = F.constrain_logits(leaf, none, given, repetition=2.0, presence=1.0, frequency=torch.ones(3, device="cuda"), allowed=flags)
        assert torch.equal(out.detach(), z.masked_fill(~flags, -math.inf))
        assert torch.equal(torch.autograd.grad(out, leaf, up)[0], flags.to(z.dtype))


def test_more_workgroups_than_a_launch_has():
    rows, classes = (1 << 20) + 5, 4104
    z = torch.randn(64, classes, device="cuda").half().repeat(rows // 64 + 1, 1)[:rows]
    history = torch.randint(0, classes, (rows, 2), device="cuda", dtype=torch.int32)
    out = F.constrain_logits(z, history, presence=8.0)
    for r in range(0, rows, 1 << 16):
        part, past = z[r:r + (1 << 16)], history[r:r + (1 << 16)].long()
        want = part.scatter(1, past, part.gather(1, past) - 8.0)        # (exact: the difference is rounded to the type once on either side)
        assert torch.equal(out[r:r + (1 << 16)], want), r


def test_captured_and_on_other_streams():
    """A graph reads histories, lengths, penalties and masks in each replay."""
    z, history, g = make(3, 9001, torch.bfloat16, 3, 50)
    lengths = torch.tensor([50, 20, 0], device="cuda")
    flags = (torch.rand(3, 9001, generator=g) < 0.5).cuda()
    rep = torch.full((3,), 1.5, device="cuda")
    leaf = z.clone().requires_grad_()
    up = torch.ones_like(z)

    def step():
        out = F.constrain_logits(leaf, history, lengths, repetition=rep, frequency=0.5, allowed=flags)
        return out.detach(), torch.autograd.grad(out, leaf, up)[0]

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    side = torch.cuda.Stream()
    for k in range(4):
        history.copy_(torch.randint(0, 9001, (3, 50), generator=g))
        lengths.copy_(torch.randint(0, 51, (3,), generator=g))
        flags.copy_(torch.rand(3, 9001, generator=g) < 0.3)
        rep.fill_(1.1 + 0.1 * k)
        graph.replay()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            want = step()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), k


def test_refusals():
    z = torch.zeros(4, 40, device="cuda")
    past, rows, flags = torch.zeros(4, 3, device="cuda", dtype=torch.int64), torch.ones(4, device="cuda"), torch.ones(4, 40, device="cuda", dtype=torch.bool)
    for match, call in [
            ("classes", lambda: F.constrain_logits(z[0])), ("classes", lambda: F.constrain_logits(z[:, :0])), ("dtype", lambda: F.constrain_logits(z.double())),
            ("history must have dtype", lambda: F.constrain_logits(z, past.float())), ("sizes of outputs", lambda: F.constrain_logits(z, past[:3])),
            ("sizes of outputs", lambda: F.constrain_logits(z, past[0])), ("history must be a CUDA", lambda: F.constrain_logits(z, past.cpu())),
            ("none was given", lambda: F.constrain_logits(z, lengths=past[:, 0])), ("lengths must have the sizes", lambda: F.constrain_logits(z, past, past[:2, 0])),
            ("lengths must have dtype", lambda: F.constrain_logits(z, past, rows)), ("repetition=0", lambda: F.constrain_logits(z, past, repetition=0)),
            ("repetition must have dtype", lambda: F.constrain_logits(z, past, repetition=rows.double())), ("presence must be a number", lambda: F.constrain_logits(z, past, presence=rows[:2])),
            ("frequency must not require", lambda: F.constrain_logits(z, past, frequency=rows.clone().requires_grad_())),
            ("bias must have dtype", lambda: F.constrain_logits(z, bias=z[0].half())), ("bias must have 40", lambda: F.constrain_logits(z, bias=z[0, :39])),
            ("bias must not require", lambda: F.constrain_logits(z, bias=z[0].clone().requires_grad_())), ("allowed must have dtype", lambda: F.constrain_logits(z, allowed=past)),
            ("allowed must have 2", lambda: F.constrain_logits(z, allowed=past[:, :1].int())), ("allowed must have 40", lambda: F.constrain_logits(z, allowed=flags[:, 1:])),
            ("sizes of outputs", lambda: F.constrain_logits(z, allowed=flags[:2])), ("torch.func", lambda: torch.func.vmap(F.constrain_logits)(z.view(2, 2, 40)))]:
        with pytest.raises(RuntimeError, match=match):
            call()
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level():
        with pytest.raises(NotImplementedError, match="forward mode"):
            F.constrain_logits(fwd.make_dual(z, z))


def _save_on_cpu_and_back(t):
    """A saved tensor as a hook that keeps it on the host hands it back: as large, contiguous."""
    return torch.empty(t.shape, dtype=t.dtype, device="cuda").copy_(t)


def _turned(t):
    """The same with another order of its last two dimensions in memory."""
    return t.transpose(-1, -2).contiguous().transpose(-1, -2) if t.dim() > 1 else t


@pytest.mark.parametrize("unpack", [_save_on_cpu_and_back, _turned])
@pytest.mark.parametrize("given", ["permuted", "padded", "contiguous"])
def test_saved_tensors_that_come_back_laid_out_otherwise(given, unpack):
    """Hooks may hand back what a call saved with other strides than it had (torch.autograd.graph.save_on_cpu does): the gradient reads it as it lies then."""
    z, history, g = make(30, 700, torch.bfloat16, 11, 40)
    z, history = z.view(6, 5, 700), history.view(6, 5, 40)
    flags = (torch.rand(6, 5, 700, generator=g) < 0.5).cuda()
    words = words_of(flags)
    lengths, numbers = torch.randint(0, 41, (6, 5), generator=g).cuda(), (1.0 + torch.rand(6, 5, generator=g)).cuda()
    up = torch.randn(6, 5, 700, generator=g).to(torch.bfloat16).cuda()

    def laid_out(t):
        if given == "permuted":
            return t.transpose(0, 1).contiguous().transpose(0, 1)
        return torch.cat((t, t), -1)[..., :t.size(-1)] if given == "padded" else t

    for allowed in (flags, words, None):
        leaf = laid_out(z).detach().requires_grad_()
        call = lambda: F.constrain_logits(leaf, laid_out(history), lengths, repetition=numbers, allowed=None if allowed is None else laid_out(allowed))
        want, = torch.autograd.grad(call(), leaf, up)
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
            out = call()
        source = up.clone().requires_grad_()
        got, = torch.autograd.grad(out, leaf, source, create_graph=True)
        assert torch.equal(got, want)
        again, = torch.autograd.grad(got, source, up)       # (the same factors once more)
        assert torch.equal(again, want)


def test_repetitions_of_rows_without_a_meaning():
    """A row's repetition that no number may be (0 or less, NaN, outside 2^-126..2^126) makes what it applies to NaN, gradients too, and nothing else."""
    odd = [0.0, -0.0, -1.5, math.nan, math.inf, -math.inf, 1e-39, 2.0 ** -149, 2.0 ** 127, 3e38, 2.0 ** -126, 2.0 ** 126, 1.5]
    rows, good = len(odd), 3
    for classes, group in ((12, "together"), (9001, "in parts")):
        z = torch.randn(rows, classes, device="cuda").clamp(-3.0, 3.0)
        history = torch.tensor([[1, 4, 1, -1]] * rows, device="cuda")
        numbers = torch.tensor(odd, dtype=torch.float32, device="cuda")
        leaf = z.clone().requires_grad_()
        out = F.constrain_logits(leaf, history, repetition=numbers)
        grad, = torch.autograd.grad(out, leaf, torch.zeros_like(out))
        for t in (out.detach(), grad):
            assert torch.isnan(t[:-good][:, [1, 4]]).all() and not torch.isnan(t[-good:]).any()
            t = t.clone()
            t[:, [1, 4]] = 0.0
            assert torch.equal(t, torch.zeros_like(t) if t[0, 0] == 0 else z.index_fill(1, torch.tensor([1, 4], device="cuda"), 0.0))
        ends = numbers[-good:].double().view(-1, 1)
        counted = z[-good:, [1, 4]].double()
        want = torch.where(counted > 0, counted / ends, counted * ends)
        assert ((out[-good:, [1, 4]].double() - want).abs() <= 3 * U * want.abs() + 2.0 ** -149).all()      # (a reciprocal and a product; the smallest numbers have fewer digits)


def test_gradient_reads_logits_where_something_counts():
    """The C entry's promise: of logits that nothing of the history names, nothing is read - the rows here are 64 classes long in memory, and named below that."""
    from sortnet_amd import _lib
    classes, rows = 1003, 1
    g = torch.Generator().manual_seed(2)
    for dtype, kind in ((torch.float32, 0), (torch.bfloat16, 1), (torch.float16, 2)):
        short = torch.randn(64, generator=g).to(dtype).cuda()
        up = torch.randn(rows, classes, generator=g).to(dtype).cuda()
        history = torch.randint(0, 64, (rows, 9), generator=g).cuda()
        got = torch.empty_like(up)
        a, c = _lib.LogitRows(), _lib.Constraints()
        a.logits, a.rows, a.inner, a.classes, a.inner_stride, a.dtype = short.data_ptr(), rows, rows, classes, classes, kind
        c.history, c.history_bytes, c.history_length, c.history_inner, c.repetition = history.data_ptr(), 8, 9, 9, 2.0
        _lib.call("sd_constrain_gradient", a, c, up.data_ptr(), got.data_ptr(), torch.cuda.current_stream().cuda_stream)
        want = up.clone()
        seen = torch.zeros(64, dtype=torch.bool, device="cuda").index_fill(0, history[0], True)
        want[0, :64] = torch.where(seen, torch.where(short > 0, up[0, :64] / 2, up[0, :64] * 2), up[0, :64])
        assert torch.equal(got, want)
