"""Dropout from the counter generator: the mask against a restatement in numpy, values bit for bit, gradients, bounds, seeds on the device,
and a hybrid model that trains with it through the losses on its logits."""
import math

import numpy as np
import pytest
import torch

from sortnet_amd import functional as F
from sortnet_amd import heads, layers, losses
from sortnet_amd.ell_inf_models import SortHybridModel
from sortnet_amd.layers import DropoutRegistry

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def mix(h):
    h = h ^ (h >> np.uint32(16))
    h = h * np.uint32(0x21f0aaad)
    h = h ^ (h >> np.uint32(15))
    h = h * np.uint32(0x735a2d97)
    return h ^ (h >> np.uint32(15))


def limit_of(q):
    return math.floor(65536 * q + 0.5)


def kept(n, q, seed, start=0):
    """Which of the values start .. start + n of a tensor stay; start a multiple of 65536."""
    out = np.empty(n, dtype=bool)
    for k in range((n + 65535) // 65536):
        row = np.array([(start // 65536 + k) & 0xFFFFFFFF], dtype=np.uint32)
        keys = [mix(np.array([seed ^ ((s * 0x9e3779b9) & 0xFFFFFFFF)], dtype=np.uint32) + row) for s in (5, 6)]
        cols = np.arange(1, 32769, dtype=np.uint32)
        words = mix(mix(keys[0] + cols * np.uint32(0x85ebca6b)) ^ keys[1])
        fields = np.stack((words & np.uint32(0xffff), words >> np.uint32(16)), 1).reshape(-1)
        part = out[k * 65536:(k + 1) * 65536]
        part[:] = fields[:part.size] < limit_of(q)
    return torch.from_numpy(out).cuda()


def expected(x, keep, q):
    scale = 65536.0 / limit_of(q) if limit_of(q) else 0.0
    return torch.where(keep.view(x.shape), x.detach().float() * scale, 0.0).to(x.dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("n, q", [(1, 0.5), (7, 0.5), (8, 0.9), (9, 0.1), (65535, 0.5), (65536, 0.25), (65537, 0.75), (1 << 20, 0.9), ((1 << 20) + 3, 0.999), (4099, 1e-5), (513, 0.0)])
def test_values_and_gradient(n, q, dtype):
    g = torch.Generator().manual_seed(n)
    seed = (n * 2654435761 + 17) & 0xFFFFFFFF
    x = torch.randn(n, generator=g).to(dtype).cuda().requires_grad_()
    up = torch.randn(n, generator=g).to(dtype).cuda()
    keep = kept(n, q, seed)
    y = F.dropout(x, q, seed)
    assert y.dtype == dtype and torch.equal(y, expected(x, keep, q))
    assert torch.equal(torch.autograd.grad(y, x, up)[0], expected(up, keep, q))
    assert torch.equal(F.dropout(x, q, seed), y) and torch.equal(F.dropout(x, q, seed + (1 << 32)), y)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", [(1, 1), (5, 7), (33, 129), (512, 512)])
def test_values_and_bounds_share_a_mask(shape, dtype):
    g = torch.Generator().manual_seed(shape[1])
    x, lower, upper = [torch.randn(shape, generator=g).to(dtype).cuda().requires_grad_() for _ in range(3)]
    ups = [torch.randn(shape, generator=g).to(dtype).cuda() for _ in range(3)]
    keep = kept(x.numel(), 0.7, 5)
    for there in ((1, 1, 1), (1, 0, 0), (0, 1, 1), (1, 1, 0), (0, 0, 1), (0, 0, 0)):
        args = [t if k else None for t, k in zip((x, lower, upper), there)]
        got = F.bound_dropout(*args, 0.7, 5)
        for a, y in zip(args, got):
            assert y is None if a is None else torch.equal(y, expected(a, keep, 0.7))
        outs = [y for y in got if y is not None]
        if outs:
            grads = torch.autograd.grad(outs, [a for a in args if a is not None], ups[:len(outs)])
            for gr, up in zip(grads, ups):
                assert torch.equal(gr, expected(up, keep, 0.7))
    # a gradient into one of three, and one alone that wants it
    got = F.bound_dropout(x, lower, upper, 0.7, 5)
    a, b = torch.autograd.grad(got[1], (x, lower), ups[0], allow_unused=True)
    assert (a is None or (a == 0).all()) and torch.equal(b, expected(ups[0], keep, 0.7))
    got = F.bound_dropout(x.detach(), lower, upper.detach(), 0.7, 5)
    assert torch.equal(torch.autograd.grad(got[1], lower, ups[1])[0], expected(ups[1], keep, 0.7))


def test_strides_alignment_and_order():
    """The mask goes by the row-major index of the tensor as it is given, wherever it lies."""
    g = torch.Generator().manual_seed(1)
    base = torch.randn(40, 61, generator=g).to(torch.bfloat16).cuda()
    for view in (base.t(), base[1:, 3:], base[::2], base.reshape(-1)[1:], base.reshape(-1)[3:102], base[:1].expand(7, 61), base.view(2, 20, 61).transpose(0, 2)):
        assert torch.equal(F.dropout(view, 0.5, 9), expected(view.contiguous(), kept(view.numel(), 0.5, 9), 0.5))
    empty = base[:0].detach().requires_grad_()
    out = F.dropout(empty, 0.5, 1)
    assert out.shape == (0, 61) and torch.autograd.grad(out.sum(), empty)[0].shape == (0, 61)


def test_dropped_values_are_zero_whatever_they_were():
    x = torch.full((4096,), math.nan, device="cuda")
    x[::2] = math.inf
    y = F.dropout(x, 0.5, 3)
    keep = kept(4096, 0.5, 3)
    assert (y[~keep] == 0).all() and not torch.isfinite(y[keep]).any()


def test_statistics():
    """Kept shares within five standard deviations of q over rows, columns, neighbours and seeds."""
    n, q = 1 << 22, 0.3
    x = torch.ones(n, device="cuda")
    a = F.dropout(x, q, 1) != 0
    qq = limit_of(q) / 65536
    dev = lambda p, m: 5 * math.sqrt(p * (1 - p) / m)
    assert abs(a.double().mean().item() - qq) <= dev(qq, n)
    blocks = a.view(64, 65536).double().mean(1)
    assert (blocks - qq).abs().max().item() <= dev(qq, 65536) * 1.2
    for shift in (1, 2, 64, 8, 65536, 65538):
        both = (a[shift:] & a[:-shift]).double().mean().item()
        assert abs(both - qq * qq) <= dev(qq * qq, n - shift) * 2, shift       # (overlapping windows: up to twice the variance)
    for other in (2, 0x80000001, 1 ^ 0x9e3779b9):
        b = F.dropout(x, q, other) != 0
        assert abs((a & b).double().mean().item() - qq * qq) <= dev(qq * qq, n)


def test_values_beyond_32_bit_indices():
    n = (1 << 32) + 70001
    x = torch.ones(n, device="cuda", dtype=torch.bfloat16)
    y = F.dropout(x, 0.5, 77)
    for start, m in ((0, 1000), ((1 << 32) - 65536, 65536), (1 << 32, 70001)):
        assert torch.equal(y[start:start + m], expected(x[start:start + m], kept(m, 0.5, 77, start), 0.5))


def test_seed_on_the_device_in_a_graph():
    """Each replay reads the seed: other masks, forward and backward alike, equal to the eager ones."""
    x = torch.randn(1000, 33, device="cuda").requires_grad_()
    up = torch.randn(1000, 33, device="cuda")
    seed = torch.tensor(5, device="cuda")

    def step(s):
        y = F.dropout(x, 0.6, s)
        return y.detach(), torch.autograd.grad(y, x, up)[0]

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step(seed)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        outs = step(seed)
    for k in (5, 6, (1 << 40) + 6, -1):
        seed.fill_(k)
        want = step(k)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
    y = F.dropout(x, 0.6, seed)
    seed.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, x, up)


def test_what_is_refused():
    x = torch.ones(4, 3, device="cuda")
    for bad in (lambda: F.dropout(x.double(), 0.5, 1), lambda: F.dropout(x, -0.1, 1), lambda: F.dropout(x, math.nan, 1), lambda: F.bound_dropout(x, x[:2], x, 0.5, 1),
                lambda: F.bound_dropout(x, x.half(), x, 0.5, 1), lambda: F.bound_dropout(x, x.cpu(), None, 0.5, 1), lambda: F.dropout(x, 0.5, torch.tensor(1)),
                lambda: F.dropout(x, 0.5, torch.tensor([1, 2], device="cuda")), lambda: F.dropout(x, 0.5, torch.tensor(1, dtype=torch.int32, device="cuda"))):
        with pytest.raises(RuntimeError):
            bad()


def test_layer_and_its_seed():
    layer = heads.BoundDropout(0.5, registry=DropoutRegistry(seed=3))
    x = torch.randn(8, 16, device="cuda")
    a, lo, up = layer(x, x - 1, None)
    assert up is None and torch.equal(a, F.dropout(x, 0.5, layer.last_seed)) and torch.equal(lo, F.dropout(x - 1, 0.5, layer.last_seed))
    b, _, _ = layer(x)
    assert not torch.equal(a, b)
    layer.registry.draws = 0
    assert torch.equal(layer(x)[0], a)
    layer.eval()
    assert layer(x)[0] is x


@pytest.mark.parametrize("kind", ["label", "preference", "policy", "certified"])
def test_a_hybrid_model_trains(kind):
    """Distance stack, dense head, dropout, final layer and a loss on its logits: gradients of all parameters against the same step with the mask multiplied
    in by torch and the loss in 64 bits.  Logits differ by nothing (the same kernels and products run), so the gradient of the logits is off by at
    most 1e-5 of its size; the parameters' are linear in it and no more than 200 times as far off through sums of both signs (checked
    against the largest entry of each)."""
    torch.manual_seed(0)
    reg = DropoutRegistry(seed=11)
    model = SortHybridModel(4, 64, (1, 8, 8), hidden=48, num_classes=7, dropout=None, registry=reg, head_dropout=0.8).cuda().train()
    assert set(model.state_dict()) == set(SortHybridModel(4, 64, (1, 8, 8), hidden=48, num_classes=7, dropout=None, registry=DropoutRegistry()).state_dict())
    x = torch.rand(12, 1, 8, 8, device="cuda")
    t = torch.arange(12, device="cuda") % 7
    ref, old, adv = torch.full((12,), -2.0, device="cuda"), torch.full((12,), -1.9, device="cuda"), torch.linspace(-1, 1, 12, device="cuda")

    def logits():
        return model(x, t, 0.1)[1] if kind == "certified" else model(x)

    out = logits()
    seed = model.head_drop.last_seed
    if kind in ("label", "certified"):
        loss = -losses.label_log_probs(out, t).mean()
    elif kind == "preference":
        loss, _ = losses.preference_loss(out, t, ref)
    else:
        loss, _ = losses.policy_loss(out, t, old, adv, ref_log_probs=ref, kl_coef=0.1, clip=0.2)
    params = [p for p in model.parameters() if p.requires_grad]
    grads = torch.autograd.grad(loss, params, allow_unused=True)

    drawn = []
    drop = model.head_drop.forward
    model.head_drop.forward = lambda *a: drawn.append(seed) or F.bound_dropout(*(list(a) + [None] * (3 - len(a))), 0.8, seed)
    out2 = logits()
    model.head_drop.forward = drop
    assert drawn and torch.equal(out, out2)         # the seed makes the mask again
    lp = torch.log_softmax(out2.double(), 1).gather(1, t.view(-1, 1)).squeeze(1)
    if kind in ("label", "certified"):
        want = -lp.mean()
    elif kind == "preference":
        m = 0.1 * ((lp - ref)[:6] - (lp - ref)[6:])
        want = torch.nn.functional.softplus(-m).mean()
    else:
        ratio = (lp - old).exp()
        apart = ref - lp
        want = (-torch.minimum(ratio * adv, ratio.clamp(0.8, 1.2) * adv) + 0.1 * (apart.exp() - apart - 1)).mean()
    assert abs(loss.item() - want.item()) <= 1e-5 * max(1.0, abs(want.item()))
    for a, b in zip(grads, torch.autograd.grad(want, params, allow_unused=True)):
        assert (a is None) == (b is None)
        if a is not None:
            assert (a - b).abs().max().item() <= 2e-3 * max(b.abs().max().item(), 1e-6)
    assert any(a is not None and (a != 0).any() for a in grads)


def test_masks_of_several_passes_are_unlike_at_any_shift():
    """The masks of the first 32 passes of a layer, each against each, shifted by up to 16 rows of 2^16 values: kept together as often as chance has it,
    within seven standard deviations (33 x 496 pairs)."""
    layer = heads.BoundDropout(0.5, registry=DropoutRegistry(seed=0))
    x = torch.ones(24, 65536, device="cuda")
    masks = torch.stack([layer(x)[0] != 0 for _ in range(32)]).to(torch.bfloat16)
    for shift in range(17):
        n = 24 - shift
        a, b = masks[:, shift:].reshape(32, -1), masks[:, :n].reshape(32, -1)
        both = sum(torch.mm(a[:, k:k + 65536].float(), b[:, k:k + 65536].float().t()) for k in range(0, n * 65536, 65536)) / (n * 65536)
        if shift == 0:
            both.fill_diagonal_(0.25)
        assert (both - 0.25).abs().max().item() <= 7 * math.sqrt(0.25 * 0.75 / (n * 65536)), shift


def test_second_derivatives():
    """A penalty on a gradient that went through the dropout, against the mask multiplied in in 64 bits.  Every value is a product of at most 16 numbers, each
    rounded once, and sums of two of one sign: off by at most 32 half steps of fp32."""
    g = torch.Generator().manual_seed(4)
    x, lower, w, v = [torch.randn(33, 70, generator=g).cuda().requires_grad_() for _ in range(4)]
    m = kept(x.numel(), 0.6, 21).view(x.shape).double() * (65536 / limit_of(0.6))

    def penalty(x, lower, w, v, drop):
        a, b = drop(x, lower)
        gx, gl = torch.autograd.grad((a * w).pow(2).sum() + (b * v).pow(2).sum(), (x, lower), create_graph=True)
        return torch.autograd.grad(gx.pow(2).sum() + gl.pow(2).sum(), (x, w, lower, v))

    def one(x, lower):
        return F.dropout(x, 0.6, 21), F.dropout(lower, 0.6, torch.tensor(21, device="cuda"))

    want = penalty(*[t.detach().double().requires_grad_() for t in (x, lower, w, v)], lambda a, b: (a * m, b * m))
    for drop in (one, lambda a, b: F.bound_dropout(a, b, None, 0.6, 21)[:2]):
        for got, exact in zip(penalty(x, lower, w, v, drop), want):
            assert ((got.double() - exact).abs() <= 32 * 2.0 ** -24 * exact.abs()).all()
    # one of two tensors alone, and a gradient that depends on nothing
    a, b, _ = F.bound_dropout(x, lower, None, 0.6, 21)
    gl, = torch.autograd.grad((a * b * v).sum(), lower, create_graph=True)
    got, exact = torch.autograd.grad(gl.pow(2).sum(), (x, v)), (2 * (m * m * x * v) * m * m * v, 2 * (m * m * x * v) * m * m * x)
    assert all(((p.double() - q).abs() <= 32 * 2.0 ** -24 * q.abs()).all() for p, q in zip(got, exact))
    gx, = torch.autograd.grad(F.dropout(x, 0.6, 21), x, torch.ones_like(x), create_graph=True)
    assert not gx.requires_grad
    # and a third derivative
    y = F.dropout(x, 0.6, 21)
    first, = torch.autograd.grad(y.pow(3).sum(), x, create_graph=True)
    second, = torch.autograd.grad(first.sum(), x, create_graph=True)
    third, = torch.autograd.grad(second.sum(), x)
    assert ((third.double() - 6 * m ** 3).abs() <= 32 * 2.0 ** -24 * 6 * m ** 3).all()


def test_activation_checkpointing():
    """A step whose forward runs again for the backward: the gradients of the step itself, with the functions and with a layer that has a seed of its own."""
    from torch.utils.checkpoint import checkpoint
    g = torch.Generator().manual_seed(9)
    x, w = torch.randn(64, 40, generator=g).cuda().requires_grad_(), torch.randn(40, 30, generator=g).cuda().requires_grad_()
    t = torch.randint(0, 30, (64,), generator=g).cuda()
    ref, adv = torch.full((64,), -3.0, device="cuda"), torch.randn(64, generator=g).cuda()
    layer = heads.BoundDropout(0.7, seed=torch.tensor(F.dropout_seed(3), device="cuda"))
    for drop in (lambda v: F.dropout(v, 0.7, 9), lambda v: layer(v)[0]):
        for loss in (lambda z: losses.label_log_probs(z, t).sum(), lambda z: losses.preference_loss(z, t, ref)[0],
                     lambda z: losses.policy_loss(z, t, ref, adv, ref_log_probs=ref, kl_coef=0.1)[0]):
            step = lambda x, w: loss(drop(torch.tanh(x)) @ w)
            want = torch.autograd.grad(step(x, w), (x, w))
            for reentrant in (False, True):
                if reentrant:       # (serves .backward() alone)
                    x.grad = w.grad = None
                    checkpoint(step, x, w, use_reentrant=True).backward()
                    got = x.grad, w.grad
                else:
                    got = torch.autograd.grad(checkpoint(step, x, w, use_reentrant=False), (x, w))
                assert all(torch.equal(a, b) for a, b in zip(got, want))
