"""The largest logits of each row against a stable sort in 64 bits: values and classes are the same, the log-sum of the others within its rounding.

Tolerance of the log-sum, with u = 2^-24: a partial sum takes classes / 64 + 128 steps at most, each of them, the exponential and its argument off by a few u of it, so
the sum is off by at most 2 (classes / 64 + 128) u of itself and its logarithm by that; the result is rounded once.  (Terms whose exponent is large are small: the
argument's rounding, |x| u, is at most 8 u of the largest term's share where the term is above e^-8, and below that its share is less than |x| e^-|x|.)"""
import math

import pytest
import torch

from sortnet_amd import functional as F

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def make(rows, classes, dtype, seed, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, classes, generator=g) * spread).to(dtype).cuda()


def check(z, k, temperature=1.0):
    values, classes, rest = F.top_logits(z, k, temperature)
    assert values.dtype == z.dtype and classes.dtype == torch.int32 and rest.dtype == torch.float32
    assert values.shape == classes.shape == (*z.shape[:-1], k) and rest.shape == z.shape[:-1]
    flat = z.detach().double().cpu().reshape(-1, z.size(-1))
    s = flat.sort(dim=1, descending=True, stable=True)
    got_classes, got_values = classes.cpu().view(-1, k), values.double().cpu().view(-1, k)
    assert torch.equal(got_classes.long(), s.indices[:, :k])
    assert torch.equal(got_values, s.values[:, :k])
    others = s.values[:, k:] / temperature
    want = torch.logsumexp(others, 1) if others.size(1) else torch.full((len(flat),), -math.inf, dtype=torch.float64)
    got = rest.double().cpu().view(-1)
    finite = torch.isfinite(want.float())       # (a log-sum above fp32's largest number, such as 3e38 / 0.01, is rounded to infinity)
    assert torch.equal(torch.isfinite(got), finite) and torch.equal(got[~finite], want.float().double()[~finite])
    assert ((got - want).abs()[finite] <= 2 * (z.size(-1) / 64 + 128) * U + 2 * U * want.abs()[finite]).all()
    return values, classes, rest


SHAPES = [(1, 1, 1), (4, 2, 1), (4, 2, 2), (512, 10, 3), (7, 33, 33), (65, 64, 5), (65, 65, 64), (9, 200, 200), (300, 256, 256), (40, 1000, 5), (40, 1000, 200), (5, 1025, 64), (12, 2049, 65),
          (7, 4099, 17), (3, 8192, 256), (6, 16385, 1), (2, 20001, 100), (1, 65537, 256), (1, 131072, 50), (300, 50001, 200), (1030, 9001, 8), (2, 300001, 256), (2100, 17000, 33), (2, 131073, 9), (1, 8193, 5), (3, 4097, 256)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows, classes, k", SHAPES)
def test_rows(rows, classes, k, dtype):
    z = make(rows, classes, dtype, rows + classes + k)
    check(z, k)
    check(z[:3], k, 0.5)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("classes, k", [(10, 3), (64, 64), (700, 20), (700, 150), (5000, 64), (40000, 256), (140000, 60)])
def test_rows_of_equal_and_ordered_values(classes, k, dtype):
    """Ties everywhere, rows that rise, fall, hold one large part, or are all masked but for a few."""
    g = torch.Generator().manual_seed(classes)
    z = make(12, classes, dtype, classes)
    z[0] = 1.25
    z[1] = -math.inf
    z[2] = torch.finfo(dtype).min
    z[3] = (torch.randn(classes, generator=g) * 2).round().to(dtype)
    z[4] = torch.arange(classes).float().div(classes).mul(100).to(dtype)
    z[5] = z[4].flip(0)
    z[6, torch.randperm(classes, generator=g)[5:]] = -math.inf
    z[7, classes // 2:] = -math.inf
    z[8] = torch.where(torch.arange(classes) % 256 < 8, 5.0, -1.0).to(dtype)        # the large ones in few work-items' hands
    z[9] = torch.where(torch.randperm(classes, generator=g) < 2 * k, 3.0, 0.0).to(dtype)
    z[10] = 0.0
    z[10, ::2] = -0.0
    z[11] = 2e38 if dtype != torch.float16 else 6e4
    z[11, ::3] = -z[11, ::3]
    values, classes_, _ = check(z, k)
    assert torch.equal(classes_[0].cpu(), torch.arange(k, dtype=torch.int32)) and torch.equal(classes_[1].cpu(), torch.arange(k, dtype=torch.int32))


@pytest.mark.parametrize("classes", [9, 500, 20000, 140000])
def test_infinities_and_nan(classes):
    z = make(6, classes, torch.float32, classes)
    z[0, 5] = math.inf
    z[1, 2] = z[1, 7] = math.inf
    z[2, ::2] = math.inf
    z[3, 4] = math.nan
    z[4, 1:] = math.nan
    z[5] = math.nan
    check(z[:2], 3)
    values, chosen, rest = F.top_logits(z[:3], 3)
    assert (values[2] == math.inf).all() and chosen[2].tolist() == [0, 2, 4] and rest[2] == math.inf
    values, chosen, rest = F.top_logits(z[3:], 3)
    assert torch.isnan(rest).all() and torch.isnan(values[0, 0]) and chosen[0, 0] == 4 and chosen[1].tolist() == [1, 2, 3] and chosen[2].tolist() == [0, 1, 2]
    assert torch.equal(values[0, 1:], torch.cat((z[3, :4], z[3, 5:])).sort(descending=True).values[:2])


@pytest.mark.parametrize("classes", [9, 500, 20000, 140000])
def test_the_largest_far_above_the_others(classes):
    """What is left keeps its size however far it lies below the k largest."""
    z = make(4, classes, torch.float32, classes)
    z[0, 3], z[0, 5] = 400.0, 300.0
    z[1, 1] = z[1, 2] = math.inf
    z[2, ::3] += 1000.0
    z[3] -= 3000.0
    z[3, 4], z[3, 8] = 0.0, 1e30
    check(z, 2)
    check(z, 2, 0.01)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("classes", [9, 500, 20000, 140000])
def test_values_of_any_size(classes, dtype):
    """Rows around any number, and rows of two numbers of one size: what is left is a few values near the ends of their spacing."""
    z = make(14, classes, dtype, classes).float()
    for r, size in enumerate((1e3, 1e5, 1e7, 3e8, 1e10, 1e20, 3e38)):
        z[2 * r] = torch.where(torch.arange(classes, device="cuda") % 3 == 0, -size, size)
        z[2 * r + 1] = (z[2 * r + 1] * size / 1e4 if size < 1e38 else 0) - size
    z = z.to(dtype)
    check(z, 2)
    check(z, 5, 0.01)
    check(z, 2, 100.0)


@pytest.mark.parametrize("classes", [10, 1000, 30000])
def test_strides(classes):
    base = make(54, classes + 3, torch.bfloat16, classes).view(6, 9, classes + 3)
    for z in (base[:, :, 1:classes + 1], base[..., :classes], base.transpose(0, 1)[..., 2:classes + 2], base[:1, :1, :classes].expand(6, 9, classes), base[2, :, :classes],
              base[..., :classes].reshape(3, 2, 9, classes), base[::2, 1::3, :classes]):
        got, want = F.top_logits(z, 4, 2.0), F.top_logits(z.contiguous().view(-1, classes), 4, 2.0)
        assert all(torch.equal(a.reshape(b.shape), b) for a, b in zip(got, want)) and got[0].shape == (*z.shape[:-1], 4)
    turned = torch.randn(classes, 5, device="cuda").t()
    assert torch.equal(F.top_logits(turned, 3)[1], F.top_logits(turned.contiguous(), 3)[1])


def test_more_rows_than_a_launch_has():
    rows = (1 << 20) + 5
    z = torch.randn(rows, 70, device="cuda").half()
    values, classes, rest = F.top_logits(z, 2)
    assert torch.equal(values, z.topk(2, dim=1).values) and torch.equal(z.gather(1, classes.long()), values)
    check(z[-40:], 2)
    for got, want in zip(F.top_logits(z[-40:], 2), (values, classes, rest)):
        assert torch.equal(got, want[-40:])


def test_no_rows_and_no_gradient():
    z = torch.empty(0, 3, 7, device="cuda")
    values, classes, rest = F.top_logits(z, 2)
    assert values.shape == classes.shape == (0, 3, 2) and rest.shape == (0, 3)
    z = torch.randn(3, 7, device="cuda", requires_grad=True)
    assert not any(t.requires_grad for t in F.top_logits(z, 2))


def test_refusals():
    z = torch.zeros(4, 9, device="cuda")
    for match, call in [("classes", lambda: F.top_logits(z[0], 1)), ("dtype", lambda: F.top_logits(z.double(), 1)), ("k=0", lambda: F.top_logits(z, 0)), ("k=10", lambda: F.top_logits(z, 10)),
                        ("k=257", lambda: F.top_logits(torch.zeros(2, 300, device="cuda"), 257)), ("temperature=0", lambda: F.top_logits(z, 1, 0)),
                        ("temperature=nan", lambda: F.top_logits(z, 1, math.nan)), ("torch.func", lambda: torch.func.vmap(lambda t: F.top_logits(t, 1))(z.view(2, 2, 9)))]:
        with pytest.raises(RuntimeError, match=match):
            call()


@pytest.mark.parametrize("rows, classes, k", [(300, 10, 3), (40, 900, 20), (3, 70001, 64), (300, 20000, 100)])
def test_captured_and_on_other_streams(rows, classes, k):
    z = make(rows, classes, torch.bfloat16, 1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = F.top_logits(z, k)
    side = torch.cuda.Stream()
    for n in range(4):
        z.copy_(make(rows, classes, torch.bfloat16, 10 + n))
        graph.replay()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            want = F.top_logits(z, k)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), n
        check(z[:5], k)


BITS = {torch.float32: torch.int32, torch.bfloat16: torch.int16, torch.float16: torch.int16}


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("classes", [9, 64, 65, 500, 20000, 140000])
def test_values_are_the_logits_bit_by_bit(classes, dtype):
    """Zeros of both signs and NaN of any payload are given as they stand, whatever form reads the row."""
    z = make(5, classes, dtype, classes)
    z[0] = -z[0].abs() - 1.0
    z[0, 2], z[0, 3], z[0, 5] = -0.0, 0.0, -0.0
    z[1] = -0.0
    z[2, 1:8:3] = math.nan
    bits = z.view(BITS[dtype])
    bits[2, 4] += 5                     # another payload
    bits[2, 7] |= -1 << (31 if dtype == torch.float32 else 15)      # and a sign
    z[3] = math.nan
    for t in (z, z[:1]):
        values, chosen, _ = F.top_logits(t, 6)
        assert torch.equal(values.view(BITS[dtype]), t.contiguous().view(BITS[dtype]).gather(1, chosen.long()))
    values, chosen, _ = F.top_logits(z, 6)
    assert chosen[0, :3].tolist() == [2, 3, 5] and torch.signbit(values[0, :3]).tolist() == [True, False, True] and torch.signbit(values[1]).all()
    assert torch.isnan(values[2, :3]).all() and chosen[2, :3].tolist() == [1, 4, 7] and torch.isnan(values[3]).all() and chosen[3].tolist() == list(range(6))
    assert not torch.isnan(values[4]).any()


@pytest.mark.parametrize("classes", [3, 9, 64, 65, 500, 20000, 140000])
def test_others_of_large_logits(classes):
    """Log-sums of some 1e5, in temperatures whose log2(e) / T is rounded by as much as a number of fp32 can be: the factor and the result are, and nothing else of their size."""
    for temperature in (1.429, 1.426, 0.713):
        z = make(40, classes, torch.float32, classes) * 3e4
        z[20:] = z[20:].abs()
        check(z, 2, temperature)
