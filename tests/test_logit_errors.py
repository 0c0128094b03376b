"""Calls of the operators that answer with logits or learn from another model's, refused before any device work."""
import math

import pytest
import torch

from sortnet_amd import _lib, losses
from sortnet_amd import functional as F

P = 1 << 20     # an address: no kernel is launched, every call is refused by its sizes
Z = torch.zeros(4, 3)


def _rows(**kw):
    rows = _lib.LogitRows()
    for k, v in dict(dict(logits=P, rows=4, inner=4, classes=3, outer_stride=0, inner_stride=3, dtype=0), **kw).items():
        setattr(rows, k, v)
    return rows


def _constraints(**kw):
    c = _lib.Constraints()
    for k, v in dict(dict(repetition=1.0), **kw).items():
        setattr(c, k, v)
    return c


BAD_ROWS = [dict(dtype=3), dict(dtype=-1), dict(rows=0), dict(rows=1 << 31), dict(classes=0), dict(classes=1 << 31), dict(inner=0), dict(inner=3), dict(logits=0),
            dict(logits=P + 2), dict(logits=P + 1, dtype=1)]


@pytest.mark.parametrize("bad", BAD_ROWS, ids=str)
def test_rows_without_a_meaning(bad):
    for name, args in (("sd_constrain_logits", (P,)), ("sd_constrain_gradient", (P, P))):
        with pytest.raises(RuntimeError, match=r"status 1\)"):
            _lib.call(name, _rows(**bad), _constraints(), *args, None)


@pytest.mark.parametrize("bad, match", [
    (dict(history=P, history_bytes=2, history_length=3), "history of"), (dict(history=P, history_bytes=8, history_length=-1), "history_length"),
    (dict(history=P, history_bytes=8, history_length=1 << 32), "history_length"), (dict(history=P + 4, history_bytes=8, history_length=3), "aligned"),
    (dict(lengths=P, length_bytes=4), "without a history"), (dict(history=P, history_bytes=4, history_length=3, lengths=P, length_bytes=3), "lengths of"),
    (dict(history=P, history_bytes=4, history_length=3, lengths=P + 2, length_bytes=4), "aligned"),
    (dict(repetition=0.0), "repetition"), (dict(repetition=-1.0), "repetition"), (dict(repetition=math.nan), "repetition"), (dict(repetition=math.inf), "repetition"),
    (dict(repetition=1e-60), "repetition"), (dict(presence=math.nan), "presence"), (dict(presence=math.inf), "presence"), (dict(frequency=-math.inf), "frequency"),
    (dict(allowed=P, allowed_kind=0), "allowed_kind"), (dict(allowed=P, allowed_kind=3), "allowed_kind"), (dict(allowed=P + 2, allowed_kind=2), "aligned"),
    (dict(bias=P + 1), "aligned"), (dict(presence_rows=P + 2), "aligned")], ids=str)
def test_constraints_without_a_meaning(bad, match):
    with pytest.raises(RuntimeError, match=match):
        _lib.call("sd_constrain_logits", _rows(), _constraints(**bad), P, None)
    with pytest.raises(RuntimeError, match=match):
        _lib.call("sd_constrain_gradient", _rows(), _constraints(**bad), P, P, None)


def test_results_out_of_line():
    for out in (None, P + 2):
        with pytest.raises(RuntimeError):
            _lib.call("sd_constrain_logits", _rows(), _constraints(), out, None)
    for grad in (None, P + 1):
        with pytest.raises(RuntimeError):
            _lib.call("sd_constrain_gradient", _rows(), _constraints(), grad, P, None)


@pytest.mark.parametrize("call", [lambda: F.constrain_logits(Z), lambda: F.constrain_logits(Z, torch.zeros(4, 2, dtype=torch.int64), presence=1.0),
                                  lambda: F.top_logits(Z, 1), lambda: losses.distill_loss(Z, Z[:, :2], torch.zeros(4, 2, dtype=torch.int32))])
def test_tensors_on_the_host(call):
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        call()


def _lists(**kw):
    lists = _lib.TopLists()
    for k, v in dict(dict(values=P, classes=P, rest=None, k=2, dtype=0, class_bytes=4), **kw).items():
        setattr(lists, k, v)
    return lists


def _distill(rows=None, lists=None, temperature=1.0, weight=1.0, stats=P, entries=P, scale=P, grad=None, loss=P, divergences=P, scratch=P):
    return _lib.call("sd_distill_loss", rows or _rows(), lists or _lists(), temperature, weight, stats, entries, scale, grad, loss, divergences, scratch, None)


@pytest.mark.parametrize("bad", BAD_ROWS, ids=str)
def test_rows_without_a_largest_logit(bad):
    assert _lib.load().sd_top_scratch(_rows(**bad), 1) == -1
    with pytest.raises(RuntimeError, match=r"status 1\)"):
        _lib.call("sd_top_logits", _rows(**bad), 1, 1.0, P, P, P, P, None)


def test_largest_logits_without_a_meaning():
    for k in (0, -1, 4, 257):
        assert _lib.load().sd_top_scratch(_rows(), k) == -1
        with pytest.raises(RuntimeError, match="k="):
            _lib.call("sd_top_logits", _rows(), k, 1.0, P, P, P, P, None)
    for t in (0.0, -1.0, 1e-5, 1e5, math.nan, math.inf):
        with pytest.raises(RuntimeError, match="temperature"):
            _lib.call("sd_top_logits", _rows(), 2, t, P, P, P, P, None)
    for values, classes, rest, match in ((None, P, P, "null"), (P, None, P, "null"), (P, P, None, "null"), (P + 2, P, P, "aligned"), (P, P + 1, P, "aligned"), (P, P, P + 2, "aligned")):
        with pytest.raises(RuntimeError, match=match):
            _lib.call("sd_top_logits", _rows(), 2, 1.0, values, classes, rest, P, None)


@pytest.mark.parametrize("bad", BAD_ROWS, ids=str)
def test_rows_without_a_meaning_to_the_teacher(bad):
    assert _lib.load().sd_distill_scratch(_rows(**bad), 2) == -1
    with pytest.raises(RuntimeError, match=r"status 1\)"):
        _distill(_rows(**bad))
    with pytest.raises(RuntimeError, match=r"status 1\)"):
        _lib.call("sd_distill_gradient", _rows(**bad), _lists(), 1.0, P, P, P, None, 0, P, None)


@pytest.mark.parametrize("bad, match", [(dict(values=0), "null"), (dict(classes=0), "null"), (dict(k=0), "k=0"), (dict(k=257), "k=257"), (dict(k=-1), "k=-1"), (dict(dtype=5), "dtype"),
                                        (dict(class_bytes=2), "classes of"), (dict(values=P + 2), "aligned"), (dict(classes=P + 4, class_bytes=8), "aligned"), (dict(rest=P + 1), "aligned")], ids=str)
def test_lists_without_a_meaning(bad, match):
    with pytest.raises(RuntimeError, match=match):
        _distill(lists=_lists(**bad))
    with pytest.raises(RuntimeError, match=match):
        _lib.call("sd_distill_gradient", _rows(), _lists(**bad), 1.0, P, P, P, None, 0, P, None)


def test_distillation_without_a_meaning():
    for k in (0, 257):
        assert _lib.load().sd_distill_scratch(_rows(), k) == -1
    for t in (0.0, -1.0, 1e-5, 1e5, math.nan, math.inf):
        with pytest.raises(RuntimeError, match="temperature"):
            _distill(temperature=t)
        with pytest.raises(RuntimeError, match="temperature"):
            _lib.call("sd_distill_gradient", _rows(), _lists(), t, P, P, P, None, 0, P, None)
    for w in (math.nan, math.inf, -math.inf, 1e39):
        with pytest.raises(RuntimeError, match="weight"):
            _distill(weight=w)
    for missing in ("loss", "divergences", "scratch"):
        with pytest.raises(RuntimeError, match="null"):
            _distill(**{missing: None})
    for missing in ("stats", "entries", "scale"):
        with pytest.raises(RuntimeError, match="needs stats"):
            _distill(**{missing: None})
    assert _lib.load().sd_distill_fuses(_rows()) == 0
    with pytest.raises(RuntimeError, match="does not leave"):       # too few rows for a gradient that leaves with them
        _distill(grad=P)
    with pytest.raises(RuntimeError, match="needs stats"):
        _distill(grad=P, stats=None, entries=None, scale=None)
    with pytest.raises(RuntimeError, match="unless_one"):
        _lib.call("sd_distill_gradient", _rows(), _lists(), 1.0, P, P, P, None, 1, P, None)
    with pytest.raises(RuntimeError, match="aligned"):
        _distill(stats=P + 4)
    with pytest.raises(RuntimeError, match="aligned"):
        _distill(scratch=P + 8)


@pytest.mark.parametrize("value", [1e-39, 2.0 ** -127, 2.0 ** 127, 3e38], ids=str)
def test_repetitions_whose_reciprocal_loses_digits(value):
    """Penalised logits are products with a repetition or its reciprocal in fp32: both have to be normal numbers."""
    for name, args in (("sd_constrain_logits", (P,)), ("sd_constrain_gradient", (P, P))):
        with pytest.raises(RuntimeError, match="repetition="):
            _lib.call(name, _rows(), _constraints(repetition=value), *args, None)


@pytest.mark.skipif(torch.cuda.is_available(), reason="where there is a GPU the kernels would be launched")
def test_launches_that_fail_name_their_kernels():
    for classes, kernel in ((60, "top_short_kernel"), (200, "top_rows_kernel"), (1 << 20, "top_join_kernel")):
        with pytest.raises(RuntimeError, match=kernel):
            _lib.call("sd_top_logits", _rows(classes=classes), 2, 1.0, P, P, P, P, None)
    for rows, kernel, slopes in ((dict(classes=60), "distill_short_kernel", "distill_short_gradient_kernel"), (dict(classes=9000), "distill_held_kernel", "distill_long_gradient_kernel"),
                                 (dict(classes=1 << 20), "distill_join_kernel", "distill_long_gradient_kernel")):
        with pytest.raises(RuntimeError, match=kernel):
            _distill(_rows(**rows))
        with pytest.raises(RuntimeError, match=slopes):
            _lib.call("sd_distill_gradient", _rows(**rows), _lists(), 1.0, P, P, P, None, 0, P, None)
    with pytest.raises(RuntimeError, match="distill_rows_that_count_kernel"):
        _distill(_rows(rows=4096, inner=4096, classes=9000), grad=P)
