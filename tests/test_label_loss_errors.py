"""Calls of the losses on label log probabilities and of the dropout that are refused before any device work."""
import math

import pytest
import torch

from sortnet_amd import _lib, ext, heads, losses
from sortnet_amd import functional as F
from sortnet_amd.layers import DropoutRegistry

Z, T = torch.zeros(4, 3), torch.zeros(4, dtype=torch.int64)
R = torch.zeros(4)


@pytest.mark.parametrize("call", [
    lambda: losses.label_log_probs(Z, T), lambda: losses.preference_loss(Z, T, R), lambda: losses.policy_loss(Z, T, R, R),
    lambda: F.dropout(Z, 0.5, 1), lambda: F.bound_dropout(None, Z, Z, 0.5, 1)])
def test_tensors_on_the_host(call):
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        call()


def _rows(**kw):
    rows = _lib.LabelRows()
    for k, v in dict(dict(logits=1 << 20, labels=1 << 20, rows=4, inner=4, classes=3, outer_stride=0, inner_stride=3, ignore_index=-100, dtype=0), **kw).items():
        setattr(rows, k, v)
    return rows


BAD_ROWS = [dict(dtype=3), dict(dtype=-1), dict(rows=0), dict(rows=1 << 31), dict(classes=0), dict(classes=1 << 31), dict(inner=0), dict(inner=3), dict(logits=0), dict(labels=0)]


@pytest.mark.parametrize("bad", BAD_ROWS, ids=str)
def test_rows_without_a_meaning(bad):
    p = 1 << 20    # no kernel is launched: every call is refused by its sizes
    rows = _rows(**bad)
    assert _lib.load().sd_label_scratch(rows, 0) == -1 and _lib.load().sd_label_scratch(rows, 1) == -1
    for name, args in [("sd_label_log_probs", (p, p, p, None)), ("sd_preference_loss", (p, None, 0, 1, 2, 0.1, 0.0, p, p, p, p, p, None)),
                       ("sd_policy_loss", (p, p, 0, 1, p, 0.2, 0.2, 0.0, p, p, p, None, p, p, p, None)), ("sd_label_gradient", (p, p, None, None, 0, p, None))]:
        with pytest.raises(RuntimeError, match=r"status 1\)"):
            _lib.call(name, rows, *args)


@pytest.mark.parametrize("bad, match", [
    (dict(pairs=0), "pairs"), (dict(pairs=-1), "pairs"), (dict(pairs=1), "pairs"), (dict(tokens=2), "pairs"), (dict(tokens=0), "pairs"), (dict(ref=None), "null"),
    (dict(offsets=1 << 20, offset_bytes=2), "bytes"), (dict(smoothing=-0.1), "smoothing"), (dict(smoothing=0.5), "smoothing"), (dict(smoothing=math.nan), "smoothing")], ids=str)
def test_preferences_without_a_meaning(bad, match):
    p = 1 << 20
    good = dict(ref=p, offsets=None, offset_bytes=0, tokens=1, pairs=2, beta=0.1, smoothing=0.0)    # of four rows
    with pytest.raises(RuntimeError, match=match):
        _lib.call("sd_preference_loss", _rows(), *dict(good, **bad).values(), p, p, p, p, p, None)


def test_buffers_out_of_line():
    p = 1 << 20
    for rows in (_rows(logits=p + 2), _rows(logits=p + 1, dtype=1), _rows(labels=p + 4)):
        with pytest.raises(RuntimeError, match="aligned"):
            _lib.call("sd_label_log_probs", rows, p, p, p, None)
    for stats, scratch in ((p + 4, p), (p, p + 8)):
        with pytest.raises(RuntimeError, match="aligned"):
            _lib.call("sd_label_log_probs", _rows(), p, stats, scratch, None)
        with pytest.raises(RuntimeError, match="aligned"):
            _lib.call("sd_preference_loss", _rows(), p, None, 0, 1, 2, 0.1, 0.0, stats, p, p, p, scratch, None)
        with pytest.raises(RuntimeError, match="aligned"):
            _lib.call("sd_policy_loss", _rows(), p, p, 0, 1, None, 0.2, 0.2, 0.0, stats, p, p, None, p, p, scratch, None)
    with pytest.raises(RuntimeError, match="aligned"):
        _lib.call("sd_label_gradient", _rows(), p + 4, p, None, None, 0, p, None)


def test_halves_of_the_gradient():
    p = 1 << 20
    with pytest.raises(RuntimeError, match="both"):
        _lib.call("sd_preference_loss", _rows(), p, None, 0, 1, 2, 0.1, 0.0, p, None, p, p, p, None)
    with pytest.raises(RuntimeError, match="both"):
        _lib.call("sd_policy_loss", _rows(), p, p, 0, 1, None, 0.2, 0.2, 0.0, None, p, p, None, p, p, p, None)
    assert _lib.load().sd_policy_fuses(_rows()) == 0
    with pytest.raises(RuntimeError, match="does not leave"):      # too few rows for a gradient that leaves with them
        _lib.call("sd_policy_loss", _rows(), p, p, 0, 1, None, 0.2, 0.2, 0.0, p, p, p, p, p, p, p, None)
    with pytest.raises(RuntimeError, match="unless_one"):
        _lib.call("sd_label_gradient", _rows(), p, p, None, None, 1, p, None)


@pytest.mark.parametrize("low, high, kl, ref, match", [(-0.1, 0.2, 0.0, 0, "clip"), (1.1, 0.2, 0.0, 0, "clip"), (0.2, -0.1, 0.0, 0, "clip"), (math.nan, 0.2, 0.0, 0, "clip"),
                                                       (0.2, math.nan, 0.0, 0, "clip"), (0.2, 0.2, 0.1, 0, "reference")])
def test_policies_without_a_meaning(low, high, kl, ref, match):
    p = 1 << 20
    with pytest.raises(RuntimeError, match=match):
        _lib.call("sd_policy_loss", _rows(), p, p, 0, 1, ref or None, low, high, kl, p, p, p, None, p, p, p, None)


def test_dropout_without_a_meaning():
    p = 1 << 20
    for q in (-0.1, 1.5, math.nan):
        with pytest.raises(RuntimeError, match="q="):
            _lib.call("sd_dropout", p, None, None, 0, 8, q, 1, None, p, None, None, None)
    with pytest.raises(RuntimeError, match="dtype"):
        _lib.call("sd_dropout", p, None, None, 7, 8, 0.5, 1, None, p, None, None, None)
    with pytest.raises(RuntimeError, match="alone"):
        _lib.call("sd_dropout", p, p, None, 0, 8, 0.5, 1, None, p, None, None, None)
    for n in (-1, 1 << 48):
        with pytest.raises(RuntimeError, match="values"):
            _lib.call("sd_dropout", p, None, None, 0, n, 0.5, 1, None, p, None, None, None)
    for q in (0.0, -1.0, 1.5, math.nan):
        with pytest.raises(ValueError):
            heads.BoundDropout(q)


def test_dropout_that_keeps_everything():
    x = torch.randn(3, 4)
    assert F.dropout(x, 1.0, 3) is x and F.dropout(x, None, 3) is x
    assert F.bound_dropout(x, None, x, 1.0, 3) == (x, None, x)
    layer = heads.BoundDropout(0.5)
    layer.eval()
    assert layer(x, None, x) == (x, None, x) and layer.last_seed is None
    assert heads.BoundDropout(1.0)(x, None, None) == (x, None, None)


def test_seeds_of_layers_continue_the_registry():
    reg, other = DropoutRegistry(seed=7), DropoutRegistry(seed=7)
    assert [reg.next_seed() for _ in range(3)] == [(7 * 1000003 + k) & 0xFFFFFFFF for k in (1, 2, 3)]
    assert other.next_seed() == (7 * 1000003 + 1) & 0xFFFFFFFF


def test_losses_keep_their_registry():
    assert set(losses.LOSSES) == {"hinge", "crossentropy", "mixture", "ce_hinge", "ce_mixture"}
    assert ext.host().label_log_probs is not None


def test_keep_probabilities_that_are_rounded_to_the_ends():
    """q is rounded to 1/65536: a layer that would keep nothing is refused, one that would keep everything draws no seed and runs no kernel."""
    x = torch.randn(3, 4)
    for q in (1e-300, 1e-6, 2.0 ** -17 * (1 - 2.0 ** -50)):
        with pytest.raises(ValueError):
            heads.BoundDropout(q)
    for q in (2.0 ** -17, 2.0 ** -16):
        assert heads.BoundDropout(q).q == q
    for q in (1.0 - 2.0 ** -17, 1.0 - 1e-9, 1.0):
        layer = heads.BoundDropout(q, registry=DropoutRegistry(seed=1))
        assert layer(x, None, x) == (x, None, x) and layer.last_seed is None and layer.registry.draws == 0
        assert F.dropout(x, q, 3) is x and F.bound_dropout(x, x, None, q, 3) == (x, x, None)
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        F.dropout(x, 1.0 - 2.0 ** -17 - 1e-9, 3)
    for q in (1.0 + 1e-9, math.inf, math.nan, -1e-9):
        with pytest.raises(ValueError):
            heads.BoundDropout(q)
