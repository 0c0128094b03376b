"""Masks of the dropout from different seeds: no row of one is a row of another, at any shift.

A row of 2^16 values is made of two keys alone, so two masks share a row where they share both keys."""
import numpy as np
import pytest

from sortnet_amd import functional as F
from sortnet_amd.layers import DropoutRegistry

WORD = 0xFFFFFFFF
FIRST, SECOND = 5 * 0x9e3779b9 & WORD, 6 * 0x9e3779b9 & WORD


def keys(seed, rows):
    """What is mixed into the two keys of rows 0 .. rows - 1, in one number (the mixing is one to one)."""
    row = np.arange(rows, dtype=np.uint32)
    a, b = (np.array([seed ^ c], dtype=np.uint32) + row for c in (FIRST, SECOND))
    return a.astype(np.uint64) << np.uint64(32) | b


def shared_rows(seeds, rows):
    every = np.concatenate([keys(s, rows) for s in seeds])
    return every.size - np.unique(every).size


def test_neighbouring_seeds_share_rows():
    """Why seeds that count up are spread."""
    assert shared_rows([1, 5], 2048) == 2044 and shared_rows([1, 2], 2048) == 0


@pytest.mark.parametrize("start", [0, 1, 17, 1000003 * 42, (1 << 26) - 60, (1 << 32) - 30, 123456789])
def test_spread_seeds_share_none(start):
    assert shared_rows([F.dropout_seed(start + k) for k in range(128)], 1 << 15) == 0


def test_spread_seeds_of_far_numbers_share_none():
    """Numbers that differ in any one or two of their low 26 bits, over 2^17 rows."""
    for a in range(0, 26, 5):
        numbers = [9] + [9 ^ 1 << a ^ (1 << b if b != a else 0) for b in range(26)]
        assert shared_rows([F.dropout_seed(n) for n in numbers], 1 << 17) == 0


def test_spread_seeds_are_all_different():
    bits = [F.dropout_seed(1 << k) for k in range(32)]
    assert sorted(bits) == [1 << k for k in range(32)]
    rng = np.random.default_rng(0)
    for n in rng.integers(0, 1 << 32, 200).tolist():
        assert F.dropout_seed(n) == sum(bits[k] for k in range(32) if n >> k & 1) == F.dropout_seed(n + (1 << 32))


def test_draws_of_a_layer_share_none():
    """The seeds that a layer takes in its passes, for several registries."""
    import torch
    from sortnet_amd import heads
    for seed in (0, 1, 42):
        layer, drawn = heads.BoundDropout(0.5, registry=DropoutRegistry(seed=seed)), []
        for _ in range(64):
            with pytest.raises(RuntimeError, match="must be a CUDA tensor"):      # the seed is drawn before the kernel refuses a tensor on the host
                layer(torch.zeros(2, 2))
            drawn.append(layer.last_seed)
        assert len(set(drawn)) == 64 and shared_rows(drawn, 1 << 14) == 0


def test_numbers_in_a_tensor():
    import torch
    numbers = [5, -1, 123456789, 1 << 31]
    assert F.dropout_seed(torch.tensor(numbers)).tolist() == [F.dropout_seed(n) for n in numbers]
