"""Hybrid models without a dropout in their head are what they were before models could have one."""
import io

import pytest
import torch

from sortnet_amd.ell_inf_models import SortHybridModel, SortHybridModel2, SortHybridModelAvg
from sortnet_amd.heads import BoundDropout
from sortnet_amd.layers import DropoutRegistry


def make(kind, **kw):
    torch.manual_seed(0)
    model = kind(4, 32, (1, 8, 8), hidden=12, num_classes=5, dropout=None, registry=DropoutRegistry(seed=2), **kw)
    features = torch.randn(6, 32 * (4 if kind is SortHybridModel2 else 1))
    model._distance_features = lambda x, eps, up, down: (features, None, None)      # the distance layers run on the GPU
    model._pool = lambda z: z
    return model.train()


@pytest.mark.parametrize("kind", [SortHybridModel, SortHybridModel2, SortHybridModelAvg])
def test_modules_of_a_model_without_dropout(kind):
    model = make(kind)
    assert not any(isinstance(m, BoundDropout) for m in model.modules()) and "head_drop" not in dict(model.named_children())
    with_one = make(kind, head_dropout=0.5)
    assert isinstance(with_one.head_drop, BoundDropout) and with_one.state_dict().keys() == model.state_dict().keys()


@pytest.mark.parametrize("kind", [SortHybridModel, SortHybridModel2, SortHybridModelAvg])
def test_a_model_kept_from_before(kind):
    """A whole model that was saved when there was no such layer, and one that is copied from one with it."""
    model = make(kind)
    want = model(torch.zeros(6, 1, 8, 8)), model(torch.zeros(6, 1, 8, 8), torch.arange(6) % 5, 0.1)
    model._modules.pop("head_drop", None)
    assert torch.equal(model(torch.zeros(6, 1, 8, 8)), want[0])
    assert all(torch.equal(a, b) for a, b in zip(model(torch.zeros(6, 1, 8, 8), torch.arange(6) % 5, 0.1), want[1]))
    del model._distance_features, model._pool
    buffer = io.BytesIO()
    torch.save(model, buffer)
    buffer.seek(0)
    again = torch.load(buffer, weights_only=False)
    assert again.state_dict().keys() == model.state_dict().keys()
