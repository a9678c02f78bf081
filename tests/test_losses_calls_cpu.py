"""Calls of the training-loss terms that are refused before anything runs, and the versions of their two libraries; without a GPU."""
import pytest
import torch

import lpmm.functional as F
from lpmm import _native


def _stored(**change):
    quant = dict(b=8, signed=True, quant_type="power-1", round_type="real-nearest", scale_type="group", qmap=torch.linspace(-1, 1, 256),
                 max1=torch.ones(1, 1), scaled_shape=torch.Size((1, 128)), dtype=torch.float32, stride=None)
    quant.update(change)
    return quant


@pytest.mark.parametrize("name,change,values", [
    ("qmap", dict(qmap={(8, True): {"power-1": None}}), torch.zeros(2049, dtype=torch.int8)),
    ("max1", dict(max1=None), torch.zeros(2049, dtype=torch.int8)),
    ("max1", dict(max1=None), torch.randn(3, 4)),  # plain values: the codes' keywords would be passed over
    ("max1", dict(max1=[1.0]), torch.zeros(2049, dtype=torch.int8)),
])
def test_a_stored_teacher_needs_its_map_and_scales(name, change, values):
    with pytest.raises(TypeError, match=f"{name} must be a tensor"):
        F.distill_loss(torch.randn(3, 20), values, torch.randint(0, 20, (3, 4)), teacher_quant=_stored(**change))


@pytest.mark.parametrize("scale,qmap", [(None, torch.linspace(-1, 1, 256)), (torch.ones(1, 1), None)])
def test_the_host_side_takes_map_and_scales_together(scale, qmap):
    with pytest.raises(RuntimeError, match="both max1 and qmap"):
        _native.losses().distill_loss(torch.randn(3, 20), torch.zeros(2049, dtype=torch.int8), torch.randint(0, 20, (3, 4)), 1.0, None, 1.0, 0.0,
                                      -100, 2, scale, qmap, 128, 8)
