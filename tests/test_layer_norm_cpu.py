"""Layer norm on host tensors, its layer and its refusals."""

import pytest
import torch

from zookeeper_amd import nn as znn
from zookeeper_amd.ops import layer_norm


@pytest.mark.parametrize("shape", [(4, 7), (3, 5, 16), (9,), (2, 1)])
def test_matches_the_formula_and_its_gradients(shape):
    torch.manual_seed(0)
    x = torch.randn(shape, dtype=torch.float64, requires_grad=True)
    w = torch.rand(shape[-1], dtype=torch.float64, requires_grad=True)
    b = torch.rand(shape[-1], dtype=torch.float64, requires_grad=True)
    ref = torch.nn.functional.layer_norm(x, (shape[-1],), w, b, eps=1e-3)
    torch.testing.assert_close(layer_norm(x, w, b), ref, rtol=1e-12, atol=1e-12)
    assert torch.autograd.gradcheck(lambda *a: layer_norm(*a), (x, w, b))


def test_layer():
    m = znn.LayerNorm(6, scale=False)
    assert m.weight is None and [n for n, _ in m.named_parameters()] == ["bias"]
    assert "eps=0.001" in repr(m)
    x = torch.randn(3, 6, dtype=torch.bfloat16)
    y = znn.LayerNorm(6)(x)
    assert y.dtype == torch.bfloat16 and y.shape == x.shape
    with pytest.raises(ValueError, match="expected shape"):
        znn.LayerNorm(5)(x)


def test_refusals():
    x = torch.randn(3, 6)
    with pytest.raises(ValueError, match="last dimension"):
        layer_norm(torch.tensor(1.0))
    with pytest.raises(ValueError, match="last dimension"):
        layer_norm(torch.randn(3, 0))
    with pytest.raises(ValueError, match="eps"):
        layer_norm(x, eps=-1.0)
    with pytest.raises(ValueError, match="eps"):
        layer_norm(x, eps=float("nan"))
    with pytest.raises(ValueError, match="weight"):
        layer_norm(x, torch.ones(5))
    with pytest.raises(ValueError, match="bias"):
        layer_norm(x, torch.ones(6), torch.ones(1, 6))
    with pytest.raises(ValueError, match="floating"):
        layer_norm(torch.ones(3, 6, dtype=torch.int32))
    with pytest.raises(ValueError, match="floating"):
        layer_norm(x, torch.ones(6, dtype=torch.int64))
