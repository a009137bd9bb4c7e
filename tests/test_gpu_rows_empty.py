"""Arrays without a row do nothing, wherever their rows would lie."""
import pytest
import torch

from anode_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape, cut", [((0, 3, 4, 8), (slice(None), slice(None), slice(0, 2))), ((3, 0, 4, 8), (slice(0, 2), slice(None), slice(1, 3))),
                                        ((2, 3, 4, 8), (slice(0, 0), slice(0, 2), slice(0, 3)))])
def test_slices_without_rows(shape, cut):
    x = torch.zeros(shape, device="cuda")[cut]
    layer = ops.RmsNormAdd(8)
    layer.dgamma.fill_(7)
    y, total = layer.forward(x, x)
    assert y.shape == total.shape == x.shape and layer.infer_quant(x, x)[0].shape == x.shape
    assert layer.backward(x, x).shape == x.shape and (layer.dgamma == 0).all()
