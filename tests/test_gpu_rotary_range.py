"""The adjoint of the rotary positions with a norm over the range of f32: heads of large values, gradients far smaller than the heads they belong
to, in both layouts and for pairs that lie anywhere.  Tolerances as in test_gpu_rotary.py."""
import pytest
import torch

from anode_b200 import ops
from tests import test_gpu_rotary as turn
from tests.test_gpu_rms_norm import EPS

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("dim, rot", [(64, 64), (128, 62), (256, 128), (33, 32), (500, 500)])
@pytest.mark.parametrize("size, small", [(1e8, 1.0), (1e13, 1.0), (1e15, 1e-9), (1e16, 1e-6), (1e17, 1.0), (1e17, 1e-15)])
def test_adjoint_of_heads_of_any_size(size, small, dim, rot, dtype):
    tokens, freq = 37, ops.rotary_frequencies(rot)
    positions = torch.arange(tokens, device="cuda") + 100
    gamma = 1 + 0.2 * turn.normal(dim, seed=5)
    for interleaved in (False, True):
        x, d = ([(turn.normal(tokens, n, dim, seed=s + n).double() * by).to(dtype) for n in (5, 2)] for s, by in ((1, size), (2, small)))
        out, dg = [torch.empty_like(t) for t in x], [torch.empty_like(gamma) for _ in x]
        ops.RotaryPositionsOp.adjoint(positions, freq, *d, *out, interleaved, 1.0, EPS, *x, gamma, gamma, *dg)
        for k in range(2):
            turn.check_backward(d[k], x[k], out[k], dg[k], positions, freq, interleaved, 1.0, True, gamma, "%d: " % k)
