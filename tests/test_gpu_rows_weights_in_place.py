"""The weights' gradient in the place of the weights: an output may be an input's array, and dx is then that of the weights as they were,
by whichever kernel the call is served."""
import pytest
import torch

from anode_b200 import ops
from tests.test_gpu_rms_norm import EPS, make, saved, weights
from tests.test_gpu_rotary import normal

pytestmark = pytest.mark.gpu


# one block, several blocks, ragged, rows that are not in step (a shift of dx), rows too wide to be held on chip
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("rows, cols, shift", [(3, 64, 0), (700, 1024, 0), (700, 1003, 0), (9, 100, 1), (700, 1000, 1), (5, 20000, 0), (300, 17000, 0)])
def test_norm(rows, cols, shift, dtype):
    dy, t, r, dt = saved(rows, cols, dtype)
    gamma = weights(cols, dtype)

    def out():
        return torch.empty(rows, cols + 8, device="cuda", dtype=dtype)[:, shift:shift + cols]
    dx, dg = out(), torch.empty_like(gamma)
    ops.RmsNormalizeAddOp.adjoint(dy, t, r, dx, gamma, dt, dg)
    both, z = gamma.clone(), out()
    ops.RmsNormalizeAddOp.adjoint(dy, t, r, z, both, dt, both)
    assert torch.equal(both, dg) and torch.equal(z, dx)


@pytest.mark.parametrize("rot", [64, 62])
def test_rotary(rot):
    tokens = 300
    q, k, dq, dk = (normal(tokens, h, 64, seed=s) for s, h in enumerate((6, 2, 6, 2)))
    freq, positions = ops.rotary_frequencies(rot), torch.arange(tokens, device="cuda")
    gq, gk = (1 + 0.2 * make(1, 64, torch.float32, s)[0] for s in (5, 6))

    def call(gq, gk, dgq, dgk):
        out = torch.empty_like(dq), torch.empty_like(dk)
        ops.RotaryPositionsOp.adjoint(positions, freq, dq, dk, *out, False, 1.0, EPS, q, k, gq, gk, dgq, dgk)
        return (*out, dgq, dgk)
    want = call(gq, gk, torch.empty_like(gq), torch.empty_like(gk))
    a, b = gq.clone(), gk.clone()
    assert all(torch.equal(x, y) for x, y in zip(call(a, b, a, b), want))
