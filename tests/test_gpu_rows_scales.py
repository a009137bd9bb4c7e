"""The 8-bit form against its forward pass: the norm is the same bits in f32, so scales are max |y|/448 rounded to nearest by whichever kernel the call is
served, and values are the nearest e4m3 of y/scale but where that is as good as the middle of two.  The quotient is y times 448/max |y|: u = 2^-24 each for that,
for the product, and for the scale that it is measured by."""
import pytest
import torch

from anode_b200 import ops
from tests.test_gpu_rms_norm import EPS, U, e4m3, make

pytestmark = pytest.mark.gpu

OFF = 3 * U


@pytest.mark.parametrize("size", [1.0, 2.0 ** -90, 2.0 ** -60, 1e20, 3e37])
@pytest.mark.parametrize("rows, cols, shift", [(700, 1024, 0), (300, 4096, 0), (300, 4099, 0), (50, 60, 0), (3000, 130, 0), (200, 16384, 0), (40, 20000, 0), (40, 30000, 0),
                                               (300, 1000, 1)])
def test_scales_are_the_nearest_quotients(rows, cols, shift, size):
    """Weights of any size: y from below the least scale to the largest numbers."""
    x, gamma = make(rows, cols, torch.float32, 1), (1 + 0.2 * make(1, cols, torch.float32, 2)[0].double()).mul(size).float()
    gamma[::31] *= 2.0 ** -12
    z, q = (torch.empty(rows, cols + 8, device="cuda", dtype=t)[:, shift:shift + cols] for t in (torch.float32, torch.float8_e4m3fn))
    ops.RmsNormalizeAddOp.apply(EPS, x, z, gamma)
    y = z.double()
    assert y.isfinite().all()
    for block in (0, 128):
        width = block or cols
        groups = -(-cols // width)
        scale = torch.empty((rows, groups) if block else (rows,), device="cuda")
        ops.RmsNormalizeAddQuantOp.apply(EPS, x, q, scale, gamma)
        peak = torch.nn.functional.pad(y.abs(), (0, groups * width - cols)).view(rows, groups, width).amax(2)
        want = (peak.clamp(min=2.0 ** -96) / 448).float()
        assert torch.equal(scale.view(rows, groups), want)
        v = y / want.double().repeat_interleave(width, 1)[:, :cols]
        nearest = e4m3(v.clamp(-448, 448))
        assert ((q.double() - v).abs() <= (nearest - v).abs() + 2 * OFF * v.abs()).all()


def test_infinite_weights():
    """An infinite y: its group's scale is infinite, the infinity is no number, and what is finite beside it is 0."""
    for rows, cols in ((3, 256), (3, 257), (3, 30000)):
        x, gamma = make(rows, cols, torch.float32, 3).abs() + 1, torch.ones(cols, device="cuda")
        gamma[5] = float("inf")
        for shape in ((rows,), (rows, -(-cols // 128))):
            q, scale = torch.empty(rows, cols, device="cuda", dtype=torch.float8_e4m3fn), torch.empty(shape, device="cuda")
            ops.RmsNormalizeAddQuantOp.apply(EPS, x, q, scale, gamma)
            first = scale.view(rows, -1)[:, 0]
            assert first.isinf().all() and q[:, 5].float().isnan().all() and (q[:, :5].float() == 0).all() and (q[:, 6:128].float() == 0).all()
            assert scale.view(rows, -1)[:, 1:].isfinite().all()
