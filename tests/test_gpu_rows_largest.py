"""How large rows may be: squares are summed in f32, so the norm holds while an rms stays below 2^64/sqrt(cols), the square root of the largest number over the
number of columns, and gives 0 beyond it."""
import math

import pytest
import torch

from anode_b200 import ops
from tests import test_gpu_rms_norm as norm
from tests.test_gpu_rms_norm import EPS, make, weights

pytestmark = pytest.mark.gpu

ROWS = 3


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("cols", [1, 64, 1003, 4096, 16384, 20000, 70001])
def test_rows_near_the_limit(cols, dtype):
    limit, gamma = 2.0 ** 64 / math.sqrt(cols), weights(cols, dtype)
    for part, held in ((0.9, True), (1.1, False)):
        # rows of one size, whose rms is that size to bf16's rounding, signs and places of larger and smaller values as they fall
        x = (make(ROWS, cols, torch.float32, 1).sign() * torch.where(torch.arange(cols, device="cuda") % 2 == 0, 1.2, math.sqrt(2 - 1.44)) * part * limit).to(dtype)
        if cols % 2:
            x[:, -1] = part * limit
        y, inv = torch.empty_like(x), torch.empty(ROWS, device="cuda")
        q, scale = torch.empty(ROWS, cols, device="cuda", dtype=torch.float8_e4m3fn), torch.empty(ROWS, -(-cols // 128), device="cuda")
        ops.RmsNormalizeAddOp.apply(EPS, x, y, gamma, None, None, inv)
        ops.RmsNormalizeAddQuantOp.apply(EPS, x, q, scale, gamma)
        if held:
            norm.check_forward(x, None, gamma, y, None, inv)
            back = (q.double() * scale.double().repeat_interleave(128, 1)[:, :cols])
            # half a step of e4m3, and of the type
            assert ((back - y.double()).abs() <= (2.0 ** -4 + 2 * norm.half_step(dtype)) * y.double().abs() + 2.0 ** -10 * scale.amax()).all()
        else:
            assert (y == 0).all() and (inv == 0).all() and (q.float() == 0).all() and (scale == 2.0 ** -96 / 448).all()
