"""The adjoint of the RMS norm over the range of f32: rows of large and of tiny values, gradients far smaller than the rows they belong to.
Every kernel that may serve a call, whole rows, ragged ones, rows that are not in step and rows too wide to be held on chip, is held to
the tolerances of test_gpu_rms_norm.py, which are relative to what the formula is made of."""
import pytest
import torch

from anode_b200 import ops
from tests import test_gpu_rms_norm as norm
from tests.test_gpu_rms_norm import make, weights

pytestmark = pytest.mark.gpu

# rows, cols, and where in a wider array the rows of dy, total and dx begin
FORMS = [(5, 64, (0, 0, 0)), (300, 96, (0, 0, 0)), (40, 1024, (0, 0, 0)), (300, 1000, (3, 3, 3)), (7, 77, (1, 1, 1)), (33, 9001, (0, 0, 0)), (5, 100, (0, 1, 2)),
         (200, 1030, (0, 3, 5)), (3, 20000, (0, 0, 0))]
# the rows' rms and the gradients' size.  Squares of 1e17 pass f32 as the sum of 3e4 columns, so that the forward pass serves these rows, too;
# products of a gradient and a row's element stay above 1e-38, the smallest normal number
SIZES = [(1e8, 1.0), (1e13, 1.0), (1e15, 1.0), (1e17, 1.0), (1e13, 1e-9), (1e15, 1e-12), (1e17, 1e-15), (1e-8, 1.0), (1e-12, 1.0), (1e-15, 1e-6), (1e-17, 1e-12)]


def saved(rows, cols, at, dtype, size, small):
    def rows_of(seed, first, scale):
        return (make(rows, cols + 8, torch.float32, seed).double() * scale).to(dtype)[:, first:first + cols]
    t = rows_of(1, at[1], size)
    return rows_of(2, at[0], small), t, t.double().square().mean(-1).rsqrt().float(), rows_of(3, at[2], small / size)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("size, small", SIZES)
def test_adjoint_of_rows_of_any_size(size, small, dtype):
    for rows, cols, at in FORMS:
        dy, t, r, dt = saved(rows, cols, at, dtype, size, small)
        for gamma, extra in ((weights(cols, dtype), None), (None, dt)):
            dx, dg = make(rows, cols + 8, dtype, 4)[:, at[2]:at[2] + cols], torch.empty(cols, device="cuda", dtype=torch.float32 if gamma is None else dtype)
            ops.RmsNormalizeAddOp.adjoint(dy, t, r, dx, gamma, extra, dg)
            norm.check_backward(dy, t, r, gamma, extra, dx, dg, "%d rows of %d at %s: " % (rows, cols, at))


@pytest.mark.parametrize("cols", [64, 77, 20000])
def test_constant_rows_have_no_gradient(cols):
    """dy along the row itself: the projection takes all of it, whatever the row's size."""
    for size in (1.0, 1e8, 1e14, 1e16):
        x = torch.full((3, cols), size, device="cuda")
        layer = ops.RmsNormAdd(cols, epsilon=0.0)
        layer.forward(x)
        dx = layer.backward(torch.ones_like(x))
        # what is left is rounding: of 1/rms, which the projection has twice, of the sum (twice row_bound), and 10u of the steps between
        assert float(dx.abs().max()) * size <= 4 * norm.row_bound(cols) + 10 * norm.U, (size, dx[0, 0])
