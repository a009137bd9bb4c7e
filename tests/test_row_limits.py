"""Rows wider than the kernels' 32-bit columns count safely are refused, on any machine, before anything is launched: the kernels' loops count up to a
block's threads beyond the last column."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from anode_b200 import _lib, ops
from tests.test_row_refusals import DIMS, norm, norm_grad, quant

MOST = 1 << 31


@pytest.mark.parametrize("rows", [0, 1, 4])
@pytest.mark.parametrize("cols", [MOST, MOST + 1, (1 << 32) - 256, (1 << 32) - 1])
def test_the_c_calls_refuse_rows_of_2_to_the_31_columns(rows, cols):
    strides = dict(x_stride=cols, residual_stride=cols, total_stride=cols)
    assert norm(rows=rows, cols=cols, y_stride=cols, **strides) == DIMS
    for block, scales in ((0, dict(scale_row_stride=1)), (128, dict(scale_row_stride=1 << 26))):
        assert quant(rows=rows, cols=cols, block=block, q_stride=cols, **strides, **scales) == DIMS
    for dgamma in (None, 7 * 0x10000):
        assert norm_grad(rows=rows, cols=cols, dy_stride=cols, total_stride=cols, dtotal_stride=cols, dx_stride=cols, dgamma=dgamma, workspace_bytes=1 << 62) == DIMS


def test_a_column_less_is_refused_for_what_is_wrong_with_it_only():
    assert norm(cols=MOST - 1, x=None) == quant(cols=MOST - 1, scale_row_stride=1 << 26, x=None) == norm_grad(cols=MOST - 1, dy=None, workspace_bytes=1 << 62) == -1


@pytest.mark.filterwarnings("ignore:Accessing the data pointer of FakeTensor")
def test_python_refuses_them_as_too_wide():
    with FakeTensorMode():
        x = torch.empty(1, MOST, device="cuda:0", dtype=torch.bfloat16)
        r = torch.empty(1, device="cuda:0")
        q = torch.empty(1, MOST, device="cuda:0", dtype=torch.float8_e4m3fn)
        for call in (lambda: ops.RmsNormalizeAddOp.apply(1e-5, x, x), lambda: ops.RmsNormalizeAddOp.adjoint(x, x, r, x), lambda: ops.RmsNormalizeAddQuantOp.apply(1e-5, x, q, r)):
            with pytest.raises(ValueError, match="too many columns"):
                call()


def test_the_error_text_names_the_reason():
    assert "2^31" in _lib.ERRORS[DIMS]
