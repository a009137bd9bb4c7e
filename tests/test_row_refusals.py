"""Row-wise operators (RMS norm with the residual's addition, its 8-bit form, rotary positions): what their entry points refuse, on any
machine.  Nothing of a refused call reaches CUDA: addresses here are numbers that no kernel may see."""
import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from anode_b200 import _lib, ops

P = 0x10000          # an address that is aligned, and never used
NULL, DIMS, WORKSPACE, ALIGN, TYPE, STRIDE = -1, -2, -3, -6, -8, -9


def norm(**change):
    a = dict(type=2, rows=4, cols=8, epsilon=1e-5, x=P, x_stride=8, residual=2 * P, residual_stride=8, gamma=3 * P, gamma_type=2, y=4 * P, y_stride=8,
             total=5 * P, total_stride=8, inv_rms=6 * P)
    a.update(change)
    return _lib.load().anode_gpu_rms_norm_add_fwd(*a.values(), None, None)


def norm_grad(**change):
    a = dict(type=2, rows=4, cols=8, dy=P, dy_stride=8, total=2 * P, total_stride=8, inv_rms=3 * P, gamma=4 * P, gamma_type=0, dtotal=5 * P, dtotal_stride=8,
             dx=6 * P, dx_stride=8, dgamma=7 * P, workspace=8 * P, workspace_bytes=1 << 30)
    a.update(change)
    return _lib.load().anode_gpu_rms_norm_add_bwd(*a.values(), None, None)


def quant(**change):
    a = dict(type=2, rows=4, cols=256, epsilon=1e-5, block=128, x=P, x_stride=256, residual=2 * P, residual_stride=256, gamma=3 * P, gamma_type=2,
             q=4 * P, q_stride=256, scale=5 * P, scale_row_stride=2, scale_group_stride=1, total=6 * P, total_stride=256)
    a.update(change)
    return _lib.load().anode_gpu_rms_norm_add_quant_fwd(*a.values(), None, None)


def heads(p, n=4, dim=8, **change):
    a = dict(data=p, batch_stride=6 * n * dim, seq_stride=n * dim, head_stride=dim, heads=n)
    a.update(change)
    return _lib.Heads(*a.values())


ROTARY = dict(type=2, batch=2, seq=6, dim=8, rot=4, interleaved=0, amplitude=1.0, freq=P, positions=2 * P, position_bytes=8, pos_batch=6, pos_seq=1,
              norm=1, epsilon=1e-5, gamma_q=3 * P, gamma_k=4 * P, gamma_type=0)


def rotary(**change):
    a = dict(ROTARY, q=heads(5 * P), k=heads(6 * P, 2), q_out=heads(7 * P), k_out=heads(8 * P, 2))
    a.update(change)
    return _lib.load().anode_gpu_rotary_positions_fwd(*[ctypes.byref(v) if isinstance(v, _lib.Heads) else v for v in a.values()], None, None)


def rotary_grad(**change):
    a = dict(ROTARY, dq_out=heads(5 * P), dk_out=heads(6 * P, 2), q=heads(7 * P), k=heads(8 * P, 2), dq=heads(9 * P), dk=heads(10 * P, 2),
             dgamma_q=11 * P, dgamma_k=12 * P, workspace=13 * P, workspace_bytes=1 << 30)
    a.update(change)
    return _lib.load().anode_gpu_rotary_positions_bwd(*[ctypes.byref(v) if isinstance(v, _lib.Heads) else v for v in a.values()], None, None)


@pytest.mark.parametrize("call, change, code", [
    (norm, dict(type=3), TYPE), (norm, dict(gamma_type=-1), TYPE), (norm, dict(cols=0), DIMS), (norm, dict(rows=1 << 41), DIMS),
    (norm, dict(x=None), NULL), (norm, dict(y=None), NULL), (norm, dict(x=P + 1), ALIGN), (norm, dict(y=P + 1), ALIGN), (norm, dict(gamma=P + 1), ALIGN),
    (norm, dict(residual=P + 1), ALIGN), (norm, dict(total=P + 1), ALIGN), (norm, dict(inv_rms=P + 2), ALIGN),
    (norm, dict(y_stride=7), STRIDE), (norm, dict(total_stride=0), STRIDE), (norm, dict(residual=None), NULL),
    (norm, dict(total=4 * P), STRIDE), (norm, dict(y=P, x_stride=16), STRIDE), (norm, dict(total=2 * P, residual_stride=16), STRIDE),
    (norm_grad, dict(type=-1), TYPE), (norm_grad, dict(gamma_type=3), TYPE), (norm_grad, dict(cols=0), DIMS), (norm_grad, dict(dy=None), NULL),
    (norm_grad, dict(total=None), NULL), (norm_grad, dict(inv_rms=None), NULL), (norm_grad, dict(dx=None), NULL), (norm_grad, dict(dx_stride=4), STRIDE),
    (norm_grad, dict(dx=P, dy_stride=16), STRIDE), (norm_grad, dict(dx=5 * P, dtotal_stride=0), STRIDE), (norm_grad, dict(workspace=None), WORKSPACE),
    (norm_grad, dict(workspace=P + 8), WORKSPACE), (norm_grad, dict(workspace_bytes=31), WORKSPACE), (norm_grad, dict(dgamma=P + 2), ALIGN),
    (norm_grad, dict(dtotal=P + 1), ALIGN), (norm_grad, dict(inv_rms=P + 1), ALIGN),
    (quant, dict(block=64), DIMS), (quant, dict(scale=None), NULL), (quant, dict(scale=P + 2), ALIGN), (quant, dict(scale_row_stride=0), STRIDE),
    (quant, dict(scale_group_stride=0), STRIDE), (quant, dict(scale_row_stride=1), STRIDE), (quant, dict(q=None), NULL), (quant, dict(q=P), STRIDE),
    (quant, dict(q_stride=255), STRIDE), (quant, dict(type=4), TYPE), (quant, dict(cols=0), DIMS),
    (rotary, dict(type=3), TYPE), (rotary, dict(position_bytes=2), TYPE), (rotary, dict(rot=3), DIMS), (rotary, dict(rot=0), DIMS), (rotary, dict(rot=10), DIMS),
    (rotary, dict(dim=1026, rot=2), DIMS), (rotary, dict(q=None), NULL), (rotary, dict(k=None), NULL), (rotary, dict(k_out=None), NULL),
    (rotary, dict(freq=None), NULL), (rotary, dict(positions=None), NULL), (rotary, dict(positions=P + 4), ALIGN), (rotary, dict(freq=P + 4), ALIGN),
    (rotary, dict(q_out=heads(7 * P, 3)), DIMS), (rotary, dict(q_out=heads(7 * P, head_stride=7)), STRIDE), (rotary, dict(q_out=heads(7 * P, seq_stride=0)), STRIDE),
    (rotary, dict(q_out=heads(7 * P, seq_stride=8)), STRIDE), (rotary, dict(q_out=heads(7 * P, batch_stride=8)), STRIDE),
    (rotary, dict(q_out=heads(5 * P, seq_stride=64, batch_stride=512)), STRIDE), (rotary, dict(q=heads(P + 1)), ALIGN), (rotary, dict(q=heads(None)), NULL),
    (rotary, dict(gamma_q=P + 2), ALIGN), (rotary, dict(gamma_type=5), TYPE), (rotary, dict(q=heads(P, 0), q_out=heads(P, 0)), DIMS),
    (rotary_grad, dict(q=None), NULL), (rotary_grad, dict(k=None), NULL), (rotary_grad, dict(workspace=None), WORKSPACE),
    (rotary_grad, dict(workspace_bytes=8), WORKSPACE), (rotary_grad, dict(norm=0), NULL), (rotary_grad, dict(dk_out=None, dk=None, k=None), NULL),
    (rotary_grad, dict(q=heads(7 * P, 3)), DIMS), (rotary_grad, dict(dq=heads(9 * P, head_stride=0)), STRIDE),
    (rotary_grad, dict(dq=heads(7 * P, seq_stride=64, batch_stride=512)), STRIDE), (rotary_grad, dict(dgamma_q=P + 2), ALIGN),
])
def test_the_c_calls_refuse(call, change, code):
    assert call(**change) == code


@pytest.mark.parametrize("call, change", [
    (rotary, dict(k_out=heads(7 * P, 2))), (rotary, dict(q_out=heads(6 * P))), (rotary, dict(k_out=heads(5 * P, 2))),
    (rotary, dict(k=heads(5 * P, 2), q_out=heads(5 * P))),
    (rotary_grad, dict(dk=heads(9 * P, 2))), (rotary_grad, dict(dq=heads(6 * P))), (rotary_grad, dict(dk=heads(5 * P, 2))),
    (rotary_grad, dict(dq=heads(8 * P))), (rotary_grad, dict(dk=heads(7 * P, 2))), (rotary_grad, dict(dgamma_k=11 * P)),
])
def test_queries_and_keys_side_by_side_share_no_output(call, change):
    """The two are worked on at the same time: an output in the place of any array of the other one has no defined result."""
    assert call(**change) == STRIDE


def test_no_rows_and_no_tokens_do_nothing():
    assert norm(rows=0, x=None, residual=None, total=None, y=None) == 0
    assert quant(rows=0, scale=None, x=None, q=None, residual=None, total=None) == 0
    assert norm_grad(rows=0, dgamma=None) == 0
    assert rotary(batch=0) == 0 and rotary(seq=0) == 0 and rotary_grad(seq=0, dgamma_q=None, dgamma_k=None) == 0


def python_calls(t, w, f32, q8, scale, heads_, pos, freq):
    norm_, quant_, turn = ops.RmsNormalizeAddOp, ops.RmsNormalizeAddQuantOp, ops.RotaryPositionsOp
    return {
        "norm": lambda: norm_.apply(1e-5, t, t, w, t, t, f32),
        "norm grad": lambda: norm_.adjoint(t, t, f32, t, w, t, w),
        "quant": lambda: quant_.apply(1e-5, t, q8, scale, w, t, t),
        "rotary": lambda: turn.apply(pos, freq, heads_, heads_, heads_, heads_),
        "rotary grad": lambda: turn.adjoint(pos, freq, heads_, heads_, heads_, heads_, False, 1.0, 1e-5, heads_, heads_, w, w, w, w),
    }


def tensors(device):
    e = lambda *s, dtype=torch.float32: torch.empty(s, device=device, dtype=dtype)      # noqa: E731
    return e(4, 8), e(8), e(4), e(4, 8, dtype=torch.float8_e4m3fn), e(4), e(4, 2, 8), e(4, dtype=torch.int64), e(4, dtype=torch.float64)


@pytest.mark.parametrize("name", sorted(python_calls(*[None] * 8)))
def test_host_tensors_are_refused_before_anything_is_asked_of_cuda(name):
    with pytest.raises(ValueError, match="CUDA tensor"):
        python_calls(*tensors("cpu"))[name]()


@pytest.mark.parametrize("name", sorted(python_calls(*[None] * 8)))
def test_what_is_no_tensor_is_refused(name):
    with pytest.raises((ValueError, TypeError)):
        python_calls(*["no"] * 8)[name]()


@pytest.mark.filterwarnings("ignore:Accessing the data pointer of FakeTensor")
def test_python_checks_of_sizes_types_and_devices():
    """Arrays that claim to be on a device: each of these is refused for what it is, before a stream or an address is needed."""
    norm_, quant_, turn = ops.RmsNormalizeAddOp, ops.RmsNormalizeAddQuantOp, ops.RotaryPositionsOp
    with FakeTensorMode():
        def e(*s, dtype=torch.float32, device="cuda:0"):
            return torch.empty(s, device=device, dtype=dtype)
        t, w, r = e(4, 8), e(8), e(4)
        cases = [
            ("sizes", lambda: norm_.apply(1e-5, t, e(4, 9))), ("type", lambda: norm_.apply(1e-5, t, e(4, 8, dtype=torch.float16))),
            ("float32, float16 or bfloat16", lambda: norm_.apply(1e-5, e(4, 8, dtype=torch.float64), t)), ("packed", lambda: norm_.apply(1e-5, e(8, 4).t(), t)),
            ("one distance", lambda: norm_.apply(1e-5, e(4, 6, 8)[:, :3], e(4, 3, 8))), ("weight per column", lambda: norm_.apply(1e-5, t, t, e(9))),
            ("without one", lambda: norm_.apply(1e-5, t, e(4, 8), w, None, e(4, 8))), ("per row", lambda: norm_.apply(1e-5, t, t, w, None, None, e(5))),
            ("other weights", lambda: norm_.adjoint(t, t, r, t, w, None, e(8, dtype=torch.float16))),
            ("Accumulate", lambda: norm_.adjoint(t, t, r, t, w, t, None, ops.WriteCap.Accumulate)), ("inv_rms", lambda: norm_.adjoint(t, t, None, t)),
            ("type", lambda: quant_.apply(1e-5, t, e(4, 8, dtype=torch.uint8), r)), ("128 columns", lambda: quant_.apply(1e-5, t, e(4, 8, dtype=torch.float8_e4m3fn), e(4, 2))),
            ("heads, dim", lambda: turn.apply(None, None, t, None, t, None)),
        ]
        h, k, pos, freq = e(4, 2, 8), e(4, 1, 8), e(4, dtype=torch.int64), e(4, dtype=torch.float64)
        cases += [
            ("number of heads", lambda: turn.apply(pos, freq, h, None, k, None)), ("given together", lambda: turn.apply(pos, freq, h, k, h, None)),
            ("one position per token", lambda: turn.apply(e(5, dtype=torch.int64), freq, h, k, h, k)), ("one position per token", lambda: turn.apply(e(4), freq, h, k, h, k)),
            ("float64", lambda: turn.apply(pos, e(4), h, k, h, k)), ("no norm", lambda: turn.apply(pos, freq, h, k, h, k, False, 1.0, None, w, w)),
            ("first array", lambda: turn.apply(pos, freq, h, e(3, 1, 8), h, k)), ("no keys", lambda: turn.adjoint(pos, freq, h, None, h, None, False, 1.0, 1e-5, h, None, w, None, w, w)),
            ("q: expected", lambda: turn.adjoint(pos, freq, h, k, h, k, False, 1.0, 1e-5)),
        ]
        for text, call in cases:
            with pytest.raises(ValueError, match=text):
                call()


@pytest.mark.skipif(torch.cuda.is_available(), reason="tensors that claim to be on a second device need a machine without a first")
@pytest.mark.filterwarnings("ignore:Accessing the data pointer of FakeTensor")
def test_tensors_of_two_devices_are_refused():
    with FakeTensorMode():
        x, y = torch.empty(4, 8, device="cuda:0"), torch.empty(4, 8, device="cuda:1")
        with pytest.raises(ValueError, match="another device"):
            ops.RmsNormalizeAddOp.apply(1e-5, x, y)


def test_layers_refuse():
    with pytest.raises(ValueError):
        ops.rotary_frequencies(3, device="cpu")
    with pytest.raises(ValueError):
        ops.rotary_frequencies(4, factor=0, device="cpu")
    with pytest.raises(ValueError):
        ops.RotaryPositions(8, rot=10, device="cpu")
    with pytest.raises(RuntimeError):
        ops.RmsNormAdd(8, device="cpu").backward(torch.zeros(1, 8))
    with pytest.raises(ValueError):
        ops.RmsNormAdd(8, device="cpu").infer_quant(torch.zeros(1, 8), block=64)


def test_frequencies():
    f = ops.rotary_frequencies(8, base=100.0, device="cpu")
    assert f.dtype == torch.float64 and torch.allclose(f, torch.tensor([1.0, 100 ** -0.25, 0.1, 100 ** -0.75], dtype=torch.float64), rtol=1e-15, atol=0)
    assert torch.equal(ops.rotary_frequencies(8, base=100.0, factor=4.0, device="cpu"), f / 4)
    s = ops.rotary_frequencies(64, factor=8.0, context=1024, device="cpu")
    plain = ops.rotary_frequencies(64, device="cpu")
    turns = 1024 * plain / 6.283185307179586
    assert torch.allclose(s[turns > 4], plain[turns > 4], rtol=1e-15, atol=0) and torch.allclose(s[turns < 1], plain[turns < 1] / 8, rtol=1e-15, atol=0)
    between = (turns > 1) & (turns < 4)
    assert between.any() and ((s < plain) & (s > plain / 8))[between].all()


def test_layers_keep_what_their_backward_pass_reads():
    """forward in place would leave the backward pass with the norm in the place of its input; infer may be in place."""
    x, pos, q = torch.zeros(4, 8), torch.arange(4), torch.zeros(4, 2, 8)
    with pytest.raises(ValueError, match="backward pass"):
        ops.RmsNormAdd(8, device="cpu").forward(x, out=x)
    turn = ops.RotaryPositions(8, norm=True, device="cpu")
    with pytest.raises(ValueError, match="backward pass"):
        turn.forward(q, None, pos, q_out=q)
    with pytest.raises(ValueError, match="backward pass"):
        turn.forward(q, q.clone(), pos, None, q.view(4, 2, 8))
    for call in (lambda: ops.RmsNormAdd(8, device="cpu").infer(x, out=x), lambda: turn.infer(q, None, pos, q_out=q),
                 lambda: ops.RotaryPositions(8, device="cpu").forward(q, None, pos, q_out=q), lambda: ops.RmsNormAdd(8, device="cpu").forward(x, x.clone(), out=x)):
        with pytest.raises(ValueError, match="CUDA tensor"):      # (as far as a machine without a device goes)
            call()
