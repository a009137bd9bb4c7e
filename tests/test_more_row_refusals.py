"""Layer norm, rows of a table by tokens and log probabilities of tokens: what their entry points refuse, on any machine.  Nothing of a refused call reaches
CUDA: addresses here are numbers that no kernel may see."""
import math

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from anode_b200 import _lib, ops

P = 0x10000          # an address that is aligned, and never used
NULL, DIMS, WORKSPACE, ALIGN, TYPE, STRIDE, VALUE = -1, -2, -3, -6, -8, -9, -10
MOST = 1 << 31


def layer(**change):
    a = dict(type=2, rows=4, cols=8, epsilon=1e-5, x=P, x_stride=8, residual=2 * P, residual_stride=8, gamma=3 * P, beta=4 * P, weight_type=2, y=5 * P, y_stride=8,
             total=6 * P, total_stride=8, mean=7 * P, inv_std=8 * P)
    a.update(change)
    return _lib.load().anode_gpu_layer_norm_add_fwd(*a.values(), None, None)


def layer_grad(**change):
    a = dict(type=2, rows=4, cols=8, dy=P, dy_stride=8, total=2 * P, total_stride=8, mean=3 * P, inv_std=4 * P, gamma=5 * P, weight_type=0, dtotal=6 * P, dtotal_stride=8,
             dx=7 * P, dx_stride=8, dgamma=8 * P, dbeta=9 * P, workspace=10 * P, workspace_bytes=1 << 30)
    a.update(change)
    return _lib.load().anode_gpu_layer_norm_add_bwd(*a.values(), None, None)


def embed(**change):
    a = dict(type=2, tokens=4, vocab=10, cols=8, scale=1.0, token=P, token_bytes=8, table=2 * P, table_stride=8, y=3 * P, y_stride=8)
    a.update(change)
    return _lib.load().anode_gpu_embed_tokens_fwd(*a.values(), None, None)


def embed_grad(**change):
    a = dict(type=2, tokens=4, vocab=10, cols=8, scale=1.0, token=P, token_bytes=8, dy=2 * P, dy_stride=8, dtable=3 * P, dtable_stride=8, dtable_type=2, accumulate=0,
             workspace=4 * P, workspace_bytes=1 << 30)
    a.update(change)
    return _lib.load().anode_gpu_embed_tokens_bwd(*a.values(), None, None)


def probs(**change):
    a = dict(type=2, rows=4, vocab=40, scale=1.0, logits=P, stride=40, token=2 * P, token_bytes=8, logprob=3 * P, entropy=4 * P, stats=5 * P, top=20, top_logprob=6 * P,
             top_token=7 * P, top_token_bytes=8)
    a.update(change)
    return _lib.load().anode_gpu_token_log_probs_fwd(*a.values(), None, None)


def probs_grad(**change):
    a = dict(type=2, rows=4, vocab=40, scale=1.0, logits=P, stride=40, token=2 * P, token_bytes=8, stats=3 * P, entropy=4 * P, dlogprob=5 * P, dentropy=6 * P, dlogits=7 * P,
             dstride=40)
    a.update(change)
    return _lib.load().anode_gpu_token_log_probs_bwd(*a.values(), None, None)


@pytest.mark.parametrize("call, change, code", [
    (layer, dict(type=3), TYPE), (layer, dict(weight_type=-1), TYPE), (layer, dict(cols=0), DIMS), (layer, dict(rows=1 << 41), DIMS), (layer, dict(cols=MOST), DIMS),
    (layer, dict(x=None), NULL), (layer, dict(y=None), NULL), (layer, dict(x=P + 1), ALIGN), (layer, dict(y=P + 1), ALIGN), (layer, dict(gamma=P + 1), ALIGN),
    (layer, dict(beta=P + 1), ALIGN), (layer, dict(gamma=None, beta=P + 1), ALIGN), (layer, dict(residual=P + 1), ALIGN), (layer, dict(total=P + 1), ALIGN),
    (layer, dict(mean=P + 2), ALIGN), (layer, dict(inv_std=P + 2), ALIGN), (layer, dict(mean=8 * P), STRIDE), (layer, dict(y_stride=7), STRIDE),
    (layer, dict(total_stride=0), STRIDE), (layer, dict(residual=None), NULL), (layer, dict(total=5 * P), STRIDE), (layer, dict(y=P, x_stride=16), STRIDE),
    (layer, dict(total=2 * P, residual_stride=16), STRIDE),
    (layer_grad, dict(type=-1), TYPE), (layer_grad, dict(weight_type=3), TYPE), (layer_grad, dict(cols=0), DIMS), (layer_grad, dict(cols=MOST), DIMS), (layer_grad, dict(dy=None), NULL),
    (layer_grad, dict(total=None), NULL), (layer_grad, dict(mean=None), NULL), (layer_grad, dict(inv_std=None), NULL), (layer_grad, dict(dx=None), NULL),
    (layer_grad, dict(dx_stride=4), STRIDE), (layer_grad, dict(dx=P, dy_stride=16), STRIDE), (layer_grad, dict(dx=6 * P, dtotal_stride=0), STRIDE),
    (layer_grad, dict(workspace=None), WORKSPACE), (layer_grad, dict(workspace=P + 8), WORKSPACE), (layer_grad, dict(workspace_bytes=255), WORKSPACE),
    (layer_grad, dict(dgamma=None, workspace=None), WORKSPACE), (layer_grad, dict(dgamma=P + 2), ALIGN), (layer_grad, dict(dbeta=P + 2), ALIGN),
    (layer_grad, dict(dbeta=8 * P), STRIDE), (layer_grad, dict(dbeta=5 * P), STRIDE), (layer_grad, dict(dtotal=P + 1), ALIGN), (layer_grad, dict(mean=P + 1), ALIGN),
    (embed, dict(type=3), TYPE), (embed, dict(token_bytes=2), TYPE), (embed, dict(cols=0), DIMS), (embed, dict(vocab=0), DIMS), (embed, dict(cols=MOST), DIMS),
    (embed, dict(vocab=MOST), DIMS), (embed, dict(tokens=MOST), DIMS), (embed, dict(token=None), NULL), (embed, dict(table=None), NULL), (embed, dict(y=None), NULL),
    (embed, dict(token=P + 4), ALIGN), (embed, dict(table=P + 1), ALIGN), (embed, dict(y=P + 1), ALIGN), (embed, dict(y_stride=7), STRIDE), (embed, dict(y=2 * P), STRIDE),
    (embed_grad, dict(type=3), TYPE), (embed_grad, dict(dtable_type=1), TYPE), (embed_grad, dict(token_bytes=1), TYPE), (embed_grad, dict(cols=0), DIMS),
    (embed_grad, dict(cols=1 << 25, dy_stride=1 << 25, dtable_stride=1 << 25, workspace_bytes=1 << 40), DIMS),
    (embed_grad, dict(vocab=0), DIMS), (embed_grad, dict(tokens=MOST), DIMS), (embed_grad, dict(token=None), NULL), (embed_grad, dict(dy=None), NULL),
    (embed_grad, dict(dtable=None), NULL), (embed_grad, dict(token=P + 2, token_bytes=4), ALIGN), (embed_grad, dict(dtable=P + 2, dtable_type=0), ALIGN),
    (embed_grad, dict(dtable_stride=7), STRIDE), (embed_grad, dict(dtable=2 * P), STRIDE), (embed_grad, dict(workspace=None), WORKSPACE),
    (embed_grad, dict(workspace=P + 8), WORKSPACE), (embed_grad, dict(workspace_bytes=15), WORKSPACE), (embed_grad, dict(tokens=0, dtable=None), NULL),
    (probs, dict(type=3), TYPE), (probs, dict(token_bytes=2), TYPE), (probs, dict(top_token_bytes=2), TYPE), (probs, dict(vocab=0, top=0), DIMS), (probs, dict(vocab=MOST), DIMS),
    (probs, dict(top=41), DIMS), (probs, dict(vocab=400, stride=400, top=129), DIMS), (probs, dict(scale=0.0), VALUE), (probs, dict(scale=-1.0), VALUE),
    (probs, dict(scale=math.inf), VALUE), (probs, dict(scale=math.nan), VALUE), (probs, dict(logits=None), NULL), (probs, dict(token=None), NULL),
    (probs, dict(top_logprob=None, top_token=None), NULL), (probs, dict(logprob=None, entropy=None, stats=None, top=0), NULL), (probs, dict(logits=P + 1), ALIGN),
    (probs, dict(token=P + 4), ALIGN), (probs, dict(logprob=P + 2), ALIGN), (probs, dict(entropy=P + 2), ALIGN), (probs, dict(stats=P + 4), ALIGN),
    (probs, dict(top_logprob=P + 2), ALIGN), (probs, dict(top_token=P + 4), ALIGN),
    (probs_grad, dict(type=3), TYPE), (probs_grad, dict(token_bytes=2), TYPE), (probs_grad, dict(vocab=0), DIMS), (probs_grad, dict(scale=0.0), VALUE),
    (probs_grad, dict(logits=None), NULL), (probs_grad, dict(token=None), NULL), (probs_grad, dict(stats=None), NULL), (probs_grad, dict(entropy=None), NULL),
    (probs_grad, dict(dlogprob=None, dentropy=None), NULL), (probs_grad, dict(dlogits=None), NULL), (probs_grad, dict(dstride=39), STRIDE),
    (probs_grad, dict(dlogits=P, dstride=48), STRIDE), (probs_grad, dict(stats=P + 4), ALIGN), (probs_grad, dict(dlogprob=P + 2), ALIGN), (probs_grad, dict(token=P + 4), ALIGN),
])
def test_the_c_calls_refuse(call, change, code):
    assert call(**change) == code


def test_no_rows_and_no_tokens_do_nothing():
    assert layer(rows=0, x=None, residual=None, total=None, y=None) == 0
    assert layer_grad(rows=0, dgamma=None, dbeta=None) == 0
    assert embed(tokens=0, token=None, table=None, y=None) == 0 and embed_grad(tokens=0, accumulate=1, dtable=None) == 0
    assert probs(rows=0, logits=None) == 0 and probs_grad(rows=0, logits=None) == 0


def python_calls(t, w, f32, pair, whole, best):
    norm, table, lp = ops.LayerNormalizeAddOp, ops.EmbedTokensOp, ops.TokenLogProbsOp
    return {
        "layer": lambda: norm.apply(1e-5, t, t, w, w, t, t, f32, f32),
        "layer grad": lambda: norm.adjoint(t, t, f32, f32, t, w, t, w, w),
        "embed": lambda: table.apply(whole, t, t),
        "embed grad": lambda: table.adjoint(whole, t, t),
        "probs": lambda: lp.apply(t, whole, f32, f32, pair, best, None),
        "probs grad": lambda: lp.adjoint(t, whole, pair, f32, t, f32, f32),
    }


NAMES = sorted(python_calls(*[None] * 6))


def tensors(device):
    e = lambda *s, dtype=torch.float32: torch.empty(s, device=device, dtype=dtype)      # noqa: E731
    return e(4, 8), e(8), e(4), e(4, 2), e(4, dtype=torch.int64), e(4, 3)


@pytest.mark.parametrize("name", NAMES)
def test_host_tensors_are_refused_before_anything_is_asked_of_cuda(name):
    with pytest.raises(ValueError, match="CUDA tensor"):
        python_calls(*tensors("cpu"))[name]()


@pytest.mark.parametrize("name", NAMES)
def test_what_is_no_tensor_is_refused(name):
    with pytest.raises((ValueError, TypeError)):
        python_calls(*["no"] * 6)[name]()


@pytest.mark.filterwarnings("ignore:Accessing the data pointer of FakeTensor")
def test_python_checks_of_sizes_types_and_devices():
    """Arrays that claim to be on a device: each of these is refused for what it is, before a stream or an address is needed."""
    norm, table, lp = ops.LayerNormalizeAddOp, ops.EmbedTokensOp, ops.TokenLogProbsOp
    with FakeTensorMode():
        def e(*s, dtype=torch.float32, device="cuda:0"):
            return torch.empty(s, device=device, dtype=dtype)
        i64, i32, f16 = torch.int64, torch.int32, torch.float16
        t, w, r, k = e(4, 8), e(8), e(4), e(4, dtype=i64)
        for text, call in [
            ("sizes", lambda: norm.apply(1e-5, t, e(4, 9))), ("type", lambda: norm.apply(1e-5, t, e(4, 8, dtype=f16))), ("packed", lambda: norm.apply(1e-5, e(8, 4).t(), t)),
            ("weight per column", lambda: norm.apply(1e-5, t, t, e(9))), ("weight per column", lambda: norm.apply(1e-5, t, t, w, e(7))),
            ("other weights", lambda: norm.apply(1e-5, t, t, w, e(8, dtype=f16))), ("without one", lambda: norm.apply(1e-5, t, e(4, 8), w, w, None, e(4, 8))),
            ("per row", lambda: norm.apply(1e-5, t, t, w, w, None, None, e(5))), ("float32, float16 or bfloat16", lambda: norm.apply(1e-5, e(4, 8, dtype=torch.float64), t)),
            ("mean: expected", lambda: norm.adjoint(t, t, None, r, t)), ("Accumulate", lambda: norm.adjoint(t, t, r, r, t, w, t, None, None, ops.WriteCap.Accumulate)),
            ("int32 or int64", lambda: table.apply(r, e(10, 8), t)), ("int32 or int64", lambda: table.apply(e(8, dtype=i64)[::2], e(10, 8), t)),
            ("vocab, cols", lambda: table.apply(k, e(2, 5, 8), t)), ("each token", lambda: table.apply(k, e(10, 8), e(5, 8))), ("each token", lambda: table.apply(k, e(10, 8), e(4, 9))),
            ("each token", lambda: table.apply(e(2, 2, dtype=i64), e(10, 8), t)), ("another type", lambda: table.apply(k, e(10, 8, dtype=f16), t)),
            ("dy's type or float32", lambda: table.adjoint(k, t, e(10, 8, dtype=f16))), ("one distance", lambda: table.adjoint(e(4, 3, dtype=i64), e(4, 6, 8)[:, :3], e(10, 8))),
            ("one token per row", lambda: lp.apply(t, e(5, dtype=i64), r)), ("log probabilities are asked for", lambda: lp.apply(t, None, r)),
            ("two values", lambda: lp.apply(t, k, r, None, r)), ("top", lambda: lp.apply(t, k, r, None, None, e(4, 2, dtype=f16))), ("top", lambda: lp.apply(t, k, r, None, None, None, e(4, 2))),
            ("sizes where both", lambda: lp.apply(t, k, r, None, None, e(4, 2), e(4, 3, dtype=i32))), ("more than 128", lambda: lp.apply(t, k, r, None, None, e(4, 9))),
            ("more than 128", lambda: lp.apply(e(4, 200), k, r, None, None, e(4, 129))), ("packed float32", lambda: lp.apply(t, k, r, None, None, e(2, 4).t())),
            ("stats: expected", lambda: lp.adjoint(t, k, None, r, t)), ("tokens of dlogprob", lambda: lp.adjoint(t, None, e(4, 2), r, t)),
            ("entropies", lambda: lp.adjoint(t, k, e(4, 2), r, t, None, r)), ("dlogprob, dentropy or both", lambda: lp.adjoint(t, k, e(4, 2), None, t)),
        ]:
            with pytest.raises(ValueError, match=text):
                call()
        wide = e(1, MOST, dtype=torch.bfloat16)
        for text, call in [("too many columns", lambda: norm.apply(1e-5, wide, wide)), ("too many columns", lambda: lp.apply(wide, None, None, e(1))),
                           ("too many rows or columns", lambda: table.apply(e(1, dtype=i64), wide, wide))]:
            with pytest.raises(ValueError, match=text):
                call()


@pytest.mark.skipif(torch.cuda.is_available(), reason="tensors that claim to be on a second device need a machine without a first")
@pytest.mark.filterwarnings("ignore:Accessing the data pointer of FakeTensor")
def test_tensors_of_two_devices_are_refused():
    with FakeTensorMode():
        x, k = torch.empty(4, 8, device="cuda:0"), torch.empty(4, device="cuda:1", dtype=torch.int64)
        for call in (lambda: ops.EmbedTokensOp.apply(k, x, x), lambda: ops.TokenLogProbsOp.apply(x, k, None, torch.empty(4, device="cuda:0"))):
            with pytest.raises(ValueError, match="another device"):
                call()


def test_layers_refuse():
    x = torch.zeros(4, 8)
    for layer_ in (ops.LayerNormAdd(8, device="cpu"), ops.TokenEmbedding(5, 8, device="cpu"), ops.TokenLogProbs()):
        with pytest.raises(RuntimeError):
            layer_.backward(x)
    with pytest.raises(ValueError, match="backward pass"):
        ops.LayerNormAdd(8, device="cpu").forward(x, out=x)
    with pytest.raises(ValueError, match="CUDA tensor"):      # (as far as a machine without a device goes)
        ops.LayerNormAdd(8, device="cpu").infer(x, out=x)
    plain = ops.LayerNormAdd(8, bias=False, device="cpu")
    assert plain.beta is None and plain.dbeta is None and ops.LayerNormAdd(8, affine=False, device="cpu").beta is None
