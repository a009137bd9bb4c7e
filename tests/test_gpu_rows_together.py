"""The row-wise operators as a transformer's layer has them: norm of the residual stream, projection, norm and rotary positions of the heads,
and back; then the serving form of the first step.  The projections are torch's."""
import pytest
import torch

from anode_b200 import ops

pytestmark = pytest.mark.gpu


def turn(x, positions, freq):
    a = positions.double()[:, None, None] * freq
    u, v = x.chunk(2, -1)
    return torch.cat((u * a.cos() - v * a.sin(), u * a.sin() + v * a.cos()), -1)


def test_a_layers_forward_and_backward_pass():
    """float32 against autograd in float64.  Products over 256 and 384 terms in f32 (sums of terms of size one, off by sqrt(n)*2^-24
    each, 1e-6) and the operators' own 1e-6 give gradients within 1e-4 of the largest; a wrong formula is off by its size."""
    tokens, cols, heads, kv, dim = 37, 256, 4, 2, 48
    g = torch.Generator(device="cuda").manual_seed(3)

    def normal(*s, scale=1.0):
        return scale * torch.randn(s, generator=g, device="cuda")
    x, res, weight = normal(tokens, cols), normal(tokens, cols), normal((heads + 2 * kv) * dim, cols, scale=cols ** -0.5)
    dq_out, dk_out, dv, dt = normal(tokens, heads, dim), normal(tokens, kv, dim), normal(tokens, kv, dim), normal(tokens, cols)
    norm, rotary = ops.RmsNormAdd(cols), ops.RotaryPositions(dim, norm=True, factor=2.0, context=64)
    for w in (norm.gamma, rotary.gamma_q, rotary.gamma_k):
        w.copy_(1 + 0.2 * normal(len(w)))
    positions = torch.arange(tokens, device="cuda") + 1000

    y, total = norm.forward(x, res)
    packed = (y @ weight.t()).view(tokens, heads + 2 * kv, dim)
    q, k, v = packed.split((heads, kv, kv), 1)
    q_out, k_out = rotary.forward(q, k, positions)
    dpacked = torch.empty_like(packed)
    rotary.backward(dq_out, dk_out, dpacked[:, :heads], dpacked[:, heads:heads + kv])
    dpacked[:, heads + kv:] = dv
    dpacked = dpacked.view(tokens, -1)
    dweight = dpacked.t() @ y
    dx = norm.backward(dpacked @ weight, dt)

    leaves = [t.double().requires_grad_() for t in (x, res, weight, norm.gamma, rotary.gamma_q, rotary.gamma_k)]
    X, R, W, G, GQ, GK = leaves

    def rms(t, gamma, eps):
        return t * (t.square().mean(-1, keepdim=True) + eps).rsqrt() * gamma
    T = X + R
    Q, K, V = (rms(T, G, norm.epsilon) @ W.t()).view(tokens, heads + 2 * kv, dim).split((heads, kv, kv), 1)
    Q, K = (turn(rms(t, w, rotary.epsilon), positions, rotary.freq) for t, w in ((Q, GQ), (K, GK)))
    torch.autograd.backward([Q, K, V, T], [t.double() for t in (dq_out, dk_out, dv, dt)])
    for what, got, want in (("total", total, T), ("q", q_out, Q), ("k", k_out, K), ("v", v, V), ("dx", dx, X.grad), ("dresidual", dx, R.grad), ("dweight", dweight, W.grad),
                            ("dgamma", norm.dgamma, G.grad), ("dgamma_q", rotary.dgamma_q, GQ.grad), ("dgamma_k", rotary.dgamma_k, GK.grad)):
        off = (got.double() - want).abs().max() / want.abs().max()
        assert off < 1e-4, (what, float(off))


def test_serving_a_token_in_eight_bits():
    """Each token of a prompt on its own gives what the whole prompt gives, bit for bit, and the 8-bit product is as near the exact one as
    half a step of e4m3 allows."""
    tokens, cols, out = 9, 1024, 64
    g = torch.Generator(device="cuda").manual_seed(4)
    x, res = (torch.randn(tokens, cols, generator=g, device="cuda").bfloat16() for _ in "xr")
    weight = torch.randn(out, cols, generator=g, device="cuda") * cols ** -0.5
    norm, rotary = ops.RmsNormAdd(cols, dtype=torch.bfloat16), ops.RotaryPositions(16, dtype=torch.bfloat16)
    positions = torch.arange(tokens, device="cuda") + 50000
    q8, scale, total = norm.infer_quant(x, res)
    y, _ = norm.infer(x, res)
    for t in range(tokens):
        one = norm.infer_quant(x[t:t + 1], res[t:t + 1])
        assert torch.equal(one[0].view(torch.uint8)[0], q8.view(torch.uint8)[t]) and torch.equal(one[1][0], scale[t]) and torch.equal(one[2][0], total[t])
        assert torch.equal(norm.infer(x[t], res[t])[0], y[t])
    back = (q8.float().view(tokens, -1, 128) * scale[:, :, None]).view(tokens, cols)
    exact = total.double() * (total.double().square().mean(-1, keepdim=True) + norm.epsilon).rsqrt()
    product, want = back.double() @ weight.double().t(), exact @ weight.double().t()
    # half a step of each value, or half the smallest step of its group
    limit = (2.0 ** -4 * exact.abs() + 2.0 ** -10 * scale.double().repeat_interleave(128, 1)) @ weight.double().abs().t()
    assert ((product - want).abs() <= limit * 1.001).all()
    heads = product.to(torch.bfloat16).view(tokens, 4, 16)
    whole, _ = rotary.infer(heads, None, positions)
    for t in range(tokens):
        one, _ = rotary.infer(heads[t:t + 1], None, positions[t:t + 1])
        assert torch.equal(one[0], whole[t])
