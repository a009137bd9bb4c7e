"""Rotary positions, with and without the norm of each head before them, against the formulas in 64 bits.

Tolerances, u = 2^-24: half a step of the type for the output's rounding; cosine and sine within 8u and the angle within 1e-7 (its
reduced form in f32) and 2^-50 of itself (products in f64, here and in the check); the norm as in the tests of rows."""
import pytest
import torch

from anode_b200 import ops
from tests.test_gpu_rms_norm import EPS, TYPES, U, half_step, near, tiny

pytestmark = pytest.mark.gpu


def normal(*shape, dtype=torch.float32, seed=0):
    g = torch.Generator(device="cuda").manual_seed(77 * seed + sum(shape))
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def table(positions, freq, amplitude, shape):
    """cos, sin and the angle's error for [..., 1, rot/2]"""
    p = positions.double()
    if len(shape) == 4 and p.dim() == 1:
        p = p.expand(shape[0], shape[1])
    a = p.unsqueeze(-1) * freq
    off = 8 * U + 1e-7 + 2.0 ** -50 * a.abs()
    return (amplitude * a.cos()).unsqueeze(-2), (amplitude * a.sin()).unsqueeze(-2), (amplitude * off).unsqueeze(-2)


def turn(x, size, cos, sin, off, rot, interleaved):
    """The turned head, and how far it may be off where x may be off by `size`."""
    u, v = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    out, far = x.clone(), size.clone()
    out[..., u], out[..., v] = x[..., u] * cos - x[..., v] * sin, x[..., u] * sin + x[..., v] * cos
    both = (x[..., u].abs() + x[..., v].abs()) * off
    far[..., u] = size[..., u] * cos.abs() + size[..., v] * sin.abs() + both
    far[..., v] = size[..., u] * sin.abs() + size[..., v] * cos.abs() + both
    return out, far


def check_forward(x, out, positions, freq, interleaved, amplitude, norm, gamma, what):
    rot, dim = 2 * len(freq), x.shape[-1]
    n = x.double()
    size = torch.zeros_like(n)
    if norm:
        n = n * (n.square().mean(-1, keepdim=True) + EPS).rsqrt() * (1 if gamma is None else gamma.double())
        size = (dim / 2 + 16) * U * n.abs()
    want, far = turn(n, size, *table(positions, freq, amplitude, x.shape), rot, interleaved)
    near(out, want, far * 1.01 + half_step(out.dtype) * (1 + 2 ** -8) * want.abs() + tiny(out.dtype), what)


def check_backward(dout, x, dx, dgamma, positions, freq, interleaved, amplitude, norm, gamma, what):
    rot, dim = 2 * len(freq), dout.shape[-1]
    cos, sin, off = table(positions, freq, amplitude, dout.shape)
    d = dout.double()
    dn, far = turn(d, torch.zeros_like(d), cos, -sin, off, rot, interleaved)
    if norm:
        x = x.double()
        r = (x.square().mean(-1, keepdim=True) + EPS).rsqrt()
        gm = torch.ones(dim, device="cuda", dtype=torch.float64) if gamma is None else gamma.double()
        g, xh, ng = dn * gm, x * r, far * gm.abs()
        c = (g * xh).mean(-1, keepdim=True)
        want = r * (g - xh * c)
        rel = (dim / 2 + 16) * U
        bound = r * (ng + xh.abs() * (ng * xh.abs()).mean(-1, keepdim=True) + 4 * rel * (g.abs() + xh.abs() * (g * xh).abs().mean(-1, keepdim=True)))
        if dgamma is not None:
            lead = tuple(range(dout.dim() - 1))
            total, size = (dn * xh).sum(lead), (dn * xh).abs().sum(lead)
            rows = dn.numel() // dim
            near(dgamma, total, (far * xh.abs()).sum(lead) + ((rows + 16) * U + 2 * rel) * size + half_step(dgamma.dtype) * (1 + 2 ** -8) * total.abs() + tiny(dgamma.dtype),
                 what + "dgamma")
    else:
        want, bound = dn, far
    near(dx, want, bound * 1.01 + half_step(dx.dtype) * (1 + 2 ** -8) * want.abs() + tiny(dx.dtype), what)


CASES = [  # tokens, heads, kv heads, dim, rot
    (1, 1, 1, 2, 2), (1, 32, 8, 128, 128), (3, 5, 1, 64, 64), (33, 7, 2, 80, 24), (17, 4, 4, 128, 64), (5, 3, 1, 7, 2), (9, 2, 1, 33, 32), (40, 8, 2, 256, 256),
    (11, 6, 3, 96, 96), (4, 2, 1, 96, 40), (3, 2, 2, 1000, 500), (2, 1, 1, 1024, 1024), (13, 64, 8, 16, 16), (257, 9, 3, 40, 20), (6, 3, 1, 130, 130), (7, 2, 1, 192, 100)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("tokens, heads, kv, dim, rot", CASES)
def test_both_directions(tokens, heads, kv, dim, rot, dtype):
    freq = ops.rotary_frequencies(rot, factor=4.0, context=512)
    for n, (interleaved, norm, weight, position_type, start, packed) in enumerate((
            (False, False, None, torch.int64, 0, False), (True, True, dtype, torch.int32, 1000000, True), (False, True, torch.float32, torch.int64, 2 ** 31 - 5, True),
            (True, False, None, torch.int64, -40, True), (False, True, None, torch.int32, 77, False))):
        amplitude = 1.0 if n % 2 else 1.2
        # (int64 positions beyond 2^31, too)
        positions = (start + 3 * torch.arange(tokens, device="cuda")).to(position_type)
        if packed:
            both, dboth = normal(tokens, heads + 2 * kv, dim, dtype=dtype, seed=n), normal(tokens, heads + 2 * kv, dim, dtype=dtype, seed=n + 9)
            (q, k), (dqo, dko) = ((b[:, :heads], b[:, heads:heads + kv]) for b in (both, dboth))
        else:
            (q, k), (dqo, dko) = ([normal(tokens, h, dim, dtype=dtype, seed=n + s + h) for h in (heads, kv)] for s in (1, 2))
        gq, gk = (1 + 0.2 * normal(dim, dtype=torch.float32, seed=s) for s in (3, 4)) if weight else (None, None)
        if weight:
            gq, gk = gq.to(weight), gk.to(weight)
        eps = EPS if norm else None
        what = "case %d " % n
        qo, ko = (torch.full(t.shape, 7.0, device="cuda", dtype=dtype) for t in (q, k))
        ops.RotaryPositionsOp.apply(positions, freq, q, k, qo, ko, interleaved, amplitude, eps, gq, gk)
        check_forward(q, qo, positions, freq, interleaved, amplitude, norm, gq, what + "q")
        check_forward(k, ko, positions, freq, interleaved, amplitude, norm, gk, what + "k")
        # queries alone, and both in place: the same bits
        alone = torch.empty_like(qo)
        ops.RotaryPositionsOp.apply(positions, freq, q, None, alone, None, interleaved, amplitude, eps, gq)
        assert torch.equal(alone, qo), what
        q2, k2 = q.clone(), k.clone()
        ops.RotaryPositionsOp.apply(positions, freq, q2, k2, q2, k2, interleaved, amplitude, eps, gq, gk)
        assert torch.equal(q2, qo) and torch.equal(k2, ko), what

        dq, dk = (torch.full(t.shape, 7.0, device="cuda", dtype=dtype) for t in (q, k))
        dgq, dgk = (torch.full((dim,), 7.0, device="cuda", dtype=weight or torch.float32) for _ in "qk") if norm else (None, None)
        more = (q, k, gq, gk, dgq, dgk) if norm else ()
        ops.RotaryPositionsOp.adjoint(positions, freq, dqo, dko, dq, dk, interleaved, amplitude, eps, *more)
        check_backward(dqo, q, dq, dgq, positions, freq, interleaved, amplitude, norm, gq, what + "dq ")
        check_backward(dko, k, dk, dgk, positions, freq, interleaved, amplitude, norm, gk, what + "dk ")
        dq2, dk2 = dqo.clone(), dko.clone()
        if norm:
            dgq2, dgk2 = torch.empty_like(dgq), torch.empty_like(dgk)
            more = (q, k, gq, gk, dgq2, dgk2)
        ops.RotaryPositionsOp.adjoint(positions, freq, dq2, dk2, dq2, dk2, interleaved, amplitude, eps, *more)
        assert torch.equal(dq2, dq) and torch.equal(dk2, dk), what
        assert not norm or (torch.equal(dgq2, dgq) and torch.equal(dgk2, dgk)), what
        if norm:
            ops.RotaryPositionsOp.adjoint(positions, freq, dqo, dko, dq2, dk2, interleaved, amplitude, eps, q, k, gq, gk)
            assert torch.equal(dq2, dq) and torch.equal(dk2, dk), what


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_batches_strides_and_what_lies_beside(dtype):
    """[batch, seq, heads, dim] at the strides of [batch, heads, seq, dim], of a packed projection, and beginning anywhere; positions per
    batch, per sequence, and broadcast; what lies beside the heads stays."""
    b, s, h, kv, dim, rot = 3, 5, 4, 2, 64, 48
    freq = ops.rotary_frequencies(rot)
    gq, gk = ((1 + 0.2 * normal(dim, seed=i)).to(dtype) for i in (1, 2))
    each = torch.randint(0, 5000, (b, s), device="cuda")
    for first in (0, 1, 4, 8):
        for positions in (each, each[0], each[:1].expand(b, s), each.int()):
            qb, kb = normal(b, h, s + 1, dim + 16, dtype=dtype, seed=3), normal(b, s, kv, dim + 16, dtype=dtype, seed=4)
            q, k = qb[:, :, :s, first:first + dim].transpose(1, 2), kb[..., first:first + dim]
            ob = normal(b, s, h + kv, dim + 16, dtype=dtype, seed=5)
            qo, ko = ob[:, :, :h, first:first + dim], ob[:, :, h:, 3:3 + dim]
            before = ob.clone()
            for norm in (False, True):
                eps, w = (EPS, (gq, gk)) if norm else (None, (None, None))
                ops.RotaryPositionsOp.apply(positions, freq, q, k, qo, ko, False, 1.0, eps, *w)
                check_forward(q, qo, positions, freq, False, 1.0, norm, w[0], "q")
                check_forward(k, ko, positions, freq, False, 1.0, norm, w[1], "k")
                before[:, :, :h, first:first + dim], before[:, :, h:, 3:3 + dim] = qo, ko
                assert torch.equal(before, ob)
                dqb = normal(b, h, s, dim, dtype=dtype, seed=6)
                dq, dk = dqb.transpose(1, 2), torch.empty(b, s, kv, dim, device="cuda", dtype=dtype)
                dg = [torch.empty_like(g) for g in (gq, gk)] if norm else []
                more = (q, k, gq, gk, *dg) if norm else ()
                douts = qo.clone(), ko.clone()
                ops.RotaryPositionsOp.adjoint(positions, freq, qo, ko, dq, dk, False, 1.0, eps, *more)
                check_backward(douts[0], q, dq, dg[0] if norm else None, positions, freq, False, 1.0, norm, w[0], "dq")
                check_backward(douts[1], k, dk, dg[1] if norm else None, positions, freq, False, 1.0, norm, w[1], "dk")


def test_turns_keep_lengths_and_relative_positions():
    """The product of two turned vectors depends on the distance of their positions alone: 100 and 4 against 1000100 and 1000004."""
    freq = ops.rotary_frequencies(128)
    q, k = normal(1, 1, 128, seed=1), normal(1, 1, 128, seed=2)
    products = []
    for at in (0, 1000000):
        turned = []
        for x, p in ((q, 100), (k, 4)):
            y = torch.empty_like(x)
            ops.RotaryPositionsOp.apply(torch.tensor([at + p], device="cuda"), freq, x, None, y, None)
            turned.append(y.double())
        # each element within 1e-7 + 10u of its pair's size
        assert abs(float(turned[0].norm() - q.double().norm())) < 1e-6 * float(q.norm())
        products.append(float((turned[0] * turned[1]).sum()))
    assert abs(products[0] - products[1]) < 4e-6 * float(q.norm() * k.norm())


def test_heads_of_zeros_and_nan():
    dim, freq = 64, ops.rotary_frequencies(64)
    q = normal(3, 2, dim, dtype=torch.bfloat16)
    q[0, 0], q[1, 1, 3] = 0, float("nan")
    out = torch.empty_like(q)
    ops.RotaryPositionsOp.apply(torch.arange(3, device="cuda"), freq, q, None, out, None, epsilon=EPS)
    assert (out[0, 0] == 0).all() and out[1, 1].isnan().all() and int(out.isnan().sum()) == dim
    ops.RotaryPositionsOp.apply(torch.arange(3, device="cuda"), freq, q, None, out, None)
    assert int(out.isnan().sum()) == 2 and out[1, 1, 3].isnan() and out[1, 1, 35].isnan()


def test_no_tokens():
    freq = ops.rotary_frequencies(32)
    for shape in ((0, 4, 32), (2, 0, 4, 32), (0, 3, 4, 32)):
        q = torch.empty(shape, device="cuda")
        positions = torch.zeros(shape[:-2], device="cuda", dtype=torch.int64)
        dg = torch.ones(32, device="cuda")
        ops.RotaryPositionsOp.apply(positions, freq, q, q, torch.empty_like(q), torch.empty_like(q))
        ops.RotaryPositionsOp.adjoint(positions, freq, q, q, torch.empty_like(q), torch.empty_like(q), epsilon=EPS, q=q, k=q, dgamma_q=dg)
        assert (dg == 0).all()


def test_heads_beyond_32_bits():
    apart = (1 << 31) + 64
    buffer = torch.empty(2 * apart + 2 * 64, device="cuda", dtype=torch.bfloat16)
    far = buffer.as_strided((3, 2, 64), (apart, 64, 1))
    q, freq, positions = normal(3, 2, 64, dtype=torch.bfloat16), ops.rotary_frequencies(64), torch.arange(3, device="cuda")
    far.copy_(q)
    ops.RotaryPositionsOp.apply(positions, freq, far, None, far, None, epsilon=EPS)
    check_forward(q, far.contiguous(), positions, freq, False, 1.0, True, None, "far")


def test_gradient_against_differences():
    layer = ops.RotaryPositions(40, 24, interleaved=True, amplitude=1.1, norm=True, epsilon=EPS)
    q, k, wq, wk = normal(5, 3, 40, seed=1), normal(5, 2, 40, seed=2), normal(5, 3, 40, seed=3), normal(5, 2, 40, seed=4)
    layer.gamma_q.copy_(1 + 0.2 * normal(40, seed=5))
    positions = torch.arange(5, device="cuda") * 11
    layer.forward(q, k, positions)
    dq, dk = layer.backward(wq, wk)

    def value(x, gamma, w):
        n = x * (x.square().mean(-1, keepdim=True) + EPS).rsqrt() * gamma
        return (turn(n, n, *table(positions, layer.freq, 1.1, x.shape), 24, True)[0] * w.double()).sum()

    for x, gamma, w, dx, dg in ((q, layer.gamma_q, wq, dq, layer.dgamma_q), (k, layer.gamma_k, wk, dk, layer.dgamma_k)):
        d, e, step = normal(*x.shape, seed=8).double(), normal(40, seed=9).double(), 1e-6
        x, gamma = x.double(), gamma.double()
        for want, got in (((value(x + step * d, gamma, w) - value(x - step * d, gamma, w)) / (2 * step), (dx.double() * d).sum()),
                          ((value(x, gamma + step * e, w) - value(x, gamma - step * e, w)) / (2 * step), (dg.double() * e).sum())):
            assert abs(float(want - got)) <= 1e-5 * float((dx.double().abs() * d.abs()).sum()) + 1e-6


def test_streams_graphs_and_calls_at_once():
    tokens, heads, kv, dim = 300, 8, 2, 128
    layer = ops.RotaryPositions(dim, norm=True, dtype=torch.bfloat16)
    positions = torch.arange(tokens, device="cuda")
    sets = [[normal(tokens, h, dim, dtype=torch.bfloat16, seed=s + i) for i, h in enumerate((heads, kv, heads, kv))] for s in (1, 20)]

    def step(q, k, dqo, dko, stream=None, workspace=None):
        out = [torch.empty_like(t) for t in (q, k, q, k)]
        dg = [torch.empty_like(layer.gamma_q) for _ in "qk"]
        ops.RotaryPositionsOp.apply(positions, layer.freq, q, k, *out[:2], False, 1.0, EPS, layer.gamma_q, layer.gamma_k, stream=stream)
        ops.RotaryPositionsOp.adjoint(positions, layer.freq, dqo, dko, *out[2:], False, 1.0, EPS, q, k, layer.gamma_q, layer.gamma_k, *dg,
                                      workspace=workspace, stream=stream)
        return out + dg
    want = [step(*s) for s in sets]
    torch.cuda.synchronize()
    other, third = torch.cuda.Stream(), torch.cuda.Stream()
    outs = []
    for _ in range(4):
        other.wait_stream(torch.cuda.current_stream())
        third.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(third):
            b = step(*sets[1])
        outs.append((step(*sets[0], stream=other), b))
    torch.cuda.synchronize()
    for a, b in outs:
        assert all(torch.equal(p, q) for p, q in zip(a, want[0])) and all(torch.equal(p, q) for p, q in zip(b, want[1]))
    ws = [torch.empty(ops.rotary_workspace_bytes(1, tokens, heads, kv, dim), device="cuda", dtype=torch.uint8), None]
    inputs = [[t.clone() for t in sets[0]] for _ in ws]
    graphs, results = [], []
    for w, inp in zip(ws, inputs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            results.append(step(*inp, workspace=w))
        graphs.append(g)
    for s, inp in zip((1, 0), inputs):
        for t, new in zip(inp, sets[s]):
            t.copy_(new)
    for _ in range(2):
        for g in graphs:
            g.replay()
    torch.cuda.synchronize()
    for s, got in zip((1, 0), results):
        assert all(torch.equal(p, q) for p, q in zip(got, want[s]))
