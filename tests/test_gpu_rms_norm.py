"""RMS norm with the residual's addition, its adjoint and its 8-bit form against the formulas in 64 bits.

Tolerances, u = 2^-24 (half a step of f32) and h = half a step of the tensors' type: a thread adds at most cols/32 of a row's terms
in turn and 16 more steps join them, so a sum of positive terms is off by (cols/32 + 16)*u of itself, r by half of that, and every other
step of the formulas by u.  A sum of rows is taken as if one after the other, rows*u of the sum of magnitudes at most."""
import pytest
import torch

from anode_b200 import ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
EPS = 1e-5
TYPES = [torch.float32, torch.float16, torch.bfloat16]
SHAPES = [(1, 1), (1, 7), (3, 32), (5, 33), (2, 127), (4, 128), (3, 129), (7, 255), (300, 96), (1, 1000), (9, 1024), (33, 2050), (2, 4096), (3, 5003),
          (1, 16384), (2, 16392), (2, 40000), (1, 70001)]


def half_step(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    return 2.0 ** -25 if t is torch.float16 else 1e-38       # half of f16's smallest step


def near(got, want, bound, what):
    got, bound = got.double(), bound.expand(want.shape) if isinstance(bound, torch.Tensor) else torch.full_like(want, bound)
    off = (got - want).abs() > bound
    off |= got.isnan() != want.isnan()
    if off.any():
        i = tuple(off.nonzero()[0].tolist())
        raise AssertionError("%s: %d of %d off; first at %s: got %r want %r bound %r" % (what, int(off.sum()), off.numel(), i, got[i].item(), want[i].item(),
                                                                                    bound[i].item()))


def make(rows, cols, dtype, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(1000 * seed + rows + 7 * cols)
    return (torch.randn(rows, cols, generator=g, device="cuda") * scale).to(dtype)


def weights(cols, dtype, seed=9):
    return (1 + 0.2 * make(1, cols, torch.float32, seed)[0]).to(dtype)


def row_bound(cols):
    return (cols / 64 + 16) * U


def check_forward(x, residual, gamma, y, total, inv_rms, what=""):
    t = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    if total is not None:
        assert torch.equal(total, t), what + "total"
        assert ((total.double() - (x.double() + residual.double())).abs() <= half_step(x.dtype) * 1.01 * t.double().abs() + tiny(x.dtype)).all()
    t = t.double()
    r = (t.square().mean(-1) + EPS).rsqrt()
    want = t * r.unsqueeze(-1) * (1 if gamma is None else gamma.double())
    d = row_bound(x.shape[-1])
    near(y, want, want.abs() * (half_step(x.dtype) * (1 + 2 ** -8) + d) + tiny(x.dtype), what + "y")
    if inv_rms is not None:
        near(inv_rms, r, r * d, what + "inv_rms")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows, cols", SHAPES)
def test_forward(rows, cols, dtype):
    x, res = make(rows, cols, dtype, 1, 2.0), make(rows, cols, dtype, 2)
    for residual, gamma in ((res, weights(cols, dtype)), (None, weights(cols, torch.float32)), (res, None)):
        y, inv = torch.full_like(x, 7.0), torch.zeros(rows, device="cuda")
        total = torch.full_like(x, 7.0) if residual is not None else None
        ops.RmsNormalizeAddOp.apply(EPS, x, y, gamma, residual, total, inv)
        check_forward(x, residual, gamma, y, total, inv)
        # the same without what need not be stored, and in place: the same bits
        z = torch.empty_like(x)
        ops.RmsNormalizeAddOp.apply(EPS, x, z, gamma, residual)
        assert torch.equal(z, y)
        if residual is not None:
            stream, out = residual.clone(), x.clone()
            ops.RmsNormalizeAddOp.apply(EPS, out, out, gamma, stream, stream)
            assert torch.equal(out, y) and torch.equal(stream, total)
            stream, out = x.clone(), residual.clone()
            ops.RmsNormalizeAddOp.apply(EPS, stream, out, gamma, out, stream)
            assert torch.equal(out, y) and torch.equal(stream, total)
        else:
            out = x.clone()
            ops.RmsNormalizeAddOp.apply(EPS, out, out, gamma)
            assert torch.equal(out, y)


def check_backward(dy, t, r, gamma, dt, dx, dgamma, what=""):
    cols, rows = dy.shape[-1], dy.shape[0]
    dtype = dx.dtype
    dy, t, r = dy.double(), t.double(), r.double().unsqueeze(-1)
    gm = torch.ones(cols, device="cuda", dtype=torch.float64) if gamma is None else gamma.double()
    g, xh = dy * gm, t * r
    c, m = (g * xh).mean(-1, keepdim=True), (g * xh).abs().mean(-1, keepdim=True)
    want = r * (g - xh * c)
    bound = r * (4 * U * g.abs() + xh.abs() * ((cols / 32 + 20) * U * m + 4 * U * c.abs()))
    if dt is not None:
        want, bound = want + dt.double(), bound + U * (want.abs() + dt.double().abs())
    near(dx, want, bound + half_step(dtype) * (1 + 2 ** -8) * want.abs() + tiny(dtype), what + "dx")
    if dgamma is not None:
        want, size = (dy * xh).sum(0), (dy * xh).abs().sum(0)
        near(dgamma, want, (rows + 16) * U * size + half_step(dgamma.dtype) * (1 + 2 ** -8) * want.abs() + tiny(dgamma.dtype), what + "dgamma")


def saved(rows, cols, dtype, seed=3):
    t = make(rows, cols, dtype, seed, 3.0)
    return make(rows, cols, dtype, seed + 1), t, (t.double().square().mean(-1) + EPS).rsqrt().float(), make(rows, cols, dtype, seed + 2)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows, cols", SHAPES + [(1000, 40), (2049, 130), (777, 1030), (150, 8192)])
def test_backward(rows, cols, dtype):
    dy, t, r, dt = saved(rows, cols, dtype)
    for gamma, extra in ((weights(cols, dtype), dt), (weights(cols, torch.float32), None), (None, dt)):
        dx, dg = torch.full_like(dy, 7.0), torch.full((cols,), 7.0, device="cuda", dtype=gamma.dtype if gamma is not None else torch.float32)
        ops.RmsNormalizeAddOp.adjoint(dy, t, r, dx, gamma, extra, dg)
        check_backward(dy, t, r, gamma, extra, dx, dg)
        # without dgamma, in dy's place, and the same call again: the same bits
        z = dy.clone()
        ops.RmsNormalizeAddOp.adjoint(z, t, r, z, gamma, extra)
        assert torch.equal(z, dx)
        z, dg2 = dy.clone(), torch.empty_like(dg)
        ops.RmsNormalizeAddOp.adjoint(z, t, r, z, gamma, extra, dg2)
        assert torch.equal(z, dx) and torch.equal(dg2, dg)
        if extra is not None:
            for how in ({"dtotal": None, "cap": ops.WriteCap.Accumulate}, {}):
                z = extra.clone()
                ops.RmsNormalizeAddOp.adjoint(dy, t, r, z, gamma, how.get("dtotal", z), dg2, how.get("cap", ops.WriteCap.Assign))
                assert torch.equal(z, dx) and torch.equal(dg2, dg)


def test_backward_is_the_gradient_of_the_forward_pass():
    """Against differences of the 64-bit forward formula along random directions."""
    rows, cols = 6, 200
    x, res, w = (make(rows, cols, torch.float32, s) for s in (11, 12, 13))
    gamma = weights(cols, torch.float32)
    layer = ops.RmsNormAdd(cols, EPS)
    layer.gamma.copy_(gamma)
    layer.forward(x, res)
    dx = layer.backward(w)

    def value(x, gamma):
        t = x + res.double()
        return (t * (t.square().mean(-1, keepdim=True) + EPS).rsqrt() * gamma * w.double()).sum()

    for seed in range(3):
        d, e, step = make(rows, cols, torch.float32, 20 + seed).double(), make(1, cols, torch.float32, 30 + seed)[0].double(), 1e-6
        for want, got in (((value(x.double() + step * d, gamma.double()) - value(x.double() - step * d, gamma.double())) / (2 * step), (dx.double() * d).sum()),
                          ((value(x.double(), gamma.double() + step * e) - value(x.double(), gamma.double() - step * e)) / (2 * step), (layer.dgamma.double() * e).sum())):
            # second differences are of the order of step^2, f64 rounding 1e-16*1e3/step, the gradients themselves 1e-6 of their size
            assert abs(float(want - got)) <= 1e-5 * float((dx.double().abs() * d.abs()).sum()) + 1e-6


def e4m3(v):
    _, e = torch.frexp(v)
    step = torch.ldexp(torch.ones_like(v), e.clamp(min=-5) - 4)
    return torch.round(v / step) * step


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows, cols", SHAPES)
def test_eight_bits(rows, cols, dtype):
    x, res = make(rows, cols, dtype, 5, 2.0), make(rows, cols, dtype, 6)
    x[:, ::17] *= 30
    groups = -(-cols // 128)
    for block, residual, gamma in ((128, res, weights(cols, dtype)), (0, None, weights(cols, torch.float32)), (128, None, None), (0, res, weights(cols, dtype))):
        q = torch.zeros(rows, cols, device="cuda", dtype=torch.float8_e4m3fn)
        shapes = [torch.zeros(rows, groups, device="cuda"), torch.zeros(groups, rows, device="cuda").t()] if block else [torch.zeros(rows, device="cuda")]
        total = torch.empty_like(x) if residual is not None else None
        for scale in shapes:
            ops.RmsNormalizeAddQuantOp.apply(EPS, x, q, scale, gamma, residual, total)
            t = x if residual is None else (x.float() + residual.float()).to(dtype)
            assert total is None or torch.equal(total, t)
            t = t.double()
            y = t * (t.square().mean(-1, keepdim=True) + EPS).rsqrt() * (1 if gamma is None else gamma.double())
            width = block or cols
            n = -(-cols // width)
            padded = torch.nn.functional.pad(y, (0, n * width - cols)).view(rows, n, width)
            want = padded.abs().amax(2).clamp(min=2.0 ** -96) / 448
            d = row_bound(cols) + 4 * U
            near(scale.reshape(rows, n), want, want * d, "scale")
            v = (padded / want.unsqueeze(2)).view(rows, n * width)[:, :cols]
            nearest = e4m3(v)
            assert (nearest.abs() <= 448).all()
            # no further than the nearest value, but for what v itself may be off by
            near(q, v, (nearest - v).abs() + 2 * (d + 4 * U) * v.abs(), "q")


def test_layer_eight_bits_and_infer_agree():
    layer = ops.RmsNormAdd(1024, dtype=torch.bfloat16)
    x, res = make(5, 1024, torch.bfloat16, 1).view(1, 5, 1024), make(5, 1024, torch.bfloat16, 2).view(1, 5, 1024)
    y, total = layer.infer(x, res)
    for block, shape in ((128, (1, 5, 8)), (None, (1, 5))):
        q, scale, t = layer.infer_quant(x, res, block)
        assert q.shape == x.shape and scale.shape == shape and torch.equal(t, total)
        back = q.float().view(1, 5, -1, 1024 // (8 if block else 1)) * scale.view(1, 5, -1, 1)
        # half a step of e4m3 (2^-4) of a value, or of the smallest step (2^-10 of the scale), and bf16's rounding of y
        assert ((back.view_as(y) - y.float()).abs() <= (2 ** -4 + 2 ** -7) * y.float().abs() + 2 ** -9 * scale.amax()).all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("cols", [64, 100, 1024, 33])
def test_strides_and_alignment(cols, dtype):
    """Slices of wider arrays that begin anywhere, broadcast inputs; what lies beside and behind the rows stays."""
    rows = 6
    wide = [make(rows + 2, 3 * cols + 5, dtype, s) for s in range(8)]
    gamma = weights(cols + 1, dtype)[1:]
    for first in (0, 1, 3, 8):
        def rows_of(i, at=first):
            return wide[i][:rows, at:at + cols]
        before = [w.clone() for w in wide]
        x, res, y, total = rows_of(0), rows_of(1, 2 * cols), rows_of(2), rows_of(3, 1)
        ops.RmsNormalizeAddOp.apply(EPS, x, y, gamma, res, total, None)
        check_forward(x, res, gamma, y, total, None, "first %d " % first)
        r = (total.double().square().mean(-1) + EPS).rsqrt().float()
        dy, dt, dx = rows_of(4), rows_of(5, 2), rows_of(6)
        dg = torch.zeros(cols + 1, device="cuda", dtype=dtype)
        ops.RmsNormalizeAddOp.adjoint(dy, total, r, dx, gamma, dt, dg[1:])
        check_backward(dy, total, r, gamma, dt, dx, dg[1:], "first %d " % first)
        assert dg[0] == 0
        for i, at in ((2, first), (3, 1), (6, first)):
            before[i][:rows, at:at + cols] = wide[i][:rows, at:at + cols]
        assert all(torch.equal(a, b) for a, b in zip(before, wide))
    one = make(1, cols, dtype, 40)
    x, y, total = make(rows, cols, dtype, 41).view(2, 3, cols), torch.empty(2, 3, cols, device="cuda", dtype=dtype), torch.empty(2, 3, cols, device="cuda", dtype=dtype)
    ops.RmsNormalizeAddOp.apply(EPS, x, y, None, one.expand(2, 3, cols), total)
    check_forward(x, one.expand(2, 3, cols), None, y, total, None, "broadcast ")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("cols", [96, 2048, 50000])
def test_rows_of_zeros_infinities_and_nan(cols, dtype):
    x = make(6, cols, dtype, 1)
    x[1] = 0
    x[2, 5] = float("inf")
    x[3, 7] = float("nan")
    x[4, 9] = float("-inf")
    y, inv = torch.empty_like(x), torch.empty(6, device="cuda")
    ops.RmsNormalizeAddOp.apply(EPS, x, y, None, None, None, inv)
    t = x.double()
    want = t * (t.square().mean(-1, keepdim=True) + EPS).rsqrt()
    assert torch.equal(y.isnan(), want.isnan())
    good = [0, 1, 5]
    check_forward(x[good], None, None, y[good], None, inv[good])
    assert torch.equal(y[1], torch.zeros_like(y[1])) and y[3].isnan().all() and y[2, 5].isnan() and (y[2, :5] == 0).all()
    for block in (0, 128):
        groups = -(-cols // 128)
        q = torch.empty(6, cols, device="cuda", dtype=torch.float8_e4m3fn)
        scale = torch.empty((6, groups) if block else (6,), device="cuda")
        ops.RmsNormalizeAddQuantOp.apply(EPS, x, q, scale)
        s = scale.view(6, -1)
        tiny_scale = torch.full_like(s[1], 2.0 ** -96 / 448)
        assert torch.equal(s[1], tiny_scale) and (q[1].float() == 0).all()
        assert s[3].isnan().all() and q[3].float().isnan().all()
        assert s[2, 0].isnan() and q[2, :min(128, cols)].float().isnan().all()
        if block and groups > 1:
            assert torch.equal(s[2, 1:], tiny_scale[1:]) and (q[2, 128:].float() == 0).all()


def test_values_that_exceed_the_type():
    x = torch.full((2, 64), 60000.0, device="cuda", dtype=torch.float16)
    y, total = torch.empty_like(x), torch.empty_like(x)
    ops.RmsNormalizeAddOp.apply(EPS, x, y, None, x, total)
    assert total.isinf().all() and y.isnan().all()        # inf * 0, as the formula says
    big = torch.full((1, 64), 1e10, device="cuda")
    out = torch.empty_like(big)
    ops.RmsNormalizeAddOp.apply(EPS, big, out)
    assert ((out - 1).abs() <= row_bound(64)).all()


def test_no_rows():
    for dtype in TYPES:
        x = torch.empty(0, 64, device="cuda", dtype=dtype)
        dg, r = torch.ones(64, device="cuda", dtype=dtype), torch.empty(0, device="cuda")
        layer = ops.RmsNormAdd(64, dtype=dtype)
        assert layer.forward(x, x)[0].shape == (0, 64)
        assert layer.infer_quant(x, x)[1].shape == (0, 1)
        ops.RmsNormalizeAddOp.adjoint(x, x, r, torch.empty_like(x), None, x, dg)
        assert (dg == 0).all()


def test_rows_beyond_32_bits():
    """Rows more than 2^31 elements apart, the last beyond 2^32 elements and 8 GiB."""
    cols, apart = 520, (1 << 31) + 64
    buffer = torch.empty(2 * apart + cols, device="cuda", dtype=torch.bfloat16)
    far = buffer.as_strided((3, cols), (apart, 1))
    x, res, gamma = make(3, cols, torch.bfloat16, 1), make(3, cols, torch.bfloat16, 2), weights(cols, torch.bfloat16)
    far.copy_(x)
    y = torch.empty_like(x)
    ops.RmsNormalizeAddOp.apply(EPS, far, y, gamma, res, far)
    check_forward(x, res, gamma, y, far.contiguous(), None)
    dy, t, r, dt = saved(3, cols, torch.bfloat16)
    far.copy_(dy)
    dg = torch.empty_like(gamma)
    ops.RmsNormalizeAddOp.adjoint(far, t, r, far, gamma, dt, dg)
    check_backward(dy, t, r, gamma, dt, far.contiguous(), dg)


def test_more_rows_than_a_launch_has_blocks():
    rows, cols = 70000, 24
    x, res = make(rows, cols, torch.float16, 1), make(rows, cols, torch.float16, 2)
    y, total, inv = torch.empty_like(x), torch.empty_like(x), torch.empty(rows, device="cuda")
    ops.RmsNormalizeAddOp.apply(EPS, x, y, None, res, total, inv)
    check_forward(x, res, None, y, total, inv)
    dx, dg = torch.empty_like(x), torch.empty(cols, device="cuda")
    ops.RmsNormalizeAddOp.adjoint(y, total, inv, dx, None, res, dg)
    check_backward(y, total, inv, None, res, dx, dg)


def test_streams_graphs_and_calls_at_once():
    rows, cols = 400, 1536
    layer = ops.RmsNormAdd(cols, EPS, dtype=torch.bfloat16)
    layer.gamma.copy_(weights(cols, torch.bfloat16))
    sets = [(make(rows, cols, torch.bfloat16, s), make(rows, cols, torch.bfloat16, s + 1), make(rows, cols, torch.bfloat16, s + 2)) for s in (1, 5)]

    def step(x, res, dy, stream=None, workspace=None):
        y, total, dx, q = (torch.empty_like(x) for _ in range(4))
        inv, dg = torch.empty(rows, device="cuda"), torch.empty_like(layer.gamma)
        ops.RmsNormalizeAddOp.apply(EPS, x, y, layer.gamma, res, total, inv, stream=stream)
        ops.RmsNormalizeAddOp.adjoint(dy, total, inv, dx, layer.gamma, y, dg, workspace=workspace, stream=stream)
        return y, total, inv, dx, dg
    want = [step(*s) for s in sets]
    torch.cuda.synchronize()
    # both at once, on streams of their own, given and current
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
    # captured, with a workspace of the caller's and without, and replayed on other inputs
    ws = [torch.empty(ops.rms_norm_workspace_bytes(rows, cols), device="cuda", dtype=torch.uint8), None]
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
