"""Layer norm with the residual's addition and its adjoint against the formulas in 64 bits.

Tolerances, u = 2^-24 (half a step of f32) and h = half a step of the tensors' type: a thread adds at most cols/32 of a row's terms in turn and
16 more steps join them, so a sum is off by D = (cols/32 + 16)*u of the sum of magnitudes.  The mean is off by a = D*mean|t|; the mean square of what
is left by 2u and D of itself and by a^2, since values less their mean add up to nothing; r by half of that and 2u; every other step of the
formulas by u of what it yields."""
import pytest
import torch

from anode_b200 import ops
from tests.test_gpu_rms_norm import EPS, SHAPES, TYPES, U, half_step, make, near, tiny, weights

pytestmark = pytest.mark.gpu


def d_of(cols):
    return (cols / 32 + 16) * U


def check_forward(x, residual, gamma, beta, y, total, mean, inv_std, what=""):
    t = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    if total is not None:
        assert torch.equal(total, t), what + "total"
    t, dtype, d = t.double(), x.dtype, d_of(x.shape[-1])
    mu = t.mean(-1, keepdim=True)
    a = d * t.abs().mean(-1, keepdim=True) + U * mu.abs()
    var = (t - mu).square().mean(-1, keepdim=True)
    r = (var + EPS).rsqrt()
    off_r = r * (d / 2 + 4 * U + a * a / (var + EPS))
    if mean is not None:
        near(mean, mu.squeeze(-1), a.squeeze(-1) + 1e-38, what + "mean")
        near(inv_std, r.squeeze(-1), off_r.squeeze(-1), what + "inv_std")
    g = 1 if gamma is None else gamma.double()
    b = 0 if beta is None else beta.double()
    xh = (t - mu) * r
    want = xh * g + b
    size = (xh * g).abs()
    bound = abs(g) * (a * r + (t - mu).abs() * off_r) + 3 * U * (size + want.abs()) + half_step(dtype) * (1 + 2 ** -8) * want.abs() + tiny(dtype)
    near(y, want, bound, what + "y")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows, cols", SHAPES)
def test_forward(rows, cols, dtype):
    x, res = make(rows, cols, dtype, 1, 2.0), make(rows, cols, dtype, 2) + 3
    for residual, gamma, beta in ((res, weights(cols, dtype), weights(cols, dtype, 8)), (None, weights(cols, torch.float32), None), (res, None, weights(cols, dtype)),
                                  (None, None, None)):
        y, mean, inv = torch.full_like(x, 7.0), torch.zeros(rows, device="cuda"), torch.zeros(rows, device="cuda")
        total = torch.full_like(x, 7.0) if residual is not None else None
        ops.LayerNormalizeAddOp.apply(EPS, x, y, gamma, beta, residual, total, mean, inv)
        check_forward(x, residual, gamma, beta, y, total, mean, inv)
        # the same without what need not be stored, and in place: the same bits
        z = torch.empty_like(x)
        ops.LayerNormalizeAddOp.apply(EPS, x, z, gamma, beta, residual)
        assert torch.equal(z, y)
        if residual is not None:
            stream, out = residual.clone(), x.clone()
            ops.LayerNormalizeAddOp.apply(EPS, out, out, gamma, beta, stream, stream)
            assert torch.equal(out, y) and torch.equal(stream, total)
            stream, out = x.clone(), residual.clone()
            ops.LayerNormalizeAddOp.apply(EPS, stream, out, gamma, beta, out, stream)
            assert torch.equal(out, y) and torch.equal(stream, total)
        else:
            out = x.clone()
            ops.LayerNormalizeAddOp.apply(EPS, out, out, gamma, beta)
            assert torch.equal(out, y)


def check_backward(dy, t, mean, r, gamma, dt, dx, dgamma, dbeta, what=""):
    rows, cols = dy.shape
    dtype, d = dx.dtype, d_of(cols)
    dy, mu, r = dy.double(), mean.double().unsqueeze(-1), r.double().unsqueeze(-1)
    gm = torch.ones(cols, device="cuda", dtype=torch.float64) if gamma is None else gamma.double()
    g, xh = dy * gm, (t.double() - mu) * r
    s, c = g.mean(-1, keepdim=True), (g * xh).mean(-1, keepdim=True)
    off_s, off_c = (d + 3 * U) * g.abs().mean(-1, keepdim=True), (d + 8 * U) * (g * xh).abs().mean(-1, keepdim=True)
    want = r * (g - s - xh * c)
    bound = r * (off_s + xh.abs() * off_c + 6 * U * (g.abs() + s.abs() + (xh * c).abs())) + 4 * U * want.abs()
    if dt is not None:
        want, bound = want + dt.double(), bound + U * (want.abs() + dt.double().abs())
    near(dx, want, bound + half_step(dtype) * (1 + 2 ** -8) * want.abs() + tiny(dtype), what + "dx")
    for got, terms, name in ((dgamma, dy * xh, "dgamma"), (dbeta, dy, "dbeta")):
        if got is not None:
            want, size = terms.sum(0), terms.abs().sum(0)
            near(got, want, (rows + 16) * U * size + half_step(got.dtype) * (1 + 2 ** -8) * want.abs() + tiny(got.dtype), what + name)


def saved(rows, cols, dtype, seed=3):
    t = make(rows, cols, dtype, seed, 3.0) + 1
    var, mean = torch.var_mean(t.double(), -1, correction=0)
    return make(rows, cols, dtype, seed + 1), t, mean.float(), (var + EPS).rsqrt().float(), make(rows, cols, dtype, seed + 2)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows, cols", SHAPES + [(1000, 40), (2049, 130), (777, 1030), (150, 8192)])
def test_backward(rows, cols, dtype):
    dy, t, mean, r, dt = saved(rows, cols, dtype)
    adjoint = ops.LayerNormalizeAddOp.adjoint
    for gamma, extra in ((weights(cols, dtype), dt), (weights(cols, torch.float32), None), (None, dt)):
        dx = torch.full_like(dy, 7.0)
        dg, db = (torch.full((cols,), 7.0, device="cuda", dtype=gamma.dtype if gamma is not None else torch.float32) for _ in range(2))
        adjoint(dy, t, mean, r, dx, gamma, extra, dg, db)
        check_backward(dy, t, mean, r, gamma, extra, dx, dg, db)
        # without the weights' gradients or with one of them, in dy's place, and the same call again: the same bits
        for which in ((False, False), (True, True), (True, False), (False, True)):
            z, again = dy.clone(), [torch.empty_like(dg) if w else None for w in which]
            adjoint(z, t, mean, r, z, gamma, extra, *again)
            assert torch.equal(z, dx) and all(a is None or torch.equal(a, b) for a, b in zip(again, (dg, db)))
        if gamma is not None:          # dgamma in gamma's place
            w, other = gamma.clone(), torch.empty_like(db)
            adjoint(dy, t, mean, r, z, w, extra, w, other)
            assert torch.equal(z, dx) and torch.equal(w, dg) and torch.equal(other, db)
        if extra is not None:
            for how in ({"dtotal": None, "cap": ops.WriteCap.Accumulate}, {}):
                z = extra.clone()
                adjoint(dy, t, mean, r, z, gamma, how.get("dtotal", z), dg, db, how.get("cap", ops.WriteCap.Assign))
                assert torch.equal(z, dx)


# rows, cols: by the slots of 16 bytes of a row, whole and ragged, several rows to each team of threads
MANY = [(40000, 32), (25000, 33), (20000, 200), (12000, 257), (5000, 640), (5001, 643), (2500, 1536), (2500, 1535), (1300, 5000), (1301, 5003), (700, 9001), (400, 10240), (500, 16384),
        (300, 16380), (301, 16381)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows, cols", MANY)
def test_many_rows(rows, cols, dtype):
    x, res, gamma, beta = make(rows, cols, dtype, 1), make(rows, cols, dtype, 2), weights(cols, dtype), weights(cols, dtype, 8)
    y, total, mean, inv = torch.empty_like(x), torch.empty_like(x), torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    ops.LayerNormalizeAddOp.apply(EPS, x, y, gamma, beta, res, total, mean, inv)
    check_forward(x, res, gamma, beta, y, total, mean, inv)
    ops.LayerNormalizeAddOp.apply(EPS, x, y, gamma, beta)
    check_forward(x, None, gamma, beta, y, None, None, None)
    dy, t, mu, r, dt = saved(rows, cols, dtype)
    dx, dg, db = torch.empty_like(dy), torch.empty_like(gamma), torch.empty_like(gamma)
    for extra in (dt, None):
        ops.LayerNormalizeAddOp.adjoint(dy, t, mu, r, dx, gamma, extra, dg, db)
        check_backward(dy, t, mu, r, gamma, extra, dx, dg, db)
    z, again = dy.clone(), [torch.empty_like(dg), torch.empty_like(db)]
    ops.LayerNormalizeAddOp.adjoint(z, t, mu, r, z, gamma, None, *again)
    assert torch.equal(z, dx) and torch.equal(again[0], dg) and torch.equal(again[1], db)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows, cols", [(1, 64), (700, 1536), (701, 515), (90, 16384), (40, 20000)])
def test_no_row_is_missing_from_the_weights_gradients(rows, cols, dtype):
    """Whole numbers whose sums are exact: means of 0, 1/std of 1."""
    g = torch.Generator(device="cuda").manual_seed(rows)
    dy, t = (torch.randint(-3, 4, (rows, cols), generator=g, device="cuda").to(dtype) for _ in range(2))
    mean, r = torch.zeros(rows, device="cuda"), torch.ones(rows, device="cuda")
    dx, dg, db = torch.empty_like(dy), torch.empty(cols, device="cuda"), torch.empty(cols, device="cuda")
    ops.LayerNormalizeAddOp.adjoint(dy, t, mean, r, dx, None, None, dg, db)
    assert torch.equal(dg, (dy.float() * t.float()).sum(0)) and torch.equal(db, dy.float().sum(0))


def test_backward_is_the_gradient_of_the_forward_pass():
    """Against differences of the 64-bit forward formula along random directions."""
    rows, cols = 6, 200
    x, res, w = (make(rows, cols, torch.float32, s) for s in (11, 12, 13))
    layer = ops.LayerNormAdd(cols, EPS)
    layer.gamma.copy_(weights(cols, torch.float32))
    layer.beta.copy_(weights(cols, torch.float32, 8))
    layer.forward(x, res)
    dx = layer.backward(w)

    def value(x, gamma, beta):
        t = x + res.double()
        c = t - t.mean(-1, keepdim=True)
        return ((c * (c.square().mean(-1, keepdim=True) + EPS).rsqrt() * gamma + beta) * w.double()).sum()

    at = [x.double(), layer.gamma.double(), layer.beta.double()]
    for seed in range(3):
        for i, grad in enumerate((dx, layer.dgamma, layer.dbeta)):
            d, step = make(*((rows, cols) if i == 0 else (1, cols)), torch.float32, 20 + seed).double(), 1e-6
            d = d if i == 0 else d[0]
            ends = [value(*[a + (sign * step * d if k == i else 0) for k, a in enumerate(at)]) for sign in (1, -1)]
            # second differences are of the order of step^2, f64 rounding 1e-16*1e3/step, the gradients themselves 1e-6 of their size
            assert abs(float((ends[0] - ends[1]) / (2 * step) - (grad.double() * d).sum())) <= 1e-5 * float((grad.double().abs() * d.abs()).sum()) + 1e-6


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("cols", [64, 100, 1024, 33])
def test_strides_and_alignment(cols, dtype):
    """Slices of wider arrays that begin anywhere, broadcast inputs; what lies beside and behind the rows stays."""
    rows = 6
    wide = [make(rows + 2, 3 * cols + 5, dtype, s) for s in range(8)]
    gamma, beta = weights(cols + 1, dtype)[1:], weights(cols + 3, dtype, 8)[3:]
    for first in (0, 1, 3, 8):
        def rows_of(i, at=first):
            return wide[i][:rows, at:at + cols]
        before = [w.clone() for w in wide]
        x, res, y, total = rows_of(0), rows_of(1, 2 * cols), rows_of(2), rows_of(3, 1)
        ops.LayerNormalizeAddOp.apply(EPS, x, y, gamma, beta, res, total)
        check_forward(x, res, gamma, beta, y, total, None, None, "first %d " % first)
        var, mean = torch.var_mean(total.double(), -1, correction=0)
        mean, r = mean.float(), (var + EPS).rsqrt().float()
        dy, dt, dx = rows_of(4), rows_of(5, 2), rows_of(6)
        dg, db = (torch.zeros(cols + 1, device="cuda", dtype=dtype) for _ in range(2))
        ops.LayerNormalizeAddOp.adjoint(dy, total, mean, r, dx, gamma, dt, dg[1:], db[1:])
        check_backward(dy, total, mean, r, gamma, dt, dx, dg[1:], db[1:], "first %d " % first)
        assert dg[0] == 0 and db[0] == 0
        for i, at in ((2, first), (3, 1), (6, first)):
            before[i][:rows, at:at + cols] = wide[i][:rows, at:at + cols]
        assert all(torch.equal(a, b) for a, b in zip(before, wide))
    one = make(1, cols, dtype, 40)
    x, y, total = make(rows, cols, dtype, 41).view(2, 3, cols), torch.empty(2, 3, cols, device="cuda", dtype=dtype), torch.empty(2, 3, cols, device="cuda", dtype=dtype)
    ops.LayerNormalizeAddOp.apply(EPS, x, y, None, None, one.expand(2, 3, cols), total)
    check_forward(x, one.expand(2, 3, cols), None, None, y, total, None, None, "broadcast ")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("cols, strides", [(1000, (1001, 1009, 1017, 1025)), (1000, (1000, 1008, 1016, 1040)), (1000, (1000, 1001, 1002, 1003)), (77, (80, 88, 96, 104))])
def test_arrays_of_different_strides(cols, strides, dtype):
    """In step with each other (they differ by whole 16 bytes), and not."""
    rows = 3000
    wide = [make(rows, s, dtype, i) for i, s in enumerate(strides)]
    x, res, y, total = (w[:, :cols] for w in wide)
    gamma, beta = weights(cols, dtype), weights(cols, dtype, 8)
    beside = [w[:, cols:].clone() for w in wide]
    mean, r = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    ops.LayerNormalizeAddOp.apply(EPS, x, y, gamma, beta, res, total, mean, r)
    check_forward(x, res, gamma, beta, y, total, mean, r)
    dy, t, dt, dx = x, total, res, y
    dg, db = torch.empty_like(gamma), torch.empty_like(gamma)
    ops.LayerNormalizeAddOp.adjoint(dy, t, mean, r, dx, gamma, dt, dg, db)
    check_backward(dy, t, mean, r, gamma, dt, dx, dg, db)
    assert all(torch.equal(a, w[:, cols:]) for a, w in zip(beside, wide))


@pytest.mark.parametrize("cols", [96, 2048, 50000])
def test_rows_far_from_zero_keep_their_spread(cols):
    """Values of 1000 with a spread of one: their squares' mean would have no digit of the spread left in f32 beyond 2^-24*1e6."""
    x = make(5, cols, torch.float32, 1) + 1000
    y, mean, inv = torch.empty_like(x), torch.empty(5, device="cuda"), torch.empty(5, device="cuda")
    ops.LayerNormalizeAddOp.apply(EPS, x, y, None, None, None, None, mean, inv)
    check_forward(x, None, None, None, y, None, mean, inv)
    var = x.double().var(-1, correction=0)
    # (the mean is off by at most 1000*d_of, 0.1 at 50000 columns, and its square adds to the variance: in fact a few of the last bits are)
    assert ((inv.double() - (var + EPS).rsqrt()).abs() <= 1e-5).all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("cols", [1, 96, 2048, 50000])
def test_constant_rows_infinities_and_nan(cols, dtype):
    x = make(6, cols, dtype, 1)
    x[1] = 0
    x[2] = 5
    x[3, cols // 2] = float("nan")
    x[4, cols // 3] = float("-inf")
    beta = weights(cols, dtype)
    y, mean, inv = torch.empty_like(x), torch.empty(6, device="cuda"), torch.empty(6, device="cuda")
    ops.LayerNormalizeAddOp.apply(EPS, x, y, None, beta, None, None, mean, inv)
    good = [0, 1, 2, 5]
    check_forward(x[good], None, None, beta, y[good], None, mean[good], inv[good])
    assert torch.equal(y[1], beta) and y[3].isnan().all() and y[4].isnan().all() and inv[3].isnan() and inv[4].isnan()


def test_no_rows():
    for dtype in TYPES:
        x = torch.empty(0, 64, device="cuda", dtype=dtype)
        dg, db, r = torch.ones(64, device="cuda", dtype=dtype), torch.ones(64, device="cuda", dtype=dtype), torch.empty(0, device="cuda")
        assert ops.LayerNormAdd(64, dtype=dtype).forward(x, x)[0].shape == (0, 64)
        ops.LayerNormalizeAddOp.adjoint(x, x, r, r.clone(), torch.empty_like(x), None, x, dg, db)
        assert (dg == 0).all() and (db == 0).all()


def test_rows_beyond_32_bits():
    """Rows more than 2^31 elements apart, the last beyond 2^32 elements and 8 GiB."""
    cols, apart = 520, (1 << 31) + 64
    buffer = torch.empty(2 * apart + cols, device="cuda", dtype=torch.bfloat16)
    far = buffer.as_strided((3, cols), (apart, 1))
    x, res, gamma, beta = make(3, cols, torch.bfloat16, 1), make(3, cols, torch.bfloat16, 2), weights(cols, torch.bfloat16), weights(cols, torch.bfloat16, 8)
    far.copy_(x)
    y = torch.empty_like(x)
    ops.LayerNormalizeAddOp.apply(EPS, far, y, gamma, beta, res, far)
    check_forward(x, res, gamma, beta, y, far.contiguous(), None, None)
    dy, t, mean, r, dt = saved(3, cols, torch.bfloat16)
    far.copy_(dy)
    dg, db = torch.empty_like(gamma), torch.empty_like(gamma)
    ops.LayerNormalizeAddOp.adjoint(far, t, mean, r, far, gamma, dt, dg, db)
    check_backward(dy, t, mean, r, gamma, dt, far.contiguous(), dg, db)


def test_more_rows_than_a_launch_has_blocks():
    rows, cols = 70000, 24
    x, res = make(rows, cols, torch.float16, 1), make(rows, cols, torch.float16, 2)
    y, total, mean, inv = torch.empty_like(x), torch.empty_like(x), torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    ops.LayerNormalizeAddOp.apply(EPS, x, y, None, None, res, total, mean, inv)
    check_forward(x, res, None, None, y, total, mean, inv)
    dx, dg, db = torch.empty_like(x), torch.empty(cols, device="cuda"), torch.empty(cols, device="cuda")
    ops.LayerNormalizeAddOp.adjoint(y, total, mean, inv, dx, None, res, dg, db)
    check_backward(y, total, mean, inv, None, res, dx, dg, db)


# rows, cols, and where in a wider array the rows of dy, total and dx begin
FORMS = [(5, 64, (0, 0, 0)), (300, 96, (0, 0, 0)), (40, 1024, (0, 0, 0)), (300, 1000, (3, 3, 3)), (7, 77, (1, 1, 1)), (33, 9001, (0, 0, 0)), (5, 100, (0, 1, 2)),
         (200, 1030, (0, 3, 5)), (3, 20000, (0, 0, 0))]


# the rows' spread and the gradients' size: squares of 1e17 pass f32 as the sum of 2e4 columns, and products of a gradient and a row's element stay above 1e-38, the smallest normal number
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("size, small", [(1e8, 1.0), (1e15, 1.0), (1e17, 1.0), (1e13, 1e-9), (1e17, 1e-15), (1e-8, 1.0), (1e-12, 1.0), (1e-15, 1e-6), (1e-17, 1e-12)])
def test_rows_of_any_size(size, small, dtype):
    for rows, cols, at in FORMS:
        def rows_of(seed, first, scale):
            return (make(rows, cols + 8, torch.float32, seed).double() * scale).to(dtype)[:, first:first + cols]
        what = "%d rows of %d at %s: " % (rows, cols, at)
        t, dy, dt = rows_of(1, at[1], size), rows_of(2, at[0], small), rows_of(3, at[2], small / size)
        gamma, beta = weights(cols, dtype), weights(cols, dtype, 8)
        y, mean, inv = torch.empty(rows, cols + 8, device="cuda", dtype=dtype)[:, at[2]:at[2] + cols], torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
        ops.LayerNormalizeAddOp.apply(EPS, t, y, gamma, beta, None, None, mean, inv)
        check_forward(t, None, gamma, beta, y, None, mean, inv, what)
        var, mean = torch.var_mean(t.double(), -1, correction=0)
        mean, r = mean.float(), var.rsqrt().float()
        for weight, extra in ((gamma, None), (None, dt)):
            dx = torch.empty(rows, cols + 8, device="cuda", dtype=dtype)[:, at[2]:at[2] + cols]
            dg, db = (torch.empty(cols, device="cuda", dtype=torch.float32 if weight is None else dtype) for _ in range(2))
            ops.LayerNormalizeAddOp.adjoint(dy, t, mean, r, dx, weight, extra, dg, db)
            check_backward(dy, t, mean, r, weight, extra, dx, dg, db, what)


@pytest.mark.parametrize("cols", [64, 77, 1024, 20000])
def test_rows_on_either_side_of_the_limits(cols):
    """Squares that leave f32 as a sum: y = beta; a sum of a row that does: NaN."""
    sign = torch.where(torch.arange(cols, device="cuda") % 2 == 0, 1.0, -1.0)
    beta, least = weights(cols, torch.float32, 8), 2.0 ** 64 / cols ** 0.5
    for first in (0, 1):            # whole and ragged rows
        x, y = (torch.empty(3, cols + 8, device="cuda")[:, first:first + cols] for _ in range(2))
        mean, inv = torch.empty(3, device="cuda"), torch.empty(3, device="cuda")
        x.copy_(sign * (0.99 * least))
        ops.LayerNormalizeAddOp.apply(EPS, x, y, None, beta, None, None, mean, inv)
        check_forward(x, None, None, beta, y, None, mean, inv)
        x.copy_(sign * (1.01 * least))
        ops.LayerNormalizeAddOp.apply(EPS, x, y, None, beta, None, None, mean, inv)
        # (the mean of an odd number of columns, 1/cols of their size, takes 1/cols^2 of the squares, 2 in 10^4 of 77)
        assert (inv == 0).all() and torch.equal(y, beta.expand_as(y))
        x.fill_(4e38 / cols)
        ops.LayerNormalizeAddOp.apply(EPS, x, y, None, beta)
        assert y.isnan().all()
