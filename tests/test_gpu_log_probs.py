"""Log probabilities of tokens, entropies, the likeliest tokens and the logits' gradient against the formulas in 64 bits.

Tolerances, u = 2^-24: z = scale*(x - m) is off by 2u of itself, its product with log2(e) by 2u more, an exponential by 4u beside that; a sum of positive terms by
D = (vocab/128 + 64)*u of itself (a thread adds at most vocab/128 of a row's terms in turn, rows of fewer than 4096 at most 32; the rest are joins and changes
of the largest).  So S is off by (4u*mean|z| + 4u + D)*S, the mean over the probabilities, and L by that and 2u*|L|."""
import math

import pytest
import torch

from anode_b200 import ops
from tests.test_gpu_rms_norm import TYPES, U, half_step, make, near, tiny

pytestmark = pytest.mark.gpu

INF = float("inf")
SHAPES = [(1, 1), (2, 2), (1, 7), (5, 33), (3, 64), (7, 129), (300, 100), (40, 1000), (9, 4096), (33, 4099), (700, 515), (2, 50021), (1, 131072), (20, 32768), (3, 262147)]


def logits_of(rows, vocab, dtype, seed=0, spread=3.0):
    return make(rows, vocab, dtype, seed, spread)


def tokens_of(rows, vocab, seed=0, kind=torch.int64, none=0.2):
    g = torch.Generator(device="cuda").manual_seed(seed + rows)
    t = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    away = torch.tensor([-1, vocab, -100, 2 ** 31 - 1], device="cuda")[torch.randint(0, 4, (rows,), generator=g, device="cuda")]
    return torch.where(torch.rand(rows, generator=g, device="cuda") < none, away, t).to(kind)


def d_of(vocab):
    return (vocab / 128 + 64) * U


class Exact:
    """The formulas in 64 bits, and how far f32 may be from them."""

    def __init__(self, logits, scale):
        x = logits.double()
        self.vocab, self.scale = x.shape[1], float(torch.tensor(scale))
        self.m = x.amax(1, keepdim=True)
        self.empty = self.m == -INF
        self.z = (x - torch.where(self.empty, 0.0, self.m)) * self.scale
        e = self.z.exp()
        s = torch.where(self.empty, 1.0, e.sum(1, keepdim=True))
        self.p = e / s
        self.L = s.log()
        near_z = torch.where(self.p > 0, self.z, 0.0)
        mean_z, mean_zz = (self.p * near_z.abs()).sum(1, keepdim=True), (self.p * near_z.square()).sum(1, keepdim=True)
        self.entropy = torch.where(self.empty, 0.0, self.L + mean_z)
        self.off_L = 4 * U * mean_z + 8 * U + d_of(self.vocab) + 2 * U * self.L.abs()
        self.off_entropy = self.off_L + 4 * U * mean_zz + (2 * d_of(self.vocab) + 16 * U) * mean_z + 2 * U * self.entropy

    def log_prob(self, index):
        """(log probabilities of the columns `index`, how far off)"""
        z = self.z.gather(1, index)
        want = torch.where(self.empty, -INF, z - self.L)
        want = torch.where(want < -3.4028235e38, -INF, want)      # (beyond f32)
        return want, torch.where(want.isfinite(), self.off_L + 3 * U * (z.abs() + want.abs()), 0.0)


def check(logits, tokens, scale, logprob=None, entropy=None, stats=None, top_logprob=None, top_token=None, what=""):
    x = Exact(logits, scale)
    if logprob is not None:
        inside = (tokens >= 0) & (tokens < x.vocab)
        want, off = x.log_prob(torch.where(inside, tokens, 0).long()[:, None])
        near(logprob, torch.where(inside, want[:, 0], 0.0), torch.where(inside, off[:, 0], 0.0), what + "logprob")
    if entropy is not None:
        near(entropy, x.entropy[:, 0], x.off_entropy[:, 0], what + "entropy")
    if stats is not None:
        assert torch.equal(stats[:, :1].double(), x.m), what + "largest"
        near(stats[:, 1:], x.L * ~x.empty, x.off_L, what + "L")
    if top_token is not None:
        order = torch.sort(logits.double(), dim=1, descending=True, stable=True)[1][:, :top_token.shape[1]]
        assert torch.equal(top_token.long(), order), what + "likeliest tokens"
        if top_logprob is not None:
            near(top_logprob, *x.log_prob(order), what + "their log probabilities")


def forward(logits, tokens, scale=1.0, top=0, kind=torch.int64, entropy=True):
    rows = logits.shape[0]
    f = lambda *s: torch.full((rows,) + s, 7.0, device="cuda")      # noqa: E731
    out = dict(logprob=f() if tokens is not None else None, entropy=f() if entropy else None, stats=f(2), top_logprob=f(top) if top else None,
               top_token=torch.full((rows, top), -7, device="cuda", dtype=kind) if top else None)
    ops.TokenLogProbsOp.apply(logits, tokens, *out.values(), scale)
    return out


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows, vocab", SHAPES)
def test_forward(rows, vocab, dtype):
    x = logits_of(rows, vocab, dtype, 1)
    for scale, top, kind in ((1.0, 0, torch.int64), (0.7, 1, torch.int32), (2.0, 5, torch.int64), (1.0, 20, torch.int32), (1.0, 64, torch.int64), (1.25, 128, torch.int64)):
        if top > vocab:
            continue
        tokens = tokens_of(rows, vocab, 2, kind)
        out = forward(x, tokens, scale, top, kind)
        check(x, tokens, scale, **out)
        # each output alone, and the same call again: the same bits
        again = forward(x, tokens, scale, top, kind)
        assert all(a is None or torch.equal(a, b) for a, b in zip(out.values(), again.values()))
        for name in out:
            if out[name] is not None:
                alone = torch.empty_like(out[name])
                ops.TokenLogProbsOp.apply(x, tokens, **{**dict.fromkeys(out), name: alone}, scale=scale)
                if name in ("stats", "top_token"):
                    assert torch.equal(alone[:, :1] if name == "stats" else alone, out[name][:, :1] if name == "stats" else out[name]), name
                check(x, tokens, scale, **({name: alone} if name != "top_logprob" else dict(top_logprob=alone, top_token=out["top_token"])), what="alone ")


def check_grad(logits, tokens, scale, stats, entropy, dlogprob, dentropy, dlogits, what=""):
    vocab, scale = logits.shape[1], float(torch.tensor(scale))
    m, L = stats.double()[:, :1], stats.double()[:, 1:]
    empty = m == -INF
    z = (logits.double() - torch.where(empty, 0.0, m)) * scale
    l = z - L
    p = l.exp()
    l = torch.where(p > 0, l, 0.0)
    dl = torch.zeros_like(L) if dlogprob is None else dlogprob.double()[:, None]
    dh = torch.zeros_like(L) if dentropy is None else dentropy.double()[:, None]
    h = torch.zeros_like(L) if dentropy is None else entropy.double()[:, None]
    hot = torch.zeros_like(z)
    if dlogprob is not None:
        inside = (tokens >= 0) & (tokens < vocab)
        dl = torch.where(inside[:, None], dl, 0.0)
        hot.scatter_(1, torch.where(inside, tokens, 0).long()[:, None], inside[:, None].double())
    want = torch.where(empty, 0.0, scale * (dl * hot - p * (dl + dh * (l + h))))
    size = dl.abs() + dh.abs() * (l.abs() + h.abs())
    # l is off by 4u of z and L, its product with log2(e) by 2u of l, the exponential by 4u beside that
    off = scale * (p * size * ((4 * z.abs() + 4 * L.abs() + 4 * l.abs()) * U + 12 * U) + p * dh.abs() * 4 * U * (z.abs() + L.abs()) + 4 * U * (dl.abs() * hot + p * size))
    off = torch.where(p > 0, off, 0.0) + 2.0 ** -126 * scale * size      # (what is below f32's smallest number may be zero)
    near(dlogits, want, off + half_step(dlogits.dtype) * (1 + 2 ** -8) * want.abs() + tiny(dlogits.dtype), what + "dlogits")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows, vocab", SHAPES)
def test_gradient(rows, vocab, dtype):
    x = logits_of(rows, vocab, dtype, 1)
    dl, dh = make(1, rows, torch.float32, 5)[0], make(1, rows, torch.float32, 6)[0]
    for scale, kind, both in ((1.0, torch.int64, (dl, dh)), (0.7, torch.int32, (dl, None)), (2.0, torch.int64, (None, dh))):
        tokens = tokens_of(rows, vocab, 3, kind)
        out = forward(x, tokens, scale)
        args = (tokens if both[0] is not None else None, out["stats"], both[0])
        dx = torch.full_like(x, 7.0)
        ops.TokenLogProbsOp.adjoint(x, *args, dx, out["entropy"] if both[1] is not None else None, both[1], scale)
        check_grad(x, tokens, scale, out["stats"], out["entropy"], *both, dx)
        z = x.clone()       # in place: the same bits
        ops.TokenLogProbsOp.adjoint(z, *args, z, out["entropy"] if both[1] is not None else None, both[1], scale)
        assert torch.equal(z, dx)


def test_gradient_is_that_of_the_forward_pass():
    """Against differences of the 64-bit forward formula along random directions."""
    rows, vocab, scale = 6, 300, 1.5
    x, w, v = logits_of(rows, vocab, torch.float32, 1), make(1, rows, torch.float32, 2)[0], make(1, rows, torch.float32, 3)[0]
    tokens = tokens_of(rows, vocab, 4)
    layer = ops.TokenLogProbs(scale)
    layer.forward(x, tokens)
    dx = layer.backward(w, v)
    inside = (tokens >= 0) & (tokens < vocab)

    def value(x):
        lp = torch.log_softmax(x * scale, 1)
        picked = lp.gather(1, torch.where(inside, tokens, 0)[:, None])[:, 0]
        return (torch.where(inside, picked, 0.0) * w.double() - (lp.exp() * lp).sum(1) * v.double()).sum()

    for seed in range(3):
        d, step = make(rows, vocab, torch.float32, 20 + seed).double(), 1e-6
        want = (value(x.double() + step * d) - value(x.double() - step * d)) / (2 * step)
        # second differences are of the order of step^2, f64 rounding 1e-16*1e3/step, the gradients themselves 1e-6 of their size
        assert abs(float(want - (dx.double() * d).sum())) <= 1e-5 * float((dx.double().abs() * d.abs()).sum()) + 1e-6


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("vocab", [200, 5000, 70001])
def test_masked_rows(vocab, dtype):
    """Masks of -infinity and of the type's lowest value: all but a few, all but one, all."""
    low = torch.finfo(dtype).min
    for mask in (-INF, low):
        x = logits_of(7, vocab, dtype, 1)
        keep = torch.zeros(7, vocab, dtype=torch.bool, device="cuda")
        keep[0], keep[1, ::3], keep[2, 5], keep[3, [7, vocab - 1, 3]] = True, True, True, True
        keep[5, vocab - 9:], keep[6, :4] = True, True
        x[~keep] = mask
        tokens = torch.tensor([3, 0, 5, 3, 1, 0, -1], device="cuda")
        for scale in (1.0, 0.5, 3.0):
            for top in (1, 20, 128):
                out = forward(x, tokens, scale, top)
                check(x, tokens, scale, **out, what="%r " % mask)
            e = Exact(x, scale)
            if mask == -INF:
                assert out["logprob"][4] == -INF and out["entropy"][4] == 0 and out["stats"][4, 0] == -INF and out["stats"][4, 1] == 0
                assert (out["top_logprob"][4] == -INF).all() and torch.equal(out["top_token"][4], torch.arange(128, device="cuda")) and out["logprob"][5] == -INF
            else:
                assert abs(float(out["entropy"][4]) - math.log(vocab)) < 1e-4 and e.entropy[4] > 0
            dl, dh = make(1, 7, torch.float32, 5)[0], make(1, 7, torch.float32, 6)[0]
            dx = torch.empty_like(x)
            ops.TokenLogProbsOp.adjoint(x, tokens, out["stats"], dl, dx, out["entropy"], dh, scale)
            check_grad(x, tokens, scale, out["stats"], out["entropy"], dl, dh, dx, "%r " % mask)
            if mask == -INF:
                assert (dx[4] == 0).all() and (dx[~keep & (torch.arange(vocab, device="cuda") != tokens[:, None])] == 0).all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("vocab", [129, 3000, 40000, 150001])
@pytest.mark.parametrize("pattern", ["equal", "rising", "falling", "two values", "few large", "striped", "strided", "zeros of both signs", "steps", "last"])
def test_patterns_of_the_likeliest(pattern, vocab, dtype):
    """Ties by the lowest index, whatever the order and however many there are; the largest ones side by side, at one distance from each other, or all of one part."""
    i = torch.arange(vocab, device="cuda", dtype=torch.float32)
    row = {"equal": 0 * i + 2, "rising": i / vocab * 8, "falling": 8 - i / vocab * 8, "two values": (i % 7 == 3).float(), "few large": torch.where(i % 4999 == 77, 9.0, 0.0),
           "striped": torch.where((i // 8) % 64 == 5, 5 + (i % 1024) / 1024, 0.1 * (i % 10)), "strided": torch.where(i % 1024 == 9, 5 + i / vocab, -i / vocab),
           "zeros of both signs": torch.where(i % 2 == 0, -0.0, 0.0), "steps": (i // 1000) % 13, "last": torch.where(i >= vocab - 100, 4.0, 1.0)}[pattern]
    x = torch.stack((row, row.flip(0), row.roll(vocab // 3))).to(dtype)
    for top in (1, 5, 20, 64, 128):
        check(x, None, 1.0, **forward(x, None, 1.0, top))
    # as one of many rows
    many = x[:1].expand(200, vocab)
    check(many, None, 1.0, **forward(many, None, 1.0, 20))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("vocab", [300, 9000, 100003])
def test_infinities_and_nan(vocab, dtype):
    x = logits_of(5, vocab, dtype, 1)
    x[1, 17], x[2, vocab - 1], x[3, 100], x[3, 50] = float("nan"), INF, float("nan"), INF
    tokens = torch.tensor([1, 2, 3, -1, 4], device="cuda")
    out = forward(x, tokens, 1.0, 8)
    good = [0, 4]
    check(x[good], tokens[good], 1.0, **{k: v[good] for k, v in out.items()})
    for k in ("logprob", "entropy"):
        assert out[k][[1, 2]].isnan().all() and (out[k][3].isnan() or k == "logprob")
    assert out["logprob"][3] == 0 and out["top_logprob"][1:4].isnan().all()
    assert torch.equal(out["top_token"], torch.sort(x.float(), dim=1, descending=True, stable=True)[1][:, :8])
    dx = torch.empty_like(x)
    w = torch.ones(5, device="cuda")
    ops.TokenLogProbsOp.adjoint(x, tokens, out["stats"], w, dx, out["entropy"], w)
    assert dx[1:3].isnan().all() and dx[good].isfinite().all()


@pytest.mark.parametrize("scale", [1e-30, 1e-3, 1.0, 50.0, 1e30])
def test_large_logits_and_far_temperatures(scale):
    """A common addend of 1e5 takes digits off the logits, none off the log probabilities; differences that scale beyond f32 are probabilities of zero."""
    x = logits_of(9, 5000, torch.float32, 1) + 1e5
    tokens = tokens_of(9, 5000, 2)
    out = forward(x, tokens, scale, 5)
    check(x, tokens, scale, **{k: v for k, v in out.items() if k in ("stats", "entropy", "top_token")})
    e = Exact(x, scale)
    inside = (tokens >= 0) & (tokens < 5000)
    want, off = e.log_prob(torch.where(inside, tokens, 0)[:, None])
    far = want.abs() > 3e38
    got = out["logprob"][:, None]
    assert (got[far & inside[:, None]] == -INF).all()
    near(torch.where(far | ~inside[:, None], 0.0, got), torch.where(far | ~inside[:, None], 0.0, want), off, "logprob")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("vocab", [64, 100, 1024, 33, 30001])
def test_strides_and_alignment(vocab, dtype):
    """Rows of a padded vocabulary that begin anywhere: what lies beside them is neither counted nor written; broadcast rows."""
    rows = 6
    wide = [make(rows + 1, 2 * vocab + 9, dtype, s, 3.0) for s in range(2)]
    tokens = tokens_of(rows, vocab, 1).view(2, 3)
    layer = ops.TokenLogProbs(0.9)
    for first in (0, 1, 3, 8):
        x, dx = (w[:rows, first:first + vocab].unflatten(0, (2, 3)) for w in wide)
        wide[0][:, first + vocab:] = INF
        before = wide[1].clone()
        logprob, entropy = layer.forward(x, tokens)
        assert logprob.shape == entropy.shape == (2, 3)
        check(x.flatten(0, 1), tokens.flatten(), 0.9, logprob.flatten(), entropy.flatten())
        best = layer.infer(x, None, 7)
        check(x.flatten(0, 1), None, 0.9, top_logprob=best[2].flatten(0, 1), top_token=best[3].flatten(0, 1))
        w = torch.ones(2, 3, device="cuda")
        layer.backward(w, w, dx)
        check_grad(x.flatten(0, 1), tokens.flatten(), 0.9, layer._saved[2].flatten(0, 1), entropy.flatten(), w.flatten(), w.flatten(), dx.flatten(0, 1))
        before[:rows, first:first + vocab] = dx.flatten(0, 1)
        assert torch.equal(before, wide[1])
        wide[0][:, first + vocab:] = 0
    one = make(1, vocab, dtype, 40).expand(9, vocab)
    check(one, tokens_of(9, vocab), 1.0, **forward(one, tokens_of(9, vocab), 1.0, 3))


def test_no_rows():
    x, none = torch.empty(0, 40, device="cuda"), torch.empty(0, device="cuda", dtype=torch.int64)
    layer = ops.TokenLogProbs()
    assert layer.forward(x, none)[0].shape == (0,) and layer.infer(x, none, 5)[3].shape == (0, 5)
    assert layer.backward(torch.empty(0, device="cuda")).shape == (0, 40)


def test_rows_beyond_32_bits():
    """Rows more than 2^31 elements apart, and one row longer than that many bytes."""
    vocab, apart = 5003, (1 << 31) + 64
    buffer = torch.empty(2 * apart + vocab, device="cuda", dtype=torch.bfloat16)
    far = buffer.as_strided((3, vocab), (apart, 1))
    x, tokens = logits_of(3, vocab, torch.bfloat16, 1), torch.tensor([1, vocab - 1, -1], device="cuda")
    far.copy_(x)
    out = forward(far, tokens, 1.0, 9)
    check(x, tokens, 1.0, **out)
    w = torch.ones(3, device="cuda")
    ops.TokenLogProbsOp.adjoint(far, tokens, out["stats"], w, far, out["entropy"], w)
    check_grad(x, tokens, 1.0, out["stats"], out["entropy"], w, w, far.contiguous())
    wide = buffer[:(1 << 30) + (1 << 29)].view(1, -1)
    wide.zero_()
    wide[0, -5], wide[0, 12345], wide[0, 7] = 30.0, 30.0, 29.0
    n = wide.shape[1]
    best = torch.empty(1, 4, device="cuda", dtype=torch.int64)
    values, entropy = torch.empty(1, 4, device="cuda"), torch.empty(1, device="cuda")
    ops.TokenLogProbsOp.apply(wide, None, None, entropy, None, values, best)
    assert best.tolist() == [[12345, n - 5, 7, 0]]
    total = math.log(2 + math.exp(-1.0) + (n - 3) * math.exp(-30.0))
    assert abs(float(values[0, 0]) + total) < 1e-4 and abs(float(values[0, 3]) + 30 + total) < 1e-4
