"""Rows of a table by tokens and the table's gradient against the formulas in 64 bits.

Tolerances, u = 2^-24 and h = half a step of the type: a row's terms are added in f32 in some order, n*u of the sum of their magnitudes for n of them, the scale
is one more product, and the result is rounded once more."""
import pytest
import torch

from anode_b200 import ops
from tests.test_gpu_rms_norm import TYPES, U, half_step, make, near, tiny

pytestmark = pytest.mark.gpu

COLS = [1, 7, 16, 33, 64, 200, 515, 1024, 4096, 8193]


def tokens_of(n, vocab, seed=0, kind=torch.int64, spread="zipf", none=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed + 31 * n + vocab)
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    t = ((vocab + 1) ** u - 1).long().clamp(0, vocab - 1) if spread == "zipf" else (u * vocab).long().clamp(0, vocab - 1) if spread == "even" else torch.full((n,), vocab // 2, device="cuda")
    away = torch.tensor([-1, vocab, -100, 2 ** 31 - 1, -2 ** 31], device="cuda")[torch.randint(0, 5, (n,), generator=g, device="cuda")]
    return torch.where(torch.rand(n, generator=g, device="cuda") < none, away, t).to(kind)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("cols", COLS)
def test_forward(cols, dtype):
    for n, vocab, kind, none in ((1, 1, torch.int32, 0), (5, 40, torch.int64, 0.3), (700, 333, torch.int32, 0.1)):
        table, tokens = make(vocab, cols, dtype, 1), tokens_of(n, vocab, 2, kind, none=none)
        inside = ((tokens >= 0) & (tokens < vocab))[:, None]
        rows = torch.where(inside, table[tokens.long().clamp(0, vocab - 1)].double(), 0.0)
        for scale in (1.0, 8.0, 45.25, -0.3):
            y = torch.full((n, cols), 7.0, device="cuda", dtype=dtype)
            ops.EmbedTokensOp.apply(tokens, table, y, scale)
            want = rows * torch.tensor(scale).double()
            near(y, want, want.abs() * (U + half_step(dtype)) * (1 + 2 ** -8) + tiny(dtype), "y")
            if scale in (1.0, 8.0):
                assert torch.equal(y, want.to(dtype))


def check_grad(tokens, dy, dtable, scale, before=None, what=""):
    vocab, cols = dtable.shape
    tokens, dy = tokens.reshape(-1).long(), dy.reshape(-1, cols).double()
    inside = (tokens >= 0) & (tokens < vocab)
    scale = float(torch.tensor(scale))
    at = tokens[inside]
    want = torch.zeros(vocab, cols, device="cuda", dtype=torch.float64).index_add_(0, at, dy[inside]) * scale
    size = torch.zeros(vocab, cols, device="cuda", dtype=torch.float64).index_add_(0, at, dy[inside].abs()) * abs(scale)
    count = torch.bincount(at, minlength=vocab)[:, None].double()
    bound = (count + 2) * U * size
    if before is not None:
        want, bound = want + before.double(), bound + U * (want + before.double()).abs()
        rest = count[:, 0] == 0
        assert torch.equal(dtable[rest], before[rest]), what + "rows that no token names"
    else:
        assert (dtable[count[:, 0] == 0] == 0).all(), what + "rows that no token names"
    near(dtable, want, bound + half_step(dtable.dtype) * (1 + 2 ** -8) * want.abs() + (count > 0) * tiny(dtable.dtype), what + "dtable")


SIZES = [(1, 1), (1, 100), (3, 7), (40, 1), (300, 50), (700, 20000), (2000, 9)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("cols", COLS)
def test_gradient(cols, dtype):
    for n, vocab in SIZES:
        for sums in {dtype, torch.float32}:
            kind, spread, none = (torch.int32, "even", 0.2) if n % 2 else (torch.int64, "zipf", 0.0)
            tokens, dy = tokens_of(n, vocab, 3, kind, spread, none), make(n, cols, dtype, 4)
            out = torch.full((vocab, cols), 7.0, device="cuda", dtype=sums)
            ops.EmbedTokensOp.adjoint(tokens, dy, out, 2.5)
            check_grad(tokens, dy, out, 2.5)
            again = torch.full((vocab, cols), float("nan"), device="cuda", dtype=sums)
            ops.EmbedTokensOp.adjoint(tokens, dy, again, 2.5)
            assert torch.equal(again, out)
            more = make(vocab, cols, sums, 5)
            before = more.clone()
            ops.EmbedTokensOp.adjoint(tokens, dy, more, 2.5, ops.WriteCap.Accumulate)
            check_grad(tokens, dy, more, 2.5, before)


@pytest.mark.parametrize("n, vocab, cols", [(1, 300000, 16), (5000, 300000, 24), (131072, 32768, 64), (131073, 100, 40), (300001, 70001, 8), (20000, 1 << 20, 20), (65536, 65536, 128),
                                            (8193, 262147, 321), (9001, 1 << 20, 72)])
@pytest.mark.parametrize("spread", ["zipf", "even", "one"])
def test_many_tokens_and_large_tables(n, vocab, cols, spread):
    """Whole numbers whose sums are exact, so that no row may be missing or come twice."""
    g = torch.Generator(device="cuda").manual_seed(n)
    tokens = tokens_of(n, vocab, 7, torch.int64, spread, 0.05)
    dy = torch.randint(-2, 3, (n, cols), generator=g, device="cuda").to(torch.bfloat16)
    inside = (tokens >= 0) & (tokens < vocab)
    want = torch.zeros(vocab, cols, device="cuda", dtype=torch.float64).index_add_(0, tokens[inside], dy[inside].double())
    out = torch.full((vocab, cols), 7.0, device="cuda")
    ops.EmbedTokensOp.adjoint(tokens, dy, out)
    assert torch.equal(out.double(), want)
    ops.EmbedTokensOp.adjoint(tokens, dy, out, 1.0, ops.WriteCap.Accumulate)
    assert torch.equal(out.double(), 2 * want)
    half = torch.full((vocab, cols), 7.0, device="cuda", dtype=torch.bfloat16)
    ops.EmbedTokensOp.adjoint(tokens, dy, half)
    assert torch.equal(half, want.to(torch.bfloat16))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("pattern", ["runs", "same", "falling", "pairs", "none", "one among none"])
def test_patterns_of_tokens(pattern, dtype):
    n, vocab, cols = 3001, 512, 72
    i = torch.arange(n, device="cuda")
    tokens = {"runs": i // 97, "same": 0 * i + 511, "falling": 511 - i % 512, "pairs": (i // 2) % 512, "none": 0 * i - 1, "one among none": torch.where(i == 1500, 17, -1)}[pattern]
    dy, out = make(n, cols, dtype, 1), torch.full((vocab, cols), 7.0, device="cuda", dtype=dtype)
    ops.EmbedTokensOp.adjoint(tokens, dy, out)
    check_grad(tokens, dy, out, 1.0, None, pattern + " ")


@pytest.mark.parametrize("pattern", ["runs", "same", "falling", "pairs", "none", "one among none"])
@pytest.mark.parametrize("n", [8193, 16385, 40001])
def test_patterns_of_many_tokens(pattern, n):
    """The same beyond the tokens that are sorted by counting, with whole numbers: both clusters of the sort give the sums exactly, and the same bits again."""
    vocab, cols = 70001, 136
    i = torch.arange(n, device="cuda")
    tokens = {"runs": i // 97, "same": 0 * i + 511, "falling": n - 1 - i, "pairs": (i // 2) % vocab, "none": 0 * i - 1, "one among none": torch.where(i == 1500, 17, -1)}[pattern]
    dy = torch.randint(-2, 3, (n, cols), generator=torch.Generator(device="cuda").manual_seed(n), device="cuda").to(torch.float16)
    inside = tokens >= 0
    want = torch.zeros(vocab, cols, device="cuda").index_add_(0, tokens[inside], dy[inside].float())
    whole, added = torch.full((vocab, cols), 7.0, device="cuda"), torch.zeros(vocab, cols, device="cuda")
    ops.EmbedTokensOp.adjoint(tokens, dy, whole)
    ops.EmbedTokensOp.adjoint(tokens, dy, added, 1.0, ops.WriteCap.Accumulate)
    assert torch.equal(whole, want) and torch.equal(added, want)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("cols", [64, 100, 33, 1000])
def test_strides_and_alignment(cols, dtype):
    """Slices that begin anywhere; what lies beside the rows stays; the gradient of a broadcast row."""
    vocab, n = 60, 50
    wide = [make(vocab, 2 * cols + 9, dtype, s) for s in range(4)]
    tokens = tokens_of(n, vocab, 1, torch.int64, "zipf", 0.1).view(5, 10)
    inside = ((tokens >= 0) & (tokens < vocab))[..., None]
    for first in (0, 1, 3, 8):
        before = [w.clone() for w in wide]
        table, y = wide[0][:, first:first + cols], wide[1][:n, first + 1:first + 1 + cols].unflatten(0, (5, 10))
        ops.EmbedTokensOp.apply(tokens, table, y, 1.0)
        assert torch.equal(y, torch.where(inside, table[tokens.clamp(0, vocab - 1)], 0))
        dy, dtable = wide[2][:n, first:first + cols].unflatten(0, (5, 10)), wide[3][:, first:first + cols]
        ops.EmbedTokensOp.adjoint(tokens, dy, dtable, 0.5)
        check_grad(tokens, dy, dtable, 0.5)
        before[1][:n, first + 1:first + 1 + cols] = wide[1][:n, first + 1:first + 1 + cols]
        before[3][:, first:first + cols] = dtable
        assert all(torch.equal(a, b) for a, b in zip(before, wide))
    one, out = make(1, cols, dtype, 9), torch.empty(vocab, cols, device="cuda", dtype=torch.float32)
    ops.EmbedTokensOp.adjoint(tokens, one.expand(5, 10, cols), out)
    check_grad(tokens, one.expand(5, 10, cols), out, 1.0)
    y = torch.empty(5, 10, cols, device="cuda", dtype=dtype)
    ops.EmbedTokensOp.apply(tokens, one.expand(vocab, cols), y)
    assert torch.equal(y, torch.where(inside, one, 0))


def test_infinities_and_nan_stay_in_their_rows():
    tokens = torch.tensor([3, 5, 3, 7], device="cuda")
    dy = make(4, 40, torch.float16, 1)
    dy[1, 4], dy[2, 5] = float("inf"), float("nan")
    out = torch.empty(9, 40, device="cuda", dtype=torch.float16)
    ops.EmbedTokensOp.adjoint(tokens, dy, out)
    bad = torch.zeros(9, 40, dtype=torch.bool, device="cuda")
    bad[5, 4] = bad[3, 5] = True
    assert torch.equal(~out.isfinite(), bad) and out[5, 4].isposinf() and out[3, 5].isnan()


def test_no_tokens():
    tokens, dy = torch.empty(0, 3, device="cuda", dtype=torch.int64), torch.empty(0, 3, 16, device="cuda")
    out = torch.ones(7, 16, device="cuda")
    ops.EmbedTokensOp.adjoint(tokens, dy, out, 1.0, ops.WriteCap.Accumulate)
    assert (out == 1).all()
    ops.EmbedTokensOp.adjoint(tokens, dy, out)
    assert (out == 0).all()
    assert ops.EmbedTokensOp.apply(tokens, out, dy).shape == (0, 3, 16)


def test_tables_beyond_32_bits():
    """A table's rows beyond 2^32 elements, and rows of dy 2^31 elements apart."""
    vocab, cols = 70000, 65536
    table = torch.zeros(vocab, cols, device="cuda", dtype=torch.bfloat16)
    tokens = torch.tensor([69999, 0, 69999, 65537, 33], device="cuda")
    for k, t in enumerate((69999, 0, 65537, 33)):
        table[t] = k + 1
    y = torch.empty(5, cols, device="cuda", dtype=torch.bfloat16)
    ops.EmbedTokensOp.apply(tokens, table, y)
    assert torch.equal(y[:, 0].float(), torch.tensor([1.0, 2, 1, 3, 4], device="cuda")) and (y == y[:, :1]).all()
    ops.EmbedTokensOp.adjoint(tokens, y, table, 0.5)
    assert torch.equal(table[[69999, 0, 65537, 33], 5].float(), torch.tensor([1.0, 1, 1.5, 2], device="cuda"))
    assert (table[1:33] == 0).all() and (table[65538:69999] == 0).all() and (table[[69999, 65537]] == table[[69999, 65537], :1]).all()
    del y
    apart = (1 << 31) + 8
    far = table.view(-1).as_strided((2, 40), (apart, 1))
    far.copy_(make(2, 40, torch.bfloat16, 1))
    out = torch.empty(3, 40, device="cuda", dtype=torch.bfloat16)
    ops.EmbedTokensOp.adjoint(torch.tensor([2, 0], device="cuda"), far, out)
    assert torch.equal(out, torch.stack((far[1], 0 * far[0], far[0])))


def test_layer_and_differences():
    """y is linear in the table, so the gradient along a direction is y of that direction, against dy."""
    layer = ops.TokenEmbedding(50, 24, 3.0)
    direction = make(50, 24, torch.float32, 1)
    layer.table.copy_(direction)
    tokens = tokens_of(200, 50, 1, torch.int32, "zipf", 0.1).view(10, 20)
    with pytest.raises(RuntimeError):
        layer.backward(direction)
    y, dy = layer.forward(tokens), make(200, 24, torch.float32, 2).view(10, 20, 24)
    d = layer.backward(dy)
    assert d is layer.dtable
    want, size = (y.double() * dy.double()).sum(), (y.double() * dy.double()).abs().sum()
    assert abs(float((d.double() * direction.double()).sum() - want)) <= 210 * U * float(size)
    once = d.clone()
    layer.backward(dy, ops.WriteCap.Accumulate)
    near(layer.dtable, 2 * once.double(), 2 * U * once.double().abs(), "accumulated")
