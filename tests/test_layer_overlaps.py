"""Layers refuse an output that touches what their backward pass reads, wherever the two meet, and take one that lies beside it."""
import pytest
import torch

from anode_b200 import ops

TAKEN = "CUDA tensor"          # (as far as a machine without a device goes)
REFUSED = "backward pass"


def norm(x, out, residual=None, total=None):
    return lambda: ops.RmsNormAdd(8, device="cpu").forward(x, residual, out, total)


def rotary(q, k, q_out, k_out, norm=True):
    return lambda: ops.RotaryPositions(8, norm=norm, device="cpu").forward(q, k, torch.arange(6), q_out, k_out)


def cases():
    wide = torch.zeros(9, 32)
    x = wide[:6, 8:16]
    rows = torch.zeros(10, 8)
    yield "the row below", norm(rows[:6], rows[1:7]), REFUSED
    yield "the last row", norm(rows[:6], rows[5:9]), REFUSED
    yield "behind the rows", norm(rows[:5], rows[5:]), TAKEN
    yield "columns behind", norm(x, wide[:6, 16:24]), TAKEN
    yield "columns before", norm(x, wide[:6, :8]), TAKEN
    yield "columns across", norm(x, wide[:6, 15:23]), REFUSED
    yield "columns across, from before", norm(x, wide[:6, 1:9]), REFUSED
    yield "columns of later rows", norm(x, wide[3:9, 16:24]), TAKEN
    yield "one column of later rows", norm(x, wide[2:8, 9:17]), REFUSED
    yield "the same memory at other strides", norm(x, wide.view(-1)[8:56].view(6, 8)), REFUSED
    yield "elsewhere", norm(x, torch.zeros(6, 8)), TAKEN
    yield "no rows", norm(rows[:0], rows[:0]), TAKEN
    yield "a broadcast row", norm(rows[:1].expand(6, 8), rows[4:]), TAKEN
    yield "a broadcast row's place", norm(rows[4:5].expand(6, 8), rows[:6]), REFUSED
    # with a residual it is the sum that is kept
    r, other = torch.zeros(6, 8), torch.zeros(6, 8)
    yield "x's place with a residual", norm(x, x, r, other), TAKEN
    yield "the sum's place", norm(x, other, r, other), REFUSED
    yield "across the sum", norm(rows[:6], wide[:6, 4:12], r, x), REFUSED
    yield "beside the sum", norm(rows[:6], wide[:6, 16:24], r, x), TAKEN
    packed = torch.zeros(6, 7, 8)
    q, k, v = packed.split((3, 2, 2), 1)
    yield "keys in the values' place", rotary(q, k, torch.zeros(6, 3, 8), v), TAKEN
    yield "queries a head on", rotary(q, k, packed[:, 1:4], torch.zeros(6, 2, 8)), REFUSED
    yield "queries' last head", rotary(q, k, torch.zeros(6, 3, 8), packed[:, 2:4]), REFUSED
    yield "queries over keys", rotary(q, k, packed[:, 4:7], None), REFUSED
    yield "one key head over a query's", rotary(q, packed[:, 3:4], None, packed[:, 2:3]), REFUSED
    yield "one key head beside", rotary(q, packed[:, 3:4], None, packed[:, 4:5]), TAKEN
    yield "without a norm nothing is read", rotary(q, k, packed[:, 1:4], v, norm=False), TAKEN
    heads_first = torch.zeros(3, 12, 8)
    yield "heads first, tokens behind", rotary(heads_first[:, :6].transpose(0, 1), None, heads_first[:, 6:].transpose(0, 1), None), TAKEN
    yield "heads first, a token across", rotary(heads_first[:, :6].transpose(0, 1), None, heads_first[:, 5:11].transpose(0, 1), None), REFUSED


@pytest.mark.skipif(torch.cuda.is_available(), reason="arrays on the host go as far as a machine without a device")
@pytest.mark.parametrize("call, why", [pytest.param(*c[1:], id=c[0]) for c in cases()])
def test_outputs_beside_and_across_what_is_kept(call, why):
    with pytest.raises(ValueError, match=why):
        call()


def test_every_pair_of_small_arrays():
    """Whether two arrays share an element, against a count of their elements."""
    base = torch.arange(700, dtype=torch.float32)
    seen = set()
    for strides in ((20, 4, 1), (1, 20, 4), (40, 5, 1), (7, 3, 1), (0, 4, 1), (6, 6, 1), (100, 25, 2)):
        for na, nb in (((3, 2, 3), (3, 2, 3)), ((3, 1, 4), (3, 4, 4)), ((1, 3, 2), (2, 3, 2)), ((2, 2, 1), (2, 3, 1))):
            a = base.as_strided(na, strides, 0)
            for at in range(0, 120):
                b = base.as_strided(nb, strides, at)
                want = bool(set(a.flatten().tolist()) & set(b.flatten().tolist()))
                assert ops._share_memory(a, b) == ops._share_memory(b, a) == want, (strides, na, nb, at)
                seen.add(want)
                other = base.as_strided(nb, (33, 5, 1), at)
                assert ops._share_memory(a, other) == bool(set(a.flatten().tolist()) & set(other.flatten().tolist())), (strides, na, nb, at)
    assert seen == {True, False}
