"""Outputs that share memory with one another, or with an input whose place they may not have, are refused, on any machine, and those that lie beside one another are
not.  Nothing of a refused call reaches CUDA: addresses here are numbers that no kernel may see."""
import itertools

import pytest
import torch

from tests.test_more_row_refusals import P, STRIDE, embed, embed_grad, layer, layer_grad, probs

LAUNCH = -4          # what a call that is taken answers on a machine without a device

no_device = pytest.mark.skipif(torch.cuda.is_available(), reason="a call that is taken would run")

# of 4 rows with 20 alternatives: each output's bytes
SIZES = dict(logprob=16, entropy=16, stats=32, top_logprob=320, top_token=640)


@pytest.mark.parametrize("a, b", list(itertools.permutations(SIZES, 2)))
def test_outputs_of_log_probabilities(a, b):
    at = 10 * P
    assert probs(**{a: at, b: at}) == STRIDE
    # the last eight bytes of one, the first of the other
    assert probs(**{a: at, b: at + SIZES[a] - 8}) == STRIDE


@no_device
def test_outputs_of_log_probabilities_side_by_side():
    ends = list(itertools.accumulate(SIZES.values(), initial=10 * P))
    assert probs(**dict(zip(SIZES, ends))) == LAUNCH
    # what is not asked for has no place
    assert probs(top=0, logprob=10 * P, entropy=10 * P + 16, top_logprob=10 * P, top_token=10 * P) == LAUNCH
    assert probs(rows=0, logprob=10 * P, entropy=10 * P) == 0


def meets(p, p_stride, p_rows, q, q_stride, q_rows, length, q_length=None):
    """Whether rows of `length` bytes have one in common, by looking at each pair of them."""
    return any(p + i * p_stride < q + j * q_stride + (q_length or length) and q + j * q_stride < p + i * p_stride + length for i in range(p_rows) for j in range(q_rows))


def rows_beside(dtype=None):
    """(first, stride, rows) of an output and of an input of 8 columns of two bytes; the output's rows do not overlap."""
    places = [0, 2, 14, 16, 18, 32, 48, 62, 64, 66, 80, 144, 158, 160, 162, 400]
    for (out, table), (s, t), (n, m) in itertools.product([(0, p) for p in places] + [(p, 0) for p in places[1:]], [(16, 16), (32, 32), (32, 16), (16, 32), (48, 32), (32, 0), (32, 6)],
                                                          [(1, 1), (4, 3), (1, 6), (5, 1)]):
        yield out, s, n, table, t, m


def test_rows_of_a_table_that_the_output_meets():
    """embed: y against the table; embed_grad: the gradient against dy.  Each place by the pairs' own comparison."""
    refused = taken = 0
    for out, s, n, other, t, m in rows_beside():
        meet = meets(out, s, n, other, t, m, 16)
        refused, taken = refused + meet, taken + (not meet)
        if not meet and torch.cuda.is_available():
            continue
        a, b = 8 * P + out, 8 * P + other
        want = STRIDE if meet else LAUNCH
        assert embed(tokens=n, vocab=m, y=a, y_stride=s // 2, table=b, table_stride=t // 2) == want, (out, s, n, other, t, m)
        assert embed_grad(vocab=n, tokens=m, dtable=a, dtable_stride=s // 2, dy=b, dy_stride=t // 2) == want, (out, s, n, other, t, m)
    assert refused > 100 and taken > 100


def test_a_gradient_in_32_bits_over_what_it_adds_up():
    """3 rows of 8 columns of four bytes, with as much between them, and 5 rows of dy of two bytes side by side."""
    for at in range(-96, 224, 4):
        meet = meets(0, 64, 3, at, 16, 5, 32, 16)
        if meet or not torch.cuda.is_available():
            assert embed_grad(vocab=3, dtable=8 * P, dtable_stride=16, dtable_type=0, tokens=5, dy=8 * P + at, dy_stride=8) == (STRIDE if meet else LAUNCH), at


@no_device
def test_many_rows_side_by_side_are_taken_at_once():
    """Rows of a packed projection's columns: 2^30 of them, which no one looks at one by one."""
    n = 1 << 30
    assert embed(tokens=n, vocab=n, y=P, y_stride=16, table=P + 16, table_stride=16) == LAUNCH
    assert embed(tokens=n, vocab=n, y=P, y_stride=16, table=P + 14, table_stride=16) == STRIDE


def test_layer_norm_y_and_the_sum():
    """4 rows of 8 columns of two bytes each, at distances of their own."""
    refused = 0
    for at, s, t in itertools.product(range(-130, 132, 2), (16, 32, 48), (16, 32)):
        meet = meets(0, s, 4, at, t, 4, 16)
        refused += meet
        if meet or not torch.cuda.is_available():
            assert layer(y=20 * P, y_stride=s // 2, total=20 * P + at, total_stride=t // 2) == (STRIDE if meet else LAUNCH), (at, s, t)
    assert refused > 100


def test_layer_norm_numbers_of_each_row():
    for at in range(-20, 24, 4):         # 4 rows of four bytes
        if abs(at) < 16 or not torch.cuda.is_available():
            assert layer(mean=20 * P, inv_std=20 * P + at) == (STRIDE if abs(at) < 16 else LAUNCH), at


def test_layer_norm_gradients_of_the_weights():
    """8 columns of four bytes: the two gradients apart, dbeta apart from gamma, dgamma in gamma's very place or apart from it."""
    for at in range(-40, 44, 4):
        meet = abs(at) < 32
        if meet or not torch.cuda.is_available():
            want = STRIDE if meet else LAUNCH
            assert layer_grad(dgamma=20 * P, dbeta=20 * P + at) == want, at
            assert layer_grad(gamma=20 * P, dbeta=20 * P + at) == want and layer_grad(gamma=20 * P, dgamma=None, dbeta=20 * P + at) == want, at
            if at:
                assert layer_grad(gamma=20 * P, dgamma=20 * P + at) == want and layer_grad(gamma=20 * P, dgamma=20 * P + at, dbeta=None) == want, at


@no_device
def test_layer_norm_gradient_in_the_weight_s_place():
    assert layer_grad(gamma=20 * P, dgamma=20 * P) == LAUNCH and layer_grad(gamma=None, dgamma=20 * P, dbeta=20 * P + 32) == LAUNCH
