"""Outputs that share memory with one another, or with an input whose place they may not have, are refused, on any machine, and those that lie beside one another are
not.  Nothing of a refused call reaches CUDA: addresses here are numbers that no kernel may see."""
import itertools

import pytest
import torch

from tests.test_more_row_refusals import P, STRIDE, probs

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
