"""The table's gradient where the count of tokens to a piece changes, and where runs of one token are as long as a piece, or one shorter or longer: whole numbers whose sums are
exact, so that no row may be missing or come twice."""
import pytest
import torch

from anode_b200 import ops

pytestmark = pytest.mark.gpu


def check(tokens, cols, dtype, sums, vocab=997):
    dy = torch.randint(-2, 3, (len(tokens), cols), generator=torch.Generator(device="cuda").manual_seed(len(tokens)), device="cuda").to(dtype)
    inside = (tokens >= 0) & (tokens < vocab)
    want = torch.zeros(vocab, cols, device="cuda").index_add_(0, tokens[inside], dy[inside].float())
    out = torch.full((vocab, cols), 7.0, device="cuda", dtype=sums)
    ops.EmbedTokensOp.adjoint(tokens, dy, out)
    assert torch.equal(out, want.to(sums))
    added = torch.ones(vocab, cols, device="cuda", dtype=torch.float32)
    ops.EmbedTokensOp.adjoint(tokens, dy, added, 1.0, ops.WriteCap.Accumulate)
    assert torch.equal(added, want + 1)


# 148 blocks twice (three times for 1001), of as many pieces as they have: the last count of tokens with 7, 8, 9, 15, 16 and 17 places to each, and the first beyond
@pytest.mark.parametrize("cols, at_once", [(1024, 592), (1001, 444), (2048, 296), (333, 1184), (520, 592)])
@pytest.mark.parametrize("places", [7, 8, 9, 15, 16, 17])
def test_counts_of_tokens_where_the_piece_changes(cols, at_once, places):
    g = torch.Generator(device="cuda").manual_seed(places)
    for n in (places * at_once, places * at_once + 1):
        u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
        check((998 ** u - 1).long().clamp(0, 996), cols, torch.float16, torch.float32)
        check((u * 1000).long(), cols, torch.bfloat16, torch.bfloat16)


@pytest.mark.parametrize("cols", [8, 40, 1001, 1024, 5001])
@pytest.mark.parametrize("run", [1, 7, 8, 9, 10, 11, 14, 15, 16, 17, 31, 32, 33, 64, 65])
def test_runs_about_as_long_as_a_piece(cols, run):
    for n in (run, 5 * run + 3, 900):
        for first in (0, 5):             # runs from a piece's border on, and across it
            i = torch.arange(n, device="cuda")
            tokens = (i + first) // run
            order = torch.randperm(n, generator=torch.Generator(device="cuda").manual_seed(run), device="cuda")
            check(tokens[order], cols, torch.float16, torch.float32)
