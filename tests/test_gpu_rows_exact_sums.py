"""The weights' gradients where every row counts.  The bounds of the other tests grow with the number of rows, so that one row of many could be lost
within them; here the sums are exact, or all of one sign, and nothing may be missing."""
import pytest
import torch

from anode_b200 import ops
from tests.test_gpu_rms_norm import U
from tests.test_gpu_rows_many import F32, HEADS, MANY

pytestmark = pytest.mark.gpu


def integers(rows, cols, seed, dtype):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(1, 4, (rows, cols), generator=g, device="cuda").to(dtype) * (2 * torch.randint(0, 2, (rows, cols), generator=g, device="cuda") - 1).to(dtype)


# (beside the shapes of other tests: as many rows as teams, one more, and one less; rows out of step; a single row)
MORE = [(1, 64), (147, 512), (148, 512), (149, 512), (2367, 256), (2368, 256), (2369, 256), (2047, 1535), (8192, 4096), (3000, 17000)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("rows, cols", MANY + F32 + MORE)
def test_norm(rows, cols, shift, dtype):
    """Products of integers from 1 to 3 with 1/rms = 1: sums below 9*40000 < 2^24 are exact in any order, and no row adds 0."""
    dy, t = integers(rows, cols, 1, dtype), integers(rows, cols, 2, dtype)
    want = (dy.double() * t.double()).sum(0).float()
    dx = torch.empty(rows, cols + 8, device="cuda", dtype=dtype)[:, shift:shift + cols]
    for extra in (None, t):
        dg = torch.full((cols,), 0.5, device="cuda")
        ops.RmsNormalizeAddOp.adjoint(dy, t, torch.ones(rows, device="cuda"), dx, None, extra, dg)
        assert torch.equal(dg, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("tokens, heads, kv, dim, rot", HEADS + [(8192, 32, 8, 128, 128), (1184, 8, 2, 64, 64), (1185, 8, 2, 64, 30)])
def test_rotary(tokens, heads, kv, dim, rot, dtype):
    """Heads of -1 and 1 at position 0 with a norm of rms 1: every term of a sum is 1/rms, as the kernel has it, of a sign that its element has.
    1/rms is within 4u of 1 (two steps); a sum of n equal terms is off by at most u for each step of the chains that it is made of: a warp's heads (no
    warp of a device that the heads fill has more than four times its share), 40 for the warps, blocks and lanes that join."""
    freq, positions = ops.rotary_frequencies(rot), torch.zeros(tokens, device="cuda", dtype=torch.int64)
    warps = 4 * 2 * torch.cuda.get_device_properties(0).multi_processor_count
    for interleaved in (False, True):
        x = [2 * torch.randint(0, 2, (tokens, n, dim), device="cuda", generator=torch.Generator(device="cuda").manual_seed(n + 7)).to(dtype) - 1 for n in (heads, kv)]
        sign = integers(1, dim, 3, dtype).sign()
        d = [sign * t for t in x]
        out, dg = [torch.empty_like(t) for t in x], [torch.empty(dim, device="cuda") for _ in x]
        ops.RotaryPositionsOp.adjoint(positions, freq, *d, *out, interleaved, 1.0, 0.0, *x, None, None, *dg)
        for n, got in zip((heads, kv), dg):
            n *= tokens
            off = (got.double() * sign.double() - n).abs().max()
            assert float(off) <= n * (4 + 4 * n / warps + 40 + 4) * U, (n, float(off))
