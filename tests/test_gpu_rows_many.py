"""Row-wise operators where a block, a team of threads or a warp has many rows or heads in turn: every form of the kernels with its loop
going round, rows that begin at different places of 16 bytes, arrays with strides of their own, and rows too wide to be held on chip.
Tolerances as in test_gpu_rms_norm.py and test_gpu_rotary.py."""
import pytest
import torch

from anode_b200 import ops
from tests import test_gpu_rms_norm as norm
from tests import test_gpu_rotary as turn
from tests.test_gpu_rms_norm import EPS, make, saved, weights

pytestmark = pytest.mark.gpu

# rows, cols: by the slots of 16 bytes of a row (up to 32, up to 127, up to 2048, more), whole and ragged, several rows to each team
MANY = [(40000, 32), (25000, 33), (20000, 200), (12000, 257), (5000, 640), (5001, 643), (2500, 1536), (2500, 1535), (1300, 5000), (1301, 5003), (700, 9001), (400, 10240), (500, 16384)]
F32 = [(500, 12288), (500, 12289), (300, 16380), (301, 16381)]


def _cases():
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        for rows, cols in MANY + (F32 if dtype is torch.float32 else []):
            yield pytest.param(rows, cols, dtype, id="%d-%d-%s" % (rows, cols, str(dtype).split(".")[1]))


CASES = list(_cases())


@pytest.mark.parametrize("rows, cols, dtype", CASES)
def test_norm_of_many_rows(rows, cols, dtype):
    x, res, gamma = make(rows, cols, dtype, 1), make(rows, cols, dtype, 2), weights(cols, dtype)
    y, total, inv = torch.empty_like(x), torch.empty_like(x), torch.empty(rows, device="cuda")
    ops.RmsNormalizeAddOp.apply(EPS, x, y, gamma, res, total, inv)
    norm.check_forward(x, res, gamma, y, total, inv)
    ops.RmsNormalizeAddOp.apply(EPS, x, y, gamma)
    norm.check_forward(x, None, gamma, y, None, None)
    dy, t, r, dt = saved(rows, cols, dtype)
    dx, dg = torch.empty_like(dy), torch.empty_like(gamma)
    for extra in (dt, None):
        ops.RmsNormalizeAddOp.adjoint(dy, t, r, dx, gamma, extra, dg)
        norm.check_backward(dy, t, r, gamma, extra, dx, dg)
    z, again = dy.clone(), torch.empty_like(dg)
    ops.RmsNormalizeAddOp.adjoint(z, t, r, z, gamma, None, again)
    assert torch.equal(z, dx) and torch.equal(again, dg)


@pytest.mark.parametrize("rows, cols, dtype", CASES)
def test_eight_bits_of_many_rows(rows, cols, dtype):
    x, res, gamma = make(rows, cols, dtype, 5), make(rows, cols, dtype, 6), weights(cols, torch.float32)
    for shape in ((rows,), (rows, -(-cols // 128))):
        q, scale, total = torch.empty(rows, cols, device="cuda", dtype=torch.float8_e4m3fn), torch.empty(shape, device="cuda"), torch.empty_like(x)
        ops.RmsNormalizeAddQuantOp.apply(EPS, x, q, scale, gamma, res, total)
        t = (x.float() + res.float()).to(dtype)
        assert torch.equal(total, t)
        t = t.double()
        y = t * (t.square().mean(-1, keepdim=True) + EPS).rsqrt() * gamma.double()
        groups = -(-cols // 128) if len(shape) == 2 else 1
        width = 128 if len(shape) == 2 else cols
        padded = torch.nn.functional.pad(y, (0, groups * width - cols)).view(rows, groups, width)
        want = padded.abs().amax(2).clamp(min=2.0 ** -96) / 448
        d = norm.row_bound(cols) + 4 * norm.U
        norm.near(scale.view(rows, groups), want, want * d, "scale")
        v = (padded / want.unsqueeze(2)).view(rows, groups * width)[:, :cols]
        nearest = norm.e4m3(v)
        norm.near(q, v, (nearest - v).abs() + 2 * (d + 4 * norm.U) * v.abs(), "q")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("cols, strides", [(1000, (1001, 1009, 1017, 1025)), (1000, (1000, 1008, 1016, 1040)), (1000, (1000, 1001, 1002, 1003)), (77, (80, 88, 96, 104))])
def test_arrays_of_different_strides(cols, strides, dtype):
    """In step with each other (they differ by whole 16 bytes), and not."""
    rows = 3000
    wide = [make(rows, s, dtype, i) for i, s in enumerate(strides)]
    x, res, y, total = (w[:, :cols] for w in wide)
    gamma = weights(cols, dtype)
    beside = [w[:, cols:].clone() for w in wide]
    ops.RmsNormalizeAddOp.apply(EPS, x, y, gamma, res, total)
    norm.check_forward(x, res, gamma, y, total, None)
    dy, t, dt, dx = x, total, res, y
    r = (t.double().square().mean(-1) + EPS).rsqrt().float()
    dg = torch.empty_like(gamma)
    ops.RmsNormalizeAddOp.adjoint(dy, t, r, dx, gamma, dt, dg)
    norm.check_backward(dy, t, r, gamma, dt, dx, dg)
    assert all(torch.equal(a, w[:, cols:]) for a, w in zip(beside, wide))


HEADS = [(9000, 3, 1, 16, 16), (6000, 5, 2, 40, 20), (1500, 32, 8, 128, 62), (1500, 32, 8, 128, 128), (3000, 8, 1, 80, 80), (4000, 6, 6, 96, 48), (2000, 4, 4, 256, 256),
         (700, 7, 3, 192, 96), (400, 3, 2, 1000, 500), (300, 2, 1, 1024, 1024), (20000, 1, 1, 64, 64), (2500, 65, 1, 64, 30)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("tokens, heads, kv, dim, rot", HEADS)
def test_heads_of_many_tokens(tokens, heads, kv, dim, rot, dtype):
    freq = ops.rotary_frequencies(rot)
    positions = torch.arange(tokens, device="cuda", dtype=torch.int32) + 5
    for interleaved, eps in ((False, EPS), (True, None), (True, EPS)):
        both, dboth = turn.normal(tokens, heads + 2 * kv, dim, dtype=dtype, seed=1), turn.normal(tokens, heads + 2 * kv, dim, dtype=dtype, seed=2)
        (q, k), (dqo, dko) = ((b[:, :heads], b[:, heads:heads + kv]) for b in (both, dboth))
        gq, gk = ((1 + 0.2 * turn.normal(dim, seed=s)).to(dtype) for s in (3, 4)) if eps else (None, None)
        out = [torch.empty(t.shape, device="cuda", dtype=dtype) for t in (q, k, q, k)]
        dg = [torch.empty_like(gq) for _ in "qk"] if eps else []
        ops.RotaryPositionsOp.apply(positions, freq, q, k, *out[:2], interleaved, 1.0, eps, gq, gk)
        for x, y, g in ((q, out[0], gq), (k, out[1], gk)):
            turn.check_forward(x, y, positions, freq, interleaved, 1.0, eps is not None, g, "forward ")
        ops.RotaryPositionsOp.adjoint(positions, freq, dqo, dko, *out[2:], interleaved, 1.0, eps, *((q, k, gq, gk, *dg) if eps else ()))
        for d, x, dx, g, s in ((dqo, q, out[2], gq, dg[:1]), (dko, k, out[3], gk, dg[1:])):
            turn.check_backward(d, x, dx, s[0] if s else None, positions, freq, interleaved, 1.0, eps is not None, g, "adjoint ")


@pytest.mark.parametrize("rot", [128, 62])
def test_a_packed_projection_in_its_own_place(rot):
    """Queries and keys turned where they lie, values beside them left alone; forward and back."""
    tokens, heads, kv, dim = 700, 12, 3, 128
    freq, positions = ops.rotary_frequencies(rot), torch.arange(tokens, device="cuda") + 9
    packed = turn.normal(tokens, heads + 2 * kv, dim, dtype=torch.bfloat16, seed=1)
    gq, gk = (1 + 0.2 * turn.normal(dim, seed=s) for s in (3, 4))
    before = packed.clone()
    q, k, v = packed.split((heads, kv, kv), 1)
    ops.RotaryPositionsOp.apply(positions, freq, q, k, q, k, False, 1.0, EPS, gq, gk)
    for x, y, g in ((before[:, :heads], q, gq), (before[:, heads:heads + kv], k, gk)):
        turn.check_forward(x, y, positions, freq, False, 1.0, True, g, "in place ")
    assert torch.equal(v, before[:, heads + kv:])
    grad = turn.normal(tokens, heads + 2 * kv, dim, dtype=torch.bfloat16, seed=2)
    given = grad.clone()
    dq, dk, dv = grad.split((heads, kv, kv), 1)
    x, dgq, dgk = before.split((heads, kv, kv), 1), torch.empty_like(gq), torch.empty_like(gk)
    ops.RotaryPositionsOp.adjoint(positions, freq, dq, dk, dq, dk, False, 1.0, EPS, x[0], x[1], gq, gk, dgq, dgk)
    for d, i, dx, g, dg in ((given[:, :heads], x[0], dq, gq, dgq), (given[:, heads:heads + kv], x[1], dk, gk, dgk)):
        turn.check_backward(d, i, dx, dg, positions, freq, False, 1.0, True, g, "in place ")
    assert torch.equal(dv, given[:, heads + kv:])


CAPTURED_FIRST = """
import torch
from anode_b200 import ops
x, r, g = torch.randn(700, 1536, device="cuda").bfloat16(), torch.randn(700, 1536, device="cuda").bfloat16(), torch.ones(1536, device="cuda")
y, t, inv, dx, dg = torch.empty_like(x), torch.empty_like(x), torch.empty(700, device="cuda"), torch.empty_like(x), torch.empty_like(g)
q, s = torch.empty(700, 1536, device="cuda", dtype=torch.float8_e4m3fn), torch.empty(700, 12, device="cuda")
h, pos, freq = x.view(700, 12, 128), torch.arange(700, device="cuda"), ops.rotary_frequencies(128)
ho, dh, w, dw = torch.empty_like(h), torch.empty_like(h), torch.ones(128, device="cuda"), torch.empty(128, device="cuda")
def step():
    ops.RmsNormalizeAddOp.apply(1e-5, x, y, g, r, t, inv)
    ops.RmsNormalizeAddOp.adjoint(y, t, inv, dx, g, r, dg)
    ops.RmsNormalizeAddQuantOp.apply(1e-5, x, q, s, g, r)
    ops.RotaryPositionsOp.apply(pos, freq, h, None, ho, None, False, 1.0, 1e-5, w)
    ops.RotaryPositionsOp.adjoint(pos, freq, ho, None, dh, None, False, 1.0, 1e-5, h, None, w, None, dw)
graph = torch.cuda.CUDAGraph()
torch.cuda.synchronize()
with torch.cuda.graph(graph):
    step()
graph.replay()
torch.cuda.synchronize()
got = [o.clone() for o in (y, t, inv, dx, dg, q.float(), s, ho, dh, dw)]
step()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, (y, t, inv, dx, dg, q.float(), s, ho, dh, dw)))
print("captured first")
"""


def test_a_process_whose_first_calls_are_captured():
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", CAPTURED_FIRST], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured first" in r.stdout, r.stdout + r.stderr


def test_calls_from_several_threads():
    """The interpreter's lock is given back during a call: threads on streams of their own, each result as alone."""
    import threading
    x, res, gamma = make(500, 1000, torch.float16, 1), make(500, 1000, torch.float16, 2), weights(1000, torch.float16)
    want, total, inv = torch.empty_like(x), torch.empty_like(x), torch.empty(500, device="cuda")
    ops.RmsNormalizeAddOp.apply(EPS, x, want, gamma, res, total, inv)
    dx, dg = torch.empty_like(x), torch.empty_like(gamma)
    ops.RmsNormalizeAddOp.adjoint(want, total, inv, dx, gamma, res, dg)
    torch.cuda.synchronize()
    bad = []

    def work():
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                y, t, i, d, w = torch.empty_like(x), torch.empty_like(x), torch.empty(500, device="cuda"), torch.empty_like(x), torch.empty_like(gamma)
                ops.RmsNormalizeAddOp.apply(EPS, x, y, gamma, res, t, i)
                ops.RmsNormalizeAddOp.adjoint(y, t, i, d, gamma, res, w)
                torch.cuda.current_stream().synchronize()
                if not (torch.equal(y, want) and torch.equal(d, dx) and torch.equal(w, dg)):
                    bad.append(1)
    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad
