"""From tokens to their log probabilities and back as a language model's step has them: rows of a table with a scale, layers' norms with the residual stream, the
tied table as the last projection, log probabilities with entropies, and the gradients' way back; serving the same step token by token; the calls captured, on
streams of their own, from several threads, and on workspaces of the caller's.  The products are torch's."""
import os
import subprocess
import sys
import threading

import pytest
import torch

from anode_b200 import ops

pytestmark = pytest.mark.gpu


def normal(*s, seed=0, dtype=torch.float32, scale=1.0):
    return (torch.randn(*s, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda") * scale).to(dtype)


def ids(n, vocab, seed=0):
    return torch.randint(0, vocab, (n,), generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def test_a_step_of_training():
    """float32 against autograd in float64.  Products over 96 and 211 terms in f32 (sums of terms of size one, off by sqrt(n)*2^-24 each, 1e-6) and the operators'
    own 1e-6 give gradients within 1e-4 of the largest; a wrong formula is off by its size."""
    vocab, cols, n, scale = 211, 96, 120, 96 ** 0.5
    tokens = ids(n, vocab, 1)
    tokens[5:9] = -1                                        # padding
    targets = torch.where(ids(n, 10, 2) == 0, -100, ids(n, vocab, 3))
    embed, norms, probs = ops.TokenEmbedding(vocab, cols, scale), [ops.LayerNormAdd(cols), ops.LayerNormAdd(cols, bias=False)], ops.TokenLogProbs(0.8)
    embed.table.copy_(normal(vocab, cols, seed=4, scale=cols ** -0.5))
    for i, layer in enumerate(norms):
        layer.gamma.copy_(1 + 0.2 * normal(cols, seed=5 + i))
    norms[0].beta.copy_(0.2 * normal(cols, seed=7))
    weight, w, v = normal(cols, cols, seed=8, scale=cols ** -0.5), normal(n, seed=9), normal(n, seed=10)

    x = embed.forward(tokens)
    y, total = norms[0].forward(x)
    z, total = norms[1].forward(y @ weight, total)
    logits = z @ embed.table.t()
    logprob, entropy = probs.forward(logits, targets)
    dlogits = probs.backward(w, v)
    dtied = dlogits.t() @ z
    dsum = norms[1].backward(dlogits @ embed.table)         # of y @ weight, and of the stream
    dweight = y.t() @ dsum
    dx = norms[0].backward(dsum @ weight.t(), dsum)
    embed.dtable.copy_(dtied)
    embed.backward(dx, ops.WriteCap.Accumulate)

    leaves = [t.double().requires_grad_() for t in (embed.table, norms[0].gamma, norms[0].beta, norms[1].gamma, weight)]
    E, G0, B0, G1, W = leaves

    def layer(t, gamma, beta, eps):
        c = t - t.mean(-1, keepdim=True)
        return c * (c.square().mean(-1, keepdim=True) + eps).rsqrt() * gamma + beta
    X = torch.where((tokens >= 0)[:, None], scale * E[tokens.clamp(min=0)], 0.0)
    Z = layer(X + layer(X, G0, B0, norms[0].epsilon) @ W, G1, 0.0, norms[1].epsilon)
    lp = torch.log_softmax(0.8 * (Z @ E.t()), 1)
    picked = torch.where(targets >= 0, lp.gather(1, targets.clamp(min=0)[:, None])[:, 0], 0.0)
    H = -(lp.exp() * lp).sum(1)
    ((picked * w.double()).sum() + (H * v.double()).sum()).backward()
    for what, got, want in (("logprob", logprob, picked), ("entropy", entropy, H), ("table", embed.dtable, E.grad), ("gamma", norms[0].dgamma, G0.grad),
                            ("beta", norms[0].dbeta, B0.grad), ("gamma of the second", norms[1].dgamma, G1.grad), ("weight", dweight, W.grad)):
        off = (got.double() - want).abs().max() / want.abs().max()
        assert off < 1e-4, (what, float(off))


def test_serving_token_by_token():
    """Rows on their own give what they give among others: the table's rows and the norms bit for bit, log probabilities to their tolerance, the likeliest tokens the same."""
    vocab, cols, n = 4096, 512, 9
    embed, norm, probs = ops.TokenEmbedding(vocab, cols, 8.0, dtype=torch.bfloat16), ops.LayerNormAdd(cols, dtype=torch.bfloat16), ops.TokenLogProbs(1.25)
    embed.table.copy_(normal(vocab, cols, seed=1))
    tokens, res = ids(n, vocab, 2), normal(n, cols, seed=3, dtype=torch.bfloat16)
    x = embed.infer(tokens)
    y, total = norm.infer(x, res)
    logits = normal(n, vocab, seed=4, dtype=torch.bfloat16, scale=3.0)
    logprob, entropy, best, best_token = probs.infer(logits, tokens, 20, True)
    for t in range(n):
        assert torch.equal(embed.infer(tokens[t:t + 1])[0], x[t])
        one = norm.infer(x[t], res[t])
        assert torch.equal(one[0], y[t]) and torch.equal(one[1], total[t])
        alone = probs.infer(logits[t:t + 1], tokens[t:t + 1], 20, True)
        assert torch.equal(alone[3][0], best_token[t])
        # (a row may be shared out in other ways; each way is within the tolerance of the formula, 2e-5 at these sizes)
        for a, b in zip(alone[:3], (logprob, entropy, best)):
            assert ((a[0] - b[t]).abs() <= 4e-5).all()


def calls(vocab=3001, cols=264, n=700, dtype=torch.bfloat16, seed=0):
    """Inputs of every call, and a function that makes them all on a stream and gives the outputs."""
    s = dict(x=normal(n, cols, seed=seed, dtype=dtype), res=normal(n, cols, seed=seed + 1, dtype=dtype), dy=normal(n, cols, seed=seed + 2, dtype=dtype),
             gamma=1 + 0.1 * normal(cols, seed=seed + 3), beta=normal(cols, seed=seed + 4), table=normal(vocab, cols, seed=seed + 5, dtype=dtype),
             tokens=ids(n, vocab // 10, seed + 6), logits=normal(n, vocab, seed=seed + 7, dtype=dtype, scale=3.0), w=normal(n, seed=seed + 8), v=normal(n, seed=seed + 9))

    def step(s=s, stream=None, spaces=(None, None)):
        f = lambda *z: torch.empty(*z, device="cuda")      # noqa: E731
        y, total, dx, e = (torch.empty_like(s["x"]) for _ in range(4))
        mean, inv, dg, db, lp, h, stats = f(n), f(n), f(cols), f(cols), f(n), f(n), f(n, 2)
        dt, dtable, dlogits, best, best_token = torch.empty_like(s["table"]), f(vocab, cols), torch.empty_like(s["logits"]), f(n, 8), torch.empty(n, 8, device="cuda", dtype=torch.int64)
        ops.LayerNormalizeAddOp.apply(1e-5, s["x"], y, s["gamma"], s["beta"], s["res"], total, mean, inv, stream=stream)
        ops.LayerNormalizeAddOp.adjoint(s["dy"], total, mean, inv, dx, s["gamma"], y, dg, db, workspace=spaces[0], stream=stream)
        ops.EmbedTokensOp.apply(s["tokens"], s["table"], e, 2.0, stream=stream)
        ops.EmbedTokensOp.adjoint(s["tokens"], s["dy"], dt, 0.5, workspace=spaces[1], stream=stream)
        ops.EmbedTokensOp.adjoint(s["tokens"], s["dy"], dtable, 0.5, workspace=spaces[1], stream=stream)
        ops.EmbedTokensOp.adjoint(s["tokens"], dx, dtable, 2.0, ops.WriteCap.Accumulate, workspace=spaces[1], stream=stream)
        ops.TokenLogProbsOp.apply(s["logits"], s["tokens"], lp, h, stats, best, best_token, 0.9, stream=stream)
        ops.TokenLogProbsOp.adjoint(s["logits"], s["tokens"], stats, s["w"], dlogits, h, s["v"], 0.9, stream=stream)
        return y, total, mean, inv, dx, dg, db, e, dt, dtable, lp, h, stats, best, best_token, dlogits
    return s, step


def same(a, b):
    return all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize("n", [700, 9000])
def test_streams_graphs_and_calls_at_once(n):
    (one, step), (two, _) = calls(n=n), calls(n=n, seed=50)
    want = [step(s) for s in (one, two)]
    torch.cuda.synchronize()
    other, third = torch.cuda.Stream(), torch.cuda.Stream()
    outs = []
    for _ in range(3):
        other.wait_stream(torch.cuda.current_stream())
        third.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(third):
            b = step(two)
        outs.append((step(one, other), b))
    torch.cuda.synchronize()
    assert all(same(a, want[0]) and same(b, want[1]) for a, b in outs)
    # captured, with workspaces of the caller's and without, and replayed on other inputs
    rows, cols, vocab = one["x"].shape + one["table"].shape[:1]
    spaces = [torch.full((b,), 255, device="cuda", dtype=torch.uint8) for b in (ops.layer_norm_workspace_bytes(rows, cols), ops.embed_workspace_bytes(rows, vocab, cols))]
    inputs = [{k: t.clone() for k, t in one.items()} for _ in range(2)]
    graphs, results = [], []
    for w, inp in zip((spaces, (None, None)), inputs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            results.append(step(inp, None, w))
        graphs.append(g)
    for s, inp in zip((two, one), inputs):
        for k, t in inp.items():
            t.copy_(s[k])
    for _ in range(2):
        for g in graphs:
            g.replay()
    torch.cuda.synchronize()
    assert same(results[0], want[1]) and same(results[1], want[0])


def test_calls_from_several_threads():
    s, step = calls(n=500)
    want = step()
    torch.cuda.synchronize()
    bad = []

    def work():
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = step()
                torch.cuda.current_stream().synchronize()
                if not same(got, want):
                    bad.append(1)
    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


CAPTURED_FIRST = """
import torch
from tests.test_gpu_tokens_together import calls, same
s, step = calls(n=9000)
graph = torch.cuda.CUDAGraph()
torch.cuda.synchronize()
with torch.cuda.graph(graph):
    got = step()
graph.replay()
torch.cuda.synchronize()
assert same([o.clone() for o in got], step())
print("captured first")
"""


def test_a_process_whose_first_calls_are_captured():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", CAPTURED_FIRST], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured first" in r.stdout, r.stdout + r.stderr


@pytest.mark.parametrize("shape, cut", [((0, 3, 4, 8), (slice(None), slice(None), slice(0, 2))), ((3, 0, 4, 8), (slice(0, 2), slice(None), slice(1, 3))),
                                        ((2, 3, 4, 8), (slice(0, 0), slice(0, 2), slice(0, 3)))])
def test_slices_without_rows(shape, cut):
    x = torch.zeros(shape, device="cuda")[cut]
    norm, embed, probs = ops.LayerNormAdd(8), ops.TokenEmbedding(5, 8), ops.TokenLogProbs()
    norm.dgamma.fill_(7), norm.dbeta.fill_(7), embed.dtable.fill_(7)
    y, total = norm.forward(x, x)
    assert y.shape == total.shape == x.shape and norm.backward(x, x).shape == x.shape and (norm.dgamma == 0).all() and (norm.dbeta == 0).all()
    none = torch.zeros(x.shape[:-1], device="cuda", dtype=torch.int64)
    assert embed.forward(none).shape == x.shape and (embed.backward(x) == 0).all()
    logprob, entropy = probs.forward(x, none)
    assert logprob.shape == entropy.shape == x.shape[:-1] and probs.backward(logprob, entropy).shape == x.shape and probs.infer(x, None, 3)[3].shape == x.shape[:-1] + (3,)


def test_accumulating_grows_from_what_is_there():
    """Ten micro-batches of whole numbers into f32 gradients: exact sums."""
    vocab, cols, n = 97, 40, 300
    embed = ops.TokenEmbedding(vocab, cols, dtype=torch.bfloat16, grad_dtype=torch.float32)
    want = torch.zeros(vocab, cols, device="cuda")
    for i in range(10):
        tokens, dy = ids(n, vocab, i), torch.randint(-3, 4, (n, cols), generator=torch.Generator(device="cuda").manual_seed(i), device="cuda").bfloat16()
        embed.forward(tokens)
        embed.backward(dy, ops.WriteCap.Accumulate if i else ops.WriteCap.Assign)
        want.index_add_(0, tokens, dy.float())
    assert torch.equal(embed.dtable, want)


def test_backward_in_the_place_of_what_it_read_is_the_last():
    """The gradient in the logits' or the sum's place leaves a second backward pass nothing to read; elsewhere, and in the incoming gradient's place, it may be repeated."""
    logits, tokens = torch.randn(6, 40, device="cuda"), ids(6, 40, 1)
    probs, w = ops.TokenLogProbs(), torch.ones(6, device="cuda")
    probs.forward(logits, tokens)
    first = probs.backward(w, w).clone()
    assert torch.equal(probs.backward(w, w), first) and torch.equal(probs.backward(w, w, out=logits), first)
    with pytest.raises(RuntimeError, match="backward before forward"):
        probs.backward(w, w)
    probs.forward(torch.randn(6, 40, device="cuda"), tokens)
    probs.backward(w, w)
    norm, x, dy = ops.LayerNormAdd(40), torch.randn(6, 40, device="cuda"), torch.randn(6, 40, device="cuda")
    _, total = norm.forward(x, x)
    dx = norm.backward(dy, total).clone()
    assert torch.equal(norm.backward(dy.clone(), total, out=torch.empty_like(dy)), dx)
    assert torch.equal(norm.backward(dy, total, out=total), dx)
    with pytest.raises(RuntimeError, match="backward before forward"):
        norm.backward(dy)
