"""Linear attention and token log probabilities as a decision loop runs them: padded
prompts, the readout of their last tokens, the chosen tokens fed back one at a time (one
row ends early), and the same step captured and replayed. Against 64 bits on the
tokens that the run chose.

Tolerance. An attention output is off by at most e = tol * size (test_linear_attention);
a logit sum w o then by d = |w| . (e + 2^-24 (8 + 6 sqrt(n)) |o|), n its terms. A log
probability moves by at most 2 max d and the entropy by 2 H max d, next to
token_log_probs' own errors (test_token_log_probs). The list is compared by the log
probabilities of the tokens it names, which are off by as much.
"""
import numpy as np
import pytest

import tenferro_ext as te
from tenferro_ext.workloads import Lcg
from test_linear_attention import cuda, host, reference as attention
from test_token_log_probs import reference as readout

R, L, H, HK, DK, DV, VOCAB, STEPS, TOP = 5, 90, 4, 2, 64, 32, 1003, 4, 3
LENGTHS = (90, 1, 64, 0, 37)  # of the prompts, padded on the left
ENDED = (1, 2)  # this row's input from this step on is masked


class Model:
    """A layer whose queries, keys, values and gates are tables by token."""

    def __init__(self, bf16):
        rng = Lcg(11)
        normal = lambda *s: rng.normal(int(np.prod(s))).astype(np.float32).reshape(s)
        unit = lambda x: x / np.sqrt((x * x).sum(2, keepdims=True))
        rounded = lambda x: te.bf16_bits_to_f32(te.to_bf16_bits(x)) if bf16 else x
        self.bf16 = bf16
        self.q, self.k = rounded(unit(normal(VOCAB, HK, DK))), rounded(unit(normal(VOCAB, HK, DK)))
        self.v = rounded(normal(VOCAB, H, DV))
        self.g = -np.abs(normal(VOCAB, H))
        self.beta = (1 / (1 + np.exp(-normal(VOCAB, H)))).astype(np.float32)
        self.w = normal(VOCAB, H * DV) / np.float32(4)  # logits = w out
        # int16, which torch can index.
        bits = (lambda x: te.to_bf16_bits(x).view(np.int16)) if bf16 else lambda x: x
        self.dev = [cuda(x) for x in (bits(self.q), bits(self.k), bits(self.v), self.g, self.beta,
                                      self.w)]

    def operands(self, tokens):
        """tokens (R, n) on the GPU -> flat q, k, v, g, beta with the tokens fastest."""
        return [x[tokens].movedim(1, -1).contiguous().view(-1) for x in self.dev[:5]]

    def logits(self, last):
        """last (R, H * DV) -> (R, VOCAB)."""
        return last @ self.dev[5].T


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
def test_prompt_readout_and_steps(bf16):
    import torch

    model = Model(bf16)
    tokens = np.zeros((R, L + STEPS), np.int64)
    mask = np.zeros((R, L + STEPS), np.float32)
    tokens[:, :L] = Lcg(29).integers(0, VOCAB - 1, R * L).reshape(R, L)
    for r, n in enumerate(LENGTHS):
        mask[r, L - n:] = 1.0
    mask[ENDED[0], L + ENDED[1]:] = 0.0
    marks = np.array([[4, -1, VOCAB - 1]] * R)
    stream = torch.cuda.Stream()
    got, outs = [], []
    with te.Context(0, stream=stream.cuda_stream) as ctx, torch.cuda.stream(stream):
        out, state = te.jeff_linear_attention_rows(
            *model.operands(cuda(tokens[:, :L])), cuda(mask[:, :L].reshape(-1)), R, L, H, HK, DK,
            DV, bf16=bf16, ctx=ctx)
        slots = cuda(marks.reshape(-1))

        def answer(last):
            x = model.logits(last)
            return te.token_log_probs(x.reshape(-1), slots, R, VOCAB, top=TOP, ctx=ctx)

        last = out.view(R, H * DV, L)[:, :, L - 1].contiguous()
        got.append([host(x) for x in answer(last)])
        outs.append(host(last))

        # One step, eager and as a graph that reads its inputs from the same tensors.
        token, on = cuda(tokens[:, :1]), cuda(mask[:, :1].reshape(-1))

        def step():
            ops = model.operands(token)
            last = te.jeff_linear_attention_step(*ops, state, R, H, HK, DK, DV, mask=on,
                                                 bf16=bf16, ctx=ctx)
            return last.view(R, -1), answer(last.view(R, -1))

        saved = state.clone()
        with te.asynchronous():
            step()
            state.copy_(saved)
            stream.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                replayed = step()
        for s in range(STEPS):
            tokens[:, L + s] = got[-1][2].reshape(R, TOP)[:, 0]  # the most likely one
            token.copy_(cuda(tokens[:, L + s:L + s + 1])), on.copy_(cuda(mask[:, L + s]))
            before = state.clone()
            eager = step()
            got.append([host(x) for x in eager[1]])
            outs.append(host(eager[0]))
            after = host(state)
            state.copy_(before)
            graph.replay()
            stream.synchronize()
            for a, b in zip((replayed[0], *replayed[1]), (outs[-1], *got[-1])):
                assert np.array_equal(host(a), b)
            assert np.array_equal(host(state), after)

    at = lambda x: np.moveaxis(x[tokens], 1, -1)
    want, S, size, A = attention(at(model.q), at(model.k), at(model.v), at(model.g),
                                 at(model.beta), mask, float(np.float32(DK ** -0.5)), None)
    tol = 2.0 ** -24 * (8 + 6 * np.sqrt(DK + 64 + L + STEPS))
    assert (np.abs(after.reshape(S.shape) - S) <= tol * A).all()
    w, n = model.w.astype(np.float64), H * DV
    own = 2.0 ** -24 * (17 + 6 * np.sqrt(VOCAB / 64 + 1))
    for s in range(STEPS + 1):
        o = want[..., L - 1 + s].reshape(R, n)
        e = tol * size[..., L - 1 + s].reshape(R, n)
        assert (np.abs(outs[s] - o) <= e).all()
        x = o @ w.T
        d = ((e + 2.0 ** -24 * (8 + 6 * np.sqrt(n)) * np.abs(o)) @ np.abs(w).T).max(
            1, keepdims=True)
        lp, entropy, order, top_lp, far = readout(x, marks, TOP)
        near = lambda a, b, t: (np.abs(a.reshape(b.shape) - b) <= t + 2.0 ** -22 * np.abs(b)).all()
        assert near(got[s][0], lp, 2 * d + own) and (got[s][0].reshape(R, 3)[:, 1] == 0).all()
        assert near(got[s][1], entropy, (2 * entropy * d[:, 0] + own * (1 + far)))
        assert near(got[s][3], top_lp, 2 * d + own)
        chosen = got[s][2].reshape(R, TOP)
        assert all(len(set(c)) == TOP for c in chosen)
        assert near(got[s][3], readout(x, chosen, TOP)[0], 2 * d + own)
    # The ended row kept its state, the empty prompt began with a uniform answer.
    np.testing.assert_array_equal(outs[1 + ENDED[1]][ENDED[0]], 0)
    assert np.array_equal(got[0][2].reshape(R, TOP)[3], np.arange(TOP))


@pytest.mark.gpu
def test_two_contexts_at_once():
    """Prompts and readouts of two contexts on two streams, in flight together: each
    has its own workspaces, so the results are those of either alone."""
    import torch

    def problem(seed, rows, length, heads, dk, dv, vocab):
        rng = Lcg(seed)
        normal = lambda *s: cuda(rng.normal(int(np.prod(s))).astype(np.float32))
        dims = (rows, length, heads, heads, dk, dv)
        kv = [normal(rows, heads, n, length) / np.sqrt(dk) for n in (dk, dk, dv)]
        gates = [-normal(rows, heads, length).abs(), torch.sigmoid(normal(rows, heads, length))]
        logits = normal(rows * heads, vocab)

        def run(ctx):
            out, state = te.jeff_linear_attention_rows(*kv, *gates, None, *dims, ctx=ctx)
            return (out, state, *te.token_log_probs(logits, None, rows * heads, vocab, top=4,
                                                    ctx=ctx)[1:])
        return run

    runs = [problem(3, 2, 700, 8, 128, 128, 70001), problem(4, 24, 200, 8, 64, 96, 50000)]
    streams = [torch.cuda.Stream() for _ in runs]
    with te.Context(0, stream=streams[0].cuda_stream) as a, \
            te.Context(0, stream=streams[1].cuda_stream) as b:
        alone = []
        for run, ctx, stream in zip(runs, (a, b), streams):
            with torch.cuda.stream(stream):
                alone.append([host(x) for x in run(ctx)])
        torch.cuda.synchronize()
        together = [[], []]
        with te.asynchronous():
            for _ in range(6):
                for i, (run, ctx, stream) in enumerate(zip(runs, (a, b), streams)):
                    with torch.cuda.stream(stream):
                        together[i].append(run(ctx))
        torch.cuda.synchronize()
    for want, tries in zip(alone, together):
        for got in tries:
            assert all(np.array_equal(host(x), y) for x, y in zip(got, want))


@pytest.mark.gpu
def test_operands_that_are_parameters(gpu_ctx, monkeypatch):
    """A program whose first call passes a module's parameters and nothing else."""
    import torch

    rng = Lcg(17)
    param = lambda *s: torch.nn.Parameter(cuda(rng.normal(int(np.prod(s))).astype(np.float32)),
                                          requires_grad=False)
    q, k, v, state = param(2, 8), param(2, 8), param(2, 4), param(2, 8, 4)
    g, beta, logits = param(2), param(2), param(3, 50)
    g.neg_().sub_(3), beta.sigmoid_()
    ops = [x.data.view(-1) for x in (q, k, v, g, beta)]
    want, after = te.jeff_linear_attention_rows(*ops, None, 1, 1, 2, 2, 8, 4,
                                                state=state.data.view(-1), ctx=gpu_ctx)
    marks = te.token_log_probs(logits.data.view(-1), None, 3, 50, top=3, ctx=gpu_ctx)
    monkeypatch.setattr(te, "_torch_types", {})
    out, new = te.jeff_linear_attention_rows(q, k, v, g, beta, None, 1, 1, 2, 2, 8, 4, state=state,
                                             ctx=gpu_ctx)
    assert torch.equal(out, want) and torch.equal(new, after)
    monkeypatch.setattr(te, "_torch_types", {})
    got = te.token_log_probs(logits, None, 3, 50, top=3, ctx=gpu_ctx)
    assert got.log_probs is None
    assert all(torch.equal(a, b) for a, b in zip(got[1:], marks[1:]))
