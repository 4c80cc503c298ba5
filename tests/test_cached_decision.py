"""The paged 8-bit cache's operators together, as a decision model with a history calls them:
left-padded prompts, single tokens whose next ones are the most likely answers (a row ends
early), a second prompt behind them; and calls of many sizes through one workspace. Each attention
against 64 bits on the codes that the formula leaves, within test_cached_attention's tolerance.
"""
import numpy as np
import pytest

import tenferro_ext as te
from tenferro_ext.workloads import Lcg
from test_cache_append import EPS, Cache
from test_cached_attention import call, check, filled, problem, reference
from test_linear_attention import cuda, host
from test_rotary import normal

R, H, HK, HD, VOCAB = 4, 8, 2, 128, 500
PROMPT, SECOND, STEPS = (70, 1, 33, 64), (1, 0, 90, 5), 4
ENDED = 2  # row 2 has no token after two steps, until the second prompt


class Model:
    """Queries, keys, values and gates of a token by table; tokens' scores by w."""

    def __init__(self, bf16):
        self.bf16 = bf16
        self.q, self.k, self.v, self.gate = (
            normal(s, VOCAB, n * HD) for s, n in ((11, H), (12, HK), (13, HK), (14, H)))
        if bf16:
            self.q, self.k, self.v, self.gate = (
                te.bf16_bits_to_f32(te.to_bf16_bits(x)) for x in (self.q, self.k, self.v, self.gate))
        self.norm = normal(15, HD) * np.float32(0.1)
        self.w = normal(16, H * HD, VOCAB) * np.float32((H * HD) ** -0.5)
        bits = te.to_bf16_bits if bf16 else lambda x: x
        self.tables = [cuda(bits(x).view(np.int16) if bf16 else x)
                       for x in (self.q, self.k, self.v, self.gate)]

    def operands(self, tokens):
        """tokens (R, L) on the device: q, k, v, gate as the calls take them."""
        import torch

        out = [t[tokens.long()].transpose(1, 2).contiguous().reshape(-1) for t in self.tables]
        return [x.view(torch.bfloat16) for x in out] if self.bf16 else out

    def at(self, x, tokens, heads):
        return np.moveaxis(x[tokens], 1, -1).reshape(R, heads, HD, tokens.shape[1])


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
def test_prompt_steps_and_another_prompt(bf16):
    import torch

    model = Model(bf16)
    rotary = te.Rotary(te.rotary_frequencies(64, 1e4), False)
    ref = Cache(R, HK, HD, 64, 5)

    def expected(tokens, counts):
        """The formula's cache moves on; outputs and tolerance on it."""
        k, v = model.at(model.k, tokens, HK), model.at(model.v, tokens, HK)
        before = ref.lengths.astype(np.int64).copy()
        ref.append(k, v, model.norm, rotary, counts)
        return reference(ref, model.at(model.q, tokens, H), model.at(model.gate, tokens, H),
                         model.norm, rotary, before, counts)

    stream = torch.cuda.Stream()
    with te.Context(0, stream=stream.cuda_stream) as ctx, torch.cuda.stream(stream):
        cache, table, norm = ref.paged(cuda), cuda(ref.table.reshape(-1)), cuda(model.norm)
        lengths, w = cuda(np.zeros(R, np.int32)), cuda(model.w)

        def forward(tokens, counts):
            q, k, v, gate = model.operands(tokens)
            L = tokens.shape[1]
            te.jeff_cache_append(k, v, norm, cache, table, lengths, counts, R, L, HK, HD, rotary, EPS,
                                 bf16=bf16, ctx=ctx)
            out = te.jeff_cached_attention(q, gate, norm, cache, table, lengths, counts, R, L, H, HK,
                                           HD, rotary, EPS, bf16=bf16, ctx=ctx)
            lengths.add_(counts)
            last = out.view(R, H * HD, L)[:, :, L - 1].contiguous()
            answer = te.token_log_probs((last @ w).reshape(-1), None, R, VOCAB, top=2, ctx=ctx)
            return out, answer.top_tokens, answer.top_log_probs

        def prompt(counts, seed):
            counts = np.array(counts)
            tokens = Lcg(seed).integers(0, VOCAB - 1, R * counts.max()).reshape(R, -1)
            got = forward(cuda(tokens), cuda(counts.astype(np.int32)))
            check(got[0], *expected(tokens, counts))
            assert ref.same(cache) == [True] * 4
            return host(got[1]).reshape(R, 2)[:, 0]

        chosen = prompt(PROMPT, 3)

        # A step, eager and captured: the graph reads its tokens, counts and lengths where they are.
        token, on = cuda(chosen.reshape(R, 1)), cuda(np.ones(R, np.int32))
        state = [*cache[:4], lengths]
        saved = [x.clone() for x in state]

        def back(to):
            for x, y in zip(state, to):
                x.copy_(y)

        with te.asynchronous():
            forward(token, on)
            back(saved)
            stream.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                replayed = forward(token, on)
        for s in range(STEPS):
            counts = np.ones(R, np.int64)
            if s >= 2:
                counts[ENDED] = 0
            token.copy_(cuda(chosen.reshape(R, 1))), on.copy_(cuda(counts.astype(np.int32)))
            saved = [x.clone() for x in state]
            got = [host(x) for x in forward(token, on)]
            after = [host(x).copy() for x in state]
            back(saved)
            graph.replay()
            stream.synchronize()
            for a, b in zip([*replayed, *state], [*got, *after]):
                assert np.array_equal(host(a).view(np.uint8), b.view(np.uint8))
            want, tol = expected(chosen.reshape(R, 1).astype(np.int64), counts)
            check(got[0], want, tol)
            assert ref.same(cache) == [True] * 4
            if s >= 2:
                np.testing.assert_array_equal(got[0].reshape(R, -1)[ENDED], 0)
            chosen = got[1].reshape(R, 2)[:, 0]
        prompt(SECOND, 9)
        assert np.array_equal(host(lengths), ref.lengths)


@pytest.mark.gpu
def test_queries_turned_before_or_inside(gpu_ctx):
    """rotary_rows and then the attention without positions, against the formula as well."""
    L, before = 20, np.array([100, 3])
    counts = np.array([L, L])
    ref = filled(2, 2, 64, 64, before + counts)
    q, _ = problem(2, 4, 64, L, False, gate=False)
    rotary = te.Rotary(te.rotary_frequencies(48, 1e4), True, 1.5)
    want, tol = reference(ref, q, None, None, rotary, before, counts)
    at = (before[:, None] + np.arange(L)).astype(np.int32)
    turned = te.rotary_rows(cuda(q.reshape(-1)), cuda(at.reshape(-1)), 2, L, 4, 64, rotary, ctx=gpu_ctx)
    check(call(gpu_ctx, ref, host(turned).reshape(q.shape), None, None, None, before, counts), want, tol)
    check(call(gpu_ctx, ref, q, None, None, rotary, before, counts), want, tol)


def shapes():
    """R, H, HK, hd, L, tokens before: few and many columns, one part and many, each width."""
    for hd in (64, 100, 192, 256):
        yield 20, 8, 1, hd, 16, (9000,) + tuple(11 * r for r in range(19))  # 128 columns, 100 parts
    yield 70, 2, 1, 128, 1, (30000,) + tuple(r for r in range(69))  # 1 long of over 64 rows
    yield 300, 4, 2, 64, 1, tuple(7 * r % 2000 for r in range(300))  # more tiles than workgroups
    yield 3, 6, 1, 40, 150, (0, 5000, 63)  # 900 columns
    yield 140, 3, 1, 72, 11, tuple(r for r in range(140))  # 33 columns: over two tiles
    yield 1, 8, 1, 64, 3000, (500,)  # 24000 columns
    yield 5, 3, 3, 1, 4, (0, 63, 64, 300, 1)  # one feature
    yield 2, 200, 1, 64, 2, (70, 600)  # a token's heads over several tiles
    yield 30, 200, 1, 64, 2, tuple(40 * r for r in range(30))
    yield 12, 300, 2, 130, 1, tuple(90 * r for r in range(12))
    yield 40, 16, 1, 2, 9, tuple(3 * r for r in range(40))


@pytest.mark.gpu
@pytest.mark.parametrize("shape", list(shapes()), ids=lambda s: "x".join(map(str, s[:5])))
def test_parts_of_ragged_rows(gpu_ctx, shape):
    R, H, HK, hd, L, before = shape
    before = np.array(before)
    counts = np.array([(L, max(1, L - 3), L, L // 2)[r % 4] for r in range(R)])
    ref = filled(R, HK, hd, 64, before + counts)
    q, gate = problem(R, H, hd, L, True)
    rotary = te.Rotary(te.rotary_frequencies(min(hd & ~1, 64), 1e4))
    want, tol = reference(ref, q, gate, None, rotary, before, counts)
    check(call(gpu_ctx, ref, q, gate, None, rotary, before, counts, True), want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("group", [1, 3, 8])
@pytest.mark.parametrize("L", [2, 3, 5, 9, 17, 33, 131])
def test_runs_of_odd_lengths(gpu_ctx, L, group):
    """Many rows, so that the longer ones take 128 columns at once."""
    R, hd = (3, 33)[L > 8], 48
    before = np.array([(61 + r) * (r % 3) for r in range(R)])
    counts = np.array([L - r % 2 for r in range(R)])
    ref = filled(R, 1, hd, 64, before + counts)
    q, gate = problem(R, group, hd, L, False)
    want, tol = reference(ref, q, gate, None, None, before, counts)
    check(call(gpu_ctx, ref, q, gate, None, None, before, counts), want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("R,L", [(2, 1), (33, 20)])
def test_scales_far_apart(gpu_ctx, R, L):
    """Blocks whose value scales lie up to 2^80 apart in any order, blocks of zeros under the least
    scale, a scale of 0; queries of 2^-60 and of 2^20."""
    hd, before, counts = 64, np.array([64 * 12 + r for r in range(R)]), np.full(R, L)
    ref = filled(R, 1, hd, 64, before + counts)
    e = Lcg(3).integers(-40, 40, ref.vs.size).reshape(ref.vs.shape)
    ref.vs[:] = 2.0 ** e
    for r in range(R):
        first, zero = ref.table[r, 0], ref.table[r, 1 + r % 3]
        ref.vs[first], ref.vs[zero] = (0.0, 2.0**-100) if r % 2 else (2.0**-30, 0.0)
        ref.values[zero] = 0
    q, _ = problem(R, 8, hd, L, False, gate=False)
    q[:, ::2] *= np.float32(2.0**-60)
    q[:, 1] *= np.float32(2.0**20)
    want, tol = reference(ref, q, None, None, None, before, counts)
    check(call(gpu_ctx, ref, q, None, None, None, before, counts), want, tol)


CALLS = [
    # R, H, HK, hd, L, tokens before
    (1, 8, 2, 256, 1, (20000,)),
    (33, 8, 1, 64, 16, (3000,) + tuple(range(32))),
    (5, 6, 3, 96, 3, (0, 700, 90, 64, 63)),
    (2, 4, 2, 128, 1, (9000, 30)),
    (20, 8, 1, 256, 16, (5000,) + tuple(range(19))),
    (64, 2, 1, 64, 1, tuple(40 * r for r in range(64))),
]


def calls(ctx):
    out = []
    for R, H, HK, hd, L, before in CALLS:
        before, counts = np.array(before), np.full(R, L)
        ref = filled(R, HK, hd, 64, before + counts)
        q, gate = problem(R, H, hd, L, False)
        operands = [cuda(np.ascontiguousarray(x).reshape(-1)) for x in
                    (q, gate, ref.table, before.astype(np.int32), counts.astype(np.int32))]
        cache = ref.paged(cuda)

        def one(ctx=ctx, o=operands, cache=cache, s=(R, L, H, HK, hd)):
            return te.jeff_cached_attention(o[0], o[1], None, cache, o[2], o[3], o[4], *s, None, EPS,
                                            ctx=ctx)
        out.append(one)
    return out


@pytest.mark.gpu
def test_one_workspace_for_all_sizes_and_two_contexts_at_once():
    """Each call alone in a new context, then in one context in many orders, then in two
    on streams of their own, none waited for: the same bits."""
    import torch

    alone = []
    for n in range(len(CALLS)):
        with te.Context(0) as ctx:
            alone.append(host(calls(ctx)[n]()))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    with te.Context(0, stream=streams[0].cuda_stream) as a, \
            te.Context(0, stream=streams[1].cuda_stream) as b:
        orders = [(0, 1, 2, 3, 4, 5), (5, 4, 3, 2, 1, 0), (1, 4, 0, 5, 2, 3), (4, 4, 1, 1, 0, 0)]
        both = []
        for ctx, stream in zip((a, b), streams):
            with torch.cuda.stream(stream):
                both.append(calls(ctx))
        torch.cuda.synchronize()
        for order in orders:
            for n in order:
                with torch.cuda.stream(streams[0]):
                    assert np.array_equal(host(both[0][n]()), alone[n]), (order, n)
        for _ in range(3):
            results = []
            with te.asynchronous():
                for order in orders:
                    for n, m in zip(order, reversed(order)):
                        with torch.cuda.stream(streams[0]):
                            results.append((n, both[0][n]()))
                        with torch.cuda.stream(streams[1]):
                            results.append((m, both[1][m]()))
            torch.cuda.synchronize()
            for n, x in results:
                assert np.array_equal(host(x), alone[n]), n


@pytest.mark.gpu
def test_a_capture_that_would_grow_the_workspace_is_refused():
    """And the workspace that is there goes on: captured calls and eager ones between replays."""
    import torch

    stream = torch.cuda.Stream()
    with te.Context(0, stream=stream.cuda_stream) as ctx, torch.cuda.stream(stream):
        ready = calls(ctx)
        small, large = ready[2], ready[4]
        want = host(small())
        held = ctx.retained_bytes()
        stream.synchronize()
        with te.asynchronous(), pytest.raises(te.Unsupported, match="workspace cannot grow"):
            with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=stream):
                large()
                raise AssertionError("captured a call whose workspace is not there")
        assert ctx.retained_bytes() == held
        # Two graphs and eager calls through one workspace, in turn.
        graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
        with te.asynchronous():
            got = []
            for g, n in zip(graphs, (2, 5)):
                host(ready[n]())
                stream.synchronize()
                with torch.cuda.graph(g, stream=stream):
                    got.append(ready[n]())
        other = host(ready[5]())
        for i in range(4):
            graphs[i & 1].replay()
            graphs[1 - (i & 1)].replay()
            stream.synchronize()
            assert np.array_equal(host(got[0]), want) and np.array_equal(host(got[1]), other)
            assert np.array_equal(host(ready[2 + 3 * (i & 1)]()), (want, other)[i & 1])


@pytest.mark.gpu
def test_many_rows_append(gpu_ctx):
    """33000 rows of one token: each leaves the codes and scales of a row alone."""
    import torch

    R, hd = 33000, 8
    k, v = normal(5, 1, 1, hd, 1), normal(6, 1, 1, hd, 1)
    ref = Cache(1, 1, hd, 64, 1)
    ref.table[:] = 0
    ref.append(k, v, None, None, np.ones(1, np.int64))
    cache = te.paged_cache(R, 1, hd, 64, device="cuda")
    every = lambda x: cuda(np.tile(x.reshape(-1), R))
    te.jeff_cache_append(every(k), every(v), None, cache, cuda(np.arange(R, dtype=np.int32)[::-1].copy()),
                         None, None, R, 1, 1, hd, None, EPS, ctx=gpu_ctx)
    keys = cache[0].view(torch.uint8).view(R, 64, 64)
    values = cache[1].view(torch.uint8).view(R, 64, 64)
    assert (keys[:, 0] == cuda(ref.keys[0, 0, 0])).all() and not keys[:, 1:].any()
    assert (values[:, :hd, 0] == cuda(ref.values[0, 0, 0, :hd, 0])).all() and not values[:, :, 1:].any()
    assert (cache[2] == float(ref.ks[0, 0, 0])).all() and (cache[3] == float(ref.vs[0, 0, 0])).all()


@pytest.mark.gpu
def test_captured_prompts():
    """Many columns in parts, captured; eager calls of other kinds between the replays."""
    import torch

    stream = torch.cuda.Stream()
    with te.Context(0, stream=stream.cuda_stream) as ctx, torch.cuda.stream(stream):
        ready = calls(ctx)
        want = [host(one()) for one in ready]
        graphs, got = [], []
        with te.asynchronous():
            for n in (1, 4):
                graphs.append(torch.cuda.CUDAGraph())
                stream.synchronize()
                with torch.cuda.graph(graphs[-1], stream=stream):
                    got.append(ready[n]())
        for i in range(4):
            for x in got:
                x.fill_(7.0)
            for g in graphs:
                g.replay()
            stream.synchronize()
            assert np.array_equal(host(got[0]), want[1]) and np.array_equal(host(got[1]), want[4])
            for n in (i, 5):
                assert np.array_equal(host(ready[n]()), want[n])


@pytest.mark.gpu
@pytest.mark.parametrize("L", [1, 70])
def test_without_lengths_and_counts(gpu_ctx, L):
    """None: no token before the call, all of its tokens new."""
    R, H, HK, hd = 3, 4, 2, 64
    k, v = normal(5, R, HK, hd, L), normal(6, R, HK, hd, L)
    q, gate = problem(R, H, hd, L, False)
    ref = Cache(R, HK, hd, 64, 2)
    cache, table = ref.paged(cuda), cuda(ref.table.reshape(-1))
    flat = lambda x: cuda(x.reshape(-1))
    ref.append(k, v, None, None, np.full(R, L))
    te.jeff_cache_append(flat(k), flat(v), None, cache, table, None, None, R, L, HK, hd, None, EPS,
                         ctx=gpu_ctx)
    assert ref.same(cache) == [True] * 4
    out = cuda(np.full(q.size, np.nan, np.float32))
    got = te.jeff_cached_attention(flat(q), flat(gate), None, cache, table, None, None, R, L, H, HK, hd,
                                   None, EPS, ctx=gpu_ctx, out=out)
    assert got is out
    check(out, *reference(ref, q, gate, None, None, np.zeros(R, np.int64), np.full(R, L)))


@pytest.mark.gpu
@pytest.mark.parametrize("weight", [3e38, 1e-30])
@pytest.mark.parametrize("L", [1, 67])
def test_norm_weights_of_any_size(gpu_ctx, L, weight):
    """Keys past f32's range, whose scales are up to 2^122, and scales that go with small ones."""
    R, HK, hd = 2, 1, 96
    k, v = normal(5, R, HK, hd, L), normal(6, R, HK, hd, L)
    norm = np.where(np.arange(hd) % 3 == 0, np.float32(weight), np.float32(weight / 3 - 1)).astype(
        np.float32)
    rotary = te.Rotary(te.rotary_frequencies(64, 1e4), True)
    ref = Cache(R, HK, hd, 64, 2)
    cache = ref.paged(cuda)
    i32 = lambda x: cuda(np.asarray(x, np.int32).reshape(-1))
    ref.append(k, v, norm, rotary, np.full(R, L))
    te.jeff_cache_append(cuda(k.reshape(-1)), cuda(v.reshape(-1)), cuda(norm), cache, i32(ref.table), None,
                         None, R, L, HK, hd, rotary, EPS, ctx=gpu_ctx)
    assert ref.same(cache) == [True] * 4


def test_nothing_to_do():
    """No rows or no tokens: nothing is read, written or launched."""
    none = np.zeros(0, np.float32)
    cache = te.paged_cache(2, 2, 64)
    i32 = lambda n: np.zeros(n, np.int32)
    with te.Context(0) as ctx:
        for R, L in ((0, 3), (2, 0)):
            te.jeff_cache_append(none, none, None, cache, i32(R), i32(R), i32(R), R, L, 2, 64, None, EPS,
                                 ctx=ctx)
            out = te.jeff_cached_attention(none, none, None, cache, i32(R), i32(R), i32(R), R, L, 4, 2, 64,
                                           None, EPS, ctx=ctx)
            assert out.size == 0
            rotary = te.Rotary(te.rotary_frequencies(32, 1e4))
            assert te.rotary_rows(none, None, R, L, 2, 64, rotary, ctx=ctx).size == 0
    assert not cache.keys.any()
