"""Token log probabilities, entropy and top alternatives against 64 bits.

Tolerance. log p = (x - m) - log z. z is a sum of positive terms, each off by the
rounding of x - m and its base-2 form (2^-23 |x - m|, weighted by e^(x - m) |x - m|
<= 1/e), the exponential (2 ulp) and the sum's roundings: at most 2^-24 (8 + n), n
additions of a lane (vocab / 64 at most, random, so 6 sqrt(n)) and 9 of the joins.
x - m and the last subtraction round once each, relative to themselves. The entropy's
second sum has the same count on sum e^(x-m) |x-m| / z.
"""
import numpy as np
import pytest

import tenferro_ext as te
from tenferro_ext.workloads import Lcg


def reference(x, tokens, top):
    """x (positions, vocab), tokens (positions, per)."""
    x = x.astype(np.float64)
    with np.errstate(all="ignore"):
        m = x.max(1, keepdims=True)
        d = x - m
        e = np.exp(d)
        z = e.sum(1, keepdims=True)
        lp = d - np.log(z)
        far = (e * np.where(e > 0, -d, 0)).sum(1) / z[:, 0]
        entropy = np.log(z)[:, 0] + far
    bad = ~np.isfinite(m[:, 0])
    lp[bad], entropy[bad] = np.nan, np.nan
    got = np.where(tokens < 0, 0.0, np.take_along_axis(
        np.concatenate((lp, np.full((len(x), 1), np.nan)), 1),
        np.clip(tokens, 0, x.shape[1]), 1)) if tokens is not None else None
    order = np.lexsort((np.arange(x.shape[1]) * np.ones_like(x, int), -np.where(
        np.isnan(x), -np.inf, x), np.isnan(x)), axis=1)[:, :top]
    return got, entropy, order, np.take_along_axis(lp, order, 1), far


def check(got, x, tokens, top):
    lp, entropy, order, top_lp, far = reference(x, tokens, top)
    tol = 2.0 ** -24 * (17 + 6 * np.sqrt(x.shape[1] / 64 + 1))

    def close(a, b, abs_tol):
        a = np.asarray(a, np.float64).reshape(b.shape)
        both = np.isfinite(b)
        assert np.array_equal(np.isnan(a), np.isnan(b))
        assert np.array_equal(a[~both & ~np.isnan(b)], b[~both & ~np.isnan(b)])
        off = np.abs(a - b)[both] - (abs_tol + 2.0 ** -22 * np.abs(b))[both]
        assert (off <= 0).all(), off.max()

    if tokens is not None:
        close(got.log_probs, lp, tol)
    close(got.entropy, entropy, tol * (1 + np.nan_to_num(far)))
    if top:
        assert np.array_equal(np.asarray(got.top_tokens).reshape(order.shape), order)
        close(got.top_log_probs, top_lp, tol)
    else:
        assert got.top_tokens is None and got.top_log_probs is None


def logits(positions, vocab, bf16, seed=0, scale=3.0):
    x = Lcg(seed * 77 + positions * 131 + vocab).normal(positions * vocab).reshape(
        positions, vocab).astype(np.float32) * np.float32(scale)
    return te.bf16_bits_to_f32(te.to_bf16_bits(x)) if bf16 else x


def some_tokens(positions, vocab, per, seed=5):
    return Lcg(seed + positions).integers(0, vocab - 1, positions * per).reshape(positions, per)


def cuda(x):
    import torch

    return torch.from_numpy(np.ascontiguousarray(x).copy()).cuda()


def run(ctx, x, tokens, top, bf16, **kw):
    bits = te.to_bf16_bits(x) if bf16 else x
    r = te.token_log_probs(cuda(bits.reshape(-1)), cuda(tokens.reshape(-1)) if tokens is not None
                           else None, x.shape[0], kw.pop("vocab", x.shape[1]), top=top, bf16=bf16,
                           ctx=ctx, **kw)
    return te.TokenLogProbs(*[a.cpu().numpy() if a is not None else None for a in r])


# ------------------------------------------------------------------ refusals (no GPU)


@pytest.fixture()
def ctx():
    c = te.Context(0)
    yield c
    c.close()


def test_refusals_before_any_device_call(ctx):
    x, t = np.zeros(20, np.float32), np.zeros(4, np.int64)
    with pytest.raises(te.InvalidArgument, match="logits: 20 elements, the shape needs 24"):
        te.token_log_probs(x, t, 4, 6, ctx=ctx)
    with pytest.raises(te.InvalidArgument, match="logits: 20 elements"):
        te.token_log_probs(x, t, 4, 4, ctx=ctx)
    with pytest.raises(te.InvalidArgument, match="tokens: 4 elements"):
        te.token_log_probs(x, t, 5, 4, ctx=ctx)
    with pytest.raises(te.InvalidArgument, match="leading dimension"):
        te.token_log_probs(x[:17], t, 4, 5, leading_dim=4, ctx=ctx)
    with pytest.raises(te.InvalidArgument, match="top must not exceed vocab"):
        te.token_log_probs(x, t, 4, 5, top=6, ctx=ctx)
    with pytest.raises(te.Unsupported, match="top 65 exceeds 64"):
        te.token_log_probs(np.zeros(100, np.float32), None, 1, 100, top=65, ctx=ctx)
    import torch

    with pytest.raises(te.InvalidArgument, match="tokens: tensor dtype int32"):
        te.token_log_probs(torch.zeros(20), torch.zeros(4, dtype=torch.int32), 4, 5, ctx=ctx)
    with pytest.raises(te.InvalidArgument, match="logits: tensor dtype bfloat16"):
        te.token_log_probs(torch.zeros(20, dtype=torch.bfloat16), None, 4, 5, ctx=ctx)
    call = ctx._lib.tfd_token_log_probs_f32
    p = x.ctypes.data
    assert call(ctx.handle, p, 0, 5, 4, None, 0, 0, None, p, None, None, 0) == te.TFD_EINVAL
    assert call(ctx.handle, p, 5, 5, 4, p, 1, 0, None, p, None, None, 0) == te.TFD_EINVAL
    assert "null buffer" in ctx._lib.tfd_last_error(ctx.handle).decode()
    assert call(ctx.handle, p, 5, 5, 4, None, 0, 1, None, p, None, p, 0) == te.TFD_EINVAL
    assert call(ctx.handle, p, 5, 1 << 62, 1 << 62, None, 0, 0, None, p, None, None,
                0) == te.TFD_EINVAL
    assert call(ctx.handle, p, 5, 5, 4, None, 0, 0, None, p, None, None, te.TFD_ASYNC) == te.TFD_EINVAL
    assert call(ctx.handle, None, 5, 5, 0, None, 0, 0, None, None, None, None, 0) == te.TFD_OK


# ------------------------------------------------------------------ on the GPU


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("positions,vocab,per,top", [
    (1, 1, 1, 1), (3, 2, 2, 2), (5, 7, 1, 0), (64, 8, 3, 2), (7, 63, 1, 63), (4, 64, 1, 64),
    (9, 1000, 2, 5), (2, 2048, 1, 20), (2, 2049, 70, 20), (600, 2300, 1, 3), (5, 20011, 4, 64),
    (1, 100003, 2, 20), (17, 131072, 4, 5)])
def test_against_64_bits(gpu_ctx, positions, vocab, per, top, bf16):
    x = logits(positions, vocab, bf16)
    t = some_tokens(positions, vocab, per)
    check(run(gpu_ctx, x, t, top, bf16), x, t, top)


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("vocab", [37, 5000, 90001])
def test_orders_ties_and_special_values(gpu_ctx, vocab, bf16):
    """Ties go to the lowest token, in rising, falling and constant rows and in runs
    of equal logits; -inf, the type's lowest value, NaN and +inf as documented."""
    low = np.float32(-3.3895314e38) if bf16 else np.finfo(np.float32).min
    x = logits(16, vocab, bf16)
    ramp = np.arange(vocab, dtype=np.float32)
    x[0], x[1], x[2], x[3] = np.floor(ramp / 8) % 128, -(np.floor(ramp / 8) % 128), 0.0, -0.0
    x[4] = np.where(ramp % 3 == 0, 0.0, -0.0)
    x[5, ::2] = -np.inf
    x[6, 1:] = -np.inf
    x[7] = -np.inf
    x[8] = low
    x[9, : vocab - 2] = low
    x[10, vocab // 2] = np.nan
    x[11, vocab // 3] = np.inf
    x[12] = np.nan
    x[13] = np.floor(x[13])
    x[14, : vocab // 2] = 200.0
    x[15] *= np.float32(1e36)
    if bf16:
        x = te.bf16_bits_to_f32(te.to_bf16_bits(x))
        x[10, vocab // 2], x[12] = np.nan, np.nan
    t = some_tokens(16, vocab, 3)
    t[:, 0], t[6, 1], t[9, 1] = -1, 0, vocab - 1
    t[13, 2], t[14, 2] = vocab, 1 << 40
    for top in (1, 8, 33):
        got = run(gpu_ctx, x, t, top, bf16)
        check(got, x, t, top)


@pytest.mark.gpu
def test_large_logits_keep_their_differences(gpu_ctx):
    """Logits around 1e6 apart by ones: the differences, not the logits, decide."""
    x = logits(8, 6000, False, scale=1.0) + np.float32(1e6)
    t = some_tokens(8, 6000, 2)
    check(run(gpu_ctx, x, t, 4, False), x, t, 4)


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("vocab,ld", [(5, 9), (1001, 1003), (2051, 2056), (70001, 70017)])
def test_leading_dimensions_offsets_and_surroundings(gpu_ctx, vocab, ld, bf16):
    """Positions further apart than vocab start at every offset from a 16-byte
    boundary; what lies between them (NaN) is not read into anything. The last one may end
    with its vocab-th logit."""
    n = 11
    x = logits(n, vocab, bf16, seed=2)
    wide = np.full((n, ld), np.nan, np.float32)
    wide[:, :vocab] = x
    t = some_tokens(n, vocab, 2)
    flat = wide.reshape(-1)[: ld * (n - 1) + vocab]
    bits = te.to_bf16_bits(flat) if bf16 else flat
    dev = cuda(np.concatenate((bits[:3], bits)))
    for start in (3, 0):
        data = dev[3:] if start else cuda(bits)
        r = te.token_log_probs(data, cuda(t.reshape(-1)), n, vocab, top=3, leading_dim=ld, bf16=bf16,
                               ctx=gpu_ctx)
        check(te.TokenLogProbs(*[a.cpu().numpy() for a in r]), x, t, 3)


@pytest.mark.gpu
def test_host_arrays_without_tokens_and_without_top(gpu_ctx):
    x = logits(6, 3000, False)
    t = some_tokens(6, 3000, 2)
    r = te.token_log_probs(x.reshape(-1), t.reshape(-1), 6, 3000, top=2, ctx=gpu_ctx)
    assert isinstance(r.top_tokens, np.ndarray)
    check(r, x, t, 2)
    r = te.token_log_probs(x.reshape(-1), None, 6, 3000, ctx=gpu_ctx)
    assert r.log_probs is None
    check(r, x, None, 0)
    check(run(gpu_ctx, x, None, 7, False), x, None, 7)
    r = te.token_log_probs(np.zeros(0, np.float32), None, 0, 50, ctx=gpu_ctx)
    assert r.entropy.size == 0


@pytest.mark.gpu
def test_repeats_streams_and_graphs():
    import torch

    stream = torch.cuda.Stream()
    with te.Context(0, stream=stream.cuda_stream) as ctx, torch.cuda.stream(stream):
        x, t = logits(2, 50000, True), some_tokens(2, 50000, 4)
        want = run(ctx, x, t, 9, True)
        check(want, x, t, 9)
        dx, dt = cuda(te.to_bf16_bits(x).reshape(-1)), cuda(t.reshape(-1))
        with te.asynchronous():
            te.token_log_probs(dx, dt, 2, 50000, top=9, bf16=True, ctx=ctx)
            stream.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                got = te.token_log_probs(dx, dt, 2, 50000, top=9, bf16=True, ctx=ctx)
        for i in range(4):
            for a in got:
                a.fill_(-5)
            graph.replay()
            stream.synchronize()
            assert all(np.array_equal(a.cpu().numpy(), b) for a, b in zip(got, want))
            if i == 1:  # a call that needs a larger workspace, eager
                y = logits(3, 160000, True)
                check(run(ctx, y, None, 64, True), y, None, 64)
        with te.asynchronous(), pytest.raises(te.InvalidArgument, match="needs TFD_ASYNC"):
            graph2 = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph2, stream=stream):
                te._async = False
                try:
                    te.token_log_probs(dx, dt, 2, 50000, top=9, bf16=True, ctx=ctx)
                finally:
                    te._async = True


@pytest.mark.gpu
def test_a_capture_that_would_grow_the_workspace_is_refused():
    import torch

    stream = torch.cuda.Stream()
    with te.Context(0, stream=stream.cuda_stream) as ctx, torch.cuda.stream(stream):
        x, t = logits(2, 50000, True), some_tokens(2, 50000, 4)
        want = run(ctx, x, t, 9, True)
        check(want, x, t, 9)
        held = ctx.retained_bytes()
        dx, dt = cuda(te.to_bf16_bits(x).reshape(-1)), cuda(t.reshape(-1))
        big = cuda(logits(3, 160000, False).reshape(-1))
        stream.synchronize()
        with te.asynchronous(), pytest.raises(te.Unsupported, match="workspace cannot grow"):
            with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=stream):
                te.token_log_probs(big, None, 3, 160000, top=64, ctx=ctx)
                raise AssertionError("captured a call whose workspace is not there")
        assert ctx.retained_bytes() == held
        graph = torch.cuda.CUDAGraph()
        with te.asynchronous(), torch.cuda.graph(graph, stream=stream):
            got = te.token_log_probs(dx, dt, 2, 50000, top=9, bf16=True, ctx=ctx)
        for _ in range(3):
            graph.replay()
            stream.synchronize()
            assert all(np.array_equal(a.cpu().numpy(), b) for a, b in zip(got, want))
            te.token_log_probs(big, None, 3, 160000, top=64, ctx=ctx)


@pytest.mark.gpu
def test_logits_past_four_gigabytes(gpu_ctx):
    """More than 2^32 bytes of logits: the last positions are read where they are."""
    import torch

    n, vocab = 33000, 65536
    x = torch.zeros(n * vocab, dtype=torch.bfloat16, device="cuda").view(n, vocab)
    rows = [0, 16384, 32767, 32768, n - 1]
    data = logits(len(rows), vocab, True, seed=4)
    x[rows] = torch.from_numpy(data).cuda().bfloat16()
    t = some_tokens(n, vocab, 1)
    r = te.token_log_probs(x.view(-1), cuda(t.reshape(-1)), n, vocab, top=2, bf16=True, ctx=gpu_ctx)
    pick = lambda a, w: a.view(n, w)[rows].cpu().numpy().reshape(-1)
    check(te.TokenLogProbs(pick(r.log_probs, 1), pick(r.entropy, 1), pick(r.top_tokens, 2),
                           pick(r.top_log_probs, 2)), data, t[rows], 2)
    assert float((r.entropy[1:1000] - np.log(vocab)).abs().max()) < 1e-5


@pytest.mark.gpu
def test_more_positions_than_one_grid_has_threads_for(gpu_ctx):
    """2^26 + 3 positions of a wavefront each: past 2^32 threads in all."""
    import torch

    n, vocab = (1 << 26) + 3, 3
    x = torch.zeros(n, vocab, device="cuda")
    rows = [0, (1 << 22) - 1, 1 << 22, (1 << 26) - 1, 1 << 26, n - 1]
    data = logits(len(rows), vocab, False, seed=6)
    x[rows] = torch.from_numpy(data).cuda()
    tokens = torch.full((n,), 2, dtype=torch.int64, device="cuda")
    r = te.token_log_probs(x.view(-1), tokens, n, vocab, top=1, ctx=gpu_ctx)
    pick = lambda a: a[rows].cpu().numpy()
    check(te.TokenLogProbs(*map(pick, r)), data, np.full((len(rows), 1), 2), 1)
    rest = torch.ones(n, dtype=torch.bool, device="cuda")
    rest[rows] = False
    assert float((r.entropy[rest] - np.log(3)).abs().max()) < 1e-6
    assert int(r.top_tokens[rest].max()) == 0
