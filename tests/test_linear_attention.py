"""Linear attention over rows, prompts and single tokens, against its recurrence
in 64 bits, token by token.

Tolerance. Without the delta rule every output and state element is a sum of
products whose terms carry at most n = key_dim + 64 + length roundings of 2^-24
each, taken on the sum of the terms' absolute values (`size`, the same recurrence
on absolute values). Roundings to nearest are independent and unbiased to first
order, so six standard deviations are 6 sqrt(n) 2^-24 of it; 8 more cover the
decays' exponentials and the scale. With the delta rule and keys of unit length the
step S -> e^g (I - beta k k^T) S does not lengthen any vector for beta in [0, 1], so
errors add up over the tokens without growing: the same count holds for a head's
errors against the largest norm its state (and with it the output) has had, plus its
largest write.
"""
import numpy as np
import pytest

import tenferro_ext as te
from tenferro_ext.workloads import Lcg


def reference(q, k, v, g, beta, mask, scale, state):
    """q, k (R, HK, dk, L), v (R, H, dv, L), g, beta (R, H, L), mask (R, L),
    state (R, H, dk, dv): out (R, H, dv, L), state, and their `size`s."""
    R, H, dv, L = v.shape
    HK, dk = q.shape[1:3]
    idx = np.arange(H) // (H // HK)
    S = np.zeros((R, H, dk, dv)) if state is None else state.astype(np.float64)
    A = np.abs(S)
    out, size = np.zeros((2, R, H, dv, L))
    norm = np.sqrt((S ** 2).sum((2, 3)))
    for t in range(L):
        on = np.ones(R, bool) if mask is None else mask[:, t] != 0
        if not on.any():
            continue
        kt, qt = k[on][..., t][:, idx].astype(np.float64), q[on][..., t][:, idx].astype(np.float64)
        f = np.exp(g[on, :, t].astype(np.float64))[..., None, None]
        D = S[on] * f
        u = v[on, :, :, t].astype(np.float64)
        if beta is not None:
            u = beta[on, :, t].astype(np.float64)[..., None] * (u - np.einsum("rhij,rhi->rhj", D, kt))
        S[on] = D + kt[..., None] * u[:, :, None]
        out[on, :, :, t] = scale * np.einsum("rhij,rhi->rhj", S[on], qt)
        if beta is None:
            A[on] = A[on] * f + np.abs(kt)[..., None] * np.abs(u)[:, :, None]
            size[on, :, :, t] = abs(scale) * np.einsum("rhij,rhi->rhj", A[on], np.abs(qt))
        else:
            norm[on] = np.maximum(norm[on], np.sqrt((S[on] ** 2).sum((2, 3))))
            norm[on] = np.maximum(norm[on], np.sqrt((u ** 2).sum(2)))
    if beta is not None:
        A = np.broadcast_to(norm[..., None, None], S.shape)
        size = abs(scale) * norm[..., None, None] * np.sqrt(
            (q.astype(np.float64) ** 2).sum(2)).max(-1, initial=0.0)[:, idx][..., None, None] * np.ones_like(out)
    return out, S, size, A


class Problem:
    def __init__(self, R, L, H, HK, dk, dv, *, bf16=False, delta=True, mask=None, state=False,
                 decay=1.0, seed=1):
        rng = Lcg(seed * 7919 + R * 1000003 + L * 1009 + H * 101 + dk * 11 + dv)

        def normal(*shape):
            return rng.normal(int(np.prod(shape))).astype(np.float32).reshape(shape)

        def unit(x):
            return x / np.sqrt((x * x).sum(2, keepdims=True))

        self.dims = (R, L, H, HK, dk, dv)
        self.q, self.k = unit(normal(R, HK, dk, L)), unit(normal(R, HK, dk, L))
        self.v = normal(R, H, dv, L)
        self.g = -np.abs(normal(R, H, L)) * np.float32(decay)
        self.beta = (1 / (1 + np.exp(-normal(R, H, L)))).astype(np.float32) if delta else None
        self.state = normal(R, H, dk, dv) if state else None
        self.bf16, self.mask = bf16, None
        if bf16:
            self.q, self.k, self.v = (te.bf16_bits_to_f32(te.to_bf16_bits(x))
                                      for x in (self.q, self.k, self.v))
        if mask == "left":  # one row of them without any active token
            self.mask = np.zeros((R, L), np.float32)
            for r in range(R):
                self.mask[r, (L * r + R - 1) // R:] = 1.0
            self.mask[-1] = 0.0
        elif mask == "holes":
            self.mask = (rng.uniform(R * L) < 0.7).astype(np.float32).reshape(R, L)

    def args(self, to=lambda x: x):
        bits = te.to_bf16_bits if self.bf16 else lambda x: x
        ops = [bits(self.q), bits(self.k), bits(self.v), self.g, self.beta, self.mask]
        return [to(np.ascontiguousarray(x).reshape(-1)) if x is not None else None for x in ops]

    def run(self, ctx, to=lambda x: x, **kw):
        R, L, H, HK, dk, dv = self.dims
        state = to(self.state.reshape(-1)) if self.state is not None else None
        return te.jeff_linear_attention_rows(*self.args(to), R, L, H, HK, dk, dv, state=state,
                                             bf16=self.bf16, ctx=ctx, **kw)

    def check(self, out, state, scale=None):
        R, L, H, HK, dk, dv = self.dims
        scale = float(np.float32(dk ** -0.5 if scale is None else scale))
        want, S, size, A = reference(self.q, self.k, self.v, self.g, self.beta, self.mask, scale,
                                     self.state)
        tol = 2.0 ** -24 * (8 + 6 * np.sqrt(dk + 64 + L))
        out = np.asarray(out, np.float64).reshape(want.shape)
        assert (np.abs(out - want) <= tol * size + 1e-37).all(), np.nanmax(
            np.abs(out - want) / (size + 1e-30))
        if state is not None:
            state = np.asarray(state, np.float64).reshape(S.shape)
            assert (np.abs(state - S) <= tol * A + 1e-37).all(), np.nanmax(
                np.abs(state - S) / (A + 1e-30))


def cut(x, bits):
    """x to nearest with that many significant bits."""
    m, e = np.frexp(x.astype(np.float64))
    return np.ldexp(np.round(np.ldexp(m, bits)), e - bits)


def column_norms(q, k, v, g, beta, mask, scale, state):
    """The bounds of `reference` for each value column by itself: the largest norm a column of
    the state has had, plus its largest write; the output's times the token's query."""
    R, H, dv, L = v.shape
    idx = np.arange(H) // (H // k.shape[1])
    S = np.zeros((R, H, k.shape[2], dv)) if state is None else state.astype(np.float64)
    norm, size = np.sqrt((S ** 2).sum(2)), np.zeros((R, H, dv, L))
    write = np.zeros((R, H, dv))
    for t in range(L):
        on = np.ones(R, bool) if mask is None else mask[:, t] != 0
        if not on.any():
            continue
        kt = k[on][..., t][:, idx].astype(np.float64)
        S[on] *= np.exp(g[on, :, t].astype(np.float64))[..., None, None]
        u = v[on, :, :, t].astype(np.float64)
        if beta is not None:
            u = beta[on, :, t].astype(np.float64)[..., None] * (
                u - np.einsum("rhij,rhi->rhj", S[on], kt))
        S[on] += kt[..., None] * u[:, :, None]
        norm[on] = np.maximum(norm[on], np.sqrt((S[on] ** 2).sum(2)))
        write[on] = np.maximum(write[on], np.abs(u))
        size[on, :, :, t] = abs(scale) * (norm + write)[on] * np.sqrt(
            (q[on][..., t].astype(np.float64) ** 2).sum(2))[:, idx][..., None]
    return size, np.broadcast_to((norm + write)[:, :, None], S.shape)


def check_columns(p, out, state):
    """`Problem.check` with two bounds that lost bits of an operand do not stay within.

    Each value column of the state evolves by itself, S_j <- e^g (I - beta k k^T) S_j + beta k
    v_j, so that the count of the module's comment holds against the column's own norm.

    Over all of a result the errors, independent and unbiased, add up in squares. From the
    state and U to an output an element takes at most 48 + 12 + 3 roundings (8 steps of 32
    features and 2 of 32 tokens, six products each, and the factors), to U as many, and 13 a
    chunk to the state; more than a token by token sum in a tree. A rounding has a standard
    deviation of at most 2^-24 / sqrt(3) of what is rounded, which is at most about twice the
    result (two terms that partly cancel): 2 * 2^-24 sqrt((126 + 13 chunks) / 3) of the
    result's 2-norm. An operand of 16 bits is off by 2^-16 / sqrt(3) or a little less."""
    R, L, H, HK, dk, dv = p.dims
    ops = (p.q, p.k, p.v, p.g, p.beta, p.mask, float(np.float32(dk ** -0.5)), p.state)
    want, S, _, _ = reference(*ops)
    size, A = column_norms(*ops)
    tol = 2.0 ** -24 * (8 + 6 * np.sqrt(dk + 64 + L))
    rms = 2 * 2.0 ** -24 * np.sqrt((126 + 13 * -(-L // 64)) / 3)
    for got, exact, bound in ((out, want, size), (state, S, A)):
        off = np.abs(np.asarray(got, np.float64).reshape(exact.shape) - exact)
        assert (off <= tol * bound + 1e-37).all(), np.max(off / (bound + 1e-30))
        whole = np.sqrt((exact ** 2).sum())
        assert np.sqrt((off ** 2).sum()) <= rms * whole, np.sqrt((off ** 2).sum()) / whole


def cuda(x):
    import torch

    return torch.from_numpy(np.ascontiguousarray(x).copy()).cuda()


def host(x):
    return x.cpu().numpy()


# ------------------------------------------------------------------ refusals (no GPU)


@pytest.fixture()
def ctx():
    c = te.Context(0)
    yield c
    c.close()


def test_refusals_before_any_device_call(ctx):
    R, L, H, HK, dk, dv = 2, 3, 4, 2, 8, 5
    f = lambda n: np.zeros(n, np.float32)
    good = dict(q=f(R * L * HK * dk), k=f(R * L * HK * dk), v=f(R * L * H * dv),
                log_decay=f(R * L * H), beta=f(R * L * H), mask=f(R * L))
    call = lambda dims=(R, L, H, HK, dk, dv), **kw: te.jeff_linear_attention_rows(
        *[kw.get(n, x) for n, x in good.items()], *dims, ctx=ctx,
        **{n: x for n, x in kw.items() if n not in good})
    for name, x in good.items():
        with pytest.raises(te.InvalidArgument, match=f"{name}: {x.size - 1} elements"):
            call(**{name: x[:-1]})
    with pytest.raises(te.InvalidArgument, match="state: 3 elements"):
        call(state=f(3))
    with pytest.raises(te.InvalidArgument, match="state_out: 3 elements"):
        call(state_out=f(3))
    with pytest.raises(te.InvalidArgument, match="multiple of key_heads"):
        call((R, L, 3, 2, dk, dv), v=f(R * L * 3 * dv), log_decay=f(R * L * 3), beta=f(R * L * 3))
    big = 257
    with pytest.raises(te.Unsupported, match="key_dim 257 exceeds 256"):
        call((R, L, H, HK, big, dv), q=f(R * L * HK * big), k=f(R * L * HK * big))
    rc = ctx._lib.tfd_jeff_linear_attention_rows_f32(
        ctx.handle, R, L, H, 0, dk, dv, *[None] * 6, 0, None, None, None, 0)
    assert rc == te.TFD_EINVAL
    rc = ctx._lib.tfd_jeff_linear_attention_rows_f32(
        ctx.handle, R, L, H, HK, dk, dv, *[None] * 6, 0, None, None, None, 0)
    assert rc == te.TFD_EINVAL and "null buffer" in ctx._lib.tfd_last_error(ctx.handle).decode()
    rc = ctx._lib.tfd_jeff_linear_attention_rows_f32(
        ctx.handle, 1 << 40, 1 << 40, H, HK, dk, dv, *[None] * 6, 0, None, None, None, 0)
    assert rc == te.TFD_EINVAL and "overflow" in ctx._lib.tfd_last_error(ctx.handle).decode()
    rc = ctx._lib.tfd_jeff_linear_attention_rows_bf16(
        ctx.handle, R, L, H, HK, dk, dv, *[None] * 6, 0, None, None, None, te.TFD_ASYNC)
    assert rc == te.TFD_EINVAL and "TFD_ASYNC" in ctx._lib.tfd_last_error(ctx.handle).decode()
    with pytest.raises(te.InvalidArgument, match="state: expected a contiguous float32 array"):
        te.jeff_linear_attention_step(f(dk), f(dk), f(dv), f(1), None, np.zeros(dk * dv), 1, 1, 1,
                                      dk, dv, ctx=ctx)


def test_results_are_not_written_to_a_copy(ctx):
    """A host array that would have to be converted is refused as a place for results, and
    keeps what it holds; the caller would never see the copy that is written."""
    R, L, H, dk, dv = 2, 3, 2, 4, 5
    f = lambda n: np.zeros(n, np.float32)
    nv, ns = R * L * H * dv, R * H * dk * dv
    ops = (f(R * L * H * dk), f(R * L * H * dk), f(nv), f(R * L * H), None, None, R, L, H, H, dk, dv)

    def wrong(n):
        fixed = f(n)
        fixed.flags.writeable = False
        return [np.zeros(n), f(2 * n)[::2], fixed, [0.0] * n]

    for x in wrong(nv):
        with pytest.raises(te.InvalidArgument, match="out: expected a contiguous float32 array"):
            te.jeff_linear_attention_rows(*ops, out=x, ctx=ctx)
    for x in wrong(ns):
        with pytest.raises(te.InvalidArgument, match="state_out: expected a contiguous float32"):
            te.jeff_linear_attention_rows(*ops, state_out=x, ctx=ctx)
        with pytest.raises(te.InvalidArgument, match="state: expected a contiguous float32"):
            te.jeff_linear_attention_rows(*ops, state=x, state_out=x, ctx=ctx)
        with pytest.raises(te.InvalidArgument, match="state: expected a contiguous float32"):
            te.jeff_linear_attention_step(f(R * H * dk), f(R * H * dk), f(R * H * dv), f(R * H), None,
                                          x, R, H, H, dk, dv, ctx=ctx)
    with pytest.raises(te.InvalidArgument, match="state: expected a contiguous float32"):
        te.jeff_linear_attention_step(f(R * H * dk), f(R * H * dk), f(R * H * dv), f(R * H), None,
                                      None, R, H, H, dk, dv, ctx=ctx)


# rows, length, heads, key_heads, key_dim, value_dim
COLUMNS = [(3, 17, 4, 2, 20, 33), (2, 65, 2, 1, 16, 130), (3, 127, 2, 2, 128, 128),
           (1, 200, 2, 1, 256, 72), (1, 600, 2, 1, 64, 64), (5, 90, 8, 4, 50, 213),
           (5, 90, 8, 4, 100, 213), (5, 90, 8, 4, 200, 100)]


@pytest.mark.parametrize("bits", [17, 16])
@pytest.mark.parametrize("delta", [True, False], ids=["delta", "plain"])
@pytest.mark.parametrize("shape", COLUMNS[:5], ids=str)
def test_the_check_finds_operands_of_fewer_bits(shape, delta, bits):
    """What a kernel computes that drops the last piece of its operands: queries, keys, values
    and every 64 tokens the state cut to 16 or 17 bits."""
    for mask in (None, "left", "holes"):
        p = Problem(*shape, delta=delta, mask=mask, state=True, decay=0.3)
        outs, state, L = [], p.state, shape[1]
        for a in range(0, L, 64):
            at = lambda x: None if x is None else x[..., a:a + 64]
            few = lambda x: cut(at(x), bits)
            out, state, _, _ = reference(few(p.q), few(p.k), few(p.v), at(p.g), at(p.beta),
                                         at(p.mask), float(np.float32(shape[4] ** -0.5)),
                                         cut(state, bits))
            outs.append(out)
        with pytest.raises(AssertionError):
            check_columns(p, np.concatenate(outs, -1), state)


def test_empty_problems_need_no_gpu(ctx):
    z = np.zeros(0, np.float32)
    out, state = te.jeff_linear_attention_rows(z, z, z, z, None, None, 0, 5, 2, 1, 4, 4, ctx=ctx)
    assert out.size == 0 and state.size == 0
    out, state = te.jeff_linear_attention_rows(z, z, z, z, None, None, 3, 0, 2, 1, 4, 4,
                                               want_state=False, ctx=ctx)
    assert out.size == 0 and state is None


# ------------------------------------------------------------------ on the GPU

SHAPES = [  # rows, length, heads, key_heads, key_dim, value_dim
    (1, 1, 1, 1, 1, 1), (2, 2, 2, 1, 5, 3), (3, 17, 4, 2, 20, 33), (2, 63, 2, 2, 32, 32),
    (1, 64, 3, 1, 64, 48), (2, 65, 2, 1, 16, 130), (3, 127, 2, 2, 128, 128), (1, 128, 2, 1, 96, 80),
    (2, 129, 4, 4, 72, 20), (1, 200, 2, 1, 256, 72), (2, 257, 3, 3, 130, 257), (1, 600, 2, 1, 64, 64)]


@pytest.mark.gpu
@pytest.mark.parametrize("delta", [True, False], ids=["delta", "plain"])
@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_against_the_recurrence(gpu_ctx, shape, bf16, delta):
    for i, mask in enumerate((None, "left", "holes")):
        p = Problem(*shape, bf16=bf16, delta=delta, mask=mask, state=i != 1, seed=i,
                    decay=(0.02, 1.0, 5.0)[i])
        out, state = p.run(gpu_ctx, cuda)
        p.check(host(out), host(state))


@pytest.mark.gpu
@pytest.mark.parametrize("delta", [True, False], ids=["delta", "plain"])
@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("value_dim", [100, 213])
@pytest.mark.parametrize("key_dim,length", [(20, 150), (50, 200), (100, 150), (200, 80)])
def test_grids_past_the_compute_units(gpu_ctx, key_dim, length, value_dim, bf16, delta):
    """280 and 560 column tiles, which other forms take than a tile per CU."""
    p = Problem(5, length, 8, 4, key_dim, value_dim, bf16=bf16, delta=delta, mask="left",
                state=True, decay=0.3)
    out, state = p.run(gpu_ctx, cuda)
    p.check(host(out), host(state))


@pytest.mark.gpu
@pytest.mark.parametrize("length", [1, 30, 150])
@pytest.mark.parametrize("delta", [True, False], ids=["delta", "plain"])
def test_decays_that_forget(gpu_ctx, length, delta):
    """log_decay -inf, very negative and very small magnitudes side by side: a sum
    of such decays over the tokens in 32 bits would lose the small ones."""
    p = Problem(2, length, 2, 1, 64, 40, delta=delta, state=True, decay=0.01)
    p.g[:, :, ::7] = -1000.0
    p.g[0, :, 3::11] = -np.inf
    p.g[1, 1, 5::9] = -100.0
    p.g[:, 0, 2::13] = 0.0
    out, state = p.run(gpu_ctx, cuda)
    p.check(host(out), host(state))


@pytest.mark.gpu
@pytest.mark.parametrize("length", [2, 150])
def test_inactive_tokens_hold_anything(gpu_ctx, length):
    for bf16 in (False, True):
        p = Problem(2, length, 4, 2, 40, 24, bf16=bf16, mask="holes", state=True)
        p.mask[0, 0], p.mask[1, -1] = 0.0, 0.0
        want = [host(x) for x in p.run(gpu_ctx, cuda)]
        off = p.mask == 0
        for x in (p.q, p.k, p.v, p.g, p.beta):
            y = np.moveaxis(x, -1, 1)  # (R, L, ...)
            y[off] = np.nan
        p.v[0, 0, 0][off[0]] = np.inf
        got = [host(x) for x in p.run(gpu_ctx, cuda)]
        for a, b in zip(got, want):
            assert np.array_equal(a, b)
        out = got[0].reshape(2, -1, length)
        assert (np.moveaxis(out, 1, 2)[off] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("delta", [True, False], ids=["delta", "plain"])
@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
def test_a_prompt_in_pieces_and_single_tokens(gpu_ctx, bf16, delta):
    """The state carries over from call to call: 100 + 75 tokens as prompts, then 5
    single tokens with the state updated in place, are the 180 tokens at once."""
    p = Problem(3, 180, 4, 2, 64, 48, bf16=bf16, delta=delta, mask="holes")
    R, L, H, HK, dk, dv = p.dims
    outs, state = [], None

    def part(a, b):
        w = Problem(R, b - a, H, HK, dk, dv, bf16=bf16, delta=delta)
        w.q, w.k, w.v, w.g, w.mask = (x[..., a:b] for x in (p.q, p.k, p.v, p.g, p.mask))
        w.beta = p.beta[..., a:b] if delta else None
        return w

    for a, b in ((0, 100), (100, 175)):
        w = part(a, b)
        out, state = te.jeff_linear_attention_rows(*w.args(cuda), *w.dims, state=state, bf16=bf16,
                                                   ctx=gpu_ctx)
        outs.append(host(out).reshape(R, H, dv, b - a))
    for t in range(175, 180):
        q, k, v, g, beta, mask = part(t, t + 1).args(cuda)
        out = te.jeff_linear_attention_step(q, k, v, g, beta, state, R, H, HK, dk, dv, mask=mask,
                                            bf16=bf16, ctx=gpu_ctx)
        outs.append(host(out).reshape(R, H, dv, 1))
    p.check(np.concatenate(outs, -1), host(state))


@pytest.mark.gpu
def test_state_in_place_zero_length_and_host_arrays(gpu_ctx):
    for L in (0, 1, 90):
        p = Problem(2, L, 2, 2, 33, 18, state=True)
        state = cuda(p.state.reshape(-1))
        dims = p.dims
        out, same = te.jeff_linear_attention_rows(*p.args(cuda), *dims, state=state,
                                                  state_out=state, ctx=gpu_ctx)
        assert same is state
        p.check(host(out), host(state))
        out, s = p.run(gpu_ctx)  # host arrays: uploaded, run, downloaded
        assert isinstance(out, np.ndarray)
        assert np.array_equal(s, host(state))
        p.check(out, s)
        out2, none = p.run(gpu_ctx, cuda, want_state=False)
        assert none is None and np.array_equal(host(out2), out)
        p.state = None
        out, s = p.run(gpu_ctx, cuda, scale=0.7)
        p.check(host(out), host(s), scale=0.7)


@pytest.mark.gpu
@pytest.mark.parametrize("length", [1, 8, 77, 256])
@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
def test_unaligned_buffers_and_their_surroundings(gpu_ctx, length, bf16):
    """Operands one element off a 16-byte boundary, outputs inside larger buffers
    that keep what is around them: the same bits as with whole buffers."""
    import torch

    p = Problem(2, length, 4, 2, 64, 36, bf16=bf16, mask="holes", state=True)
    want = [host(x) for x in p.run(gpu_ctx, cuda)]

    def shifted(x):
        y = cuda(np.concatenate((x[:1], x.reshape(-1), x[:1])))
        return y[1:-1]

    buf = [torch.full((w.size + 2,), 7.0, device="cuda") for w in want]
    p.run(gpu_ctx, shifted, out=buf[0][1:-1], state_out=buf[1][1:-1])
    for b, w in zip(buf, want):
        b = host(b)
        assert b[0] == 7.0 and b[-1] == 7.0 and np.array_equal(b[1:-1], w)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1, 1, 16, 16, 128, 128), (2, 300, 4, 2, 128, 64)], ids=str)
def test_repeats_streams_and_graphs(shape):
    """The same bits on every run, on another stream, and on every replay of a graph,
    also after a larger call of the same context."""
    import torch

    stream = torch.cuda.Stream()
    with te.Context(0, stream=stream.cuda_stream) as ctx, torch.cuda.stream(stream):
        p = Problem(*shape, state=True, mask="holes")
        R, L, H, HK, dk, dv = shape
        want = [host(x) for x in p.run(ctx, cuda)]
        ops = p.args(cuda)
        state, out, new = cuda(p.state.reshape(-1)), cuda(want[0] * 0), cuda(want[1] * 0)
        call = lambda: te.jeff_linear_attention_rows(*ops, *p.dims, state=state, state_out=new,
                                                     ctx=ctx, out=out)
        with te.asynchronous():
            call()
            stream.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                call()
        for i in range(4):
            out.fill_(-1.0), new.fill_(-1.0)
            graph.replay()
            stream.synchronize()
            assert np.array_equal(host(out), want[0]) and np.array_equal(host(new), want[1])
            if i == 1:  # a larger call in between, eager
                b = Problem(2 * R, L + 200, H, HK, dk, dv)
                b.check(*[host(x) for x in b.run(ctx, cuda)])
        with te.asynchronous(), pytest.raises(te.TenferroExtError):
            big = Problem(9, 1500, H, HK, dk, 256)
            args = big.args(cuda)
            o, s = torch.empty(9 * 1500 * H * 256, device="cuda"), torch.empty(
                9 * H * dk * 256, device="cuda")
            stream.synchronize()
            graph2 = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph2, stream=stream):
                te.jeff_linear_attention_rows(*args, *big.dims, state_out=s, out=o, ctx=ctx)
                raise te.TenferroExtError(0, "captured without growing")
    with te.Context(0) as own:  # the context's own stream, ordered against torch's
        got = [host(x) for x in p.run(own, cuda)]
        assert all(np.array_equal(a, b) for a, b in zip(got, want))
        assert own.retained_bytes() > 0


@pytest.mark.gpu
def test_states_past_four_gigabytes(gpu_ctx):
    """Single tokens of so many rows that the states' offsets pass 32 bits."""
    import torch

    R, H, dk, dv = 4200, 16, 128, 128
    gen = torch.Generator(device="cuda").manual_seed(3)
    new = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    q, k = (torch.nn.functional.normalize(new(R, H, dk), dim=2) for _ in range(2))
    v, g, beta = new(R, H, dv), -new(R, H).abs(), torch.rand(R, H, generator=gen, device="cuda")
    state = new(R, H, dk, dv)
    rows = torch.tensor([0, 2047, 2048, 4095, 4096, R - 1])
    before = state[rows.cuda()].cpu().numpy()
    out = te.jeff_linear_attention_step(q.view(-1), k.view(-1), v.view(-1), g.view(-1),
                                        beta.view(-1), state.view(-1), R, H, H, dk, dv,
                                        ctx=gpu_ctx)
    part = lambda x: x[rows.cuda()].cpu().numpy()
    p = Problem(len(rows), 1, H, H, dk, dv)
    p.q, p.k, p.v, p.g, p.beta = part(q)[..., None], part(k)[..., None], part(v)[..., None], \
        part(g)[..., None], part(beta)[..., None]
    p.state = before
    p.check(part(out.view(R, -1)), part(state))


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
def test_more_rows_than_one_workspace_holds(gpu_ctx, bf16):
    """2300 rows of two chunks and 16 heads, over 2 GiB of operands: runs of rows follow
    each other through the workspace."""
    import torch

    R, L, H, HK, dk, dv = 2300, 70, 16, 8, 32, 32
    gen = torch.Generator(device="cuda").manual_seed(8)
    new = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    q, k = (torch.nn.functional.normalize(new(R, HK, dk, L), dim=2) for _ in range(2))
    v, g, beta = new(R, H, dv, L), -new(R, H, L).abs(), torch.rand(R, H, L, generator=gen,
                                                                   device="cuda")
    state, mask = new(R, H, dk, dv), (torch.rand(R, L, generator=gen, device="cuda") < 0.9).float()
    if bf16:
        q, k, v = (x.bfloat16() for x in (q, k, v))
    flat = [x.reshape(-1) for x in (q, k, v, g, beta, mask)]
    out, after = te.jeff_linear_attention_rows(*flat, R, L, H, HK, dk, dv, state=state.view(-1),
                                               bf16=bf16, ctx=gpu_ctx)
    assert gpu_ctx.retained_bytes() < 3 << 30
    rows = [0, 500, 1000, 1023, 1500, 2047, 2048, R - 1]
    part = lambda x: x[rows].float().cpu().numpy()
    p = Problem(len(rows), L, H, HK, dk, dv)
    p.q, p.k, p.v, p.g, p.beta, p.mask, p.state = map(part, (q, k, v, g, beta, mask, state))
    p.check(part(out.view(R, -1)), part(after.view(R, -1)))
    assert bool((out.view(R, H, dv, L) != 0).any(3).all())


@pytest.mark.gpu
@pytest.mark.parametrize("length", [1 << 20, (1 << 20) + 5])
def test_the_longest_chunked_row_and_past_it(gpu_ctx, length):
    """The last tokens of a row of 2^20 tokens, and of one past what the chunks
    address. e^(sum of the decays) of 300 tokens is below 2^-200: only those count."""
    import torch

    H, dk, dv, last = 2, 8, 8, 300
    gen = torch.Generator(device="cuda").manual_seed(9)
    new = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    q, k = (torch.nn.functional.normalize(new(1, H, dk, length), dim=2) for _ in range(2))
    v, g, beta = new(1, H, dv, length), -new(1, H, length).abs(), torch.rand(
        1, H, length, generator=gen, device="cuda")
    out, state = te.jeff_linear_attention_rows(*(x.reshape(-1) for x in (q, k, v, g, beta)), None, 1,
                                               length, H, H, dk, dv, ctx=gpu_ctx)
    part = lambda x: x[..., length - last:].cpu().numpy()
    q, k, v, g, beta = map(part, (q, k, v, g, beta))
    assert (g[..., :200].sum(-1) < -139).all()
    scale = float(np.float32(dk ** -0.5))
    want, S, size, A = reference(q, k, v, g, beta, None, scale, None)
    tol = 2.0 ** -24 * (8 + 6 * np.sqrt(dk + 64 + last))
    got = part(out.view(1, H, dv, length))
    assert (np.abs(got - want) <= tol * size)[..., 200:].all()
    assert (np.abs(state.view(1, H, dk, dv).cpu().numpy() - S) <= tol * A).all()


@pytest.mark.gpu
@pytest.mark.parametrize("delta,key_heads", [(False, 820), (True, 2)])
def test_a_row_of_more_columns_than_one_grid_has_threads_for(gpu_ctx, delta, key_heads):
    """4100 heads of 65536 value features: 2^32 threads and more for one row, whose heads go in
    runs, of whole groups of a key head (5 heads) and of parts of one (2050 heads)."""
    import torch

    L, H, dk, dv = 7, 4100, 8, 65536
    gen = torch.Generator(device="cuda").manual_seed(12)
    new = lambda *s, **kw: torch.randn(*s, generator=gen, device="cuda", **kw)
    q, k = (torch.nn.functional.normalize(new(key_heads, dk, L), dim=1).bfloat16() for _ in "qk")
    v, g = new(H, dv, L, dtype=torch.bfloat16), -new(H, L).abs()
    beta = torch.rand(H, L, generator=gen, device="cuda") if delta else None
    mask = torch.tensor([1.0, 1, 0, 1, 1, 1, 1], device="cuda")
    state = new(H, dk, dv)
    heads = [0, 4, 5, 1019, 1020, 1023, 1024, 2047, 2048, 2049, 2050, 3073, 3074, 4097, 4098, H - 1]
    cols = [*range(5), *range(32760, 32775), *range(dv - 20, dv)]
    part = lambda x: x[heads][:, cols].float().cpu().numpy()[None]
    of_key = [h // (H // key_heads) for h in heads]
    p = Problem(1, L, len(heads), len(heads), dk, len(cols), delta=delta)
    p.q, p.k = (x[of_key].float().cpu().numpy()[None] for x in (q, k))
    p.v, p.state = part(v), part(state.transpose(1, 2)).transpose(0, 1, 3, 2)
    p.g, p.mask = g[heads].cpu().numpy()[None], mask.cpu().numpy()[None]
    p.beta = beta[heads].cpu().numpy()[None] if delta else None
    flat = [x.reshape(-1) if x is not None else None for x in (q, k, v, g, beta)]
    out, _ = te.jeff_linear_attention_rows(*flat, mask, 1, L, H, key_heads, dk, dv,
                                           state=state.view(-1), state_out=state.view(-1),
                                           bf16=True, ctx=gpu_ctx)
    p.check(part(out.view(H, dv, L)), part(state.transpose(1, 2)).transpose(0, 1, 3, 2))


@pytest.mark.gpu
def test_single_tokens_of_more_rows_than_two_to_the_32_threads(gpu_ctx):
    import torch

    R, H, dk, dv = 65535, 260, 1, 32
    gen = torch.Generator(device="cuda").manual_seed(13)
    new = lambda *s, **kw: torch.randn(*s, generator=gen, device="cuda", **kw)
    q, k = (new(R, H, dk).sign().bfloat16() for _ in "qk")
    v, g = new(R, H, dv, dtype=torch.bfloat16), -new(R, H).abs()
    beta, state = torch.rand(R, H, generator=gen, device="cuda"), new(R, H, dk, dv)
    rows = [0, 1, 32767, 32768, 64000, R - 1]
    part = lambda x: x[rows].float().cpu().numpy()
    p = Problem(len(rows), 1, H, H, dk, dv)
    p.q, p.k, p.v, p.g, p.beta = (part(x)[..., None] for x in (q, k, v, g, beta))
    p.state = part(state)
    out = te.jeff_linear_attention_step(*(x.reshape(-1) for x in (q, k, v, g, beta)),
                                        state.view(-1), R, H, H, dk, dv, bf16=True, ctx=gpu_ctx)
    p.check(part(out.view(R, H, dv, 1)), part(state))


@pytest.mark.gpu
@pytest.mark.parametrize("delta", [True, False], ids=["delta", "plain"])
@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("dk", [30, 64, 128, 256])
def test_the_workspace_holds_what_is_used(dk, bf16, delta):
    """Per (row, key head, chunk): queries, with the delta rule keys by tokens, and keys by
    features, except f32 keys of up to 128 features, which are read where they are. Per (row,
    head, chunk): scores, with the delta rule the solve operand, and three factors a token."""
    R, L, H, HK, dv = 2, 100, 4, 2, 20
    p = Problem(R, L, H, HK, dk, dv, bf16=bf16, delta=delta, state=True)
    with te.Context(0) as ctx:
        ctx.stream()
        before = ctx.retained_bytes()
        out, state = p.run(ctx, cuda)
        used = ctx.retained_bytes() - before
    p.check(host(out), host(state))
    chunks, wide = 2, max(32, 1 << (dk - 1).bit_length())
    parts = 1 + delta + (bf16 or dk > 128)
    assert used == R * chunks * (HK * parts * 64 * wide * (2 if bf16 else 4)
                                 + H * (1 + delta) * 18 * 1024 + H * 3 * 64 * 4 + 8)


@pytest.mark.gpu
@pytest.mark.parametrize("delta", [True, False], ids=["delta", "plain"])
@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", COLUMNS, ids=str)
def test_every_column_against_its_own_norm(gpu_ctx, shape, bf16, delta):
    for mask in (None, "left", "holes"):
        p = Problem(*shape, bf16=bf16, delta=delta, mask=mask, state=True, decay=0.3)
        check_columns(p, *[host(x) for x in p.run(gpu_ctx, cuda)])


@pytest.mark.gpu
@pytest.mark.parametrize("delta", [True, False], ids=["delta", "plain"])
@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("heads,key_heads,dk,dv", [(4, 2, 40, 24), (8, 4, 50, 200),
                                                   (8, 4, 100, 260), (4, 2, 200, 24)])
def test_more_than_64_chunks_in_a_row_without_an_active_token(gpu_ctx, heads, key_heads, dk, dv,
                                                              bf16, delta):
    """Rows of 73 chunks with 150 active tokens: in the first and the last ones with 68 dead
    chunks between, only in the last, only in the first, and none. The others hold NaN."""
    R, n, L = 4, 150, 64 * 72 + 10
    p = Problem(R, n, heads, key_heads, dk, dv, bf16=bf16, delta=delta, state=True, decay=0.3)
    p.mask = np.ones((R, n), np.float32)
    p.mask[3] = 0.0
    at = np.array([[*range(75), *range(L - 75, L)], range(L - n, L), range(n), range(n)])
    mask = np.zeros((R, L), np.float32)
    for r in range(3):
        mask[r, at[r]] = 1.0

    def long(x, fill=np.nan):
        if x is None:
            return None
        y = np.full((*x.shape[:-1], L), fill, np.float32)
        for r in range(R):
            y[r][..., at[r]] = x[r]
        return y

    w = Problem(1, 1, 1, 1, 1, 1, bf16=bf16)
    w.dims = (R, L, heads, key_heads, dk, dv)
    w.q, w.k, w.v, w.g, w.beta = (long(x) for x in (p.q, p.k, p.v, p.g, p.beta))
    w.mask, w.state = mask, p.state
    out, state = [host(x) for x in w.run(gpu_ctx, cuda)]
    out = out.reshape(R, heads, dv, L)
    assert (np.moveaxis(out, 3, 1)[mask == 0] == 0).all()
    check_columns(p, np.stack([out[r][..., at[r]] for r in range(R)]), state)
    assert np.array_equal(state.reshape(p.state.shape)[3], p.state[3])


@pytest.mark.gpu
def test_a_capture_that_would_grow_the_workspace_is_refused():
    """And what the context had stays as it was: the call before it runs, captured and eager."""
    import torch

    stream = torch.cuda.Stream()
    with te.Context(0, stream=stream.cuda_stream) as ctx, torch.cuda.stream(stream):
        small, big = Problem(1, 100, 2, 2, 40, 24), Problem(3, 500, 2, 2, 40, 24)
        want = [host(x) for x in small.run(ctx, cuda)]
        held = ctx.retained_bytes()
        ops, more = small.args(cuda), big.args(cuda)
        stream.synchronize()
        with te.asynchronous(), pytest.raises(te.Unsupported, match="workspace cannot grow"):
            with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=stream):
                te.jeff_linear_attention_rows(*more, *big.dims, ctx=ctx)
                raise AssertionError("captured a call whose workspace is not there")
        assert ctx.retained_bytes() == held
        graph = torch.cuda.CUDAGraph()
        with te.asynchronous(), torch.cuda.graph(graph, stream=stream):
            got = te.jeff_linear_attention_rows(*ops, *small.dims, ctx=ctx)
        for _ in range(3):
            graph.replay()
            stream.synchronize()
            assert all(np.array_equal(host(a), b) for a, b in zip(got, want))
            big.check(*[host(x) for x in big.run(ctx, cuda)])


# Shapes whose prompts take, of the delta rule: the token-by-token kernel, the path kernel on
# one and two column tiles, four waves on two and four tiles, eight waves on one and two; the
# same shapes without it: the plain kernel on one and two tiles.
EVERY_KERNEL = [(2, 5, 4, 2, 40, 24), (2, 150, 4, 2, 40, 24), (5, 90, 8, 4, 50, 100),
                (5, 90, 8, 4, 50, 213), (5, 90, 8, 4, 100, 213), (2, 150, 4, 2, 200, 24),
                (5, 90, 8, 4, 200, 213)]


@pytest.mark.gpu
@pytest.mark.parametrize("delta", [True, False], ids=["delta", "plain"])
@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", EVERY_KERNEL, ids=str)
def test_inactive_tokens_beside_inf_and_nan(gpu_ctx, shape, bf16, delta):
    """A state and active tokens that hold inf and NaN: the outputs of inactive tokens are 0
    all the same, and a value column without any of it has the bits it had before."""
    R, L, H, HK, dk, dv = shape
    p = Problem(*shape, bf16=bf16, delta=delta, mask="holes", state=True, decay=0.1)
    p.mask[:, 1], p.mask[:, 2] = 1.0, 0.0
    clean = [host(x) for x in p.run(gpu_ctx, cuda)]
    p.state[:, :, dk // 2, 3], p.state[:, :, 0, 4] = np.inf, np.nan
    p.v[:, :, 5, 1], p.v[:, :, 6, 1] = np.nan, -np.inf
    out, state = [host(x) for x in p.run(gpu_ctx, cuda)]
    off = p.mask == 0
    tokens = lambda x: np.moveaxis(x.reshape(R, H, dv, L), 3, 1)  # (R, L, H, dv)
    assert (tokens(out)[off] == 0).all()
    whole = [j for j in range(dv) if j not in (3, 4, 5, 6)]
    assert np.array_equal(tokens(out)[..., whole], tokens(clean[0])[..., whole])
    cols = lambda x: x.reshape(R, H, dk, dv)[..., whole]
    assert np.array_equal(cols(state), cols(clean[1]))
    last = tokens(out)[np.arange(R), [np.flatnonzero(m)[-1] for m in p.mask]]
    assert not np.isfinite(last[..., 3:7]).any()
    p.k[:, :, 0, 1] = np.nan  # every column of the heads from here on
    out = host(p.run(gpu_ctx, cuda)[0])
    assert (tokens(out)[off] == 0).all()
