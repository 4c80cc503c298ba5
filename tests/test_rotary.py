"""Rotary positions against the formula in 64 bits.

Tolerance. The turn is taken in 64 bits and rounded once, to within 2^-25 of a turn or pi
2^-24 of an angle; a sine is off by 2 steps of 2^-24, its product with the magnitude, the
product with a feature and the sum by one rounding each: 9 2^-24 m (|a| + |b|) covers all.
A bf16 result is rounded once more, by 2^-8 of itself.
"""
import numpy as np
import pytest

import tenferro_ext as te
from tenferro_ext.workloads import Lcg
from test_linear_attention import cuda, host


def pair_index(rotary_dim, interleaved):
    i = np.arange(rotary_dim // 2)
    return (2 * i, 2 * i + 1) if interleaved else (i, i + rotary_dim // 2)


def turned(x, positions, rotary, inverse=False):
    """x (R, H, hd, L) in 64 bits, positions (R, L): turned, and the terms' absolute sum."""
    f, interleaved, magnitude = rotary
    t = positions.astype(np.float64)[:, None, :] * np.asarray(f)[None, :, None]
    t = 2 * np.pi * (t - np.rint(t))
    c, s = np.cos(t)[:, None], np.sin(t)[:, None] * (-1 if inverse else 1)
    a, b = pair_index(2 * len(f), interleaved)
    y, size = x.astype(np.float64).copy(), np.zeros(x.shape)
    y[:, :, a], y[:, :, b] = (magnitude * (x[:, :, a] * c - x[:, :, b] * s),
                              magnitude * (x[:, :, a] * s + x[:, :, b] * c))
    size[:, :, a] = size[:, :, b] = abs(magnitude) * (np.abs(x[:, :, a]) + np.abs(x[:, :, b]))
    return y, size


def normal(seed, *shape):
    return Lcg(seed).normal(int(np.prod(shape))).astype(np.float32).reshape(shape)


def as_float(y):
    """Values of a result of either type, on the host."""
    y = host(y)
    return te.bf16_bits_to_f32(y.view(np.uint16)) if y.dtype.itemsize == 2 else y


CASES = [
    # rows, length, heads, head_dim, rotary_dim, interleaved, first position
    (64, 1, 8, 256, 64, False, 5000),
    (3, 1, 2, 10, 2, True, 1),
    (1, 7, 1, 33, 32, False, 0),
    (2, 64, 3, 128, 128, True, 1 << 20),
    (2, 1003, 5, 96, 48, False, 100000),
    (1, 130, 17, 512, 256, True, 2**31 - 200),
    (2, 9, 4, 6, 0, False, 3),
]


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c[:5])))
def test_against_the_formula(gpu_ctx, case, inverse, bf16):
    R, L, H, hd, rot, interleaved, first = case
    x = normal(1 + L, R, H, hd, L)
    if bf16:
        x = te.bf16_bits_to_f32(te.to_bf16_bits(x))
    f = te.rotary_frequencies(rot, 1e4)
    rotary = te.Rotary(f, interleaved, 1.25)
    positions = (first + 11 * np.arange(R)[:, None] + np.arange(L)).astype(np.int32)
    bits = te.to_bf16_bits if bf16 else lambda v: v
    got = te.rotary_rows(cuda(bits(x).reshape(-1)), cuda(positions.reshape(-1)), R, L, H, hd, rotary,
                         inverse=inverse, bf16=bf16, ctx=gpu_ctx)
    want, size = turned(x, positions, rotary, inverse)
    tol = 9 * 2.0**-24 * size + (2.0**-8 * np.abs(want) if bf16 else 0)
    off = np.abs(as_float(got).reshape(want.shape).astype(np.float64) - want)
    assert (off <= tol).all(), (off / (size + 1e-30)).max()


@pytest.mark.gpu
def test_places_none_negative_and_in_place(gpu_ctx):
    R, L, H, hd = 2, 37, 3, 40
    x = normal(3, R, H, hd, L)
    rotary = te.Rotary(te.rotary_frequencies(20, 1e4))
    at = np.broadcast_to(np.arange(L, dtype=np.int32), (R, L))
    one = te.rotary_rows(x.reshape(-1), None, R, L, H, hd, rotary, ctx=gpu_ctx)  # host arrays
    d = cuda(x.reshape(-1))
    two = te.rotary_rows(d, cuda(at.reshape(-1).copy()), R, L, H, hd, rotary, ctx=gpu_ctx, out=d)
    assert two is d and np.array_equal(one, host(two))
    # Turning by -p is the inverse, bit for bit, and undoes the turn.
    back = te.rotary_rows(two, cuda(-at.reshape(-1)), R, L, H, hd, rotary, ctx=gpu_ctx)
    inverse = te.rotary_rows(two, None, R, L, H, hd, rotary, inverse=True, ctx=gpu_ctx)
    assert np.array_equal(host(back), host(inverse))
    _, size = turned(x, at, rotary)
    off = np.abs(host(back).reshape(x.shape) - x)
    assert (off <= 2 * 9 * 2.0**-24 * 1.5 * (size + np.abs(x))).all()


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
def test_inverse_is_the_gradient(gpu_ctx, interleaved):
    """For y = R x the gradient of w . y is R^T w: against differences of the op itself, which
    is linear, with steps along each feature of a head."""
    L, hd, rot = 5, 12, 8
    rotary = te.Rotary(te.rotary_frequencies(rot, 100.0), interleaved, 0.75)
    w = normal(9, 1, 1, hd, L)
    grad = as_float(te.rotary_rows(cuda(w.reshape(-1)), None, 1, L, 1, hd, rotary, inverse=True,
                                   ctx=gpu_ctx)).reshape(hd, L)
    for i in range(hd):
        e = np.zeros((1, 1, hd, L), np.float32)
        e[:, :, i] = 1
        y = as_float(te.rotary_rows(cuda(e.reshape(-1)), None, 1, L, 1, hd, rotary, ctx=gpu_ctx))
        diff = (y.reshape(hd, L).astype(np.float64) * w[0, 0]).sum(0)
        # Two errors of 9 2^-24 of the terms: of the pair's row and of its column.
        assert (np.abs(diff - grad[i]) <= 2 * 9 * 2.0**-24 * np.abs(w[0, 0]).sum(0)).all()


@pytest.mark.gpu
def test_captured_with_positions_that_move(gpu_ctx):
    import torch

    R, L, H, hd = 4, 1, 2, 64
    x = cuda(normal(4, R, H, hd, L).reshape(-1))
    p = cuda(np.arange(R, dtype=np.int32))
    rotary = te.Rotary(te.rotary_frequencies(hd, 1e4), True)
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with te.Context(0, stream=side.cuda_stream) as ctx, te.asynchronous():
        with torch.cuda.graph(graph, stream=side):
            out = te.rotary_rows(x, p, R, L, H, hd, rotary, ctx=ctx)
            p += 1
        for step in range(4):
            graph.replay()
            torch.cuda.synchronize()
            at = torch.arange(R, device="cuda", dtype=torch.int32) + step
            want = te.rotary_rows(x, at, R, L, H, hd, rotary, ctx=gpu_ctx)
            torch.cuda.synchronize()
            assert torch.equal(out, want), step


def test_frequencies():
    f = te.rotary_frequencies(64, 1e4)
    assert f.dtype == np.float64 and np.allclose(
        f, 1e4 ** (-np.arange(32) / 32) / (2 * np.pi), rtol=1e-14)
    assert np.allclose(te.rotary_frequencies(64, 1e4, scaling="linear", factor=4), f / 4, rtol=1e-15)
    base = te.rotary_frequencies(64, 1e4, scaling="base", factor=4)
    assert np.isclose(base[0], f[0]) and np.isclose(base[-1], f[-1] / 4)
    bands = te.rotary_frequencies(64, 1e4, scaling="bands", factor=8, trained_length=1000,
                                  low_turns=1, high_turns=4)
    turns = f * 1000
    assert np.array_equal(bands[turns >= 4], f[turns >= 4])
    assert np.array_equal(bands[turns <= 1], f[turns <= 1] / 8)
    between = (turns > 1) & (turns < 4)
    assert between.any() and ((bands < f) & (bands > f / 8))[between].all()
    assert te.rotary_frequencies(0, 1e4).size == 0
    for bad in (dict(rotary_dim=3, theta=1e4), dict(rotary_dim=4, theta=0.0),
                dict(rotary_dim=4, theta=1.0, scaling="linear", factor=0.0),
                dict(rotary_dim=2, theta=1.0, scaling="base", factor=2.0),
                dict(rotary_dim=4, theta=1.0, scaling="bands", factor=2.0),
                dict(rotary_dim=4, theta=1.0, scaling="twist")):
        with pytest.raises(te.InvalidArgument):
            te.rotary_frequencies(**bad)


def test_refusals():
    x = np.zeros(2 * 3 * 8, np.float32)
    f = te.rotary_frequencies(8, 1e4)
    call = lambda x=x, p=None, hd=8, rotary=te.Rotary(f), **kw: te.rotary_rows(
        x, p, 2, 3, 1, hd, rotary, ctx=te.Context(0), **kw)
    for kw, text in ((dict(x=x[:-1]), "x: 47"), (dict(p=np.zeros(5, np.int32)), "positions: 5"),
                     (dict(rotary=te.Rotary(np.zeros(5))), "rotary_dim must not exceed"),
                     (dict(rotary=te.Rotary(np.array([np.nan]))), "finite"),
                     (dict(out=np.zeros(48, np.float64)), "to update"),
                     (dict(out=np.zeros(47, np.float32)), "out: 47")):
        with pytest.raises(te.InvalidArgument, match=text):
            call(**kw)
    with pytest.raises(te.Unsupported, match="rotary_dim 260"):
        te.rotary_rows(np.zeros(260, np.float32), None, 1, 1, 1, 260, te.Rotary(np.zeros(130)),
                       ctx=te.Context(0))
    # At the C entry: odd dims, missing frequencies, unknown flags.
    with te.Context(0) as ctx:
        fn = ctx._lib.tfd_rotary_rows_f32
        bits = te.f32_bits(1.0)
        for dim, freq, flags, text in ((3, f.ctypes.data, 0, "even"), (4, None, 0, "frequencies"),
                                       (4, f.ctypes.data, te.TFD_TRIM_LEADING, "flag"),
                                       (4, f.ctypes.data, te.TFD_ASYNC, "TFD_ASYNC")):
            with pytest.raises(te.InvalidArgument, match=text):
                ctx.check(fn(ctx.handle, 2, 3, 1, 8, dim, x.ctypes.data, None, freq, bits,
                             x.ctypes.data, flags))
        with pytest.raises(te.InvalidArgument, match="null buffer"):
            ctx.check(fn(ctx.handle, 2, 3, 1, 8, 4, None, None, f.ctypes.data, bits, x.ctypes.data, 0))
        with pytest.raises(te.InvalidArgument, match="overflow"):
            ctx.check(fn(ctx.handle, 1 << 40, 1 << 40, 1, 8, 4, x.ctypes.data, None, f.ctypes.data,
                         bits, x.ctypes.data, 0))
        assert fn(ctx.handle, 0, 3, 1, 8, 4, None, None, f.ctypes.data, bits, None, 0) == te.TFD_OK
    assert ctx is not None
