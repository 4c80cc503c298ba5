"""Attention over the paged 8-bit cache against the formula in 64 bits, on the codes and scales
that the cache holds.

Tolerance, in units of u = 2^-24. A normalized, turned query feature carries at most 28 roundings
(norm: 9 of a sum of 256 squares, its root, reciprocal, two products; turn: 9 of
test_rotary; two fp16 pieces of 11 bits: 2^-22, which is 4), each at most u of the features that
enter it; a score's sum of 3 hd products
six standard deviations of independent roundings, 6 sqrt(3 hd). All are taken on the sum of the
products' absolute values (`size`; a turned pair mixes two features, which 2 covers), and
e^score is off by twice that (numerator and denominator) plus 4 u |score| of the score's scaling and
its difference from the reference. exp2, two fp16 pieces, scales and sums over T keys add 20 + 6 sqrt(3 T)
u, the gate 8 + 2 |gate|. All on the sum of p |v| times the gate. Beside it a probability, which
is at most 1 against the row's largest, is held times 2^11 to 2^15 in fp16 pieces whose last step is 2^-24:
it is off by up to 2^-25 / 2^11 = 2^-36 however small it is, on the sum of |v| (the sum of the
probabilities, which divides it, is at least 1). That shows where the largest probabilities meet
values of 0.
"""
import numpy as np
import pytest

import tenferro_ext as te
from test_cache_append import E4M3, EPS, Cache
from test_linear_attention import cuda, host
from test_rotary import normal, pair_index, turned

U = 2.0**-24


def reference(ref, q, gate, norm, rotary, before, counts):
    """q, gate (R, H, hd, L); the cache holds before[r] + counts[r] tokens: out and tolerance."""
    R, H, hd, L = q.shape
    x, group = q.astype(np.float64), H // ref.HK
    with np.errstate(invalid="ignore", over="ignore"):
        if norm is not None:
            x = x / np.sqrt((x * x).mean(2, keepdims=True) + float(np.float32(EPS)))
            x = x * (1 + norm.astype(np.float64))[:, None]
        at = before[:, None] + np.arange(L) - (L - counts[:, None])
        mag = np.abs(x)
        if rotary is not None:
            x = turned(x, at, rotary)[0]
            a, b = pair_index(2 * len(rotary.frequencies), rotary.interleaved)
            mag[:, :, a] = mag[:, :, b] = (mag[:, :, a] + mag[:, :, b]) * abs(rotary.magnitude)
    out, tol = np.zeros((2, R, H, hd, L))
    for r in range(R):
        n, c = int(before[r]), int(counts[r])
        if not c:
            continue
        pages = ref.table[r, :-(-(n + c) // ref.page)]
        for h in range(ref.HK):
            k = E4M3[ref.keys[pages, h]] * np.repeat(ref.ks[pages, h], 64, 1)[:, :, None]
            v = E4M3[ref.values[pages, h]].transpose(0, 1, 3, 2) * ref.vs[pages, h][:, :, None, None]
            k = k.reshape(-1, ref.wide)[:n + c, :hd]
            v = v.reshape(-1, ref.wide)[:n + c, :hd]
            for j in range(h * group, (h + 1) * group):
                with np.errstate(invalid="ignore", over="ignore"):
                    s = x[r, j].T[L - c:] @ k.T / np.sqrt(hd)
                    size = mag[r, j].T[L - c:] @ np.abs(k).T / np.sqrt(hd)
                    seen = np.arange(n + c) <= at[r, L - c:, None]
                    s = np.where(seen, s, -np.inf)
                    p = np.exp(s - s.max(1, keepdims=True))
                    p /= p.sum(1, keepdims=True)
                    pv = np.where(seen[:, :, None], p[:, :, None] * v, 0).sum(1) if np.isnan(
                        v).any() else p @ v
                    e = 2 * ((28 + 6 * np.sqrt(3 * hd)) * 2 * np.where(seen, size, 0).max(1)
                             + 4 * np.where(seen, np.abs(s), 0).max(1)) + 20 + 6 * np.sqrt(3 * (n + c))
                    g = 1.0 if gate is None else 1 / (1 + np.exp(-gate[r, j].T[L - c:].astype(float)))
                    extra = 8 if gate is None else 8 + 2 * np.abs(gate[r, j].T[L - c:])
                    out[r, j, :, L - c:] = (pv * g).T
                    tol[r, j, :, L - c:] = ((e[:, None] + extra) * U * (p @ np.abs(np.nan_to_num(v)))
                                            * g).T
                    tol[r, j, :, L - c:] += 2.0**-36 * (seen @ np.abs(np.nan_to_num(v)) * g).T
    return out, tol


def filled(R, HK, hd, page, total, seed=3):
    """A cache whose rows hold total[r] tokens of ordinary codes, NaN codes behind them."""
    ref = Cache(R, HK, hd, page, max(1, -(-int(max(total)) // page)) + 1)
    rng = np.random.default_rng(seed)

    def codes(*shape):
        c = rng.integers(0, 0x77, shape).astype(np.uint8)  # up to 240
        return c | (rng.integers(0, 2, shape) * 128).astype(np.uint8)

    for r in range(R):
        for n in range(0, int(total[r]), 64):
            p, i = ref.table[r, n // page], n % page // 64
            m = min(64, int(total[r]) - n)
            ref.keys[p, :, 64 * i:64 * i + m, :hd] = codes(HK, m, hd)
            ref.keys[p, :, 64 * i:64 * i + m, hd:] = 0
            ref.values[p, :, i, :hd, :m] = codes(HK, hd, m)
            ref.ks[p, :, i] = 2.0 ** rng.integers(-9, -6, HK)
            ref.vs[p, :, i] = 2.0 ** rng.integers(-9, -6, HK)
    return ref


def call(ctx, ref, q, gate, norm, rotary, before, counts, bf16=False, to=cuda, cache=None, **kw):
    R, H, hd, L = q.shape
    bits = te.to_bf16_bits if bf16 else lambda x: x
    i32 = lambda x: to(np.ascontiguousarray(x, dtype=np.int32).reshape(-1))
    return te.jeff_cached_attention(
        to(bits(q).reshape(-1)), None if gate is None else to(bits(gate).reshape(-1)),
        None if norm is None else to(norm), ref.paged(to) if cache is None else cache,
        i32(ref.table), i32(before), i32(counts), R, L, H, ref.HK, hd, rotary, EPS, bf16=bf16,
        ctx=ctx, **kw)


def check(got, want, tol):
    got = (got if isinstance(got, np.ndarray) else host(got)).reshape(want.shape).astype(np.float64)
    bad = np.isnan(want)
    assert np.array_equal(np.isnan(got), bad), (np.isnan(got) != bad).sum()
    off = np.abs(got - want)[~bad]
    assert (off <= tol[~bad]).all(), (off / (tol[~bad] + 1e-30)).max()


def problem(R, H, hd, L, bf16, gate=True, seed=4):
    q, g = normal(seed, R, H, hd, L), normal(seed + 1, R, H, hd, L) if gate else None
    if bf16:
        q = te.bf16_bits_to_f32(te.to_bf16_bits(q))
        g = None if g is None else te.bf16_bits_to_f32(te.to_bf16_bits(g))
    return q, g


CASES = [
    # H, HK, head_dim, rotary_dim, interleaved, page, L, tokens before by row
    (8, 2, 256, 64, False, 64, 1, (0, 1, 62, 63, 64, 1000)),
    (4, 4, 128, 128, True, 128, 1, (127, 128, 5, 300)),
    (17, 1, 64, 64, False, 64, 1, (200, 0)),
    (6, 3, 33, 32, False, 64, 3, (0, 61, 62, 63, 64, 500)),
    (2, 2, 8, 8, True, 256, 17, (0, 250, 40)),
    (6, 2, 192, 192, False, 64, 70, (0, 1, 130)),
    (8, 2, 256, 64, False, 128, 200, (0, 77, 400)),
    (5, 1, 96, 0, False, 64, 40, (30, 2000)),
    (16, 2, 128, 64, True, 64, 5, (700, 3)),
    (8, 8, 64, 32, False, 64, 130, (0, 64)),
]


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, (*c[:4], c[6]))))
def test_against_the_formula(gpu_ctx, case, bf16):
    H, HK, hd, rot, interleaved, page, L, before = case
    R = len(before)
    before = np.array(before)
    counts = np.array([(L, L - L // 3, L, max(L - 1, 0), 0, L)[r] for r in range(R)])
    ref = filled(R, HK, hd, page, before + counts)
    q, gate = problem(R, H, hd, L, bf16, gate=H != 17)
    norm = None if H == 5 else normal(2, hd) * np.float32(0.1)
    rotary = te.Rotary(te.rotary_frequencies(rot, 1e4), interleaved, 1.25) if rot else None
    want, tol = reference(ref, q, gate, norm, rotary, before, counts)
    for r in range(R):
        q[r, :, :, :L - counts[r]] = np.nan  # not active: not used
    check(call(gpu_ctx, ref, q, gate, norm, rotary, before, counts, bf16), want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("R,H,HK,hd,L,before", [
    (1, 8, 2, 256, 1, (20000,)), (1, 1, 1, 64, 1, (40000,)), (2, 4, 2, 128, 4, (9000, 30)),
    (40, 4, 2, 128, 1, tuple(37 * r for r in range(40))),
    (1, 4, 1, 256, 300, (3000,)),
], ids=lambda x: str(x) if isinstance(x, int) else "")
def test_long_rows_in_parts(gpu_ctx, R, H, HK, hd, L, before):
    before, counts = np.array(before), np.full(R, L)
    ref = filled(R, HK, hd, 256, before + counts)
    q, gate = problem(R, H, hd, L, False)
    norm = normal(2, hd) * np.float32(0.1)
    rotary = te.Rotary(te.rotary_frequencies(hd, 1e6, scaling="linear", factor=4.0))
    want, tol = reference(ref, q, gate, norm, rotary, before, counts)
    check(call(gpu_ctx, ref, q, gate, norm, rotary, before, counts), want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("L", [1, 6, 150])
def test_large_scores(gpu_ctx, L):
    """Queries times 64: the softmax picks few keys, references move by hundreds."""
    before, counts = np.array([700, 90]), np.array([L, L])
    ref = filled(2, 1, 128, 64, before + counts)
    q, gate = problem(2, 4, 128, L, False)
    q *= np.float32(64)
    want, tol = reference(ref, q, gate, None, None, before, counts)
    check(call(gpu_ctx, ref, q, gate, None, None, before, counts), want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("L", [1, 7, 140])
def test_nan_reaches_what_sees_its_token(gpu_ctx, L):
    """NaN codes in keys and values of cached and of new tokens."""
    before, counts = np.array([100, 130, 3]), np.array([L, L, L])
    R, H, HK, hd = 3, 4, 2, 64
    ref = filled(R, HK, hd, 64, before + counts)

    def spoil(r, token, h, key):
        p, i = ref.table[r, token // 64], token % 64
        if key:
            ref.keys[p, h, i, 5] = 0x7F
        else:
            ref.values[p, h, 0, 7:9, i] = 0xFF
    spoil(0, 100 + L // 2, 0, False)  # seen by the second half of the new tokens, two features
    spoil(1, 130 + L // 2, 1, True)   # as a key: every feature
    spoil(1, 20, 0, False)
    q, gate = problem(R, H, hd, L, False)
    want, tol = reference(ref, q, gate, None, None, before, counts)
    assert np.isnan(want).any() and not np.isnan(want[2]).any()
    if L > 1:
        assert not np.isnan(want[0, :, :, 0]).any()
    check(call(gpu_ctx, ref, q, gate, None, None, before, counts), want, tol)


@pytest.mark.gpu
def test_rows_and_pages_that_do_not_fit_give_nan(gpu_ctx):
    """Device operands, which only the kernel sees."""
    R, H, HK, hd, L = 6, 4, 2, 64, 2
    before, counts = np.array([70, 70, 70, 70, 70, 70]), np.full(6, L)
    ref = filled(R, HK, hd, 64, before + counts)
    q, gate = problem(R, H, hd, L, False)
    want, tol = reference(ref, q, gate, None, None, before, counts)
    before[1], before[2], counts[3] = -1, 64 * ref.per_row - 1, L + 1
    ref.table[4, 0], ref.table[5, 1] = ref.pages, -5
    want[1:] = np.nan
    check(call(gpu_ctx, ref, q, gate, None, None, before, counts), want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("trim", [False, True])
def test_as_the_rows_op(gpu_ctx, trim):
    """Prompts whose normalized keys and whose values are e4m3 values: the same as the Jeff rows
    op, whose own error is within 2e-5."""
    R, H, HK, hd, L = 3, 8, 2, 256, 150
    q, gate = problem(R, H, hd, L, False)
    k = np.sign(normal(6, R, HK, hd, L))
    v = E4M3[np.abs(normal(7, R, HK, hd, L) * 20).astype(np.int64).clip(0, 60)].astype(np.float32) * k
    norm = normal(2, hd) * np.float32(0.1)
    counts = np.array([150, 90, 1]) if trim else np.full(R, L)
    mask = (np.arange(L) >= L - counts[:, None]).astype(np.float32)
    flat = lambda x: cuda(np.ascontiguousarray(x).reshape(-1))
    want = te.jeff_full_attention_rows(
        flat(q), flat(k), flat(v), flat(gate), cuda(norm), cuda(np.zeros(hd, np.float32)), flat(mask),
        R, L, H, HK, hd, 0, 1e4, 0.0, trim_leading=trim, ctx=gpu_ctx)
    cache = te.paged_cache(R * 3, HK, hd, device="cuda")
    table, n = cuda(np.arange(R * 3, dtype=np.int32)), flat(counts.astype(np.int32))
    te.jeff_cache_append(flat(k), flat(v), cuda(np.zeros(hd, np.float32)), cache, table, None, n, R, L,
                         HK, hd, None, 0.0, ctx=gpu_ctx)
    got = te.jeff_cached_attention(flat(q), flat(gate), cuda(norm), cache, table, None, n, R, L, H, HK,
                                   hd, None, 0.0, ctx=gpu_ctx)
    assert float((got - want).abs().max()) <= 4e-5


@pytest.mark.gpu
def test_host_arrays_out_and_shared_pages(gpu_ctx):
    R, H, HK, hd, L = 3, 4, 2, 40, 2
    before, counts = np.array([70, 64, 0]), np.array([2, 1, 2])
    ref = filled(R, HK, hd, 64, before + counts)
    ref.table[1, 0] = ref.table[0, 0]  # a shared prefix
    q, gate = problem(R, H, hd, L, False)
    want, tol = reference(ref, q, gate, None, None, before, counts)
    out = np.full(R * H * hd * L, np.nan, np.float32)
    got = call(gpu_ctx, ref, q, gate, None, None, before, counts, to=lambda x: x, out=out)
    assert got is out
    check(out, want, tol)
    check(call(gpu_ctx, ref, q, gate, None, None, before, counts), want, tol)


@pytest.mark.gpu
def test_same_bits_every_time(gpu_ctx):
    for L, before in ((1, (5000, 300)), (90, (2000, 10))):
        before, counts = np.array(before), np.array([L, L])
        ref = filled(2, 2, 256, 64, before + counts)
        q, gate = problem(2, 8, 256, L, False)
        first = host(call(gpu_ctx, ref, q, gate, None, None, before, counts))
        for _ in range(3):
            assert np.array_equal(first, host(call(gpu_ctx, ref, q, gate, None, None, before, counts)))


@pytest.mark.gpu
def test_past_31_bits_of_a_cache(gpu_ctx):
    """2.2e9 bytes of keys: the rows' pages are the last ones."""
    import torch

    R, H, HK, hd, page, L = 2, 4, 2, 256, 1024, 1
    before, counts = np.array([1500, 30]), np.array([1, 1])
    ref = filled(R, HK, hd, page, before + counts)
    pages = 4200
    big = te.paged_cache(pages, HK, hd, page, device="cuda")
    assert big.keys.numel() > 2**31
    for x, y in zip(big[:4], ref.paged(cuda)[:4]):
        x.view(y.dtype)[-y.numel():] = y
    q, gate = problem(R, H, hd, L, False)
    want, tol = reference(ref, q, gate, None, None, before, counts)
    ref.table += pages - ref.pages
    check(call(gpu_ctx, ref, q, gate, None, None, before, counts, cache=big), want, tol)
    del big
    torch.cuda.empty_cache()


@pytest.mark.parametrize("change,text", [
    (dict(q=lambda x: x[1:]), "q: "),
    (dict(gate=lambda x: x[1:]), "gate: "),
    (dict(q_norm=lambda x: x[1:]), "q_norm: 63"),
    (dict(kv_heads=3), "whole pages|multiple|elements"),
    (dict(heads=3, q=lambda x: x[:384], gate=None), "multiple of kv_heads"),
    (dict(pages=lambda x: x + 4), "outside the cache"),
    (dict(lengths=lambda x: x + 200), "do not hold"),
    (dict(counts=lambda x: x - 4), "negative"),
    (dict(out=np.zeros(5, np.float32)), "out: 5"),
    (dict(out=np.zeros(1536, np.float64)), "to update"),
    (dict(rotary=te.Rotary(np.zeros(40))), "rotary_dim must not exceed"),
])
def test_refusals(change, text):
    R, H, HK, hd, L = 2, 4, 2, 64, 3
    a = dict(q=np.zeros(R * H * hd * L, np.float32), gate=np.zeros(R * H * hd * L, np.float32),
             q_norm=np.zeros(hd, np.float32), cache=te.paged_cache(4, HK, hd),
             pages=np.arange(4, dtype=np.int32), lengths=np.zeros(R, np.int32),
             counts=np.full(R, L, np.int32), rows=R, length=L, heads=H, kv_heads=HK, head_dim=hd,
             rotary=None, eps=EPS)
    if change.get("heads") == 3:
        a.update(length=2, counts=np.full(R, 2, np.int32), q=np.zeros(768, np.float32))
        change = dict(change, q=a["q"])
    a.update({n: (f(a[n]) if callable(f) else f) for n, f in change.items()})
    with te.Context(0) as ctx, pytest.raises(te.InvalidArgument, match=text):
        te.jeff_cached_attention(**a, ctx=ctx)


def test_refuses_wide_heads():
    with te.Context(0) as ctx, pytest.raises(te.Unsupported, match="head_dim 300"):
        te.jeff_cached_attention(np.zeros(300, np.float32), None, None, te.paged_cache(1, 1, 300),
                                 np.zeros(1, np.int32), None, None, 1, 1, 1, 1, 300, None, EPS, ctx=ctx)
