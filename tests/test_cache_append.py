"""Appending to the paged 8-bit cache against the formula in 64 bits, code for code.

Keys are computed in 64 bits, as they are here: the two differ by some 2^-50 of a value, so
no value of these inputs is near enough to a border between codes for them to differ.
"""
import numpy as np
import pytest

import tenferro_ext as te
from test_linear_attention import cuda, host
from test_rotary import normal, turned

EPS = 1e-6


def _e4m3():
    """Value of every code."""
    c = np.arange(256)
    e, m = (c >> 3) & 15, c & 7
    v = np.where(e == 0, m * 2.0**-9, (1 + m / 8) * 2.0 ** (e.astype(float) - 7))
    v = np.where((c & 127) == 127, np.nan, v)
    return np.where(c & 128, -v, v)


E4M3 = _e4m3()


def encode(x):
    """Codes of x (64 bits) to nearest even; what is over 448 or not finite the code of NaN."""
    a = np.abs(x)
    with np.errstate(invalid="ignore", divide="ignore"):
        step = np.exp2(np.maximum(np.floor(np.log2(np.where(a > 0, a, 1))), -6) - 3)
        r = np.rint(a / step) * step
    found = np.searchsorted(E4M3[:127], np.nan_to_num(np.minimum(r, 448.0)))
    code = np.where(np.signbit(x), found | 128, found)
    return np.where(a <= 448, code, 127).astype(np.uint8)


def scale_for(most):
    """Smallest power of two s >= 2^-100 with most <= 448 s."""
    m, e = np.frexp(most)
    return 2.0 ** max(-100, e - 9 + (m > 0.875)) if most > 0 else 2.0**-100


class Cache:
    """A cache and its rows on the host, updated by the formula; `paged` copies it."""

    def __init__(self, R, HK, hd, page, per_row, spare=3, seed=5, fill=0x7F):
        self.R, self.HK, self.hd, self.page, self.per_row = R, HK, hd, page, per_row
        self.wide = -(-hd // 64) * 64
        self.pages = R * per_row + spare
        rng = np.random.default_rng(seed)
        self.table = rng.permutation(self.pages)[:R * per_row].astype(np.int32).reshape(R, per_row)
        # What was in memory: NaN codes everywhere, and scales that nothing may read.
        self.keys = np.full((self.pages, HK, page, self.wide), fill, np.uint8)
        self.values = np.full((self.pages, HK, page // 64, self.wide, 64), fill, np.uint8)
        self.ks = np.full((self.pages, HK, page // 64), 2.0**60, np.float32)
        self.vs = np.full((self.pages, HK, page // 64), 2.0**60, np.float32)
        self.lengths = np.zeros(R, np.int32)

    def paged(self, to=lambda x: x):
        return te.PagedCache(*(to(x.reshape(-1).copy()) for x in
                               (self.keys, self.values, self.ks, self.vs)), self.page)

    def same(self, cache):
        """Where the flat buffers of `cache` hold what this one does."""
        got = [(x if isinstance(x, np.ndarray) else host(x)).reshape(-1) for x in cache[:4]]
        return [np.array_equal(g.view(np.uint8), w.reshape(-1).view(np.uint8))
                for g, w in zip(got, (self.keys, self.values, self.ks, self.vs))]

    def append(self, k, v, norm, rotary, counts):
        """k, v (R, HK, hd, L): the last counts[r] tokens of each row."""
        R, HK, hd, L = k.shape
        k, v = k.astype(np.float64), v.astype(np.float64)
        with np.errstate(invalid="ignore", over="ignore"):
            if norm is not None:
                k = k / np.sqrt((k * k).mean(2, keepdims=True) + float(np.float32(EPS)))
                k = k * (1 + norm.astype(np.float64))[:, None]
            at = self.lengths[:, None] + np.arange(L) - (L - counts[:, None])
            if rotary is not None:
                k = turned(k, at, rotary)[0]
        for r in range(R):
            for h in range(HK):
                n = int(self.lengths[r])
                while n < self.lengths[r] + counts[r]:
                    b = n // 64
                    end = min(64 * b + 64, int(self.lengths[r] + counts[r]))
                    p, i = self.table[r, b * 64 // self.page], b % (self.page // 64)
                    t = slice(L - counts[r] + n - self.lengths[r], L - counts[r] + end - self.lengths[r])
                    s = slice(n - 64 * b, end - 64 * b)
                    keys = self.keys[p, h, 64 * i:64 * i + 64]
                    vals = self.values[p, h, i].T  # (64, wide)
                    for x, codes, scales in ((k, keys, self.ks), (v, vals, self.vs)):
                        new = x[r, h, :, t].T
                        scale = scale_for(np.abs(np.where(np.isfinite(new), new, 0)).max())
                        if s.start:
                            before = float(scales[p, h, i])
                            if before >= scale:
                                scale = before
                            else:
                                again = encode(E4M3[codes[:s.start]] * before / scale)
                                kept = (codes[:s.start] & 127) == 127
                                codes[:s.start] = np.where(kept, codes[:s.start], again)
                        codes[s, :hd] = encode(new / scale)
                        scales[p, h, i] = scale
                    keys[s, hd:] = 0
                    n = end
        self.lengths = self.lengths + counts.astype(np.int32)


def operands(seed, R, HK, hd, L, bf16):
    k, v = normal(seed, R, HK, hd, L), normal(seed + 1, R, HK, hd, L) * np.float32(0.3)
    if bf16:
        k, v = (te.bf16_bits_to_f32(te.to_bf16_bits(x)) for x in (k, v))
    return k, v


def run(ctx, ref, cache, k, v, norm, rotary, counts, lengths, bf16, to=cuda):
    R, HK, hd, L = k.shape
    bits = te.to_bf16_bits if bf16 else lambda x: x
    i32 = lambda x: to(np.ascontiguousarray(x, dtype=np.int32).reshape(-1))
    te.jeff_cache_append(to(bits(k).reshape(-1)), to(bits(v).reshape(-1)),
                         None if norm is None else to(norm), cache, i32(ref.table), i32(lengths),
                         i32(counts), R, L, HK, hd, rotary, EPS, bf16=bf16, ctx=ctx)


CASES = [
    # HK, head_dim, rotary_dim, interleaved, page, lengths of the calls
    (2, 256, 64, False, 64, (1, 1, 70, 1)),
    (1, 8, 8, True, 64, (3, 61, 1, 64)),
    (3, 33, 32, False, 128, (65, 1, 5)),
    (2, 96, 96, True, 64, (1, 63, 130)),
    (1, 128, 0, False, 256, (200, 2, 1, 1)),
    (1, 192, 192, False, 64, (64, 64, 1)),
    (2, 256, 256, True, 128, (127, 2, 300)),
]


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c[:3])))
def test_code_for_code(gpu_ctx, case, bf16):
    """Several calls one after another, of ragged rows, one of which never gets a token."""
    HK, hd, rot, interleaved, page, calls = case
    R = 4
    ref = Cache(R, HK, hd, page, -(-sum(calls) // page) + 1)
    cache = ref.paged(cuda)
    rotary = te.Rotary(te.rotary_frequencies(rot, 1e4), interleaved, 1.5) if rot else None
    norm = None if hd == 128 else normal(2, hd) * np.float32(0.1)
    for n, L in enumerate(calls):
        k, v = operands(17 * n + hd, R, HK, hd, L, bf16)
        # Each call larger than the one before: scales grow within blocks.
        k, v = k * np.float32(2.0**n), v * np.float32(2.0 ** (2 * n))
        counts = np.array([L, (L + 1) // 2, 0, max(0, L - 7)], np.int32)
        k[1, :, :, :L - counts[1]] = np.nan  # not active: not used
        lengths = ref.lengths.copy()
        ref.append(k, v, norm, rotary, counts)
        run(gpu_ctx, ref, cache, k, v, norm, rotary, counts, lengths, bf16)
        assert ref.same(cache) == [True] * 4, (n, ref.same(cache))


@pytest.mark.gpu
def test_single_tokens_leave_a_prompts_codes(gpu_ctx):
    """Falling sizes: no scale grows, so the order of the calls does not matter."""
    R, HK, hd, L = 2, 2, 64, 150
    k, v = operands(3, R, HK, hd, L, False)
    fall = (2.0 ** (-np.arange(L) // 8)).astype(np.float32)
    k, v = np.abs(k).clip(1, 1.5) * fall, np.abs(v).clip(1, 1.5) * fall
    rotary = None
    one, many = (Cache(R, HK, hd, 64, 3) for _ in range(2))
    a, b = one.paged(cuda), many.paged(cuda)
    run(gpu_ctx, one, a, k, v, None, rotary, np.full(R, L), np.zeros(R), False)
    for t in range(L):
        run(gpu_ctx, many, b, np.ascontiguousarray(k[..., t:t + 1]),
            np.ascontiguousarray(v[..., t:t + 1]), None, rotary, np.ones(R), np.full(R, t), False)
    for x, y in zip(a[:4], b[:4]):
        assert np.array_equal(host(x).view(np.uint8), host(y).view(np.uint8))


@pytest.mark.gpu
def test_sizes_at_the_borders(gpu_ctx):
    """All codes and the middles between them, scales at 448 and just over, blocks of zeros, tiny
    and huge values, NaN and inf."""
    R, HK, hd, L = 1, 1, 64, 64 * 9
    v = np.zeros((hd, L), np.float32)
    grid = np.concatenate([E4M3[:127], (E4M3[1:127] + E4M3[:126]) / 2])
    grid = np.concatenate([grid, -grid, grid * (1 + 2.0**-20), -grid * (1 - 2.0**-20)])
    v[:, :64] = np.resize(grid.astype(np.float32), (hd, 64)).clip(-448, 448)
    v[:, 64:128] = v[:, :64] * 2.0**-30
    v[0, 128] = 448.0
    v[0, 192] = np.nextafter(np.float32(448.0), np.float32(500.0))
    v[:, 320:384] = np.float32(1e-38) * np.arange(64)
    v[:, 384:448] = np.float32(3e38) * (np.arange(64) - 32) / 32
    v[:, 448:512] = 1.0
    v[3, 450], v[4, 451], v[5, 452] = np.nan, np.inf, -np.inf
    v[:, 512:] = 1.0
    v[:, 513] = np.nan
    v = v.reshape(R, HK, hd, L)
    ref = Cache(R, HK, hd, 64, 9)
    cache = ref.paged(cuda)
    counts = np.full(1, L)
    ref.append(v, v, None, None, counts)
    run(gpu_ctx, ref, cache, v, v, None, None, counts, np.zeros(1), False)
    assert ref.same(cache) == [True] * 4


@pytest.mark.gpu
def test_host_arrays_and_defaults(gpu_ctx):
    R, HK, hd, L = 2, 1, 20, 5
    k, v = operands(8, R, HK, hd, L, False)
    ref = Cache(R, HK, hd, 64, 1)
    cache = ref.paged()
    te.jeff_cache_append(k.reshape(-1), v.reshape(-1), None, cache, ref.table.reshape(-1), None, None,
                         R, L, HK, hd, None, EPS, ctx=gpu_ctx)
    ref.append(k, v, None, None, np.full(R, L))
    assert ref.same(cache) == [True] * 4


@pytest.mark.gpu
def test_rows_and_pages_that_do_not_fit_are_left(gpu_ctx):
    """Device operands, which only the kernel sees: such a row or page is not written."""
    R, HK, hd, L = 6, 2, 64, 3
    k, v = operands(8, R, HK, hd, L, False)
    ref = Cache(R, HK, hd, 64, 2)
    cache = ref.paged(cuda)
    table = ref.table.copy()
    table[3, 0], table[4, 0] = ref.pages, -1
    lengths = np.array([126, -1, 0, 0, 0, 62])  # row 5 crosses into its second page
    counts = np.array([3, 3, 4, 3, 3, 3])
    table[5, 1] = 2**31 - 1
    te.jeff_cache_append(cuda(k.reshape(-1)), cuda(v.reshape(-1)), None, cache,
                         cuda(table.reshape(-1)), cuda(lengths.astype(np.int32)),
                         cuda(counts.astype(np.int32)), R, L, HK, hd, None, EPS, ctx=gpu_ctx)
    # Of all the rows only row 5's first page gets its two tokens.
    got = host(cache[0]).view(np.uint8).reshape(ref.keys.shape)
    p = table[5, 0]
    assert (got[p, :, 62:] == encode_block(k[5, :, :, :2], ref, host(cache[2]), p)).all()
    got[p, :, 62:] = 0x7F
    assert (got[p, :, :62] == 0x7F).all() and (np.delete(got, p, 0) == 0x7F).all()


def encode_block(k, ref, scales, p):
    s = scales.reshape(ref.ks.shape)[p]  # (HK, 1): that of the block before, which never falls
    assert (s == 2.0**60).all()
    return encode(k.transpose(0, 2, 1).astype(np.float64) / s[:, :, None])


def refusal_call(**change):
    R, HK, hd, L = 2, 2, 64, 3
    cache = te.paged_cache(4, HK, hd)
    a = dict(k=np.zeros(R * HK * hd * L, np.float32), v=np.zeros(R * HK * hd * L, np.float32),
             k_norm=np.zeros(hd, np.float32), cache=cache, pages=np.arange(4, dtype=np.int32),
             lengths=np.zeros(R, np.int32), counts=np.full(R, L, np.int32), rows=R, length=L,
             kv_heads=HK, head_dim=hd, rotary=te.Rotary(te.rotary_frequencies(32, 1e4)), eps=EPS)
    a.update({n: (f(a[n]) if callable(f) else f) for n, f in change.items()})
    with te.Context(0) as ctx:
        te.jeff_cache_append(**a, ctx=ctx)


@pytest.mark.parametrize("change,text", [
    (dict(k=lambda x: x[1:]), "k: 767"),
    (dict(v=lambda x: x[1:]), "v: 767"),
    (dict(k_norm=lambda x: x[1:]), "k_norm: 63"),
    (dict(cache=lambda c: c._replace(keys=c.keys[1:])), "to update|elements"),
    (dict(cache=lambda c: c._replace(keys=c.keys[:-1].copy())), "values|whole pages"),
    (dict(cache=lambda c: c._replace(keys=c.keys.astype(np.int16))), "keys: expected a contiguous uint8"),
    (dict(cache=lambda c: c._replace(key_scales=c.key_scales[:-1].copy())), "key_scales: 7"),
    (dict(cache=lambda c: c._replace(value_scales=c.value_scales.astype(np.float64))), "value_scales"),
    (dict(cache=lambda c: c._replace(page_tokens=96)), "power of two"),
    (dict(cache=lambda c: c._replace(page_tokens=32)), "power of two"),
    (dict(pages=lambda x: x[1:]), "pages: 3"),
    (dict(pages=lambda x: x + 4), "outside the cache"),
    (dict(pages=lambda x: -x), "outside the cache"),
    (dict(pages=lambda x: x * 0), "append to one page"),
    (dict(lengths=lambda x: x - 1), "negative"),
    (dict(lengths=lambda x: x + 126), "do not hold"),
    (dict(lengths=lambda x: x[1:]), "lengths: 1"),
    (dict(counts=lambda x: x + 1), "more than its tokens"),
    (dict(counts=lambda x: x - 4), "negative"),
    (dict(counts=lambda x: x[1:]), "counts: 1"),
    (dict(rotary=te.Rotary(np.zeros(33))), "rotary_dim must not exceed"),
    (dict(rotary=te.Rotary(np.array([np.inf]))), "finite"),
])
def test_refusals(change, text):
    with pytest.raises(te.InvalidArgument, match=text):
        refusal_call(**change)


def test_refusals_of_the_c_entry():
    with te.Context(0) as ctx:
        fn = ctx._lib.tfd_jeff_cache_append_f32
        c = te.paged_cache(1, 1, 64)
        s = te._PagedCacheStruct(*(x.ctypes.data for x in c[:4]), 1, 64)
        x, table = np.zeros(64, np.float32), np.zeros(1, np.int32)
        import ctypes

        def call(hd=64, struct=s, per_row=1, pages=table.ctypes.data, flags=0, rows=1, length=1, heads=1):
            ctx.check(fn(ctx.handle, rows, length, heads, hd, 0, x.ctypes.data, x.ctypes.data, None,
                         None, te.f32_bits(1.0), te.f32_bits(EPS),
                         None if struct is None else ctypes.byref(struct), pages, per_row, None, None,
                         flags))

        bad = te._PagedCacheStruct(None, *(x.ctypes.data for x in c[1:4]), 1, 64)
        odd = te._PagedCacheStruct(c[0].ctypes.data + 1, *(x.ctypes.data for x in c[1:4]), 1, 64)
        for kw, text in ((dict(struct=None), "null cache"), (dict(struct=bad), "null buffer"),
                         (dict(pages=None), "null buffer"), (dict(per_row=0), "need a page"),
                         (dict(flags=te.TFD_INVERSE), "flag"),
                         (dict(struct=odd, flags=te.TFD_DEVICE_PTRS), "16-byte"),
                         (dict(rows=1 << 40, length=1 << 40), "overflow")):
            with pytest.raises(te.InvalidArgument, match=text):
                call(**kw)
        for kw, text in ((dict(hd=257), "head_dim 257"), (dict(per_row=1 << 26), "31 bits"),
                         (dict(length=1 << 25), "launch grid")):
            with pytest.raises(te.Unsupported, match=text):
                call(**kw)
        call(rows=0)
        call(length=0)
