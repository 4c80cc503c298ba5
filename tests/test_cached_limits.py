"""The paged cache's operators and the turns at their limits: more rows than one launch's grid holds in
one dimension (rows repeat, so that the first ones are checked against the formula and all others
against them), caches and features past 2^31, and rows and pages that do not fit."""
import numpy as np
import pytest

import tenferro_ext as te
from test_cache_append import EPS, Cache, operands, run
from test_cached_attention import call, check, filled, problem, reference
from test_linear_attention import cuda, host
from test_rotary import normal, turned


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
def test_turns_of_70000_rows(gpu_ctx, bf16):
    R, of, H, hd = 70000, 7, 2, 10
    x = normal(3, of, H, hd, 1)
    if bf16:
        x = te.bf16_bits_to_f32(te.to_bf16_bits(x))
    at = 1000 * np.arange(of, dtype=np.int32)
    rotary = te.Rotary(te.rotary_frequencies(8, 1e4), True)
    bits = te.to_bf16_bits(x).view(np.int16) if bf16 else x
    got = te.rotary_rows(cuda(bits.reshape(-1)).repeat(R // of), cuda(at).repeat(R // of), R, 1, H, hd,
                         rotary, bf16=bf16, ctx=gpu_ctx).view(R // of, -1)
    assert (got == got[0]).all()
    y = host(got[0])
    y = te.bf16_bits_to_f32(y.view(np.uint16)) if bf16 else y
    want, size = turned(x, at[:, None], rotary)
    off = np.abs(y.reshape(want.shape) - want)
    assert (off <= 9 * 2.0**-24 * size + (2.0**-8 * np.abs(want) if bf16 else 0)).all()


@pytest.mark.gpu
def test_attention_of_4_million_tiles(gpu_ctx):
    """65535 rows of 65 kv heads, which share five rows' pages."""
    R, of, H, hd = 65535, 5, 65, 8
    before, counts = np.array([0, 1, 17, 62, 63]), np.ones(of, np.int64)
    ref = filled(of, H, hd, 64, before + counts)
    q = normal(4, of, H, hd, 1)
    want, tol = reference(ref, q, None, None, None, before, counts)
    i32 = lambda x: cuda(np.ascontiguousarray(x, dtype=np.int32).reshape(-1)).repeat(R // of)
    got = te.jeff_cached_attention(cuda(q.reshape(-1)).repeat(R // of), None, None, ref.paged(cuda),
                                   i32(ref.table), i32(before), None, R, 1, H, H, hd, None, EPS,
                                   ctx=gpu_ctx).view(R // of, -1)
    assert (got == got[0]).all()
    check(host(got[0]), want, tol)


@pytest.mark.gpu
def test_append_of_a_million_heads(gpu_ctx):
    """65535 rows of 17 kv heads: 9 GB of pages."""
    import torch

    R, HK, hd = 65535, 17, 8
    k, v = normal(5, 1, HK, hd, 1), normal(6, 1, HK, hd, 1)
    ref = Cache(1, HK, hd, 64, 1)
    ref.table[:] = 0
    ref.append(k, v, None, None, np.ones(1, np.int64))
    cache = te.paged_cache(R, HK, hd, 64, device="cuda")
    te.jeff_cache_append(cuda(k.reshape(-1)).repeat(R), cuda(v.reshape(-1)).repeat(R), None, cache,
                         torch.arange(R, dtype=torch.int32, device="cuda").flip(0), None, None, R, 1, HK,
                         hd, None, EPS, ctx=gpu_ctx)
    keys = cache.keys.view(torch.uint8).view(R, HK, 64, 64)
    values = cache.values.view(torch.uint8).view(R, HK, 64, 64)
    assert (keys[:, :, 0] == cuda(ref.keys[0, :, 0])).all()
    assert (values[:, :, :hd, 0] == cuda(ref.values[0, :, 0, :hd, 0])).all()
    for got, want in ((cache.key_scales, ref.ks), (cache.value_scales, ref.vs)):
        assert (got.view(R, HK) == cuda(want[0, :, 0])).all()
    del cache, keys, values
    torch.cuda.empty_cache()


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("L", [1, 130])
def test_append_past_31_bits_of_a_cache(gpu_ctx, L, bf16):
    """2.2e9 bytes of keys, the rows' pages the last ones; the others stay as they were."""
    import torch

    R, HK, hd, page, pages = 2, 2, 256, 1024, 4200
    ref = Cache(R, HK, hd, page, 1, spare=0)
    ref.lengths[:] = 30, 890
    for x in (ref.keys, ref.values):
        x[:] = 0x38
    ref.ks[:] = ref.vs[:] = 2.0**-8
    big = te.paged_cache(pages, HK, hd, page, device="cuda")
    assert big.keys.numel() > 2**31
    for x, y in zip(big[:4], ref.paged(cuda)[:4]):
        x.view(y.dtype)[-y.numel():] = y
    k, v = operands(7, R, HK, hd, L, bf16)
    rotary = te.Rotary(te.rotary_frequencies(64, 1e4))
    norm, counts, lengths = normal(2, hd) * np.float32(0.1), np.array([L, L]), ref.lengths.copy()
    ref.append(k, v, norm, rotary, counts)
    ref.table += pages - ref.pages
    run(gpu_ctx, ref, big, k, v, norm, rotary, counts, lengths, bf16)
    ends = [x.view(torch.uint8 if i < 2 else torch.float32)[-y.size:] for i, (x, y) in enumerate(
        zip(big[:4], (ref.keys, ref.values, ref.ks, ref.vs)))]
    assert ref.same(ends) == [True] * 4
    for x, end in zip(big[:2], ends):
        assert not x.view(torch.int64)[:-end.numel() // 8].any()
    del big, ends, x, end
    torch.cuda.empty_cache()


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("R,L", [(2, 1), (33, 20)], ids=["single", "prompt"])
def test_attention_past_31_bits_of_a_cache(gpu_ctx, R, L, bf16):
    import torch

    H, HK, hd, page, pages = 16, 2, 256, 128, 33600
    before, counts = np.array([(1500, 30)[r % 2] + r for r in range(R)]), np.full(R, L)
    ref = filled(R, HK, hd, page, before + counts)
    big = te.paged_cache(pages, HK, hd, page, device="cuda")
    assert big.keys.numel() > 2**31
    for x, y in zip(big[:4], ref.paged(cuda)[:4]):
        x.view(y.dtype)[-y.numel():] = y
    q, gate = problem(R, H, hd, L, bf16)
    want, tol = reference(ref, q, gate, None, None, before, counts)
    ref.table += pages - ref.pages
    check(call(gpu_ctx, ref, q, gate, None, None, before, counts, bf16, cache=big), want, tol)
    del big, x, y
    torch.cuda.empty_cache()


@pytest.mark.gpu
@pytest.mark.parametrize("R,L,H,hd", [(130, 8192, 16, 128), (1, 1 << 24, 1, 130)])
def test_turns_past_31_bits(gpu_ctx, R, L, H, hd):
    """2.2e9 bf16 features, by rows and in one: the same ones for every token, so that the turns of the
    first and the last tokens of the last row tell whether all are where they belong."""
    import torch

    x = normal(3, H * hd)
    x = te.bf16_bits_to_f32(te.to_bf16_bits(x))
    rotary = te.Rotary(te.rotary_frequencies(64, 1e7), False, 1.25)
    features = cuda(te.to_bf16_bits(x).view(np.int16)).view(torch.bfloat16)
    whole = features[:, None].expand(R, H * hd, L).reshape(-1)
    assert whole.numel() > 2**31
    got = te.rotary_rows(whole, None, R, L, H, hd, rotary, bf16=True, ctx=gpu_ctx)
    got = got.view(R, H * hd, L)
    at = np.r_[0:3, L // 2:L // 2 + 3, L - 3:L]
    want, size = turned(np.repeat(x.reshape(1, H, hd, 1), at.size, 3), at[None], rotary)
    for r in (0, R - 1):
        y = host(got[r][:, cuda(at)].float()).reshape(want.shape)
        assert (np.abs(y - want) <= 9 * 2.0**-24 * size + 2.0**-8 * np.abs(want)).all()
    assert all((got[r] == got[0]).all() for r in range(1, R))
    del whole, got
    torch.cuda.empty_cache()


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
def test_of_rows_and_pages_that_do_not_fit_nothing_is_written(gpu_ctx, bf16):
    """Device operands: keys, values and both scales stay, but for the tokens of a row whose pages are
    sound up to them."""
    R, HK, hd, L = 6, 2, 64, 3
    k, v = operands(8, R, HK, hd, L, bf16)
    ref = Cache(R, HK, hd, 64, 2)
    p = ref.table[5, 0]  # row 5 goes from its first page to one that is not there
    ref.keys[p, :, :62], ref.values[p, ..., :62] = 0x30, 0xB1
    ref.ks[p] = ref.vs[p] = 2.0**-10
    cache = ref.paged(cuda)
    lengths = np.array([126, -1, 0, 0, 0, 62], np.int32)
    ref.lengths[5] = 62
    ref.append(k[..., :2], v[..., :2], None, None, np.array([0, 0, 0, 0, 0, 2]))
    assert ref.ks[p].min() > 2.0**-10 and ref.vs[p].min() > 2.0**-10  # earlier codes go on, too
    ref.table[3, 0], ref.table[4, 0], ref.table[5, 1] = ref.pages, -1, 2**31 - 1
    run(gpu_ctx, ref, cache, k, v, None, None, np.array([3, 3, 4, 3, 3, 3]), lengths, bf16)
    assert ref.same(cache) == [True] * 4
