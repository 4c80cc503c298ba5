"""Many rows of the paged cache's operators and of the turns: calls past what one launch's grid holds
in one dimension. Rows repeat, so that the first ones are checked against the formula and all others
against them."""
import numpy as np
import pytest

import tenferro_ext as te
from test_cache_append import EPS, Cache
from test_cached_attention import check, filled, reference
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
