"""The attention over the paged 8-bit cache where blocks' value scales lie far apart: the unit that
outputs are kept in follows the blocks, and must leave f32's range nowhere.

Queries are 0, so that all keys of a row weigh the same and the outputs are means of its values,
whose codes have one sign: sums are then as large as they can be. Tolerances are
test_cached_attention's.
"""
import numpy as np
import pytest

import tenferro_ext as te
from test_cache_append import Cache
from test_cached_attention import call, check, reference

HD, ZERO = 64, 2.0**-100  # ZERO: the scale that the append gives to a block of zeros

# R, H, HK, L. Single tokens: more (row, head) tiles than CUs, so that a row stays in one part and
# each of eight waves has every eighth of its blocks. Prompts: as many
# tiles of 128 columns, whose waves see every block.
SINGLE, PROMPT = (40, 16, 8, 1), (130, 8, 1, 20)


def blocks_of(scales, codes, R, HK, last=64):
    """R rows of len(scales) blocks of 64 tokens (the last one of `last`) on the same pages: block b's
    values are codes[b], its scale scales[b]; keys as they come."""
    n = len(scales)
    ref = Cache(1, HK, HD, 64, n, spare=0)
    for b, (scale, code) in enumerate(zip(scales, codes)):
        p = ref.table[0, b]
        ref.keys[p], ref.values[p], ref.vs[p], ref.ks[p] = 0x38, code, scale, 1.0
        if b == n - 1:
            ref.keys[p, :, last:], ref.values[p, ..., last:] = 0x7F, 0x7F  # behind the row
    ref.table = np.repeat(ref.table, R, 0)
    ref.R = R
    return ref, 64 * (n - 1) + last


def attend(ctx, ref, total, shape, bf16):
    R, H, HK, L = shape
    q = np.zeros((R, H, HD, L), np.float32)
    before, counts = np.full(R, total - L), np.full(R, L)
    want, tol = reference(ref, q[:1], None, None, None, before[:1], counts[:1])
    assert np.isfinite(want).all()
    got = call(ctx, ref, q, None, None, None, before, counts, bf16)
    check(got, np.repeat(want, R, 0), np.repeat(tol, R, 0))


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", [SINGLE, PROMPT], ids=["single", "prompt"])
@pytest.mark.parametrize("every", [1, 8], ids=["next_block", "next_of_eight"])
@pytest.mark.parametrize("first", [1.0, 2.0**-1, 2.0**-4, 2.0])
@pytest.mark.parametrize("zero", [ZERO, 0.0])
def test_zeros_behind_large_values(gpu_ctx, shape, every, first, zero, bf16):
    """Large values, zeros, larger ones, zeros, smaller ones, and a last block of a token's zeros."""
    scales = np.repeat([first, zero, 2.0**6, zero, 2.0**-3, 2.0**-9, zero], every)
    codes = np.repeat([0x7E, 0x00, 0x7E, 0x00, 0x7C, 0x7E, 0x00], every)
    R, H, HK, L = shape
    ref, total = blocks_of(scales, codes, R, HK, last=1)
    attend(gpu_ctx, ref, total, shape, bf16)


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", [SINGLE, PROMPT], ids=["single", "prompt"])
@pytest.mark.parametrize("first", [1.0, 2.0**-1])
def test_only_large_values_and_zeros(gpu_ctx, shape, first, bf16):
    """Nothing behind the zeros takes the unit back."""
    R, H, HK, L = shape
    ref, total = blocks_of([first] * 8 + [ZERO] * 8, [0x7E] * 8 + [0] * 8, R, HK)
    attend(gpu_ctx, ref, total, shape, bf16)


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape,large,zeros", [((256, 1, 1, 1), 2600, 8), (PROMPT, 330, 2)],
                         ids=["single", "prompt"])
def test_long_rows_of_large_values_and_zeros(gpu_ctx, shape, large, zeros, bf16):
    """A wave sums up 20800 values of 896: 2^15 times that is 2^39 units of 2."""
    R, H, HK, L = shape
    ref, total = blocks_of([2.0] * large + [ZERO] * zeros, [0x7E] * large + [0] * zeros, R, HK)
    attend(gpu_ctx, ref, total, shape, bf16)
