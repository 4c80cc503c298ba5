"""Host arrays that the cache's operators would have to convert: numbers that a 32-bit integer does
not hold, and codes that are not bytes, are refused before anything else happens."""
import numpy as np
import pytest

import tenferro_ext as te
from test_cache_append import EPS

R, H, HK, HD, L = 2, 4, 2, 64, 3


def attention(**change):
    a = dict(q=np.zeros(R * H * HD * L, np.float32), gate=None, q_norm=None, cache=te.paged_cache(4, HK, HD),
             pages=np.arange(4, dtype=np.int32), lengths=np.zeros(R, np.int32),
             counts=np.full(R, L, np.int32), rows=R, length=L, heads=H, kv_heads=HK, head_dim=HD,
             rotary=None, eps=EPS)
    a.update({n: f(a[n]) for n, f in change.items()})
    with te.Context(0) as ctx:
        te.jeff_cached_attention(**a, ctx=ctx)


@pytest.mark.parametrize("change,text", [
    (dict(pages=lambda x: x.astype(np.int64) + 2**32), "pages: not all"),
    (dict(lengths=lambda x: x.astype(np.int64) - 2**32), "lengths: not all"),
    (dict(counts=lambda x: x.astype(np.uint64) + 2**32), "counts: not all"),
    (dict(lengths=lambda x: x + 0.5), "lengths: not all"),
    (dict(lengths=lambda x: x + np.nan), "lengths: not all"),
    (dict(cache=lambda c: c._replace(keys=c.keys.astype(np.float32))), "keys: expected"),
    (dict(cache=lambda c: c._replace(values=c.values.astype(np.int64))), "values: expected"),
])
def test_refused(change, text):
    with pytest.raises(te.InvalidArgument, match=text):
        attention(**change)


def test_positions_past_31_bits_are_refused():
    x = np.zeros(8, np.float32)
    with te.Context(0) as ctx, pytest.raises(te.InvalidArgument, match="positions: not all"):
        te.rotary_rows(x, np.array([2**31]), 1, 1, 1, 8, te.Rotary(np.zeros(4)), ctx=ctx)


def test_other_integers_that_fit_are_taken():
    """Up to the next refusal."""
    with pytest.raises(te.InvalidArgument, match="outside the cache"):
        attention(pages=lambda x: list(x.astype(np.int64) + 4), lengths=lambda x: x.astype(np.float64),
                  counts=lambda x: x.astype(np.uint8))
