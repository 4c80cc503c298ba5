"""Cases of the rotary positions, of appending to a paged cache in 8 bits, and of the attention over it.

``kind`` names the operator:

* ``rotary``  rotary positions of heads of features (``rotary_rows``): pairs by halves or
              interleaved, on the first ``rotary`` features of a head, forwards or ``inverse``
              (the gradient)
* ``append``  keys (normalized, rotated) and values of new tokens into a paged cache
              (``jeff_cache_append``)
* ``attend``  causal attention of new tokens over the cache that holds them and the row's
              earlier ones (``jeff_cached_attention``), queries normalized and rotated, outputs gated

Layouts are the framework's: rows of (length, width) with the tokens contiguous. The cache's
pages hold whole blocks of 64 tokens; a head's features are padded with zeros to a multiple of 64
(``wide``). Per page and head: keys (page, wide), features contiguous; values (page / 64, wide, 64),
a block's tokens contiguous; a power of two per block of keys and of values, the scale of its e4m3
codes. ``pages`` (rows, pages a row) says where a row's tokens are. Row r holds ``lengths[r]``
tokens before the call, which brings the last ``counts[r]`` of its ``length`` tokens.
"""
import math
import os
import sys

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
_BLOCK = 64
_EPS = 1e-6
_LOWEST = -100  # exponent of the smallest scale


def _rotary(name, rows, length, heads, head_dim, rotary, *, dtype="f32", interleaved=False,
            inverse=False, scaled=False, far=8192):
    return dict(kind="rotary", name=name, rows=rows, length=length, heads=heads, head_dim=head_dim,
                rotary=rotary, dtype=dtype, interleaved=interleaved, inverse=inverse, scaled=scaled,
                far=far)


def _append(name, rows, length, kv_heads, head_dim, rotary, *, shortest=None, cached=(0, 0),
            page=64, dtype="f32", interleaved=False):
    return dict(kind="append", name=name, rows=rows, length=length, kv_heads=kv_heads,
                head_dim=head_dim, rotary=rotary, shortest=length if shortest is None else shortest,
                cached_low=cached[0], cached=cached[1], page=page, dtype=dtype,
                interleaved=interleaved)


def _attend(name, rows, length, heads, kv_heads, head_dim, rotary, *, shortest=None, cached=(0, 0),
            page=64, dtype="f32", interleaved=False):
    return dict(_append(name, rows, length, kv_heads, head_dim, rotary, shortest=shortest,
                        cached=cached, page=page, dtype=dtype, interleaved=interleaved),
                kind="attend", heads=heads)


def listed():
    return [
        # One new token of each row of a batch, part of the head: latency.
        _rotary("rotary_step", 64, 1, 8, 256, 64, dtype="bf16"),
        # Long prompts at far positions, whole heads interleaved, stretched frequencies.
        _rotary("rotary_long", 2, 8192, 16, 128, 128, interleaved=True, scaled=True, far=1 << 20),
        # Gradient of odd shapes.
        _rotary("rotary_gradient", 3, 1003, 5, 96, 48, dtype="bf16", inverse=True),
        # The keys and values of one generated token a row.
        _append("append_step", 64, 1, 2, 256, 64, cached=(5, 4000), dtype="bf16"),
        # All question rows of a decision into empty caches, left-padded.
        _append("append_rows", 16, 256, 2, 256, 64, shortest=32),
        # Long prompts behind what is cached, interleaved positions, large pages, one odd length.
        _append("append_long", 4, 8191, 4, 128, 128, shortest=8000, cached=(100, 3000), page=256,
                dtype="bf16", interleaved=True),
        # One row generating behind a short prompt: latency.
        _attend("attend_first", 1, 1, 8, 2, 256, 64, cached=(300, 300)),
        # A batch of ragged rows generating a token each.
        _attend("attend_batch", 64, 1, 8, 2, 256, 64, cached=(200, 4000), page=128, dtype="bf16"),
        # One row generating behind a long context.
        _attend("attend_long", 1, 1, 8, 2, 256, 64, cached=(131000, 131000), page=256, dtype="bf16"),
        # A few tokens a row at once, head widths off the tiles, an empty cache among the rows.
        _attend("attend_few", 5, 3, 6, 3, 96, 96, shortest=0, cached=(0, 1500), interleaved=True),
        # The next turn's prompt behind a cached one.
        _attend("attend_prompt", 2, 1024, 8, 2, 256, 64, shortest=900, cached=(8000, 8192), page=128,
                dtype="bf16"),
        # A large batch with long rows: the cache's traffic.
        _attend("attend_wide", 128, 1, 8, 2, 256, 64, cached=(8000, 8192), page=256),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("rotary", "append", "attend", "attend"))
    dtype = rng.choice(("f32", "bf16"))
    interleaved = rng.random() < 0.4
    head_dim = rng.choice((32, 64, 96, 128, 256, 256, rng.randint(8, 256)))
    rotary = min(head_dim // 2 * 2, 2 * rng.randint(1, 128)) if rng.random() < 0.5 else head_dim // 2 * 2
    if kind == "rotary":
        heads = rng.randint(1, 16)
        length = 1 if rng.random() < 0.3 else _log_int(rng, 2, 16384)
        most = 2 * 8192 * 16 * 128 // (length * heads * head_dim)
        return dict(kind=kind, rows=_log_int(rng, 1, max(1, min(256, most))), length=length,
                    heads=heads, head_dim=head_dim, rotary=rotary, dtype=dtype,
                    interleaved=interleaved, inverse=rng.random() < 0.4, scaled=rng.random() < 0.5,
                    far=_log_int(rng, 100, 1 << 20))
    kv_heads = rng.choice((1, 2, 2, 3, 4, 8))
    case = dict(kind=kind, rows=1, length=1, kv_heads=kv_heads, head_dim=head_dim, rotary=rotary,
                shortest=1, cached_low=0, cached=0, page=rng.choice((64, 128, 256)), dtype=dtype,
                interleaved=interleaved)
    if kind == "append":
        length = 1 if rng.random() < 0.4 else _log_int(rng, 2, 8192)
        most = 4 * 8191 * 4 * 128 // (length * kv_heads * head_dim)
        case.update(length=length, rows=_log_int(rng, 1, max(1, min(256, most))),
                    cached=rng.choice((0, _log_int(rng, 1, 4096))))
    else:
        case["heads"] = kv_heads * rng.choice((1, 2, 3, 4, 4, 8))
        length = 1 if rng.random() < 0.6 else _log_int(rng, 2, 1024)
        most = 2 * 8 * 1024 * 9216 // (length * case["heads"])
        cached = min(_log_int(rng, 1, 131072), max(1, most - length))
        total = cached + length
        most = min(most // total, 128 * 8192 * 2 * 256 // (total * kv_heads * (-(-head_dim // 64) * 64)))
        case.update(length=length, rows=_log_int(rng, 1, max(1, min(256, most))), cached=cached)
    case["cached_low"] = rng.choice((case["cached"], case["cached"] // rng.randint(2, 9)))
    case["shortest"] = case["length"] if rng.random() < 0.5 else case["length"] // rng.randint(2, 9)
    return case


# ------------------------------------------------------------------ inputs


def _spread(low, high, rows):
    """One whole number a row, from low to high."""
    return [high if rows == 1 else low + (high - low) * r // (rows - 1) for r in range(rows)]


def _frequencies(pairs, scaled):
    """Turns per token of each pair; stretched by 8 where a pair turns less than once in 8192
    tokens, not at all where more than 32 times, blended by its turns between."""
    f = 1e7 ** (-torch.arange(pairs, dtype=torch.float64) / max(pairs, 1)) / (2 * math.pi)
    if scaled:
        keep = ((f * 8192 - 1) / 31).clamp(0, 1)
        f = f * (keep + (1 - keep) / 8)
    return f


def prepare(case, seed):
    dev = torch.device("cuda", 0)
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    rows, length, hd = case["rows"], case["length"], case["head_dim"]
    s = dict(case)
    host = _frequencies(case["rotary"] // 2, case.get("scaled", False))
    s.update(frequencies=host.numpy(), turns=host.to(dev))
    if case["kind"] == "rotary":
        s["x"] = normal(rows * case["heads"] * hd * length).to(dtype)
        first = torch.randint(case["far"], (rows, 1), generator=gen, device=dev, dtype=torch.int32)
        s["positions"] = (first + torch.arange(length, device=dev, dtype=torch.int32)).view(-1)
        return s
    kv_heads, page = case["kv_heads"], case["page"]
    wide = -(-hd // 64) * 64
    order = torch.randperm(rows, generator=gen, device=dev)
    lengths, counts = (torch.tensor(_spread(lo, hi, rows), dtype=torch.int32, device=dev) for lo, hi in
                       ((case["cached_low"], case["cached"]), (case["shortest"], length)))
    s.update(lengths=lengths[order], counts=counts[torch.randperm(rows, generator=gen, device=dev)])
    per_row = -(-(case["cached"] + length) // page)
    pool = rows * per_row + 1
    s["pages"] = torch.randperm(pool, generator=gen, device=dev)[:rows * per_row].to(torch.int32)
    # What a cache holds: normalized keys, and values of unit size, in 1/256 or 1/512.
    size = pool * kv_heads * page * wide
    codes = [(torch.randn(size, generator=gen, device=dev, dtype=torch.bfloat16) * 110.0).clamp(-448, 448)
             .to(torch.float8_e4m3fn) for _ in range(2)]
    codes[0].view(-1, wide)[:, hd:] = torch.zeros((), device=dev).to(torch.float8_e4m3fn)
    scales = [2.0 ** -torch.randint(7, 9, (size // (wide * _BLOCK),), generator=gen, device=dev).float()
              for _ in range(2)]
    s.update(keys=codes[0], values=codes[1], key_scales=scales[0], value_scales=scales[1],
             norm=normal(hd) * 0.02)
    if case["kind"] == "append":
        s.update(k=(normal(rows * kv_heads * hd * length) * 0.64).to(dtype),
                 v=(normal(rows * kv_heads * hd * length) * 0.64).to(dtype))
    else:
        n = rows * case["heads"] * hd * length
        s.update(q=(normal(n) * 0.64).to(dtype), gate=(normal(n) * 0.64).to(dtype))
    return s


# ------------------------------------------------------------------ plain forms


def _cos_sin(positions, turns):
    """cos and sin (rows, 1, pairs, length) in 64 bits of positions (rows, length)."""
    t = positions.double()[:, None, None, :] * turns[None, None, :, None]
    t = 2 * math.pi * (t - torch.round(t))
    return torch.cos(t), torch.sin(t)


def _turn(x, cos, sin, interleaved):
    """x (rows, heads, features, length), its first pairs turned."""
    pairs = cos.shape[2]
    if interleaved:
        a, b = x[:, :, 0:2 * pairs:2], x[:, :, 1:2 * pairs:2]
    else:
        a, b = x[:, :, :pairs], x[:, :, pairs:2 * pairs]
    y, z = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack([y, z], 3).flatten(2, 3) if interleaved else torch.cat([y, z], 2)
    return torch.cat([turned, x[:, :, 2 * pairs:]], 2)


def _normalized(x, weight):
    return x * torch.rsqrt(x.square().mean(2, keepdim=True) + _EPS) * (1 + weight.to(x.dtype))[:, None]


def _plain_rotary(s):
    rows, length = s["rows"], s["length"]
    x = s["x"].view(rows, s["heads"], s["head_dim"], length).float()
    cos, sin = _cos_sin(s["positions"].view(rows, length), s["turns"])
    sin = -sin if s["inverse"] else sin
    return _turn(x, cos.float(), sin.float(), s["interleaved"]).to(s["x"].dtype).view(-1)


def _token_positions(s):
    """Place in its row's cache of every token (rows, length), negative where it is none."""
    t = torch.arange(s["length"], device=s["lengths"].device)
    behind = s["length"] - s["counts"].long()[:, None]
    return torch.where(t >= behind, s["lengths"].long()[:, None] + t - behind, -1)


def _to_codes(v):
    """v to the nearest e4m3 value, in 64 bits."""
    step = torch.exp2((torch.frexp(v).exponent - 1).clamp(min=-6).double() - 3)
    return torch.round(v / step) * step


def _plain_append(s):
    """In 64 bits: a value next to a border goes to its own side."""
    rows, length, kv_heads, hd, page = (s[n] for n in ("rows", "length", "kv_heads", "head_dim", "page"))
    wide, dev = -(-hd // 64) * 64, s["k"].device
    pages = s["pages"].view(rows, -1).long()
    per_page = page // _BLOCK
    blocks = pages.shape[1] * per_page
    at = _token_positions(s)
    active = at >= 0
    k = _normalized(s["k"].view(rows, kv_heads, hd, length).double(), s["norm"])
    k = _turn(k, *_cos_sin(at.clamp(min=0), s["turns"]), s["interleaved"])
    v = s["v"].view(rows, kv_heads, hd, length).double()
    row, token = torch.nonzero(active, as_tuple=True)
    place = at[row, token]
    # Blocks of the pool, (page * kv_heads + head) * per_page + block, of every token and head.
    head = torch.arange(kv_heads, device=dev)[None, :]
    of_token = ((pages[row, place // page][:, None] * kv_heads + head) * per_page
                + (place % page // _BLOCK)[:, None])
    # Rows whose first block holds earlier tokens.
    first = s["lengths"].long()
    kept = torch.nonzero((s["counts"] > 0) & (first % _BLOCK > 0))[:, 0]
    of_kept = ((pages[kept, first[kept] // page][:, None] * kv_heads + head) * per_page
               + (first[kept] % page // _BLOCK)[:, None])
    older = torch.arange(_BLOCK, device=dev) < (first[kept] % _BLOCK)[:, None]  # (kept, 64)
    for x, codes, scales, by_token in ((k, s["keys"], s["key_scales"], True),
                                       (v, s["values"], s["value_scales"], False)):
        new = x[row, :, :, token]  # (tokens, kv_heads, hd)
        most = torch.zeros(scales.numel(), dtype=torch.float64, device=dev)
        most.scatter_reduce_(0, of_token.flatten(), new.abs().amax(2).flatten(), "amax")
        m, e = torch.frexp(most)
        need = torch.where(most > 0, e - 9 + (m > 0.875).int(), _LOWEST).clamp(min=_LOWEST)
        scale = torch.where(torch.zeros_like(most).index_fill_(0, of_token.flatten(), 1.0) > 0,
                            torch.exp2(need.double()), scales.double())
        before = scales.double()[of_kept]
        scale[of_kept] = torch.maximum(scale[of_kept], before)
        # Codes as (block, 64 tokens, features), in either layout.
        view = codes.view(torch.uint8).view(-1, _BLOCK, wide) if by_token else codes.view(
            torch.uint8).view(-1, wide, _BLOCK).transpose(1, 2)
        old = view[of_kept].view(torch.float8_e4m3fn) if by_token else view[of_kept].contiguous().view(
            torch.float8_e4m3fn)
        again = _to_codes(old.float().double() * (before / scale[of_kept])[..., None, None])
        again = torch.where(older[:, None, :, None], again, old.float().double())
        view[of_kept] = again.float().to(torch.float8_e4m3fn).view(torch.uint8)
        new = _to_codes(new / scale[of_token][..., None]).float().to(torch.float8_e4m3fn).view(torch.uint8)
        slot = (place % _BLOCK)[:, None].expand_as(of_token)
        view[of_token, slot, :hd] = new
        scales.copy_(scale)
    return {"keys": s["keys"], "values": s["values"], "key_scales": s["key_scales"],
            "value_scales": s["value_scales"]}


def _plain_attend(s):
    rows, length, heads, kv_heads, hd, page = (
        s[n] for n in ("rows", "length", "heads", "kv_heads", "head_dim", "page"))
    wide = -(-hd // 64) * 64
    at = _token_positions(s)
    pages = s["pages"].view(rows, -1).long()
    total = pages.shape[1] * page
    # (rows, kv_heads, tokens, features) of keys and values
    k = s["keys"].view(torch.uint8).view(-1, kv_heads, page, wide)[pages].view(torch.float8_e4m3fn).float()
    k = k.view(*k.shape[:3], -1, _BLOCK, wide) * s["key_scales"].view(-1, kv_heads, page // _BLOCK)[
        pages][..., None, None]
    k = k.transpose(1, 2).reshape(rows, kv_heads, total, wide)[..., :hd].contiguous()
    v = s["values"].view(torch.uint8).view(-1, kv_heads, page // _BLOCK, wide, _BLOCK)[pages].view(
        torch.float8_e4m3fn).float()
    v = v * s["value_scales"].view(-1, kv_heads, page // _BLOCK)[pages][..., None, None]
    v = v.permute(0, 2, 1, 3, 5, 4).reshape(rows, kv_heads, total, wide)[..., :hd].contiguous()
    q = _normalized(s["q"].view(rows, heads, hd, length).float(), s["norm"])
    cos, sin = _cos_sin(at.clamp(min=0), s["turns"])
    q = _turn(q, cos.float(), sin.float(), s["interleaved"])
    q = q.transpose(2, 3).reshape(rows, kv_heads, -1, hd)
    scores = q @ k.transpose(2, 3).contiguous() / math.sqrt(hd)
    scores = scores.view(rows, heads, length, total)
    hidden = torch.arange(total, device=q.device) > at[:, None, :, None]
    scores = scores.masked_fill_(hidden, -math.inf)
    high = scores.amax(3, keepdim=True)
    p = torch.exp(scores - torch.where(high == -math.inf, 0.0, high))
    z = p.sum(3, keepdim=True)
    out = (p.view(rows, kv_heads, -1, total) @ v).view(rows, heads, length, hd)
    out = torch.where(z > 0, out / z, 0.0).transpose(2, 3)
    gate = s["gate"].view(rows, heads, hd, length).float()
    return (out / (1 + torch.exp(-gate))).reshape(-1)


# ------------------------------------------------------------------ the framework's operators


_kept = {}


def _framework():
    """The package, and a context on torch's stream, as a program that runs torch beside it keeps."""
    if not _kept:
        package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                               "tenferro-decision-rs_amd")
        if package not in sys.path:
            sys.path.insert(0, package)
        import tenferro_ext

        _kept["te"] = tenferro_ext
        _kept["ctx"] = tenferro_ext.Context(0, stream=torch.cuda.current_stream().cuda_stream)
    return _kept["te"], _kept["ctx"]


def _own(s):
    te, ctx = _framework()
    bf16 = s["dtype"] == "bf16"
    rotary = te.Rotary(s["frequencies"], s["interleaved"])
    with te.asynchronous():
        if s["kind"] == "rotary":
            return te.rotary_rows(s["x"], s["positions"], s["rows"], s["length"], s["heads"],
                                  s["head_dim"], rotary, inverse=s["inverse"], bf16=bf16, ctx=ctx)
        cache = te.PagedCache(s["keys"], s["values"], s["key_scales"], s["value_scales"], s["page"])
        if s["kind"] == "append":
            te.jeff_cache_append(s["k"], s["v"], s["norm"], cache, s["pages"], s["lengths"],
                                 s["counts"], s["rows"], s["length"], s["kv_heads"], s["head_dim"],
                                 rotary, _EPS, bf16=bf16, ctx=ctx)
            return {"keys": s["keys"], "values": s["values"], "key_scales": s["key_scales"],
                    "value_scales": s["value_scales"]}
        return te.jeff_cached_attention(s["q"], s["gate"], s["norm"], cache, s["pages"],
                                        s["lengths"], s["counts"], s["rows"], s["length"],
                                        s["heads"], s["kv_heads"], s["head_dim"], rotary, _EPS,
                                        bf16=bf16, ctx=ctx)


def run(state):
    if own:
        return _own(state)
    return {"rotary": _plain_rotary, "append": _plain_append, "attend": _plain_attend}[
        state["kind"]](state)


# ------------------------------------------------------------------ work


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    rows, length, hd = case["rows"], case["length"], case["head_dim"]
    if case["kind"] == "rotary":
        n = rows * length * case["heads"]
        # A pair takes four products and two sums.
        return {"bytes": 2 * size * n * hd + 4 * rows * length, "flops": 3 * n * case["rotary"]}
    kv_heads = case["kv_heads"]
    counts = _spread(case["shortest"], length, rows)
    if case["kind"] == "append":
        n = sum(counts) * kv_heads
        # Codes and, per started block, two scales; a square, a sum, two products and the scaling of
        # a key, the scaling of a value.
        return {"bytes": 2 * n * hd * (size + 1) + 8 * n // _BLOCK + 12 * rows,
                "flops": n * (6 * hd + 3 * case["rotary"])}
    cached = _spread(case["cached_low"], case["cached"], rows)
    heads = case["heads"]
    # Which row has which count goes by the seed: on average a row's tokens see its cached ones.
    held = sum(cached) + sum(counts)
    pairs = sum(cached) * sum(counts) / rows + sum(c * (c + 1) / 2 for c in counts)
    n = sum(counts) * heads * hd
    return {"bytes": int(held * kv_heads * (2 * hd + 8 / _BLOCK) + held // case["page"] * 4
                         + n * 2 * size + rows * length * heads * hd * 4 + 8 * rows),
            "flops": int(4 * pairs * heads * hd)}


# ------------------------------------------------------------------ 64 bits


def _exact_turned(x, place, turns, interleaved):
    """x (..., features) of one token each, in 64 bits, as complex numbers times e^(2 pi i p f)."""
    pairs = turns.numel()
    t = place.double()[:, None] * turns
    w = torch.polar(torch.ones_like(t), 2 * math.pi * (t - torch.round(t)))
    out = x.clone()
    if interleaved:
        z = torch.view_as_complex(x[..., :2 * pairs].reshape(*x.shape[:-1], pairs, 2).contiguous())
        out[..., :2 * pairs] = torch.view_as_real(z * w[:, None]).flatten(-2)
    else:
        z = torch.complex(x[..., :pairs].contiguous(), x[..., pairs:2 * pairs].contiguous()) * w[:, None]
        out[..., :pairs], out[..., pairs:2 * pairs] = z.real, z.imag
    return out


def _exact_normalized(x, weight):
    return x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + _EPS) * (weight.double() + 1)


def _tokens_of(x, r, heads, hd, length):
    """Row r of rows x (length, heads * hd) as (length, heads, hd) in 64 bits."""
    n = heads * hd * length
    return x[r * n:(r + 1) * n].double().view(heads, hd, length).permute(2, 0, 1)


def _exact_rotary(s):
    out = []
    for r in range(s["rows"]):
        place = s["positions"].view(s["rows"], -1)[r].double() * (-1 if s["inverse"] else 1)
        x = _tokens_of(s["x"], r, s["heads"], s["head_dim"], s["length"])
        out.append(_exact_turned(x, place, s["turns"], s["interleaved"]).permute(1, 2, 0).reshape(-1))
    return torch.cat(out)


def _exact_append(s):
    """Block by block. All e4m3 values, so that the nearest is looked up."""
    kv_heads, hd, page, rows = s["kv_heads"], s["head_dim"], s["page"], s["rows"]
    wide = -(-hd // 64) * 64
    dev = s["k"].device
    values = torch.arange(0x7F, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn).float().double()
    middles = (values[1:] + values[:-1]) / 2

    def nearest(x):
        a = x.abs().contiguous()
        i = torch.bucketize(a, middles)  # the border itself to the lower value
        tie = (i < middles.numel()) & (middles[i.clamp(max=middles.numel() - 1)] == a)
        i = torch.where(tie & (i % 2 == 1), i + 1, i)
        return torch.copysign(values[i], x)

    keys = s["keys"].float().double().view(-1, kv_heads, page, wide)
    vals = s["values"].float().double().view(-1, kv_heads, page // _BLOCK, wide, _BLOCK)
    scales = [s[n].double().view(-1, kv_heads, page // _BLOCK).clone()
              for n in ("key_scales", "value_scales")]
    first, counts = s["lengths"].tolist(), s["counts"].tolist()
    pages = s["pages"].view(rows, -1).tolist()
    for r in range(rows):
        n, c = first[r], counts[r]
        if not c:
            continue
        k = _exact_normalized(_tokens_of(s["k"], r, kv_heads, hd, s["length"])[-c:], s["norm"])
        k = _exact_turned(k, torch.arange(n, n + c, device=dev), s["turns"], s["interleaved"])
        v = _tokens_of(s["v"], r, kv_heads, hd, s["length"])[-c:]
        for block in range(n // _BLOCK, (n + c - 1) // _BLOCK + 1):
            p, b = pages[r][block * _BLOCK // page], block % (page // _BLOCK)
            lo, hi = max(n, block * _BLOCK), min(n + c, (block + 1) * _BLOCK)
            at = slice(lo - block * _BLOCK, hi - block * _BLOCK)
            for x, held, scale in ((k, keys[p, :, b * _BLOCK:(b + 1) * _BLOCK], scales[0]),
                                   (v, vals[p, :, b].transpose(1, 2), scales[1])):
                new = x[lo - n:hi - n].transpose(0, 1)  # (kv_heads, tokens, hd)
                need = torch.exp2(torch.ceil(torch.log2(new.abs().amax((1, 2)) / 448)))
                need = torch.where(new.abs().amax((1, 2)) <= 224 * need, need / 2, need)
                need = torch.where(new.abs().amax((1, 2)) > 448 * need, need * 2, need)
                need = need.clamp(min=2.0 ** _LOWEST)
                if lo % _BLOCK:
                    before = scale[p, :, b].clone()
                    need = torch.maximum(need, before)
                    old = held[:, :at.start]
                    held[:, :at.start] = nearest(old * (before / need)[:, None, None])
                held[:, at, :hd] = nearest(new / need[:, None, None])
                scale[p, :, b] = need
    return {"keys": keys.reshape(-1), "values": vals.reshape(-1), "key_scales": scales[0].reshape(-1),
            "value_scales": scales[1].reshape(-1)}


def _exact_attend(s):
    rows, length, heads, kv_heads, hd, page = (
        s[n] for n in ("rows", "length", "heads", "kv_heads", "head_dim", "page"))
    wide, dev = -(-hd // 64) * 64, s["q"].device
    out = torch.zeros(rows, heads, hd, length, dtype=torch.float64, device=dev)
    keys = s["keys"].view(torch.uint8).view(-1, kv_heads, page, wide)
    vals = s["values"].view(torch.uint8).view(-1, kv_heads, page // _BLOCK, wide, _BLOCK)
    ks, vs = (s[n].view(-1, kv_heads, page // _BLOCK) for n in ("key_scales", "value_scales"))
    first, counts = s["lengths"].tolist(), s["counts"].tolist()
    for r in range(rows):
        n, c = first[r], counts[r]
        if not c:
            continue
        place = torch.arange(n, n + c, device=dev)
        q = _exact_normalized(_tokens_of(s["q"], r, heads, hd, length)[-c:], s["norm"])
        q = _exact_turned(q, place, s["turns"], s["interleaved"])
        g = _tokens_of(s["gate"], r, heads, hd, length)[-c:]
        p = s["pages"].view(rows, -1)[r].long()
        for h in range(kv_heads):
            k = keys[p, h].view(torch.float8_e4m3fn).float().double().view(-1, wide)
            k = k * ks[p, h].double().reshape(-1).repeat_interleave(_BLOCK)[:, None]
            v = vals[p, h].view(torch.float8_e4m3fn).float().double().transpose(2, 3).reshape(-1, wide)
            v = v * vs[p, h].double().reshape(-1).repeat_interleave(_BLOCK)[:, None]
            k, v = k[:n + c, :hd], v[:n + c, :hd].contiguous()
            for j in range(h * (heads // kv_heads), (h + 1) * (heads // kv_heads)):
                scores = (q[:, j].contiguous() @ k.T.contiguous()) * hd ** -0.5
                scores[torch.arange(n + c, device=dev) > place[:, None]] = -math.inf
                o = torch.softmax(scores, 1) @ v * torch.sigmoid(g[:, j])
                out[r, j, :, length - c:] = o.T
    return out.reshape(-1)


def exact(case, seed):
    if case["kind"] == "append" and case["rows"] * (1 + case["length"] // _BLOCK) > 6000:
        return None  # block by block it would take too long
    s = prepare(case, seed)
    return {"rotary": _exact_rotary, "append": _exact_append, "attend": _exact_attend}[case["kind"]](s)
