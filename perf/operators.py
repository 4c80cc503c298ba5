"""Cases of the linear attention and of the token log probabilities.

``kind`` names the operator:

* ``prompt``   linear attention over rows of tokens (``jeff_linear_attention_rows``): decayed state
               per head, with ``delta`` the gated delta-rule write, from a given state with ``continues``
* ``step``     the same for one token a row, the state updated in place
               (``jeff_linear_attention_step``)
* ``answer``   log probabilities of given tokens, the entropy and the ``top`` alternatives at
               every position of a matrix of logits (``token_log_probs``)

Layouts are the framework's: rows of (length, width) with the tokens contiguous, states
(value_dim, key_dim) per row and head with the value features contiguous, logits (vocab, positions)
with a position's logits contiguous.
"""
import math
import os
import sys

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
_CHUNK = 64  # tokens that the plain form of a prompt takes at once


def _prompt(name, rows, length, heads, key_heads, key_dim, value_dim, *, shortest=None,
            dtype="f32", delta=True, continues=False):
    return dict(kind="prompt", name=name, rows=rows, length=length, heads=heads,
                key_heads=key_heads, key_dim=key_dim, value_dim=value_dim,
                shortest=shortest or length, dtype=dtype, delta=delta, continues=continues)


def _step(name, rows, heads, key_heads, key_dim, value_dim, *, dtype="f32", delta=True):
    return dict(kind="step", name=name, rows=rows, heads=heads, key_heads=key_heads,
                key_dim=key_dim, value_dim=value_dim, dtype=dtype, delta=delta)


def _answer(name, positions, vocab, per_position, top, *, dtype="f32", banned=False):
    return dict(kind="answer", name=name, positions=positions, vocab=vocab,
                per_position=per_position, top=top, dtype=dtype, banned=banned)


def listed():
    return [
        # One short question: latency and launches.
        _prompt("prompt_short", 1, 48, 4, 4, 32, 32),
        # All question rows of a decision in one call, left-padded, delta rule.
        _prompt("prompt_rows", 16, 256, 16, 16, 128, 128, shortest=32),
        # Rows of an odd length and head widths off the tiles that continue from a state, plain decay.
        _prompt("prompt_odd", 3, 777, 6, 3, 96, 80, shortest=300, delta=False, continues=True),
        # Wide heads with shared keys, as the full-attention layers have them, plain decay, bf16.
        _prompt("prompt_wide", 8, 1024, 8, 2, 256, 256, dtype="bf16", delta=False),
        # Long-context prefill, delta rule, bf16.
        _prompt("prompt_long", 2, 8192, 16, 16, 128, 128, dtype="bf16"),
        # One row generating a token: latency.
        _step("step_single", 1, 16, 16, 128, 128),
        # A batch of rows generating a token each, bf16 operands.
        _step("step_batch", 64, 16, 8, 128, 128, dtype="bf16"),
        # A large batch with wide heads, plain decay: the states' traffic.
        _step("step_wide", 128, 8, 2, 256, 256, delta=False),
        # Marker logits of a batch of decision prompts.
        _answer("answer_markers", 64, 8, 1, 2),
        # Label tokens at the last position of each question row.
        _answer("answer_labels", 16, 131072, 4, 5),
        # One position of a model with an odd vocabulary, half of it banned by a grammar.
        _answer("answer_single", 1, 100003, 2, 20, dtype="bf16", banned=True),
        # Every token of a batch of prompts scored.
        _answer("answer_prompt", 4096, 65536, 1, 0, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("prompt", "prompt", "step", "answer"))
    dtype = rng.choice(("f32", "bf16"))
    if kind == "answer":
        vocab = _log_int(rng, 2, 160000)
        return dict(kind=kind, positions=_log_int(rng, 1, max(1, min(8192, (1 << 27) // vocab))),
                    vocab=vocab, per_position=rng.randint(1, 8), top=rng.randint(0, min(vocab, 32)),
                    dtype=dtype, banned=rng.random() < 0.3)
    key_heads = rng.choice((1, 2, 4, 8, 16))
    heads = key_heads * rng.choice([m for m in (1, 2, 4) if key_heads * m <= 16])
    key_dim = rng.choice((32, 64, 128, 256, rng.randint(8, 256)))
    value_dim = rng.choice((32, 64, 128, 256, key_dim, rng.randint(8, 256)))
    case = dict(kind=kind, rows=0, heads=heads, key_heads=key_heads, key_dim=key_dim,
                value_dim=value_dim, dtype=dtype, delta=rng.random() < 0.6)
    size = heads * key_dim * value_dim
    if kind == "step":
        case["rows"] = _log_int(rng, 1, max(1, min(256, (1 << 26) // size)))
        return case
    length = _log_int(rng, 2, 8192)
    most = 2 * 8192 * 16 * 128 * 128 // (length * size)
    while most < 1:
        length //= 2
        most = 2 * 8192 * 16 * 128 * 128 // (length * size)
    case.update(length=length, rows=_log_int(rng, 1, min(32, most)),
                shortest=length if rng.random() < 0.4 else max(1, length // rng.randint(2, 8)),
                continues=rng.random() < 0.4)
    return case


# ------------------------------------------------------------------ inputs


def _unit_heads(x, width):
    """x (rows, heads * width, length) with every head's vector of unit length."""
    r, w, n = x.shape
    y = x.view(r, w // width, width, n)
    return (y / y.square().sum(2, keepdim=True).sqrt()).view(r, w, n)


def prepare(case, seed):
    dev = torch.device("cuda", 0)
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    def uniform(*shape):
        return torch.rand(*shape, generator=gen, device=dev)

    s = dict(case)
    if case["kind"] == "answer":
        n, vocab, m = case["positions"], case["vocab"], case["per_position"]
        # Logits of a model: a wide bulk, and at half of the positions one token that stands out.
        x = normal(n, vocab) * 2.5
        peak = torch.randint(vocab, (n, 1), generator=gen, device=dev)
        x.scatter_add_(1, peak, (uniform(n, 1) < 0.5) * 12.0)
        tokens = torch.randint(vocab, (n, m), generator=gen, device=dev)
        tokens[:, 0] = peak[:, 0]
        if case["banned"]:
            x[uniform(n, vocab) < 0.5] = -math.inf
            x.scatter_(1, peak, 3.0)  # a grammar leaves something to say
        s.update(logits=x.to(dtype).view(-1), tokens=tokens.view(-1))
        return s
    length = 1 if case["kind"] == "step" else case["length"]
    rows, heads, key_heads = case["rows"], case["heads"], case["key_heads"]
    dk, dv = case["key_dim"], case["value_dim"]
    # Keys and queries of unit length, decays from nearly none to strong ones, as a layer's gates
    # give them: -rate * softplus(.), one rate a head.
    rate = torch.exp(uniform(1, heads, 1) * math.log(400.0) + math.log(0.01))
    soft = torch.nn.functional.softplus(normal(rows, heads, length))
    s.update(q=_unit_heads(normal(rows, key_heads * dk, length), dk).to(dtype).view(-1),
             k=_unit_heads(normal(rows, key_heads * dk, length), dk).to(dtype).view(-1),
             v=normal(rows, heads * dv, length).to(dtype).view(-1),
             log_decay=(-rate * soft).view(-1),
             beta=torch.sigmoid(normal(rows, heads, length)).view(-1) if case["delta"] else None,
             state=None, mask=None)
    if case["kind"] == "step" or case["continues"]:
        s["state"] = (normal(rows, heads, dk, dv) * 0.3).view(-1)
    if case["kind"] == "prompt":
        lo = case["shortest"]
        if lo < length or rows > 1:
            valid = torch.linspace(lo, length, rows, device=dev).round().to(torch.int64)
            valid = valid[torch.randperm(rows, generator=gen, device=dev)]
            at = torch.arange(length, device=dev)
            s["mask"] = (at[None, :] >= length - valid[:, None]).float().view(-1)
    return s


# ------------------------------------------------------------------ plain forms


def _heads_first(x, rows, heads, width, length, times):
    """(rows, heads * times, length, width) in 32 bits of rows x (length, heads * width)."""
    y = x.float().view(rows, heads, width, length).transpose(2, 3)
    return y.repeat_interleave(times, 1) if times > 1 else y


def _plain_prompt(s):
    """The recurrence in blocks of _CHUNK tokens: within a block the decayed products of all pairs,
    between blocks the state. The block's writes solve a unit lower triangular system, by rows."""
    rows, length, heads, key_heads = s["rows"], s["length"], s["heads"], s["key_heads"]
    dk, dv, dev = s["key_dim"], s["value_dim"], s["q"].device
    times = heads // key_heads
    pad = -length % _CHUNK
    blocks = (length + pad) // _CHUNK

    def cut(x, width):  # (rows, heads, blocks, chunk, width), zeros behind the end
        x = torch.cat([x, x.new_zeros(rows, heads, pad, width)], 2) if pad else x
        return x.reshape(rows, heads, blocks, _CHUNK, width)

    active = torch.ones(rows, 1, length, 1, dtype=torch.bool, device=dev)
    if s["mask"] is not None:
        active = (s["mask"] != 0).view(rows, 1, length, 1)
    zero = torch.zeros((), device=dev)
    q, k, v, g = (cut(torch.where(active, x, zero), w) for x, w in (
        (_heads_first(s["q"], rows, key_heads, dk, length, times), dk),
        (_heads_first(s["k"], rows, key_heads, dk, length, times), dk),
        (_heads_first(s["v"], rows, heads, dv, length, 1), dv),
        (s["log_decay"].view(rows, heads, length, 1), 1)))
    cum = g.double().cumsum(3)
    seen = torch.ones(_CHUNK, _CHUNK, dtype=torch.bool, device=dev).tril()
    decay = torch.exp((cum - cum.transpose(3, 4)).masked_fill(~seen, -math.inf)).float()
    from_start, to_end = torch.exp(cum).float(), decay[..., -1, :, None]
    solve = None
    if s["beta"] is not None:
        beta = cut(torch.where(active, s["beta"].view(rows, heads, length, 1), zero), 1)
        pairs = (beta * (k @ k.transpose(3, 4)) * decay).tril(-1)
        solve = torch.eye(_CHUNK, device=dev).repeat(rows, heads, blocks, 1, 1)
        for t in range(1, _CHUNK):
            solve[..., t, :t] = -(pairs[..., t, None, :t] @ solve[..., :t, :t])[..., 0, :]
    scores = (q @ k.transpose(3, 4)) * decay
    scale = 1.0 / math.sqrt(dk)
    state = torch.zeros(rows, heads, dk, dv, device=dev)
    if s["state"] is not None:
        state = s["state"].view(rows, heads, dk, dv)
    out = torch.empty(rows, heads, blocks, _CHUNK, dv, device=dev)
    for n in range(blocks):
        write = v[:, :, n]
        if solve is not None:
            write = beta[:, :, n] * (write - from_start[:, :, n] * (k[:, :, n] @ state))
            write = solve[:, :, n] @ write
        out[:, :, n] = scale * (from_start[:, :, n] * (q[:, :, n] @ state) + scores[:, :, n] @ write)
        state = (from_start[:, :, n, -1:] * state
                 + k[:, :, n].transpose(2, 3) @ (to_end[:, :, n] * write))
    out = out.view(rows, heads, length + pad, dv)[:, :, :length]
    return {"out": out.transpose(2, 3).reshape(-1), "state": state.reshape(-1)}


def _plain_step(s):
    rows, heads, key_heads, dk, dv = (s[n] for n in ("rows", "heads", "key_heads", "key_dim",
                                                     "value_dim"))
    q, k = (s[n].float().view(rows, key_heads, dk, 1).repeat_interleave(heads // key_heads, 1)
            for n in ("q", "k"))
    state = s["state"].view(rows, heads, dk, dv)
    decayed = state * torch.exp(s["log_decay"]).view(rows, heads, 1, 1)
    write = s["v"].float().view(rows, heads, 1, dv)
    if s["beta"] is not None:
        write = s["beta"].view(rows, heads, 1, 1) * (write - (decayed * k).sum(2, keepdim=True))
    state.copy_(decayed + k * write)
    return {"out": ((state * q).sum(2) / math.sqrt(dk)).view(-1), "state": s["state"]}


def _plain_answer(s):
    n, vocab, m, top = s["positions"], s["vocab"], s["per_position"], s["top"]
    x = s["logits"].view(n, vocab).float()
    high = x.max(1, keepdim=True).values
    y = x - high
    e = torch.exp(y)
    z = e.sum(1, keepdim=True)
    log_z = torch.log(z)
    tokens = s["tokens"].view(n, m)
    r = {"log_probs": (y.gather(1, tokens) - log_z).view(-1),
         "entropy": (log_z - (e * torch.where(e > 0, y, 0.0)).sum(1, keepdim=True) / z).view(-1)}
    if top:
        # One whole number per logit, larger for larger logits and, among equal ones, lower indexes.
        bits = (x + 0.0).view(torch.int32).to(torch.int64)
        order = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
        key = (order << 32) + (vocab - 1 - torch.arange(vocab, device=x.device))
        ids = vocab - 1 - (key.topk(top, 1).values & 0xFFFFFFFF)
        r.update(top_tokens=ids.view(-1), top_log_probs=(y.gather(1, ids) - log_z).view(-1))
    return r


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
    with te.asynchronous():
        if s["kind"] == "answer":
            r = te.token_log_probs(s["logits"], s["tokens"], s["positions"], s["vocab"],
                                   top=s["top"], bf16=bf16, ctx=ctx)
            more = {} if not s["top"] else {"top_tokens": r.top_tokens,
                                            "top_log_probs": r.top_log_probs}
            return {"log_probs": r.log_probs, "entropy": r.entropy, **more}
        if s["kind"] == "step":
            out = te.jeff_linear_attention_step(
                s["q"], s["k"], s["v"], s["log_decay"], s["beta"], s["state"], s["rows"],
                s["heads"], s["key_heads"], s["key_dim"], s["value_dim"], bf16=bf16, ctx=ctx)
            return {"out": out, "state": s["state"]}
        out, state = te.jeff_linear_attention_rows(
            s["q"], s["k"], s["v"], s["log_decay"], s["beta"], s["mask"], s["rows"], s["length"],
            s["heads"], s["key_heads"], s["key_dim"], s["value_dim"], state=s["state"], bf16=bf16,
            ctx=ctx)
        return {"out": out, "state": state}


def run(state):
    if own:
        return _own(state)
    return {"prompt": _plain_prompt, "step": _plain_step, "answer": _plain_answer}[
        state["kind"]](state)


# ------------------------------------------------------------------ work


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "answer":
        n, vocab = case["positions"], case["vocab"]
        # Per logit: a subtraction, an exponential, a product and two sums.
        return {"bytes": n * (vocab * size + case["per_position"] * 12 + 4 + case["top"] * 12),
                "flops": 5 * n * vocab}
    step = case["kind"] == "step"
    tokens = case["rows"] * (1 if step else case["length"])
    heads, key_heads, dk, dv = (case[n] for n in ("heads", "key_heads", "key_dim", "value_dim"))
    states = 4 * case["rows"] * heads * dk * dv
    moved = tokens * (size * (2 * key_heads * dk + heads * dv) + 4 * heads * dv
                      + 4 * heads * (2 if case["delta"] else 1))
    moved += states * (2 if step or case["continues"] else 1)
    if not step and (case["shortest"] < case["length"] or case["rows"] > 1):
        moved += 4 * tokens
    # The state's decay is not counted, its update and its product with the query (and the key) are.
    return {"bytes": moved, "flops": tokens * heads * dk * dv * (6 if case["delta"] else 4)}


# ------------------------------------------------------------------ 64 bits


def _exact_answer(s):
    n, vocab, m, top = s["positions"], s["vocab"], s["per_position"], s["top"]
    found = {"log_probs": [], "entropy": [], "top_tokens": [], "top_log_probs": []}
    for part, tokens in zip(s["logits"].view(n, vocab).split(256),
                            s["tokens"].view(n, m).split(256)):
        x = part.double()
        p = x - torch.logsumexp(x, 1, keepdim=True)
        found["log_probs"].append(p.gather(1, tokens))
        found["entropy"].append(-torch.where(p.exp() > 0, p.exp() * p, 0.0).sum(1))
        if top:
            values, ids = x.sort(dim=1, descending=True, stable=True)
            found["top_tokens"].append(ids[:, :top])
            found["top_log_probs"].append(p.gather(1, ids[:, :top]))
    return {name: torch.cat(v).reshape(-1) for name, v in found.items() if v}


def _exact_linear(s):
    """Token by token, by the definition."""
    rows, heads, key_heads, dk, dv = (s[n] for n in ("rows", "heads", "key_heads", "key_dim",
                                                     "value_dim"))
    length = s.get("length", 1)
    group = torch.arange(heads, device=s["q"].device) // (heads // key_heads)
    q = s["q"].double().view(rows, key_heads, dk, length)[:, group].permute(3, 0, 1, 2).contiguous()
    k = s["k"].double().view(rows, key_heads, dk, length)[:, group].permute(3, 0, 1, 2).contiguous()
    v = s["v"].double().view(rows, heads, dv, length).permute(3, 0, 1, 2).contiguous()
    keep = s["log_decay"].double().exp().view(rows, heads, length).permute(2, 0, 1).contiguous()
    on = torch.ones(length, rows, 1, dtype=torch.float64, device=q.device)
    if s["mask"] is not None:
        on = (s["mask"] != 0).double().view(rows, length, 1).transpose(0, 1).contiguous()
    keep = keep * on + (1 - on)
    write = on.expand(length, rows, heads)
    if s["beta"] is not None:
        write = write * s["beta"].double().view(rows, heads, length).permute(2, 0, 1)
    state = torch.zeros(rows, heads, dk, dv, dtype=torch.float64, device=q.device)
    if s["state"] is not None:
        state = s["state"].double().view(rows, heads, dk, dv)
    out = torch.empty(length, rows, heads, dv, dtype=torch.float64, device=q.device)
    for t in range(length):
        state = state * keep[t, :, :, None, None]
        u = v[t]
        if s["beta"] is not None:
            u = u - (k[t][..., None] * state).sum(2)
        state = state + k[t][..., None] * (write[t][..., None] * u)[:, :, None, :]
        out[t] = (q[t][..., None] * state).sum(2) * on[t][..., None]
    out = out / math.sqrt(dk)
    return {"out": out.permute(1, 2, 3, 0).reshape(-1), "state": state.reshape(-1)}


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_answer(s) if case["kind"] == "answer" else _exact_linear(s)
