"""Measured cases of the rotary append and of the 8-bit paged KV cache.

Four operators, each with a plain form in elementary torch operations and the call that a
user makes of the framework:

  append      kernels.rope_append into 16/32-bit pools: QK-norm (optional), rotary positions
              (half or interleaved pairs, part of the head, scaled for long contexts) and the
              write of K and V rows at their slots, for any number of tokens
  append_q8   the same call into pools of e4m3 values with one power-of-two scale for each
              page and KV head; a page that already holds rows is rescaled when its scale grows
  decode_q8   kernels.paged_decode_attention_q8: one query token per request over such pools
  prefill_q8  kernels.paged_prefill_attention_q8: one request's query tokens over its pages

Pools are [num_pages, kv_heads, page_size, head_dim], slots are page * page_size + offset.
"""

import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4}
_E4M3_MAX = 448.0
_MIN_EXP = -118  # smallest scale exponent: scale and 1 / scale are both normal fp32 values


def listed():
    return [
        # a decode step of 64 requests, 8B head shape with QK-norm: latency counts
        {"name": "append_step", "op": "append", "dtype": "bf16", "tokens": 64, "requests": 64,
         "start": 4000, "hq": 32, "hkv": 8, "dim": 128, "rot": 128, "pairs": "half", "norm": True,
         "base": 1e6, "factor": 1.0, "page": 16},
        # the prompts of four requests in one launch
        {"name": "append_prompt", "op": "append", "dtype": "bf16", "tokens": 8192, "requests": 4,
         "start": 0, "hq": 32, "hkv": 8, "dim": 128, "rot": 128, "pairs": "half", "norm": True,
         "base": 1e6, "factor": 1.0, "page": 16},
        # odd token count far into a stretched context, interleaved pairs over half the head
        {"name": "append_far", "op": "append", "dtype": "f32", "tokens": 1337, "requests": 3,
         "start": 250001, "hq": 14, "hkv": 2, "dim": 64, "rot": 32, "pairs": "interleaved",
         "norm": False, "base": 1e4, "factor": 8.0, "page": 32},
        # the same step into the 8-bit cache: most pages already hold rows
        {"name": "append_q8_step", "op": "append_q8", "dtype": "bf16", "tokens": 64, "requests": 64,
         "start": 4000, "hq": 32, "hkv": 8, "dim": 128, "rot": 128, "pairs": "half", "norm": True,
         "base": 1e6, "factor": 1.0, "page": 16},
        # prompts into the 8-bit cache
        {"name": "append_q8_prompt", "op": "append_q8", "dtype": "bf16", "tokens": 8192,
         "requests": 4, "start": 0, "hq": 32, "hkv": 8, "dim": 128, "rot": 128, "pairs": "half",
         "norm": True, "base": 1e6, "factor": 1.0, "page": 16},
        # ragged chunks of prompts that continue inside a page, pages of 32
        {"name": "append_q8_chunks", "op": "append_q8", "dtype": "f16", "tokens": 777,
         "requests": 5, "start": 1003, "hq": 14, "hkv": 2, "dim": 64, "rot": 32,
         "pairs": "interleaved", "norm": False, "base": 1e4, "factor": 4.0, "page": 32},
        # one user's step: latency of the split and the join
        {"name": "decode_q8_one", "op": "decode_q8", "dtype": "bf16", "requests": 1, "low": 1000,
         "high": 1000, "hq": 32, "hkv": 8, "dim": 128, "page": 16},
        # a step of 64 requests of very different lengths, 8B head shape
        {"name": "decode_q8_batch", "op": "decode_q8", "dtype": "bf16", "requests": 64, "low": 512,
         "high": 8192, "hq": 32, "hkv": 8, "dim": 128, "page": 16},
        # a mixture-of-experts model's heads: eight query heads for each KV head
        {"name": "decode_q8_wide", "op": "decode_q8", "dtype": "bf16", "requests": 128, "low": 200,
         "high": 4096, "hq": 32, "hkv": 4, "dim": 128, "page": 16},
        # few requests with long histories
        {"name": "decode_q8_long", "op": "decode_q8", "dtype": "f16", "requests": 8, "low": 30011,
         "high": 32768, "hq": 32, "hkv": 8, "dim": 128, "page": 32},
        # a chunk of a long prompt over what is cached already
        {"name": "prefill_q8_chunk", "op": "prefill_q8", "dtype": "bf16", "queries": 1024,
         "start": 7000, "hq": 32, "hkv": 8, "dim": 128, "page": 16},
        # a short continuation of a long history
        {"name": "prefill_q8_few", "op": "prefill_q8", "dtype": "f16", "queries": 17,
         "start": 20011, "hq": 32, "hkv": 8, "dim": 128, "page": 16},
    ]


def _spread(rng, low, high):
    """A whole number, spread evenly over the logarithm of low .. high."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng):
    op = rng.choice(["append", "append_q8", "decode_q8", "prefill_q8"])
    hkv = rng.choice([1, 2, 4, 8])
    case = {"op": op, "dtype": rng.choice(["bf16", "f16"]), "hkv": hkv,
            "hq": hkv * rng.choice([1, 2, 4]), "dim": rng.choice([64, 128]),
            "page": rng.choice([16, 32])}
    if op in ("append", "append_q8"):
        tokens = _spread(rng, 1, 8192)
        dim = case["dim"]
        if op == "append" and tokens <= 4096:
            case["dtype"] = rng.choice(["bf16", "f16", "f32"])
        case |= {"tokens": tokens, "requests": rng.randint(1, min(tokens, 64)),
                 "start": rng.choice([0, _spread(rng, 1, 300000)]),
                 "rot": rng.choice([dim, dim, dim // 2]),
                 "pairs": rng.choice(["half", "interleaved"]), "norm": rng.random() < 0.5,
                 "base": rng.choice([1e4, 1e6]), "factor": rng.choice([1.0, 4.0, 16.0])}
    elif op == "decode_q8":
        case["hq"] = hkv * rng.choice([1, 2, 4, 5, 8])
        requests = _spread(rng, 1, 128)
        high = _spread(rng, 1, min(32768, 262144 // requests))
        case |= {"requests": requests, "low": rng.randint(0, high), "high": high}
    else:
        queries = _spread(rng, 1, 1024)
        start = _spread(rng, 1, min(32768, 7_000_000 // queries))
        case |= {"queries": queries, "start": rng.choice([0, start, start])}
    return case


def _lengths(case):
    """The lengths of the case's requests, by the case alone: decode contexts between low and
    high, or how the tokens of an append fall to its requests."""
    n = case["requests"]
    if case["op"] == "decode_q8":
        low, high = case["low"], case["high"]
        return [low + int(round((high - low) * ((0.5 + 0.6180339887498949 * i) % 1.0)))
                for i in range(n)]
    spare = case["tokens"] - n
    cuts = sorted(int(spare * ((0.31 + 0.6180339887498949 * i) % 1.0)) for i in range(n - 1))
    return [1 + b - a for a, b in zip([0] + cuts, cuts + [spare])]


def _starts(case):
    """Where each request's tokens of an append begin in its sequence."""
    return [case["start"] + 5 * i if case["start"] else 0 for i in range(case["requests"])]


# ---------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------


def _rotary(rot, base, factor):
    """Frequencies of the pairs and the factor on cosine and sine. Beyond the trained length
    the slow pairs are interpolated and the fast ones kept, with a ramp between them, and the
    scores are sharpened a little (the YaRN rule, trained length 32768)."""
    inv = 1.0 / base ** (torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    if factor == 1.0:
        return inv.float(), 1.0
    turns = 32768.0 * inv / (2 * math.pi)
    keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0, 1)
    return (inv / factor * (1 - keep) + inv * keep).float(), 0.1 * math.log(factor) + 1.0


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(1_000_003 * int(seed) + 17)


def _normal(shape, gen):
    return torch.randn(shape, device="cuda", generator=gen)


def _keys(shape, gen):
    """Key rows: a few channels of each head are much larger than the others."""
    loud = 1 + 7 * (torch.rand(shape[-1], device="cuda", generator=gen) < 0.04)
    return _normal(shape, gen) * loud


def _filled_pools(pages, case, gen):
    """8-bit pools as appends leave them: e4m3 values and power-of-two scales."""
    shape = (pages, case["hkv"], case["page"], case["dim"])
    pools = []
    for x in (_keys(shape, gen), _normal(shape, gen)):
        x *= torch.exp(0.7 * _normal((pages, case["hkv"], 1, 1), gen))
        s = torch.exp2(_exponent(x.abs().amax((-2, -1))).float())
        pools += [(x / s[:, :, None, None]).to(torch.float8_e4m3fn), s]
    return pools


def prepare(case, seed):
    gen = _gen(seed)
    dt = _TYPES[case["dtype"]]
    hq, hkv, dim, page = case["hq"], case["hkv"], case["dim"], case["page"]
    state = {"case": case, "err": None}
    if case["op"] in ("append", "append_q8"):
        lens, starts = _lengths(case), _starts(case)
        # each request's new rows go to pages of its own, at the offsets its positions have
        spans = [(s % page + n + page - 1) // page for n, s in zip(lens, starts)]
        pages = sum(spans) + 7
        order = torch.randperm(pages, device="cuda", generator=gen)
        slots, positions, at = [], [], 0
        for n, s, span in zip(lens, starts, spans):
            rows = torch.arange(s % page, s % page + n, device="cuda")
            slots.append(order[at + rows // page] * page + rows % page)
            positions.append(torch.arange(s, s + n, device="cuda"))
            at += span
        tokens = case["tokens"]
        # q, k and v are the three parts of one projection's output
        qkv = torch.empty((tokens, (hq + 2 * hkv) * dim), dtype=dt, device="cuda")
        qkv[:, :hq * dim] = _normal((tokens, hq * dim), gen).to(dt)
        qkv[:, hq * dim:(hq + hkv) * dim] = _keys((tokens, hkv * dim), gen).to(dt)
        qkv[:, (hq + hkv) * dim:] = _normal((tokens, hkv * dim), gen).to(dt)
        inv, factor = _rotary(case["rot"], case["base"], case["factor"])
        state |= {"q": qkv[:, :hq * dim].view(tokens, hq, dim),
                  "k": qkv[:, hq * dim:(hq + hkv) * dim].view(tokens, hkv, dim),
                  "v": qkv[:, (hq + hkv) * dim:].view(tokens, hkv, dim),
                  "positions": torch.cat(positions), "slots": torch.cat(slots),
                  "inv_freq": inv.cuda(), "rope_scale": factor,
                  "qw": (1 + 0.2 * _normal((dim,), gen)).to(dt) if case["norm"] else None,
                  "kw": (1 + 0.2 * _normal((dim,), gen)).to(dt) if case["norm"] else None}
        if case["op"] == "append":
            state["k_pool"] = _normal((pages, hkv, page, dim), gen).to(dt)
            state["v_pool"] = _normal((pages, hkv, page, dim), gen).to(dt)
        else:
            state |= dict(zip(("k_pool", "k_scale", "v_pool", "v_scale"),
                              _filled_pools(pages, case, gen)))
        return state
    if case["op"] == "decode_q8":
        lens, queries = _lengths(case), case["requests"]
    else:
        lens, queries = [case["start"] + case["queries"]], case["queries"]
    spans = [(n + page - 1) // page for n in lens]
    pages = sum(spans) + 5
    pools = _filled_pools(pages, case, gen)
    order = torch.randperm(pages, device="cuda", generator=gen).to(torch.int32)
    width = max(1, max(spans))
    tables = torch.zeros((len(lens), width), dtype=torch.int32, device="cuda")
    ends, at = [], 0
    for i, (n, span) in enumerate(zip(lens, spans)):
        tables[i, :span] = order[at:at + span]
        at += span
        if n % page:
            ends.append((i, span - 1, n % page))
    # what lies behind a request's last row, and in pages of nobody, was never written
    for pool, scale in (pools[:2], pools[2:]):
        raw = pool.view(torch.uint8)
        raw[order[at:].long()] = 0x7F
        scale[order[at:].long()] = math.nan
        for i, last, used in ends:
            raw[tables[i, last].long(), :, used:] = 0x7F
    state |= dict(zip(("k_pool", "k_scale", "v_pool", "v_scale"), pools))
    state |= {"q": _normal((queries, hq, dim), gen).to(dt), "tables": tables,
              "lens": torch.tensor(lens, dtype=torch.int32, device="cuda")}
    return state


# ---------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------


def _rotated(x, state, weight):
    """QK-norm and rotary positions of the rows x [tokens, heads, dim], in fp32."""
    x = x.float()
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-5) * weight.float()
    angle = state["positions"].double()[:, None] * state["inv_freq"].double()
    c = (angle.cos() * state["rope_scale"]).float()[:, None]
    s = (angle.sin() * state["rope_scale"]).float()[:, None]
    rot = 2 * c.shape[-1]
    if state["case"]["pairs"] == "half":
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat((a * c - b * s, b * c + a * s), -1)
    else:
        a, b = x[..., :rot:2], x[..., 1:rot:2]
        turned = torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2)
    return torch.cat((turned, x[..., rot:]), -1)


def _exponent(amax):
    """Smallest e >= _MIN_EXP with amax <= 448 * 2^e (448 = 0.875 * 2^9)."""
    m, e = torch.frexp(amax)
    return torch.where(amax > 0, e - 9 + (m > 0.875), _MIN_EXP).clamp(min=_MIN_EXP)


def _to_e4m3(x):
    return x.clamp(-_E4M3_MAX, _E4M3_MAX).to(torch.float8_e4m3fn)


def _append_8bit(rows, slots, pool, scale):
    """Rows [tokens, kv_heads, dim] into their pages; a page's scale covers its kept rows
    (those before the first new one) and the new ones."""
    page_size = pool.shape[2]
    pages, which = torch.unique(slots // page_size, return_inverse=True)
    n, heads = pages.shape[0], rows.shape[1]
    first = torch.full((n,), page_size, device=rows.device)
    first = first.scatter_reduce(0, which, slots % page_size, "amin")
    amax = torch.where(rows.isfinite(), rows.abs(), 0).amax(-1)
    amax = torch.zeros((n, heads), device=rows.device).scatter_reduce(
        0, which[:, None].expand_as(amax), amax, "amax")
    before = scale[pages]
    kept = (first > 0)[:, None]
    exponent = torch.maximum(_exponent(amax),
                             torch.where(kept, torch.frexp(before)[1] - 1, _MIN_EXP))
    after = torch.exp2(exponent.float())
    ratio = torch.where(kept, before / after, 1)
    tiles = pool[pages]
    moved = _to_e4m3(tiles.float() * ratio[:, :, None, None]).view(torch.uint8)
    keep = (torch.arange(page_size, device=rows.device) < first[:, None])[:, None, :, None]
    raw = pool.view(torch.uint8)
    raw[pages] = torch.where(keep, moved, tiles.view(torch.uint8))
    raw[slots // page_size, :, slots % page_size] = _to_e4m3(
        rows / after[which][..., None]).view(torch.uint8)
    scale[pages] = after


def _append(state):
    slots, k_pool, v_pool = state["slots"], state["k_pool"], state["v_pool"]
    q = _rotated(state["q"], state, state["qw"])
    k = _rotated(state["k"], state, state["kw"])
    if state["case"]["op"] == "append":
        page, offset = slots // k_pool.shape[2], slots % k_pool.shape[2]
        k_pool[page, :, offset] = k.to(k_pool.dtype)
        v_pool[page, :, offset] = state["v"].to(v_pool.dtype)
        return {"q": q.to(k_pool.dtype), "k_pool": k_pool, "v_pool": v_pool}
    _append_8bit(k, slots, k_pool, state["k_scale"])
    _append_8bit(state["v"].float(), slots, v_pool, state["v_scale"])
    return {"q": q.to(state["q"].dtype), "k_pool": k_pool, "v_pool": v_pool,
            "k_scale": state["k_scale"], "v_scale": state["v_scale"]}


def _values(pool, scale, tables):
    """[requests, kv_heads, tokens, dim] in fp32 of the pages that the tables name."""
    x = pool[tables.long()].float() * scale[tables.long()][..., None, None]
    return x.transpose(1, 2).flatten(2, 3)


def _attend(q, k, v, seen):
    """q [b, h, group, n, d], k and v [b, h, t, d], seen [b, n, t]: softmax over the seen keys
    of each row; zeros where none is seen."""
    b, h, g, n, d = q.shape
    x = torch.matmul(q.reshape(b, h, g * n, d), k.transpose(-1, -2)) / math.sqrt(d)
    x = torch.where(seen[:, None, None], x.view(b, h, g, n, -1), -math.inf)
    top = x.amax(-1, keepdim=True)
    w = torch.exp(x - torch.where(top.isinf(), 0, top))
    total = w.sum(-1, keepdim=True)
    v = torch.where(seen.any(1)[:, None, :, None], v, 0)
    out = torch.matmul(w.view(b, h, g * n, -1), v).view(b, h, g, n, d)
    return torch.where(total > 0, out / total, 0)


def _attention(state):
    case = state["case"]
    k = _values(state["k_pool"], state["k_scale"], state["tables"])
    v = _values(state["v_pool"], state["v_scale"], state["tables"])
    q = state["q"].float()
    rows, hq, dim = q.shape
    group = hq // case["hkv"]
    t = torch.arange(k.shape[2], device=q.device)
    if case["op"] == "decode_q8":
        x = q.view(rows, case["hkv"], group, 1, dim)
        out = _attend(x, k, v, (t < state["lens"][:, None])[:, None])
    else:
        x = q.view(rows, case["hkv"], group, dim).permute(1, 2, 0, 3)[None]
        at = case["start"] + torch.arange(rows, device=q.device)
        out = _attend(x, k, v, (t <= at[:, None])[None])
        out = out[0].permute(2, 0, 1, 3)
    return out.reshape(rows, hq, dim).to(state["q"].dtype)


def _with_framework(state):
    from plastic_infer_b200 import kernels

    case = state["case"]
    if case["op"] in ("append", "append_q8"):
        q = kernels.rope_append(
            state["q"], state["k"], state["v"], state["positions"], state["inv_freq"],
            state["slots"], state["k_pool"], state["v_pool"], q_norm_weight=state["qw"],
            k_norm_weight=state["kw"], eps=1e-5, interleaved=case["pairs"] == "interleaved",
            rope_scale=state["rope_scale"], k_scale=state.get("k_scale"),
            v_scale=state.get("v_scale"))
        out = {"q": q, "k_pool": state["k_pool"], "v_pool": state["v_pool"]}
        if case["op"] == "append_q8":
            out |= {"k_scale": state["k_scale"], "v_scale": state["v_scale"]}
        return out
    pools = (state["k_pool"], state["v_pool"], state["k_scale"], state["v_scale"])
    if case["op"] == "decode_q8":
        return kernels.paged_decode_attention_q8(state["q"], *pools, state["tables"], state["lens"])
    return kernels.paged_prefill_attention_q8(state["q"], *pools, state["tables"][0],
                                              case["start"] + case["queries"],
                                              q_start=case["start"], causal=True)


def run(state):
    if own:
        return _with_framework(state)
    if state["case"]["op"] in ("append", "append_q8"):
        return _append(state)
    return _attention(state)


# ---------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------


def work(case):
    size = _BYTES[case["dtype"]]
    hq, hkv, dim, page = case["hq"], case["hkv"], case["dim"], case["page"]
    if case["op"] in ("append", "append_q8"):
        n = case["tokens"]
        moved = n * (hq + 2 * hkv) * dim * size + n * 16 + n * hq * dim * size
        if case["op"] == "append":
            moved += n * 2 * hkv * dim * size
        else:
            lens, starts = _lengths(case), _starts(case)
            touched = sum((s % page + m + page - 1) // page for m, s in zip(lens, starts))
            moved += n * 2 * hkv * dim + touched * 2 * hkv * 4
        return {"bytes": moved, "flops": n * (hq + hkv) * (3 * case["rot"] + 4 * dim * case["norm"])}
    if case["op"] == "decode_q8":
        lens, queries = _lengths(case), case["requests"]
        pairs = sum(lens)
    else:
        queries = case["queries"]
        lens = [case["start"] + queries]
        pairs = queries * case["start"] + queries * (queries + 1) // 2
    pages = sum((n + page - 1) // page for n in lens)
    moved = 2 * sum(lens) * hkv * dim + pages * (2 * hkv * 4 + 4) + 2 * queries * hq * dim * size
    return {"bytes": moved, "flops": 4 * pairs * hq * dim}


# ---------------------------------------------------------------------------------------
# 64 bits, from the definitions
# ---------------------------------------------------------------------------------------


def _exact_turn(x, state, weight):
    x = x.double()
    if weight is not None:
        x = x * (x.square().mean(-1, keepdim=True) + 1e-5).rsqrt() * weight.double()
    half = state["inv_freq"].numel()
    turn = torch.polar(torch.full((1, 1), state["rope_scale"], dtype=torch.float64, device="cuda"),
                       state["positions"].double()[:, None] * state["inv_freq"].double())
    first = torch.arange(half, device="cuda")
    if state["case"]["pairs"] == "half":
        i, j = first, first + half
    else:
        i, j = 2 * first, 2 * first + 1
    z = torch.complex(x[..., i], x[..., j]) * turn[:, None]
    out = x.clone()
    out[..., i], out[..., j] = z.real, z.imag
    return out


def _exact_e4m3(x):
    """The e4m3 value nearest to x (ties to even), at most 448 in size."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(x / step) * step).clamp(-_E4M3_MAX, _E4M3_MAX)


def _exact_blocks(rows, state, pool, scale):
    values, scale = pool.double(), scale.double()
    size = pool.shape[2]
    slots = state["slots"].tolist()
    at = 0
    while at < len(slots):
        page, offset = divmod(slots[at], size)
        n = 1
        while at + n < len(slots) and offset + n < size and slots[at + n] == slots[at] + n:
            n += 1
        for h in range(rows.shape[1]):
            new = rows[at:at + n, h]
            top = float(new.abs().max())
            e = max(_MIN_EXP, math.ceil(math.log2(top / _E4M3_MAX))) if top > 0 else _MIN_EXP
            if top > 0 and top <= _E4M3_MAX * 2.0 ** (e - 1) and e > _MIN_EXP:
                e -= 1
            if offset:
                e = max(e, int(round(math.log2(float(scale[page, h])))))
                values[page, h, :offset] = _exact_e4m3(
                    values[page, h, :offset] * (float(scale[page, h]) / 2.0 ** e))
            values[page, h, offset:offset + n] = _exact_e4m3(new / 2.0 ** e)
            scale[page, h] = 2.0 ** e
        at += n
    return values, scale


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] in ("append", "append_q8"):
        q = _exact_turn(state["q"], state, state["qw"])
        k = _exact_turn(state["k"], state, state["kw"])
        v = state["v"].double()
        if case["op"] == "append":
            out = {"q": q}
            for name, rows in (("k_pool", k), ("v_pool", v)):
                flat = state[name].double().transpose(1, 2).flatten(0, 1)
                flat[state["slots"]] = rows
                out[name] = flat.unflatten(0, (-1, case["page"])).transpose(1, 2)
            return out
        kp, ks = _exact_blocks(k, state, state["k_pool"], state["k_scale"])
        vp, vs = _exact_blocks(v, state, state["v_pool"], state["v_scale"])
        return {"q": q, "k_pool": kp, "v_pool": vp, "k_scale": ks, "v_scale": vs}
    hkv, dim, page = case["hkv"], case["dim"], case["page"]
    group = case["hq"] // hkv
    lens = state["lens"].tolist()
    out = torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        if n == 0:
            continue
        ids = state["tables"][b, :(n + page - 1) // page].long()
        k, v = (torch.einsum("phtd,ph->hptd", state[p][ids].double(), state[s][ids].double())
                .flatten(1, 2)[:, :n] for p, s in (("k_pool", "k_scale"), ("v_pool", "v_scale")))
        for h in range(hkv):
            heads = slice(h * group, (h + 1) * group)
            if case["op"] == "decode_q8":
                p = torch.softmax(state["q"][b, heads].double() @ k[h].T * dim ** -0.5, -1)
                out[b, heads] = p @ v[h]
            else:
                q = state["q"][:, heads].double().transpose(0, 1)
                hidden = torch.ones((q.shape[1], n), dtype=torch.bool, device="cuda").triu(
                    case["start"] + 1)
                p = torch.softmax((q @ k[h].T * dim ** -0.5).masked_fill(hidden, -math.inf), -1)
                out[:, heads] = (p @ v[h]).transpose(0, 1)
    return out
