"""Cases of the paged-serving operators: page planning, cache append, attention of a
chunk of new tokens over the paged cache, and the residual RMS norm with an int8 output.

`run` computes an operator in its plain form (elementary torch operations in 32 bits,
rounded once at the end), or, where `own` is true, through the calls a user makes of
`thunderllamax_b200`.  `exact` computes the same from the definitions in 64 bits.
"""
import math

import torch

own = False

HEADS = {  # query heads, KV heads, head dim
    "a": (24, 4, 256),   # the full-attention layers of this repository's attention
    "b": (32, 8, 128),
    "c": (8, 8, 64),
    "d": (16, 1, 128),
    "e": (12, 2, 64),
}
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


# ---------------------------------------------------------------------- cases
def listed():
    return [
        # one decode step's bookkeeping for a modest batch: pure latency
        {"name": "plan_decode_64", "op": "plan", "requests": 64, "new": 1, "kv_hi": 8192, "page": 16,
         "short": False},
        # a step that admits many prompts at once: 1000 requests of ragged chunks, 16-token pages
        {"name": "plan_admit_1000", "op": "plan", "requests": 1000, "new": 120, "kv_hi": 4000, "page": 16,
         "short": False},
        # the new rows of one decode step into the int8 cache
        {"name": "append_decode_i8", "op": "append", "tokens": 64, "heads": "a", "cache": "i8", "x": "f16", "page": 64},
        # a large prefill chunk into a bf16 cache
        {"name": "append_chunk_bf16", "op": "append", "tokens": 8191, "heads": "b", "cache": "bf16", "x": "bf16",
         "page": 16},
        # the norm before the FFN for the rows of one verify step (fp32 residual stream)
        {"name": "norm_rows_11", "op": "norm", "m": 11, "k": 5120, "x": "f32", "r": "f32"},
        # the same for a prefill chunk
        {"name": "norm_chunk_2048", "op": "norm", "m": 2048, "k": 5120, "x": "f32", "r": "f32"},
        # a long chunk of a narrower model with a 16-bit residual stream, odd row count
        {"name": "norm_chunk_16bit", "op": "norm", "m": 8193, "k": 2048, "x": "f16", "r": "f16"},
        # one request, one new token: the latency of a single user's decode
        {"name": "attn_decode_1", "op": "attn", "requests": 1, "new_lo": 1, "new_hi": 1, "kv_lo": 4097, "kv_hi": 4097,
         "heads": "a", "cache": "i8", "q": "f16", "page": 64, "gate": True},
        # a decode batch of ragged contexts
        {"name": "attn_decode_64", "op": "attn", "requests": 64, "new_lo": 1, "new_hi": 1, "kv_lo": 300,
         "kv_hi": 16000, "heads": "a", "cache": "i8", "q": "f16", "page": 64, "gate": True},
        # the verify rows of one request at a long context
        {"name": "attn_verify_100k", "op": "attn", "requests": 1, "new_lo": 11, "new_hi": 11, "kv_lo": 100011,
         "kv_hi": 100011, "heads": "a", "cache": "i8", "q": "f16", "page": 64, "gate": True},
        # a mixed step: requests from a single token to a full chunk, small pages
        {"name": "attn_mixed_bf16", "op": "attn", "requests": 9, "new_lo": 1, "new_hi": 1000, "kv_lo": 200,
         "kv_hi": 7001, "heads": "b", "cache": "bf16", "q": "bf16", "page": 16, "gate": False},
        # a prefill chunk over an equally long cached prefix: compute bound
        {"name": "attn_chunk_4096", "op": "attn", "requests": 1, "new_lo": 4096, "new_hi": 4096, "kv_lo": 8192,
         "kv_hi": 8192, "heads": "a", "cache": "f16", "q": "f16", "page": 64, "gate": True},
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over the logarithm."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))
    v = min(hi, max(lo, v))
    return v + 1 if v == 3072 else v


def draw(rng):
    op = rng.choice(["plan", "append", "norm", "attn", "attn", "attn"])
    if op == "plan":
        return {"op": op, "requests": _log(rng, 1, 1000), "new": _log(rng, 1, 120), "kv_hi": _log(rng, 1, 8000),
                "page": rng.choice([8, 16, 64, 256]), "short": rng.random() < 0.3}
    if op == "append":
        heads, cache = rng.choice("abcde"), rng.choice(["f16", "bf16", "i8"])
        return {"op": op, "tokens": _log(rng, 1, 8000), "heads": heads, "cache": cache,
                "x": rng.choice(["f16", "bf16", "f32"]) if cache == "i8" else cache,
                "page": rng.choice([8, 16, 64, 256])}
    if op == "norm":
        k = 128 * _log(rng, 1, 63)
        k = k + 128 if k == 3072 else k
        x = rng.choice(["f16", "bf16", "f32"])
        return {"op": op, "m": _log(rng, 1, 16000000 // k), "k": k, "x": x, "r": rng.choice([x, "f32"])}
    heads, cache = rng.choice("aabcde"), rng.choice(["f16", "bf16", "i8"])
    hq, hkv, d = HEADS[heads]
    new_hi = _log(rng, 1, rng.choice([1, 16, 4000]))
    kv_hi = _log(rng, max(new_hi, 2), 16000)
    most = min(2.4e9 / (hkv * d * 4.0 * kv_hi), 2.4e9 / (hq * 4.0 * new_hi * kv_hi),
               2e11 / (hq * d * 2.0 * new_hi * kv_hi))
    return {"op": op, "requests": _log(rng, 1, max(1, min(96, int(most)))), "new_lo": _log(rng, 1, new_hi),
            "new_hi": new_hi, "kv_lo": _log(rng, 1, kv_hi), "kv_hi": kv_hi, "heads": heads, "cache": cache,
            "q": "f16" if cache == "i8" else cache, "page": rng.choice([8, 16, 64, 256]),
            "gate": rng.random() < 0.5}


def _spread(lo, hi, n, step):
    """n whole numbers from lo to hi, evenly over the logarithm, in a shuffled but fixed order; the first is hi."""
    v = [hi if i == 0 else int(round(lo * (hi / lo) ** ((i * step % n) / max(1, n - 1)))) for i in range(n)]
    return [min(hi, max(lo, x + (x == 3072))) for x in v]


def _lengths(case):
    """(new tokens, cached and new tokens) of each request: fixed by the case."""
    if case["op"] == "plan":
        n = case["requests"]
        new = [1 + (i * 7919) % (2 * case["new"] - 1) for i in range(n)]
        cached = [0 if i % 5 == 4 else (i * 104729 + 11) % (case["kv_hi"] + 1) for i in range(n)]
        return new, [a + b for a, b in zip(new, cached)]
    n = case["requests"]
    new = _spread(case["new_lo"], case["new_hi"], n, 7)
    kv = _spread(case["kv_lo"], case["kv_hi"], n, 11)
    return new, [max(a, b) for a, b in zip(new, kv)]


def _ceil(a, b):
    return -(-a // b)


def work(case):
    op = case["op"]
    if op == "plan":
        new, kv = _lengths(case)
        got = sum(_ceil(t, case["page"]) - _ceil(t - n, case["page"]) for n, t in zip(new, kv))
        # lengths and held counts in; starts, lengths, held counts and status out; a free page id read and
        # a table entry written for each page taken; a slot and a position for each token
        return {"bytes": 4 * (7 * len(new) + 3) + 8 * got + 8 * sum(new), "flops": 0}
    if op == "append":
        _, h, d = HEADS[case["heads"]]
        t = case["tokens"]
        size = TYPES[case["x"]].itemsize
        row = d + d // 16 if case["cache"] == "i8" else 2 * d
        return {"bytes": 2 * t * h * (d * size + row) + 4 * t, "flops": 0}
    if op == "norm":
        m, k = case["m"], case["k"]
        return {"bytes": m * k * (TYPES[case["x"]].itemsize + 2 * TYPES[case["r"]].itemsize + 1) + m * k // 32 + 4 * k,
                "flops": 0}
    hq, hkv, d = HEADS[case["heads"]]
    new, kv = _lengths(case)
    row = d + d // 16 if case["cache"] == "i8" else 2 * d
    q = sum(new) * hq * d * 2
    pairs = sum(n * (t - n) + n * (n + 1) // 2 for n, t in zip(new, kv))
    return {"bytes": 2 * sum(kv) * hkv * row + q * (3 if case["gate"] else 2) + 4 * sum(_ceil(t, case["page"]) for t in kv),
            "flops": 4 * hq * d * pairs}


# --------------------------------------------------------------------- inputs
def _randn(g, shape, dtype, scale=1.0):
    """Normal values of projections and residual streams, a few channels of them larger."""
    x = torch.randn(shape, generator=g, device="cuda")
    x.mul_(scale)
    x[..., ::61] *= 3.0
    return x.to(dtype)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _cache(g, case, pages):
    """A cache of random pages [page][head][slot][dim]: (k, v, k scales, v scales)."""
    _, h, d = HEADS[case["heads"]]
    shape = (pages, h, case["page"], d)
    if case["cache"] == "i8":
        made = [torch.randint(1, 256, shape, dtype=torch.uint8, generator=g, device="cuda") for _ in range(2)]
        scales = [torch.rand(shape[:3] + (d // 32,), generator=g, device="cuda").mul_(0.018).add_(0.012).half()
                  for _ in range(2)]
        return made + scales
    return [_randn(g, shape, TYPES[case["cache"]]) for _ in range(2)] + [None, None]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(1000003 * (seed + 1) + 17)
    st = {"case": dict(case)}
    make = {"plan": _prepare_plan, "append": _prepare_append, "norm": _prepare_norm, "attn": _prepare_attn}
    make[case["op"]](case, g, st)
    return st


def _prepare_plan(case, g, st):
    new, kv = _lengths(case)
    n, page = len(new), case["page"]
    had = [_ceil(t - a, page) for a, t in zip(new, kv)]
    width = max(_ceil(t, page) for t in kv) + 1
    pages = sum(_ceil(t, page) for t in kv) + 7
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    st["table"] = torch.full((n, width), -1, dtype=torch.int32, device="cuda")
    held = _ints(had)
    col = torch.arange(width, device="cuda")
    mine = col[None, :] < held[:, None]
    st["table"][mine] = order[:sum(had)]
    st["held"], st["free"] = held, torch.full_like(order, -1)
    st["free"][:pages - sum(had)] = order[sum(had):]
    # a pool that runs short serves the first requests of the batch and refuses the rest
    st["n_free"] = _ints([(pages - sum(had)) // (2 if case["short"] else 1)])
    st["new"], st["cached"] = _ints(new), _ints([t - a for a, t in zip(new, kv)])
    st["tokens"] = sum(new)
    st["held_out"], st["n_free_out"] = torch.empty_like(held), torch.empty_like(st["n_free"])
    if own:
        from thunderllamax_b200 import paged

        st["pages"] = paged.PageTable(n, width, pages, page, table=st["table"], held=st["held"], free=st["free"],
                                      n_free=st["n_free"])
        st["plan"] = paged.Plan(n, st["tokens"])


def _prepare_append(case, g, st):
    _, h, d = HEADS[case["heads"]]
    t, page = case["tokens"], case["page"]
    pages = _ceil(t, page) + 2
    st["cache"] = _cache(g, case, pages)
    # the projections' rows hold k and v of a token side by side
    kv = _randn(g, (t, 2, h, d), TYPES[case["x"]])
    st["k"], st["v"] = kv[:, 0], kv[:, 1]
    st["slots"] = (torch.randperm(pages, generator=g, device="cuda")[:, None] * page
                   + torch.arange(page, device="cuda")[None, :]).reshape(-1)[:t].to(torch.int32)
    st["slots"][::97] = -1                      # tokens of requests that got no pages
    if own:
        from thunderllamax_b200 import paged

        st["store"] = paged.PagedCache(*st["cache"])


def _prepare_norm(case, g, st):
    m, k = case["m"], case["k"]
    st["x"] = _randn(g, (m, k), TYPES[case["x"]])
    st["r"] = _randn(g, (m, k), TYPES[case["r"]], 2.0)
    st["w"] = 1.0 + 0.2 * torch.randn(k, generator=g, device="cuda")
    st["out"] = torch.empty_like(st["r"])
    st["xq"] = torch.empty((m, k), dtype=torch.int8, device="cuda")
    st["sx"] = torch.empty((m, k // 128), device="cuda")


def _prepare_attn(case, g, st):
    hq, hkv, d = HEADS[case["heads"]]
    new, kv = _lengths(case)
    page = case["page"]
    need = [_ceil(t, page) for t in kv]
    pages, n = sum(need) + 3, len(new)
    st["cache"] = _cache(g, case, pages)
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    st["table"] = torch.full((n, max(need)), -1, dtype=torch.int32, device="cuda")
    mine = torch.arange(max(need), device="cuda")[None, :] < _ints(need)[:, None]
    st["table"][mine] = order[:sum(need)]
    if case["cache"] != "i8":
        # what follows a request's last token in its last page was never written
        last = st["table"][torch.arange(n, device="cuda"), _ints(need).long() - 1].long()
        stale = torch.arange(page, device="cuda")[None, :] >= (_ints(kv) - (_ints(need) - 1) * page)[:, None]
        hole = stale[:, None, :, None]
        for c in st["cache"][:2]:
            c[last] = torch.where(hole, torch.full_like(c[last], float("nan")), c[last])
    st["q_start"] = _ints([0] + torch.tensor(new).cumsum(0).tolist())
    st["kv_len"] = _ints(kv)
    st["new_hi"], st["kv_hi"], st["scale"] = max(new), max(kv), d ** -0.5
    st["q"] = _randn(g, (sum(new), hq, d), TYPES[case["q"]])
    st["gate"] = _randn(g, (sum(new), hq, d), TYPES[case["q"]]) if case["gate"] else None
    st["out"] = torch.empty_like(st["q"])
    if own:
        from thunderllamax_b200 import paged

        st["store"] = paged.PagedCache(*st["cache"])
        st["attn"] = paged.PagedAttention(hq, hkv, d)


# ------------------------------------------------------------------------ run
def run(st):
    op = st["case"]["op"]
    if op == "plan":
        return _run_plan(st)
    if op == "append":
        return _run_append(st)
    if op == "norm":
        return _run_norm(st)
    return _run_attn(st)


def _run_plan(st):
    page = st["case"]["page"]
    if own:
        p = st["pages"].plan(st["cached"], st["new"], st["plan"], held_out=st["held_out"], n_free_out=st["n_free_out"])
        return {"table": st["table"], "held": st["held_out"], "n_free": st["n_free_out"], "q_start": p.q_start,
                "kv_len": p.kv_len, "slots": p.slots, "positions": p.positions, "status": p.status}
    cached, new, held, table = st["cached"].long(), st["new"].long(), st["held"].long(), st["table"]
    need = (cached + new + page - 1) // page
    take = (need - held).clamp(min=0)
    end = take.cumsum(0)
    n_free = st["n_free"].long()
    ok = ((take == 0) | (end <= n_free)) & (need <= table.shape[1])
    # the i-th page that the batch takes comes from the end of the free pages
    col = torch.arange(table.shape[1], device="cuda")[None, :]
    rank = (end - take)[:, None] + col - held[:, None]
    fresh = (col >= held[:, None]) & (col < need[:, None]) & ok[:, None]
    page_id = st["free"][(n_free - 1 - rank).clamp(0, st["free"].numel() - 1)]
    table.copy_(torch.where(fresh, page_id, table))
    held_out = torch.where(ok, held + take, held)
    start = torch.cat([torch.zeros_like(new[:1]), new.cumsum(0)])
    tok = torch.arange(st["tokens"], device="cuda")
    b = torch.searchsorted(start, tok, right=True) - 1
    pos = cached[b] + tok - start[b]
    slot = torch.where(ok[b], table[b, pos // page].long() * page + pos % page, torch.full_like(pos, -1))
    i32 = torch.int32
    return {"table": table, "held": held_out.to(i32), "n_free": (n_free - torch.where(ok, take, 0 * take).sum()).to(i32),
            "q_start": start.to(i32), "kv_len": torch.where(ok, cached + new, 0 * new).to(i32), "slots": slot.to(i32),
            "positions": pos.to(i32), "status": (~ok).to(i32)}


def _stands_for(st):
    """The values an int8 cache stands for (16-bit caches are returned as they are)."""
    k, v, ks, vs = st["cache"]
    if ks is None:
        return {"k": k, "v": v}
    k, v = ((c.view(*s.shape, 32).to(torch.int16) - 128) * s[..., None] for c, s in ((k, ks), (v, vs)))
    return {"k": k, "v": v, "k_scale": ks, "v_scale": vs}


def _run_append(st):
    if own:
        st["store"].append(st["k"], st["v"], st["slots"])
        return _stands_for(st)
    k, v, ks, vs = st["cache"]
    pages, h, page, d = k.shape
    slot = st["slots"].long()
    slot = torch.where(slot < 0, torch.full_like(slot, pages * page), slot)
    at = (slot // page, slice(None), slot % page)
    x = {"k": st["k"].float(), "v": st["v"].float()}
    if ks is not None:
        a = {n: t.view(-1, h, d // 32, 32) for n, t in x.items()}
        top = {n: t.abs().amax(-1) for n, t in a.items()}
        s = {n: torch.where(t > 0, t * (1.0 / 127.0), torch.full_like(t, 1e-8)).half() for n, t in top.items()}
        x = {n: ((t / s[n].float()[..., None]).nan_to_num(nan=-127.0).clamp(-127, 127).round() + 128).reshape(-1, h, d)
             for n, t in a.items()}
        _put(ks, at, s["k"])
        _put(vs, at, s["v"])
    _put(k, at, x["k"].to(k.dtype))
    _put(v, at, x["v"].to(v.dtype))
    return _stands_for(st)


def _put(cache, at, rows):
    """cache[page, :, slot] = rows, with a spare page for the tokens that have no slot."""
    wide = torch.cat([cache, cache[:1]])
    wide[at] = rows
    cache.copy_(wide[:-1])


def _run_norm(st):
    m, k = st["case"]["m"], st["case"]["k"]
    if own:
        from thunderllamax_b200 import prefill

        out, xq, sx = prefill.add_rms_norm_q8(st["x"], st["r"], st["w"], 1e-6, out=st["out"], xq=st["xq"], sx=st["sx"])
        return {"residual": out, "values": xq.view(m, k // 128, 128) * sx.half()[..., None], "scales": sx}
    h = st["x"].float() + st["r"].float()
    y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + 1e-6) * st["w"]
    y = y.view(m, k // 128, 128)
    sx = y.abs().amax(-1).clamp(min=1e-6) * (1.0 / 127.0)
    q = (y / sx[..., None]).round().clamp(-127, 127)
    return {"residual": h.to(st["r"].dtype), "values": q.half() * sx.half()[..., None], "scales": sx}


def _rows(cache, scale, table, page, most):
    """The cached rows of each request in order: [request][KV head][position][dim] in 32 bits."""
    idx = table[:, :_ceil(most, page)].clamp(min=0).long()
    x = cache[idx]
    if scale is None:
        x = x.float()
    else:   # an int8 cache stands for code * scale, rounded to fp16
        s = scale[idx]
        x = ((x.view(*s.shape, 32).float() - 128.0) * s.float()[..., None]).half().float().flatten(-2)
    return x.permute(0, 2, 1, 3, 4).flatten(2, 3)


def _run_attn(st):
    if own:
        return st["attn"](st["store"], st["table"], st["q_start"], st["kv_len"], st["q"], gate=st["gate"],
                          scale=st["scale"], max_new=st["new_hi"], out=st["out"])
    case = st["case"]
    hq, hkv, d = HEADS[case["heads"]]
    kc, vc, ks, vs = st["cache"]
    k = _rows(kc, ks, st["table"], case["page"], st["kv_hi"])
    v = _rows(vc, vs, st["table"], case["page"], st["kv_hi"])
    n_req, most = st["kv_len"].numel(), st["new_hi"]
    start, kv = st["q_start"].long(), st["kv_len"].long()
    key, t = torch.arange(k.shape[2], device="cuda"), torch.arange(most, device="cuda")
    v = torch.where((key[None, :] < kv[:, None])[:, None, :, None], v, 0.0)
    tokens = st["q"].shape[0]
    q = st["q"][(start[:-1, None] + t).clamp(max=tokens - 1)].float()        # [request][t][head][dim]
    q = q.view(n_req, most, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(n_req, hkv, -1, d)
    s = (q @ k.transpose(-1, -2)).mul_(st["scale"]).view(n_req, hkv, hq // hkv, most, -1)
    limit = (kv - (start[1:] - start[:-1]))[:, None] + t                      # the last key a token sees
    seen = (key <= limit[..., None]) & (key < kv[:, None, None])
    s.masked_fill_(~seen[:, None, None], float("-inf"))
    top = s.amax(-1, keepdim=True)
    p = s.sub_(torch.where(top.isinf(), 0.0, top)).exp_()
    total = p.sum(-1)
    o = (p.view(n_req, hkv, -1, p.shape[-1]) @ v).view(n_req, hkv, hq // hkv, most, d)
    o = o / torch.where(total == 0, 1.0, total)[..., None]
    tok = torch.arange(tokens, device="cuda")
    b = torch.searchsorted(start, tok, right=True) - 1
    o = o.permute(0, 3, 1, 2, 4).reshape(n_req * most, hq, d)[b * most + tok - start[b]]
    if st["gate"] is not None:
        o = o / (1.0 + torch.exp(-st["gate"].float()))
    return o.to(st["q"].dtype)


# ---------------------------------------------------------------------- exact
def exact(case, seed):
    """What `run` returns, from the definitions, one request or row at a time, in 64 bits."""
    if case["op"] == "plan":
        return None
    st = prepare(case, seed)
    with torch.no_grad():
        return {"append": _exact_append, "norm": _exact_norm, "attn": _exact_attn}[case["op"]](st)


def _exact_append(st):
    k, v, ks, vs = st["cache"]
    pages, h, page, d = k.shape
    out = {}
    for name, cache, scale, rows in (("k", k, ks, st["k"]), ("v", v, vs, st["v"])):
        if scale is None:
            flat = cache.double().permute(0, 2, 1, 3).reshape(pages * page, h, d)
        else:
            flat = (cache.view(pages, h, page, d // 32, 32).double() - 128) * scale.double()[..., None]
            flat = flat.flatten(-2).permute(0, 2, 1, 3).reshape(pages * page, h, d)
            sflat = scale.double().permute(0, 2, 1, 3).reshape(pages * page, h, d // 32)
        use = st["slots"] >= 0
        to, x = st["slots"][use].long(), rows[use].double()
        if scale is not None:
            g = x.reshape(-1, h, d // 32, 32)
            s = (g.abs().amax(-1) / 127.0).half().double()
            x = ((g / s[..., None]).clamp(-127, 127).round() * s[..., None]).flatten(-2)
            sflat[to] = s
            out[name + "_scale"] = sflat.view(pages, page, h, d // 32).permute(0, 2, 1, 3).contiguous()
        flat[to] = x
        got = flat.view(pages, page, h, d).permute(0, 2, 1, 3).contiguous()
        out[name] = got if scale is None else got.view(pages, h, page, d // 32, 32)
    return out


def _exact_norm(st):
    m, k = st["case"]["m"], st["case"]["k"]
    h = st["x"].double() + st["r"].double()
    y = h / torch.sqrt((h * h).sum(-1, keepdim=True) / k + 1e-6) * st["w"].double()
    y = y.reshape(m, k // 128, 128)
    s = torch.maximum(y.abs().amax(-1), torch.tensor(1e-6, dtype=torch.float64, device="cuda")) / 127.0
    return {"residual": h, "values": torch.round(y / s[..., None]).clamp(-127, 127) * s[..., None], "scales": s}


def _exact_attn(st):
    case = st["case"]
    hq, hkv, d = HEADS[case["heads"]]
    new, kv = _lengths(case)
    if 4.0 * hq * d * sum(a * b for a, b in zip(new, kv)) > 4e12:
        return None
    page, outs, at = case["page"], [], 0
    for b, (n, total) in enumerate(zip(new, kv)):
        ids = st["table"][b, :_ceil(total, page)].long()
        heads = []
        for h in range(hkv):
            parts = []
            for cache, scale in (st["cache"][0::2], st["cache"][1::2]):
                x = cache[ids, h].double()
                if scale is not None:
                    x = (x - 128.0) * scale[ids, h].double().repeat_interleave(32, -1)
                    x = x.half().double()
                parts.append(x.reshape(-1, d)[:total])
            k, v = parts
            g = hq // hkv
            q = st["q"][at:at + n, h * g:(h + 1) * g].double().reshape(n * g, d)
            s = (q @ k.T) * st["scale"]
            row = torch.arange(n, device="cuda").repeat_interleave(g)[:, None]
            s = s.masked_fill(torch.arange(total, device="cuda")[None, :] > total - n + row, float("-inf"))
            heads.append((torch.softmax(s, -1) @ v).reshape(n, g, d))
        o = torch.cat(heads, 1)
        if st["gate"] is not None:
            o = o * torch.sigmoid(st["gate"][at:at + n].double())
        outs.append(o)
        at += n
    return torch.cat(outs)
