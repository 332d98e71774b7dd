"""The operators of a packed serving step: what is measured, and their plain forms.

A step of a server that packs its requests one behind the other goes: `page_plan` turns request lengths into block tables, slots
and positions; `PagedKvCache.append` rounds the new keys and values to four bits and stores them at their slots (`read` gives
them back); `prompt_attention` is the causal attention of whole packed prompts; `PagedKvCache.decode_attention` is the
attention of one new token per request over the four-bit pages.

`run` computes a case with elementary torch operations, or — where `own` is true — through the public calls of atlas_b200.
"""
import math

import torch

own = False
DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # block tables and slots: a decode step of a small server (one new token per request) …
        dict(name="plan_decode_48", op="plan", batch=48, cached_max=6000, new_max=1, page=16, spare=40),
        # … a step that takes in hundreds of prompts at once …
        dict(name="plan_prompts_700", op="plan", batch=700, cached_max=900, new_max=400, page=32, spare=1000),
        # four-bit cache: the new rows of one decode step of a 32-request batch, as the f32 activations that a product leaves
        dict(name="cache_step_32_f32", op="cache", tokens=32, n_kv=8, hd=128, group=32, page=16, dtype="f32", fused=False),
        # a long prompt's rows, bf16, taken out of the middle of fused query|key|value rows; all heads hold keys of their own
        dict(name="cache_prompt_8191_bf16", op="cache", tokens=8191, n_kv=32, hd=128, group=64, page=64, dtype="bf16", fused=True),
        # decode attention: a single chat, where latency counts
        dict(name="decode_1x700", op="decode", batch=1, len_min=700, len_max=700, n_heads=32, n_kv=8, hd=128, group=32, page=16, window=0),
        # a ragged batch, no heads shared, sliding window of 4096
        dict(name="decode_12_window_mha", op="decode", batch=12, len_min=1, len_max=9001, n_heads=32, n_kv=32, hd=128, group=64, page=64, window=4096),
        # one very long document
        dict(name="decode_1x131071", op="decode", batch=1, len_min=131071, len_max=131071, n_heads=32, n_kv=8, hd=128, group=32, page=16, window=0),
        # a full server: 64 requests of up to 8 k
        dict(name="decode_64x8k", op="decode", batch=64, len_min=2000, len_max=8192, n_heads=32, n_kv=8, hd=128, group=32, page=32, window=0),
        # prompt attention: one short question
        dict(name="prompt_1x37", op="prompt", batch=1, len_min=37, len_max=37, past_max=0, n_heads=32, n_kv=8, hd=128, window=0, dtype="bf16", fused=True),
        # a pack of prompts of very different lengths, some behind a prefix that is cached already
        dict(name="prompt_24_ragged", op="prompt", batch=24, len_min=1, len_max=1200, past_max=700, n_heads=32, n_kv=8, hd=128, window=0, dtype="bf16", fused=False),
        # narrow heads in f16 under a sliding window
        dict(name="prompt_3_window_f16", op="prompt", batch=3, len_min=2500, len_max=4100, past_max=0, n_heads=16, n_kv=4, hd=64, window=1024, dtype="f16", fused=True),
        # one long prompt, every head with keys of its own
        dict(name="prompt_1x8192_mha", op="prompt", batch=1, len_min=8192, len_max=8192, past_max=0, n_heads=32, n_kv=32, hd=128, window=0, dtype="bf16", fused=True),
    ]


def _between(rng, lo, hi):
    """A whole number spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["plan", "cache", "decode", "decode", "prompt", "prompt"])
    page = rng.choice([16, 32, 48, 64, 128])
    hd, group = rng.choice([(128, 32), (128, 64), (64, 32), (64, 64)])
    n_kv = rng.choice([1, 2, 4, 8, 16])
    n_heads = n_kv * rng.choice([1, 2, 3, 4, 6, 8, 12])
    if op == "plan":
        return dict(op=op, batch=_between(rng, 1, 1000), cached_max=_between(rng, 1, 20000), new_max=_between(rng, 1, 300), page=page,
                    spare=_between(rng, 1, 2000))
    if op == "cache":
        return dict(op=op, tokens=min(_between(rng, 1, 20000), 200000 // n_kv), n_kv=n_kv, hd=hd, group=group, page=page,
                    dtype=rng.choice(["f32", "bf16", "f16"]), fused=rng.choice([True, False]))
    if op == "decode":
        batch = _between(rng, 1, 200)
        most = max(1, min(100000, 250000 // batch, 2000000 // (batch * n_kv)))
        hi = _between(rng, 1, most)
        return dict(op=op, batch=batch, len_min=_between(rng, 1, hi), len_max=hi, n_heads=n_heads, n_kv=n_kv, hd=hd, group=group, page=page,
                    window=rng.choice([0, 0, _between(rng, 1, 5000)]))
    n_heads, n_kv = rng.choice([(32, 8), (32, 32), (16, 4), (8, 1), (12, 4), (6, 2), (5, 5)])
    batch = _between(rng, 1, 60)
    hi = _between(rng, 1, max(1, int(math.sqrt(1.0e9 / (batch * n_heads)))))
    return dict(op=op, batch=batch, len_min=_between(rng, 1, hi), len_max=hi, past_max=rng.choice([0, 0, _between(rng, 1, hi)]), n_heads=n_heads,
                n_kv=n_kv, hd=rng.choice([64, 128]), window=rng.choice([0, 0, _between(rng, 1, 2000)]), dtype=rng.choice(["bf16", "f16"]),
                fused=rng.choice([True, False]))


def _lengths(case, n, lo, hi):
    """Request lengths belong to the case (a server knows them): the same for every seed."""
    g = torch.Generator().manual_seed(1000003 * n + 1009 * lo + hi)
    return torch.randint(lo, hi + 1, (n,), generator=g)


def work(case):
    if case["op"] == "plan":
        b = case["batch"]
        cached, new = _lengths(case, b, 0, case["cached_max"]), _lengths(case, b, 1, case["new_max"])
        pages = -(-(cached + new) // case["page"])
        had = -(-cached // case["page"])
        n = int(new.sum())
        # lengths in, lengths and row starts out, slots and positions out, the pages taken read and written
        return {"bytes": 4.0 * (4 * b + 1 + 2 * n + 2 * int((pages - had).sum())), "flops": 0.0}
    if case["op"] == "cache":
        e = case["tokens"] * case["n_kv"] * case["hd"] * 2
        size = {"f32": 4, "bf16": 2, "f16": 2}[case["dtype"]]
        held = e / 2 + e / case["group"] * 2
        return {"bytes": e * size + 2 * held + e * 4 + 8.0 * case["tokens"], "flops": 0.0}
    if case["op"] == "decode":
        rows = _lengths(case, case["batch"], case["len_min"], case["len_max"])
        if case["window"]:
            rows = rows.clamp(max=case["window"])
        r = int(rows.sum())
        e = case["hd"]
        return {"bytes": r * 2.0 * case["n_kv"] * (e / 2 + e / case["group"] * 2) + 8.0 * case["batch"] * case["n_heads"] * e,
                "flops": 4.0 * r * case["n_heads"] * e}
    lq, lp = _prompt_lengths(case)
    pairs = 0
    for q, p in zip(lq.tolist(), lp.tolist()):
        w = case["window"] or (q + p)
        full = max(0, min(q, q + p - w))              # rows that see a whole window
        rest = q - full                               # rows that see all behind them
        pairs += full * w + rest * p + rest * (rest + 1) // 2
    t, k = int(lq.sum()), int((lq + lp).sum())
    return {"bytes": 2.0 * case["hd"] * (2 * t * case["n_heads"] + 2 * k * case["n_kv"]), "flops": 4.0 * pairs * case["n_heads"] * case["hd"]}


def _prompt_lengths(case):
    lq = _lengths(case, case["batch"], case["len_min"], case["len_max"])
    lp = _lengths(case, case["batch"], 0, case["past_max"]) if case["past_max"] else torch.zeros(case["batch"], dtype=torch.long)
    return lq, lp


def _rows(gen, shape, hd):
    """Keys or values as a model makes them: normal, a few channels far larger than the rest."""
    x = torch.randn(*shape, device=DEV, generator=gen)
    x[..., 3] *= 6.0
    x[..., hd // 2 + 5] *= -4.0
    return x


def _fused(parts, yes):
    """Rows [tokens, heads, hd]: each tensor by itself, or all as column ranges of one buffer, as one product leaves them."""
    if not yes:
        return [p.contiguous() for p in parts]
    t, hd = parts[0].shape[0], parts[0].shape[2]
    buf = torch.cat([p.reshape(t, -1) for p in parts], dim=1)
    out, at = [], 0
    for p in parts:
        w = p.shape[1] * hd
        out.append(buf[:, at:at + w].unflatten(1, (p.shape[1], hd)))
        at += w
    return out


def _ints(x):
    return x.to(torch.int32).to(DEV)


def _table(lens, page, n_pages, gen, width):
    """Block table of requests whose pages lie anywhere in the pool."""
    need = -(-lens // page)
    order = torch.randperm(n_pages, generator=gen)
    table = torch.full((len(lens), width), -1, dtype=torch.long)
    at = 0
    for i, m in enumerate(need.tolist()):
        table[i, :m] = order[at:at + m]
        at += m
    return table, order[at:]


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    s = {"case": dict(case)}
    page = case.get("page")
    if case["op"] == "plan":
        b = case["batch"]
        cached, new = _lengths(case, b, 0, case["cached_max"]), _lengths(case, b, 1, case["new_max"])
        width = int((-(-(case["cached_max"] + case["new_max"]) // page)))
        had = int((-(-cached // page)).sum())
        taken = int((-(-(cached + new) // page)).sum()) - had
        n_pages = had + taken + case["spare"]
        table, free = _table(cached, page, n_pages, host, width)
        n = int(new.sum())
        s.update(cached=_ints(cached), new=_ints(new), table=_ints(table), free=_ints(free), n_pages=n_pages, tokens=n,
                 cu=torch.empty(b + 1, dtype=torch.int32, device=DEV), lens=torch.empty(b, dtype=torch.int32, device=DEV),
                 slots=torch.empty(n, dtype=torch.int32, device=DEV), pos=torch.empty(n, dtype=torch.int32, device=DEV),
                 status=torch.empty(3, dtype=torch.int32, device=DEV))
        if own:
            import atlas_b200
            s["ab"], s["ctx"] = atlas_b200, atlas_b200.Context.default()
        return s
    if case["op"] == "prompt":
        lq, lp = _prompt_lengths(case)
        hd, nh, nk = case["hd"], case["n_heads"], case["n_kv"]
        t, tk = int(lq.sum()), int((lq + lp).sum())
        dt = TYPES[case["dtype"]]
        q = torch.randn(t, nh, hd, device=DEV, generator=gen).to(dt)
        k = _rows(gen, (tk, nk, hd), hd).to(dt)
        v = _rows(gen, (tk, nk, hd), hd).to(dt)
        if t == tk:
            q, k, v = _fused([q, k, v], case["fused"])
        else:
            (q,), (k, v) = _fused([q], False), _fused([k, v], case["fused"])
        zero = torch.zeros(1, dtype=torch.long)
        s.update(q=q, k=k, v=v, cu_q=_ints(torch.cat([zero, lq.cumsum(0)])), cu_k=_ints(torch.cat([zero, (lq + lp).cumsum(0)])),
                 max_q=int(lq.max()), max_k=int((lq + lp).max()), out=torch.empty(t, nh, hd, dtype=dt, device=DEV))
        if own:
            import atlas_b200
            s["ab"], s["ctx"] = atlas_b200, atlas_b200.Context.default()
        return s
    hd, nk, group = case["hd"], case["n_kv"], case["group"]
    if case["op"] == "cache":
        n = case["tokens"]
        n_pages = -(-n // page) + 7
        k, v = _rows(gen, (n, nk, hd), hd), _rows(gen, (n, nk, hd), hd)
        k, v = _fused([k.to(TYPES[case["dtype"]]), v.to(TYPES[case["dtype"]])], case["fused"])
        slots = _ints(torch.randperm(n_pages, generator=host)[:, None] * page + torch.arange(page)[None, :]).flatten()[:n].contiguous()
        s.update(k=k, v=v, slots=slots, out_k=torch.empty(n, nk, hd, device=DEV), out_v=torch.empty(n, nk, hd, device=DEV))
    else:
        lens = _lengths(case, case["batch"], case["len_min"], case["len_max"])
        n_pages = int((-(-lens // page)).sum()) + 5
        table, _ = _table(lens, page, n_pages, host, -(-int(lens.max()) // page))
        b, nh = case["batch"], case["n_heads"]
        s.update(q=torch.randn(b, nh, hd, device=DEV, generator=gen), table=_ints(table.clamp(min=0)), lens=_ints(lens), max_len=int(lens.max()),
                 out=torch.empty(b, nh, hd, device=DEV))
    # the pool in four bits: pages of nibbles with a bf16 scale per group
    if not own:
        s["held"] = torch.zeros(2, n_pages * page, nk, hd // 2, dtype=torch.uint8, device=DEV)
        s["scales"] = torch.ones(2, n_pages * page, nk, hd // group, dtype=torch.bfloat16, device=DEV)
    else:
        import atlas_b200
        s["ab"], s["ctx"] = atlas_b200, atlas_b200.Context.default()
        s["pool"] = atlas_b200.PagedKvCache(n_pages, page, nk, hd, group=group, ctx=s["ctx"])
    if case["op"] == "decode":                       # the cache that earlier steps have filled
        at = 0
        while at < n_pages * page:
            m = min(65536, n_pages * page - at)
            k, v = _rows(gen, (m, nk, hd), hd).bfloat16(), _rows(gen, (m, nk, hd), hd).bfloat16()
            slots = torch.arange(at, at + m, dtype=torch.int32, device=DEV)
            if own:
                torch.cuda.synchronize()
                s["pool"].append(k, v, slots)
                s["ctx"].sync()
            else:
                _store(s, k, v, slots.long())
            at += m
    return s


# ── plain forms ──────────────────────────────────────────────────────────────────
def _quantise(x, group):
    """Groups of `group` numbers → whole numbers −7..7 and one bf16 scale each: scale = bf16(max|x| / 7), 1 where that is below the
    smallest normal number (a group of zeros); the number is x times the scale's f32 reciprocal, rounded half away from zero."""
    g = x.float().unflatten(-1, (-1, group))
    top = g.abs().amax(-1)
    scale = (top / 7.0).bfloat16()
    scale = torch.where(scale < 2.0 ** -126, torch.ones_like(scale), scale)
    y = (g * (1.0 / scale.float())[..., None]).double()
    n = (torch.sign(y) * torch.floor(y.abs() + 0.5)).clamp(-7, 7)
    return n.to(torch.int8).flatten(-2), scale


def _store(s, k, v, slots):
    for i, x in enumerate((k, v)):
        n, scale = _quantise(x, s["case"]["group"])
        u = (n + 8).to(torch.uint8)
        s["held"][i, slots] = (u[..., 0::2] << 4) | u[..., 1::2]
        s["scales"][i, slots] = scale


def _fetch(s, i, slots):
    b = s["held"][i, slots]
    n = torch.stack([b >> 4, b & 15], dim=-1).flatten(-2).float() - 8.0
    return (n.unflatten(-1, (-1, s["case"]["group"])) * s["scales"][i, slots].float()[..., None]).flatten(-2)


def _plan_plain(s):
    page, n = s["case"]["page"], s["tokens"]
    cached, new, free = s["cached"].long(), s["new"].long(), s["free"].long()
    had, need = (cached + page - 1) // page, (cached + new + page - 1) // page
    cu = torch.cat([new.new_zeros(1), new.cumsum(0)])
    first = (need - had).cumsum(0) - (need - had)                  # place in the free list of a request's first new page
    col = torch.arange(s["table"].shape[1], device=DEV)[None, :]
    fresh = (col >= had[:, None]) & (col < need[:, None])
    table = torch.where(fresh, free[(first[:, None] + col - had[:, None]).clamp(0, len(free) - 1)], s["table"].long())
    token = torch.arange(n, device=DEV)
    seq = torch.searchsorted(cu[1:], token, right=True)
    pos = cached[seq] + token - cu[seq]
    slots = table[seq, pos // page] * page + pos % page
    taken = (need - had).sum()
    status = torch.stack([taken, torch.zeros_like(taken), torch.zeros_like(taken)])
    return [x.to(torch.int32) for x in (table, cu, cached + new, slots, pos, status)]


def _decode_plain(s):
    c = s["case"]
    b, nh, nk, hd = c["batch"], c["n_heads"], c["n_kv"], c["hd"]
    t = torch.arange(s["max_len"], device=DEV)
    lens = s["lens"].long()[:, None]
    slots = s["table"].long()[:, t // c["page"]] * c["page"] + t % c["page"]
    seen = (t < lens) & ((lens - 1 - t < c["window"]) if c["window"] else True)
    k, v = _fetch(s, 0, slots), _fetch(s, 1, slots)                # [b, t, n_kv, hd]
    q = s["q"].view(b, nk, nh // nk, hd)
    a = torch.matmul(q, k.permute(0, 2, 3, 1)) / math.sqrt(hd)     # [b, n_kv, heads of the group, t]
    a = a.masked_fill(~seen[:, None, None, :], -math.inf)
    p = torch.exp(a - a.amax(-1, keepdim=True))
    return (torch.matmul(p, v.permute(0, 2, 1, 3)) / p.sum(-1, keepdim=True)).reshape(b, nh, hd)


def _prompt_plain(s):
    c = s["case"]
    nh, nk, hd = c["n_heads"], c["n_kv"], c["hd"]
    cu_q, cu_k = s["cu_q"].long(), s["cu_k"].long()
    i, j = torch.arange(s["max_q"], device=DEV), torch.arange(s["max_k"], device=DEV)
    lq, lk = (cu_q[1:] - cu_q[:-1])[:, None], (cu_k[1:] - cu_k[:-1])[:, None]
    rq = (cu_q[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)
    rk = (cu_k[:-1, None] + j).clamp(max=s["k"].shape[0] - 1)
    at = (i + lk - lq)[:, :, None] - j                             # how far key j lies behind query i
    seen = (at >= 0) & (j < lk)[:, None, :]
    if c["window"]:
        seen &= at < c["window"]
    q = s["q"][rq].float().unflatten(2, (nk, nh // nk)).permute(0, 2, 3, 1, 4).flatten(2, 3)    # [b, n_kv, heads·max_q, hd]
    k = s["k"][rk].float().permute(0, 2, 3, 1)
    v = s["v"][rk].float().permute(0, 2, 1, 3)
    a = torch.matmul(q, k).mul_(1.0 / math.sqrt(hd)).unflatten(2, (nh // nk, -1))
    a.masked_fill_(~seen[:, None, None], -1e30)
    a.sub_(a.amax(-1, keepdim=True)).exp_()
    z = a.sum(-1, keepdim=True)
    o = torch.matmul(a.flatten(2, 3), v).unflatten(2, (nh // nk, -1)).div_(z)                   # [b, n_kv, heads, max_q, hd]
    o = o.permute(0, 3, 1, 2, 4).flatten(2, 3)                                                  # [b, max_q, heads, hd]
    return o[i < lq].to(s["q"].dtype)


def run(s):
    c = s["case"]
    if c["op"] == "plan":
        if own:
            s["ab"].page_plan(s["cached"], s["new"], s["free"], s["table"], s["cu"], s["lens"], s["slots"], s["pos"], s["status"],
                              page_size=c["page"], n_pages=s["n_pages"], ctx=s["ctx"])
            out = [s["table"], s["cu"], s["lens"], s["slots"], s["pos"], s["status"]]
        else:
            out = _plan_plain(s)
        return dict(zip(("table", "cu", "lens", "slots", "pos", "status"), out))
    if c["op"] == "cache":
        if own:
            s["pool"].append(s["k"], s["v"], s["slots"])
            s["pool"].read(s["slots"], s["out_k"], s["out_v"])
            return {"k": s["out_k"], "v": s["out_v"]}
        slots = s["slots"].long()
        _store(s, s["k"], s["v"], slots)
        return {"k": _fetch(s, 0, slots), "v": _fetch(s, 1, slots)}
    if c["op"] == "decode":
        if own:
            s["pool"].decode_attention(s["q"], s["out"], s["table"], s["lens"], 1.0 / math.sqrt(c["hd"]), c["window"])
            return s["out"]
        return _decode_plain(s)
    if own:
        s["ab"].prompt_attention(s["q"], s["k"], s["v"], s["out"], s["cu_q"], s["cu_k"], scale=1.0 / math.sqrt(c["hd"]),
                                 window_size=c["window"], ctx=s["ctx"])
        return s["out"]
    return _prompt_plain(s)


# ── the definitions in 64 bits, request by request ───────────────────────────────
def _held_values(x, group):
    """What the four-bit format holds for x: nearest of the fifteen multiples of each group's scale; the scale itself is a bf16 number
    and the product with its reciprocal an f32 number by the format's definition."""
    t, h, hd = x.shape
    g = x.to(torch.float32).reshape(t, h, hd // group, group)
    s = torch.div(g.abs().max(dim=3, keepdim=True).values, 7.0).to(torch.bfloat16).to(torch.float32)
    s[s < 2.0 ** -126] = 1.0
    y = torch.mul(g, torch.reciprocal(s)).to(torch.float64)
    m = torch.where(y >= 0, torch.floor(y + 0.5), torch.ceil(y - 0.5))
    return (m.clamp(min=-7.0, max=7.0) * s.to(torch.float64)).reshape(t, h, hd)


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if case["op"] == "plan":
        page = case["page"]
        table, free = s["table"].tolist(), s["free"].tolist()
        cu, lens, slots, pos, at = [0], [], [], [], 0
        for i, (c, m) in enumerate(zip(s["cached"].tolist(), s["new"].tolist())):
            for j in range(-(-c // page), -(-(c + m) // page)):
                table[i][j] = free[at]
                at += 1
            for p in range(c, c + m):
                slots.append(table[i][p // page] * page + p % page)
                pos.append(p)
            cu.append(cu[-1] + m)
            lens.append(c + m)
        got = dict(table=table, cu=cu, lens=lens, slots=slots, pos=pos, status=[at, 0, 0])
        return {k: torch.tensor(v, dtype=torch.int32) for k, v in got.items()}
    if case["op"] == "cache":
        return {"k": _held_values(s["k"], case["group"]), "v": _held_values(s["v"], case["group"])}
    nh, nk, hd, w = case["n_heads"], case["n_kv"], case["hd"], case["window"]
    if case["op"] == "decode":
        page, out = case["page"], torch.empty(case["batch"], nh, hd, dtype=torch.float64, device=DEV)
        for b, n in enumerate(s["lens"].tolist()):
            lo = max(0, n - w) if w else 0
            t = torch.arange(lo, n, device=DEV)
            slots = s["table"][b].long()[torch.div(t, page, rounding_mode="floor")] * page + torch.remainder(t, page)
            kv = []
            for i in (0, 1):
                raw = s["held"][i][slots].to(torch.int16)
                n16 = torch.empty(*raw.shape[:-1], hd, dtype=torch.float64, device=DEV)
                n16[..., 0::2], n16[..., 1::2] = torch.div(raw, 16, rounding_mode="floor").double() - 8, torch.remainder(raw, 16).double() - 8
                kv.append(n16 * s["scales"][i][slots].double().repeat_interleave(case["group"], dim=-1))
            for h in range(nh):
                kh = h // (nh // nk)
                p = torch.softmax((kv[0][:, kh] @ s["q"][b, h].double()) / math.sqrt(hd), dim=0)
                out[b, h] = p @ kv[1][:, kh]
        return out
    cq, ck = s["cu_q"].tolist(), s["cu_k"].tolist()
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEV)
    for b in range(case["batch"]):
        lq, lk = cq[b + 1] - cq[b], ck[b + 1] - ck[b]
        i = torch.arange(lk - lq, lk, device=DEV)[:, None]
        j = torch.arange(lk, device=DEV)[None, :]
        hidden = j > i
        if w:
            hidden = hidden | (j <= i - w)
        for h in range(nh):
            q, k, v = (x[r0:r1, z].double() for x, r0, r1, z in ((s["q"], cq[b], cq[b + 1], h), (s["k"], ck[b], ck[b + 1], h // (nh // nk)),
                                                                (s["v"], ck[b], ck[b + 1], h // (nh // nk))))
            p = (q @ k.T / math.sqrt(hd)).masked_fill(hidden, -math.inf)
            out[cq[b]:cq[b + 1], h] = torch.softmax(p, dim=1) @ v
    return out
