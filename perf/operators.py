"""The paged-cache operators, measured: what serving many requests at once puts around the quantized linears.

A server that runs EPTQ layers for many requests keeps keys and values in pages.  One step of it is: pages and cache
slots for the new tokens of every request (`plan_pages`), rotary embedding and the store into the pages
(`rope_append_paged`), attention of the new rows over the pages (`paged_attention`: one row per request while tokens
are generated, many for a chunk of a prompt, both in one batch), or, for prompts that start from an empty cache,
attention straight over the packed projections (`prompt_attention`).  Head layouts are those of the architectures that
`eptq_b200.engine` names (32 heads over 32 or 8 key/value heads of 128, 64 over 8, or a rank's share of them) and of the
smaller decoders with heads of 64.

`run` computes an operator in plain torch operations, or, where `own` is true, makes the call that a user makes.
"""
import random

import torch

own = False

DEV = "cuda"
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


# ---- cases -----------------------------------------------------------------------------------------------------
# Lengths are whole numbers from lo to hi, spread evenly over their logarithm by `mix` alone, so that a case says all.
def _case(name, op, **kw):
    c = {"name": name, "op": op, "dtype": "fp16", "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 16, "batch": 1,
         "cached_lo": 0, "cached_hi": 0, "new_lo": 1, "new_hi": 1, "chunks": 0, "chunk": 0, "pad": 0, "mix": 1}
    c.update(kw)
    return c


def listed():
    return [
        # one token for each of 64 running requests: what a server plans between two decode steps
        _case("plan_decode_64", "plan", batch=64, cached_lo=1, cached_hi=4096),
        # a step full of new prompts, some rows of padding, and too few free pages for the last requests
        _case("plan_prompts_512", "plan", batch=512, cached_lo=0, cached_hi=4096, new_lo=0, new_hi=700, pad=77, short=True),
        # decode step of 8 requests, every head with its own keys (7B architecture)
        _case("append_8_rows", "append", kv_heads=32, batch=8, cached_lo=20, cached_hi=2000),
        # a prompt chunk far into long contexts, grouped heads, bf16, padded to a fixed number of rows
        _case("append_chunk_bf16", "append", dtype="bf16", batch=16, page=64, cached_lo=30000, cached_hi=120000, new_lo=100, new_hi=900, pad=31),
        # one chat: the smallest decode call
        _case("decode_1", "attend", cached_lo=907, cached_hi=907),
        # heads of 64, each with its own keys, bf16
        _case("decode_32_h64_bf16", "attend", dtype="bf16", heads=12, kv_heads=12, head_dim=64, page=32, batch=32, cached_lo=1, cached_hi=2000, pad=3),
        # a full server: 64 requests from a few tokens to 16 thousand
        _case("decode_64_long", "attend", batch=64, cached_lo=100, cached_hi=16000),
        # a chunk of one long document over what is cached of it (70B architecture)
        _case("chunk_long", "attend", heads=64, batch=1, page=64, cached_lo=24001, cached_hi=24001, new_lo=509, new_hi=509),
        # chunks of two prompts beside 32 running requests
        _case("mixed_34", "attend", dtype="bf16", batch=34, cached_lo=50, cached_hi=3500, chunks=2, chunk=411),
        # the smallest prompt
        _case("prompt_77_h64", "prompt", heads=12, kv_heads=12, head_dim=64, new_lo=77, new_hi=77),
        # prompts of many lengths packed into one call, padded
        _case("prompt_packed", "prompt", batch=12, new_lo=1, new_hi=2500, pad=9),
        # one long prompt, every head with its own keys (7B architecture), bf16
        _case("prompt_8191_bf16", "prompt", dtype="bf16", kv_heads=32, new_lo=8191, new_hi=8191),
    ]


def _between(rng, lo, hi):
    """A whole number from lo (>= 1) to hi, spread evenly over its logarithm."""
    return min(hi, max(lo, int(lo * ((hi + 1) / lo) ** rng.random())))


def draw(rng):
    op = rng.choice(["plan", "append", "attend", "attend", "attend", "prompt", "prompt"])
    heads, kv, hd = rng.choice([(32, 32, 128), (32, 8, 128), (64, 8, 128), (8, 1, 128), (28, 4, 128), (12, 12, 64), (16, 2, 64), (15, 5, 64)])
    c = _case("", op, dtype=rng.choice(["fp16", "bf16"]), heads=heads, kv_heads=kv, head_dim=hd, page=rng.choice([16, 32, 64, 128]),
              pad=rng.choice([0, 0, 0, rng.randint(1, 60)]), mix=rng.randrange(1 << 30))
    if op == "plan":
        b = _between(rng, 1, 512)
        c.update(batch=b, cached_lo=0, cached_hi=_between(rng, 1, 4096), new_lo=0, new_hi=_between(rng, 1, min(700, 1 + 60000 // b)), short=rng.random() < 0.3)
    elif op == "append":
        rows = _between(rng, 1, 4000)
        b = _between(rng, 1, min(rows, 64))
        c.update(batch=b, cached_lo=0, cached_hi=_between(rng, 1, 100000), new_lo=1, new_hi=max(1, rows // b))
    elif op == "attend":
        kind = rng.choice(["decode", "few", "chunk", "mixed"])
        if kind == "decode":
            b = _between(rng, 1, 64)
            c.update(batch=b, cached_lo=0, cached_hi=_between(rng, 1, min(16000, 200000 // b)))
        elif kind == "few":
            b = _between(rng, 1, 24)
            c.update(batch=b, cached_lo=0, cached_hi=_between(rng, 1, min(8000, 60000 // b)), new_lo=1, new_hi=rng.randint(1, 16))
        elif kind == "chunk":
            b = _between(rng, 1, 4)
            c.update(batch=b, cached_lo=0, cached_hi=_between(rng, 1, 24000 // b), new_lo=1, new_hi=_between(rng, 16, 509))
        else:
            b = _between(rng, 3, 32)
            c.update(batch=b, cached_lo=0, cached_hi=_between(rng, 50, 3500), chunks=rng.randint(1, 2), chunk=_between(rng, 20, 411))
    else:
        b = _between(rng, 1, 16)
        c.update(batch=b, new_lo=rng.choice([0, 1]), new_hi=_between(rng, 2, 6000 // b))
    del c["name"]
    return c


def _lengths(c):
    """(cached, new) lengths of every request."""
    rng = random.Random(c["mix"])

    def some(lo, hi):
        return 0 if lo == 0 and rng.random() < 0.1 else _between(rng, max(lo, 1), max(hi, 1)) if hi else 0

    cached = [some(c["cached_lo"], c["cached_hi"]) for _ in range(c["batch"])]
    new = [some(c["new_lo"], c["new_hi"]) for _ in range(c["batch"])]
    for i in range(c["chunks"]):
        new[(i * 7 + 3) % c["batch"]] = c["chunk"] - i
    if not any(new):
        new[0] = 1
    return cached, new


def _ceil(a, b):
    return -(-a // b)


# ---- inputs ----------------------------------------------------------------------------------------------------
def _normal(gen, dtype, *shape):
    return torch.randn(*shape, generator=gen, device=DEV, dtype=torch.float32 if shape[0] < 4096 else dtype).to(dtype)


def _whole(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=DEV)


def prepare(case, seed):
    c = case
    gen = torch.Generator(device=DEV).manual_seed(seed)
    cached, new = _lengths(c)
    dt, nh, nkv, hd, ps = TYPES[c["dtype"]], c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    s = {"op": c["op"], "page": ps, "head_dim": hd, "rows": sum(new) + c["pad"], "max_new": max(new)}
    rows = s["rows"]
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    s["cu_rows"] = _whole(starts)
    if c["op"] == "prompt":
        s["q"] = _normal(gen, dt, rows, nh * hd) * 2
        s["k"] = _normal(gen, dt, rows, nkv * hd)
        s["v"] = _normal(gen, dt, rows, nkv * hd)
        s["out"] = torch.zeros(rows, nh * hd, dtype=dt, device=DEV)
        return s
    # pages in no order, a few more than are needed; every request's table names the pages of what it has cached
    held = [_ceil(n, ps) for n in cached]
    want = [_ceil(a + b, ps) for a, b in zip(cached, new)]
    used = held if c["op"] == "plan" else want
    n_pages, width = sum(want) + 5, max(want) + 1
    pages = torch.randperm(n_pages, generator=gen, device=DEV).to(torch.int32)
    ends = torch.tensor(used, device=DEV).cumsum(0)
    first, col = ends - torch.tensor(used, device=DEV), torch.arange(width, device=DEV)[None]
    inside = col < torch.tensor(used, device=DEV)[:, None]
    s["tables"] = torch.where(inside, pages[(first[:, None] + col).clamp(max=n_pages - 1)], -1).to(torch.int32)
    s["cached"], s["new"] = _whole(cached), _whole(new)
    if c["op"] == "plan":
        s["free"] = pages[sum(used):].contiguous()
        s["n_free"] = _whole([max(0, (sum(want) - sum(held)) * 9 // 10) if c.get("short") else s["free"].numel()])
        return s
    s["kv_lens"] = _whole([a + b for a, b in zip(cached, new)])
    s["q"] = _normal(gen, dt, rows, nh * hd) * 2
    if c["op"] == "append":
        s["k"], s["v"] = _normal(gen, dt, rows, nkv * hd), _normal(gen, dt, rows, nkv * hd)
        s["inv_freq"] = 1.0 / (10000.0 ** (torch.arange(0, hd, 2, device=DEV).float() / hd))
        s["k_cache"] = torch.zeros(n_pages, nkv, ps, hd, dtype=dt, device=DEV)
        s["v_cache"] = torch.zeros_like(s["k_cache"])
        r = torch.arange(rows, device=DEV)
        b = torch.searchsorted(s["cu_rows"][1:], r, right=True)
        live, b = b < c["batch"], b.clamp(max=c["batch"] - 1)
        s["positions"] = torch.where(live, s["cached"][b] + r - s["cu_rows"][b], 0)
        page = s["tables"][b, s["positions"] // ps].long()
        s["slots"] = torch.where(live, page * ps + s["positions"] % ps, -1)
        return s
    s["k_cache"] = _normal(gen, dt, n_pages, nkv, ps, hd)
    s["v_cache"] = _normal(gen, dt, n_pages, nkv, ps, hd)
    s["out"] = torch.zeros(rows, nh * hd, dtype=dt, device=DEV)
    return s


# ---- plain forms -----------------------------------------------------------------------------------------------
def _plan(s):
    ps, rows, tables = s["page"], s["rows"], s["tables"]
    cached, new = s["cached"].long(), s["new"].long()
    B, width = tables.shape
    total, n_free = cached + new, s["n_free"].long()
    held, want = (cached + ps - 1) // ps, (total + ps - 1) // ps
    ends = new.cumsum(0)
    fits = (total <= width * ps) & (ends <= rows)
    need = torch.where(fits, want - held, 0)
    upto = need.cumsum(0)
    served = fits & ((need == 0) | (upto <= n_free))
    cu_rows = torch.cat((ends.new_zeros(1), ends)).clamp(max=rows)
    col = torch.arange(width, device=DEV)[None]
    gets = served[:, None] & (col >= held[:, None]) & (col < want[:, None])
    nth = (upto - need - held)[:, None] + col
    tables = torch.where(gets, s["free"][(n_free - 1 - nth).clamp(0, s["free"].numel() - 1)], tables)
    r = torch.arange(rows, device=DEV)
    b = torch.searchsorted(cu_rows[1:], r, right=True)
    live, b = b < B, b.clamp(max=B - 1)
    pos = torch.where(live, cached[b] + r - cu_rows[b], 0)
    page = tables[b, (pos // ps).clamp(max=width - 1)].long()
    slots = torch.where(live & served[b], page * ps + pos % ps, -1)
    left = n_free - torch.where(served & (need > 0), upto, 0).amax()
    return {"tables": tables, "cu_rows": cu_rows.int(), "kv_lens": torch.where(served, total, 0).int(), "positions": pos, "slots": slots, "n_free": left.int()}


def _turned(x, cos, sin):
    a, b = x.float().chunk(2, dim=-1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1).to(x.dtype)


def _append(s):
    hd, ps, slots, kc, vc = s["head_dim"], s["page"], s["slots"], s["k_cache"], s["v_cache"]
    rows = slots.shape[0]
    angle = s["positions"].double()[:, None, None] * s["inv_freq"].double()        # far positions: 32 bits lose the angle
    cos, sin = angle.cos().float(), angle.sin().float()
    q = _turned(s["q"].reshape(rows, -1, hd), cos, sin).reshape(rows, -1)
    k = _turned(s["k"].reshape(rows, -1, hd), cos, sin)
    v = s["v"].reshape(rows, -1, hd)
    src = torch.where(slots >= 0, torch.arange(rows, device=DEV), 0)               # rows without a slot: row 0 once more
    page, at = slots[src] // ps, slots[src] % ps
    kc[page, :, at] = k[src]
    vc[page, :, at] = v[src]
    return {"q": q, "k_cache": kc, "v_cache": vc}


def _softmax_product(q, k, v, seen, scale):
    """q (B, G, R, T, hd), k and v (B, G, L, hd), seen (B, T, L) -> (B, G, R, T, hd)."""
    B, G, R, T, hd = q.shape
    p = (q.reshape(B, G, R * T, hd) * scale) @ k.transpose(-1, -2)
    p = p.reshape(B, G, R, T, -1).masked_fill_(~seen[:, None, None], float("-inf"))
    p = p.sub_(p.amax(dim=-1, keepdim=True).clamp_(min=-1e30)).exp_()
    total = p.sum(dim=-1, keepdim=True)
    return (p.reshape(B, G, R * T, -1) @ v).reshape(B, G, R, T, hd) / torch.where(total > 0, total, 1)


def _rows_to_batch(s, x, width):
    """Packed rows (rows, n * hd) -> (B, width, n, hd), and for every packed row its request and place."""
    cu, rows = s["cu_rows"].long(), x.shape[0]
    at = cu[:-1, None] + torch.arange(width, device=DEV)
    r = torch.arange(rows, device=DEV)
    b = torch.searchsorted(cu[1:], r, right=True)
    live, b = b < cu.numel() - 1, b.clamp(max=cu.numel() - 2)
    return x[at.clamp(max=rows - 1)].reshape(cu.numel() - 1, width, -1, s["head_dim"]), live, b, torch.where(live, r - cu[b], 0)


def _attend(s):
    hd, T, dt = s["head_dim"], s["max_new"], s["q"].dtype
    q, live, b, t = _rows_to_batch(s, s["q"], T)
    B, nkv = q.shape[0], s["k_cache"].shape[1]
    k, v = (c[s["tables"].clamp(min=0).long()].transpose(1, 2).reshape(B, nkv, -1, hd).float() for c in (s["k_cache"], s["v_cache"]))
    q = q.float().reshape(B, T, nkv, -1, hd).permute(0, 2, 3, 1, 4)
    kv, cu = s["kv_lens"].long(), s["cu_rows"].long()
    last = (kv - (cu[1:] - cu[:-1]))[:, None] + torch.arange(T, device=DEV)        # the last key that a row sees
    key = torch.arange(k.shape[2], device=DEV)
    o = _softmax_product(q, k, v, key <= torch.minimum(last, kv[:, None] - 1)[..., None], hd ** -0.5)
    o = o.permute(0, 3, 1, 2, 4).reshape(B, T, -1)
    return torch.where(live[:, None], o[b, t], 0).to(dt)


def _prompt(s):
    hd, T, dt = s["head_dim"], s["max_new"], s["q"].dtype
    q, live, b, t = _rows_to_batch(s, s["q"], T)
    k, v = (_rows_to_batch(s, x, T)[0].float().transpose(1, 2) for x in (s["k"], s["v"]))
    B, nkv = k.shape[:2]
    q = q.float().reshape(B, T, nkv, -1, hd).permute(0, 2, 3, 1, 4)
    at = torch.arange(T, device=DEV)
    o = _softmax_product(q, k, v, (at[None] <= at[:, None])[None].expand(B, T, T), hd ** -0.5)
    o = o.permute(0, 3, 1, 2, 4).reshape(B, T, -1)
    return torch.where(live[:, None], o[b, t], 0).to(dt)


# ---- one pass --------------------------------------------------------------------------------------------------
def run(state):
    s = state
    if own:
        from eptq_b200.kernels import paged

        if s["op"] == "plan":
            p = paged.plan_pages(s["cached"], s["new"], s["tables"], s["free"], s["n_free"], s["page"], s["rows"])
            return {"tables": s["tables"], "cu_rows": p.cu_rows, "kv_lens": p.kv_lens, "positions": p.positions, "slots": p.slots, "n_free": p.n_free}
        if s["op"] == "append":
            q = paged.rope_append_paged(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["positions"], s["slots"], s["inv_freq"])
            return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
        if s["op"] == "attend":
            return paged.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["tables"], s["kv_lens"], s["cu_rows"], s["max_new"], out=s["out"])
        return paged.prompt_attention(s["q"], s["k"], s["v"], s["cu_rows"], s["head_dim"], out=s["out"])
    return {"plan": _plan, "append": _append, "attend": _attend, "prompt": _prompt}[s["op"]](s)


# ---- what a pass cannot do without -----------------------------------------------------------------------------
def work(case):
    c = case
    cached, new = _lengths(c)
    rows, B, nh, nkv, hd, ps = sum(new) + c["pad"], c["batch"], c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    live = sum(new)
    if c["op"] == "plan":                    # two lengths in, two out; a page id out and in for each page; position and slot of each row
        pages = sum(_ceil(a + b, ps) - _ceil(a, ps) for a, b in zip(cached, new))
        return {"bytes": 16 * B + 8 * pages + 16 * rows, "flops": 4 * rows + 8 * B}
    if c["op"] == "append":
        return {"bytes": 2 * hd * (2 * rows * nh + 4 * live * nkv) + 16 * rows, "flops": 3 * hd * rows * (nh + nkv)}
    if c["op"] == "prompt":
        cached = [0] * B
    seen = sum(n * a + n * (n + 1) // 2 for a, n in zip(cached, new))
    keys = sum(a + n for a, n in zip(cached, new) if n)
    return {"bytes": 2 * hd * (2 * live * nh + 2 * keys * nkv), "flops": 4 * hd * nh * seen}


# ---- in 64 bits, request by request ----------------------------------------------------------------------------
def exact(case, seed):
    c = case
    s = prepare(case, seed)
    cached, new = _lengths(c)
    nh, nkv, hd, ps = c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    if c["op"] == "plan":
        return None                          # whole numbers
    if c["op"] == "append":
        rows = s["rows"]
        turn = torch.polar(torch.ones(rows, hd // 2, dtype=torch.float64, device=DEV), s["positions"].double()[:, None] * s["inv_freq"].double()[None])

        def rotated(x):
            x = x.double().reshape(rows, -1, 2, hd // 2)
            z = torch.complex(x[:, :, 0], x[:, :, 1]) * turn[:, None]
            return torch.stack((z.real, z.imag), dim=2).reshape(rows, -1, hd)

        kc = torch.zeros(s["k_cache"].shape, dtype=torch.float64, device=DEV)
        vc = torch.zeros_like(kc)
        live = s["slots"] >= 0
        at = s["slots"][live]
        kc[at // ps, :, at % ps] = rotated(s["k"])[live]
        vc[at // ps, :, at % ps] = s["v"].double().reshape(rows, nkv, hd)[live]
        return {"q": rotated(s["q"]).reshape(rows, -1), "k_cache": kc, "v_cache": vc}
    out = torch.zeros(s["rows"], nh, hd, dtype=torch.float64, device=DEV)
    start = 0
    for i, n in enumerate(new):
        if n:
            q = s["q"][start:start + n].double().reshape(n, nh, hd)
            if c["op"] == "prompt":
                past = 0
                k, v = (s[x][start:start + n].double().reshape(n, nkv, hd).transpose(0, 1) for x in ("k", "v"))
            else:
                past = cached[i]
                ids = s["tables"][i, :_ceil(past + n, ps)].long()
                k, v = (s[x][ids].double().transpose(0, 1).reshape(nkv, -1, hd)[:, :past + n] for x in ("k_cache", "v_cache"))
            hidden = torch.ones(n, past + n, dtype=torch.bool, device=DEV).triu(past + 1)
            for h in range(nh):
                z = (q[:, h] @ k[h * nkv // nh].T) / hd ** 0.5
                out[start:start + n, h] = torch.softmax(z.masked_fill(hidden, float("-inf")), dim=-1) @ v[h * nkv // nh]
        start += n
    return out.reshape(s["rows"], nh * hd)
