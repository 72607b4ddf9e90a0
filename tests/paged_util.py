"""Reference and tolerances of the paged-cache operators, in 64 bits from their formulas."""
import math

import torch

HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}     # a rounding is off by at most this, relative to the value


def attention_reference(q, keys, values, past, scale):
    """q (n, nh, hd), keys and values (L, nkv, hd) of one request whose rows stand behind `past` keys; `past` < 0 leaves rows
    that see nothing.  Returns (o, tol) in 64 bits, (n, nh, hd).

    tol, per value: the output is rounded once; p is rounded once before it meets v (below 2^-14 of its scale fp16 has a
    fixed step: 2^-25 a key); each logit is an fp32 sum of hd products in any order, so within (hd + 8) 2^-24 of the sum of
    their magnitudes, which moves p by twice that, relatively; exp is within 2^-20; sums over the keys are fp32."""
    n, nh, hd = q.shape
    L, nkv = keys.shape[0], keys.shape[1]
    step = HALF_STEP[q.dtype]
    o = torch.zeros(n, nh, hd, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(o)
    t = torch.arange(n, device=q.device)[:, None]
    seen = (torch.arange(L, device=q.device)[None] <= past + t)
    some = seen.any(dim=1)
    for h in range(nh):
        if L == 0:
            break
        k, v = keys[:, h * nkv // nh].double(), values[:, h * nkv // nh].double()
        x = q[:, h].double()
        z = (x @ k.T * scale).masked_fill(~seen, -math.inf)
        p = torch.softmax(z[some], dim=-1)
        o[some, h] = p @ v
        spread = (x.abs() @ k.abs().T * abs(scale)).masked_fill(~seen, 0).amax(dim=1)[some] * (hd + 8) * 2.0 ** -24 + 2.0 ** -20
        mass = p @ v.abs()
        tol[some, h] = (step * o[some, h].abs() + (step + 2 * spread[:, None] + 3 * L * 2.0 ** -24) * mass
                        + (L * 2.0 ** -25 * v.abs().max() if q.dtype == torch.float16 else 0))
    return o, tol


def check(got, want, tol, what=""):
    off = (got.double() - want).abs()
    worst = float((off - tol).max()) if off.numel() else 0.0
    assert bool(torch.isfinite(got).all()), f"{what}: not finite"
    assert worst <= 0, f"{what}: {float(off.max()):.3g} off, {worst:.3g} over the tolerance"


def gather(cache, table, n, n_pages=None):
    """Keys or values 0 .. n-1 of a request: (n, nkv, hd)."""
    ps, hd = cache.shape[2], cache.shape[3]
    ids = table[: -(-n // ps)].long()
    return cache[ids].transpose(1, 2).reshape(-1, cache.shape[1], hd)[:n]


def make_step(lens, nh, nkv, hd, ps, dtype, seed, device="cuda", pad=0, spare=3, fill=float("nan")):
    """A step over a paged cache: lens is [(kv_len, new)].  Pages are in random order; what no request holds is `fill`."""
    g = torch.Generator(device="cpu").manual_seed(seed)
    need = [-(-kv // ps) for kv, _ in lens]
    n_pages, width = sum(need) + spare, max([1] + need) + 1
    perm = torch.randperm(n_pages, generator=g)
    tables = torch.full((len(lens), width), -7, dtype=torch.int32)
    k_cache = torch.full((n_pages, nkv, ps, hd), fill, dtype=torch.float32)
    v_cache = torch.full((n_pages, nkv, ps, hd), fill, dtype=torch.float32)
    at = 0
    for b, (kv, _) in enumerate(lens):
        ids = perm[at:at + need[b]]
        at += need[b]
        tables[b, :need[b]] = ids.int()
        for j, page in enumerate(ids.tolist()):
            live = min(ps, kv - j * ps)
            k_cache[page, :, :live] = torch.randn(nkv, live, hd, generator=g)
            v_cache[page, :, :live] = torch.randn(nkv, live, hd, generator=g)
    new = [n for _, n in lens]
    rows = sum(new) + pad
    q = 2 * torch.randn(rows, nh * hd, generator=g)
    if pad:
        q[-pad:] = float("nan")
    cu = torch.tensor([0] + new).cumsum(0).int()
    return {"q": q.to(dtype).to(device), "k_cache": k_cache.to(dtype).to(device), "v_cache": v_cache.to(dtype).to(device),
            "tables": tables.to(device), "kv_lens": torch.tensor([kv for kv, _ in lens], dtype=torch.int32, device=device),
            "cu_rows": cu.to(device), "max_rows": max([0] + new), "rows": rows, "lens": lens, "pad": pad}


def step_reference(s, nh, scale=None):
    hd = s["k_cache"].shape[3]
    scale = hd ** -0.5 if scale is None else scale
    outs, tols, at = [], [], 0
    for b, (kv, n) in enumerate(s["lens"]):
        q = s["q"][at:at + n].reshape(n, nh, hd)
        at += n
        keys, values = (gather(s[c], s["tables"][b], kv) for c in ("k_cache", "v_cache"))
        o, t = attention_reference(q, keys, values, kv - n, scale)
        outs.append(o.reshape(n, nh * hd))
        tols.append(t.reshape(n, nh * hd))
    return torch.cat(outs), torch.cat(tols)


def plan_reference(cached, new, tables, free, n_free, ps, rows):
    """plan_pages, request by request.  Lists in, (tables, cu_rows, kv_lens, positions, slots, n_free) out."""
    tables = [list(t) for t in tables]
    width = len(tables[0]) if tables else 0
    left = max(0, min(n_free, len(free)))
    cu, kv, pos, slots, at, stopped = [0], [], [], [], 0, False
    for b, (c, n) in enumerate(zip(cached, new)):
        c, n = max(c, 0), max(n, 0)
        held, want = -(-c // ps), -(-(c + n) // ps)
        fits = c + n <= width * ps and at + n <= rows
        served = fits and (want == held or (not stopped and want - held <= left))
        if fits and want > held:
            if served:
                for j in range(held, want):
                    left -= 1
                    tables[b][j] = free[left]
            else:
                stopped = True
        kv.append(c + n if served else 0)
        for t in range(n):
            if at + t < rows:
                pos.append(c + t)
                slots.append(tables[b][(c + t) // ps] * ps + (c + t) % ps if served else -1)
        at += n
        cu.append(min(at, rows))
    pos += [0] * (rows - len(pos))
    slots += [-1] * (rows - len(slots))
    return tables, cu, kv, pos, slots, left
