"""Paged-cache operators (plan, rotary append, attention over pages, packed prompts) against 64-bit references."""
import pytest
import torch

from tests.paged_util import attention_reference, check, gather, make_step, plan_reference, step_reference

pytestmark = pytest.mark.gpu
FP16, BF16 = torch.float16, torch.bfloat16


def _attend(s, **kw):
    from eptq_b200.kernels import paged
    kw.setdefault("max_rows", s["max_rows"])
    return paged.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["tables"], s["kv_lens"], s["cu_rows"], **kw)


# ---- plan ----------------------------------------------------------------------------------------------------
def _plan_case(B, ps, seed, short=False, most=90, rows_cut=0, width_cut=0):
    g = torch.Generator().manual_seed(seed)
    cached = torch.randint(0, 3 * most, (B,), generator=g).tolist()
    new = [0 if i % 5 == 3 else int(torch.randint(0, most, (1,), generator=g)) for i in range(B)]
    held = [-(-c // ps) for c in cached]
    want = [-(-(c + n) // ps) for c, n in zip(cached, new)]
    width = max(1, max(want) - width_cut)
    perm = torch.randperm(sum(want) + 9, generator=g).tolist()
    tables, at = [], 0
    for h in held:
        tables.append((perm[at:at + h] + [-1] * width)[:width])
        at += h
    free = perm[at:]
    n_free = (sum(want) - sum(held)) // 2 if short else len(free)
    return cached, new, tables, free, n_free, sum(new) + 7 - rows_cut


@pytest.mark.parametrize("B,ps,kw", [(1, 16, {}), (3, 64, {}), (64, 16, {}), (200, 32, {"short": True}), (1024, 16, {}),
                                     (1025, 128, {}), (2500, 16, {"short": True, "most": 40}), (40, 16, {"rows_cut": 300}),
                                     (40, 16, {"width_cut": 6}), (33, 16, {"most": 3000})])
def test_plan_pages(B, ps, kw):
    from eptq_b200.kernels import paged
    cached, new, tables, free, n_free, rows = _plan_case(B, ps, seed=B + ps, **kw)
    want = plan_reference(cached, new, tables, free, n_free, ps, rows)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")            # noqa: E731
    wide = torch.full((B, len(tables[0]) + 3), -5, dtype=torch.int32, device="cuda")
    wide[:, :-3] = i32(tables)
    t, count = wide[:, :-3], i32([n_free])                                       # rows of the table farther apart than wide
    for _ in range(2):                                                           # again over the same tables: the same plan
        p = paged.plan_pages(i32(cached), i32(new), t, i32(free), count, ps, rows)
        assert t.tolist() == want[0] and bool((wide[:, -3:] == -5).all())
        assert p.cu_rows.tolist() == want[1] and p.kv_lens.tolist() == want[2]
        assert p.positions.tolist() == want[3] and p.slots.tolist() == want[4]
        assert p.n_free.tolist() == [want[5]] and count.tolist() == [n_free]


def test_plan_pages_edges():
    """No requests, no rows, lengths below zero, a free count beyond the list."""
    from eptq_b200.kernels import paged
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")            # noqa: E731
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    p = paged.plan_pages(none, none, none.reshape(0, 4), i32([3]), i32([1]), 16, 5)
    assert p.cu_rows.tolist() == [0] and p.slots.tolist() == [-1] * 5 and p.positions.tolist() == [0] * 5 and p.n_free.tolist() == [1]
    t = i32([[-1, -1], [-1, -1], [-1, -1]])
    p = paged.plan_pages(i32([-4, 0, 0]), i32([3, -2, 17]), t, i32([9, 8]), i32([50]), 16, 20)
    assert p.cu_rows.tolist() == [0, 3, 3, 20] and p.kv_lens.tolist() == [3, 0, 0] and p.n_free.tolist() == [1]
    assert t.tolist() == [[8, -1], [-1, -1], [-1, -1]] and p.slots.tolist() == [128, 129, 130] + [-1] * 17
    p = paged.plan_pages(i32([0]), i32([0]), i32([[-1]]), none, i32([0]), 16, 0)
    assert p.kv_lens.tolist() == [0] and p.slots.numel() == 0
    p = paged.plan_pages(i32([2 ** 31 - 1, 0]), i32([2 ** 31 - 1, 1]), i32([[0], [0]]), i32([4]), i32([1]), 16, 8)
    assert p.kv_lens.tolist() == [0, 0] and p.cu_rows.tolist() == [0, 8, 8]


# ---- rotary embedding + store ----------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("rows,nh,nkv,hd,ps,far", [(1, 32, 32, 128, 16, 0), (37, 8, 2, 64, 32, 5000), (5, 28, 4, 128, 64, 131000),
                                                   (3, 1, 1, 16, 16, 2 ** 31), (2, 5, 5, 256, 128, 77), (300, 12, 12, 64, 16, 90)])
def test_rope_append_paged(dtype, rows, nh, nkv, hd, ps, far):
    from eptq_b200.kernels import paged
    g = torch.Generator(device="cuda").manual_seed(rows + hd)
    qkv = torch.randn(rows, (nh + 2 * nkv) * hd, generator=g, device="cuda").to(dtype)      # one projection's output
    q, k, v = qkv[:, :nh * hd], qkv[:, nh * hd:(nh + nkv) * hd], qkv[:, (nh + nkv) * hd:]
    n_pages = -(-rows // ps) + 2
    kc = torch.full((n_pages, nkv, ps, hd), 7.0, device="cuda", dtype=dtype)
    vc = torch.full_like(kc, 7.0)
    slots = torch.randperm(n_pages * ps, generator=g, device="cuda")[:rows]
    if rows > 2:
        slots[1], slots[-1] = -1, n_pages * ps                                              # neither is in the cache
    pos = far + torch.arange(rows, device="cuda") * 3
    inv_freq = 1.0 / (10000.0 ** (torch.arange(0, hd, 2, device="cuda").float() / hd))
    scaling = 1.25
    before = qkv.clone()
    out = paged.rope_append_paged(q, k, v, kc, vc, pos, slots, inv_freq, scaling)
    assert torch.equal(qkv, before)
    ang = pos.double()[:, None] * inv_freq.double()
    cos, sin = ang.cos()[:, None] * scaling, ang.sin()[:, None] * scaling
    # one rounding of the output; cos and sin within 2^-20 (their argument is at most pi, to 2^-22), products and the sum in fp32
    step = {FP16: 2.0 ** -11, BF16: 2.0 ** -8}[dtype]

    def rotated(x, n):
        a, b = x.double().reshape(rows, n, hd).chunk(2, dim=-1)
        want = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
        size = (a.abs() + b.abs()) * scaling
        tol = step * want.abs() + torch.cat((size, size), dim=-1) * 2.0 ** -19 + 2.0 ** -25      # (2^-25: fp16 below its normal range)
        return want, tol

    want, tol = rotated(q, nh)
    check(out.reshape(rows, nh, hd), want, tol, "q")
    live = (slots >= 0) & (slots < n_pages * ps)
    at = slots[live]
    want, tol = rotated(k, nkv)
    check(kc[at // ps, :, at % ps], want[live], tol[live], "k")
    assert torch.equal(vc[at // ps, :, at % ps], v.reshape(rows, nkv, hd)[live])
    rest = torch.ones(n_pages * ps, dtype=torch.bool, device="cuda")
    rest[at] = False
    for c in (kc, vc):
        assert bool((c.transpose(1, 2).reshape(n_pages * ps, -1)[rest] == 7).all())
    q2 = q.contiguous()
    assert paged.rope_append_paged(q2, k, v, kc, vc, pos, slots, inv_freq, scaling, out=q2) is q2 and torch.equal(q2, out)


# ---- attention over pages ----------------------------------------------------------------------------------------
SHAPES = [(32, 8, 128), (4, 4, 128), (28, 4, 128), (12, 12, 64), (16, 1, 64), (15, 5, 64), (64, 8, 128)]
LENS = {
    "tokens": [(1, 1), (17, 1), (16, 1), (128, 1), (129, 1), (700, 1), (2049, 1)],
    "empty": [(0, 0), (5, 0), (0, 3), (33, 1), (2, 5), (64, 64), (0, 0)],                 # no rows, no keys, more rows than keys
    "few": [(200, 5), (31, 7), (1000, 16), (16, 2)],
    "chunks": [(300, 129), (128, 128), (517, 257), (1, 1), (260, 3)],
    "mixed": [(900, 1), (140, 140), (33, 1), (1200, 77), (450, 1)],
}


@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("lens", sorted(LENS))
@pytest.mark.parametrize("nh,nkv,hd", SHAPES)
def test_paged_attention(dtype, lens, nh, nkv, hd):
    """Every kernel the call may choose, by the row bound that it is told; what lies behind a request's keys is NaN."""
    ps = [16, 32, 64, 128][(nh + len(lens)) % 4]
    s = make_step(LENS[lens], nh, nkv, hd, ps, dtype, seed=nh + len(lens), pad=3)
    want, tol = step_reference(s, nh)
    for told in (1, s["max_rows"], 100000):
        out = torch.full_like(s["q"], 9.0)
        assert _attend(s, max_rows=told, out=out) is out
        check(out[:-3], want, tol, f"told {told}")
        assert bool((out[-3:] == 9).all())                                                 # rows behind the last request


@pytest.mark.parametrize("told", [1, 100000])
@pytest.mark.parametrize("dtype", [FP16, BF16])
def test_paged_attention_long(dtype, told):
    """One long request beside short ones: work cut over many blocks and joined, the same bits every time."""
    s = make_step([(20011, 1), (3, 1), (9000, 21), (1, 1)], 8, 2, 128, 16, dtype, seed=3)
    want, tol = step_reference(s, 8)
    first = _attend(s, max_rows=told)
    check(first, want, tol)
    for _ in range(5):
        assert torch.equal(_attend(s, max_rows=told), first)


@pytest.mark.parametrize("told", [1, 100000])
@pytest.mark.parametrize("batch,hd", [(300, 64), (1100, 128)])
def test_paged_attention_many_requests(batch, hd, told):
    lens = [((i * 37) % 190, 1 if i % 11 else 0) for i in range(batch)]
    s = make_step(lens, 4, 2, hd, 32, FP16, seed=batch)
    want, tol = step_reference(s, 4)
    check(_attend(s, max_rows=told), want, tol)


@pytest.mark.parametrize("told", [1, 100000])
def test_paged_attention_pages_outside_the_cache(told):
    """Keys on a page id outside the cache do not count; a request with no other pages gives zeros."""
    nh, nkv, hd, ps = 8, 2, 128, 16
    s = make_step([(200, 3), (40, 1), (16, 16)], nh, nkv, hd, ps, FP16, seed=11)
    n_pages = s["k_cache"].shape[0]
    s["tables"][0, 2], s["tables"][0, 5], s["tables"][0, 12] = -1, n_pages, 2 ** 31 - 1
    s["tables"][1, :] = -(2 ** 31)
    out = _attend(s, max_rows=told)
    keep = torch.ones(200, dtype=torch.bool)
    for j in (2, 5, 12):
        keep[j * ps:(j + 1) * ps] = False
    ids = s["tables"][0].clone()
    ids[(ids < 0) | (ids >= n_pages)] = 0
    keys, values = (gather(s[c], ids, 200)[keep.cuda()] for c in ("k_cache", "v_cache"))
    for t in range(3):
        seen = int(keep[:198 + t].sum())                                    # keys 0 .. 197 + t, without the lost pages
        o, tol = attention_reference(s["q"][t:t + 1].reshape(1, nh, hd), keys[:seen], values[:seen], seen - 1, hd ** -0.5)
        check(out[t:t + 1].reshape(1, nh, hd), o, tol)
    assert bool((out[3] == 0).all())
    o, tol = attention_reference(s["q"][4:].reshape(16, nh, hd), gather(s["k_cache"], s["tables"][2], 16), gather(s["v_cache"], s["tables"][2], 16), 0, hd ** -0.5)
    check(out[4:].reshape(16, nh, hd), o, tol)


@pytest.mark.parametrize("told", [1, 100000])
@pytest.mark.parametrize("dtype", [FP16, BF16])
def test_paged_attention_far_logits(dtype, told):
    """Logits from -30000 to 30000, rising and falling along the keys: the running maximum moves all the time, or never."""
    nh, nkv, hd, ps = 4, 2, 64, 16
    s = make_step([(600, 2), (600, 2), (333, 130)], nh, nkv, hd, ps, dtype, seed=5)
    for b, sign in ((0, 1.0), (1, -1.0)):
        for j in range(-(-600 // ps)):
            page = int(s["tables"][b, j])
            s["k_cache"][page, :, :, 0] = sign * torch.linspace(-170, 170, 600 + ps, device="cuda")[j * ps:(j + 1) * ps].to(dtype)
    s["q"][:, 0::hd] = 200.0
    want, tol = step_reference(s, nh, 1.0)
    check(_attend(s, max_rows=told, scale=1.0), want, tol)


@pytest.mark.parametrize("told", [1, 100000])
def test_paged_attention_scale(told):
    """A scale of zero weighs all keys alike; a negative one turns the order round."""
    s = make_step([(77, 4), (300, 1)], 8, 8, 128, 16, FP16, seed=6)
    for scale in (0.0, -0.1):
        want, tol = step_reference(s, 8, scale)
        check(_attend(s, max_rows=told, scale=scale), want, tol)


@pytest.mark.parametrize("told", [1, 100000])
def test_paged_attention_large_offsets(told):
    """Pages beyond 2^32 bytes of a cache, and pages farther apart than they are long."""
    nh, nkv, hd, ps = 8, 4, 128, 64
    s = make_step([(500, 3), (90, 1)], nh, nkv, hd, ps, FP16, seed=8)
    n = s["k_cache"].shape[0]
    per_page = 2 * nkv * ps * hd
    n_pages = (2 ** 32) // per_page + n                                   # over 2^32 values with both caches in one tensor
    both = torch.empty(n_pages, 2, nkv, ps, hd, dtype=FP16, device="cuda")
    both[-n:, 0], both[-n:, 1] = s["k_cache"], s["v_cache"]
    want, tol = step_reference(s, nh)
    s["k_cache"], s["v_cache"] = both[:, 0], both[:, 1]
    s["tables"] = torch.where(s["tables"] >= 0, s["tables"] + (n_pages - n), s["tables"])
    check(_attend(s, max_rows=told), want, tol)


def test_paged_attention_strided_q():
    s = make_step([(130, 5), (64, 1)], 8, 2, 64, 16, BF16, seed=9)
    want, tol = step_reference(s, 8)
    wide = torch.full((s["rows"], 8 * 64 + 256), float("nan"), dtype=BF16, device="cuda")
    wide[:, 128:128 + 512] = s["q"]
    s["q"] = wide[:, 128:128 + 512]
    for told in (1, 100000):
        check(_attend(s, max_rows=told), want, tol)


@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("nh,nkv,hd,lens,told", [(8, 2, 128, [(300, 40)], 100000), (4, 4, 64, [(513, 300), (70, 2)], 100000), (8, 2, 128, [(90, 4), (33, 2)], 4),
                                                 (6, 2, 64, [(64, 5)], 5), (7, 1, 128, [(1500, 140)], 100000)])
def test_paged_attention_values_not_finite(dtype, nh, nkv, hd, lens, told):
    """A value that is not finite reaches the rows that see it, in its column, and no other row: not the request's earlier ones."""
    s = make_step(lens, nh, nkv, hd, 16, dtype, seed=12)
    want, tol = step_reference(s, nh)
    want, tol = want.reshape(-1, nh, hd).clone(), tol.reshape(-1, nh, hd)
    at = 0
    for b, (kv, n) in enumerate(lens):
        for key, col, head, value in ((kv - n + 1, 3, 0, float("inf")), (kv - 1, 5, nkv - 1, float("nan")), (kv - (n + 1) // 2, hd - 1, 0, float("-inf"))):
            page = int(s["tables"][b, key // 16])
            s["v_cache"][page, head, key % 16, col] = value
            rows = slice(at + key - (kv - n), at + n)
            want[rows, head * (nh // nkv):(head + 1) * (nh // nkv), col] += value
        at += n
    out = _attend(s, max_rows=told).double().reshape(-1, nh, hd)
    finite = torch.isfinite(want)
    assert torch.equal(torch.isfinite(out), finite)
    assert bool((((out - want).abs() <= tol) | ~finite).all())
    assert torch.equal(torch.isnan(out), torch.isnan(want)) and bool((out[~finite & ~torch.isnan(want)] == want[~finite & ~torch.isnan(want)]).all())


# ---- packed prompts --------------------------------------------------------------------------------------------
def _prompt_reference(q, k, v, lens, nh, nkv, hd, scale=None):
    outs, tols, at = [], [], 0
    for n in lens:
        o, t = attention_reference(q[at:at + n].reshape(n, nh, hd), k[at:at + n].reshape(n, nkv, hd), v[at:at + n].reshape(n, nkv, hd), 0,
                                   hd ** -0.5 if scale is None else scale)
        outs.append(o.reshape(n, nh * hd))
        tols.append(t.reshape(n, nh * hd))
        at += n
    return torch.cat(outs), torch.cat(tols)


@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("nh,nkv,hd", SHAPES)
@pytest.mark.parametrize("lens", [[1], [77], [128, 0, 129, 1, 127], [255, 256, 257], [0, 0, 900], [3] * 40, [2050, 5]])
def test_prompt_attention(dtype, nh, nkv, hd, lens):
    """q, k, v as columns of one projection; rows behind the last prompt are NaN and leave no trace."""
    from eptq_b200.kernels import paged
    rows, pad = sum(lens), 5
    g = torch.Generator(device="cuda").manual_seed(rows + nh)
    qkv = torch.randn(rows + pad, (nh + 2 * nkv) * hd, generator=g, device="cuda").to(dtype)
    qkv[rows:] = float("nan")
    q, k, v = qkv[:, :nh * hd], qkv[:, nh * hd:(nh + nkv) * hd], qkv[:, (nh + nkv) * hd:]
    cu = torch.tensor([0] + lens, device="cuda").cumsum(0).int()
    out = torch.full((rows + pad, nh * hd), 9.0, dtype=dtype, device="cuda")
    assert paged.prompt_attention(q, k, v, cu, hd, out=out) is out
    want, tol = _prompt_reference(q, k, v, lens, nh, nkv, hd)
    check(out[:rows], want, tol)
    assert bool((out[rows:] == 9).all())
    assert torch.equal(paged.prompt_attention(q.contiguous(), k.contiguous(), v.contiguous(), cu, hd)[:rows], out[:rows])


def test_prompt_attention_values_not_finite():
    """A prompt that overflowed leaves its neighbours in the call alone."""
    from eptq_b200.kernels import paged
    nh, nkv, hd, lens = 8, 2, 128, [40, 100, 30]
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = (torch.randn(170, n * hd, generator=g, device="cuda").half() for n in (nh, nkv, nkv))
    k[40:140], v[40:140] = float("inf"), float("nan")
    cu = torch.tensor([0, 40, 140, 170], dtype=torch.int32, device="cuda")
    out = paged.prompt_attention(q, k, v, cu, hd)
    for lo, hi in ((0, 40), (140, 170)):
        want, tol = _prompt_reference(q[lo:hi], k[lo:hi], v[lo:hi], [hi - lo], nh, nkv, hd)
        check(out[lo:hi], want, tol)


# ---- together ------------------------------------------------------------------------------------------------
def _serve(dtype, nh, nkv, hd, ps, prompts, new_tokens, chunk, seed=0):
    """Prompts fed in chunks and then token by token, requests joining one after the other; compares every row of every
    step with causal attention over the request's whole history in 64 bits."""
    from eptq_b200.kernels import paged
    B = len(prompts)
    total = [p + new_tokens for p in prompts]
    g = torch.Generator(device="cuda").manual_seed(seed)
    qs, ks, vs = ([torch.randn(n, h * hd, generator=g, device="cuda").to(dtype) for n in total] for h in (nh, nkv, nkv))
    width = max(-(-n // ps) for n in total)
    n_pages = sum(-(-n // ps) for n in total) + 2
    kc = torch.full((n_pages, nkv, ps, hd), float("nan"), dtype=dtype, device="cuda")
    vc = kc.clone()
    tables = torch.full((B, width), -1, dtype=torch.int32, device="cuda")
    free = torch.randperm(n_pages, generator=g, device="cuda").int()
    n_free = torch.tensor([n_pages], dtype=torch.int32, device="cuda")
    inv_freq = 1.0 / (10000.0 ** (torch.arange(0, hd, 2, device="cuda").float() / hd))
    done = [0] * B
    rot_q, outs = [[] for _ in range(B)], [[] for _ in range(B)]
    step = 0
    while any(d < n for d, n in zip(done, total)):
        new = [0 if b > step else min(chunk, prompts[b] - done[b]) if done[b] < prompts[b] else min(1, total[b] - done[b]) for b in range(B)]
        rows = sum(new) + 2
        x = [torch.cat([t[b][done[b]:done[b] + new[b]] for b in range(B)] + [torch.full_like(t[0][:1], float("nan")).expand(2, -1)]) for t in (qs, ks, vs)]
        plan = paged.plan_pages(torch.tensor(done, dtype=torch.int32, device="cuda"), torch.tensor(new, dtype=torch.int32, device="cuda"),
                                tables, free, n_free, ps, rows)
        n_free.copy_(plan.n_free)
        q = paged.rope_append_paged(*x, kc, vc, plan.positions, plan.slots, inv_freq)
        out = paged.paged_attention(q, kc, vc, tables, plan.kv_lens, plan.cu_rows, max(new))
        at = 0
        for b in range(B):
            rot_q[b].append(q[at:at + new[b]])
            outs[b].append(out[at:at + new[b]])
            at += new[b]
            done[b] += new[b]
        step += 1
    assert int(n_free) == 2
    for b in range(B):
        n = total[b]
        keys, values = gather(kc, tables[b], n), gather(vc, tables[b], n)
        assert torch.equal(values.reshape(n, -1), vs[b])
        want, tol = attention_reference(torch.cat(rot_q[b]).reshape(n, nh, hd), keys, values, 0, hd ** -0.5)
        check(torch.cat(outs[b]).reshape(n, nh, hd), want, tol, f"request {b}")
        cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
        whole = paged.prompt_attention(torch.cat(rot_q[b]), keys.reshape(n, -1).contiguous(), vs[b], cu, hd)
        check(whole.reshape(n, nh, hd), want, tol, f"request {b} as one prompt")


@pytest.mark.parametrize("dtype,nh,nkv,hd,ps", [(FP16, 8, 2, 128, 16), (BF16, 4, 4, 64, 32), (FP16, 7, 1, 64, 64)])
def test_serving_steps(dtype, nh, nkv, hd, ps):
    _serve(dtype, nh, nkv, hd, ps, prompts=[100, 7, 333], new_tokens=9, chunk=64)


def test_captured_step_follows_the_lengths():
    """One captured step (plan, append, attention), replayed for other lengths; two graphs of it on two streams at once."""
    from eptq_b200.kernels import paged
    nh, nkv, hd, ps, B, rows = 8, 2, 128, 16, 5, 40

    def build(seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        st = {"cached": torch.zeros(B, dtype=torch.int32, device="cuda"), "new": torch.zeros(B, dtype=torch.int32, device="cuda"),
              "tables": torch.full((B, 200), -1, dtype=torch.int32, device="cuda"), "free": torch.randperm(900, generator=g, device="cuda").int(),
              "n_free": torch.tensor([900], dtype=torch.int32, device="cuda")}
        st["q"], st["k"], st["v"] = (torch.randn(rows, h * hd, generator=g, device="cuda").half() for h in (nh, nkv, nkv))
        st["kc"], st["vc"] = (torch.randn(900, nkv, ps, hd, generator=g, device="cuda").half() for _ in range(2))
        st["inv_freq"] = 1.0 / (10000.0 ** (torch.arange(0, hd, 2, device="cuda").float() / hd))
        st["all"] = torch.randperm(900, generator=g, device="cuda").int().reshape(B, 180)

        def step():
            p = paged.plan_pages(st["cached"], st["new"], st["tables"], st["free"], st["n_free"], ps, rows)
            q = paged.rope_append_paged(st["q"], st["k"], st["v"], st["kc"], st["vc"], p.positions, p.slots, st["inv_freq"])
            st["out"] = paged.paged_attention(q, st["kc"], st["vc"], st["tables"], p.kv_lens, p.cu_rows, rows, out=st.setdefault("buf", torch.zeros_like(q)))
            st["plan"], st["qr"] = p, q
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step()
        return st, graph, stream

    sides = [build(1), build(2)]
    for lens in ([(300, 1), (0, 20), (2500, 1), (17, 3), (0, 0)], [(0, 1), (1, 1), (2, 1), (3, 1), (4, 1)], [(2800, 7), (2800, 7), (2800, 7), (5, 7), (800, 7)]):
        for st, _, _ in sides:
            st["cached"].copy_(torch.tensor([c for c, _ in lens], dtype=torch.int32))
            st["new"].copy_(torch.tensor([n for _, n in lens], dtype=torch.int32))
            for b, (c, _) in enumerate(lens):
                st["tables"][b, :180] = st["all"][b]
        torch.cuda.synchronize()
        for _ in range(3):
            for _, graph, stream in sides:
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        for st, _, _ in sides:
            at = 0
            for b, (c, n) in enumerate(lens):
                keys, values = (gather(st[x], st["tables"][b], c + n) for x in ("kc", "vc"))
                want, tol = attention_reference(st["qr"][at:at + n].reshape(n, nh, hd), keys, values, c, hd ** -0.5)
                check(st["out"][at:at + n].reshape(n, nh, hd), want, tol)
                at += n


def test_streams_and_threads():
    """Calls on streams of their own, at once, from two threads."""
    import threading
    steps = [make_step([(3000, 1), (50, 1), (4000, 3)], 8, 2, 128, 16, FP16, seed=20 + i) for i in range(2)]
    wants = [step_reference(s, 8) for s in steps]
    torch.cuda.synchronize()
    outs = [None, None]

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for j in range(30):
                outs[i] = _attend(steps[i], max_rows=1 if j % 2 else 1000)
        stream.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for o, (want, tol) in zip(outs, wants):
        check(o, want, tol)


def test_nothing_to_do():
    from eptq_b200.kernels import paged
    e = lambda *shape, dtype=FP16: torch.empty(*shape, dtype=dtype, device="cuda")     # noqa: E731
    i = lambda *shape: torch.zeros(*shape, dtype=torch.int32, device="cuda")            # noqa: E731
    cache = e(4, 2, 16, 64)
    assert paged.paged_attention(e(0, 256), cache, cache, i(3, 5), i(3), i(4), 1).shape == (0, 256)
    out = torch.full((2, 256), 5.0, dtype=FP16, device="cuda")
    paged.paged_attention(torch.zeros_like(out), cache, cache, i(0, 5), i(0), i(1), 1, out=out)
    assert bool((out == 5).all())
    for told in (2, 1000):                                                 # a cache without pages
        out.fill_(5)
        paged.paged_attention(torch.zeros_like(out), cache[:0], cache[:0], i(1, 0), i(1) + 9, torch.tensor([0, 2], dtype=torch.int32, device="cuda"), told, out=out)
        assert bool((out == 0).all())
    assert paged.prompt_attention(e(0, 256), e(0, 128), e(0, 128), i(1), 64).shape == (0, 256)
    assert paged.rope_append_paged(e(0, 256), e(0, 128), e(0, 128), cache, cache, e(0, dtype=torch.int64), e(0, dtype=torch.int64), e(32, dtype=torch.float32)).shape == (0, 256)
