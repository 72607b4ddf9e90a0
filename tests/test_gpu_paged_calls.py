"""What a call of the paged-cache operators leaves alone, clears, refuses and reports."""
import pytest
import torch

from tests.paged_util import check, make_step, step_reference

pytestmark = pytest.mark.gpu
FP16, BF16 = torch.float16, torch.bfloat16


def _attend(s, **kw):
    from eptq_b200.kernels import paged
    kw.setdefault("max_rows", s["max_rows"])
    return paged.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["tables"], s["kv_lens"], s["cu_rows"], **kw)


def _soil(like):
    """The allocator's next block of this size is full of NaN."""
    x = torch.full_like(like, float("nan"))
    torch.cuda.synchronize()
    del x


# ---- rows of no request ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("told", [1, 100000])
@pytest.mark.parametrize("dtype,hd,pad", [(FP16, 128, 1), (BF16, 64, 700), (FP16, 64, 37)])
def test_rows_of_no_request_are_zeros_without_out(dtype, hd, pad, told):
    nh = 6
    s = make_step([(90, 4), (33, 2), (0, 3)], nh, 2, hd, 16, dtype, seed=pad, pad=pad)
    want, tol = step_reference(s, nh)
    _soil(s["q"])
    out = _attend(s, max_rows=told)
    check(out[:-pad], want, tol)
    assert bool((out[-pad:] == 0).all())
    # five rows ahead of the first request as well
    s["q"], s["cu_rows"] = torch.cat((s["q"][-1:].expand(5, -1), s["q"])), s["cu_rows"] + 5
    _soil(s["q"])
    out = _attend(s, max_rows=told)
    check(out[5:-pad], want, tol)
    assert bool((out[:5] == 0).all()) and bool((out[-pad:] == 0).all())
    kept = _attend(s, max_rows=told, out=torch.full_like(s["q"], 9.0))
    assert bool((kept[:5] == 9).all()) and bool((kept[-pad:] == 9).all()) and torch.equal(kept[5:-pad], out[5:-pad])


def test_rows_of_no_prompt_are_zeros_without_out():
    from eptq_b200.kernels import paged
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = (torch.randn(300, n * 128, generator=g, device="cuda").half() for n in (4, 2, 2))
    q[200:] = k[200:] = v[200:] = float("nan")
    cu = torch.tensor([0, 60, 200], dtype=torch.int32, device="cuda")
    _soil(q)
    out = paged.prompt_attention(q, k, v, cu, 128)
    assert bool(torch.isfinite(out[:200]).all()) and bool((out[200:] == 0).all())
    _soil(q)
    assert bool((paged.prompt_attention(q, k, v, cu[:1], 128) == 0).all())                    # no prompt at all
    kept = torch.full_like(q, 9.0)
    assert bool((paged.prompt_attention(q, k, v, cu[:1], 128, out=kept) == 9).all())
