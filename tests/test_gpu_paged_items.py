"""Attention where a block of the launch goes from a tile with one empty half to a short one, against 64-bit references."""
import pytest
import torch

from tests.paged_util import attention_reference, check, make_step, step_reference

pytestmark = pytest.mark.gpu
FP16, BF16 = torch.float16, torch.bfloat16


@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("lens,nh,nkv,hd", [([(1500, 1)] * 32 + [(50, 50)], 32, 8, 128),
                                            (([(2000, 1)] * 3 + [(45, 45)]) * 16, 32, 8, 128),
                                            (([(1300, 1)] * 3 + [(77, 76)]) * 12, 16, 4, 64)])
def test_new_prompts_beside_running_requests(dtype, lens, nh, nkv, hd):
    """Running requests leave half 1 of their tiles empty; a short prompt follows in the same block.  Behind every request's keys
    stand NaN."""
    from eptq_b200.kernels import paged
    s = make_step(lens, nh, nkv, hd, 16, dtype, seed=len(lens))
    want, tol = step_reference(s, nh)
    first = paged.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["tables"], s["kv_lens"], s["cu_rows"], s["max_rows"])
    check(first, want, tol)
    for _ in range(20):
        again = paged.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["tables"], s["kv_lens"], s["cu_rows"], s["max_rows"])
        assert torch.equal(again, first)


@pytest.mark.parametrize("lens,nh,nkv,hd,dtype", [([3970], 28, 4, 128, FP16), ([8002], 28, 4, 128, BF16), ([2105, 2105], 24, 8, 128, FP16),
                                                  ([990, 45] * 6, 32, 8, 128, BF16), ([990, 45] * 6, 32, 8, 64, FP16)])
def test_prompts_that_end_in_one_half(lens, nh, nkv, hd, dtype):
    """A prompt's last tile has rows in one half only, the next head group's or prompt's first tile is short."""
    from eptq_b200.kernels import paged
    rows, pad = sum(lens), 7
    g = torch.Generator(device="cuda").manual_seed(rows + nh)
    qkv = torch.randn(rows + pad, (nh + 2 * nkv) * hd, generator=g, device="cuda").to(dtype)
    qkv[rows:] = float("nan")
    q, k, v = qkv[:, :nh * hd], qkv[:, nh * hd:(nh + nkv) * hd], qkv[:, (nh + nkv) * hd:]
    cu = torch.tensor([0] + lens, device="cuda").cumsum(0).int()
    first = paged.prompt_attention(q, k, v, cu, hd)[:rows].clone()
    at = 0
    for n in lens:
        o, t = attention_reference(*(x[at:at + n].reshape(n, -1, hd) for x in (q, k, v)), 0, hd ** -0.5)
        check(first[at:at + n].reshape(n, nh, hd), o, t, f"prompt of {n} at {at}")
        at += n
    for _ in range(20):
        assert torch.equal(paged.prompt_attention(q, k, v, cu, hd)[:rows], first)
