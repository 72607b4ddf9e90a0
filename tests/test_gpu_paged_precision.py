"""Attention weights of the kernel for few rows: kept in more bits than the inputs have."""
import math

import pytest
import torch

from tests.paged_util import HALF_STEP, check, gather, make_step

pytestmark = pytest.mark.gpu
FP16, BF16 = torch.float16, torch.bfloat16


@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("nh,nkv,hd", [(8, 2, 128), (4, 4, 64), (16, 1, 64), (28, 4, 128)])
@pytest.mark.parametrize("lens", [[(3, 1), (2, 1), (40, 1), (333, 1)] * 6, [(5, 2), (70, 2), (19, 1)] * 5])
def test_weights_of_few_rows(dtype, nh, nkv, hd, lens):
    _weights_of_few_rows(dtype, nh, nkv, hd, lens, 1)


@pytest.mark.parametrize("nh,nkv,hd,n", [(8, 2, 128, 4), (16, 1, 64, 2), (8, 8, 64, 32), (15, 5, 64, 10), (8, 8, 128, 16)])
def test_most_rows_that_count_as_few(nh, nkv, hd, n):
    """As many rows of a key/value head as the documentation names: a tile of 16, or two with heads of 64."""
    _weights_of_few_rows(FP16, nh, nkv, hd, [(n + 3, n), (90, 1), (400, 2)] * 2, n)


def _weights_of_few_rows(dtype, nh, nkv, hd, lens, max_rows):
    """The weight meets its value as two 16-bit values: the first cut off behind its last bit, so the second is below 2 steps of it and
    rounded by half a step of its own: 2 * 2^-11 * 2^-11 of the weight in fp16, 2 * 2^-8 * 2^-8 in bf16.  fp16 has a fixed step of
    2^-24 below its normal range: half a step of the first value and one of the second (which is not let become zero), of weights
    whose largest is 2^7 at least, so below 2^-30 a key.  What is left is the output's rounding, and what scores and sums in
    fp32 are off by: small logits keep that below it."""
    from eptq_b200.kernels import paged
    s = make_step(lens, nh, nkv, hd, 16, dtype, seed=nh + hd + len(lens))
    s["q"] /= 16
    got = paged.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["tables"], s["kv_lens"], s["cu_rows"], max_rows)
    step, scale, at = HALF_STEP[dtype], hd ** -0.5, 0
    for b, (kv, n) in enumerate(lens):
        keys, values = (gather(s[c], s["tables"][b], kv).double() for c in ("k_cache", "v_cache"))
        for t in range(n):
            seen = kv - n + t + 1
            q = s["q"][at].reshape(nkv, nh // nkv, hd).double()
            k, v = keys[:seen].transpose(0, 1), values[:seen].transpose(0, 1)
            p = torch.softmax(q @ k.mT * scale, dim=-1)
            o, mass = p @ v, p @ v.abs()
            spread = float((q.abs() @ k.abs().mT * scale).max()) * (hd + 8) * 2.0 ** -24 + 2.0 ** -20
            fixed = seen * 2.0 ** -30 * float(v.abs().max()) if dtype == FP16 else 0.0
            tol = step * o.abs() + (2 * step * step + 2 * spread + 3 * seen * 2.0 ** -24) * mass + fixed
            check(got[at].reshape(o.shape), o, tol, f"request {b}, row {t}")
            at += 1


@pytest.mark.parametrize("dtype", [FP16, BF16])
def test_infinite_values_stay_infinite(dtype):
    """Both parts of a weight meet an infinite value, also where one of them is small or the weight has few bits."""
    from eptq_b200.kernels import paged
    nh, nkv, hd = 4, 2, 64
    s = make_step([(200, 1), (64, 1)], nh, nkv, hd, 16, dtype, seed=2)
    s["q"].zero_()                                                               # all weights alike: a power of two, no rest
    for b, kv in enumerate((200, 64)):
        for j, key in enumerate((0, 17, kv - 1)):
            page = int(s["tables"][b, key // 16])
            s["v_cache"][page, :, key % 16, 3 * j] = math.inf if j != 1 else -math.inf
    out = paged.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["tables"], s["kv_lens"], s["cu_rows"], 1).reshape(2, nh, hd)
    assert bool((out[:, :, 0] == math.inf).all()) and bool((out[:, :, 3] == -math.inf).all()) and bool((out[:, :, 6] == math.inf).all())
    rest = [c for c in range(hd) if c not in (0, 3, 6)]
    assert bool(torch.isfinite(out[:, :, rest]).all())
