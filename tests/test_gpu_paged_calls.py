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


# ---- what is written is marked as written --------------------------------------------------------------------------
def _append_case(rows=4, nh=4, nkv=2, hd=64, ps=16):
    g = torch.Generator(device="cuda").manual_seed(rows)
    q, k, v = (torch.randn(rows, n * hd, generator=g, device="cuda").half() for n in (nh, nkv, nkv))
    kc, vc = (torch.zeros(3, nkv, ps, hd, dtype=FP16, device="cuda") for _ in range(2))
    pos = torch.arange(rows, device="cuda")
    return q, k, v, kc, vc, pos, pos + ps, 1.0 / (10000.0 ** (torch.arange(0, hd, 2, device="cuda").float() / hd))


def _plan_case():
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")            # noqa: E731
    return [i32([0, 3]), i32([20, 1]), i32([[-1, -1], [2, -1]]), i32([0, 1, 3]), i32([3]), 16, 21]


def test_versions_of_written_tensors_move():
    from eptq_b200.kernels import paged
    q, k, v, kc, vc, pos, slots, inv = _append_case()
    both = torch.zeros(2, *kc.shape, dtype=FP16, device="cuda")
    before = q._version, kc._version, vc._version, both._version
    assert paged.rope_append_paged(q, k, v, kc, vc, pos, slots, inv, out=q) is q
    assert q._version > before[0] and kc._version > before[1] and vc._version > before[2]
    paged.rope_append_paged(q, k, v, both[0], both[1], pos, slots, inv)
    assert both._version > before[3]                                            # through views
    plan = _plan_case()
    versions = [t._version for t in plan[:5]]
    paged.plan_pages(*plan)
    assert [t._version > v for t, v in zip(plan[:5], versions)] == [False, False, True, False, False]
    s = make_step([(20, 2)], 4, 2, 64, 16, FP16, seed=1)
    out = torch.zeros_like(s["q"])
    version = out._version, s["k_cache"]._version
    _attend(s, out=out)
    assert out._version > version[0] and s["k_cache"]._version == version[1]
    version = out._version
    paged.prompt_attention(s["q"], k[:2], v[:2], s["cu_rows"], 64, out=out)
    assert out._version > version


def test_autograd_sees_an_overwritten_tensor():
    w = torch.ones(2, 256, dtype=FP16, device="cuda", requires_grad=True)
    s = make_step([(20, 2)], 4, 2, 64, 16, FP16, seed=1)
    out = torch.ones_like(s["q"])
    y = (w * out).sum()
    _attend(s, out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_a_lazy_copy_keeps_its_values():
    from eptq_b200.kernels import paged
    q, k, v, kc, vc, pos, slots, inv = _append_case()
    copies = [torch._lazy_clone(t) for t in (q, kc, vc)]
    want = [t.clone() for t in (q, kc, vc)]
    paged.rope_append_paged(q, k, v, kc, vc, pos, slots, inv, out=q)
    assert all(torch.equal(c, w) for c, w in zip(copies, want))
    assert not torch.equal(q, want[0]) and bool((kc[1, :, :4] != 0).any()) and torch.equal(vc[1, :, :4].transpose(0, 1).reshape(4, -1), v)
    plan = _plan_case()
    copy, old = torch._lazy_clone(plan[2]), plan[2].clone()
    paged.plan_pages(*plan)
    assert torch.equal(copy, old) and plan[2].tolist() == [[3, 1], [2, -1]]


def test_tensors_made_in_inference_mode():
    from eptq_b200.kernels import paged
    with torch.inference_mode():
        case, plan = _append_case(), _plan_case()
        inside = paged.rope_append_paged(*case)
        paged.plan_pages(*plan)
    assert torch.equal(paged.rope_append_paged(*case), inside)
    assert plan[2].tolist() == [[3, 1], [2, -1]]
    paged.plan_pages(*plan)


# ---- refusals --------------------------------------------------------------------------------------------------------
def test_gradients_and_tangents_are_refused():
    import torch.autograd.forward_ad as fwAD
    from eptq_b200.kernels import paged
    q, k, v, kc, vc, pos, slots, inv = _append_case()
    cu = torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    want = paged.prompt_attention(q, k, v, cu, 64)
    for i in range(3):
        x = [q, k, v]
        x[i] = x[i].clone().requires_grad_()
        with pytest.raises(RuntimeError, match="gradient"):
            paged.prompt_attention(*x, cu, 64)
        with torch.no_grad():
            assert torch.equal(paged.prompt_attention(*x, cu, 64), want)
        with fwAD.dual_level():
            x[i] = fwAD.make_dual([q, k, v][i], torch.ones_like([q, k, v][i]))
            with pytest.raises(RuntimeError, match="tangent"):
                paged.prompt_attention(*x, cu, 64)
            with pytest.raises(RuntimeError, match="tangent"):
                paged.rope_append_paged(*x, kc, vc, pos, slots, inv)
            with torch.no_grad(), fwAD._set_fwd_grad_enabled(False):
                assert torch.equal(paged.prompt_attention(*x, cu, 64), want)
            assert torch.equal(paged.prompt_attention(q, k, v, cu, 64), want)
    assert bool((kc == 0).all())


def test_outputs_that_overlap_are_refused():
    from eptq_b200.kernels import paged
    q, k, v, kc, vc, pos, slots, inv = _append_case(nh=2)
    cu = torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    flat = torch.zeros(5 * 128, dtype=FP16, device="cuda")
    shifted, ahead = flat[128:].view(4, 128), flat[:-128].view(4, 128)
    for out, what in ((k, "k"), (v, "v"), (kc.view(-1)[:512].view(4, 128), "k_cache"), (vc.view(-1)[-512:].view(4, 128), "v_cache")):
        with pytest.raises(RuntimeError, match=f"`out` overlaps `{what}`"):
            paged.rope_append_paged(q, k, v, kc, vc, pos, slots, inv, out=out)
    with pytest.raises(RuntimeError, match="`out` overlaps `q`"):
        paged.rope_append_paged(shifted, k, v, kc, vc, pos, slots, inv, out=ahead)
    with pytest.raises(RuntimeError, match="the same memory"):
        paged.rope_append_paged(q, k, v, kc, kc, pos, slots, inv)
    for out, what in ((k, "k"), (v, "v")):
        with pytest.raises(RuntimeError, match=f"`out` overlaps `{what}`"):
            paged.prompt_attention(q, k, v, cu, 64, out=out)
    with pytest.raises(RuntimeError, match="`out` overlaps `q`"):
        paged.prompt_attention(shifted, k, v, cu, 64, out=ahead)
    wide = torch.zeros(4, 512, dtype=FP16, device="cuda")
    with pytest.raises(RuntimeError, match="`out` overlaps `q`"):
        paged.prompt_attention(wide[:, :128], k, v, cu, 64, out=wide.view(-1)[:512].view(4, 128))
    tables, kv = torch.zeros(1, 2, dtype=torch.int32, device="cuda"), torch.tensor([4], dtype=torch.int32, device="cuda")
    for out, what in ((kc.view(-1)[:512].view(4, 128), "k_cache"), (vc.view(-1)[-512:].view(4, 128), "v_cache")):
        with pytest.raises(RuntimeError, match=f"`out` overlaps `{what}`"):
            paged.paged_attention(q, kc, vc, tables, kv, cu, 4, out=out)
    torch.cuda.synchronize()
    assert bool((kc == 0).all()) and bool((vc == 0).all())


@pytest.mark.parametrize("told", [1, 100000])
def test_attention_in_place_of_q(told):
    """Tiles that are cut and tiles that are not."""
    from eptq_b200.kernels import paged
    s = make_step([(9000, 21), (40, 40), (333, 1)], 8, 2, 128, 16, FP16, seed=4)
    want = _attend(s, max_rows=told)
    assert _attend(s, max_rows=told, out=s["q"]) is s["q"] and torch.equal(s["q"], want)
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = (torch.randn(3000, n * 64, generator=g, device="cuda").half() for n in (4, 2, 2))
    cu = torch.tensor([0, 700, 3000], dtype=torch.int32, device="cuda")
    want = paged.prompt_attention(q, k, v, cu, 64)
    assert paged.prompt_attention(q, k, v, cu, 64, out=q) is q and torch.equal(q, want)


# ---- waits that ran out ------------------------------------------------------------------------------------------------
def test_status_word_of_the_stream_is_read():
    """The word that the attention kernels are given is one that `workspace_status_all` reads: set here by hand, no wait runs out."""
    from eptq_b200 import _lib
    from eptq_b200.kernels import workspace_status_all
    s = make_step([(20, 2), (300, 1)], 4, 2, 64, 16, FP16, seed=1)
    device = s["q"].device
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        for told in (1, 1000):
            _attend(s, max_rows=told)
        mine = _lib.host().scratch(device.index, 0)                                 # of this stream
        assert mine.data_ptr() in {t.data_ptr() for t in _lib.host().scratch_of_device(device.index)}
        assert workspace_status_all(device) == 0                                    # waits that did not run out
        word = mine[4092:4096].view(torch.int32)
        word.fill_(6)
        assert workspace_status_all(device) == 6 and workspace_status_all(device) == 0 and int(word) == 0


def test_scratch_made_in_a_capture():
    """A stream's first call is a captured one: its scratch is zero at once, and no replay clears a code that stands there."""
    from eptq_b200 import _lib
    from eptq_b200.kernels import workspace_status_all
    s = make_step([(20, 2), (300, 1)], 4, 2, 64, 16, FP16, seed=1)
    want, device = _attend(s), s["q"].device
    before = {t.data_ptr() for t in _lib.host().scratch_of_device(device.index)}
    for _ in range(64):                                                             # a stream that has no scratch yet
        stream = torch.cuda.Stream()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = _attend(s)
        with torch.cuda.stream(stream):
            mine = _lib.host().scratch(device.index, 0)
        if mine.data_ptr() not in before:
            break
    else:
        pytest.skip("every stream of the pool has scratch by now")
    assert bool((mine[:1 << 20] == 0).all())                                        # before any replay
    mine[4092:4096].view(torch.int32).fill_(6)
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and workspace_status_all(device) == 6 and workspace_status_all(device) == 0


def test_lazy_copies_of_inputs_are_outputs():
    """A lazy copy shares its original's memory until it is written; that is no overlap."""
    from eptq_b200.kernels import paged
    q, k, v, kc, vc, pos, slots, inv = _append_case(nh=2)
    cu = torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    want = paged.prompt_attention(q, k, v, cu, 64)
    old = k.clone()
    assert torch.equal(paged.prompt_attention(q, k, v, cu, 64, out=torch._lazy_clone(k)), want) and torch.equal(k, old)
    paged.rope_append_paged(q, k, v, kc, torch._lazy_clone(kc), pos, slots, inv)
    assert bool((kc[1] != 0).any())
