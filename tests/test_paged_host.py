"""Refusals of the paged-cache operators, and their 64-bit references checked against themselves; no GPU."""
import ctypes as C

import pytest
import torch

from tests.paged_util import attention_reference, make_step, plan_reference, step_reference


def test_cpu_tensors_raise(built_library):
    from eptq_b200.kernels import paged
    i32, f16 = torch.zeros(2, dtype=torch.int32), torch.zeros(2, 128, dtype=torch.float16)
    cache = torch.zeros(2, 1, 16, 128, dtype=torch.float16)
    i64 = torch.zeros(2, dtype=torch.int64)
    for call in (lambda: paged.plan_pages(i32, i32, i32.reshape(2, 1), i32, i32[:1], 16, 2),
                 lambda: paged.rope_append_paged(f16, f16, f16, cache, cache, i64, i64, torch.zeros(64)),
                 lambda: paged.paged_attention(f16, cache, cache, i32.reshape(2, 1), i32, torch.zeros(3, dtype=torch.int32), 1),
                 lambda: paged.prompt_attention(f16, f16, f16, i32, 128)):
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            call()


def _attention(**kw):
    from eptq_b200 import _lib
    a = _lib.EptqAttention()
    values = dict(dtype=0, rows=4, batch=2, n_heads=8, n_kv_heads=2, head_dim=128, max_rows=2, page_size=16, n_pages=5, table_width=3,
                  scale=0.1, q_stride=1024, k_stride=4096, v_stride=4096, table_stride=3, q=256, k=256, v=256, tables=256, kv_lens=256,
                  cu_rows=256, out=256)
    values.update(kw)
    for k, v in values.items():
        setattr(a, k, v)
    return a


NULL, SHAPE, ALIGN, WORKSPACE, UNSUPPORTED = 1, 2, 3, 5, 7


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=2), UNSUPPORTED), (dict(head_dim=96), UNSUPPORTED), (dict(head_dim=256), UNSUPPORTED), (dict(rows=-1), SHAPE),
    (dict(batch=-1), SHAPE), (dict(n_heads=7), SHAPE), (dict(n_heads=0), SHAPE), (dict(n_kv_heads=0), SHAPE), (dict(page_size=24), SHAPE),
    (dict(page_size=8), SHAPE), (dict(page_size=256), SHAPE), (dict(page_size=-16), SHAPE), (dict(n_pages=-1), SHAPE), (dict(table_stride=2), SHAPE),
    (dict(q_stride=1000), SHAPE), (dict(k_stride=4088), SHAPE), (dict(q_stride=1028), ALIGN), (dict(v_stride=4100), ALIGN), (dict(q=264), ALIGN),
    (dict(out=257), ALIGN), (dict(q=None), NULL), (dict(out=None), NULL), (dict(k=None), NULL), (dict(kv_lens=None), NULL), (dict(cu_rows=None), NULL),
    (dict(tables=None), NULL), (dict(page_size=0, k_stride=128, v_stride=256), SHAPE)])
def test_attention_refusals(built_library, kw, status):
    """Found before anything touches a device."""
    from eptq_b200 import _lib
    lib = _lib.load()
    a = _attention(**kw)
    assert lib.eptq_ragged_attention(C.byref(a), 4096, 1 << 40, None) == status
    assert status == NULL or lib.eptq_ragged_attention_workspace_bytes(C.byref(a)) == 0


def test_attention_null_and_nothing(built_library):
    from eptq_b200 import _lib
    lib = _lib.load()
    assert lib.eptq_ragged_attention(None, None, 0, None) == NULL
    for kw in (dict(rows=0), dict(batch=0)):
        assert lib.eptq_ragged_attention(C.byref(_attention(**kw)), None, 0, None) == 0


@pytest.mark.parametrize("change,status", [
    (dict(page_size=20), SHAPE), (dict(rows=-1), SHAPE), (dict(B=-1), SHAPE), (dict(width=9), SHAPE), (dict(free_cap=-1), SHAPE),
    (dict(cu_rows=None), NULL), (dict(n_free=None), NULL), (dict(cached=None), NULL), (dict(tables=None), NULL), (dict(slots=None), NULL),
    (dict(free_pages=None), NULL)])
def test_plan_refusals(built_library, change, status):
    from eptq_b200 import _lib
    a = dict(cached=256, fresh=256, B=3, tables=256, table_stride=4, width=4, free_pages=256, free_cap=9, n_free=256, page_size=16, rows=5,
             cu_rows=256, kv_lens=256, positions=256, slots=256, n_free_out=256, stream=None)
    a.update(change)
    assert _lib.load().eptq_plan_pages(*a.values()) == status


@pytest.mark.parametrize("change,status", [
    (dict(dtype=3), UNSUPPORTED), (dict(hd=24), UNSUPPORTED), (dict(hd=512), UNSUPPORTED), (dict(ps=48), SHAPE), (dict(rows=-2), SHAPE),
    (dict(q_stride=100), SHAPE), (dict(page_stride=100), SHAPE), (dict(k_stride=268), ALIGN), (dict(v=264), ALIGN), (dict(q=None), NULL),
    (dict(slots=None), NULL), (dict(k_cache=None), NULL)])
def test_append_refusals(built_library, change, status):
    from eptq_b200 import _lib
    a = dict(dtype=0, q=256, q_stride=1024, k=256, k_stride=256, v=256, v_stride=256, q_out=256, k_cache=256, v_cache=256, page_stride=4096,
             positions=256, slots=256, inv_freq=256, rows=3, nh=8, nkv=2, hd=128, n_pages=4, ps=16, scaling=1.0, stream=None)
    a.update(change)
    assert _lib.load().eptq_rope_append_paged(*a.values()) == status


def test_references_agree():
    """Attention over a request's pages is attention over its keys in order; a row without keys is zero."""
    s = make_step([(40, 5), (0, 2), (3, 5)], 4, 2, 64, 16, torch.float16, seed=1, device="cpu")
    want, tol = step_reference(s, 4)
    assert bool((want[5:7] == 0).all()) and bool((want[7:9] == 0).all()) and bool(torch.isfinite(want).all()) and bool(torch.isfinite(tol).all())
    ids = s["tables"][0, :3].long()
    k = s["k_cache"][ids].transpose(1, 2).reshape(48, 2, 64)[:40].double()
    v = s["v_cache"][ids].transpose(1, 2).reshape(48, 2, 64)[:40].double()
    q = s["q"][4].reshape(4, 64).double()
    for h in range(4):
        p = torch.softmax(k[:, h // 2] @ q[h] / 8.0, dim=0)
        assert torch.allclose(want[4].reshape(4, 64)[h], p @ v[:, h // 2], rtol=1e-12, atol=1e-12)
    o, _ = attention_reference(s["q"][:5].reshape(5, 4, 64), k.half(), v.half(), 35, 0.125)
    assert torch.allclose(o.reshape(5, -1), want[:5], rtol=1e-12, atol=1e-12)


def test_plan_reference_by_hand():
    tables, cu, kv, pos, slots, left = plan_reference([16, 5, 0], [2, 3, 20], [[4, -1], [2, -1], [-1, -1]], [7, 9, 1], 3, 16, 30)
    assert tables == [[4, 1], [2, -1], [9, 7]] and cu == [0, 2, 5, 25] and kv == [18, 8, 20] and left == 0
    assert pos == [16, 17, 5, 6, 7] + list(range(20)) + [0] * 5
    assert slots == [16, 17, 37, 38, 39] + [144 + i for i in range(16)] + [112 + i for i in range(4)] + [-1] * 5
    tables, cu, kv, pos, slots, left = plan_reference([16, 5, 0], [2, 3, 20], [[4, -1], [2, -1], [-1, -1]], [7, 9], 2, 16, 25)
    assert kv == [18, 8, 0] and left == 1 and slots[5:] == [-1] * 20


def test_schedule_takes_every_block_once(tmp_path):
    """The device's schedule, compiled for the host: shares of random calls cover the work once, cut tiles know their pieces."""
    import shutil
    import subprocess
    from pathlib import Path
    source = Path(__file__).with_name("schedule_check.cpp")
    program = tmp_path / "schedule_check"
    subprocess.run([shutil.which("g++") or "g++", "-O1", "-std=c++17", "-o", str(program), str(source)], check=True)
    out = subprocess.run([str(program)], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and out.stdout.startswith("ok"), out.stdout
    assert int(out.stdout.split()[1]) > 10000
