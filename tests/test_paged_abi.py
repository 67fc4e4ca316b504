"""The paged cache's C ABI on the CPU: structure layouts against gcc, and the host checks that answer
with a status and a message before anything touches a device (the pointers are never read)."""
import ctypes

import pytest
import torch

from modelcore_b200 import _native
from modelcore_b200._native import PagedAppendArgs, PagedAttnArgs, PagePlanArgs, PageReleaseArgs
from test_abi import _c_layout

INVALID, UNSUPPORTED, ALIGNMENT = (_native.MCB_ERR_INVALID_ARG, _native.MCB_ERR_UNSUPPORTED,
                                   _native.MCB_ERR_ALIGNMENT)


@pytest.mark.parametrize("cls,cname", [(PagePlanArgs, "mcb_page_plan_args"), (PageReleaseArgs, "mcb_page_release_args"),
                                       (PagedAppendArgs, "mcb_paged_append_args"),
                                       (PagedAttnArgs, "mcb_paged_attn_args")])
def test_ctypes_structures_match_the_c_layout(cls, cname):
    fields = [f for f, _ in cls._fields_]
    c = _c_layout(cname, fields)
    assert c == [ctypes.sizeof(cls)] + [getattr(cls, f).offset for f in fields]


def _call(entry, cls, good, **kw):
    a = cls()
    for k, v in {**good, **kw}.items():
        if isinstance(v, tuple):
            getattr(a, k)[:] = v
        else:
            setattr(a, k, v)
    return getattr(_native.load(), entry)(ctypes.byref(a), None), _native.last_error()


def _rejects(entry, cls, good, cases):
    assert getattr(_native.load(), entry)(None, None) == INVALID
    for kw, status, words in cases:
        st, msg = _call(entry, cls, good, **kw)
        assert st == status and words in msg, (kw, st, msg)


P = 1 << 20
PLAN = dict(cache_seqlens=P, new_lens=P, block_table=P, free_pages=P, free_state=P, free_state_out=P, cu_new=P,
            positions=P, slot_map=P, counter=P, table_stride=8, R=2, N=4, n_pages=9, max_pages=8, page_size=16)


def test_plan_and_release_reject_bad_arguments():
    common = [(dict(R=-1), INVALID, "R=-1"), (dict(n_pages=0), INVALID, "n_pages"),
              (dict(max_pages=0), INVALID, "max_pages"), (dict(page_size=8), UNSUPPORTED, "power of two"),
              (dict(page_size=24), UNSUPPORTED, "power of two"), (dict(page_size=2048), UNSUPPORTED, "power of two"),
              (dict(max_pages=1 << 28, table_stride=1 << 28), UNSUPPORTED, "positions a request"),
              (dict(table_stride=7), INVALID, "table_stride"), (dict(block_table=None), INVALID, "NULL"),
              (dict(free_state_out=None), INVALID, "NULL"), (dict(counter=None), INVALID, "NULL")]
    _rejects("mcb_page_plan", PagePlanArgs, PLAN,
             common + [(dict(N=-1), INVALID, "N=-1"), (dict(slot_map=None), INVALID, "NULL")])
    release = dict(done=P, cache_seqlens=P, block_table=P, free_pages=P, free_state=P, free_state_out=P,
                   seqlens_out=P, counter=P, table_stride=8, R=2, n_pages=9, max_pages=8, page_size=16)
    _rejects("mcb_page_release", PageReleaseArgs, release, common + [(dict(done=None), INVALID, "NULL")])


def test_append_rejects_bad_arguments():
    good = dict(q=P, k=P, v=P, q_stride=(256, 64), k_stride=(128, 64), v_stride=(128, 64), q_out=P, k_pages=P,
                v_pages=P, positions=P, slot_map=P, cos=P, sin=P, N=3, Hq=4, Hkv=2, D=64, n_pages=5, page_size=16,
                rot_len=10, eps=1e-6, scale=1.2, rotate_k=1)
    _rejects("mcb_paged_append_rope", PagedAppendArgs, good, [
        (dict(N=-1), INVALID, "N=-1"), (dict(Hq=0), INVALID, "Hq=0"), (dict(D=96), UNSUPPORTED, "head_dim 96"),
        (dict(v=None), INVALID, "come together"), (dict(slot_map=None), INVALID, "NULL"),
        (dict(q_out=None), INVALID, "NULL"), (dict(rot_len=0), INVALID, "rot_len"),
        (dict(page_size=20), UNSUPPORTED, "power of two"), (dict(n_pages=0), INVALID, "n_pages"),
        (dict(k_stride=(-128, 64)), INVALID, "negative"), (dict(q_stride=(256, 68)), ALIGNMENT, "16-byte"),
        (dict(k_pages=P + 8), ALIGNMENT, "16-byte"), (dict(cos=P + 2), ALIGNMENT, "16-byte"),
        (dict(N=1 << 30), UNSUPPORTED, "vectors in one call")])
    assert _call("mcb_paged_append_rope", PagedAppendArgs, good, N=0)[0] == 0  # nothing to do


def test_attention_rejects_bad_arguments():
    good = dict(q=P, q_stride=(256, 64), k_pages=P, v_pages=P, block_table=P, table_stride=8, cache_seqlens=P,
                cu_new=P, out=P, R=2, N=4, Hq=4, Hkv=2, D=64, n_pages=9, max_pages=8, page_size=16, window=-1,
                softmax_scale=0.125)
    _rejects("mcb_paged_attn", PagedAttnArgs, good, [
        (dict(R=-1), INVALID, "R=-1"), (dict(N=-1), INVALID, "N=-1"), (dict(max_new=-1), INVALID, "max_new=-1"),
        (dict(Hq=5), INVALID, "divisible"), (dict(Hq=258), UNSUPPORTED, "at most 128"),
        (dict(D=256), UNSUPPORTED, "head_dim 256"), (dict(page_size=40), UNSUPPORTED, "power of two"),
        (dict(softmax_scale=0.0), INVALID, "softmax_scale"), (dict(softmax_scale=float("nan")), INVALID, "softmax_scale"),
        (dict(softmax_scale=float("inf")), INVALID, "softmax_scale"), (dict(out=None), INVALID, "NULL"),
        (dict(block_table=None), INVALID, "NULL"), (dict(table_stride=7), INVALID, "table_stride"),
        (dict(q_stride=(-256, 64)), INVALID, "negative"), (dict(q_stride=(256, 60)), ALIGNMENT, "16-byte"),
        (dict(v_pages=P + 8), ALIGNMENT, "16-byte"), (dict(n_pages=1 << 30, Hkv=4), UNSUPPORTED, "2^31")])
    assert _call("mcb_paged_attn", PagedAttnArgs, good, N=0)[0] == 0
    WORKSPACE, ws = _native.MCB_ERR_WORKSPACE, dict(workspace=P, workspace_bytes=1 << 30)
    _rejects("mcb_paged_attn", PagedAttnArgs, good, [
        ({}, WORKSPACE, "workspace"), (dict(workspace=P, workspace_bytes=16), WORKSPACE, "workspace"),
        (dict(ws, workspace=P + 16), WORKSPACE, "256-byte"), (dict(ws, counters=None), WORKSPACE, "counters"),
        (dict(ws, counters=P, counter_count=3), WORKSPACE, "counters")])


def test_shape_functions_on_meta_tensors():
    import modelcore_b200.torch_ops  # noqa: F401
    ints = dict(device="meta", dtype=torch.int32)
    lens, table, queue = torch.empty(5, **ints), torch.empty(5, 9, **ints), torch.empty(40, **ints)
    st = torch.empty(2, device="meta", dtype=torch.int64)
    cu, pos, slots = torch.ops.mcb200.page_plan(lens, lens, table, queue, st, st, 16, 11)
    assert cu.shape == (6,) and pos.shape == slots.shape == (11,)
    assert cu.dtype == pos.dtype == torch.int32 and slots.dtype == torch.int64
    q = torch.empty(11, 8, 128, device="meta", dtype=torch.bfloat16)
    pages = torch.empty(40, 2, 16, 128, device="meta", dtype=torch.bfloat16)
    assert torch.ops.mcb200.paged_attn(q, pages, pages, table, lens, cu).shape == q.shape
    cos = torch.empty(100, 64, device="meta", dtype=torch.bfloat16)
    assert torch.ops.mcb200.paged_append_rope(q, None, None, None, None, pos, None, cos, cos).shape == q.shape
    s = str(torch.ops.mcb200.paged_append_rope.default._schema)
    assert "Tensor(a!)? k_pages" in s and "Tensor(b!)? v_pages" in s
    assert "(a!)" not in str(torch.ops.mcb200.paged_attn.default._schema)
