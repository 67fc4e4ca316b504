"""The C ABI of speculative decoding and shared pages on the CPU: structure layouts against gcc, and the
host checks that answer with a status and a message before anything touches a device (the pointers are
never read)."""
import ctypes

import pytest
import torch

from modelcore_b200 import _native
from modelcore_b200._native import (DraftTreeArgs, PagedAttnArgs, PagedKeepArgs, PagedTreeAttnArgs, PageForkArgs,
                                    VerifyDraftsArgs)
from test_abi import _c_layout

INVALID, UNSUPPORTED, ALIGNMENT, WORKSPACE = (_native.MCB_ERR_INVALID_ARG, _native.MCB_ERR_UNSUPPORTED,
                                              _native.MCB_ERR_ALIGNMENT, _native.MCB_ERR_WORKSPACE)
P = 1 << 20


@pytest.mark.parametrize("cls,cname", [(DraftTreeArgs, "mcb_draft_tree_args"),
                                       (PagedTreeAttnArgs, "mcb_paged_tree_attn_args"),
                                       (VerifyDraftsArgs, "mcb_verify_drafts_args"),
                                       (PagedKeepArgs, "mcb_paged_keep_args"), (PageForkArgs, "mcb_page_fork_args")])
def test_ctypes_structures_match_the_c_layout(cls, cname):
    fields = [f for f, _ in cls._fields_]
    assert _c_layout(cname, fields) == [ctypes.sizeof(cls)] + [getattr(cls, f).offset for f in fields]


def _fill(cls, values):
    a = cls()
    for k, v in values.items():
        if isinstance(v, dict):
            setattr(a, k, _fill(PagedAttnArgs, v))
        elif isinstance(v, tuple):
            getattr(a, k)[:] = v
        else:
            setattr(a, k, v)
    return a


def _rejects(entry, cls, good, cases):
    fn = getattr(_native.load(), entry)
    assert fn(None, None) == INVALID
    for kw, status, words in cases:
        st, msg = fn(ctypes.byref(_fill(cls, {**good, **kw})), None), _native.last_error()
        assert st == status and words in msg, (kw, st, msg)
    return lambda **kw: fn(ctypes.byref(_fill(cls, {**good, **kw})), None)


def test_draft_tree_rejects_bad_arguments():
    good = dict(parents=P, cu_new=P, cache_seqlens=P, positions=P, mask=P, R=2, N=5, words=2)
    call = _rejects("mcb_draft_tree", DraftTreeArgs, good, [
        (dict(R=-1), INVALID, "R=-1"), (dict(N=-1), INVALID, "N=-1"), (dict(words=0), UNSUPPORTED, "words 0"),
        (dict(words=9), UNSUPPORTED, "words 9"), (dict(parents=None), INVALID, "NULL"), (dict(mask=None), INVALID, "NULL"),
        (dict(cache_seqlens=None), INVALID, "NULL")])
    assert call(N=0) == 0


def test_tree_attention_rejects_bad_arguments():
    attn = dict(q=P, q_stride=(256, 64), k_pages=P, v_pages=P, block_table=P, table_stride=8, cache_seqlens=P, cu_new=P,
                out=P, R=2, N=4, Hq=4, Hkv=2, D=64, n_pages=9, max_pages=8, page_size=16, window=-1, softmax_scale=0.125)
    good = dict(attn=attn, positions=P, mask=P, words=1)
    of_attn = [(dict(R=-1), INVALID, "R=-1"), (dict(Hq=5), INVALID, "divisible"), (dict(Hq=258), UNSUPPORTED, "at most 128"),
               (dict(D=256), UNSUPPORTED, "head_dim 256"), (dict(page_size=40), UNSUPPORTED, "power of two"),
               (dict(softmax_scale=0.0), INVALID, "softmax_scale"), (dict(out=None), INVALID, "NULL"),
               (dict(table_stride=7), INVALID, "table_stride"), (dict(q_stride=(-256, 64)), INVALID, "negative"),
               (dict(q_stride=(256, 60)), ALIGNMENT, "16-byte"), (dict(v_pages=P + 8), ALIGNMENT, "16-byte"),
               (dict(n_pages=1 << 30, Hkv=4), UNSUPPORTED, "2^31")]
    call = _rejects("mcb_paged_tree_attn", PagedTreeAttnArgs, good,
                    [(dict(attn={**attn, **kw}), status, words) for kw, status, words in of_attn]
                    + [(dict(words=0), UNSUPPORTED, "words 0"), (dict(words=9), UNSUPPORTED, "words 9"),
                       (dict(mask=None), INVALID, "NULL"), (dict(positions=None), INVALID, "NULL")])
    assert call(attn={**attn, "N": 0}) == 0


def test_verify_rejects_bad_arguments():
    good = dict(logits=P, logits_stride=100, tokens=P, parents=P, cu_new=P, accept=P, draws=P, accepted=P, path=P,
                next_token=P, R=2, N=5, V=100, max_path=4, temperature=1.0)
    call = _rejects("mcb_verify_drafts", VerifyDraftsArgs, good, [
        (dict(R=-1), INVALID, "R=-1"), (dict(V=0), INVALID, "V=0"), (dict(V=(1 << 30) + 1), UNSUPPORTED, "2^30"), (dict(max_path=0), INVALID, "max_path=0"),
        (dict(temperature=-1.0), INVALID, "temperature"), (dict(temperature=float("nan")), INVALID, "temperature"),
        (dict(temperature=float("inf")), INVALID, "temperature"), (dict(logits=None), INVALID, "NULL"),
        (dict(draws=None), INVALID, "NULL"), (dict(path=None), INVALID, "NULL"),
        (dict(logits_stride=99), INVALID, "closer together"),
        (dict(draft_probs=P, draft_stride=99), INVALID, "closer together")])
    assert call(R=0) == 0


POOL = dict(k_pages=P, v_pages=P, R=2, slots=3, Hkv=2, D=64, n_pages=9, max_pages=8, page_size=16, table_stride=8)
OF_POOL = [(dict(R=-1), INVALID, "R=-1"), (dict(slots=0), INVALID, "slots=0"), (dict(Hkv=0), INVALID, "Hkv=0"),
           (dict(D=96), UNSUPPORTED, "head_dim 96"), (dict(n_pages=0), INVALID, "n_pages"),
           (dict(page_size=24), UNSUPPORTED, "power of two"), (dict(k_pages=None), INVALID, "NULL"),
           (dict(free_state_out=None), INVALID, "NULL"), (dict(table_stride=7), INVALID, "table"),
           (dict(v_pages=P + 8), ALIGNMENT, "16-byte"), (dict(max_pages=1 << 28, table_stride=1 << 28), UNSUPPORTED, "2^31"),
           (dict(n_pages=1 << 30, Hkv=4), UNSUPPORTED, "2^31")]


def test_keep_rejects_bad_arguments():
    good = dict(POOL, path=P, path_stride=5, accepted=P, cache_seqlens=P, new_lens=P, block_table=P, free_pages=P,
                free_state=P, free_state_out=P, seqlens_out=P, counter=P, P=5)
    _rejects("mcb_paged_keep", PagedKeepArgs, good, OF_POOL + [
        (dict(P=-1), INVALID, "P=-1"), (dict(path=None), INVALID, "NULL"), (dict(counter=None), INVALID, "NULL"),
        (dict(path_stride=4), INVALID, "path_stride")])


def test_fork_rejects_bad_arguments():
    good = dict(POOL, source=P, cache_seqlens=P, block_table=P, shares=P, free_pages=P, free_state=P, block_table_out=P,
                table_out_stride=8, shares_out=P, free_state_out=P, seqlens_out=P)
    _rejects("mcb_page_fork", PageForkArgs, good, OF_POOL + [
        (dict(source=None), INVALID, "NULL"), (dict(shares=None), INVALID, "NULL"),
        (dict(table_out_stride=7), INVALID, "table"), ({}, WORKSPACE, "workspace"),
        (dict(workspace=P, workspace_bytes=16), WORKSPACE, "workspace"),
        (dict(workspace=P + 16, workspace_bytes=1 << 30), WORKSPACE, "256-byte")])


def test_shape_functions_on_meta_tensors():
    import modelcore_b200.torch_ops  # noqa: F401
    ints = dict(device="meta", dtype=torch.int32)
    n, rows = torch.empty(11, **ints), torch.empty(5, **ints)
    cu, table = torch.empty(6, **ints), torch.empty(5, 9, **ints)
    pos, mask = torch.ops.mcb200.draft_tree(n, cu, rows, 40)
    assert pos.shape == (11,) and mask.shape == (11, 2) and mask.dtype == torch.int32
    q = torch.empty(11, 8, 128, device="meta", dtype=torch.bfloat16)
    pages = torch.empty(40, 2, 16, 128, device="meta", dtype=torch.bfloat16)
    assert torch.ops.mcb200.paged_tree_attn(q, pages, pages, table, rows, cu, pos, mask).shape == q.shape
    logits, u = torch.empty(11, 99, device="meta"), torch.empty(11, device="meta")
    kept, path, token = torch.ops.mcb200.verify_drafts(logits, n.long(), n, cu, u, u[:5], 1.0, None, 7)
    assert kept.shape == (5,) and path.shape == (5, 7) and token.shape == (5,) and token.dtype == torch.int64
    assert kept.dtype == path.dtype == torch.int32
    assert "(e!) v_pages" in str(torch.ops.mcb200.paged_keep.default._schema)
    assert "Tensor(a!) free_pages" in str(torch.ops.mcb200.page_fork.default._schema)
    assert "!" not in str(torch.ops.mcb200.paged_tree_attn.default._schema)
