"""Limits of the C ABI of speculative decoding and shared pages, on the CPU: what is refused with a status and a
message, and what is not (the pointers are never read)."""
from modelcore_b200._native import PagedKeepArgs, VerifyDraftsArgs
from test_draft_abi import INVALID, POOL, UNSUPPORTED, P, _rejects


def test_verify_takes_temperatures_of_forty_orders():
    good = dict(logits=P, logits_stride=100, tokens=P, parents=P, cu_new=P, accept=P, draws=P, accepted=P, path=P,
                next_token=P, R=2, N=5, V=100, max_path=4, temperature=1.0)
    call = _rejects("mcb_verify_drafts", VerifyDraftsArgs, good, [
        (dict(temperature=9e-21), UNSUPPORTED, "from 1e-20"), (dict(temperature=1e-45), UNSUPPORTED, "from 1e-20"),
        (dict(temperature=2e20), UNSUPPORTED, "to 1e20"), (dict(temperature=3.3e38), INVALID, "finite")])
    for fine in (0.0, 1e-20, 1e20):
        assert call(R=0, temperature=fine) == 0


def test_keep_refuses_what_no_grid_holds():
    good = dict(POOL, path=P, path_stride=5, accepted=P, cache_seqlens=P, new_lens=P, block_table=P, free_pages=P,
                free_state=P, free_state_out=P, seqlens_out=P, counter=P, P=5)
    _rejects("mcb_paged_keep", PagedKeepArgs, good, [
        (dict(R=65535), UNSUPPORTED, "at most 65,534"),
        (dict(R=1000, slots=1 << 20, Hkv=512), UNSUPPORTED, "above 2^41")])
