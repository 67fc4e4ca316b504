"""PagedKVCache's steps of trees against calls that do not fit them."""
import pytest
import torch

from test_gpu_speculative import check, make, put, rows_of

pytestmark = pytest.mark.gpu


def test_advance_takes_chains_and_refuses_trees():
    """advance leaves keys where they lie: row 0 has a chunk, row 1 a chain, row 2 a chain that branches at its third
    token, row 3 two roots."""
    g = torch.Generator("cuda").manual_seed(0)
    parents = [t - 1 for t in range(70)] + [-1, 0, 1, 2] + [-1, 0, 0, 1] + [-1, -1]
    new = [70, 4, 4, 2]
    for as_list in (True, False):
        cache = make()
        cache.advance(cache.plan([3, 20, 0, 17]))
        given = parents if as_list else torch.tensor(parents, dtype=torch.int32, device="cuda")
        step = cache.plan(new, parents=given, max_tree=32)
        put(cache, step, g)
        for kept, row in ((None, 2), ([70, 4, 3, 1], 2), ([0, 0, 0, 2], 3), ([70, 4, 4, 0], 2)):
            with pytest.raises(RuntimeError, match=f"of row {row} are a tree"):
                cache.advance(step, kept=kept)
        before = [x.clone() for x in rows_of(cache)]
        cache.advance(step, kept=[70, 3, 2, 1])  # (the refusals have left the step)
        check(cache)
        assert cache.host_lens().tolist() == [73, 23, 2, 18, 0, 0]
        for old, now in zip(before, rows_of(cache)):
            assert torch.equal(now[:len(old)], old)
    cache = make()
    step = cache.plan([5, 40], parents=[t - 1 for t in range(5)] + [t - 1 for t in range(40)], max_tree=32)
    cache.advance(step)
    check(cache)
    assert cache.host_lens().tolist() == [5, 40, 0, 0, 0, 0]


@pytest.mark.parametrize("bad", [dict(max_tree=0), dict(max_tree=257), dict(dtype=torch.int64), dict(device="cpu")])
def test_a_refused_plan_of_trees_drops_the_step_before(bad):
    """Row 1's pages of the step before are in the table as another row's by the time the parents are refused."""
    cache = make()
    cache.advance(cache.plan([5, 5]))
    step = cache.plan([0, 40])
    max_tree = bad.get("max_tree", 32)
    parents = torch.full((40,), -1, dtype=bad.get("dtype", torch.int32), device=bad.get("device", "cuda"))
    with pytest.raises(RuntimeError):
        cache.plan([20, 20], parents=parents, max_tree=max_tree)
    with pytest.raises(RuntimeError, match="not the planned one"):
        cache.advance(step)
    check(cache)
    cache.advance(cache.plan([20, 20]))
    check(cache)


def test_pages_shared_by_many_are_counted_when_they_change(monkeypatch):
    """16 samples each of two prompts of 40 pages that go on to share more, part by part; a plan and a count of free pages
    walk nothing that grows with the pages."""
    cache = make(n_pages=600, rows=32, max_len=1200, slots=1)
    cache.advance(cache.plan([645] + [0] * 15 + [640]))
    cache.fork([0] * 16 + [16] * 16)
    check(cache)
    cache.advance(cache.plan([30] * 32))
    cache.fork([0] * 8 + [1] * 8 + [17] * 16)
    check(cache)
    cache.advance(cache.plan([1, 40] * 16))
    cache.fork([-1, 1] * 8 + list(range(16, 32)))
    check(cache)
    cache.release([3, 17])
    check(cache)
    monkeypatch.setattr(cache, "_shared_count", lambda: pytest.fail("counted again"))
    free = cache.free_page_count()
    cache.advance(cache.plan([16] * 32))
    assert cache.free_page_count() == free - 32
    check(cache)
