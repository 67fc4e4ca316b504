"""PagedKVCache's steps that do not go from plan to advance one after another: planned again, dropped, rows
released in between.  Whatever the order, the queue on the GPU and the host's count agree and every page has
one owner."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

PAGE = 16


def make(n_pages=10, rows=3, max_len=160):
    from modelcore_b200 import PagedKVCache
    return PagedKVCache(n_pages, PAGE, 2, 64, 1, rows, max_len, "cuda")


def check(cache):
    """The cache's state read from the GPU: lengths, owned and free pages."""
    from modelcore_b200 import ops
    code, what = ops.device_error()
    assert code == 0, what
    lens = cache.host_lens()
    assert cache.cache_seqlens.tolist() == lens.tolist()
    head, tail = cache.free_state.tolist()
    assert tail - head == cache.free_page_count()
    queue, table = cache.free_pages.tolist(), cache.block_table.tolist()
    free = [queue[x % cache.n_pages] for x in range(head, tail)]
    owned = [p for r, n in enumerate(lens.tolist()) for p in table[r][:-(-n // PAGE)]]
    assert sorted(free + owned) == list(range(cache.n_pages))


def slots_of(cache, step):
    return step.plan.slot_map.tolist()


def test_planning_again_takes_no_more_pages():
    cache = make()
    first = cache.plan([90])
    second = cache.plan([90])
    assert slots_of(cache, first) == slots_of(cache, second) and cache.free_page_count() == 10
    check(cache)
    third = cache.plan([70, 80])  # all ten pages: there if the dropped plans took none
    assert len(set(slots_of(cache, third))) == 150 and min(slots_of(cache, third)) >= 0
    cache.advance(third)
    assert cache.free_page_count() == 0
    check(cache)


def test_a_dropped_or_advanced_step_is_refused():
    from modelcore_b200 import ops  # noqa: F401
    cache = make()
    q = torch.zeros(20, 2, 64, device="cuda", dtype=torch.bfloat16)
    cos = torch.ones(160, 32, device="cuda", dtype=torch.bfloat16)
    old = cache.plan([20])
    step = cache.plan([10, 10])
    uses = (lambda s: cache.append(0, q, q, q, s, cos, cos), lambda s: cache.attend(0, q, s), cache.advance)
    for use in uses:
        with pytest.raises(RuntimeError, match="not the planned one"):
            use(old)
    for use in uses:
        use(step)
    for use in uses:
        with pytest.raises(RuntimeError, match="not the planned one"):
            use(step)
    check(cache)
    assert cache.host_lens().tolist() == [10, 10, 0]


def test_rows_released_while_a_step_is_planned():
    cache = make()
    cache.advance(cache.plan([40, 30, 20]))
    step = cache.plan([10, 0, 1])  # one new page, for row 0
    cache.release([1])             # not in the step
    check(cache)
    cache.advance(step)
    check(cache)
    assert cache.host_lens().tolist() == [50, 0, 21] and cache.free_page_count() == 4
    step = cache.plan([30, 5])
    cache.release([0])             # in the step, which is dropped
    with pytest.raises(RuntimeError, match="not the planned one"):
        cache.advance(step)
    check(cache)
    cache.advance(cache.plan([120]))
    check(cache)
    assert cache.free_page_count() == 0


def test_a_long_life_with_dropped_plans():
    rng = np.random.default_rng(3)
    cache = make(60, 7, 300)
    for _ in range(150):
        lens = cache.host_lens()
        gone = np.nonzero((rng.random(7) < 0.1) | (lens > 250))[0]
        cache.release(gone)
        for attempt in range(rng.integers(1, 4)):
            new = np.where(rng.random(7) < 0.3, rng.integers(0, 45, 7), 1)
            while cache.pages_needed(new) > cache.free_page_count():
                new[rng.integers(0, 7)] = 0
            step = cache.plan(new, num_tokens=int(new.sum()) + int(rng.integers(0, 3)))
        if rng.random() < 0.2:
            idle = np.nonzero(new == 0)[0]
            cache.release(idle[:1])
        if rng.random() < 0.9:
            cache.advance(step)
        check(cache)


def test_a_step_kept_in_part_gives_the_other_pages_back():
    cache = make()
    cache.advance(cache.plan([14, 16, 15]))
    step = cache.plan([4, 4, 4])
    with pytest.raises(RuntimeError, match="not 5 to keep"):
        cache.advance(step, kept=[1, 5, 0])
    cache.advance(step, kept=[1, 4, 0])  # rows 0 and 2 do not need their second page after all
    check(cache)
    assert cache.host_lens().tolist() == [15, 20, 15] and cache.free_page_count() == 6
    rng = np.random.default_rng(4)
    cache = make(60, 7, 300)
    for _ in range(150):
        lens = cache.host_lens()
        cache.release(np.nonzero((rng.random(7) < 0.05) | (lens > 240))[0])
        new = rng.integers(0, 40, 7)
        while cache.pages_needed(new) > cache.free_page_count():
            new[rng.integers(0, 7)] = 0
        step = cache.plan(new)
        cache.advance(step, kept=rng.integers(0, new + 1))
        check(cache)


def test_what_is_kept_is_what_was_written():
    """Attention after partial steps against the same tokens written whole: the kept ones are in the rows'
    pages, the rejected ones in nobody's."""
    from modelcore_b200 import ops
    g = torch.Generator("cuda").manual_seed(2)
    cos, sin = (torch.randn(160, 32, device="cuda", generator=g).to(torch.bfloat16) for _ in range(2))
    new = lambda n: torch.randn(n, 6, 64, device="cuda", generator=g).to(torch.bfloat16).split([2, 2, 2], 1)
    a, b = make(30), make(30)
    ks, vs = [[], [], []], [[], [], []]
    for i in range(20):
        kept = [(i + r) % 5 for r in range(3)]
        step = a.plan([4, 4, 4])
        q, k, v = new(12)
        a.append(0, q, k, v, step, cos, sin)
        a.advance(step, kept=kept)
        for r in range(3):
            ks[r].append(k[4 * r:4 * r + kept[r]])
            vs[r].append(v[4 * r:4 * r + kept[r]])
    check(a)
    lens = [sum(map(len, x)) for x in ks]
    step = b.plan(lens)
    k, v = (torch.cat([torch.cat(x) for x in y]) for y in (ks, vs))
    b.append(0, k, k, v, step, cos, sin)
    b.advance(step)
    assert a.host_lens().tolist() == b.host_lens().tolist() == lens
    q, k, v = new(6)
    outs = []
    for cache in (a, b):
        step = cache.plan([1, 2, 3])
        outs.append(cache.attend(0, cache.append(0, q, k, v, step, cos, sin), step))
    assert torch.equal(*outs) and ops.device_error()[0] == 0
