"""The paged operators where their parts meet: blocks of unlike size one after another on an SM, sums and
windows at the ends of their types, tables with holes, steps that are dropped or kept in part, captured
graphs that go.  Plain forms and tolerances are test_gpu_paged's."""
import numpy as np
import pytest
import torch

from test_gpu_paged import U, attn_case, attn_ref, check_attn, i32  # noqa: F401
from test_gpu_paged import expects_device_error, no_device_error, ops  # noqa: F401  (fixtures)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("Hq,Hkv,D,block", [(16, 4, 128, 64), (4, 4, 64, 256), (8, 1, 128, 32)])
def test_a_full_block_and_then_a_ragged_one(ops, Hq, Hkv, D, block):
    """Many units an SM, blocks whose row quarters are all taken before blocks of a few rows: the results
    are right and repeat themselves bit for bit."""
    fresh = [block + 1 + r % 40 for r in range(150)]
    cached = [(r * 37) % 300 for r in range(150)]
    c = check_attn(ops, cached, fresh, Hq, Hkv, D, 64)
    call = lambda: ops.paged_attn(c["q"], c["kp"], c["vp"], c["table"], c["cached"], c["cu"])
    want = call()
    assert all(torch.equal(call(), want) for _ in range(20))


@pytest.mark.parametrize("D,G,fresh", [(128, 4, 40), (64, 1, 200), (128, 1, 128)])
@pytest.mark.parametrize("pattern", ["both halves, every tile", "both, then one", "halves in turn"])
def test_references_that_move_again_and_again(ops, pattern, D, G, fresh):
    """Scores that leave the exponent's range tile after tile for thousands of keys: the two warps of a row
    quarter move its reference together, or one of them does, in every order, and none waits for one
    that has gone on (the wait's limit would set a device error).  Enough requests that an SM has runs of
    a dozen tiles and more."""
    cached, scale, R = 6000, 8.0, 24
    c, ks, vs = attn_case([cached] * R, [fresh] * R, 2 * G, 2, D, 64, seed=7)
    key = torch.arange(cached + fresh, device="cuda")
    n, half = key // 128, key // 64 % 2
    level = {"both halves, every tile": 2 * n + half, "both, then one": 2 * n - n % 2 * half * 3,
             "halves in turn": n + (n + half) % 2 * 2}[pattern]
    rise = (4.0 * level).to(torch.bfloat16)  # (integers up to 400, a multiple of 4: exact)
    sign = (torch.arange(R * fresh, device="cuda") % 3 - 1).to(torch.bfloat16)[:, None]
    q = c["q"].contiguous().mul(0.25)
    q[..., 0] = sign * 4
    for r in range(R):
        ks[r][..., 0] = rise[:, None]
        page = c["table"][r].long()
        c["kp"][page[key // 64], :, key % 64] = ks[r]
    want, bound = attn_ref(q, ks, vs, [cached] * R, [fresh] * R, -1, scale)
    got = ops.paged_attn(q, c["kp"], c["vp"], c["table"], c["cached"], c["cu"], softmax_scale=scale)
    err = np.abs(got.double().cpu().numpy() - want)
    # a score of up to 1600 x 8 is a sum of fp32 products: off by up to 2^-20 of it
    slack = (2.25 * U + 8.0 * 1600 * 2.0 ** -20) * bound
    assert np.isfinite(err).all() and (err <= slack).all(), (err - slack).max()


HUGE = 2 ** 31 - 1


@pytest.mark.parametrize("new", [[HUGE] * 3, [HUGE] * 5, [20] + [HUGE] * 4 + [20], [HUGE] * 1000, [16] * 1023 + [HUGE] * 3,
                                 [40] * 1024 + [HUGE] * 1025])
def test_new_tokens_past_32_bits_stay_in_the_table(ops, expects_device_error, new):
    """Lengths that sum to 2^32 and more (a tensor never written, say): the errors are set, each row takes the
    pages of its own table row and no more, what fits the batch is planned, nothing else is written."""
    R, width, page, N = len(new), 4, 16, 300
    need = [min(-(-n // page), width) for n in new]
    have = sum(need) + 10
    whole = torch.full((R + 4, width), -77, dtype=torch.int32, device="cuda")
    outs = ops.page_plan(i32([0] * R), i32(new), whole[:R], i32(range(have)), torch.tensor([0, have], device="cuda"),
                         page_size=page, num_tokens=N)
    assert ops.device_error()[0] in (1, 7)
    start = np.concatenate([[0], np.cumsum(need)])
    want = np.where(np.arange(width)[None] < np.array(need)[:, None], start[:-1, None] + np.arange(width)[None], -77)
    assert np.array_equal(whole.cpu().numpy(), np.concatenate([want, np.full((4, width), -77)]))
    assert outs.free_state.tolist() == [sum(need), have]
    cu = np.minimum(np.concatenate([[0], np.cumsum(np.array(new, dtype=np.int64))]), HUGE)
    assert outs.cu_new.tolist() == cu.tolist()
    pos, slots = np.zeros(N, np.int64), np.full(N, -1)
    for t in range(N):
        r = int(np.searchsorted(cu, t, side="right")) - 1
        pos[t] = t - cu[r]
        if pos[t] < width * page:
            slots[t] = want[r, pos[t] // page] * page + pos[t] % page
    assert outs.positions.tolist() == pos.tolist() and outs.slot_map.tolist() == slots.tolist()


@pytest.mark.parametrize("window", [HUGE, HUGE - 1, HUGE - 62, HUGE - 200, 2 ** 30, 1000])
@pytest.mark.parametrize("Hq,Hkv,D", [(16, 4, 128), (6, 6, 64)])
def test_a_window_wider_than_the_positions(ops, window, Hq, Hkv, D):
    """The widest windows are no windows, for the first tokens of a prompt too."""
    check_attn(ops, [0, 0, 70, 5], [300, 1, 200, 3], Hq, Hkv, D, 64, window, hints=(0, 300))
    check_attn(ops, [0, 3, 70, 500], [1, 1, 1, 1], Hq, Hkv, D, 64, window, hints=(0, 1))


def test_release_after_the_queue_ran_out(ops, expects_device_error):
    """Entries that plan left at -1 for want of pages (or that name no page) do not go into the queue: it holds
    every real page once again, and later plans take them."""
    page, n_pages = 16, 10
    table = torch.full((2, 8), -1, dtype=torch.int32, device="cuda")
    queue, state = i32(range(n_pages)), torch.tensor([0, n_pages], device="cuda")
    lens = i32([0, 0])
    ops.page_plan(lens, i32([96, 96]), table, queue, state, page_size=page, num_tokens=192, free_state_out=state)
    assert ops.device_error()[0] == 5 and table.tolist() == [[0, 1, 2, 3, 4, 5, -1, -1], [6, 7, 8, 9, -1, -1, -1, -1]]
    lens.copy_(i32([96, 96]))
    for done in ([0, 1], [1, 0]):
        ops.page_release(i32(done), lens, table, queue, state, page_size=page, free_state_out=state, seqlens_out=lens)
    assert ops.device_error()[0] == 6 and lens.tolist() == [0, 0] and state.tolist() == [10, 20]
    assert queue.tolist() == [6, 7, 8, 9, 0, 1, 2, 3, 4, 5]
    plan = ops.page_plan(lens, i32([80, 80]), table, queue, state, page_size=page, num_tokens=160, free_state_out=state)
    assert ops.device_error()[0] == 0 and sorted(table[:, :5].flatten().tolist()) == list(range(10))
    assert state.tolist() == [20, 20] and (plan.slot_map >= 0).all()


@pytest.mark.parametrize("R,hi,holes", [(3, 100, 0.5), (40, 2000, 0.1), (40, 2000, 0.001), (1500, 3000, 0.02), (700, 60, 1.0)])
def test_release_of_tables_with_holes(ops, expects_device_error, R, hi, holes):
    """Holes anywhere, over one CTA and many: the pages go back in order without them."""
    rng = np.random.default_rng(R)
    page, cached = 16, rng.integers(0, hi, R)
    held = -(-cached // page)
    total = int(held.sum()) + 5
    table = np.full((R, int(held.max()) + 2), 12345678, np.int64)
    order, at, want = rng.permutation(total), 0, []
    done = (rng.random(R) < 0.8).astype(int)
    for r in range(R):
        table[r, :held[r]] = order[at:at + held[r]]
        at += held[r]
        bad = rng.random(held[r]) < holes
        table[r, :held[r]][bad] = rng.choice([-1, total, 2 ** 31 - 1, -2 ** 31], bad.sum())
        want += table[r, :held[r]][~bad].tolist() if done[r] else []
    queue = np.arange(total) + 1000
    head, tail = 7 * total + total - 3, 7 * total + total  # three free ones, the queue going round at once
    got = i32(queue)
    st, lens = ops.page_release(i32(done), i32(cached), i32(table), got, torch.tensor([head, tail], device="cuda"),
                                page_size=page)
    ops.device_error()
    assert st.tolist() == [head, tail + len(want)] and lens.tolist() == np.where(done, 0, cached).tolist()
    got = got.cpu().numpy()
    assert got[(tail + np.arange(len(want))) % total].tolist() == want
    assert got[(head + np.arange(3)) % total].tolist() == queue[(head + np.arange(3)) % total].tolist()


@pytest.mark.parametrize("R,hi,page,in_place", [(1, 50, 16, True), (40, 3000, 16, False), (1500, 700, 32, True),
                                                (64, 30000, 64, False)])
def test_release_down_to_a_length(ops, R, hi, page, in_place):
    """keep_lens: below, at and above the length, negative; only of the requests that are done."""
    rng = np.random.default_rng(R)
    cached, done = rng.integers(0, hi, R), (rng.random(R) < 0.7).astype(int)
    keep = np.where(rng.random(R) < 0.2, rng.choice([-3, hi + 5, 0], R), (cached * rng.random(R)).astype(int))
    held = -(-cached // page)
    total, width = int(held.sum()) + 4, int(held.max()) + 2
    table, order, at = np.full((R, width), -1, np.int64), rng.permutation(total), 0
    left = np.where(done, np.clip(keep, 0, cached), cached)
    want = []
    for r in range(R):
        table[r, :held[r]] = order[at:at + held[r]]
        at += held[r]
        want += table[r, -(-left[r] // page):held[r]].tolist()
    head, tail = 5 * total + 2, 5 * total + 6
    queue, lens, st = i32(np.arange(total)), i32(cached), torch.tensor([head, tail], device="cuda")
    out = dict(free_state_out=st, seqlens_out=lens) if in_place else {}
    st, new = ops.page_release(i32(done), lens, i32(table), queue, st, page_size=page, keep_lens=i32(keep), **out)
    assert new.tolist() == left.tolist() and st.tolist() == [head, tail + len(want)]
    assert queue.cpu().numpy()[(tail + np.arange(len(want))) % total].tolist() == want
    for bad in (i32(keep[:-1]), i32(keep).long(), i32(keep).cpu(), new):
        with pytest.raises(RuntimeError):
            ops.page_release(i32(done), i32(cached), i32(table), queue, st, page_size=page, seqlens_out=new,
                             keep_lens=bad)


def test_captures_leave_no_memory_behind(ops):
    """Steps captured again and again (a server that meets new shapes) and dropped: what the captures took is
    given back, and the graphs that live on count arrivals of their own."""
    c, _, _ = attn_case([3000] * 4, [1] * 4, 16, 4, 128, 16, seed=1)
    call = lambda: ops.paged_attn(c["q"], c["kp"], c["vp"], c["table"], c["cached"], c["cu"], max_new=1)
    want = call()

    def capture():
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        return graph, out

    def reserved():
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        return torch.cuda.memory_reserved()

    keep, out = capture()
    capture()
    before = reserved()
    for _ in range(12):
        graph, got = capture()
        graph.replay()
        assert torch.equal(got, want)
        del graph, got
    assert reserved() <= before
    for _ in range(3):
        out.zero_()
        keep.replay()
        assert torch.equal(out, want)


@pytest.mark.parametrize("D,G,fresh", [(128, 4, 100), (64, 1, 300), (128, 8, 1), (64, 4, 5)])
@pytest.mark.parametrize("rise", [7, 14, 30, 60])
def test_large_values_behind_scores_that_rise(ops, D, G, fresh, rise):
    """Values of 2^60 (and enough requests that an SM has runs of tiles): weights relative to a reference that
    lies far behind would carry the sums past fp32's range, the result is finite."""
    cached, scale, R = 1400, 1.0, 60
    c, ks, vs = attn_case([cached] * R, [fresh] * R, 2 * G, 2, D, 64, seed=11)
    key = torch.arange(cached + fresh, device="cuda")
    up = torch.where(key % 512 >= 128, float(rise), 0.0).to(torch.bfloat16)[:, None]
    q = c["q"].contiguous().mul(0.25)
    q[..., 0] = 1
    for r in range(R):
        ks[r][..., 0] = up
        vs[r].mul_(2.0 ** 60)
        page = c["table"][r].long()
        for pool, x in ((c["kp"], ks[r]), (c["vp"], vs[r])):
            pool[page[key // 64], :, key % 64] = x
    want, bound = attn_ref(q, ks, vs, [cached] * R, [fresh] * R, -1, scale)
    got = ops.paged_attn(q, c["kp"], c["vp"], c["table"], c["cached"], c["cu"], softmax_scale=scale)
    err = np.abs(got.double().cpu().numpy() - want)
    # (a score below 2^7 is a sum of fp32 products: off by 2^-13 at most, its weight by that relatively)
    assert np.isfinite(err).all() and (err <= (2.25 * U + 8.0 * 2.0 ** -13) * bound).all(), (err / bound).max()


def test_a_dimension_of_one_has_any_stride(ops):
    """One token, or one head: torch may give its dimension any stride, and it is not used."""
    from test_gpu_paged import append_inputs, tables
    cos, sin = tables(300, 64)
    odd = lambda x, d: x.contiguous().as_strided(x.shape, [13 if i == d else s for i, s in
                                                           enumerate(x.contiguous().stride())])
    for N, H, d in ((1, 4, 0), (6, 1, 1)):
        (q, k, v), slots, pos, (kp, vp) = append_inputs(N, H, H, 64, 16, 9)
        kp2, vp2 = kp.clone(), vp.clone()
        want = ops.paged_append_rope(q, k, v, kp, vp, pos, slots, cos, sin)
        got = ops.paged_append_rope(odd(q, d), odd(k, d), odd(v, d), kp2, vp2, pos, slots, cos, sin)
        assert torch.equal(got, want) and torch.equal(kp2[slots // 16, :, slots % 16], kp[slots // 16, :, slots % 16])
        assert torch.equal(vp2[slots // 16, :, slots % 16], vp[slots // 16, :, slots % 16])


def test_one_query_for_all(ops):
    """Queries expanded over tokens or heads (a stride of 0) are what their copies are."""
    for fresh in ([40, 3], [1, 1]):
        c, _, _ = attn_case([90, 10], fresh, 4, 2, 64, 16)
        for q in (c["q"][:1].expand(sum(fresh), 4, 64), c["q"][:, :1].expand(sum(fresh), 4, 64)):
            call = lambda x: ops.paged_attn(x, c["kp"], c["vp"], c["table"], c["cached"], c["cu"])
            assert torch.equal(call(q), call(q.contiguous()))


def test_the_paged_step_under_torch_compile(ops):
    """plan, append (keys and values, and queries alone), attention and release as nodes of a compiled graph:
    the results and what is written in place are the eager step's."""
    from test_gpu_paged import tables
    Hq, Hkv, D, page, R = 8, 2, 128, 16, 3
    cos, sin = tables(400, D)
    g = torch.Generator("cuda").manual_seed(5)
    qkv = torch.randn(R, Hq + 2 * Hkv, D, device="cuda", generator=g).to(torch.bfloat16)
    q, k, v = qkv.split([Hq, Hkv, Hkv], 1)
    ones, done = i32([1] * R), i32([0, 1, 0])
    from modelcore_b200 import torch_ops  # noqa: F401
    m = torch.ops.mcb200

    def step(lens, table, queue, state, kp, vp):
        state2 = torch.empty_like(state)
        cu, pos, slots = m.page_plan(lens, ones, table, queue, state, state2, page, R)
        qr = m.paged_append_rope(q, k, v, kp, vp, pos, slots, cos, sin)
        alone = m.paged_append_rope(q, None, None, None, None, pos, None, cos, sin)
        out = m.paged_attn(qr, kp, vp, table, lens, cu, window=100, max_new=1)
        lens += ones
        m.page_release(done, lens, table, queue, state2, state2, lens, page)
        return out * 1.0, alone, state2, cu, pos, slots

    def fresh():
        pool = lambda s: torch.randn(40, Hkv, page, D, device="cuda", generator=torch.Generator("cuda").manual_seed(s)
                                     ).to(torch.bfloat16)
        return [i32([0, 90, 300]), i32(np.arange(R * 30).reshape(R, 30) % 30), i32(np.arange(40)),
                torch.tensor([30, 40], device="cuda"), pool(1), pool(2)]

    compiled = torch.compile(step, fullgraph=True, backend="aot_eager")
    a, b = fresh(), fresh()
    for _ in range(3):
        for x, y in zip(step(*a), compiled(*b)):
            assert torch.equal(x, y)
        for x, y in zip(a, b):
            assert torch.equal(x, y)
        a[3], b[3] = (torch.tensor([30, 40], device="cuda") for _ in range(2))


def test_tokens_before_the_first_request_are_padding_too(ops):
    """A batch whose first request starts after token 0: nobody's tokens come out as zeros, before and after."""
    for fresh in ([1, 2], [70, 5]):
        c, ks, vs = attn_case([30, 200], fresh, 4, 2, 64, 16, tail=9)
        at = c["cu"] + 4
        want = ops.paged_attn(c["q"][4:].contiguous(), c["kp"], c["vp"], c["table"], c["cached"], c["cu"])
        junk = torch.full_like(c["q"].contiguous(), float("nan"))
        del junk  # (the output's memory, as like as not)
        got = ops.paged_attn(c["q"], c["kp"], c["vp"], c["table"], c["cached"], at)
        assert not got[:4].any() and torch.equal(got[4:], want)
