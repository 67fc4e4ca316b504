"""The paged cache's operators against plain implementations in 64 bits (numpy): page_plan and
page_release entry for entry, the append against kv_append_rope's bits and a 64-bit rope and norm,
the attention over ragged batches, page sizes, windows and head layouts.

Attention tolerance, per output element: with A = softmax(q K^T) |V| the weights' rounding to bf16
(unit roundoff u = 2^-8) moves the sum by at most u A, the output's rounding by u |out| <= u A, and
fp32 sums and exponentials by far less than u A / 4: |got - want| <= (2 + 1/4) u A."""
import numpy as np
import pytest
import torch

from oracle import kv_path as O

pytestmark = pytest.mark.gpu

U = 2.0 ** -8


@pytest.fixture(scope="module")
def ops():
    from modelcore_b200 import ops
    return ops


@pytest.fixture(autouse=True)
def no_device_error(request, ops):
    ops.device_error()
    yield
    if "expects_device_error" not in request.fixturenames:
        code, what = ops.device_error()
        assert code == 0, what


@pytest.fixture
def expects_device_error():
    """Named by a test that reads the device errors itself."""


def i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def ceil_div(a, b):
    return -(-a // b)


# ---------------------------------------------------------------------------------------------
# page_plan / page_release
def plan_ref(cached, fresh, table, queue, state, page, n):
    cu, table, head = [0], table.copy(), state[0]
    pos, slots = np.full(n, -1, np.int64), np.full(n, -1, np.int64)
    for r, (a, b) in enumerate(zip(cached, fresh)):
        for j in range(ceil_div(a, page), ceil_div(a + b, page)):
            table[r, j] = queue[head % len(queue)]
            head += 1
        for t in range(b):
            if cu[-1] + t < n:
                pos[cu[-1] + t] = a + t
                slots[cu[-1] + t] = int(table[r, (a + t) // page]) * page + (a + t) % page
        cu.append(cu[-1] + b)
    return np.array(cu), pos, slots, table, np.array([head, state[1]])


def make_tables(rng, cached, page, width, spare, head0):
    """A block table holding every request's pages in shuffled order and the queue of the others."""
    held = [ceil_div(a, page) for a in cached]
    total = sum(held) + spare
    order = rng.permutation(total)
    table = np.full((len(cached), width), -1, np.int64)
    at = 0
    for r, n in enumerate(held):
        table[r, :n] = order[at:at + n]
        at += n
    queue = np.full(total, -1, np.int64)
    queue[(head0 + np.arange(spare)) % total] = order[at:]
    return table, queue, [head0, head0 + spare]


def run_plan(ops, cached, fresh, table, queue, state, page, n, stride_pad=0):
    wide = np.full((table.shape[0], table.shape[1] + stride_pad), 123456789)
    wide[:, :table.shape[1]] = table
    bt = i32(wide)[:, :table.shape[1]]
    st = torch.tensor(state, dtype=torch.int64, device="cuda")
    p = ops.page_plan(i32(cached), i32(fresh), bt, i32(queue), st, page_size=page, num_tokens=n)
    return p, bt, st


@pytest.mark.parametrize("cached,fresh,page,pad,head0,stride_pad", [
    ([0], [1], 16, 0, 0, 0),
    ([15, 16, 17], [1, 1, 1], 16, 0, 5, 3),
    ([0, 0, 31, 32, 33, 100], [0, 70, 1, 0, 32, 500], 32, 7, 10 ** 12 + 3, 1),
    ([], [], 16, 4, 0, 0),
    ([7], [0], 64, 0, 2, 0),
    (list(range(0, 1300)), [i % 5 for i in range(1300)], 16, 11, 77, 0),       # more than one scan of 1,024 rows
    ([i * 7 % 900 for i in range(2500)], [1 if i % 9 else 60 for i in range(2500)], 64, 1, 3, 2),
    ([3, 1000], [9000, 20000], 1024, 0, 1, 0),
])
def test_plan_matches_the_plain_one(ops, cached, fresh, page, pad, head0, stride_pad):
    rng = np.random.default_rng(len(cached) + page)
    width = max([ceil_div(a + b, page) for a, b in zip(cached, fresh)] + [1]) + 2
    need = sum(ceil_div(a + b, page) - ceil_div(a, page) for a, b in zip(cached, fresh))
    table, queue, state = make_tables(rng, cached, page, width, need + 3, head0)
    n = sum(fresh) + pad
    want = plan_ref(cached, fresh, table, queue, state, page, n)
    for _ in range(2):  # planning again from the same inputs gives the same step
        p, bt, st = run_plan(ops, cached, fresh, table, queue, state, page, n, stride_pad)
        for got, ref in zip((p.cu_new, p.positions, p.slot_map, bt, p.free_state), want):
            assert np.array_equal(got.cpu().numpy(), ref)
        assert st.tolist() == state and p.slot_map.dtype == torch.int64


def test_plan_and_release_in_place_over_many_steps(ops):
    """A life of a small cache: requests come, grow and go; the counters, lengths and tables are
    updated in place, and at every step no page belongs to two requests."""
    rng = np.random.default_rng(8)
    R, page, n_pages = 9, 16, 60
    table, queue = torch.full((R, 12), -1, dtype=torch.int32, device="cuda"), i32(rng.permutation(n_pages))
    state = torch.tensor([0, n_pages], dtype=torch.int64, device="cuda")
    lens = torch.zeros(R, dtype=torch.int32, device="cuda")
    for step in range(60):
        host = lens.cpu().numpy()
        done = (rng.random(R) < 0.2) | (host > 80)
        ops.page_release(i32(done.astype(int)), lens, table, queue, state, page_size=page, free_state_out=state,
                         seqlens_out=lens)
        host = np.where(done, 0, host)
        assert lens.tolist() == host.tolist()
        fresh = np.where(rng.random(R) < 0.3, rng.integers(0, 20, R), 1)
        before, q, s, bt = host, queue.cpu().numpy(), state.tolist(), table.cpu().numpy()
        p = ops.page_plan(lens, i32(fresh), table, queue, state, page_size=page, num_tokens=int(fresh.sum()) + 2,
                          free_state_out=state)
        want = plan_ref(before, fresh, bt, q, s, page, int(fresh.sum()) + 2)
        assert np.array_equal(table.cpu().numpy(), want[3]) and state.tolist() == want[4].tolist()
        assert np.array_equal(p.slot_map.cpu().numpy(), want[2])
        lens += i32(fresh)
        host = lens.cpu().numpy()
        owned = [int(x) for r in range(R) for x in table[r, :ceil_div(int(host[r]), page)].tolist()]
        free = [int(queue[x % n_pages]) for x in range(*state.tolist())]
        assert sorted(owned + free) == list(range(n_pages))


@pytest.mark.parametrize("R,lo,hi,page,every", [(1, 0, 0, 16, 1), (5, 0, 40, 16, 2), (1500, 0, 700, 32, 3),
                                                (40, 1, 30000, 16, 1), (64, 0, 100, 1024, 70)])
def test_release_matches_the_plain_one(ops, R, lo, hi, page, every):
    rng = np.random.default_rng(R)
    cached = rng.integers(lo, hi + 1, R)
    width = ceil_div(hi, page) + 1
    table, queue, state = make_tables(rng, cached, page, width, 4, 10 * R + 1)
    done = (np.arange(R) % every == 0).astype(int) * 3  # any non-zero value
    want_q, tail = queue.copy(), state[1]
    for r in range(R):
        for j in range(ceil_div(int(cached[r]), page) if done[r] else 0):
            want_q[tail % len(queue)] = table[r, j]
            tail += 1
    q = i32(queue)
    st, lens = ops.page_release(i32(done), i32(cached), i32(table), q, torch.tensor(state, device="cuda"),
                                page_size=page)
    assert np.array_equal(q.cpu().numpy(), want_q)
    assert st.tolist() == [state[0], tail]
    assert lens.tolist() == np.where(done != 0, 0, cached).tolist()


def test_plan_reports_what_does_not_fit(ops, expects_device_error):
    table, queue = np.full((2, 4), -1), np.arange(3)
    p, bt, _ = run_plan(ops, [0, 0], [20, 60], table, queue, [0, 3], 16, 80)  # six pages, three free
    assert ops.device_error()[0] == 5
    assert bt.tolist() == [[0, 1, -1, -1], [2, -1, -1, -1]] and p.free_state.tolist() == [3, 3]
    slots = p.slot_map.tolist()
    assert slots[:20] == list(range(20)) and slots[20:36] == list(range(32, 48)) and set(slots[36:]) == {-1}
    p, bt, _ = run_plan(ops, [60], [10], np.array([[5, 6, 7, 8]]), np.arange(20), [0, 20], 16, 10)
    assert ops.device_error()[0] == 1                                           # past the table's 64 positions
    assert p.slot_map.tolist() == [8 * 16 + 12 + i for i in range(4)] + [-1] * 6
    p, _, _ = run_plan(ops, [0], [5], np.full((1, 4), -1), np.arange(20), [0, 20], 16, 3)
    assert ops.device_error()[0] == 7 and p.slot_map.tolist() == [0, 1, 2] and p.cu_new.tolist() == [0, 5]
    run_plan(ops, [5], [1], np.full((1, 4), -1), np.arange(20), [0, 20], 16, 1)
    assert ops.device_error()[0] == 6                                           # a held page the table lacks


def test_plan_out_of_pages_over_many_ctas(ops, expects_device_error):
    """The CTAs that write slots and those that write table entries meet the queue's end in any order:
    what is reported is the queue's end, and the pages go to the first requests."""
    R, page, have = 900, 16, 1000
    fresh = [40] * R  # three pages each
    for _ in range(20):
        p, bt, _ = run_plan(ops, [0] * R, fresh, np.full((R, 4), -1), np.arange(have), [0, have], page, 40 * R)
        assert ops.device_error()[0] == 5
        assert p.free_state.tolist() == [have, have]
        k = np.arange(3 * R).reshape(R, 3)
        assert np.array_equal(bt.cpu().numpy()[:, :3], np.where(k < have, k, -1))
        t = np.arange(40 * R)
        k = t // 40 * 3 + t % 40 // page
        assert np.array_equal(p.slot_map.cpu().numpy(), np.where(k < have, k * page + t % 40 % page, -1))
    ops.page_release(i32([1]), i32([40]), i32([[1, 2, 3]]), i32(np.arange(4)),
                     torch.tensor([0, 3], device="cuda"), page_size=16)
    assert ops.device_error()[0] == 5                                           # three pages into room for one


# ---------------------------------------------------------------------------------------------
# the append
def tables(rot, D):
    cos, sin = O.rotary_tables(rot, D)
    as_dev = lambda b: torch.from_numpy(np.ascontiguousarray(b).view(np.int16)).view(torch.bfloat16).cuda()
    return as_dev(cos), as_dev(sin)


APPEND = [(1, 1, 1, 64, 16), (5, 4, 2, 128, 16), (37, 12, 12, 64, 32), (130, 16, 4, 128, 64), (1000, 15, 5, 128, 128),
          (3, 3, 1, 64, 1024)]


def append_inputs(N, Hq, Hkv, D, page, seed=0):
    g = torch.Generator("cuda").manual_seed(seed + N)
    qkv = torch.randn(N, Hq + 2 * Hkv, D, device="cuda", generator=g).mul_(2).to(torch.bfloat16)
    n_pages = ceil_div(N, page) + 2
    slots = torch.randperm(n_pages * page, device="cuda", generator=g)[:N]
    pos = torch.randint(0, 300, (N,), device="cuda", generator=g, dtype=torch.int32)
    pools = [torch.full((n_pages, Hkv, page, D), float("nan"), device="cuda", dtype=torch.bfloat16) for _ in range(2)]
    return qkv.split([Hq, Hkv, Hkv], 1), slots, pos, pools


@pytest.mark.parametrize("N,Hq,Hkv,D,page", APPEND)
def test_append_writes_the_bits_of_the_contiguous_append(ops, N, Hq, Hkv, D, page):
    (q, k, v), slots, pos, (kp, vp) = append_inputs(N, Hq, Hkv, D, page)
    cos, sin = tables(300, D)
    out = ops.paged_append_rope(q, k, v, kp, vp, pos, slots, cos, sin)
    # the same tokens as rows of a contiguous cache, one token a row
    kc = torch.zeros(N, 300, Hkv, D, device="cuda", dtype=torch.bfloat16)
    vc = torch.zeros_like(kc)
    want = ops.kv_append_rope(q[:, None], k[:, None], v[:, None], kc, vc, pos, cos, sin)
    assert torch.equal(out, want[:, 0])
    rows = torch.arange(N, device="cuda")
    for pool, cache in ((kp, kc), (vp, vc)):
        assert torch.equal(pool[slots // page, :, slots % page], cache[rows, pos.long()])
        untouched = torch.ones(pool.shape[0] * page, dtype=torch.bool, device="cuda")
        untouched[slots] = False
        assert pool.transpose(1, 2).reshape(-1, Hkv, D)[untouched].isnan().all()


@pytest.mark.parametrize("N,Hq,Hkv,D,page", APPEND)
def test_append_rounded_once_matches_64_bits(ops, N, Hq, Hkv, D, page):
    """One rounding: |got - want| <= u |want| (1 + 2^-8) + 2^-20 for fp32's share (a handful of fp32
    roundings, 2^-24 relative each, of terms at most |x| <= 2^4)."""
    (q, k, v), slots, pos, (kp, vp) = append_inputs(N, Hq, Hkv, D, page, 1)
    cos, sin = tables(300, D)
    out = ops.paged_append_rope(q, k, v, kp, vp, pos, slots, cos, sin, round_each=False)
    c, s = (x.double().cpu().numpy().reshape(-1, D // 2)[pos.cpu().numpy()][:, None] for x in (cos, sin))

    def ref(x):
        x = x.double().cpu().numpy()
        x1, x2 = x[..., :D // 2], x[..., D // 2:]
        y = np.concatenate([x1 * c + x2 * s, x2 * c - x1 * s], -1)
        return 1.2 * y / np.sqrt((y * y).mean(-1, keepdims=True) + np.finfo(np.float32).eps)

    for got, want in ((out, ref(q)), (kp[slots // page, :, slots % page], ref(k))):
        err = np.abs(got.double().cpu().numpy() - want)
        assert (err <= U * np.abs(want) * (1 + U) + 2.0 ** -20).all(), err.max()
    assert torch.equal(vp[slots // page, :, slots % page], v)


def test_append_skips_padding_and_reads_only_q_when_told(ops):
    (q, k, v), slots, pos, (kp, vp) = append_inputs(40, 8, 2, 128, 16, 2)
    cos, sin = tables(300, 128)
    full = ops.paged_append_rope(q, k, v, kp.clone(), vp.clone(), pos, slots, cos, sin)
    keep_k = kp.clone()
    pos2, slots2 = pos.clone(), slots.clone()
    pos2[30:], slots2[25:] = -1, -1
    out = ops.paged_append_rope(q, k, v, kp, vp, pos2, slots2, cos, sin)
    assert torch.equal(out[:30], full[:30]) and not out[30:].any()
    assert kp.transpose(1, 2).reshape(-1, 2, 128)[slots[25:]].isnan().all()
    only_q = ops.paged_append_rope(q, None, None, None, None, pos, None, cos, sin)
    assert torch.equal(only_q, full)
    raw = ops.paged_append_rope(q, k, v, keep_k, vp, pos, slots, cos, sin, rotate_k=False)
    assert torch.equal(raw, full) and torch.equal(keep_k[slots // 16, :, slots % 16], k)
    assert ops.paged_append_rope(q[:0], k[:0], v[:0], kp, vp, pos[:0], slots[:0], cos, sin).shape == (0, 8, 128)


def test_append_reports_slots_and_positions_out_of_range(ops, expects_device_error):
    (q, k, v), slots, pos, (kp, vp) = append_inputs(10, 4, 2, 64, 16, 3)
    cos, sin = tables(300, 64)
    bad = slots.clone()
    bad[3] = kp.shape[0] * 16
    ops.paged_append_rope(q, k, v, kp, vp, pos, bad, cos, sin)
    assert ops.device_error()[0] == 6
    far = pos.clone()
    far[4] = 300
    out = ops.paged_append_rope(q, k, v, kp, vp, far, slots, cos, sin)
    assert ops.device_error()[0] == 2 and not out[4].any()


# ---------------------------------------------------------------------------------------------
# the attention
def attn_case(cached, fresh, Hq, Hkv, D, page, seed=0, spare=3, poison=float("nan"), extra=0, tail=0, pool_pages=None):
    """Packed q, pools whose every position no request owns holds `poison`, and the block table."""
    g = torch.Generator("cuda").manual_seed(seed)
    held = [ceil_div(a + b, page) for a, b in zip(cached, fresh)]
    width, total = max(held + [1]) + extra, pool_pages or sum(held) + spare
    first = total - sum(held) - 1 if pool_pages else 0
    order = first + torch.randperm(sum(held) + 1, generator=torch.Generator().manual_seed(seed)).numpy()
    table = np.full((len(cached), width), 2 ** 31 - 1)  # entries past a request's pages are never read
    q = torch.randn(sum(fresh) + tail, Hq + 2, D, device="cuda", generator=g).to(torch.bfloat16)[:, :Hq]
    make = torch.empty if pool_pages else (lambda *a, **k: torch.full(*a, poison, **k))
    kp, vp = (make((total, Hkv, page, D), device="cuda", dtype=torch.bfloat16) for _ in range(2))
    at = 0
    ks, vs = [], []
    for r, (a, b) in enumerate(zip(cached, fresh)):
        pages = order[at:at + held[r]]
        at += held[r]
        table[r, :held[r]] = pages
        k, v = (torch.randn(a + b, Hkv, D, device="cuda", generator=g).to(torch.bfloat16) for _ in range(2))
        for pool, x in ((kp, k), (vp, v)):
            c = torch.arange(a + b, device="cuda")
            pool[torch.from_numpy(pages).cuda()[c // page], :, c % page] = x
        ks.append(k)
        vs.append(v)
    cu = np.concatenate([[0], np.cumsum(fresh)])
    return dict(q=q, kp=kp, vp=vp, table=i32(table), cached=i32(cached), cu=i32(cu)), ks, vs


def attn_ref(q, ks, vs, cached, fresh, window, scale=None):
    """(out, A) in 64 bits."""
    N, Hq, D = q.shape
    out, bound = np.zeros((N, Hq, D)), np.zeros((N, Hq, D))
    at = 0
    q = q.double()
    for a, b, k, v in zip(cached, fresh, ks, vs):
        if b == 0:
            continue
        G = Hq // k.shape[1]
        k, v = (x.double().repeat_interleave(G, 1) for x in (k, v))
        pos = torch.arange(a, a + b, device="cuda")[:, None]
        key = torch.arange(a + b, device="cuda")[None]
        seen = (key <= pos) & ((pos - key <= window) if window >= 0 else True)
        s = torch.einsum("thd,chd->htc", q[at:at + b], k) * (D ** -0.5 if scale is None else scale)
        w = torch.softmax(s.masked_fill(~seen, -np.inf), -1)
        out[at:at + b] = torch.einsum("htc,chd->thd", w, v).cpu().numpy()
        bound[at:at + b] = torch.einsum("htc,chd->thd", w, v.abs()).cpu().numpy()
        at += b
    return out, bound


def check_attn(ops, cached, fresh, Hq, Hkv, D, page, window=-1, hints=(0,), scale=None, **kw):
    c, ks, vs = attn_case(cached, fresh, Hq, Hkv, D, page, **kw)
    want, bound = attn_ref(c["q"], ks, vs, cached, fresh, window, scale)
    for hint in hints:
        got = ops.paged_attn(c["q"], c["kp"], c["vp"], c["table"], c["cached"], c["cu"], window=window,
                             max_new=hint, softmax_scale=scale)
        assert got.is_contiguous() and got.shape == c["q"].shape
        err = np.abs(got.double().cpu().numpy() - want)
        worst = (err - 2.25 * U * bound).max() if err.size else 0.0
        assert np.isfinite(err).all() and worst <= 0, (hint, worst, np.unravel_index(np.nanargmax(err), err.shape))
    return c


RAGGED = ([0, 1, 15, 16, 63, 64, 127, 200, 511, 0], [1, 1, 1, 17, 1, 2, 0, 3, 1, 0])
HEADS = [(1, 1, 64), (12, 12, 64), (4, 2, 128), (16, 4, 128), (3, 1, 64), (15, 5, 128), (32, 1, 128), (10, 2, 64),
         (128, 1, 64)]


@pytest.mark.parametrize("Hq,Hkv,D", HEADS)
@pytest.mark.parametrize("window", [-1, 0, 20, 64])
def test_attention_over_short_ragged_chunks(ops, Hq, Hkv, D, window):
    check_attn(ops, *RAGGED, Hq, Hkv, D, 16, window, hints=(0, 17), tail=3, extra=2)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256, 1024])
@pytest.mark.parametrize("Hq,Hkv,D", [(12, 12, 64), (8, 2, 128)])
def test_attention_over_every_page_size(ops, page, Hq, Hkv, D):
    check_attn(ops, [0, 700, 1023, 129], [300, 1, 2, 65], Hq, Hkv, D, page, -1)
    check_attn(ops, [0, 700, 1023, 129], [300, 1, 2, 65], Hq, Hkv, D, page, 100)


@pytest.mark.parametrize("cached", [[n] for n in (0, 1, 62, 63, 64, 127, 128, 129, 1000, 5000)] +
                         [[0, 4999], list(range(0, 700, 10)), [3000] * 33])
@pytest.mark.parametrize("Hq,Hkv,D", [(12, 12, 64), (16, 4, 128), (15, 5, 128)])
def test_single_token_steps(ops, cached, Hq, Hkv, D):
    """The serving form: one new token a request, the hint given and not."""
    check_attn(ops, cached, [1] * len(cached), Hq, Hkv, D, 32, -1, hints=(1, 0))
    check_attn(ops, cached, [1] * len(cached), Hq, Hkv, D, 32, 130, hints=(1,))


@pytest.mark.parametrize("fresh", [1, 2, 4, 5, 16, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 600])
@pytest.mark.parametrize("Hq,Hkv,D,window", [(16, 4, 128, -1), (16, 4, 128, 90), (6, 6, 64, -1), (5, 1, 64, 300)])
def test_chunk_lengths_around_the_tiles(ops, fresh, Hq, Hkv, D, window):
    check_attn(ops, [0, 333], [fresh, fresh], Hq, Hkv, D, 64, window, hints=(0, fresh))


def test_a_mixed_batch_of_many_requests(ops):
    rng = np.random.default_rng(1)
    cached = rng.integers(0, 900, 150).tolist()
    fresh = [1 if i % 7 else int(rng.integers(0, 200)) for i in range(150)]
    check_attn(ops, cached, fresh, 16, 4, 128, 16, -1)
    check_attn(ops, cached, fresh, 12, 12, 64, 64, 256)


def test_a_hint_that_is_too_small_costs_speed_only(ops):
    check_attn(ops, [10, 0, 500], [1, 40, 300], 16, 4, 128, 16, -1, hints=(1,))


def test_the_rows_do_not_see_what_lies_outside_them(ops):
    """Infinities and NaN before the window, after the last position and in pages nobody owns."""
    for poison in (float("inf"), float("-inf"), float("nan")):
        c = check_attn(ops, [300, 5, 1000], [1, 70, 3], 8, 2, 128, 16, 50, poison=poison)
        before = ops.paged_attn(c["q"], c["kp"], c["vp"], c["table"], c["cached"], c["cu"], window=50)
        t = c["table"].long()
        for r, lo in ((0, 300 - 50), (2, 1000 - 50)):  # pages wholly before the window, and the
            for pool in (c["kp"], c["vp"]):            # positions of its first page before it
                pool[t[r, :lo // 16]] = poison
                pool[t[r, lo // 16], :, :lo % 16] = poison
        after = ops.paged_attn(c["q"], c["kp"], c["vp"], c["table"], c["cached"], c["cu"], window=50)
        assert torch.equal(before, after)


def test_large_scores_and_a_given_scale(ops):
    check_attn(ops, [130, 700], [1, 90], 8, 2, 128, 32, -1, scale=1.0)
    check_attn(ops, [130, 700], [1, 90], 8, 2, 64, 32, -1, scale=3.0)
    check_attn(ops, [130, 700], [1, 90], 8, 2, 64, 32, -1, scale=1e-4)


SPIKES = {
    # score of key c when q's first element is +1 (integers exact in bf16, times the scale)
    "one key of a first half": lambda c: 60.0 * (c == 390),
    "one key of a second half": lambda c: 60.0 * (c == 450),
    "a jump inside a first half": lambda c: 60.0 * (c >= 400),
    "a jump inside a second half": lambda c: 60.0 * (c >= 500),
    "a step every 64 keys": lambda c: 40.0 * (c // 64),
    "a step every 128 keys": lambda c: 40.0 * (c // 128),
    "up and down": lambda c: 50.0 * ((c // 64) % 3),
    "the last keys of the cache": lambda c: 60.0 * (c >= 636),
}


@pytest.mark.parametrize("pattern", SPIKES)
@pytest.mark.parametrize("D,G,fresh", [(128, 4, 100), (64, 1, 300), (128, 8, 1), (64, 4, 5)])
def test_scores_that_leap_by_hundreds(ops, pattern, D, G, fresh):
    """Far more than an exponential's range between one block of keys and the next: every running
    reference has to move, for some rows and not for others (q's first element is +1, 0 or -1)."""
    cached = 640
    c, ks, vs = attn_case([cached], [fresh], 2 * G, 2, D, 64, seed=3)
    key = torch.arange(cached + fresh, device="cuda")
    ks[0][..., 0] = SPIKES[pattern](key).to(torch.bfloat16)[:, None]
    sign = (torch.arange(fresh, device="cuda") % 3 - 1).to(torch.bfloat16)[:, None]
    q = c["q"].contiguous().mul(0.25)
    q[..., 0] = sign
    page = c["table"][0].long()
    c["kp"][page[key // 64], :, key % 64] = ks[0]
    scale = 8.0
    want, bound = attn_ref(q, ks, vs, [cached], [fresh], -1, scale)
    got = ops.paged_attn(q, c["kp"], c["vp"], c["table"], c["cached"], c["cu"], softmax_scale=scale)
    err = np.abs(got.double().cpu().numpy() - want)
    # a score of s = 480 is a sum of fp32 products: off by up to s 2^-20, its weight by that relatively
    slack = (2.25 * U + 8.0 * 480 * 2.0 ** -20) * bound
    assert np.isfinite(err).all() and (err <= slack).all(), (err - slack).max()


@pytest.mark.parametrize("D,G,fresh", [(128, 4, 200), (64, 1, 300), (128, 4, 1), (64, 12, 1)])
def test_what_a_row_sees_reaches_it(ops, D, G, fresh):
    """A NaN key makes the rows that see it NaN and no others; an infinite value is infinite there."""
    cached = 300
    for at, what in ((100, "k"), (310, "k"), (20, "v"), (299, "v")):
        if at >= cached + fresh:
            continue
        c, ks, vs = attn_case([cached, 50], [fresh, 3], 2 * G, 2, D, 32, seed=at)
        page = c["table"][0].long()
        pool = c["kp"] if what == "k" else c["vp"]
        pool[page[at // 32], :, at % 32] = float("nan") if what == "k" else float("inf")
        got = ops.paged_attn(c["q"], c["kp"], c["vp"], c["table"], c["cached"], c["cu"]).float()
        sees = torch.arange(cached, cached + fresh, device="cuda") >= at
        assert got[fresh:].isfinite().all()
        if what == "k":
            assert torch.equal(got[:fresh].isnan().all(-1).all(-1), sees)
            assert got[:fresh][~sees].isfinite().all()
        else:
            assert (got[:fresh][sees] == float("inf")).all()


def test_pages_beyond_32_bit_offsets(ops):
    """A pool of more than 2^31 elements, the requests' pages at its end."""
    pages = (1 << 31) // (2 * 64 * 128) + 200
    check_attn(ops, [400, 3], [1, 150], 4, 2, 128, 64, -1, pool_pages=pages)
    cos, sin = tables(64, 128)
    kp = torch.empty(pages, 2, 64, 128, device="cuda", dtype=torch.bfloat16)
    k = torch.randn(3, 2, 128, device="cuda").to(torch.bfloat16)
    slots = torch.tensor([pages * 64 - 1, pages * 64 - 64, 5], device="cuda")
    pos = torch.tensor([1, 2, 3], dtype=torch.int32, device="cuda")
    ops.paged_append_rope(k, k, k, torch.empty_like(kp), kp, pos, slots, cos, sin)
    assert torch.equal(kp[slots // 64, :, slots % 64], k)


def test_empty_batches(ops):
    c, _, _ = attn_case([5, 9], [1, 1], 4, 2, 64, 16)
    none = ops.paged_attn(c["q"][:0], c["kp"], c["vp"], c["table"], c["cached"], i32([0, 0, 0]))
    assert none.shape == (0, 4, 64)
    out = ops.paged_attn(c["q"], c["kp"], c["vp"], c["table"], c["cached"], i32([0, 0, 0]))
    assert not out.any()  # only padding
    out = ops.paged_attn(c["q"], c["kp"], c["vp"], c["table"][:0], c["cached"][:0], i32([0]))
    assert not out.any()


def test_attention_reports_bad_tables_and_lengths(ops, expects_device_error):
    c, _, _ = attn_case([40, 9], [1, 20], 4, 2, 64, 16)
    args = (c["q"], c["kp"], c["vp"])
    bad = c["table"].clone()
    bad[0, 1] = c["kp"].shape[0]
    ops.paged_attn(*args, bad, c["cached"], c["cu"])
    assert ops.device_error()[0] == 6
    bad[0, 1] = -1
    ops.paged_attn(*args, bad, c["cached"], c["cu"])
    assert ops.device_error()[0] == 6
    ops.paged_attn(*args, c["table"][:, :2].contiguous(), c["cached"], c["cu"])
    assert ops.device_error()[0] == 1
    ops.paged_attn(*args, c["table"], i32([-3, 9]), c["cu"])
    assert ops.device_error()[0] == 1
    c["kp"].nan_to_num_(0.0)
    c["vp"].nan_to_num_(0.0)
    good = ops.paged_attn(*args, c["table"], c["cached"], c["cu"])
    assert ops.device_error()[0] == 0 and good.isfinite().all()


def test_a_captured_step_follows_its_lengths(ops):
    """plan + append + attention in a CUDA graph, replayed as the lengths grow, against the same
    calls made eagerly."""
    Hq, Hkv, D, page, R = 8, 2, 128, 16, 3
    cos, sin = tables(400, D)
    g = torch.Generator("cuda").manual_seed(5)
    qkv = torch.randn(R, Hq + 2 * Hkv, D, device="cuda", generator=g).to(torch.bfloat16)
    q, k, v = qkv.split([Hq, Hkv, Hkv], 1)

    def fresh_state():
        return dict(lens=i32([0, 90, 300]), table=i32(np.arange(R * 30).reshape(R, 30)),
                    queue=i32(np.concatenate([np.arange(90, 180), np.full(90, -1)])), state=torch.tensor([0, 90], device="cuda"),
                    kp=torch.randn(180, Hkv, page, D, device="cuda", generator=torch.Generator("cuda").manual_seed(1)
                                   ).to(torch.bfloat16),
                    vp=torch.randn(180, Hkv, page, D, device="cuda", generator=torch.Generator("cuda").manual_seed(2)
                                   ).to(torch.bfloat16))

    ones = i32([1] * R)

    def step(s):
        p = ops.page_plan(s["lens"], ones, s["table"], s["queue"], s["state"], page_size=page, num_tokens=R,
                          free_state_out=s["state"])
        qr = ops.paged_append_rope(q, k, v, s["kp"], s["vp"], p.positions, p.slot_map, cos, sin)
        out = ops.paged_attn(qr, s["kp"], s["vp"], s["table"], s["lens"], p.cu_new, max_new=1)
        ops.kv_advance(s["lens"], 1)
        return out

    eager = fresh_state()
    want = [step(eager).clone() for _ in range(40)]
    s = fresh_state()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(s)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(s)
    for name, x in fresh_state().items():
        s[name].copy_(x)
    for w in want:
        graph.replay()
        assert torch.equal(out, w)
    assert torch.equal(s["kp"], eager["kp"]) and s["state"].tolist() == eager["state"].tolist()


def test_two_streams_at_once(ops):
    c1, _, _ = attn_case([3000] * 4, [1] * 4, 16, 4, 128, 16, seed=1)
    c2, _, _ = attn_case([2000] * 3, [40] * 3, 16, 4, 128, 64, seed=2)
    call = lambda c: ops.paged_attn(c["q"], c["kp"], c["vp"], c["table"], c["cached"], c["cu"])
    want = call(c1), call(c2)
    torch.cuda.synchronize()
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    got = [[], []]
    for _ in range(20):
        for i, c in enumerate((c1, c2)):
            with torch.cuda.stream(streams[i]):
                got[i].append(call(c))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


# ---------------------------------------------------------------------------------------------
# refusals
def test_what_is_refused(ops):
    c, _, _ = attn_case([5, 49], [1, 3], 4, 2, 64, 16)
    call = lambda **kw: ops.paged_attn(*({**c, **{k: v for k, v in kw.items() if k in c}}[k] for k in
                                         ("q", "kp", "vp", "table", "cached", "cu")),
                                       **{k: v for k, v in kw.items() if k not in c})
    call()
    bad = [dict(q=c["q"].float()), dict(q=c["q"].cpu()), dict(q=c["q"][0]), dict(q=c["q"].transpose(1, 2)),
           dict(q=c["q"][:, :3]), dict(q=c["q"][..., :32]), dict(kp=c["kp"][:, :, :8].contiguous()),
           dict(kp=c["kp"].transpose(1, 2)), dict(kp=c["kp"].half()), dict(vp=c["vp"][:1]),
           dict(table=c["table"].long()), dict(table=c["table"][:1]), dict(table=c["table"].t().contiguous().t()),
           dict(cached=c["cached"][:1]), dict(cached=c["cached"].cpu()), dict(cu=c["cu"][:2]), dict(cu=c["cu"].long()),
           dict(softmax_scale=0.0), dict(softmax_scale=-1.0), dict(softmax_scale=float("nan")), dict(max_new=-1)]
    D96 = torch.zeros(4, 4, 96, device="cuda", dtype=torch.bfloat16)
    P96 = torch.zeros(8, 2, 16, 96, device="cuda", dtype=torch.bfloat16)
    bad += [dict(q=D96, kp=P96, vp=P96)]
    P24 = torch.zeros(8, 2, 24, 64, device="cuda", dtype=torch.bfloat16)
    bad += [dict(kp=P24, vp=P24)]
    odd = torch.zeros(4 * 4 * 65, device="cuda", dtype=torch.bfloat16).as_strided((4, 4, 64), (260, 65, 1))
    bad += [dict(q=odd)]
    for kw in bad:
        with pytest.raises(RuntimeError):
            call(**kw)
    (q, k, v), slots, pos, (kp, vp) = append_inputs(6, 4, 2, 64, 16)
    cos, sin = tables(300, 64)
    ok = [q, k, v, kp, vp, pos, slots, cos, sin]
    for i, x in ((0, q.half()), (1, k[:, :1]), (1, None), (2, v[:3]), (3, kp.half()), (4, vp[:, :, :8]), (5, pos.long()),
                 (5, pos[:3]), (6, slots.int()), (6, None), (7, cos.float()), (8, sin[:, :16].contiguous()),
                 (7, cos[:100].contiguous())):
        with pytest.raises(RuntimeError):
            ops.paged_append_rope(*ok[:i], x, *ok[i + 1:])
    st = torch.tensor([0, 9], device="cuda")
    plan = dict(cache_seqlens=i32([1, 2]), new_lens=i32([1, 1]), block_table=i32([[1, 2], [3, 4]]),
                free_pages=i32(range(9)), free_state=st)
    ops.page_plan(*plan.values(), page_size=16, num_tokens=2)
    for kw in (dict(new_lens=i32([1])), dict(new_lens=plan["new_lens"].long()), dict(block_table=i32([[1, 2]])),
               dict(free_state=st.int()), dict(free_state=st[:1]), dict(free_pages=i32([])),
               dict(cache_seqlens=plan["cache_seqlens"].cpu())):
        with pytest.raises(RuntimeError):
            ops.page_plan(*{**plan, **kw}.values(), page_size=16, num_tokens=2)
    for kw in (dict(page_size=8), dict(page_size=48), dict(page_size=2048), dict(num_tokens=-1)):
        with pytest.raises(RuntimeError):
            ops.page_plan(*plan.values(), **{**dict(page_size=16, num_tokens=2), **kw})
    with pytest.raises(RuntimeError):
        ops.page_release(i32([1]), *[plan[k] for k in ("cache_seqlens", "block_table", "free_pages", "free_state")],
                         page_size=16)
