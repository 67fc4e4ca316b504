"""Trees of drafted tokens over the paged cache against plain implementations in 64 bits: positions and
masks, attention, verification, the kept path's move, and rows that share pages.

Attention tolerance, per output element: as in test_gpu_paged.py -- with A = softmax(q K^T) |V| over the
keys a row sees, the weights' rounding to bf16 (unit roundoff u = 2^-8) moves the sum by at most u A, the
output's rounding by u |out| <= u A, fp32 sums and exponentials by far less than u A / 4."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -8
NEG = -math.inf


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


def offsets(lens):
    return np.concatenate([[0], np.cumsum(lens)]).astype(int)


def random_parents(rng, n, kind="any"):
    if kind == "chain":
        return [t - 1 for t in range(n)]
    if kind == "roots":
        return [-1] * n
    return [-1 if t == 0 else int(rng.integers(-1 if kind == "forest" else 0, t)) for t in range(n)]


# ---------------------------------------------------------------------------------------------
# draft_tree
def tree_ref(cached, parents, words):
    """Of one request: positions and rows of bits."""
    n = len(parents)
    if n > 32 * words:
        return [cached + t for t in range(n)], np.zeros((n, 32 * words), bool)
    bits, pos = np.zeros((n, 32 * words), bool), []
    for t, p in enumerate(parents):
        if p >= 0:
            bits[t] = bits[p]
        bits[t, t] = True
        pos.append(cached + int(bits[t].sum()) - 1)
    return pos, bits


def pack(bits):
    return np.packbits(bits, axis=-1, bitorder="little").view(np.int32).reshape(bits.shape[0], bits.shape[1] // 32)


@pytest.mark.parametrize("fresh,max_tree,kind", [
    ([1], 1, "any"), ([0, 5, 0], 32, "any"), ([32, 33, 31, 64], 64, "any"), ([7, 300, 8], 40, "any"),
    ([256, 257, 1, 255], 256, "any"), ([100, 200], 256, "chain"), ([96, 3], 96, "roots"), ([50] * 40, 160, "forest"),
    (list(range(1200)), 192, "any"), ([], 32, "any"), ([129], 129, "any"),
])
def test_tree_positions_and_masks(ops, fresh, max_tree, kind):
    rng = np.random.default_rng(len(fresh) + max_tree)
    cached = [int(rng.integers(0, 5000)) for _ in fresh]
    parents = [random_parents(rng, n, kind) for n in fresh]
    words, pad = ceil_div(max_tree, 32), 3
    pos, masks = [], [np.zeros((0, words), np.int32)]
    for c, p in zip(cached, parents):
        a, b = tree_ref(c, p, words)
        pos += a
        masks.append(pack(b))
    flat = sum(parents, []) + [-1] * pad
    t = ops.draft_tree(i32(flat).reshape(-1), i32(offsets(fresh)), i32(cached).reshape(-1), max_tree=max_tree)
    assert t.positions.tolist() == pos + [-1] * pad
    assert np.array_equal(t.mask.cpu().numpy(), np.concatenate(masks + [np.zeros((pad, words), np.int32)]))


def test_tree_reports_parents_that_are_no_earlier_tokens(ops, expects_device_error):
    for bad in (2, 9, -2, 1 << 30, -(1 << 31)):
        t = ops.draft_tree(i32([-1, 0, bad, 2]), i32([0, 4]), i32([10]), max_tree=32)
        assert ops.device_error()[0] == 8
        assert t.positions.tolist() == [10, 11, 10, 11] and t.mask.flatten().tolist() == [1, 3, 4, 12]


def test_tree_positions_stop_at_31_bits(ops):
    t = ops.draft_tree(i32([-1, 0, 1]), i32([0, 3]), i32([2 ** 31 - 2]), max_tree=32)
    assert t.positions.tolist() == [2 ** 31 - 2, 2 ** 31 - 1, 2 ** 31 - 1]


def test_tokens_before_the_first_request(ops):
    t = ops.draft_tree(i32([5, 5, -1, 0, 7]), i32([2, 4]), i32([10]), max_tree=64)
    assert t.positions.tolist() == [-1, -1, 10, 11, -1]
    assert t.mask.tolist() == [[0, 0], [0, 0], [1, 0], [3, 0], [0, 0]]


# ---------------------------------------------------------------------------------------------
# paged_tree_attn
def attn_case(cached, fresh, parents, Hq, Hkv, D, page, max_tree, seed=0, poison=None, masks=None, spare=4):
    """A batch of requests with their keys and values in pages in shuffled order; what no request holds, and
    the last pages' positions past their ends, are `poison`."""
    g = torch.Generator("cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, device="cuda", dtype=torch.bfloat16, generator=g)
    R, cu, words = len(cached), offsets(fresh), ceil_div(max_tree, 32)
    counts = [ceil_div(a + b, page) for a, b in zip(cached, fresh)]
    n_pages = sum(counts) + spare
    order = torch.randperm(n_pages, device="cuda", generator=g)
    table = torch.full((R, max(counts + [1]) + 2), -1, device="cuda", dtype=torch.int32)
    fill = 0.0 if poison is None else poison
    kp = torch.full((n_pages, Hkv, page, D), fill, device="cuda", dtype=torch.bfloat16)
    vp = kp.clone()
    ks, vs, at = [], [], 0
    for r, n in enumerate(counts):
        table[r, :n] = order[at:at + n].to(torch.int32)
        at += n
        k, v = rand(cached[r] + fresh[r], Hkv, D), rand(cached[r] + fresh[r], Hkv, D)
        c = torch.arange(k.shape[0], device="cuda")
        kp[table[r, :n].long()[c // page], :, c % page] = k
        vp[table[r, :n].long()[c // page], :, c % page] = v
        ks.append(k)
        vs.append(v)
    if masks is None:
        both = [tree_ref(c, p, words) for c, p in zip(cached, parents)]
        pos, bits = [b[0] for b in both], [b[1] for b in both]
    else:
        pos, bits = masks
    q = rand(int(cu[-1]) + 2, Hq, 2 * D)[..., :D]  # (two padding tokens, strided rows)
    none = [np.zeros((0, 32 * words), bool)]
    packed = np.concatenate([pack(b) for b in bits + none] + [np.zeros((2, words), np.int32)])
    return dict(q=q, kp=kp, vp=vp, table=table, cached=i32(cached).reshape(-1), cu=i32(cu), ks=ks, vs=vs,
                pos=i32(sum(pos, []) + [-1, -1]).reshape(-1), mask=torch.from_numpy(packed).cuda(), words=words, bits=bits,
                positions=pos)


def attn_ref(c, cached, fresh, window, scale):
    """(want, bound) of the tokens that requests have, in 64 bits."""
    want, bound, at = [], [], 0
    for r, (a, b) in enumerate(zip(cached, fresh)):
        q = c["q"][at:at + b].double()
        at += b
        group = q.shape[1] // c["ks"][r].shape[1]
        k, v = (x.double().repeat_interleave(group, 1) for x in (c["ks"][r], c["vs"][r]))
        seen = torch.zeros(b, a + b, dtype=torch.bool, device="cuda")
        seen[:, :a] = True
        pos = torch.tensor(c["positions"][r], device="cuda", dtype=torch.long).clamp(min=a)
        if b > 32 * c["words"]:
            seen[:, a:] = torch.ones(b, b, device="cuda").tril() > 0
            pos = a + torch.arange(b, device="cuda")
        else:
            seen[:, a:] = torch.from_numpy(c["bits"][r][:, :b]).cuda()
        if window >= 0:
            where = torch.cat([torch.arange(a, device="cuda"), pos])
            seen &= pos[:, None] - where[None] <= window
        s = torch.einsum("thd,chd->thc", q, k) * scale
        s = s.masked_fill(~seen[:, None], NEG)
        w = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e300))
        w = w / w.sum(-1, keepdim=True).clamp(min=1e-300)
        want.append(torch.einsum("thc,chd->thd", w, v))
        bound.append(torch.einsum("thc,chd->thd", w, v.abs()))
    return torch.cat(want), torch.cat(bound)


def check_attn(ops, cached, fresh, Hq, Hkv, D, page, window=-1, max_tree=64, kind="any", scale=None, hints=None, seed=0,
               poison=None, masks=None, parents=None):
    rng = np.random.default_rng(seed)
    if parents is None:
        parents = [random_parents(rng, n, kind) for n in fresh]
    c = attn_case(cached, fresh, parents, Hq, Hkv, D, page, max_tree, seed, poison, masks)
    want, bound = attn_ref(c, cached, fresh, window, scale or D ** -0.5)
    for hint in hints or (max(fresh), 0):
        got = ops.paged_tree_attn(c["q"], c["kp"], c["vp"], c["table"], c["cached"], c["cu"], c["pos"], c["mask"],
                                  window=window, softmax_scale=scale, max_new=hint)
        assert not got[-2:].any()
        err = (got[:-2].double() - want).abs()
        assert err.isfinite().all()
        slack = 2.25 * U * bound + 1e-30
        assert (err <= slack).all(), f"hint {hint}: {(err / slack).max()} of the bound"
    return c


HEADS = [(12, 12, 64), (16, 4, 128), (6, 2, 64), (15, 5, 128), (8, 1, 64), (2, 2, 128), (128, 1, 128), (40, 1, 64)]


@pytest.mark.parametrize("Hq,Hkv,D", HEADS)
@pytest.mark.parametrize("page", [16, 64, 128])
def test_attention_of_ragged_trees(ops, Hq, Hkv, D, page):
    check_attn(ops, [0, 1, 127, 128, 129, 700, 33], [5, 1, 16, 9, 33, 64, 0], Hq, Hkv, D, page)


@pytest.mark.parametrize("n", [1, 2, 7, 8, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256])
@pytest.mark.parametrize("Hq,Hkv,D", [(4, 4, 128), (8, 2, 128), (8, 1, 64)])
def test_tree_sizes_around_the_tiles(ops, n, Hq, Hkv, D):
    check_attn(ops, [0, 300], [n, n], Hq, Hkv, D, 32, max_tree=256)


@pytest.mark.parametrize("past", [0, 1, 63, 64, 65, 111, 112, 113, 120, 127, 128, 129, 255, 256, 1000])
@pytest.mark.parametrize("D", [64, 128])
def test_cached_lengths_around_the_tiles(ops, past, D):
    check_attn(ops, [past, past + 1], [16, 5], 8, 2, D, 16)


@pytest.mark.parametrize("window", [0, 1, 3, 60, 128, 1000])
@pytest.mark.parametrize("kind", ["any", "chain", "forest"])
@pytest.mark.parametrize("Hq,Hkv,D", [(16, 4, 128), (6, 6, 64)])
def test_windows(ops, window, kind, Hq, Hkv, D):
    check_attn(ops, [0, 2, 200, 500], [20, 64, 40, 3], Hq, Hkv, D, 32, window=window, kind=kind)


@pytest.mark.parametrize("Hq,Hkv,D", [(16, 4, 128), (12, 12, 64), (64, 2, 64)])
@pytest.mark.parametrize("window", [-1, 100])
def test_trees_beside_prompt_chunks(ops, Hq, Hkv, D, window):
    check_attn(ops, [0, 300, 40, 7], [33, 20, 400, 1], Hq, Hkv, D, 16, window=window, max_tree=32, hints=(400, 0))


def test_a_hint_that_is_too_small_costs_speed_only(ops):
    check_attn(ops, [10, 0, 500], [1, 40, 300], 16, 4, 128, 16, hints=(1, 40), max_tree=64)


def test_many_requests(ops):
    rng = np.random.default_rng(1)
    cached = rng.integers(0, 1500, 150).tolist()
    fresh = [int(rng.integers(0, 30)) for _ in cached]
    check_attn(ops, cached, fresh, 16, 4, 128, 16)
    check_attn(ops, cached, fresh, 12, 12, 64, 64, window=256)


def test_long_requests_cut_between_many_blocks(ops):
    check_attn(ops, [20000], [63], 8, 2, 128, 64)
    check_attn(ops, [30011, 5], [9, 2], 4, 1, 64, 16)
    check_attn(ops, [12345, 9000], [100, 250], 8, 1, 128, 32, max_tree=256)


@pytest.mark.parametrize("Hq,Hkv,D,fresh", [(16, 4, 128, 5), (16, 4, 128, 30), (16, 4, 128, 63), (4, 4, 64, 14),
                                            (8, 8, 64, 30), (12, 6, 64, 64), (32, 4, 128, 3), (6, 6, 128, 1)])
@pytest.mark.parametrize("page", [16, 128])
def test_long_runs_of_tiles(ops, Hq, Hkv, D, fresh, page):
    """Some 25 tiles a block in one or two runs: every stage of its rings turns many times."""
    check_attn(ops, [20000, 17777, 23456, 20001], [fresh] * 4, Hq, Hkv, D, page)


@pytest.mark.parametrize("Hq,Hkv,D,fresh", [(8, 1, 64, 2), (8, 1, 128, 2), (8, 1, 64, 20), (4, 4, 128, 20)])
def test_positions_up_to_31_bits(ops, Hq, Hkv, D, fresh):
    """The last tokens that a table of 1,024-position pages can hold, their window's pages the only real ones."""
    page, window = 1024, 700
    width = (2 ** 31 - 1) // page
    past = width * page - fresh
    parents = random_parents(np.random.default_rng(1), fresh)
    first = past - past % page - page  # the first position that has a page of its own
    c = attn_case([past - first], [fresh], [parents], Hq, Hkv, D, page, 32)
    table = torch.full((1, width), 2 ** 31 - 1, device="cuda", dtype=torch.int32)
    table[0, first // page:] = c["table"][0, :width - first // page]
    want, bound = attn_ref(c, [past - first], [fresh], window, D ** -0.5)
    t = ops.draft_tree(i32(parents + [-1, -1]), c["cu"], i32([past]), max_tree=32)
    for hint in (0, fresh):
        got = ops.paged_tree_attn(c["q"], c["kp"], c["vp"], table, i32([past]), c["cu"], t.positions, t.mask, window=window,
                                  max_new=hint)
        assert ((got[:-2].double() - want).abs() <= 2.25 * U * bound).all()


@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 128), (3, 3, 64)])
def test_masks_of_any_kind(ops, Hq, Hkv, D):
    """Rows that see nothing, later tokens, not themselves; positions below the cached length."""
    rng = np.random.default_rng(5)
    cached, fresh = [0, 0, 90, 300], [40, 1, 64, 17]
    bits = [rng.random((n, 64)) < 0.3 for n in fresh]
    for b in bits:
        b[::3] = False
    bits[1][:] = False
    pos = [[int(x) for x in rng.integers(0, a + n + 1, n)] for a, n in zip(cached, fresh)]
    for window in (-1, 5, 40):
        c = check_attn(ops, cached, fresh, Hq, Hkv, D, 16, window=window, masks=(pos, bits), parents=[[]] * 4)
    assert c["mask"].shape == (sum(fresh) + 2, 2)


def test_a_row_that_sees_nothing_is_zero(ops):
    bits = [np.zeros((n, 32), bool) for n in (1, 20)]
    c = attn_case([0, 0], [1, 20], None, 8, 2, 128, 16, 32, masks=([[0], list(range(20))], bits), poison=float("nan"))
    got = ops.paged_tree_attn(c["q"], c["kp"], c["vp"], c["table"], c["cached"], c["cu"], c["pos"], c["mask"])
    assert not got.any()


@pytest.mark.parametrize("poison", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 128), (12, 12, 64)])
def test_what_lies_outside_a_request_does_not_reach_it(ops, poison, Hq, Hkv, D):
    window = 50
    c = check_attn(ops, [300, 5, 1000, 64], [1, 60, 3, 64], Hq, Hkv, D, 16, window=window, poison=poison)
    call = lambda: ops.paged_tree_attn(c["q"], c["kp"], c["vp"], c["table"], c["cached"], c["cu"], c["pos"], c["mask"],
                                       window=window)
    before = call()
    t = c["table"].long()
    for r, lo in ((0, 300 - window), (2, 1000 - window)):  # what lies wholly before the window
        for pool in (c["kp"], c["vp"]):
            pool[t[r, :lo // 16]] = poison
            pool[t[r, lo // 16], :, :lo % 16] = poison
    assert torch.equal(before, call())


@pytest.mark.parametrize("D", [64, 128])
def test_keys_that_a_token_does_not_see(ops, D):
    """NaN and infinite keys of the tree's other branches."""
    parents = [[-1, 0, 0, 1, 2, 3, 4]]
    c = attn_case([100], [7], parents, 8, 2, D, 16, 32)
    call = lambda: ops.paged_tree_attn(c["q"], c["kp"], c["vp"], c["table"], c["cached"], c["cu"], c["pos"], c["mask"])
    before = call()
    for poison in (float("nan"), float("inf"), float("-inf")):
        c["kp"][c["table"][0, 104 // 16].long(), :, 104 % 16] = poison  # token 4's key: 4 and 6 see it
        after = call()
        assert torch.equal(before[[0, 1, 2, 3, 5]], after[[0, 1, 2, 3, 5]])
    c = attn_case([100], [7], parents, 8, 2, D, 16, 32)
    c["kp"][c["table"][0, 104 // 16].long(), :, 104 % 16] = float("nan")
    got = ops.paged_tree_attn(c["q"], c["kp"], c["vp"], c["table"], c["cached"], c["cu"], c["pos"], c["mask"])
    assert got[[4, 6]].isnan().all() and got[[0, 1, 2, 3, 5]].isfinite().all()


SPIKES = {
    "one key": lambda c: 60.0 * (c == 390),
    "a jump": lambda c: 60.0 * (c >= 500),
    "a step every 64 keys": lambda c: 40.0 * (c // 64),
    "a step every 128 keys": lambda c: 40.0 * (c // 128),
    "up and down": lambda c: 50.0 * ((c // 64) % 3),
    "the last keys of the cache": lambda c: 60.0 * (c >= 636),
}


@pytest.mark.parametrize("pattern", SPIKES)
@pytest.mark.parametrize("D,G,fresh", [(128, 4, 60), (64, 1, 30), (128, 8, 64), (64, 4, 5)])
def test_scores_that_leap_by_hundreds(ops, pattern, D, G, fresh):
    """Far more than an exponential's range between one block of keys and the next, for some rows and not
    for others (q's first element is +1, 0 or -1)."""
    cached, scale = 640, 8.0
    c = attn_case([cached], [fresh], [random_parents(None, fresh, "chain")], 2 * G, 2, D, 64, 64, seed=3)
    key = torch.arange(cached + fresh, device="cuda")
    c["ks"][0][..., 0] = SPIKES[pattern](key).to(torch.bfloat16)[:, None]
    q = c["q"].contiguous().mul(0.25)
    q[:fresh, :, 0] = (torch.arange(fresh, device="cuda") % 3 - 1).to(torch.bfloat16)[:, None]
    c["q"] = q
    c["kp"][c["table"][0].long()[key // 64], :, key % 64] = c["ks"][0]
    want, bound = attn_ref(c, [cached], [fresh], -1, scale)
    got = ops.paged_tree_attn(q, c["kp"], c["vp"], c["table"], c["cached"], c["cu"], c["pos"], c["mask"],
                              softmax_scale=scale)[:fresh]
    err = (got.double() - want).abs()
    # a score of s = 480 is a sum of fp32 products: off by up to s 2^-20, its weight by that relatively
    slack = (2.25 * U + 8.0 * 480 * 2.0 ** -20) * bound
    assert err.isfinite().all() and (err <= slack).all(), (err - slack).max()


def test_a_chain_is_what_paged_attn_gives(ops):
    """To the rounding of either: a chain's masks are the causal ones."""
    for Hq, Hkv, D in ((16, 4, 128), (12, 12, 64)):
        cached, fresh = [100, 0, 999], [9, 17, 64]
        c = check_attn(ops, cached, fresh, Hq, Hkv, D, 16, kind="chain")
        other = ops.paged_attn(c["q"], c["kp"], c["vp"], c["table"], c["cached"], c["cu"])
        got = ops.paged_tree_attn(c["q"], c["kp"], c["vp"], c["table"], c["cached"], c["cu"], c["pos"], c["mask"])
        _, bound = attn_ref(c, cached, fresh, -1, D ** -0.5)
        assert ((got - other)[:-2].abs().double() <= 4.5 * U * bound).all()


def test_pages_outside_the_pool_are_reported(ops, expects_device_error):
    c = attn_case([100], [7], [random_parents(None, 7, "chain")], 8, 2, 128, 16, 32)
    for bad in (-1, c["kp"].shape[0], 2 ** 31 - 1):
        table = c["table"].clone()
        table[0, 2] = bad
        got = ops.paged_tree_attn(c["q"], c["kp"], c["vp"], table, c["cached"], c["cu"], c["pos"], c["mask"])
        assert ops.device_error()[0] == 6 and got.isfinite().all()


def test_lengths_past_the_table_are_reported(ops, expects_device_error):
    c = attn_case([100], [7], [random_parents(None, 7, "chain")], 8, 2, 64, 16, 32)
    for bad in (16 * c["table"].shape[1] - 6, 2 ** 31 - 1, -1):
        ops.paged_tree_attn(c["q"], c["kp"], c["vp"], c["table"].clamp(min=0), i32([bad]), c["cu"], c["pos"], c["mask"])
        assert ops.device_error()[0] == 1


def test_the_same_call_gives_the_same_bits(ops):
    c = check_attn(ops, [3000, 100, 0], [60, 20, 5], 16, 4, 128, 32)
    call = lambda: ops.paged_tree_attn(c["q"], c["kp"], c["vp"], c["table"], c["cached"], c["cu"], c["pos"], c["mask"])
    first = call()
    assert all(torch.equal(first, call()) for _ in range(5))


# ---------------------------------------------------------------------------------------------
# verify_drafts
def verify_ref(logits, tokens, parents, accept, draw, temperature, probs, max_path):
    """One request's walk, in 64 bits on the host."""
    n, V = logits.shape
    if n == 0:
        return 0, [], -1
    node, path = 0, [0]
    while True:
        row = logits[node]
        best = int(row.argmax())
        if temperature > 0:
            p = np.exp((row - row.max()) / temperature)
            p /= p.sum()
            rest, mass = p, 1.0
        following = -1
        for c in [j for j in range(node + 1, n) if parents[j] == node] if len(path) < max_path else []:
            x = tokens[c]
            if temperature == 0:
                if x == best:
                    following = c
                    break
                continue
            q = 1.0 if probs is None else probs[node][x]
            if accept[c] * q * mass < rest[x]:
                following = c
                break
            if probs is None:
                rest = rest.copy()
                rest[x] = 0
            else:
                rest = np.maximum(rest / mass - probs[node], 0)
            mass = rest.sum()
            if not mass > 0:
                rest, mass = p, 1.0
        if following < 0:
            break
        path.append(following)
        node = following
    if temperature == 0:
        return len(path), path, best
    sums = np.cumsum(rest)
    above = np.nonzero(sums > draw * sums[-1])[0]
    return len(path), path, int(above[0]) if len(above) else int(np.nonzero(rest > 0)[0][-1])


def verify_case(rng, fresh, V, draft, dtype=torch.float32, kind="any", spread=3.0, few=12):
    """Trees whose tokens are among a row's likely ones (a few tokens carry most of the probability)."""
    n = sum(fresh)
    parents = [random_parents(rng, m, kind) for m in fresh]
    cu = offsets(fresh)
    logits = rng.normal(size=(n, V)) * 0.5
    top = rng.integers(0, V, (n, few))
    np.put_along_axis(logits, top, rng.normal(size=(n, few)) * spread + 5, 1)
    logits = torch.tensor(logits, dtype=dtype)
    tokens = rng.integers(0, V, n)
    for r, m in enumerate(fresh):
        for t in range(1, m):
            if parents[r][t] >= 0:
                tokens[cu[r] + t] = top[cu[r] + parents[r][t], rng.integers(0, few)]
    probs = None
    if draft:
        near = logits.double().numpy() + rng.normal(size=(n, V)) * draft
        probs = np.exp(near - near.max(1, keepdims=True))
        probs = torch.tensor(probs / probs.sum(1, keepdims=True), dtype=torch.float32)
    return dict(logits=logits, tokens=tokens, parents=parents, probs=probs, cu=cu, accept=rng.random(n, dtype=np.float32),
                draws=rng.random(len(fresh), dtype=np.float32), fresh=fresh)


def run_verify(ops, c, temperature, max_path, pad=0):
    wide = torch.zeros(c["logits"].shape[0], c["logits"].shape[1] + pad, dtype=c["logits"].dtype)
    wide[:, :c["logits"].shape[1]] = c["logits"]
    probs = None if c["probs"] is None else c["probs"].cuda()
    return ops.verify_drafts(wide.cuda()[:, :c["logits"].shape[1]], torch.tensor(c["tokens"]).cuda(),
                             i32(sum(c["parents"], [])).reshape(-1), i32(c["cu"]), torch.tensor(c["accept"]).cuda(),
                             torch.tensor(c["draws"]).cuda(), temperature=temperature, draft_probs=probs, max_path=max_path)


def check_verify(ops, c, temperature, max_path=None, pad=0):
    width = max_path or max(c["fresh"] + [1])
    got = run_verify(ops, c, temperature, width, pad)
    logits = c["logits"].double().numpy()
    probs = None if c["probs"] is None else c["probs"].double().numpy()
    T = float(np.float32(temperature))
    lengths = []
    for r, m in enumerate(c["fresh"]):
        a, b = c["cu"][r], c["cu"][r] + m
        want = verify_ref(logits[a:b], c["tokens"][a:b], c["parents"][r], c["accept"][a:b].astype(float),
                          float(c["draws"][r]), T, None if probs is None else probs[a:b], width)
        kept = int(got.accepted[r])
        assert (kept, got.path[r].tolist()[:kept], int(got.next_token[r])) == want, r
        assert got.path[r].tolist()[kept:] == [-1] * (width - kept)
        lengths.append(kept)
    return got, lengths


@pytest.mark.parametrize("temperature", [0.0, 0.6, 1.0, 2.5])
@pytest.mark.parametrize("draft", [0.0, 0.2, 2.0])
@pytest.mark.parametrize("fresh,V", [([1], 7), ([0, 3, 1, 20], 1000), ([16] * 40, 4099), ([9] * 200, 517),
                                     ([64, 2], 32768), ([5, 5], 100003), ([1, 2, 3], 1)])
def test_walks(ops, temperature, draft, fresh, V):
    rng = np.random.default_rng(V + len(fresh))
    c = verify_case(rng, fresh, V, draft)
    check_verify(ops, c, temperature, pad=3)


@pytest.mark.parametrize("draft", [0.0, 0.3])
def test_walks_in_bf16_and_by_chains(ops, draft):
    rng = np.random.default_rng(3)
    c = verify_case(rng, [12] * 30 + [0, 1], 3001, draft, torch.bfloat16, "chain", spread=0.5, few=2)
    c["accept"] *= 0.3
    _, lengths = check_verify(ops, c, 1.0, pad=1)
    assert max(lengths) >= (5 if draft else 2)  # (they do go on)
    check_verify(ops, c, 1.0, max_path=3)
    check_verify(ops, c, 1.0, max_path=1)


def test_flat_rows(ops):
    """Every token as likely as the next: the draw is next to a border everywhere."""
    V = 50021
    for pad in (0, 1, 2, 3):
        u = (torch.arange(64) * 777 + 5 + pad).double()
        draws = ((u + 0.5) / V).float()
        logits = torch.full((64, V + pad), 1.5, device="cuda")[:, :V]
        got = ops.verify_drafts(logits, torch.zeros(64, dtype=torch.long, device="cuda"), i32([-1] * 64), i32(range(65)),
                                torch.zeros(64, device="cuda"), draws.cuda(), max_path=1)
        assert got.next_token.tolist() == torch.floor(draws.double() * V).long().tolist()


def test_a_large_vocabulary(ops):
    rng = np.random.default_rng(8)
    c = verify_case(rng, [4, 7], 262147, 0.4)
    check_verify(ops, c, 1.0)
    check_verify(ops, c, 0.0)


def test_many_children_and_the_same_token_twice(ops):
    """Refused again and again; a refused token that comes back has nothing left."""
    rng = np.random.default_rng(4)
    for draft in (0.0, 0.5):
        c = verify_case(rng, [60], 97, draft)
        c["parents"] = [[-1] + [0] * 59]
        c["tokens"][1:] = rng.integers(0, 20, 59)
        c["accept"][:] = 0.999
        check_verify(ops, c, 1.0)
        c["accept"][:] = rng.random(60) * 0.2 + 0.6
        check_verify(ops, c, 1.3)


def test_a_draft_that_is_the_target_is_kept(ops):
    """Its probabilities in 32 bits are off by up to 2^-24: a uniform of at most 1 - 2^-20 keeps it."""
    rng = np.random.default_rng(5)
    c = verify_case(rng, [10, 10], 1000, 0.0, kind="chain")
    c["probs"] = torch.softmax(c["logits"].double(), -1).float()
    c["accept"][:] = 1 - 2.0 ** -20
    got, lengths = check_verify(ops, c, 1.0)
    assert lengths == [10, 10]


def test_nothing_left_falls_back_to_the_target(ops):
    # all of the target's probability on a token that is refused (its uniform is 1)
    logits = torch.full((2, 50), -math.inf, device="cuda")
    logits[:, 7] = 1.0
    args = (torch.tensor([0, 7]).cuda(), i32([-1, 0]), i32([0, 2]), torch.ones(2, device="cuda"),
            torch.tensor([0.5], device="cuda"))
    for probs in (None, torch.softmax(logits, -1)):
        got = ops.verify_drafts(logits, *args, draft_probs=probs, max_path=2)
        assert (got.accepted.tolist(), got.next_token.tolist()) == ([1], [7])


@pytest.mark.parametrize("draw", [0.0, 1.0, 1 - 2.0 ** -24])
def test_draws_at_the_ends(ops, draw):
    logits = torch.full((3, 5000), -math.inf, device="cuda")
    logits[:, [17, 300, 4711]] = 0.0
    got = ops.verify_drafts(logits, torch.zeros(3, dtype=torch.long, device="cuda"), i32([-1] * 3), i32([0, 1, 2, 3]),
                            torch.zeros(3, device="cuda"), torch.full((3,), draw, device="cuda"), max_path=4)
    assert got.next_token.tolist() == [17 if draw == 0 else 4711] * 3


def test_greedy_ties_go_to_the_first(ops):
    logits = torch.zeros(2, 9000, device="cuda")
    logits[0, [123, 8000]] = 4.0
    logits[1, [5, 6]] = 1.0
    for x, want in ((123, ([2], 5)), (8000, ([1], 123))):
        got = ops.verify_drafts(logits, torch.tensor([0, x]).cuda(), i32([-1, 0]), i32([0, 2]),
                                torch.zeros(2, device="cuda"), torch.zeros(1, device="cuda"), temperature=0, max_path=2)
        assert (got.accepted.tolist(), int(got.next_token)) == want


def test_rows_without_probabilities(ops, expects_device_error):
    for bad in (float("nan"), float("inf")):
        for temperature in (0.0, 1.0):
            logits = torch.zeros(4, 3000, device="cuda")
            logits[1, 2999] = bad
            logits[2] = -math.inf
            got = ops.verify_drafts(logits, torch.zeros(4, dtype=torch.long, device="cuda"), i32([-1] * 4),
                                    i32([0, 1, 2, 3, 4]), torch.zeros(4, device="cuda"), torch.zeros(4, device="cuda"),
                                    temperature=temperature, max_path=1)
            assert got.next_token.tolist() == [0, -1, -1, 0] and got.accepted.tolist() == [1] * 4
            assert ops.device_error()[0] == 9


def test_drafted_tokens_outside_the_vocabulary(ops, expects_device_error):
    for x in (-1, 100, 1 << 40):
        logits = torch.zeros(3, 100, device="cuda")
        got = ops.verify_drafts(logits, torch.tensor([0, x, 3]).cuda(), i32([-1, 0, 0]), i32([0, 3]),
                                torch.zeros(3, device="cuda"), torch.zeros(1, device="cuda"), max_path=3)
        assert ops.device_error()[0] == 4 and got.path.tolist() == [[0, 2, -1]]


def test_the_tokens_have_the_targets_distribution(ops):
    """20,000 requests with the same rows and other uniforms: the first new token, kept or drawn, against
    the target's probabilities.  A count of n draws has variance n p (1 - p): 5 of its deviations."""
    n, V = 20000, 6
    g = torch.Generator("cuda").manual_seed(1)
    logits = torch.tensor([1.0, 0.2, -0.5, 0.8, -2.0, 0.0], device="cuda")
    q = torch.softmax(torch.tensor([0.1, 1.2, 0.0, 0.3, -1.0, 0.4], device="cuda"), -1)
    rand = lambda *s: torch.rand(*s, device="cuda", generator=g)
    p = torch.softmax(logits.double(), -1).cpu()
    for draft in (True, False):
        children = torch.multinomial(q.expand(n, V), 2, replacement=True, generator=g) if draft else torch.tensor(
            [[1, 3]], device="cuda").expand(n, 2)
        tokens = torch.cat([torch.zeros(n, 1, dtype=torch.long, device="cuda"), children], 1).reshape(-1)
        got = ops.verify_drafts(logits.expand(3 * n, V).contiguous(), tokens, i32([-1, 0, 0] * n), i32(np.arange(n + 1) * 3),
                                rand(3 * n), rand(n), draft_probs=q.expand(3 * n, V).contiguous() if draft else None,
                                max_path=2)
        kept = got.accepted > 1
        first = torch.where(kept, tokens.view(n, 3).gather(1, got.path[:, 1:].long().clamp(min=0))[:, 0], got.next_token)
        count = torch.bincount(first, minlength=V).cpu().double()
        assert ((count - n * p).abs() <= 5 * (n * p * (1 - p)).sqrt()).all(), (count, n * p)
        assert kept.float().mean() > 0.3


# ---------------------------------------------------------------------------------------------
# paged_keep
def pools(g, slots, n_pages, Hkv, page, D):
    shape = (slots, n_pages, Hkv, page, D) if slots else (n_pages, Hkv, page, D)
    return [torch.randn(shape, device="cuda", dtype=torch.bfloat16, generator=g) for _ in range(2)]


def tables(rng, lens, page, width, spare, head):
    held = [ceil_div(a, page) for a in lens]
    order = rng.permutation(sum(held) + spare)
    table, at = np.full((len(lens), width), -1), 0
    for r, n in enumerate(held):
        table[r, :n] = order[at:at + n]
        at += n
    queue = np.full(len(order), -1)
    queue[(head + np.arange(spare)) % len(order)] = order[at:]
    return table, queue, [head, head + spare]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("cached,fresh,slots,Hkv,D,page", [
    ([0], [1], 1, 1, 64, 16), ([5, 16, 31, 0, 40], [20, 1, 64, 0, 17], 3, 2, 128, 16), ([100], [300], 0, 3, 64, 32),
    ([i * 7 % 300 for i in range(90)], [i * 5 % 40 for i in range(90)], 2, 4, 64, 16),
    ([17] * 700, [9] * 700, 1, 1, 64, 64), ([1000, 3], [600, 2], 5, 1, 128, 1024),
])
def test_keep_moves_the_path_and_gives_pages_back(ops, in_place, cached, fresh, slots, Hkv, D, page):
    rng = np.random.default_rng(len(cached) + page)
    g = torch.Generator("cuda").manual_seed(1)
    R, P = len(cached), max(fresh) + 1
    lens = [a + b for a, b in zip(cached, fresh)]
    table, queue, state = tables(rng, lens, page, ceil_div(max(lens), page) + 2, 4, 10 ** 12 + 1)
    kp, vp = pools(g, slots, len(queue), Hkv, page, D)
    kept = [int(rng.integers(0, n + 1)) for n in fresh]
    path = np.full((R, P + 2), -1)
    for r, (n, k) in enumerate(zip(fresh, kept)):
        path[r, :k] = np.sort(rng.permutation(n)[:k])
    want = [x.clone() for x in (kp, vp)]
    for pool in want:
        flat = pool.view(-1, len(queue), Hkv, page, D)
        for r in range(R):
            at = lambda t: (int(table[r, (cached[r] + t) // page]), (cached[r] + t) % page)
            moved = [flat[:, at(t)[0], :, at(t)[1]].clone() for t in path[r, :kept[r]]]
            for i, v in enumerate(moved):
                flat[:, at(i)[0], :, at(i)[1]] = v
    q2, tail = queue.copy(), state[1]
    for r in range(R):
        for c in range(ceil_div(cached[r] + kept[r], page), ceil_div(lens[r], page)):
            q2[tail % len(queue)] = table[r, c]
            tail += 1
    st, cl, fp = torch.tensor(state, device="cuda"), i32(cached), i32(queue)
    out = dict(free_state_out=st, seqlens_out=cl) if in_place else {}
    state2, lens2 = ops.paged_keep(i32(path)[:, :P], i32(kept), cl, i32(fresh), i32(table), fp, st, kp, vp, **out)
    assert torch.equal(kp, want[0]) and torch.equal(vp, want[1])
    assert fp.tolist() == q2.tolist() and state2.tolist() == [state[0], tail]
    assert lens2.tolist() == [a + k for a, k in zip(cached, kept)]
    assert in_place or (st.tolist() == state and cl.tolist() == cached)


def test_keep_with_paths_that_do_not_fit(ops, expects_device_error):
    g = torch.Generator("cuda").manual_seed(1)
    for path, kept, want in (([[0, 0, 3]], 3, 3), ([[0, 9, 3]], 3, 3), ([[0, 1, 2]], 7, 3),
                             ([[0, -1, 2]], 3, 3)):
        kp, vp = pools(g, 1, 4, 1, 16, 64)
        before = kp.clone()
        state, lens = ops.paged_keep(i32(path), i32([kept]), i32([3]), i32([5]), i32([[2, 1]]), i32([0, 3, -1, -1]),
                                     torch.tensor([0, 2], device="cuda"), kp, vp)
        assert ops.device_error()[0] == 8 and lens.tolist() == [3 + want]
        moved = [p for p in range(16) if not torch.equal(kp[0, 2, :, p], before[0, 2, :, p])]
        assert moved == ([5] if path[0][2] == 3 else [])


def test_keep_and_fork_past_32_bits(ops):
    """A pool of 2^32 bytes and more a slot: the last slot's last pages."""
    slots, n_pages, Hkv, page, D = 2, 34000, 8, 64, 128
    kp, vp = (torch.zeros(slots, n_pages, Hkv, page, D, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    g = torch.Generator("cuda").manual_seed(1)
    for pool in (kp, vp):
        pool[:, -2] = torch.randn(slots, Hkv, page, D, device="cuda", dtype=torch.bfloat16, generator=g)
    before = [pool[:, -2].clone() for pool in (kp, vp)]
    queue, state = torch.arange(n_pages, device="cuda", dtype=torch.int32), torch.tensor([n_pages - 1, n_pages], device="cuda")
    ops.paged_keep(i32([[0, 5, 40]]), i32([3]), i32([10]), i32([50]), i32([[n_pages - 2]]), queue.clone(), state, kp, vp)
    f = ops.page_fork(i32([0, 0]), i32([13, 0]), i32([[n_pages - 2], [-1]]), torch.zeros_like(queue), queue, state, kp, vp)
    assert f.block_table.tolist() == [[n_pages - 2], [n_pages - 1]]
    for pool, old in zip((kp, vp), before):
        for i, at in enumerate((0, 5, 40)):
            assert torch.equal(pool[:, -2, :, 10 + i], old[:, :, 10 + at])
        assert torch.equal(pool[:, -1, :, :13], pool[:, -2, :, :13]) and not pool[:, -1, :, 13:].any()
        assert not pool[:, :-2].any()


def test_keep_of_whole_steps(ops):
    """accepted < 0: as it is, its path not read; the pages up to its end stay."""
    g = torch.Generator("cuda").manual_seed(1)
    kp, vp = pools(g, 2, 8, 1, 16, 64)
    before = kp.clone()
    state, lens = ops.paged_keep(i32([[9, 9], [0, 3]]), i32([-1, 2]), i32([3, 20]), i32([40, 30]),
                                 i32([[2, 1, 0, -1], [3, 4, 5, 6]]), i32([7, -1, -1, -1, -1, -1, -1, -1]),
                                 torch.tensor([0, 1], device="cuda"), kp, vp)
    assert lens.tolist() == [43, 22] and state.tolist() == [0, 3]
    assert torch.equal(kp[:, 4, :, 5], before[:, 4, :, 7])
    kp[:, 4, :, 5] = before[:, 4, :, 5]
    assert torch.equal(kp, before)


def test_keep_without_requests(ops):
    g = torch.Generator("cuda").manual_seed(1)
    kp, vp = pools(g, 2, 4, 1, 16, 64)
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    state, lens = ops.paged_keep(none.view(0, 3), none, none, none, none.view(0, 2), i32([0, 1, 2, 3]),
                                 torch.tensor([5, 9], device="cuda"), kp, vp)
    assert state.tolist() == [5, 9] and lens.numel() == 0


# ---------------------------------------------------------------------------------------------
# page_fork
def fork_ref(source, lens, table, shares, queue, state, pools, page):
    table, shares, queue, (head, tail) = table.copy(), shares.copy(), queue.copy(), state
    new, n, out = np.full_like(table, -1), len(queue), [p.clone() for p in pools]
    first, new_lens = {}, []
    for r, s in enumerate(source):
        if not 0 <= s < len(source):
            new_lens.append(0)
            continue
        full, part = divmod(lens[s], page)
        new[r, :full] = table[s, :full]
        new_lens.append(lens[s])
        if part:
            old = int(table[s, full])
            if s in first:
                page_new = int(queue[head % n])
                head += 1
                for pool, dst in zip(pools, out):
                    dst[:, page_new, :, :part] = pool[:, old, :, :part]
                new[r, full] = page_new
            else:
                new[r, full] = old
        first.setdefault(s, r)
    holders = np.zeros(n, int)
    for r, m in enumerate(new_lens):
        for c in range(ceil_div(m, page)):
            holders[new[r, c]] += 1
    for r, m in enumerate(lens):
        for c in range(ceil_div(m, page)):
            if holders[table[r, c]] == 0 and shares[table[r, c]] >= 0:
                shares[table[r, c]] = -1
    for x in np.nonzero(shares < 0)[0]:
        queue[tail % n] = x
        tail += 1
    return new, np.maximum(holders - 1, 0), queue, [head, tail], new_lens, out


def fork_state(rng, groups, page, slots, Hkv, D, width, spare, head=7):
    """Rows in groups that share full pages: groups = [(shared pages, [row lengths])]."""
    lens, rows, n = [], [], 0
    for shared, lengths in groups:
        common = list(range(n, n + shared))
        n += shared
        for m in lengths:
            own = list(range(n, n + ceil_div(m, page) - min(shared, m // page)))
            n += len(own)
            rows.append(common[:m // page] + own)
            lens.append(m)
    total = n + spare
    order = rng.permutation(total)
    table, holders = np.full((len(rows), width), -1), np.zeros(total, int)
    for r, pages in enumerate(rows):
        table[r, :len(pages)] = order[pages]
        holders[order[pages]] += 1
    held = np.zeros(total, bool)
    held[table[table >= 0]] = True
    free = np.nonzero(~held)[0]
    queue = np.full(total, -1)
    queue[(head + np.arange(len(free))) % total] = rng.permutation(free)
    g = torch.Generator("cuda").manual_seed(2)
    return lens, table, np.maximum(holders - 1, 0), queue, [head, head + len(free)], pools(g, slots, total, Hkv, page, D)


GROUPS = {
    "one row": [(0, [37])],
    "prompts": [(0, [100]), (0, [0]), (0, [64]), (0, [0]), (0, [0]), (0, [5])],
    "beams": [(3, [50, 70, 48, 63]), (2, [32, 33, 90, 40]), (0, [1, 16, 15, 17])],
    "many": [(i % 5, [i * 3 % 90 + 80, i * 7 % 60 + 80, 96]) for i in range(400)],
}


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("kind", ["random", "same", "none", "one", "reverse"])
@pytest.mark.parametrize("name", GROUPS)
@pytest.mark.parametrize("slots,Hkv,D", [(2, 2, 64), (1, 1, 128)])
def test_fork_against_the_plain_one(ops, in_place, kind, name, slots, Hkv, D):
    rng = np.random.default_rng(len(name) + slots)
    page, R = 16, sum(len(b) for _, b in GROUPS[name])
    lens, table, shares, queue, state, (kp, vp) = fork_state(rng, GROUPS[name], page, slots, Hkv, D, 13, R + 2)
    source = {"random": rng.integers(-1, R, R), "same": np.arange(R), "none": np.full(R, -1),
              "one": np.zeros(R, int), "reverse": np.arange(R)[::-1]}[kind].tolist()
    want = fork_ref(source, lens, table, shares, queue, state, (kp, vp), page)
    wide = i32(np.pad(table, ((0, 0), (0, 3)), constant_values=99))
    args = dict(source=i32(source), cache_seqlens=i32(lens), block_table=wide[:, :13], shares=i32(shares),
                free_pages=i32(queue), free_state=torch.tensor(state, device="cuda"), k_pages=kp, v_pages=vp)
    keys = dict(block_table_out="block_table", shares_out="shares", free_state_out="free_state",
                seqlens_out="cache_seqlens")
    f = ops.page_fork(**args, **({k: args[v] for k, v in keys.items()} if in_place else {}))
    assert np.array_equal(f.block_table.cpu().numpy(), want[0])
    assert f.shares.tolist() == want[1].tolist() and args["free_pages"].tolist() == want[2].tolist()
    assert f.free_state.tolist() == want[3] and f.seqlens.tolist() == want[4]
    assert torch.equal(kp, want[5][0]) and torch.equal(vp, want[5][1])
    assert (wide[:, 13:] == 99).all()
    if not in_place:
        assert np.array_equal(args["block_table"].cpu().numpy(), table) and args["shares"].tolist() == shares.tolist()


def test_calls_without_requests_or_tokens(ops):
    g = torch.Generator("cuda").manual_seed(1)
    kp, vp = pools(g, 1, 40, 1, 16, 64)
    none, state = torch.zeros(0, dtype=torch.int32, device="cuda"), torch.tensor([7, 9], device="cuda")
    queue = i32(range(40))
    f = ops.page_fork(none, none, none.view(0, 2), torch.zeros_like(queue), queue, state, kp, vp)
    assert f.free_state.tolist() == [7, 9] and f.shares.tolist() == [0] * 40 and queue.tolist() == list(range(40))
    empty = torch.zeros(0, 50, device="cuda")
    got = ops.verify_drafts(empty, none.long(), none, i32([0, 0, 0]), empty[:, 0], torch.zeros(2, device="cuda"), max_path=3)
    assert got.accepted.tolist() == [0, 0] and got.next_token.tolist() == [-1, -1] and (got.path == -1).all()
    got = ops.verify_drafts(empty, none.long(), none, i32([0]), empty[:, 0], empty[:, 0], max_path=3)
    assert got.path.shape == (0, 3)
    q = torch.zeros(3, 2, 64, device="cuda", dtype=torch.bfloat16)
    out = ops.paged_tree_attn(q + 1, kp[0], vp[0], none.view(0, 2), none, i32([0]), i32([0] * 3), i32([[1]] * 3))
    assert not out.any()
    out = ops.paged_tree_attn(q[:0], kp[0], vp[0], i32([[0]]), i32([5]), i32([0, 0]), none, none.view(0, 1))
    assert out.shape == (0, 2, 64)


def test_a_large_pool_is_counted_and_placed_by_blocks(ops):
    """Above 32 blocks of 1,024 pages: freed pages in page order across them, the queue's ring included."""
    rng = np.random.default_rng(3)
    n, rows, page = 40000, 50, 16
    order = rng.permutation(n)
    table = np.full((rows, 500), -1)
    lens = rng.integers(1, 500 * page, rows)
    at = 0
    for r in range(rows):
        held = ceil_div(int(lens[r]), page)
        table[r, :held] = order[at:at + held]
        at += held
    queue = np.full(n, -1)
    head = n - 5
    queue[(head + np.arange(n - at)) % n] = order[at:]
    g = torch.Generator("cuda").manual_seed(1)
    kp, vp = pools(g, 0, n, 1, page, 64)
    source = [r if r % 3 else -1 for r in range(rows)]
    want = fork_ref(source, lens.tolist(), table, np.zeros(n, int), queue, [head, head + n - at], (kp, vp), page)
    q = i32(queue)
    f = ops.page_fork(i32(source), i32(lens), i32(table), i32(np.zeros(n)), q, torch.tensor([head, head + n - at], device="cuda"),
                      kp, vp)
    assert q.tolist() == want[2].tolist() and f.free_state.tolist() == want[3]
    assert np.array_equal(f.block_table.cpu().numpy(), want[0]) and not f.shares.any()


def test_fork_step_after_step(ops):
    """Random steps on the same tables: every page is free or held, and shared by as many as its shares say."""
    rng = np.random.default_rng(0)
    page, R, width = 16, 12, 9
    lens, table, shares, queue, state, (kp, vp) = fork_state(rng, [(0, [100])] + [(0, [0])] * 11, page, 1, 1, 64, width, 60)
    t = [i32(lens), i32(table), i32(shares), i32(queue), torch.tensor(state, device="cuda")]
    for _ in range(25):
        lens_now = t[0].tolist()
        live = [r for r, n in enumerate(lens_now) if n]
        source = [int(rng.choice(live)) if rng.random() < 0.8 else -1 for _ in range(R)]
        if max(source) < 0:
            source[0] = live[0]
        ops.page_fork(i32(source), t[0], t[1], t[2], t[3], t[4], kp, vp, block_table_out=t[1], shares_out=t[2],
                      free_state_out=t[4], seqlens_out=t[0])
        # the rows grow by a few tokens
        lens_now = np.array(t[0].tolist())
        fresh = np.where(lens_now > 0, np.minimum(rng.integers(0, 9, R), 130 - lens_now), 0)
        ops.page_plan(t[0], i32(fresh), t[1], t[3], t[4], page_size=page, num_tokens=int(fresh.sum()),
                      free_state_out=t[4])
        t[0] += i32(fresh)
        lens_now, tab = t[0].tolist(), t[1].tolist()
        holders = {}
        for r, n in enumerate(lens_now):
            for x in tab[r][:ceil_div(n, page)]:
                holders[x] = holders.get(x, 0) + 1
        head, tail = t[4].tolist()
        free = [t[3].tolist()[x % len(queue)] for x in range(head, tail)]
        assert sorted(free + list(holders)) == list(range(len(queue)))
        assert all(t[2].tolist()[x] == holders.get(x, 1) - 1 for x in range(len(queue)))
        for r, n in enumerate(lens_now):  # a page that is not full is one row's own
            assert n % page == 0 or holders[tab[r][n // page]] == 1


def test_fork_reports_what_does_not_fit(ops, expects_device_error):
    g = torch.Generator("cuda").manual_seed(1)
    for source, queue, state, code in (([0, 2], [2, 3, -1, -1], [0, 2], 8), ([0, 0], [2, 3, -1, -1], [2, 2], 5),
                                       ([0, 0], [9, 3, -1, -1], [0, 2], 6), ([0, 0], [-1, 3, -1, -1], [0, 2], 6)):
        kp, vp = pools(g, 1, 4, 1, 16, 64)
        f = ops.page_fork(i32(source), i32([20, 0]), i32([[0, 1], [-1, -1]]), i32([0] * 4), i32(queue),
                          torch.tensor(state, device="cuda"), kp, vp)
        assert ops.device_error()[0] == code
        assert f.block_table.tolist() == [[0, 1], [-1, -1] if code == 8 else [0, -1]]
    kp, vp = pools(g, 1, 4, 1, 16, 64)
    f = ops.page_fork(i32([0]), i32([50]), i32([[0, 1]]), i32([0] * 4), i32([2, 3, -1, -1]),
                      torch.tensor([0, 2], device="cuda"), kp, vp)
    assert ops.device_error()[0] == 1 and f.seqlens.tolist() == [32]
    f = ops.page_fork(i32([-1]), i32([20]), i32([[0, 7]]), i32([0] * 4), i32([2, 3, 1, -1]),
                      torch.tensor([0, 3], device="cuda"), kp, vp)
    assert ops.device_error()[0] == 6 and f.free_state.tolist() == [0, 4]
