"""Speculative decoding and shared pages where their parts meet: a cluster's blocks that decide alike, sums
and comparisons at their bounds, extreme temperatures, many requests of many heads, steps that follow one
another.  Plain forms and tolerances are test_gpu_draft's."""
import math

import numpy as np
import pytest
import torch

from test_gpu_draft import U, attn_case, attn_ref, check_verify, i32, random_parents, verify_case
from test_gpu_draft import expects_device_error, no_device_error, ops  # noqa: F401  (fixtures)

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------------------------
# paged_tree_attn
@pytest.mark.parametrize("Hq,Hkv,D,fresh", [(8, 2, 128, 4), (8, 1, 64, 2), (16, 4, 128, 8), (4, 1, 64, 7)])
def test_maxima_at_every_place_of_a_tile(ops, Hq, Hkv, D, fresh):
    """Few rows a kv head, tile after tile of 128 keys whose maximum is 40 above the tile's before, at another key for each
    of 128 requests: every thread's maximum, reference and sum in turn is the one that counts, for rows that
    see it rise, fall or not at all.  Tolerance as for scores that leap by hundreds (test_gpu_draft)."""
    R, cached, scale = 128, 640, 8.0
    c = attn_case([cached] * R, [fresh] * R, [random_parents(None, fresh, "chain")] * R, Hq, Hkv, D, 64, 32, seed=5)
    key = torch.arange(cached + fresh, device="cuda")
    at = key.new_tensor([[t * 128 + (r * 37 + t * 11) % 128 for t in range(5)] for r in range(R)])
    q = c["q"].contiguous().mul(0.25)
    q[:-2, :, 0] = (torch.arange(R * fresh, device="cuda") % 3 - 1).to(torch.bfloat16)[:, None]
    c["q"] = q
    for r in range(R):
        c["ks"][r][..., 0] = 0
        c["ks"][r][at[r], :, 0] = (40.0 * torch.arange(1, 6, device="cuda")).to(torch.bfloat16)[:, None]
        c["kp"][c["table"][r].long()[key // 64], :, key % 64] = c["ks"][r]
    want, bound = attn_ref(c, [cached] * R, [fresh] * R, -1, scale)
    call = lambda: ops.paged_tree_attn(q, c["kp"], c["vp"], c["table"], c["cached"], c["cu"], c["pos"], c["mask"],
                                       softmax_scale=scale, max_new=fresh)
    got = call()
    err = (got[:-2].double() - want).abs()
    # scores up to 8 * 200 and some tens: 1,700 2^-20 of a weight
    slack = (2.25 * U + 8.0 * 1700 * 2.0 ** -20) * bound
    assert err.isfinite().all() and (err <= slack).all(), (err - slack).max()
    assert all(torch.equal(call(), got) for _ in range(20))


# ---------------------------------------------------------------------------------------------
# verify_drafts
@pytest.mark.parametrize("V,R", [(16384, 30), (9000, 60), (5000, 120), (40000, 18)])
def test_comparisons_near_the_bound_of_the_32_bit_sums(ops, V, R):
    """Chains whose tokens are all kept, by 1e-5 to 5e-5: what a comparison is short of lies around the distance at
    which the row is summed again, now and then within an ulp of it.  Requests of 8, 4 and 2 blocks: all of a
    request's take the second sum, or none does (a block alone in it would wait at another barrier)."""
    T = 40
    g = torch.Generator("cuda").manual_seed(V)
    logits = torch.randn(R * T, V, device="cuda", generator=g) * 2
    tokens = torch.randint(0, V, (R, T), device="cuda", generator=g)
    x = tokens.roll(-1, 1).reshape(-1, 1)  # the token of the only child
    logits.scatter_(1, x, -math.inf)
    logits.scatter_(1, x, torch.logsumexp(logits, 1, keepdim=True) - 0.5)
    p = torch.softmax(logits.double(), 1)
    short = 1e-5 + 4e-5 * torch.rand(R * T, device="cuda", generator=g, dtype=torch.float64)
    accept = torch.zeros(R * T, device="cuda")
    accept.view(R, T)[:, 1:] = (p.gather(1, x)[:, 0] - short).float().view(R, T)[:, :-1]
    draws = torch.rand(R, device="cuda", generator=g)
    sums = p.view(R, T, V)[:, -1].cumsum(1)
    want = (sums <= draws[:, None].double() * sums[:, -1:]).sum(1)
    for _ in range(10):
        got = ops.verify_drafts(logits, tokens.reshape(-1), i32([t - 1 for t in range(T)] * R), i32(np.arange(R + 1) * T),
                                accept, draws, max_path=T)
        assert got.accepted.tolist() == [T] * R and got.path.tolist() == [list(range(T))] * R
        assert torch.equal(got.next_token, want)
        accept.view(R, T)[:, 1:] += 2.0 ** -25  # (3e-8, ten times: far less than 1e-5)


def test_rows_of_unlike_length_back_to_back(ops):
    """Requests with and without tokens, clusters that end at once beside ones that walk, launch after launch: a block's
    shared memory is written by the others of its cluster once it has started, and as long as it is there."""
    V = 16384  # 8 blocks of 2,048 tokens
    g = torch.Generator("cuda").manual_seed(0)
    fresh = [r % 4 for r in range(37)]
    cu = np.concatenate([[0], np.cumsum(fresh)])
    best = torch.randint(0, V, (int(cu[-1]),), device="cuda", generator=g)
    logits = torch.zeros(len(best), V, device="cuda").scatter_(1, best[:, None], 60.0)  # (others: e^-60 each)
    parents = i32(sum(([-1, 0, 0][:n] for n in fresh), []))
    tokens = best.roll(1)  # the first child is kept
    accept, draws = (torch.full((n,), 0.5, device="cuda") for n in (len(best), len(fresh)))
    got = [ops.verify_drafts(logits, tokens, parents, i32(cu), accept, draws, max_path=2) for _ in range(200)]
    last = [cu[r] + min(n, 2) - 1 for r, n in enumerate(fresh)]
    for v in got:
        assert v.accepted.tolist() == [min(n, 2) for n in fresh]
        assert v.next_token.tolist() == [int(best[t]) if n else -1 for t, n in zip(last, fresh)]


def adding(inc, n):
    """n times inc added up in 32 bits."""
    s, inc = np.float32(0), np.float32(inc)
    for _ in range(n):
        s += inc
    return float(s)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_vocabulary_whose_32_bit_sums_are_far_off(ops, dtype):
    """2^25 tokens and one block (more requests than half of a GPU's blocks, all but one without tokens): a lane adds
    16,384 equal groups, one rounding after another the same way.  Token 7 has half of the probability; a uniform a
    little above it refuses it, one a little below keeps it, at distances that 1e-5 would take for settled."""
    V, x = 1 << 25, 7
    if dtype == torch.float32:
        tail = math.log(2.0 ** -25 * (1 + 0.75 * 2.0 ** -9))
    else:
        tail = -17.25  # (exact)
    logits = torch.full((2, V), tail, device="cuda", dtype=dtype)
    tail = float(logits[0, 0])
    peak = 0.0 if dtype == torch.float32 else 0.125
    logits[:, x] = peak
    w = math.exp(tail - peak)
    exact = 1 / (1 + (V - 1) * w)
    in32 = 1 / (1 + 512 * adding(4 * np.float32(w), V // 2048))
    if dtype == torch.float32:
        assert abs(in32 - exact) > 5e-5  # (what the test is about: more than a bound of 1e-5 allows)
    R = 300
    cu = i32([0] + [2] * R)
    tokens, parents, draws = torch.tensor([0, x], device="cuda"), i32([-1, 0]), torch.full((R,), 0.25, device="cuda")
    for near in (1e-6, 1e-5, 2.5e-5, 4e-5, 1e-4, 1e-3):
        for side in (-1, 1):
            u = np.float32(exact + side * near)
            got = ops.verify_drafts(logits, tokens, parents, cu, torch.full((2,), float(u), device="cuda"), draws, max_path=2)
            assert got.accepted.tolist() == [2 if u < exact else 1] + [0] * (R - 1), (near, side)
            # the draw at a quarter: of the whole row at token 1, of the row without x at token 0
            if u < exact:
                want = x if 7 * w <= 0.25 / exact < 7 * w + 1 else 0.25 / exact / w
            else:
                want = 0.25 * (V - 1) + 1
            assert abs(int(got.next_token[0]) - want) <= 1


@pytest.mark.parametrize("bad", [math.nan, -1e-3, -math.inf])
@pytest.mark.parametrize("V", [50, 20000])
def test_uniforms_that_are_none(ops, expects_device_error, bad, V):
    """A draw that is NaN or below 0 gives no token, such an accept keeps none, and both are reported; the other requests
    are as ever, and temperature 0 reads no uniforms."""
    logits = torch.zeros(6, V, device="cuda")
    logits[:, 3] = 60.0  # (the others: e^-60 each)
    tokens, parents, cu = torch.tensor([0, 3] * 3, device="cuda"), i32([-1, 0] * 3), i32([0, 2, 4, 6])
    fine, half = torch.full((6,), 0.5, device="cuda"), torch.full((3,), 0.5, device="cuda")
    bent = torch.tensor([0.5, bad, 0.5], device="cuda")
    for probs in (None, torch.softmax(logits, 1)):
        got = ops.verify_drafts(logits, tokens, parents, cu, fine, bent, draft_probs=probs, max_path=2)
        assert ops.device_error()[0] == 10
        assert got.accepted.tolist() == [2, 2, 2] and got.next_token.tolist() == [3, -1, 3]
        got = ops.verify_drafts(logits, tokens, parents, cu, bent.repeat_interleave(2), half, draft_probs=probs, max_path=2)
        assert ops.device_error()[0] == 10
        assert got.accepted.tolist() == [2, 1, 2] and got.next_token.tolist() == [3, 3, 3]
    got = ops.verify_drafts(logits, tokens, parents, cu, fine * bad, half * bad, temperature=0, max_path=2)
    assert ops.device_error()[0] == 0 and got.accepted.tolist() == [2, 2, 2] and got.next_token.tolist() == [3, 3, 3]


@pytest.mark.parametrize("temperature", [1e-20, 1e-15, 1e-10, 1e-6, 1e20])
@pytest.mark.parametrize("draft", [0.0, 0.3])
def test_extreme_temperatures(ops, temperature, draft):
    """Almost greedy and almost flat, among ties of the largest logit, logits of hundreds and of -infinity."""
    rng = np.random.default_rng(3)
    c = verify_case(rng, [1, 9, 0, 30, 12], 3001, draft, kind="chain")
    logits = (c["logits"] * 40).round()  # (whole numbers: equal ones are equal)
    logits[:, ::7] = -math.inf
    logits[:, [0, 70]] = 0.0
    rows, top = torch.arange(len(logits)), torch.tensor(c["tokens"]).roll(-1)
    logits[rows, top] = logits.amax(1)  # a drafted token shares the first place
    c["logits"] = logits
    for scale in (0.3, 1.0):
        c["accept"] = (rng.random(len(logits)) * scale).astype(np.float32)
        check_verify(ops, c, temperature)


@pytest.mark.parametrize("V", [5, 58, 20000])
def test_a_rest_of_one_token_refusal_after_refusal(ops, V):
    """p has 1e-8 on a token and all else on another, q more of the first, up to 1e-3.  A child of the first token
    is refused; what is left is the other token alone, and of p's 1e-8 nothing: no child of the first is kept any more,
    however small its uniform, and the other one is drawn."""
    x, y = 1, V - 2
    parents, uniforms = [-1] + [0] * 12, [0.0] + [0.9] * 6 + [1e-3] * 6
    logits = torch.full((13, V), -math.inf, device="cuda")
    logits[:, x], logits[:, y] = math.log(1e-8), 0.0
    for b in (2e-7, 1.5e-6, 3e-6, 1e-5, 7e-5, 1e-4, 1e-3):
        probs = torch.zeros(13, V, device="cuda")
        probs[:, x], probs[:, y] = b, 1 - b
        for draw in (0.0, 0.4, 0.99):
            got = ops.verify_drafts(logits, torch.full((13,), x, device="cuda"), i32(parents), i32([0, 13]),
                                    torch.tensor(uniforms, device="cuda"), torch.tensor([draw], device="cuda"),
                                    draft_probs=probs, max_path=3)
            assert (got.accepted.tolist(), got.next_token.tolist()) == ([1], [y]), (b, draw)


@pytest.mark.parametrize("V", [5, 58, 1525, 20000])
@pytest.mark.parametrize("near", [1e-4, 1e-3, 0.3])
def test_refusal_after_refusal_of_a_draft_that_is_nearly_the_target(ops, V, near):
    """Rows with most of the probability on one token, drafts near them, and children that the draft would hardly have
    drawn, refused one after another: what is left of p is 1e-3 to 1e-7 each time, and is divided by itself each time."""
    rng = np.random.default_rng(V)
    for spread in (8.0, 14.0):
        fresh = [20, 7, 3, 12, 25, 2, 9, 16]
        c = verify_case(rng, fresh, V, near, kind="forest", spread=1.0, few=2)
        rows = np.arange(len(c["tokens"]))
        top = rng.integers(0, V, len(rows))
        logits = c["logits"].double().numpy()
        logits[rows, top] += spread
        bent = logits + rng.normal(size=logits.shape) * near
        probs = np.exp(bent - bent.max(1, keepdims=True))
        c["logits"] = torch.tensor(logits, dtype=torch.float32)
        c["probs"] = torch.tensor(probs / probs.sum(1, keepdims=True), dtype=torch.float32)
        c["tokens"] = rng.integers(0, V, len(rows))
        c["accept"] = (0.5 + 0.49 * c["accept"]).astype(np.float32)
        check_verify(ops, c, 1.0)


# ---------------------------------------------------------------------------------------------
# paged_keep
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("R,slots,Hkv,D", [(520, 32, 32, 128), (1100, 80, 8, 128), (3000, 12, 12, 64)])
def test_keep_of_many_requests_of_many_heads(ops, in_place, R, slots, Hkv, D):
    """More blocks than 2^16 (but for the last): every slot's and head's move, the lengths and
    the counter, twice."""
    page, g = 16, torch.Generator("cuda").manual_seed(R)
    kp, vp = (torch.zeros(slots, R + 1, Hkv, page, D, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    table = torch.randperm(R, device="cuda", generator=g).to(torch.int32).view(R, 1)
    new, cached = torch.full((R,), 6, device="cuda", dtype=torch.int32), torch.full((R,), 3, device="cuda", dtype=torch.int32)
    path, kept = i32([[0, 2, 5]] * R), i32([3, 2, 1, 0] * (R // 4))
    queue, state = torch.full((R + 1,), R, device="cuda", dtype=torch.int32), torch.tensor([0, 1], device="cuda")
    lens = cached.clone()
    for turn in range(2):
        want = []
        for pool in (kp, vp):
            pool[:, :, :, 3 + 2 * turn:9 + 2 * turn] = torch.randn(Hkv, 6, D, device="cuda", dtype=torch.bfloat16, generator=g)
            pool[:, :, :, 3 + 2 * turn:9 + 2 * turn] += torch.arange(R + 1, device="cuda").view(1, -1, 1, 1, 1) % 7
        cached = lens.clone() if turn == 0 else torch.full_like(lens, 5)
        start = cached.clone()
        before = [pool.clone() for pool in (kp, vp)]
        out = dict(free_state_out=state, seqlens_out=cached) if in_place else {}
        state, lens = ops.paged_keep(path, kept, cached, new, table, queue, state, kp, vp, **out)
        assert torch.equal(lens, start + kept) and state.tolist() == [0, 1]
        at = int(start[0])
        rows = table[:, 0].long()
        for pool, old in zip((kp, vp), before):
            for i, src in ((1, 2), (2, 5)):
                moves = rows[kept > i]
                old[:, moves, :, at + i] = old[:, moves, :, at + src]
            assert torch.equal(pool, old)
        del before
