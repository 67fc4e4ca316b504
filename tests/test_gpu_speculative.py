"""PagedKVCache's trees, forks and kept paths, and the speculative-decoding example, on the GPU."""
import importlib.util
import os

import numpy as np
import pytest
import torch

from conftest import REPO

pytestmark = pytest.mark.gpu

PAGE = 16


def _load(folder, name):
    spec = importlib.util.spec_from_file_location(name, os.path.join(REPO, folder, name + ".py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


@pytest.fixture(scope="module")
def example():
    return _load("examples", "paged_speculative")


def make(n_pages=60, rows=6, max_len=200, slots=2):
    from modelcore_b200 import PagedKVCache
    return PagedKVCache(n_pages, PAGE, 2, 64, slots, rows, max_len, "cuda")


def check(cache):
    """The cache's state read from the GPU: lengths, every page free or held by as many rows as it says."""
    from modelcore_b200 import ops
    code, what = ops.device_error()
    assert code == 0, what
    lens = cache.host_lens()
    assert cache.cache_seqlens.tolist() == lens.tolist()
    head, tail = cache.free_state.tolist()
    assert tail - head == cache.free_page_count()
    queue, table = cache.free_pages.tolist(), cache.block_table.tolist()
    free = [queue[x % cache.n_pages] for x in range(head, tail)]
    holders = {}
    for r, n in enumerate(lens.tolist()):
        for p in table[r][:-(-n // PAGE)]:
            holders[p] = holders.get(p, 0) + 1
        assert n % PAGE == 0 or holders[table[r][n // PAGE]] == 1
    assert sorted(free + list(holders)) == list(range(cache.n_pages))
    assert cache.page_shares.tolist() == [holders.get(p, 1) - 1 for p in range(cache.n_pages)]


def rows_of(cache, slot=0):
    """Every row's keys, (length, Hkv, D)."""
    out = []
    for r, n in enumerate(cache.host_lens().tolist()):
        pages = cache.block_table[r, :-(-n // PAGE)].long()
        out.append(cache.k_pages[slot][pages].transpose(1, 2).reshape(-1, 2, 64)[:n])
    return out


def put(cache, step, g):
    """Random keys and values for a step's tokens, in every slot."""
    cos, sin = torch.ones(400, 32, device="cuda", dtype=torch.bfloat16), torch.zeros(400, 32, device="cuda",
                                                                                     dtype=torch.bfloat16)
    for slot in range(cache.n_slots):
        x = [torch.randn(step.num_tokens, 2, 64, device="cuda", dtype=torch.bfloat16, generator=g) for _ in range(3)]
        cache.append(slot, *x, step, cos, sin, rotate_k=False)


def test_a_long_life_of_trees_forks_and_releases():
    rng = np.random.default_rng(0)
    g = torch.Generator("cuda").manual_seed(0)
    cache = make()
    shared = 0
    for _ in range(80):
        lens = cache.host_lens()
        want = rows_of(cache)
        what = rng.random()
        if what < 0.25 and lens.any():
            live = np.nonzero(lens)[0]
            source = [int(rng.choice(live)) if rng.random() < 0.5 else r for r in range(6)]
            if rng.random() < 0.3:
                source[int(rng.integers(0, 6))] = -1
            cache.fork(source)
            want = [want[s] if s >= 0 else want[0][:0] for s in source]
        elif what < 0.4:
            gone = np.nonzero((rng.random(6) < 0.3) | (lens > 140))[0]
            cache.release(gone)
            want = [w[:0] if r in gone else w for r, w in enumerate(want)]
        else:
            new = np.where((rng.random(6) < 0.7) & (lens < 150), rng.integers(1, 20, 6), 0)
            while cache.pages_needed(new) > cache.free_page_count():
                new[rng.integers(0, 6)] = 0
            parents = [int(rng.integers(-1, t)) if t else -1 for n in new for t in range(n)]
            pad = int(rng.integers(0, 3))
            step = cache.plan(new, int(new.sum()) + pad, parents=parents + [-1] * pad)
            put(cache, step, g)
            fresh = [w[n:] for w, n in zip(rows_of_step(cache, new), lens)]
            kept = [int(rng.integers(0, n + 1)) if rng.random() < 0.9 else -1 for n in new]
            path = np.full((6, 20), -1)
            for r, (n, k) in enumerate(zip(new, kept)):
                path[r, :max(k, 0)] = np.sort(rng.permutation(n)[:max(k, 0)])
            got = cache.keep(step, torch.tensor(path, dtype=torch.int32, device="cuda"),
                             torch.tensor(kept, dtype=torch.int32, device="cuda"))
            assert got == [int(n) if k < 0 else k for n, k in zip(new, kept)]
            want = [torch.cat([w, f if k < 0 else f[path[r, :k]]]) for r, (w, f, k) in enumerate(zip(want, fresh, kept))]
        check(cache)
        assert all(torch.equal(a, b) for a, b in zip(rows_of(cache), want))
        shared = max(shared, int(cache.page_shares.sum()))
    assert shared > 5


def rows_of_step(cache, new):
    """rows_of with a planned step's tokens."""
    lens = cache._host_lens
    cache._host_lens = lens + new
    out = [x.clone() for x in rows_of(cache)]
    cache._host_lens = lens
    return out


def test_refusals():
    cache = make(10, 4, 150, 1)
    cache.advance(cache.plan([100]))
    with pytest.raises(RuntimeError, match="source must name"):
        cache.fork([4])
    with pytest.raises(RuntimeError, match="source must name"):
        cache.fork([-2])
    cache.advance(cache.plan([0, 45]))  # the pages are all taken
    with pytest.raises(RuntimeError, match="copies 1 pages and 0 are free"):
        cache.fork([0, 1, 1])
    with pytest.raises(RuntimeError, match="a row for each"):
        step = cache.plan([1])
        cache.keep(step, torch.zeros(3, 2, dtype=torch.int32, device="cuda"),
                   torch.zeros(3, dtype=torch.int32, device="cuda"))
    with pytest.raises(RuntimeError, match="parents must name"):
        cache.plan([2], parents=[-1])
    check(cache)


def test_a_planned_step_is_dropped_by_a_fork():
    cache = make()
    cache.advance(cache.plan([40, 10]))
    step = cache.plan([20])
    cache.fork([0, 1, 0])
    with pytest.raises(RuntimeError, match="not the planned one"):
        cache.advance(step)
    check(cache)
    cache.advance(cache.plan([20, 1, 3]))
    check(cache)


@pytest.mark.parametrize("head_dim,heads,kv_heads,samples", [(64, 8, 2, 3), (128, 4, 4, 1)])
def test_speculative_tokens_are_the_model_s_own(example, head_dim, heads, kv_heads, samples):
    """Greedy: every token, drafted or not, is the model's own choice over the same text, its logit the largest up to the
    two paths' difference (test_gpu_paged_serving.py derives the 0.15)."""
    from modelcore_b200 import ops
    alone = _load("tests", "test_gpu_paged_serving").alone
    rng = np.random.default_rng(0)
    model = example.SpeculativeDecoder(head_dim=head_dim, heads=heads, kv_heads=kv_heads)
    prompts = [(rng.integers(0, model.vocab, 9).tolist() * 40)[:int(n)] for n in rng.integers(1, 300, 5)]
    ends = []
    tokens, steps, drafted = example.generate(model, prompts, samples=samples, max_tokens=30, chunk=100,
                                              on_step=lambda c, t, r: (check(c), ends.append(c.free_page_count())))
    assert all(len(t) == 30 for t in tokens) and len(tokens) == 5 * samples and steps <= 29
    for r, t in enumerate(tokens):
        prompt = prompts[r // samples]
        logits = alone(model, prompt + t)[len(prompt) - 1:-1]
        picked = logits.gather(1, torch.tensor(t, device="cuda")[:, None])[:, 0]
        assert (logits.amax(-1) - picked).max() < 0.15
    code, what = ops.device_error()
    assert code == 0, what


def test_sampled_text_and_its_pages(example):
    model = example.SpeculativeDecoder()
    caches = []
    tokens, steps, drafted = example.generate(model, [[1, 2, 3] * 30, [5] * 50], samples=4, max_tokens=20, temperature=0.5,
                                              on_step=lambda c, t, r: (check(c), caches.append(c)))
    assert all(len(t) == 20 and all(0 <= x < model.vocab for x in t) for t in tokens)
    assert caches[-1].free_page_count() == caches[-1].n_pages and not caches[-1].host_lens().any()
    check(caches[-1])


# ---------------------------------------------------------------------------------------------
# captured, on other streams
def tree_step(seed=0, R=3, T=12, past=100):
    """The inputs of a step of trees: (arguments of each operator in turn)."""
    g = torch.Generator("cuda").manual_seed(seed)
    ints = dict(dtype=torch.int32, device="cuda")
    page, Hq, Hkv, D, V = 16, 8, 2, 64, 501
    n_pages = R * 8 + 9
    lens = torch.randint(past, past + 10, (R,), generator=g, **ints)
    order = torch.randperm(n_pages, device="cuda", generator=g).to(torch.int32)
    table = torch.full((R, 9), -1, **ints)
    table[:, :7] = order[:7 * R].view(R, 7)
    queue = torch.full((n_pages,), -1, **ints)
    queue[:n_pages - 7 * R] = order[7 * R:]
    pool = lambda: torch.randn(2, n_pages, Hkv, page, D, device="cuda", dtype=torch.bfloat16, generator=g)
    parents = (torch.rand(R * T, device="cuda", generator=g) * (torch.arange(R * T, device="cuda") % T)).to(torch.int32)
    parents[::T] = -1
    return dict(lens=lens, new=torch.full((R,), T, **ints), table=table, queue=queue,
                state=torch.tensor([0, n_pages - 7 * R], device="cuda"), k=pool(), v=pool(), parents=parents,
                q=torch.randn(R * T, Hq, D, device="cuda", dtype=torch.bfloat16, generator=g),
                logits=torch.randn(R * T, V, device="cuda", generator=g) * 4,
                tokens=torch.randint(0, V, (R * T,), device="cuda", generator=g),
                accept=torch.rand(R * T, device="cuda", generator=g) * 0.01, draws=torch.rand(R, device="cuda", generator=g),
                shares=torch.zeros(n_pages, **ints), source=torch.arange(R, **ints).flip(0) // 2)


def run_step(ops, s):
    page = s["k"].shape[3]
    p = ops.page_plan(s["lens"], s["new"], s["table"], s["queue"], s["state"], page_size=page, num_tokens=s["q"].shape[0])
    t = ops.draft_tree(s["parents"], p.cu_new, s["lens"], max_tree=32)
    y = ops.paged_tree_attn(s["q"], s["k"][0], s["v"][0], s["table"], s["lens"], p.cu_new, t.positions, t.mask)
    z = ops.paged_tree_attn(s["q"], s["k"][1], s["v"][1], s["table"], s["lens"], p.cu_new, t.positions, t.mask, max_new=12)
    v = ops.verify_drafts(s["logits"], s["tokens"], s["parents"], p.cu_new, s["accept"], s["draws"], max_path=12)
    state, lens = ops.paged_keep(v.path, v.accepted, s["lens"], s["new"], s["table"], s["queue"], p.free_state, s["k"],
                                 s["v"])
    f = ops.page_fork(s["source"], lens, s["table"], s["shares"], s["queue"], state, s["k"], s["v"])
    return [*t, y, z, *v, state, lens, *f, s["queue"], s["k"], s["v"]]


def clone(s):
    return {k: v.clone() for k, v in s.items()}


def test_a_step_captured_and_replayed():
    from modelcore_b200 import ops
    first, second = tree_step(0), tree_step(1)
    want = [[x.clone() for x in run_step(ops, clone(s))] for s in (first, second)]
    static = clone(first)
    graph = torch.cuda.CUDAGraph()
    run_step(ops, clone(first))
    with torch.cuda.graph(graph):
        got = run_step(ops, static)
    for s, w in ((first, want[0]), (second, want[1]), (first, want[0])):
        for k in static:
            static[k].copy_(s[k])
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, w))
    code, what = ops.device_error()
    assert code == 0, what


def test_two_graphs_and_two_streams_at_once():
    from modelcore_b200 import ops
    steps = [tree_step(s, R=5 + s) for s in range(2)]
    want = [[x.clone() for x in run_step(ops, clone(s))] for s in steps]
    streams = [torch.cuda.Stream() for _ in steps]
    torch.cuda.synchronize()
    for _ in range(5):
        got, held = [], []
        for st, s in zip(streams, steps):
            with torch.cuda.stream(st):
                held.append(clone(s))
                got.append(run_step(ops, held[-1]))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))
    static, graphs, got = [clone(s) for s in steps], [torch.cuda.CUDAGraph() for _ in steps], []
    for gr, s in zip(graphs, static):
        with torch.cuda.graph(gr):
            got.append(run_step(ops, s))
    for _ in range(5):
        for s, x in zip(static, steps):
            for k in s:
                s[k].copy_(x[k])
        torch.cuda.synchronize()
        for st, gr in zip(streams, graphs):
            with torch.cuda.stream(st):
                gr.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))


def test_arguments_that_do_not_fit():
    from modelcore_b200 import ops
    s = tree_step()
    cpu = s["lens"].cpu()
    p = ops.page_plan(s["lens"], s["new"], s["table"], s["queue"], s["state"], page_size=16, num_tokens=36)
    t = ops.draft_tree(s["parents"], p.cu_new, s["lens"], max_tree=32)
    attn = lambda **kw: ops.paged_tree_attn(*{**dict(q=s["q"], k=s["k"][0], v=s["v"][0], table=s["table"], lens=s["lens"],
                                                     cu=p.cu_new, pos=t.positions, mask=t.mask), **kw}.values())
    verify = lambda **kw: ops.verify_drafts(**{**dict(logits=s["logits"], tokens=s["tokens"], parents=s["parents"],
                                                      cu_new=p.cu_new, accept=s["accept"], draws=s["draws"], max_path=4), **kw})
    v = verify()
    keep = lambda **kw: ops.paged_keep(**{**dict(path=v.path, accepted=v.accepted, cache_seqlens=s["lens"], new_lens=s["new"],
                                                 block_table=s["table"], free_pages=s["queue"], free_state=p.free_state,
                                                 k_pages=s["k"], v_pages=s["v"]), **kw})
    fork = lambda **kw: ops.page_fork(**{**dict(source=s["source"], cache_seqlens=s["lens"], block_table=s["table"],
                                                shares=s["shares"], free_pages=s["queue"], free_state=s["state"],
                                                k_pages=s["k"], v_pages=s["v"]), **kw})
    half = s["k"].half()
    for call, words in (
            (lambda: ops.draft_tree(s["parents"], p.cu_new, s["lens"], max_tree=0), "max_tree"),
            (lambda: ops.draft_tree(s["parents"], p.cu_new, s["lens"], max_tree=257), "max_tree"),
            (lambda: ops.draft_tree(s["parents"].long(), p.cu_new, s["lens"], max_tree=32), "parents"),
            (lambda: ops.draft_tree(s["parents"], p.cu_new[:-1], s["lens"], max_tree=32), "cu_new"),
            (lambda: attn(mask=t.mask[:-1]), "mask"), (lambda: attn(mask=t.mask.expand(-1, 9).contiguous()), "words 9"),
            (lambda: attn(pos=t.positions[:-1]), "positions"), (lambda: attn(q=s["q"].half()), "q must be"),
            (lambda: attn(lens=cpu), "cache_seqlens"), (lambda: attn(q=s["q"][:, :7]), "divisible"),
            (lambda: verify(logits=s["logits"].half()), "logits"), (lambda: verify(tokens=s["tokens"].int()), "tokens"),
            (lambda: verify(temperature=-1.0), "temperature"), (lambda: verify(max_path=0), "max_path"),
            (lambda: verify(draws=s["draws"][:-1]), "draws"), (lambda: verify(logits=s["logits"].t()), "tokens|rows"),
            (lambda: verify(draft_probs=s["logits"][:, 1:]), "draft_probs"),
            (lambda: verify(draft_probs=s["logits"].double()), "draft_probs"),
            (lambda: keep(k_pages=half, v_pages=half), "k_pages"), (lambda: keep(path=v.path[:-1]), "path"),
            (lambda: keep(free_pages=s["queue"][:-1]), "free_pages"), (lambda: keep(accepted=cpu), "accepted"),
            (lambda: fork(shares=s["shares"][:-1]), "shares"), (lambda: fork(source=s["source"].long()), "source"),
            (lambda: fork(v_pages=s["v"][0]), "v_pages"), (lambda: fork(block_table_out=s["table"][:, 1:]), "block_table_out")):
        with pytest.raises(RuntimeError, match=words):
            call()
    code, what = ops.device_error()
    assert code == 0, what
