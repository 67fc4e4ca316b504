"""What the operators of speculative decoding and of shared pages are measured on: the cases, their
inputs, and each operator in its plain form beside the call a user makes.

  tree      draft_tree: positions and ancestor masks of trees of drafted tokens, from their parents
  attn      paged_tree_attn: attention of such trees over a paged cache
  verify    verify_drafts: which drafted tokens the target's probabilities keep, and the next token
  keep      paged_keep: the kept path's keys and values moved together, the other pages given back
  fork      page_fork: rows become copies of rows, sharing the pages that are full

The lengths of a case and the shapes of its paths follow from the case alone ("lens"), the values, the
trees' branches and the placement of the pages from the seed."""
import math
import random

import torch

own = False

SCALE = 1.2


def listed():
    return [
        # one step of 64 requests with 16 drafted tokens each
        dict(name="tree_64", op="tree", rows=64, nodes=16, wide=4, chunks=0, chunk=0, most=32, lo=512, hi=1023, lens=1,
             pad=0),
        # a full server with large trees, prompt chunks beside them, a padded token count
        dict(name="tree_1000", op="tree", rows=1000, nodes=200, wide=7, chunks=9, chunk=700, most=256, lo=100, hi=8191,
             lens=2, pad=37),
        # three requests of the quickstart model (12 heads of 64): the smallest step
        dict(name="attn_tree_3", op="attn", rows=3, nodes=8, wide=3, chunks=0, chunk=0, most=32, lo=500, hi=1023, hq=12,
             hkv=12, d=64, page=16, window=-1, lens=3),
        # an ordinary batch of the grouped-query model
        dict(name="attn_tree_32", op="attn", rows=32, nodes=16, wide=4, chunks=0, chunk=0, most=32, lo=1024, hi=8192,
             hq=16, hkv=4, d=128, page=64, window=-1, lens=4),
        # large trees over long requests, small pages
        dict(name="attn_tree_long", op="attn", rows=13, nodes=63, wide=9, chunks=0, chunk=0, most=64, lo=8192, hi=32700,
             hq=32, hkv=8, d=128, page=16, window=-1, lens=5),
        # the window layers' step: trees of odd sizes beside two prompt chunks
        dict(name="attn_tree_window", op="attn", rows=24, nodes=41, wide=5, chunks=2, chunk=300, most=64, lo=0, hi=6000,
             hq=16, hkv=4, d=128, page=32, window=1024, lens=6),
        # three requests, each drafted token the draft's best guess: latency
        dict(name="verify_3", op="verify", rows=3, nodes=8, wide=2, vocab=32768, temperature=0.8, probs=False,
             dtype="float32", lens=7),
        # a batch whose drafted tokens were drawn from the draft's probabilities, a large vocabulary
        dict(name="verify_64", op="verify", rows=64, nodes=16, wide=3, vocab=131071, temperature=1.0, probs=True,
             dtype="float32", lens=8),
        # the quickstart model's twelve layers, a few requests
        dict(name="keep_8", op="keep", rows=8, nodes=16, wide=4, lo=500, hi=1000, slots=12, hkv=12, d=64, page=16,
             lens=9),
        # the grouped-query model's layers, a full batch
        dict(name="keep_128", op="keep", rows=128, nodes=47, wide=6, lo=100, hi=400, slots=24, hkv=4, d=128, page=32,
             lens=10),
        # one prompt becomes eight samples
        dict(name="fork_16", op="fork", rows=16, group=8, prefix=700, tail=0, slots=12, hkv=12, d=64, page=16, beam=False,
             lens=11),
        # a beam search's step: every group of four rows goes on with some of its rows
        dict(name="fork_beam_256", op="fork", rows=256, group=4, prefix=1500, tail=200, slots=12, hkv=4, d=128, page=64,
             beam=True, lens=12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tree", "attn", "attn", "attn", "verify", "verify", "keep", "fork"])
    page = rng.choice([16, 32, 64, 128])
    lens = rng.randrange(1 << 30)
    wide = rng.randint(1, 9)
    hq, hkv, d = rng.choice([(12, 12, 64), (16, 4, 128), (32, 8, 128), (6, 2, 64), (15, 5, 128), (8, 1, 64),
                             (24, 24, 128)])
    while True:
        rows = _log(rng, 1, 1000 if op == "tree" else 128)
        if op in ("tree", "attn"):
            most = rng.choice([32, 64, 128, 256])
            lo = _log(rng, 1, 8000)
            chunks = rng.choice([0, 0, rng.randint(0, max(1, rows // 8))])
            c = dict(op=op, rows=rows, nodes=_log(rng, 1, most), wide=wide, chunks=chunks,
                     chunk=_log(rng, most + 1, 700) if chunks else 0, most=most, lo=lo, hi=lo + _log(rng, 1, 16000),
                     lens=lens)
            if op == "tree":
                return c | dict(pad=rng.choice([0, 0, 5]))
            c |= dict(hq=hq, hkv=hkv, d=d, page=page, window=rng.choice([-1, -1, -1, 5, 128, 1024, 4000]))
            longest = c["hi"] + max(c["nodes"], c["chunk"])
            w = work(c)
            # no more work than the largest listed case, and a plain form whose padded scores fit
            if (w["flops"] <= 0.26e12 and w["bytes"] <= 1e9 and rows * longest * hkv * d <= 0.6e9
                    and rows * max(c["nodes"], c["chunk"]) * hq * longest <= 2.5e9):
                return c
        elif op == "verify":
            c = dict(op=op, rows=rows, nodes=_log(rng, 1, 64), wide=wide, vocab=_log(rng, 500, 200000),
                     temperature=rng.choice([0.0, 0.7, 1.0, 1.3]), probs=rng.random() < 0.5,
                     dtype=rng.choice(["float32", "bfloat16"]), lens=lens)
            if rows * c["nodes"] * c["vocab"] <= 1.3e8:
                return c
        elif op == "keep":
            lo = _log(rng, 1, 1000)
            c = dict(op=op, rows=rows, nodes=_log(rng, 1, 128), wide=wide, lo=lo, hi=lo + _log(rng, 1, 300),
                     slots=_log(rng, 1, 32), hkv=hkv, d=d, page=page, lens=lens)
            if rows * (_pages(c["hi"] + c["nodes"], page) + 1) * page * c["slots"] * hkv * d <= 1e9:
                return c
        else:
            c = dict(op=op, rows=rows, group=rng.randint(1, min(rows, 9)), prefix=_log(rng, 1, 4000),
                     tail=rng.choice([0, _log(rng, 1, 300)]), slots=_log(rng, 1, 32), hkv=hkv, d=d, page=page,
                     beam=rng.random() < 0.6, lens=lens)
            held = rows * _pages(c["tail"] + 1, page) + rows // c["group"] * _pages(c["prefix"], page)
            if (held + rows) * page * c["slots"] * hkv * d <= 1e9:
                return c


def _pages(n, page):
    return -(-n // page)


def _lengths(case):
    """(cached tokens, new tokens) of every request, as lists."""
    rng = random.Random(case["lens"])
    rows = case["rows"]
    cached = [rng.randint(case["lo"], case["hi"]) for _ in range(rows)]
    # most trees are full; some requests are near their end and draft fewer
    fresh = [case["nodes"] if rng.random() < 0.7 else rng.randint(1, case["nodes"]) for _ in range(rows)]
    for r in rng.sample(range(rows), case.get("chunks", 0)):
        fresh[r] = case["chunk"]
    return cached, fresh


def _paths(case, fresh):
    """How many tokens of each request's tree are kept, its root among them."""
    rng = random.Random(case["lens"] + 1)
    levels = [_pages(n - 1, case["wide"]) + 1 for n in fresh]
    return [1 + min(sum(rng.random() < 0.7 for _ in range(8)), n - 1) for n in levels]


def _moves(case, fresh):
    """(kept, in place) of each request: of its kept tokens the first ones -- the draft's best guesses come
    first -- are where they belong, the others behind all the places of kept ones, so that a pass can be
    repeated."""
    rng = random.Random(case["lens"] + 2)
    return [(n, min(n, max(2 * n - count, rng.randint(1, 2)))) for n, count in zip(_paths(case, fresh), fresh)]


def _trees(case, fresh, gen):
    """Parents (N,) of trees in levels of `wide` tokens under a root, each token's parent drawn from the
    level before; -1 for roots, and a prompt chunk's tokens follow one another."""
    wide = case["wide"]
    n = torch.tensor(fresh, device="cuda")
    local = torch.arange(sum(fresh), device="cuda") - (n.cumsum(0) - n).repeat_interleave(n)
    level = (local - 1) // wide + 1
    up = 1 + (level - 2) * wide + torch.randint(0, wide, local.shape, device="cuda", generator=gen)
    parent = torch.where(local == 0, -1, torch.where(level <= 1, 0, up))
    if case.get("chunks"):
        parent = torch.where(n.repeat_interleave(n) > case["most"], local - 1, parent)
    return parent.to(torch.int32), local


def _normed(shape, gen):
    """Vectors as the append leaves them: rms 1.2."""
    x = torch.randn(shape, device="cuda", dtype=torch.bfloat16, generator=gen)
    r = x.float().square().mean(-1, keepdim=True).rsqrt_().mul_(SCALE).to(torch.bfloat16)
    return x.mul_(r)


def _offsets(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return torch.tensor(cu, dtype=torch.int32, device="cuda")


def _tables(counts, spare, gen):
    """A block table of counts[r] pages each, in shuffled order, and the order of all pages."""
    n_pages, width = sum(counts) + spare, max(counts) + 1
    order = torch.randperm(n_pages, device="cuda", generator=gen).to(torch.int32)
    n = torch.tensor(counts, device="cuda")
    col = torch.arange(width, device="cuda")[None]
    index = (col + (n.cumsum(0) - n)[:, None]).clamp_(max=n_pages - 1)
    return torch.where(col < n[:, None], order[index], -1).contiguous(), order


def _queue(order, used, head):
    """The free-page queue and its counters: the pages of `order` from `used` on, from entry `head`."""
    total = order.numel()
    queue = torch.full((total,), -1, dtype=torch.int32, device="cuda")
    queue[(head + torch.arange(total - used, device="cuda")) % total] = order[used:]
    return queue, torch.tensor([head, head + total - used], dtype=torch.int64, device="cuda")


def prepare(case, seed):
    op = case["op"]
    gen = torch.Generator("cuda").manual_seed(seed)
    s = dict(case=case)
    ints = dict(dtype=torch.int32, device="cuda")
    if op == "fork":
        return _prepare_fork(s, gen, seed)
    if op == "verify":
        return _prepare_verify(s, gen)
    cached, fresh = _lengths(case)
    s |= dict(cached=torch.tensor(cached, **ints), fresh=torch.tensor(fresh, **ints), cu=_offsets(fresh))
    parents, _ = _trees(case, fresh, gen)
    if op == "tree":
        # (what is read is the lengths' values alone: from the seed)
        return s | dict(parents=torch.cat([parents, parents.new_full((case["pad"],), -1)]),
                        cached=torch.randint(case["lo"], case["hi"] + 1, (case["rows"],), generator=gen, **ints))
    page, hkv, d = case["page"], case["hkv"], case["d"]
    counts = [_pages(a + b, page) for a, b in zip(cached, fresh)]
    s["table"], order = _tables(counts, 5, gen)
    if op == "keep":
        s["queue"], s["state"] = _queue(order, sum(counts), 3 * order.numel() - 2)
        rng = random.Random(seed)
        kept = _moves(case, fresh)
        path = [list(range(stay)) + sorted(rng.sample(range(n, count), n - stay)) + [-1] * (case["nodes"] - n)
                for (n, stay), count in zip(kept, fresh)]
        pool = (case["slots"], order.numel(), hkv, page, d)
        return s | dict(path=torch.tensor(path, **ints), kept=torch.tensor([n for n, _ in kept], **ints), page=page,
                        k_pages=torch.randn(pool, device="cuda", dtype=torch.bfloat16, generator=gen),
                        v_pages=torch.randn(pool, device="cuda", dtype=torch.bfloat16, generator=gen))
    pool = (order.numel(), hkv, page, d)
    t = dict(s, parents=parents)
    s["positions"], s["mask"] = _plain_tree(t)
    return s | dict(q=_normed((sum(fresh), case["hq"], d), gen), k_pages=_normed(pool, gen),
                    v_pages=torch.randn(pool, device="cuda", dtype=torch.bfloat16, generator=gen), page=page,
                    most=max(fresh), longest=max(a + b for a, b in zip(cached, fresh)))


def _prepare_verify(s, gen):
    """Logits like a target's (a few tokens hold most of the probability) and drafts that it keeps for a
    path as long as _paths says."""
    case = s["case"]
    rows, vocab = case["rows"], case["vocab"]
    _, fresh = _lengths(dict(case, lo=1, hi=1))
    n = sum(fresh)
    parents, local = _trees(case, fresh, gen)
    kept = torch.tensor(_paths(case, fresh), device="cuda")
    count = torch.tensor(fresh, device="cuda")
    first = count.cumsum(0) - count
    start = first.repeat_interleave(count)
    tokens = torch.randint(0, vocab, (n,), device="cuda", generator=gen)
    temperature = case["temperature"] or 1.0
    logits = torch.randn(n, vocab, device="cuda", generator=gen)
    parent = (start + parents).clamp_(min=0)
    # on the path: each level's token of which the one before is the parent (the last such one)
    line = torch.zeros(n, dtype=torch.bool, device="cuda")
    at = first.clone()
    index = torch.arange(n, device="cuda")
    for _ in range(int(kept.max()) - 1):
        child = torch.full((n,), -1, device="cuda").scatter_reduce_(
            0, torch.where(local > 0, parent, index), torch.where(local > 0, index, -1), "amax")
        at = torch.where(child[at] >= 0, child[at], at)
        line[at] = True
    depth = (local - 1) // case["wide"] + 1
    line &= (depth > 0) & (depth < kept.repeat_interleave(count))
    # a drafted token has some 0.05 to 0.5 of its parent's probability, or nearly all of it on the path
    share = torch.rand(n, device="cuda", generator=gen) * 0.45 + 0.05
    boost = math.log(vocab) + 0.5 / temperature ** 2 + torch.log(torch.where(line, 20.0, share / (1 - share)))
    drafted = local > 0
    logits.view(-1).scatter_reduce_(0, (parent * vocab + tokens)[drafted], (boost * temperature)[drafted], "amax")
    if case["probs"]:
        noise = torch.randn(n, vocab, device="cuda", generator=gen).mul_(0.3).add_(logits, alpha=1 / temperature)
        s["probs"] = torch.softmax(noise, -1)
    else:
        s["probs"] = None
    u = torch.rand(n, device="cuda", generator=gen)
    # the path's tokens are kept, those after it are not
    s["accept"] = torch.where(line, u * 0.5, 1 - 0.05 * u).clamp_(max=1 - 2.0 ** -24)
    return s | dict(logits=logits.to(getattr(torch, case["dtype"])), tokens=tokens, parents=parents, cu=_offsets(fresh),
                    last=torch.rand(rows, device="cuda", generator=gen), most=max(fresh),
                    depth=_pages(case["nodes"] - 1, case["wide"]) + 1, temperature=case["temperature"])


def _forks(case):
    """(lengths, sources) of every row, as lists: groups of rows that share a prefix and went on each for
    itself; a beam search's rows go on with one of their group's, the others with the group's first."""
    rng = random.Random(case["lens"])
    rows, group = case["rows"], case["group"]
    lens, source, prefix = [0] * rows, [-1] * rows, [0] * rows
    for a in range(0, rows, group):
        shared = rng.randint((case["prefix"] + 1) // 2, case["prefix"])
        mine = range(a, min(a + group, rows))
        for r in mine:
            # samples: the prompt's row is forked into the empty rows beside it
            if case["beam"] or r == a:
                lens[r] = shared + (rng.randint(0, case["tail"]) if case["beam"] else 0)
                prefix[r] = shared // case["page"]
            source[r] = rng.choice(mine) if case["beam"] else a
        if rng.random() < 0.1:  # a group that has finished
            for r in mine:
                source[r] = -1
    return lens, source, prefix


def _prepare_fork(s, gen, seed):
    case = s["case"]
    page, rows = case["page"], case["rows"]
    lens, source, prefix = _forks(case)
    table, owners, used = [], {}, 0
    for r in range(rows):
        a = r - r % case["group"]
        mine = []
        for j in range(_pages(lens[r], page)):
            if j < prefix[r] and r != a:
                mine.append(table[a][j])
            else:
                mine.append(used)
                used += 1
            owners[mine[-1]] = owners.get(mine[-1], 0) + 1
        table.append(mine)
    total = used + rows + 3
    order = torch.randperm(total, device="cuda", generator=gen).to(torch.int32)
    width = max(len(t) for t in table) + 2
    at = torch.tensor([t + [0] * (width - len(t)) for t in table], device="cuda")
    held = torch.tensor([len(t) for t in table], device="cuda")
    ints = dict(dtype=torch.int32, device="cuda")
    shares = torch.zeros(total, **ints)
    shares[order[torch.tensor(list(owners), device="cuda")].long()] = torch.tensor(list(owners.values()), **ints) - 1
    queue, state = _queue(order, used, 5 * total - 1)
    pool = (case["slots"], total, case["hkv"], page, case["d"])
    return s | dict(page=page, source=torch.tensor(source, **ints), cached=torch.tensor(lens, **ints), shares=shares,
                    table=torch.where(torch.arange(width, device="cuda")[None] < held[:, None], order[at], -1).contiguous(),
                    queue=queue, state=state,
                    k_pages=torch.randn(pool, device="cuda", dtype=torch.bfloat16, generator=gen),
                    v_pages=torch.randn(pool, device="cuda", dtype=torch.bfloat16, generator=gen))


# -- one pass ------------------------------------------------------------------------------------
def run(s):
    return (_own if own else _plain)[s["case"]["op"]](s)


def _own_tree(s):
    from modelcore_b200 import ops
    t = ops.draft_tree(s["parents"], s["cu"], s["cached"], max_tree=s["case"]["most"])
    return t.positions, t.mask


def _own_attn(s):
    from modelcore_b200 import ops
    return ops.paged_tree_attn(s["q"], s["k_pages"], s["v_pages"], s["table"], s["cached"], s["cu"], s["positions"],
                               s["mask"], window=s["case"]["window"], max_new=s["most"])


def _own_verify(s):
    from modelcore_b200 import ops
    v = ops.verify_drafts(s["logits"], s["tokens"], s["parents"], s["cu"], s["accept"], s["last"],
                          temperature=s["temperature"], draft_probs=s["probs"], max_path=s["most"])
    return v.accepted, v.path, v.next_token


def _own_keep(s):
    from modelcore_b200 import ops
    state, lens = ops.paged_keep(s["path"], s["kept"], s["cached"], s["fresh"], s["table"], s["queue"], s["state"],
                                 s["k_pages"], s["v_pages"])
    return s["k_pages"], s["v_pages"], s["queue"], state, lens


def _own_fork(s):
    from modelcore_b200 import ops
    f = ops.page_fork(s["source"], s["cached"], s["table"], s["shares"], s["queue"], s["state"], s["k_pages"],
                      s["v_pages"])
    return f.block_table, f.shares, f.free_state, f.seqlens, s["queue"], s["k_pages"], s["v_pages"]


def _row_of(cu, n):
    """The request of every packed token, and whether it has one."""
    t = torch.arange(n, device="cuda")
    row = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    return row.clamp_(max=cu.numel() - 2), t < cu[-1]


def _plain_tree(s):
    most, parents, cu = s["case"]["most"], s["parents"].long(), s["cu"].long()
    n, words = parents.numel(), (most + 31) // 32
    row, live = _row_of(cu, n)
    first = cu[row]
    local = torch.arange(n, device="cuda") - first
    tree = live & ((cu[1:] - cu[:-1])[row] <= 32 * words)
    # every token's ancestors by doubling; the last row is nobody's
    up = torch.cat([torch.where(tree & (parents >= 0), first + parents, n), torch.tensor([n], device="cuda")])
    seen = torch.zeros(n + 1, 32 * words, dtype=torch.bool, device="cuda")
    seen[:n] = (torch.arange(32 * words, device="cuda")[None] == local[:, None]) & tree[:, None]
    for _ in range((32 * words - 1).bit_length()):
        seen |= seen[up]
        up = up[up]
    seen = seen[:n]
    past = s["cached"].long()[row]
    positions = torch.where(live, past + torch.where(tree, seen.sum(-1) - 1, local), -1)
    bits = (seen.view(n, words, 32).long() << torch.arange(32, device="cuda")).sum(-1)
    return positions.to(torch.int32), torch.where(bits >= 1 << 31, bits - (1 << 32), bits).to(torch.int32)


def _plain_attn(s):
    page, window, cached, cu = s["page"], s["case"]["window"], s["cached"].long(), s["cu"].long()
    n, hq, d = s["q"].shape
    hkv, rows, most = s["k_pages"].shape[1], cached.numel(), s["most"]
    width = _pages(s["longest"], page)
    table = s["table"][:, :width].long().clamp(min=0)
    # every request padded to the longest: (rows, Hkv, keys, D)
    k = s["k_pages"][table].transpose(1, 2).reshape(rows, hkv, width * page, d).float()
    v = s["v_pages"][table].transpose(1, 2).reshape(rows, hkv, width * page, d).float()
    t = torch.arange(most, device="cuda")
    token = (cu[:-1, None] + t[None]).clamp(max=n - 1)
    q = s["q"][token].view(rows, most, hkv, hq // hkv, d).permute(0, 2, 1, 3, 4).float()
    score = (q.reshape(rows, hkv, -1, d) @ k.transpose(-1, -2)).mul_(1.0 / math.sqrt(d))
    score = score.view(rows, hkv, most, hq // hkv, width * page)
    # of the new tokens: a tree's by its mask, a chunk's all before; of the cached ones all
    words = s["mask"].shape[1]
    word = s["mask"][token][:, :, (t // 32).clamp(max=words - 1)]
    chunk = (cu[1:] - cu[:-1] > 32 * words)[:, None, None]
    new = torch.where(chunk, t[None, None] <= t[None, :, None], (word >> (t % 32)) & 1 > 0)
    pos = s["positions"].long()[token]
    if window >= 0:
        new = new & (pos[:, :, None] - pos[:, None, :] <= window)
    key = torch.arange(width * page, device="cuda")[None, None]
    past = cached[:, None, None]
    seen = (key < past) & ((pos[..., None] - key <= window) if window >= 0 else True)
    at = (key - past).expand(rows, most, -1)
    count = (cu[1:] - cu[:-1])[:, None, None]
    seen = seen | ((at >= 0) & (at < count) & new.gather(2, at.clamp(0, most - 1)))
    score.masked_fill_(~seen[:, None, :, None], float("-inf"))
    score.sub_(score.amax(-1, keepdim=True).clamp_(min=-1e30)).exp_()
    total = score.sum(-1, keepdim=True)
    out = (score.view(rows, hkv, -1, width * page) @ v).view(rows, hkv, most, hq // hkv, d)
    out = torch.where(total > 0, out / total, 0.0).permute(0, 2, 1, 3, 4).reshape(rows, most, hq, d)
    live = t[None] < (cu[1:] - cu[:-1])[:, None]
    return torch.zeros(n, hq, d, device="cuda").index_put_((token[live],), out[live]).to(torch.bfloat16)


def _plain_verify(s):
    """Level by level, all requests at once; in 64 bits, since a draw is next to a border now and then."""
    logits, tokens, probs, cu = s["logits"], s["tokens"], s["probs"], s["cu"].long()
    n, vocab = logits.shape
    rows, most, temperature = cu.numel() - 1, s["most"], s["temperature"]
    row, live = _row_of(cu, n)
    index = torch.arange(n, device="cuda")
    child_of = torch.where((index > cu[row]) & (s["parents"] >= 0), cu[row] + s["parents"], -1)
    here, ok = cu[:-1].clone(), cu[1:] > cu[:-1]
    here = here.clamp(max=n - 1)
    path = torch.full((rows, most), -1, device="cuda")
    path[:, 0] = torch.where(ok, 0, -1)
    accepted, going, answer = ok.long(), ok.clone(), torch.full((rows,), -1, device="cuda")
    for level in range(s["depth"]):
        row_logits = logits[here].double()
        if temperature == 0:
            best = row_logits.argmax(-1)
        else:
            p = torch.softmax(row_logits / temperature, -1)
            r, mass = p.clone(), p.sum(-1)
            q = probs[here].double() if probs is not None else None
        found = torch.full((rows,), -1, device="cuda")
        last = torch.full((rows,), -1, device="cuda")
        for _ in range(min(s["case"]["wide"], n) if level + 1 < s["depth"] else 0):
            # the next child of `here`, in the tokens' order
            mine = (child_of[None] == here[:, None]) & (index[None] > last[:, None]) & live[None]
            has = mine.any(-1) & going & (found < 0)
            c = torch.where(has, torch.argmax(mine.to(torch.int8), -1), 0)
            x = tokens[c][:, None]
            if temperature == 0:
                yes = has & (x[:, 0] == best)
            else:
                of_draft = q.gather(1, x)[:, 0] if q is not None else 1.0
                yes = has & (s["accept"][c].double() * of_draft * mass < r.gather(1, x)[:, 0])
                if q is not None:
                    rest = (r / mass[:, None] - q).clamp_(min=0)
                else:
                    rest = r.scatter(1, x, 0.0)
                left = rest.sum(-1)
                rest = torch.where((left > 0)[:, None], rest, p)
                no = has & ~yes
                r, mass = torch.where(no[:, None], rest, r), torch.where(no, rest.sum(-1), mass)
            found = torch.where(yes, c, found)
            last = torch.where(has, c, last)
        stop = going & (found < 0)
        if temperature == 0:
            pick = best
        else:
            sums = r.cumsum(-1)
            pick = (sums <= s["last"].double()[:, None] * sums[:, -1:]).sum(-1)
            pick = torch.minimum(pick, vocab - 1 - (r > 0).flip(-1).to(torch.int8).argmax(-1))
        answer = torch.where(stop, pick, answer)
        going = going & (found >= 0)
        here = torch.where(going, found, here)
        if level + 1 < most:
            path[:, level + 1] = torch.where(going, found - cu[:-1], -1)
        accepted = accepted + going
    return accepted.to(torch.int32), path.to(torch.int32), answer


def _plain_keep(s):
    page, table = s["page"], s["table"].long()
    cached, fresh, kept, path = s["cached"].long(), s["fresh"].long(), s["kept"].long(), s["path"].long()
    i = torch.arange(path.shape[1], device="cuda")[None]
    moved = (i < kept[:, None]) & (path != i)
    r, i = moved.nonzero(as_tuple=True)
    src, dst = cached[r] + path[r, i], cached[r] + i
    for pool in (s["k_pages"], s["v_pages"]):
        pool[:, table[r, dst // page], :, dst % page] = pool[:, table[r, src // page], :, src % page]
    lens = cached + kept
    held = (lens + page - 1) // page
    count = (cached + fresh + page - 1) // page - held
    before = count.cumsum(0) - count
    col = torch.arange(table.shape[1], device="cuda")[None]
    back = (col >= held[:, None]) & (col < (held + count)[:, None])
    to = (s["state"][1] + before[:, None] + col - held[:, None]) % s["queue"].numel()
    s["queue"][to[back]] = s["table"][back]
    return (s["k_pages"], s["v_pages"], s["queue"], torch.stack([s["state"][0], s["state"][1] + count.sum()]),
            lens.to(torch.int32))


def _plain_fork(s):
    page, table, queue, shares = s["page"], s["table"], s["queue"], s["shares"].long()
    rows, width = table.shape
    source, cached = s["source"].long(), s["cached"].long()
    goes = source >= 0
    src = source.clamp(min=0)
    lens = torch.where(goes, cached[src], 0)
    full, part = lens // page, lens % page
    r = torch.arange(rows, device="cuda")
    heirs = torch.zeros(rows, dtype=torch.long, device="cuda").index_add_(0, src, goes.long())
    first = torch.full((rows,), rows, device="cuda").scatter_reduce_(0, src, torch.where(goes, r, rows), "amin")
    fresh = goes & (part > 0) & (first[src] != r)
    page_of = queue[(s["state"][0] + fresh.cumsum(0) - 1) % queue.numel()]
    col = torch.arange(width, device="cuda")[None]
    out = torch.where(col < (full + (part > 0))[:, None], table[src], -1)
    out = torch.where((col == full[:, None]) & fresh[:, None], page_of[:, None], out)
    # one row each for every page it holds; only the first heir keeps a page that is not full
    held = col < ((cached + page - 1) // page)[:, None]
    change = torch.where(col < (cached // page)[:, None], heirs[:, None] - 1, -(heirs == 0)[:, None].long())
    shares = shares.index_add(0, table[held].long(), change[held])
    freed = shares < 0
    tail = s["state"][1]
    queue[(tail + freed.cumsum(0) - 1)[freed] % queue.numel()] = freed.nonzero()[:, 0].to(torch.int32)
    new, old, upto = page_of[fresh].long(), table[src, full.clamp(max=width - 1)][fresh].long(), part[fresh]
    keep = (torch.arange(page, device="cuda")[None] < upto[:, None])[None, :, None, :, None]
    for pool in (s["k_pages"], s["v_pages"]):
        pool[:, new] = torch.where(keep, pool[:, old], pool[:, new])
    state = torch.stack([s["state"][0] + fresh.sum(), tail + freed.sum()])
    return out, shares.clamp(min=0).to(torch.int32), state, lens.to(torch.int32), queue, s["k_pages"], s["v_pages"]


_own = dict(tree=_own_tree, attn=_own_attn, verify=_own_verify, keep=_own_keep, fork=_own_fork)
_plain = dict(tree=_plain_tree, attn=_plain_attn, verify=_plain_verify, keep=_plain_keep, fork=_plain_fork)


# -- what a pass cannot do without ---------------------------------------------------------------
def work(case):
    op = case["op"]
    if op == "fork":
        lens, source, _ = _forks(case)
        page, vec = case["page"], 2 * case["slots"] * case["hkv"] * case["d"] * 2
        taken, moved, entries = set(), 0, 0
        for src in source:
            if src >= 0:
                entries += _pages(lens[src], page)
                if src in taken:
                    moved += lens[src] % page
                taken.add(src)
        return dict(bytes=2 * moved * vec + 8 * entries + 12 * len(lens), flops=0)
    cached, fresh = _lengths(case if "lo" in case else dict(case, lo=1, hi=1))
    n = sum(fresh)
    if op == "tree":
        return dict(bytes=(n + case["pad"]) * (8 + case["most"] // 8) + 8 * len(fresh), flops=0)
    if op == "verify":
        # the rows of the kept tokens, and the draft's rows where the walk ends
        size = (4 if case["dtype"] == "float32" else 2) * sum(_paths(case, fresh))
        return dict(bytes=case["vocab"] * (size + (4 * len(fresh) if case["probs"] else 0)) + 16 * n, flops=0)
    if op == "keep":
        kept = sum(n - stay for n, stay in _moves(case, fresh))
        vec = 2 * case["slots"] * case["hkv"] * case["d"] * 2
        return dict(bytes=2 * kept * vec + 4 * kept + 16 * len(fresh), flops=0)
    window, pairs, keys, d = case["window"], 0, 0, case["d"]
    for a, b in zip(cached, fresh):
        deep = b - 1 if b > case["most"] else _pages(b - 1, case["wide"])
        # a tree's token sees its ancestors, half the levels on average, and itself
        own_keys = 1 + (b - 1) / 2 if b > case["most"] else 1 + deep / 2
        past = a if window < 0 else min(a, max(0, window - deep / 2))
        pairs += b * (past + own_keys)
        keys += b + (a if window < 0 else min(a, window))
    return dict(bytes=int(4 * keys * case["hkv"] * d + 4 * n * case["hq"] * d + n * (4 + case["most"] // 8)),
                flops=int(4 * d * case["hq"] * pairs))


# -- the definition in 64 bits, for computed numbers ---------------------------------------------
def exact(case, seed):
    """Request by request, token by token's list of keys, for attention; the others give whole numbers or
    move what is there."""
    if case["op"] != "attn" or work(case)["flops"] > 1e12:
        return None
    s = prepare(case, seed)
    page, window, words = s["page"], case["window"], s["mask"].shape[1]
    n, hq, d = s["q"].shape
    group = hq // s["k_pages"].shape[1]
    cached, cu = s["cached"].tolist(), s["cu"].tolist()
    positions = s["positions"].long()
    out = torch.zeros(n, hq, d, dtype=torch.float64, device="cuda")
    for r, past in enumerate(cached):
        a, b = cu[r], cu[r + 1]
        count = b - a
        end = past + count
        pages = s["table"][r, :_pages(end, page)].long()
        where = torch.cat([torch.arange(past, device="cuda"), positions[a:b]])
        seen = torch.ones(count, end, dtype=torch.bool, device="cuda")
        if count > 32 * words:
            seen[:, past:] = torch.ones(count, count, device="cuda").tril() > 0
        else:
            j = torch.arange(count, device="cuda")
            seen[:, past:] = (s["mask"][a:b][:, j // 32] >> (j % 32)) & 1 > 0
        if window >= 0:
            seen &= positions[a:b, None] - where[None] <= window
        for h in range(hq // group):
            k = s["k_pages"][pages, h].reshape(-1, d)[:end].double()
            v = s["v_pages"][pages, h].reshape(-1, d)[:end].double()
            q = s["q"][a:b, h * group:(h + 1) * group].double()
            w = torch.einsum("tgd,kd->tgk", q, k) / math.sqrt(d)
            w = torch.softmax(w.masked_fill_(~seen[:, None], -math.inf), -1)
            out[a:b, h * group:(h + 1) * group] = torch.einsum("tgk,kd->tgd", w, v)
    return out
