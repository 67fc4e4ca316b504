"""What the paged-cache operators are measured on: the cases, their inputs, and each operator in its
plain form beside the call a user makes.

  plan      page_plan: offsets, positions, slot map and block tables of one step, from the lengths
  release   page_release: a finished request's pages back to the free queue
  append    paged_append_rope: rope, norm and scale of packed tokens, keys and values into pages
  attn      paged_attn: attention of ragged chunks of new tokens over the pages

The lengths of a case follow from the case alone ("lens"), the values and the placement of the pages
from the seed."""
import math
import random

import torch

own = False

EPS = torch.finfo(torch.float32).eps  # the epsilon of rms_norm when none is given
SCALE = 1.2


def listed():
    return [
        # one decode step of 64 requests of the quickstart model, small pages: pure latency
        dict(name="plan_decode_64", op="plan", rows=64, lo=512, hi=1023, chunks=0, chunk=0, page=16, lens=1, pad=0),
        # a full server's step: 60 prompt chunks beside 940 decoding requests, a padded token count
        dict(name="plan_chunks_1000", op="plan", rows=1000, lo=100, hi=8191, chunks=60, chunk=512, page=64, lens=2,
             pad=37),
        # a quarter of a batch finishes at once
        dict(name="release_256", op="release", rows=256, lo=1, hi=8192, every=4, page=16, lens=3),
        # many long requests cancelled together
        dict(name="release_999", op="release", rows=999, lo=8000, hi=32768, every=3, page=16, lens=4),
        # the quickstart model's decode step (12 heads of 64)
        dict(name="append_decode_64", op="append", tokens=64, hq=12, hkv=12, d=64, page=16, pad=0),
        # the grouped-query model's prompt chunks, an odd number of tokens with a padded tail
        dict(name="append_chunks_16381", op="append", tokens=16381, hq=16, hkv=4, d=128, page=64, pad=5),
        # three requests of the quickstart model decoding: the smallest serving step
        dict(name="attn_decode_3", op="attn", rows=3, lo=500, hi=1023, chunks=0, chunk=0, hq=12, hkv=12, d=64,
             page=16, window=-1, lens=5),
        # the grouped-query model's decode step at batch 128
        dict(name="attn_decode_128", op="attn", rows=128, lo=1024, hi=8192, chunks=0, chunk=0, hq=16, hkv=4, d=128,
             page=64, window=-1, lens=6),
        # long requests decoding four tokens at a time (drafted tokens to verify), small pages
        dict(name="attn_verify_long", op="attn", rows=13, lo=8192, hi=32700, chunks=13, chunk=4, hq=32, hkv=8, d=128,
             page=16, window=-1, lens=7),
        # prompt chunks beside decoding requests: the continuous batch
        dict(name="attn_mixed_64", op="attn", rows=64, lo=1024, hi=7600, chunks=7, chunk=509, hq=16, hkv=4, d=128,
             page=64, window=-1, lens=8),
        # the window layers' chunks, odd sizes
        dict(name="attn_window_chunks", op="attn", rows=5, lo=0, hi=6000, chunks=5, chunk=2041, hq=16, hkv=4, d=128,
             page=32, window=1024, lens=9),
        # one long prompt's second half
        dict(name="attn_chunk_8192", op="attn", rows=1, lo=8192, hi=8192, chunks=1, chunk=8192, hq=16, hkv=4, d=128,
             page=64, window=-1, lens=10),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "release", "append", "attn", "attn", "attn"])
    page = rng.choice([16, 32, 64, 128])
    lens = rng.randrange(1 << 30)
    if op == "plan":
        rows = _log(rng, 1, 1000)
        lo = _log(rng, 1, 4000)
        chunks = rng.randint(0, min(rows, 60))
        return dict(op=op, rows=rows, lo=lo, hi=lo + _log(rng, 1, 4000), chunks=chunks,
                    chunk=_log(rng, 2, 512) if chunks else 0, page=page, lens=lens, pad=rng.choice([0, 0, 1, 100]))
    if op == "release":
        lo = _log(rng, 1, 16000)
        return dict(op=op, rows=_log(rng, 1, 999), lo=lo, hi=lo + _log(rng, 1, 16000), every=rng.randint(1, 9),
                    page=page, lens=lens)
    hq, hkv, d = rng.choice([(12, 12, 64), (16, 4, 128), (32, 8, 128), (6, 2, 64), (15, 5, 128), (8, 1, 64),
                             (24, 24, 128)])
    if op == "append":
        tokens = _log(rng, 1, 16000)
        tokens = max(1, min(tokens, 16000 * (16 + 8) * 128 // ((hq + 2 * hkv) * d)))
        return dict(op=op, tokens=tokens, hq=hq, hkv=hkv, d=d, page=page, pad=rng.choice([0, 0, 3]))
    window = rng.choice([-1, -1, -1, 128, 1024, 4000])
    while True:
        rows = _log(rng, 1, 128)
        lo = _log(rng, 1, 8000)
        hi = lo + _log(rng, 1, 16000)
        kind = rng.choice(["decode", "chunks", "mixed"])
        chunks = dict(decode=0, chunks=rows, mixed=(rows + 3) // 4)[kind]
        chunk = _log(rng, 2, 4096) if chunks else 0
        c = dict(op=op, rows=rows, lo=lo, hi=hi, chunks=chunks, chunk=chunk, hq=hq, hkv=hkv, d=d, page=page,
                 window=window, lens=lens)
        longest = hi + max(1, chunk)
        # no more work than the largest listed case, and a plain form whose padded scores fit
        if (work(c)["flops"] <= 0.9e12 and work(c)["bytes"] <= 1.5e9
                and rows * max(1, chunk) * hq * longest <= 4.2e9 and rows * longest * hkv * d <= 0.6e9):
            return c


def _lengths(case):
    """(cached tokens, new tokens) of every request, as lists: chunks first in a shuffled order."""
    rng = random.Random(case["lens"])
    rows = case["rows"]
    cached = [rng.randint(case["lo"], case["hi"]) for _ in range(rows)]
    fresh = [1] * rows
    for r in rng.sample(range(rows), case.get("chunks", 0)):
        # most chunks are full; some are a prompt's ragged end
        fresh[r] = case["chunk"] if rng.random() < 0.7 else rng.randint(1, case["chunk"])
    return cached, fresh


def _pages(n, page):
    return -(-n // page)


def _tables(d, device="cuda"):
    """Rotary tables (positions, D/2) in bf16, base 10000."""
    inv = 10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64, device=device) / d)
    ang = torch.arange(40000, dtype=torch.float64, device=device)[:, None] * inv[None]
    return ang.cos().to(torch.bfloat16), ang.sin().to(torch.bfloat16)


def _normed(shape, gen):
    """Vectors as the append leaves them: rms 1.2."""
    x = torch.randn(shape, device="cuda", dtype=torch.bfloat16, generator=gen)
    r = x.float().square().mean(-1, keepdim=True).rsqrt_().mul_(SCALE).to(torch.bfloat16)
    return x.mul_(r)


def prepare(case, seed):
    op, page = case["op"], case["page"]
    gen = torch.Generator("cuda").manual_seed(seed)
    s = dict(case=case, page=page)
    ints = dict(dtype=torch.int32, device="cuda")
    if op in ("plan", "release", "attn"):
        cached, fresh = _lengths(case)
        s["cached"] = torch.tensor(cached, **ints)
        held = [_pages(n, page) for n in cached]
    if op in ("plan", "release"):
        rows = case["rows"]
        width = max(_pages(a + b, page) for a, b in zip(cached, fresh)) + 3
        total = sum(_pages(a + b, page) for a, b in zip(cached, fresh)) + 100
        order = torch.randperm(total, device="cuda", generator=gen).to(torch.int32)
        held_t = torch.tensor(held, device="cuda")
        index = torch.arange(width, device="cuda")[None] + (held_t.cumsum(0) - held_t)[:, None]
        table = torch.where(torch.arange(width, device="cuda")[None] < held_t[:, None],
                            order[index.clamp_(max=total - 1)], -1)
        used = sum(held)
        # a queue that has gone round: the free pages start in its middle
        head = 1000 * total + total - min(total, 7)
        queue = torch.full((total,), -1, **ints)
        at = (head + torch.arange(total - used, device="cuda")) % total
        queue[at] = order[used:]
        s |= dict(table=table.contiguous(), queue=queue,
                  state=torch.tensor([head, head + total - used], dtype=torch.int64, device="cuda"),
                  state_out=torch.zeros(2, dtype=torch.int64, device="cuda"))
        if op == "plan":
            s |= dict(fresh=torch.tensor(fresh, **ints), tokens=sum(fresh) + case["pad"])
        else:
            done = [int(r % case["every"] == seed % case["every"]) for r in range(rows)]
            s |= dict(done=torch.tensor(done, **ints), cached_out=torch.zeros(rows, **ints))
        return s
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    if op == "append":
        n = case["tokens"]
        n_pages = _pages(n, page) + 3
        # a whole projection of the packed tokens; q, k and v are views of it
        qkv = torch.randn(n + case["pad"], hq + 2 * hkv, d, device="cuda", dtype=torch.bfloat16, generator=gen)
        place = torch.randperm(n_pages, device="cuda", generator=gen)
        start = int(torch.randint(0, 20000, (1,), generator=torch.Generator().manual_seed(seed)))
        t = torch.arange(n + case["pad"], device="cuda")
        slots = torch.where(t < n, place[(t // page).clamp_(max=n_pages - 1)] * page + t % page, -1)
        pos = torch.where(t < n, start + t, -1).to(torch.int32)
        cos, sin = _tables(d)
        return s | dict(qkv=qkv, slots=slots, pos=pos, cos=cos, sin=sin,
                        k_pages=torch.zeros(n_pages, hkv, page, d, device="cuda", dtype=torch.bfloat16),
                        v_pages=torch.zeros(n_pages, hkv, page, d, device="cuda", dtype=torch.bfloat16))
    counts = [_pages(a + b, page) for a, b in zip(cached, fresh)]
    width, n_pages = max(counts) + 1, sum(counts) + 5
    order = torch.randperm(n_pages, device="cuda", generator=gen).to(torch.int32)
    count_t = torch.tensor(counts, device="cuda")
    col = torch.arange(width, device="cuda")[None]
    index = (col + (count_t.cumsum(0) - count_t)[:, None]).clamp_(max=n_pages - 1)
    cu = [0]
    for n in fresh:
        cu.append(cu[-1] + n)
    return s | dict(
        q=_normed((cu[-1], hq, d), gen), k_pages=_normed((n_pages, hkv, page, d), gen),
        v_pages=torch.randn(n_pages, hkv, page, d, device="cuda", dtype=torch.bfloat16, generator=gen),
        table=torch.where(col < count_t[:, None], order[index], -1).contiguous(),
        cu=torch.tensor(cu, **ints), most=max(fresh), longest=max(a + b for a, b in zip(cached, fresh)))


# -- one pass ------------------------------------------------------------------------------------
def run(s):
    return (_own if own else _plain)[s["case"]["op"]](s)


def _own_plan(s):
    from modelcore_b200 import ops
    p = ops.page_plan(s["cached"], s["fresh"], s["table"], s["queue"], s["state"], page_size=s["page"],
                      num_tokens=s["tokens"], free_state_out=s["state_out"])
    return p.cu_new, p.positions, p.slot_map, s["table"], s["state_out"]


def _own_release(s):
    from modelcore_b200 import ops
    ops.page_release(s["done"], s["cached"], s["table"], s["queue"], s["state"], page_size=s["page"],
                     free_state_out=s["state_out"], seqlens_out=s["cached_out"])
    return s["queue"], s["state_out"], s["cached_out"]


def _own_append(s):
    from modelcore_b200 import ops
    hq, hkv = s["case"]["hq"], s["case"]["hkv"]
    q, k, v = s["qkv"].split([hq, hkv, hkv], 1)
    out = ops.paged_append_rope(q, k, v, s["k_pages"], s["v_pages"], s["pos"], s["slots"], s["cos"], s["sin"],
                                round_each=False)
    return out, s["k_pages"], s["v_pages"]


def _own_attn(s):
    from modelcore_b200 import ops
    return ops.paged_attn(s["q"], s["k_pages"], s["v_pages"], s["table"], s["cached"], s["cu"],
                          window=s["case"]["window"], max_new=s["most"])


def _plain_plan(s):
    page, n, table, queue = s["page"], s["tokens"], s["table"], s["queue"]
    cached, fresh, head = s["cached"].long(), s["fresh"].long(), s["state"][0]
    cu = torch.cat([fresh.new_zeros(1), fresh.cumsum(0)])
    first = (cached + page - 1) // page
    need = (cached + fresh + page - 1) // page - first
    taken = need.cumsum(0)
    before = taken - need
    col = torch.arange(table.shape[1], device="cuda")[None]
    new = (col >= first[:, None]) & (col < (first + need)[:, None])
    source = (head + before[:, None] + col - first[:, None]) % queue.numel()
    table = torch.where(new, queue[source], table)
    t = torch.arange(n, device="cuda")
    row = torch.searchsorted(cu[1:], t, right=True)
    live = t < cu[-1]
    row = row.clamp(max=cached.numel() - 1)
    pos = cached[row] + t - cu[row]
    at = (pos // page).clamp(max=table.shape[1] - 1)
    slot = table[row, at].long() * page + pos % page
    state = torch.stack([head + taken[-1], s["state"][1]])
    return (cu.to(torch.int32), torch.where(live, pos, -1).to(torch.int32), torch.where(live, slot, -1), table,
            state)


def _plain_release(s):
    page, table, queue = s["page"], s["table"], s["queue"]
    gone = s["done"] != 0
    count = torch.where(gone, (s["cached"].long() + page - 1) // page, 0)
    total = count.cumsum(0)
    col = torch.arange(table.shape[1], device="cuda")[None]
    back = col < count[:, None]
    to = (s["state"][1] + (total - count)[:, None] + col) % queue.numel()
    queue[to[back]] = table[back]
    return queue, torch.stack([s["state"][0], s["state"][1] + total[-1]]), torch.where(gone, 0, s["cached"])


def _rope_norm(x, c, s):
    x1, x2 = x.float().chunk(2, -1)
    y = torch.cat([x1 * c + x2 * s, x2 * c - x1 * s], -1)
    return y * (y.square().mean(-1, keepdim=True) + EPS).rsqrt() * SCALE


def _plain_append(s):
    hq, hkv, page = s["case"]["hq"], s["case"]["hkv"], s["page"]
    q, k, v = s["qkv"].split([hq, hkv, hkv], 1)
    live = s["pos"] >= 0
    at = s["pos"].long().clamp(min=0)
    c, sn = s["cos"][at].float()[:, None], s["sin"][at].float()[:, None]
    out = torch.where(live[:, None, None], _rope_norm(q, c, sn), 0.0).to(torch.bfloat16)
    slots = s["slots"][live]
    s["k_pages"][slots // page, :, slots % page] = _rope_norm(k, c, sn)[live].to(torch.bfloat16)
    s["v_pages"][slots // page, :, slots % page] = v[live]
    return out, s["k_pages"], s["v_pages"]


def _plain_attn(s):
    page, window, cached, cu = s["page"], s["case"]["window"], s["cached"].long(), s["cu"].long()
    n, hq, d = s["q"].shape
    hkv, rows, most = s["k_pages"].shape[1], cached.numel(), s["most"]
    width = _pages(s["longest"], page)
    table = s["table"][:, :width].long().clamp(min=0)
    # every request padded to the longest: (rows, Hkv, keys, D)
    k = s["k_pages"][table].transpose(1, 2).reshape(rows, hkv, width * page, d).float()
    v = s["v_pages"][table].transpose(1, 2).reshape(rows, hkv, width * page, d).float()
    t = torch.arange(most, device="cuda")[None]
    token = (cu[:-1, None] + t).clamp(max=n - 1)
    q = s["q"][token].view(rows, most, hkv, hq // hkv, d).permute(0, 2, 1, 3, 4).float()
    score = (q.reshape(rows, hkv, -1, d) @ k.transpose(-1, -2)).mul_(1.0 / math.sqrt(d))
    score = score.view(rows, hkv, most, hq // hkv, width * page)
    key = torch.arange(width * page, device="cuda")
    pos = (cached[:, None] + t)[..., None]
    seen = key <= pos
    if window >= 0:
        seen = seen & (pos - key <= window)
    score.masked_fill_(~seen[:, None, :, None], float("-inf"))
    score.sub_(score.amax(-1, keepdim=True)).exp_()
    total = score.sum(-1, keepdim=True)
    out = (score.view(rows, hkv, -1, width * page) @ v).view(rows, hkv, most, hq // hkv, d) / total
    out = out.permute(0, 2, 1, 3, 4).reshape(rows, most, hq, d)
    return out[t < (cu[1:] - cu[:-1])[:, None]].to(torch.bfloat16)


_own = dict(plan=_own_plan, release=_own_release, append=_own_append, attn=_own_attn)
_plain = dict(plan=_plain_plan, release=_plain_release, append=_plain_append, attn=_plain_attn)


# -- what a pass cannot do without ---------------------------------------------------------------
def work(case):
    op, page = case["op"], case["page"]
    if op == "append":
        n, vec = case["tokens"], case["d"] * 2
        heads = case["hq"] + 2 * case["hkv"]
        return dict(bytes=n * (2 * heads * vec + vec + 12), flops=n * (case["hq"] + case["hkv"]) * case["d"] * 8)
    cached, fresh = _lengths(case)
    if op == "plan":
        new = sum(_pages(a + b, page) - _pages(a, page) for a, b in zip(cached, fresh))
        return dict(bytes=16 * len(cached) + 8 * new + 12 * (sum(fresh) + case["pad"]) + 32, flops=0)
    if op == "release":
        back = sum(_pages(a, page) for a in cached) / case["every"]
        return dict(bytes=int(8 * back) + 12 * len(cached) + 32, flops=0)
    window, pairs, keys = case["window"], 0, 0
    for a, b in zip(cached, fresh):
        # token t of the chunk sees min(a + t, window) + 1 keys
        whole = b if window < 0 else max(0, min(b, window - a))
        pairs += whole * (a + 1) + whole * (whole - 1) // 2 + (b - whole) * (window + 1)
        keys += a + b - (0 if window < 0 else max(0, a - window))
    d = case["d"]
    return dict(bytes=4 * keys * case["hkv"] * d + 4 * sum(fresh) * case["hq"] * d + 4 * sum(
        _pages(a + b, page) for a, b in zip(cached, fresh)), flops=4 * d * case["hq"] * pairs)


# -- the definitions in 64 bits, for computed numbers --------------------------------------------
def exact(case, seed):
    if case["op"] in ("plan", "release"):
        return None  # whole numbers
    s = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(s)
    return _exact_attn(s) if work(case)["flops"] < 3e12 else None


def _exact_append(s):
    """Token by position: each pair of halves turned by its angle as a complex number."""
    hq, hkv, page = s["case"]["hq"], s["case"]["hkv"], s["page"]
    half = s["case"]["d"] // 2
    n = s["case"]["tokens"]
    turn = torch.complex(s["cos"].double(), -s["sin"].double())[s["pos"][:n].long()][:, None]
    x = s["qkv"].double()

    def turned(y):
        z = torch.complex(y[..., :half].contiguous(), y[..., half:].contiguous()) * turn
        z = torch.cat([z.real, z.imag], -1)
        return SCALE * z / torch.sqrt((z * z).sum(-1, keepdim=True) / (2 * half) + EPS)

    out = torch.zeros(x.shape[0], hq, 2 * half, dtype=torch.float64, device="cuda")
    out[:n] = turned(x[:n, :hq])
    pools = []
    for rows, pool in ((turned(x[:n, hq:hq + hkv]), s["k_pages"]), (x[:n, hq + hkv:], s["v_pages"])):
        flat = pool.double().transpose(1, 2).reshape(-1, hkv, 2 * half)
        flat[s["slots"][:n]] = rows
        pools.append(flat.view(-1, page, hkv, 2 * half).transpose(1, 2).contiguous())
    return out, pools[0], pools[1]


def _exact_attn(s):
    """Request by request, head by head, a block of tokens at a time."""
    page, window = s["page"], s["case"]["window"]
    n, hq, d = s["q"].shape
    group = hq // s["k_pages"].shape[1]
    cached, cu = s["cached"].tolist(), s["cu"].tolist()
    out = torch.zeros(n, hq, d, dtype=torch.float64, device="cuda")
    for r, past in enumerate(cached):
        end = past + cu[r + 1] - cu[r]
        pages = s["table"][r, :_pages(end, page)].long()
        step = max(1, (1 << 26) // (end * group))
        for h in range(hq // group):
            k = s["k_pages"][pages, h].reshape(-1, d)[:end].double()
            v = s["v_pages"][pages, h].reshape(-1, d)[:end].double()
            for a in range(cu[r], cu[r + 1], step):
                b = min(a + step, cu[r + 1])
                p = torch.arange(past + a - cu[r], past + b - cu[r], device="cuda")
                lag = p[:, None] - torch.arange(end, device="cuda")[None]
                hide = (lag < 0) | ((lag > window) if window >= 0 else False)
                q = s["q"][a:b, h * group:(h + 1) * group].double()
                w = torch.einsum("tgd,kd->tgk", q, k) / math.sqrt(d)
                w = torch.softmax(w.masked_fill_(hide[:, None], -math.inf), -1)
                out[a:b, h * group:(h + 1) * group] = torch.einsum("tgk,kd->tgd", w, v)
    return out
