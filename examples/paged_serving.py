"""Continuous batching over a paged KV cache: prompts arrive, are prefilled in chunks beside the
requests that are already generating, and hand their pages on when they finish.

    python examples/paged_serving.py [--requests 40] [--rows 16] [--pages 400]

The model is a small random-weight decoder in modelcore's architecture (RMSNorm blocks, rotary, QK-norm,
gated silu, softcapped greedy head) stepping on packed tokens; every step is one forward over whatever
the scheduler put together.
"""
import argparse
import os
import sys
import time
from collections import deque

import torch
import torch.nn.functional as F

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from modelcore_b200 import PagedKVCache, ops  # noqa: E402


class PackedDecoder:
    """A stack of attention and gated MLP blocks on packed tokens."""

    def __init__(self, vocab=1000, width=512, layers=4, heads=8, kv_heads=2, head_dim=64, hidden=1024, max_len=2048,
                 softcap=15.0, seed=0, device="cuda"):
        g = torch.Generator(device).manual_seed(seed)
        w = lambda *shape: (torch.randn(*shape, device=device, generator=g) * shape[-1] ** -0.5).to(torch.bfloat16)
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, head_dim
        self.vocab, self.softcap, self.max_len, self.device = vocab, softcap, max_len, torch.device(device)
        self.embed, self.head = w(vocab, width), w(vocab, width)
        self.layers = [dict(qkv=w((heads + 2 * kv_heads) * head_dim, width), out=w(width, heads * head_dim),
                            gate_up=w(2 * hidden, width), down=w(width, hidden), window=-1 if i % 2 else 256)
                       for i in range(layers)]
        freq = 10000.0 ** (-torch.arange(0, head_dim, 2, device=device, dtype=torch.float64) / head_dim)
        angle = torch.arange(max_len, device=device, dtype=torch.float64)[:, None] * freq
        self.cos, self.sin = angle.cos().to(torch.bfloat16), angle.sin().to(torch.bfloat16)

    def new_cache(self, pages, page_size, rows):
        return PagedKVCache(pages, page_size, self.kv_heads, self.head_dim, len(self.layers), rows, self.max_len,
                            self.device)

    def forward(self, ids, cache, step):
        """Hidden states (N, width) of the packed ids (N,)."""
        x, h = ops.embed_rms_norm(ids, self.embed)
        for slot, layer in enumerate(self.layers):
            qkv = F.linear(h, layer["qkv"]).view(-1, self.heads + 2 * self.kv_heads, self.head_dim)
            q, k, v = qkv.split([self.heads, self.kv_heads, self.kv_heads], 1)
            q = cache.append(slot, q, k, v, step, self.cos, self.sin)
            y = cache.attend(slot, q, step, window=layer["window"])
            x, h = ops.add_rms_norm(x, F.linear(y.flatten(1), layer["out"]))
            gate, up = F.linear(h, layer["gate_up"]).chunk(2, -1)
            x, h = ops.add_rms_norm(x, F.linear(ops.gated_silu(gate, up), layer["down"]))
        return h

    def next_tokens(self, h):
        """The greedy token of each of the given hidden states (rows, width)."""
        out = torch.empty(h.shape[0], dtype=torch.int64, device=h.device)
        ops.softcap_argmax(F.linear(h, self.head), self.vocab, self.softcap, want_logits=False, argmax_out=out)
        return out


def serve(model, prompts, *, max_tokens, rows=16, pages=400, page_size=16, chunk=128, on_step=None):
    """Generates max_tokens[i] tokens after each prompt (a list of ids).  At most `rows` requests run at a
    time; a prompt is taken in when its pages fit beside what the running requests can still need.
    Returns the generated tokens, a list a prompt, and the number of steps."""
    cache = model.new_cache(pages, page_size, rows)
    waiting = deque(range(len(prompts)))
    running = {}  # row -> request
    done = [None] * len(prompts)
    need = lambda i: -(-(len(prompts[i]) + max_tokens[i]) // page_size)
    steps = 0
    while waiting or running:
        promised = sum(need(r["request"]) for r in running.values())
        for row in (r for r in range(rows) if r not in running):
            if not waiting or promised + need(waiting[0]) > pages:
                break
            i = waiting.popleft()
            running[row] = dict(request=i, todo=list(prompts[i]), out=[])
            promised += need(i)
        if not running:
            raise RuntimeError(f"prompt {waiting[0]} needs {need(waiting[0])} pages of {pages}")
        new = [0] * rows
        ids = []
        for row in sorted(running):
            take = running[row]["todo"][:chunk]
            new[row] = len(take)
            ids += take
        step = cache.plan(new)
        h = model.forward(torch.tensor(ids, device=model.device), cache, step)
        cache.advance(step)
        last, who = step.last_tokens()
        tokens = model.next_tokens(h[torch.from_numpy(last).to(h.device)]).tolist()
        finished = []
        for row, token in zip(who.tolist(), tokens):
            r = running[row]
            del r["todo"][:new[row]]
            if r["todo"]:
                continue  # a prompt's chunk before its last
            r["out"].append(token)
            r["todo"] = [token]
            if len(r["out"]) == max_tokens[r["request"]]:
                done[r["request"]] = r["out"]
                finished.append(row)
        if finished:
            cache.release(finished)
            for row in finished:
                del running[row]
        steps += 1
        if on_step is not None:
            on_step(cache, step, running)
    return done, steps


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--requests", type=int, default=40)
    ap.add_argument("--rows", type=int, default=16)
    ap.add_argument("--pages", type=int, default=400)
    args = ap.parse_args()
    g = torch.Generator().manual_seed(1)
    rand = lambda lo, hi: int(torch.randint(lo, hi + 1, (1,), generator=g))
    model = PackedDecoder()
    prompts = [torch.randint(0, model.vocab, (rand(5, 700),), generator=g).tolist() for _ in range(args.requests)]
    wanted = [rand(1, 60) for _ in prompts]
    serve(model, prompts[:2], max_tokens=wanted[:2], rows=args.rows, pages=args.pages)  # warm up
    torch.cuda.synchronize()
    start = time.perf_counter()
    tokens, steps = serve(model, prompts, max_tokens=wanted, rows=args.rows, pages=args.pages)
    seconds = time.perf_counter() - start
    code, what = ops.device_error()
    assert code == 0, what
    print(f"{len(prompts)} requests, {sum(map(len, prompts))} prompt tokens and {sum(map(len, tokens))} generated in "
          f"{steps} steps, {seconds * 1e3:.0f} ms")


if __name__ == "__main__":
    main()
