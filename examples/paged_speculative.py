"""Speculative decoding over a paged KV cache: several samples of each prompt share the prompt's pages, and every
step verifies a tree of drafted tokens a sample.

    python examples/paged_speculative.py [--prompts 6] [--samples 4] [--tokens 60] [--temperature 0.1]

The draft is the text itself: what followed the last tokens where they stood before, as a tree of the continuations
found.  The model is paged_serving.py's small random-weight decoder, whose text repeats itself at low temperatures.
"""
import argparse
import importlib.util
import os
import sys
import time

import numpy as np
import torch
import torch.nn.functional as F

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from modelcore_b200 import ops  # noqa: E402


def _serving():
    spec = importlib.util.spec_from_file_location(
        "paged_serving", os.path.join(os.path.dirname(os.path.abspath(__file__)), "paged_serving.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def draft(text, most, depth=6, branches=4):
    """A tree of at most `most` tokens after text: (tokens, parents), text's last token first."""
    tokens, parents, children = [text[-1]], [-1], [{}]
    for n in (3, 2, 1):
        tail = text[-n:]
        for at in range(len(text) - n - 1, -1, -1):
            if len(children[0]) >= branches and n < 3:
                break
            if text[at:at + n] != tail:
                continue
            here = 0
            for x in text[at + n:at + n + depth]:
                if x not in children[here]:
                    if len(tokens) == most:
                        return tokens, parents
                    children[here][x] = len(tokens)
                    tokens.append(x)
                    parents.append(here)
                    children.append({})
                here = children[here][x]
    return tokens, parents


def generate(model, prompts, *, samples=1, max_tokens=40, most=16, temperature=0.0, pages=400, page_size=16, chunk=256,
             seed=0, on_step=None):
    """max_tokens tokens after each prompt, `samples` times.  Returns (tokens, a list a sample, the samples of a prompt
    after one another; steps; tokens kept of drafts)."""
    rows = len(prompts) * samples
    cache = model.new_cache(pages, page_size, rows)
    g = torch.Generator(model.device).manual_seed(seed)
    rand = lambda n: torch.rand(n, device=model.device, generator=g)
    text = [list(prompts[r // samples]) for r in range(rows)]
    # the prompts, once each, in chunks; the last hidden state of each is its samples' first
    todo = {i * samples: list(p) for i, p in enumerate(prompts)}
    first = {}
    while todo:
        new = [len(todo.get(r, [])[:chunk]) for r in range(rows)]
        ids = [x for r in sorted(todo) for x in todo[r][:chunk]]
        step = cache.plan(new)
        h = model.forward(torch.tensor(ids, device=model.device), cache, step)
        cache.advance(step)
        last, who = step.last_tokens()
        for at, r in zip(last.tolist(), who.tolist()):
            del todo[r][:chunk]
            if not todo[r]:
                first[r] = h[at]
                del todo[r]
    cache.fork([r - r % samples for r in range(rows)])
    logits = model.logits(torch.stack([first[r - r % samples] for r in range(rows)]))
    tokens = ops.sample(logits, rand(rows), temperature=temperature).flatten().tolist()
    for r, x in enumerate(tokens):
        text[r].append(x)
    goal = [len(prompts[r // samples]) + max_tokens for r in range(rows)]
    running, steps, drafted = set(range(rows)), 0, 0
    done = [r for r in running if len(text[r]) >= goal[r]]
    while True:
        running -= set(done)
        cache.release(done)
        if not running:
            break
        trees = [draft(text[r], most) if r in running else ([], []) for r in range(rows)]
        ids = torch.tensor([x for t, _ in trees for x in t], device=model.device)
        parents = torch.tensor([x for _, p in trees for x in p], dtype=torch.int32, device=model.device)
        step = cache.plan([len(t) for t, _ in trees], parents=parents, max_tree=most)
        logits = model.logits(model.forward(ids, cache, step))
        v = ops.verify_drafts(logits, ids, parents, step.plan.cu_new, rand(len(ids)), rand(rows), temperature=temperature,
                              max_path=step.max_new)
        kept = cache.keep(step, v.path, v.accepted)
        path, tokens = v.path.tolist(), v.next_token.tolist()
        for r in running:
            text[r] += [trees[r][0][i] for i in path[r][1:kept[r]]] + [tokens[r]]
            drafted += kept[r] - 1
        done = [r for r in running if len(text[r]) >= goal[r]]
        steps += 1
        if on_step is not None:
            on_step(cache, text, running)
    return [t[len(prompts[r // samples]):goal[r]] for r, t in enumerate(text)], steps, drafted


class SpeculativeDecoder(_serving().PackedDecoder):
    """PackedDecoder with the logits of given hidden states."""

    def logits(self, h):
        return ops.softcap_argmax(F.linear(h, self.head), self.vocab, self.softcap)


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--prompts", type=int, default=6)
    ap.add_argument("--samples", type=int, default=4)
    ap.add_argument("--tokens", type=int, default=60)
    ap.add_argument("--temperature", type=float, default=0.1)
    args = ap.parse_args()
    rng = np.random.default_rng(1)
    model = SpeculativeDecoder()
    # prompts that repeat themselves, as documents do
    prompts = [(rng.integers(0, model.vocab, 40).tolist() * 8)[:int(rng.integers(60, 300))] for _ in range(args.prompts)]
    run = lambda: generate(model, prompts, samples=args.samples, max_tokens=args.tokens, temperature=args.temperature,
                           pages=1000)
    run()  # warm up
    torch.cuda.synchronize()
    start = time.perf_counter()
    tokens, steps, drafted = run()
    seconds = time.perf_counter() - start
    code, what = ops.device_error()
    assert code == 0, what
    print(f"{len(prompts)} prompts, {args.samples} samples each, {sum(map(len, tokens))} tokens in {steps} steps, {drafted} "
          f"of them drafted, {seconds * 1e3:.0f} ms")


if __name__ == "__main__":
    main()
