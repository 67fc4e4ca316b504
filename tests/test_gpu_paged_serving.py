"""PagedKVCache and the continuous-batching example, on the GPU: a served request's tokens against the
same model run alone over a contiguous KVCache, pages never shared, refusals before any launch."""
import importlib.util
import os

import numpy as np
import pytest
import torch
import torch.nn.functional as F

from conftest import REPO

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("paged_serving", os.path.join(REPO, "examples", "paged_serving.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def alone(model, ids):
    """Logits (T, vocab) after every token of one request, the whole of it in one forward over KVCache."""
    from modelcore_b200 import KVCache, ops
    T = len(ids)
    cache = KVCache(1, model.kv_heads, T, model.head_dim, len(model.layers), model.device, torch.bfloat16)
    cos, sin = model.cos.view(1, -1, 1, model.head_dim // 2), model.sin.view(1, -1, 1, model.head_dim // 2)
    x, h = ops.embed_rms_norm(torch.tensor(ids, device=model.device), model.embed)
    for slot, layer in enumerate(model.layers):
        qkv = F.linear(h, layer["qkv"]).view(1, T, -1, model.head_dim)
        q, k, v = qkv.split([model.heads, model.kv_heads, model.kv_heads], 2)
        kc, vc = cache.get_slot_cache(slot)
        q = ops.kv_append_rope(q, k, v, kc, vc, cache.cache_seqlens, cos, sin)
        y = ops.decode_attn(q, kc, vc, cache.cache_seqlens, window=layer["window"])
        x, h = ops.add_rms_norm(x, F.linear(y.view(T, -1), layer["out"]))
        gate, up = F.linear(h, layer["gate_up"]).chunk(2, -1)
        x, h = ops.add_rms_norm(x, F.linear(ops.gated_silu(gate, up), layer["down"]))
    return ops.softcap_argmax(F.linear(h, model.head), model.vocab, model.softcap)


@pytest.mark.parametrize("head_dim,heads,kv_heads,page_size,chunk", [(64, 8, 2, 16, 50), (128, 4, 4, 64, 400)])
def test_served_tokens_are_the_model_s_own(example, head_dim, heads, kv_heads, page_size, chunk):
    """Every generated token is a greedy choice of the model run alone over the same tokens: its logit there
    is the largest up to the two paths' difference.  The logits are of unit scale (unit-rms states times
    weights of variance 1 / width) and each of the eight block halves adds bf16 roundings of relative
    2^-9 or so to the states in either path: a few hundredths; 0.15 leaves a factor of three or more."""
    from modelcore_b200 import ops
    rng = np.random.default_rng(0)
    model = example.PackedDecoder(head_dim=head_dim, heads=heads, kv_heads=kv_heads)
    prompts = [rng.integers(0, model.vocab, int(n)).tolist() for n in rng.integers(1, 500, 14)]
    wanted = [int(n) for n in rng.integers(1, 25, 14)]
    owned = []

    def check(cache, step, running):
        lens = cache.host_lens()
        assert cache.cache_seqlens.tolist() == lens.tolist()
        table = cache.block_table.cpu().numpy()
        pages = [int(p) for r in range(cache.max_rows) for p in table[r, :-(-int(lens[r]) // page_size)]]
        assert len(set(pages)) == len(pages) and cache.n_pages - len(pages) == cache.free_page_count()
        head, tail = cache.free_state.tolist()
        assert tail - head == cache.free_page_count()
        owned.append(len(pages))

    tokens, steps = example.serve(model, prompts, max_tokens=wanted, rows=5, pages=2600 // page_size,
                                  page_size=page_size, chunk=chunk, on_step=check)
    assert [len(t) for t in tokens] == wanted and owned[-1] == 0 and max(owned) > 0
    code, what = ops.device_error()
    assert code == 0, what
    for prompt, out in zip(prompts, tokens):
        logits = alone(model, prompt + out[:-1])[len(prompt) - 1:]
        chosen = logits.gather(1, torch.tensor(out, device=logits.device)[:, None])[:, 0]
        assert (logits.max(-1).values - chosen).max().item() <= 0.15


def test_what_the_cache_refuses():
    from modelcore_b200 import PagedKVCache
    make = lambda **kw: PagedKVCache(**{**dict(n_pages=10, page_size=16, n_kv_head=2, head_dim=64, num_kv_slots=1,
                                               max_rows=3, max_seq_len=100, device="cuda"), **kw})
    for kw in (dict(device="cpu"), dict(dtype=torch.float16), dict(head_dim=96), dict(page_size=24), dict(page_size=8)):
        with pytest.raises(RuntimeError):
            make(**kw)
    cache = make()
    for new in ([101], [1, 1, 1, 1], [-1], [[1]]):
        with pytest.raises(RuntimeError):
            cache.plan(new)
    with pytest.raises(RuntimeError):
        cache.plan([5, 5], num_tokens=9)
    with pytest.raises(RuntimeError, match="are free"):
        cache.plan([90, 80])
    step = cache.plan([90, 60], num_tokens=160)
    cache.advance(step)
    assert cache.free_page_count() == 0 and cache.plan([6, 4]).num_tokens == 10  # the pages' own room
    with pytest.raises(RuntimeError, match="are free"):
        cache.plan([0, 0, 1])
    cache.release([0])
    assert cache.free_page_count() == 6 and cache.host_lens().tolist() == [0, 60, 0]
    assert cache.cache_seqlens.tolist() == [0, 60, 0]
