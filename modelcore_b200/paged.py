"""PagedKVCache: a KV cache in pages, shared by requests of any length that come, grow and go.

modelcore's KVCache (modelcore/cache.py:13-119) gives every row T_max positions of its own and adds
the same number of new tokens to every row.  Here the positions of all requests live in one pool of
pages, a request holds the pages its length needs, a step takes any number of new tokens of each
request (a prompt's chunk beside other requests' single tokens), packed one after another, and a
finished request's pages serve the next:

    cache = PagedKVCache(n_pages, 64, n_kv_head, head_dim, n_slots, max_rows, max_seq_len, device)
    step = cache.plan([1, 0, 512, 1])                 # new tokens of rows 0..3
    for slot, layer in enumerate(layers):
        q, k, v = layer.project(x)                    # (step.num_tokens, heads, head_dim), packed
        q = cache.append(slot, q, k, v, step, cos, sin)
        y = cache.attend(slot, q, step, window=layer.window)
    cache.advance(step)
    cache.release([2])                                # row 2 is done: its pages are free

Of drafted tokens that were verified in one step, advance(step, kept=[2, 0, 1, 4]) keeps the accepted ones.

A plan takes its pages only when the step is advanced: until then it can be dropped (planned again, or
never followed), and the cache is what it was.

Everything that depends on the lengths happens on the GPU (ops.page_plan and the kernels that read its
tables); the class keeps a host mirror of the lengths only to refuse a step that does not fit
before anything is launched, as KVCache does.
"""
from typing import NamedTuple, Optional

import numpy as np
import torch

from . import _native, ops
from .cache import _aligned_zeros


class PagedStep(NamedTuple):
    """One planned step (PagedKVCache.plan): the cache's current one until it is advanced or dropped."""
    plan: ops.PagePlan
    new_lens: torch.Tensor     # (max_rows,) int32
    host_lens: np.ndarray      # the same, on the host
    num_tokens: int            # of the packed batch, padding included
    max_new: int

    def last_tokens(self):
        """Indices into the packed batch of the last new token of every row that has any, and those rows
        (host arrays)."""
        rows = np.nonzero(self.host_lens)[0]
        return np.cumsum(self.host_lens)[rows] - 1, rows


class PagedKVCache:
    """k_pages / v_pages: (n_slots, n_pages, n_kv_head, page_size, head_dim) bf16, a head's page one
    contiguous block.  Rows are requests: block_table (max_rows, max_pages) and cache_seqlens
    (max_rows,), both int32, describe them; free_pages and free_state are the queue of free pages."""

    def __init__(self, n_pages, page_size, n_kv_head, head_dim, num_kv_slots, max_rows, max_seq_len, device,
                 dtype=torch.bfloat16):
        _native.load()
        device = torch.device(device)
        if device.type != "cuda":
            raise RuntimeError(f"PagedKVCache lives on a CUDA device, got {device}")
        if dtype != torch.bfloat16:
            raise RuntimeError(f"PagedKVCache stores bf16, got {dtype}")
        if head_dim not in (64, 128):
            raise RuntimeError(f"PagedKVCache needs head_dim 64 or 128, got {head_dim}")
        if page_size < 16 or page_size > 1024 or page_size & (page_size - 1):
            raise RuntimeError(f"page_size must be a power of two from 16 to 1024, got {page_size}")
        self.page_size, self.n_pages, self.n_slots = page_size, n_pages, num_kv_slots
        self.n_kv_head, self.head_dim = n_kv_head, head_dim
        self.max_rows, self.max_seq_len = max_rows, max_seq_len
        self.max_pages = -(-max_seq_len // page_size)
        shape = (num_kv_slots, n_pages, n_kv_head, page_size, head_dim)
        self.k_pages = _aligned_zeros(shape, device)
        self.v_pages = _aligned_zeros(shape, device)
        ints = dict(dtype=torch.int32, device=device)
        self.block_table = torch.full((max_rows, self.max_pages), -1, **ints)
        self.cache_seqlens = torch.zeros(max_rows, **ints)
        self.free_pages = torch.arange(n_pages, **ints)
        self.free_state = torch.tensor([0, n_pages], dtype=torch.int64, device=device)
        self._host_lens = np.zeros(max_rows, dtype=np.int64)
        self._step = None  # the planned step that advance has not followed yet

    def _held(self, lens):
        return -(-lens // self.page_size)

    def _to_device(self, values):
        return torch.from_numpy(np.ascontiguousarray(values, dtype=np.int32)).pin_memory().to(
            self.cache_seqlens.device, non_blocking=True)

    def host_lens(self):
        """Row lengths as this cache's methods have set them (no device read)."""
        return self._host_lens.copy()

    def free_page_count(self):
        """Pages that no row holds (no device read)."""
        return int(self.n_pages - self._held(self._host_lens).sum())

    def pages_needed(self, new_lens):
        """Pages a step of these new tokens a row would take from the free ones."""
        new = self._rows(new_lens)
        return int((self._held(self._host_lens + new) - self._held(self._host_lens)).sum())

    def _rows(self, new_lens):
        new = np.zeros(self.max_rows, dtype=np.int64)
        given = np.asarray(new_lens, dtype=np.int64)
        if given.ndim != 1 or given.size > self.max_rows or (given < 0).any():
            raise RuntimeError(f"new_lens must be at most {self.max_rows} counts, got {new_lens}")
        new[:given.size] = given
        return new

    def plan(self, new_lens, num_tokens: Optional[int] = None):
        """Plans a step of new_lens[r] new tokens for each row (missing rows: 0): pages are chosen for
        them and the packed batch's offsets, positions and slots computed, on the GPU.  num_tokens pads
        the batch (for a fixed shape).  The rows' lengths and the free pages stay until advance(step);
        planning again drops a step that has not been advanced."""
        new = self._rows(new_lens)
        total = int(new.sum())
        num_tokens = total if num_tokens is None else int(num_tokens)
        if num_tokens < total:
            raise RuntimeError(f"{total} new tokens do not fit a batch of {num_tokens}")
        end = self._host_lens + new
        if (end > self.max_seq_len).any():
            row = int(end.argmax())
            raise RuntimeError(f"row {row} would grow to {int(end[row])} tokens, beyond {self.max_seq_len}")
        if self.pages_needed(new) > self.free_page_count():
            raise RuntimeError(f"the step needs {self.pages_needed(new)} pages and {self.free_page_count()} are free")
        lens = self._to_device(new)
        p = ops.page_plan(self.cache_seqlens, lens, self.block_table, self.free_pages, self.free_state,
                          page_size=self.page_size, num_tokens=num_tokens)
        self._step = PagedStep(p, lens, new, num_tokens, int(new.max(initial=0)))
        return self._step

    def _current(self, step):
        # another plan may have given this one's pages to other rows, and its positions are behind once advanced
        if step is not self._step:
            raise RuntimeError("the step is not the planned one: it has been advanced, or dropped by a later plan or "
                               "by the release of one of its rows")

    def append(self, slot, q, k, v, step, cos, sin, *, eps=None, scale=1.2, rotate_k=True, round_each=True):
        """Rope, norm and scale of the packed q (N, Hq, D) and k (N, Hkv, D), k and v into the step's
        slots; k = v = None for a layer that reads slot's pages but adds nothing (modelcore's
        produces_kv=False).  Returns the processed q."""
        self._current(step)
        pages = (self.k_pages[slot], self.v_pages[slot], step.plan.slot_map) if k is not None else (None,) * 3
        return ops.paged_append_rope(q, k, v, pages[0], pages[1], step.plan.positions, pages[2], cos, sin, eps=eps,
                                     scale=scale, rotate_k=rotate_k, round_each=round_each)

    def attend(self, slot, q, step, *, window=-1, softmax_scale=None):
        """Attention of the step's packed queries over their rows' pages of one slot."""
        self._current(step)
        return ops.paged_attn(q, self.k_pages[slot], self.v_pages[slot], self.block_table, self.cache_seqlens,
                              step.plan.cu_new, window=window, softmax_scale=softmax_scale, max_new=step.max_new)

    def advance(self, step, kept=None):
        """The step's new tokens become part of their rows, and its pages theirs.  kept: how many of its new
        tokens each row keeps, the first ones (a list as plan's; drafted tokens that verification
        rejects are not kept); the pages that only the others needed are free again."""
        self._current(step)
        if kept is not None:
            kept = self._rows(kept)
            if (kept > step.host_lens).any():
                row = int((kept - step.host_lens).argmax())
                raise RuntimeError(f"row {row} has {step.host_lens[row]} new tokens in the step, not {kept[row]} to keep")
        self._step = None
        self.cache_seqlens.add_(step.new_lens)
        self.free_state = step.plan.free_state
        if kept is None:
            self._host_lens += step.host_lens
            return
        self._host_lens += kept
        fewer = kept < step.host_lens
        if fewer.any():
            self._release(fewer, self._to_device(self._host_lens))

    def release(self, rows):
        """Frees the pages of the given rows and sets their lengths to 0.  A planned step that has new tokens
        of one of them is dropped; any other stays the current one."""
        done = np.zeros(self.max_rows, dtype=bool)
        done[np.asarray(rows, dtype=np.int64)] = True
        if self._step is not None and self._step.host_lens[done].any():
            self._step = None
        self._release(done)
        if self._step is not None:
            self._step.plan.free_state[1:].copy_(self.free_state[1:])  # its tail: the pages that have come back
        self._host_lens[done] = 0

    def _release(self, done, keep_lens=None):
        ops.page_release(self._to_device(done), self.cache_seqlens, self.block_table, self.free_pages,
                         self.free_state, page_size=self.page_size, free_state_out=self.free_state,
                         seqlens_out=self.cache_seqlens, keep_lens=keep_lens)
