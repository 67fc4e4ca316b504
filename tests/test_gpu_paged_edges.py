"""The paged operators where their parts meet: blocks of unlike size one after another on an SM, sums and
windows at the ends of their types, tables with holes, steps that are dropped or kept in part, captured
graphs that go.  Plain forms and tolerances are test_gpu_paged's."""
import numpy as np
import pytest
import torch

from test_gpu_paged import U, attn_case, attn_ref, check_attn, i32  # noqa: F401
from test_gpu_paged import expects_device_error, no_device_error, ops  # noqa: F401  (fixtures)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("Hq,Hkv,D,block", [(16, 4, 128, 64), (4, 4, 64, 256), (8, 1, 128, 32)])
def test_a_full_block_and_then_a_ragged_one(ops, Hq, Hkv, D, block):
    """Many units an SM, blocks whose row quarters are all taken before blocks of a few rows: the results
    are right and repeat themselves bit for bit."""
    fresh = [block + 1 + r % 40 for r in range(150)]
    cached = [(r * 37) % 300 for r in range(150)]
    c = check_attn(ops, cached, fresh, Hq, Hkv, D, 64)
    call = lambda: ops.paged_attn(c["q"], c["kp"], c["vp"], c["table"], c["cached"], c["cu"])
    want = call()
    assert all(torch.equal(call(), want) for _ in range(20))
