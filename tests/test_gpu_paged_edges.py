"""The paged-cache operators at the edges of what their header allows: kernels that end right
after their last MMA, long lines, tails of a softmax far below its largest weight, signed
limits of the eviction, keys past shared memory."""

import numpy as np
import pytest
import torch

from oracle import paged as opg
from webyiq_b200 import W4A8Error, ops

from test_gpu_paged import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("H,KVH,D,lens,news", [
    (8, 2, 256, [40, 65, 1, 90], [33, 1, 1, 65]),   # pairs of CTAs, second row tiles of one token and of none
    (8, 2, 256, [70, 0, 3], [3, 0, 5]),             # one row tile; tokens that see nothing
    (32, 8, 128, [40, 65, 1, 90], [33, 1, 1, 65]),  # two row tiles a CTA
    (6, 2, 192, [300, 2], [70, 2]), (16, 1, 64, [129, 1], [9, 1])])
def test_back_to_back(cuda, H, KVH, D, lens, news):
    """Short items with little or no output, call after call: a CTA's last barrier arrivals come before it
    leaves, and its successor's barriers are its own.  The same bits every time, no wait that gave up."""
    c = Case(cuda, lens, news, H, KVH, D, seed=D)
    o, lse = ops.attn_paged(c.q, c.kv, c.batch)
    c.check(o, lse)
    acc = ops.attn_weights(c.q, lse, c.kv, c.batch, torch.zeros((c.B, KVH, c.batch.max_kv), device=cuda))
    got = []
    for _ in range(100):
        o2, lse2 = ops.attn_paged(c.q, c.kv, c.batch)
        got.append((o2, lse2, ops.attn_weights(c.q, lse2, c.kv, c.batch, torch.zeros_like(acc))))
    assert ops.device_error() == 0
    assert all(torch.equal(a, o) and torch.equal(b, lse) and torch.equal(w, acc) for a, b, w in got)


def test_line_too_long(cuda):
    """Lengths and starts whose work passes 2^31 steps (the page table leads all of it to one page): nothing is
    computed, the device error word says why, and the next call is as ever."""
    T, L = 1 << 17, 1 << 30
    k = torch.zeros((1, 16, 1024, 16), dtype=torch.float16, device=cuda)
    kv = ops.PagedKV(k, k.clone())

    def i32(*a):
        return torch.tensor(a, dtype=torch.int32, device=cuda)

    batch = ops.PagedBatch(i32(0, T), i32(L), torch.zeros((1, 1 << 20), dtype=torch.int32, device=cuda), T, 1000)
    q = torch.zeros((T, 16, 16), dtype=torch.float16, device=cuda)
    o, lse = torch.full_like(q, 7), torch.full((T, 16), 7.0, device=cuda)
    ops.attn_paged(q, kv, batch, o=o, lse=lse)
    with pytest.raises(W4A8Error, match="0x20"):
        ops.device_error()
    assert (o == 7).all() and (lse == 7).all()
    acc = torch.zeros((1, 16, 1 << 24), device=cuda)
    ops.attn_weights(q, lse, kv, batch, acc)
    with pytest.raises(W4A8Error, match="0x20"):
        ops.device_error()
    assert not acc.any()
    c = Case(cuda, [300], [40], 8, 2, 128)
    c.check(*ops.attn_paged(c.q, c.kv, c.batch))
    assert ops.device_error() == 0
