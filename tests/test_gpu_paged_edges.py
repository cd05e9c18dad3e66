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


def _dense(c, abs_v=False):
    """Float64 attention on the GPU, one sequence and head at a time."""
    o = torch.zeros((c.T, c.H, c.D), dtype=torch.float64, device=c.cuda)
    lse = torch.full((c.T, c.H), -torch.inf, dtype=torch.float64, device=c.cuda)
    G = c.H // c.KVH
    for b in range(c.B):
        n, L = int(c.news[b]), int(c.lens[b])
        pg, row = (torch.from_numpy(x).to(c.cuda) for x in opg.slots(c.table, b, L, c.page))
        k, v = c.k[pg, :, row].double(), c.v[pg, :, row].double()
        v = v.abs() if abs_v else v
        t = slice(int(c.q_start[b]), int(c.q_start[b]) + n)
        sees = torch.ones((n, L), dtype=torch.bool, device=c.cuda).tril(L - n)
        for h in range(c.H):
            s = (c.q[t, h].double() @ k[:, h // G].T / c.D ** 0.5).masked_fill(~sees, -torch.inf)
            lse[t, h] = s.logsumexp(1)
            o[t, h] = s.softmax(1) @ v[:, h // G]
    return o, lse


@pytest.mark.parametrize("lens,news,H,KVH,D", [
    ([100003], [1], 8, 2, 256),                                                   # one item over all CTAs
    ([6000] * 24, [1] * 24, 32, 8, 128), ([6000] * 24, [40] * 24, 32, 8, 128),    # a CTA has whole items
    ([6000] * 80, [1] * 80, 8, 2, 256), ([6000] * 40, [40] * 40, 8, 2, 256), ([9000] * 150, [1] * 150, 4, 1, 64)])
@pytest.mark.parametrize("below", [5.4, 16.0, 17.5])
def test_tail_beside_a_sink(cuda, lens, news, H, KVH, D, below):
    """One slot with a score far above all others and a V row of zeros (an attention sink), f16: the output is
    what the many small weights give.  A weight w, relative to the row's largest, is stored with an error of
    at most max(2^-11 w, 2^-32) (f16 of 2^7 w, whose subnormal step is 2^-24); f32 scores of up to 20 add 2e-5 w.
    So |err| <= (2^-11 + 2e-5) sum p |v| + 2^-32 sum |v|, sums over the slots seen."""
    c = Case(cuda, lens, news, H, KVH, D, "f16", page=64, seed=int(below))
    rng = np.random.default_rng(7)
    c.q.copy_(torch.from_numpy(rng.standard_normal((c.T, H, D)) * 0.1).to(cuda))
    c.q[:, :, 0] = 4
    at = 300 if below < 8 else 0  # a late one: the reference that the weights are taken against stays below it
    for b, L in enumerate(lens):
        pg, row = (torch.from_numpy(x).to(cuda) for x in opg.slots(c.table, b, L, c.page))
        k, v = c.k[pg, :, row], c.v[pg, :, row] + 1
        k[:, :, 0] = 0
        k[at], v[at] = 0, 0
        k[at, :, 0] = below * D ** 0.5 / 4
        c.k[pg, :, row], c.v[pg, :, row] = k, v
    o, lse = ops.attn_paged(c.q, c.kv, c.batch, o=torch.empty((c.T, H, D), device=cuda))
    assert ops.device_error() == 0
    ro, rl = _dense(c)
    size = _dense(c, abs_v=True)[0]
    many = torch.repeat_interleave(torch.tensor(lens, device=cuda), torch.tensor(news, device=cuda))[:, None, None]
    bad = (o.double() - ro).abs() > (2.0 ** -11 + 2e-5) * size + 2.0 ** -32 * 1.5 * many
    assert not bad.any(), (int(bad.sum()), ((o.double() - ro).abs() / ro.abs()).max().item())
    assert ((lse.double() - rl).abs() <= 1e-5 * (1 + rl.abs())).all()
