"""The paged-cache operators at the edges of what their header allows: kernels that end right
after their last MMA, long lines, tails of a softmax far below its largest weight, signed
limits of the eviction, keys past shared memory."""

import ctypes

import numpy as np
import pytest
import torch

from oracle import paged as opg
from webyiq_b200 import W4A8Error, _lib, ops

from test_gpu_paged import Case, test_evict as check_evict

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


def _evicted(cuda, lens, keep, low, sink, acc, pos, seed=0):
    """(positions kept of each head, len_out) of an eviction, checked against rows of the cache that moved with them."""
    KVH, D = acc.shape[1], 64
    c = Case(cuda, lens, [0] * len(lens), KVH, KVH, D, seed=seed)
    k0 = c.host(c.k)
    a, p, n = ops.kv_evict(c.kv, c.batch, torch.from_numpy(acc).to(cuda), c.i32(pos), c.i32(keep), c.i32(low), sink=sink)
    p, n, k1 = p.cpu().numpy(), n.cpu().tolist(), c.host(c.k)
    for b, L in enumerate(lens):
        pg, row = opg.slots(c.table, b, L, c.page)
        for h in range(KVH):
            slot_of = {x: j for j, x in enumerate(pos[b, h, :L])}
            came = [slot_of[x] for x in p[b, h, :n[b]]]
            np.testing.assert_array_equal(k1[pg[:n[b]], h, row[:n[b]]], k0[pg[came], h, row[came]])
    return [[sorted(p[b, h, :n[b]].tolist()) for h in range(KVH)] for b in range(len(lens))], n


def test_evict_limits_are_signed(cuda):
    """protect_from at or below zero protects every slot (a sequence shorter than its window of latest tokens),
    so the lowest slots stay; a negative keep keeps none."""
    rng = np.random.default_rng(1)
    acc = rng.random((4, 2, 100)).astype(np.float32)
    pos = np.stack([[rng.permutation(100) for _ in range(2)] for _ in range(4)])
    kept, n = _evicted(cuda, [100] * 4, [40, 40, -3, 40], [-28, 0, 50, 2 ** 31 - 1], 0, acc, pos)
    assert n == [40, 40, 0, 40]
    for b in (0, 1):
        assert kept[b] == [sorted(pos[b, h, :40].tolist()) for h in range(2)]
    # protect_from past every position: by weight alone
    assert kept[3] == [sorted(pos[3, h, np.argsort(-acc[3, h], kind="stable")[:40]].tolist()) for h in range(2)]
    # the unsigned entry point takes the same bits as large values: nothing protected, everything kept
    c = Case(cuda, [100] * 4, [0] * 4, 2, 2, 64)
    dacc, dpos, n = torch.from_numpy(acc).to(cuda), c.i32(pos), torch.zeros(4, dtype=torch.int32, device=cuda)
    ws = ops.kv_evict_workspace(c.batch, 2, cuda, 100)
    keep, low = c.i32([40, 40, -3, 40]), c.i32([-28, 0, 50, 2 ** 31 - 1])
    p = [ctypes.c_void_p(t.data_ptr()) for t in (c.k, c.v, c.batch.kv_len, c.batch.table, dacc, dpos, keep, low, n, ws)]
    st = _lib.load().w4a8_kv_evict(p[0], p[1], *c.kv.layout, 2, 64, p[2], p[3], 4, c.batch.table.shape[1], p[4], p[5], 100,
                                   p[6], p[7], 0, p[4], p[5], p[8], p[9], ws.numel(), None)
    torch.cuda.synchronize()
    assert st == _lib.OK and n.cpu().tolist() == [40, 40, 100, 40]
    got = sorted(dpos[0, 0, :40].cpu().tolist())
    assert got == sorted(pos[0, 0, np.argsort(-acc[0, 0], kind="stable")[:40]].tolist())


def test_evict_infinite_weight_is_no_protection(cuda):
    """Protected slots come before any weight, +inf too, whatever the slots' order."""
    acc = np.ones((1, 2, 64), np.float32)
    acc[0, 0, :30] = np.inf
    acc[0, 1, 3:50:2] = np.inf
    pos = np.tile(np.arange(64), (1, 2, 1))
    kept, n = _evicted(cuda, [64], [16], [56], 4, acc, pos)
    assert n == [16]
    assert kept[0][0] == [*range(8), *range(56, 64)]                         # 4 sinks, the first 4 infinite, the latest 8
    assert kept[0][1] == [0, 1, 2, 3, 5, 7, 9, 11, *range(56, 64)]


@pytest.mark.parametrize("stride,kind,dtype", [(49152, "ties", "f16"), (49153, "ties", "f16"), (49153, "odd", "bf16"),
                                               (70000, "spread", "bf16"), (70000, "ties", "f16")])
def test_evict_keys_in_the_workspace(cuda, stride, kind, dtype):
    """So many heads that each gets one CTA, whose keys lie in shared memory up to 49152 slots of a head and in the
    workspace past that: both sides of it, with a separate output and in place."""
    B, KVH = 26, 3
    assert B * KVH * 2 > torch.cuda.get_device_properties(cuda).multi_processor_count  # (no clusters)
    big = torch.zeros((B, KVH, stride), dtype=torch.float32, device=cuda)
    keys = _lib.load().w4a8_kv_evict_workspace_bytes(B, KVH, stride) - 2 * B * KVH * (stride // 2 + 1) * 4
    assert (keys >= big.numel() * 4) == (stride > 49152)
    lens = [stride - 3, 20011] + [20 + b for b in range(B - 2)]  # (the helper's weights have three slots more)
    check_evict(cuda, KVH, 16, 16, lens, [20001, 20000] + [13] * (B - 2), kind, dtype)


@pytest.mark.parametrize("over", ["keep", "low"])
def test_evict_length_over_a_limit(cuda, over):
    """len_out in the place of keep or of protect_from: every head still goes by the limits as they were."""
    rng = np.random.default_rng(2)
    B, KVH, L = 24, 16, 700
    acc, pos = rng.random((B, KVH, L)).astype(np.float32), np.tile(np.arange(L), (B, KVH, 1))
    for _ in range(5):
        c = Case(cuda, [L] * B, [0] * B, KVH, KVH, 16)
        limits = {"keep": c.i32([150 + b for b in range(B)]), "low": c.i32([L - 60 - b for b in range(B)])}
        _, p, n = ops.kv_evict(c.kv, c.batch, torch.from_numpy(acc).to(cuda), c.i32(pos), limits["keep"], limits["low"],
                               len_out=limits[over])
        assert n is limits[over] and n.cpu().tolist() == [150 + b for b in range(B)]
        p = p.cpu().numpy()
        for b in range(B):
            low = L - 60 - b
            for h in range(KVH):
                best = np.argsort(-acc[b, h, :low], kind="stable")[:150 + b - 60 - b]
                assert sorted(p[b, h, :150 + b].tolist()) == sorted([*best.tolist(), *range(low, L)])


@pytest.mark.parametrize("T,H", [(1, 8), (5, 1), (1, 1)])
def test_gate_strides_of_one(cuda, T, H):
    """A dimension of one has no stride: whatever the gate's tensor gives for it is taken."""
    c = Case(cuda, [77], [T], H, 1, 64, seed=T)
    row, head = 3 if T == 1 else 64 * H + 4, 7 if H == 1 else 64
    buf = torch.randn(T * (64 * H + 8) + 16, device=cuda)
    gate = buf.as_strided((T, H, 64), (row, head, 1))
    o, lse = ops.attn_paged(c.q, c.kv, c.batch, gate=gate)
    c.check(o, lse, gate=gate.cpu().numpy())


def test_cache_strides_of_one(cuda):
    """One kv head and one page: whatever strides the tensors give for those dimensions, each its own."""
    c = Case(cuda, [100], [9], 4, 1, 64, page=112)
    one = int(c.table[0, 0])
    k = torch.empty(112 * 64, dtype=c.k.dtype, device=cuda).as_strided((1, 1, 112, 64), (3, 5, 64, 1))
    v = torch.empty(112 * 64, dtype=c.k.dtype, device=cuda).as_strided((1, 1, 112, 64), (7, 2 ** 40, 64, 1))
    k.copy_(c.k[one:one + 1])
    v.copy_(c.v[one:one + 1])
    batch = ops.PagedBatch(c.batch.q_start, c.batch.kv_len, torch.zeros_like(c.batch.table), 9, 100)
    c.check(*ops.attn_paged(c.q, ops.PagedKV(k, v), batch))
