"""The paged-cache operators on the GPU against oracle/paged.py (float64): append with norm
and rotation, attention of new tokens, accumulated weights, eviction.

Tolerances, from the arithmetic (u16 = 2^-11 for f16, 2^-8 for bf16, the unit roundoff):
 - q, k, v rows: one rounding of a f32 result, |err| <= u16 |x| + 1e-5 max|x| (the second
   term: the f32 norm, table products of two, and f16's subnormals).
 - o: weights rounded to 16 bits each carry a relative error up to u16, so the sum is
   off by at most u16 * sum p |v| <= u16 max|v|; one rounding of the result adds
   u16 |o|; f32 scores of size up to 30 add 1e-5 max|v|.
   |err| <= u16 (max|v| + |o|) + 2e-5 max|v|.
 - lse: f32 scores and sums, |err| <= 1e-5 (1 + |lse|).
 - weights: each term off by a factor 1 + 2e-5 (f32 score of size up to 30, and the
   exponential of it), all terms positive: |err| <= 4e-5 (|acc|) + 1e-6.
 - eviction moves values: exact."""

import numpy as np
import pytest
import torch

from oracle import paged as opg
from webyiq_b200 import W4A8Error, ops

pytestmark = pytest.mark.gpu

DT = {"f16": torch.float16, "bf16": torch.bfloat16}
U = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}


class Case:
    """A batch with random pages; slots past every length hold NaN."""

    def __init__(self, cuda, lens, news, H, KVH, D, dtype="f16", page=16, seed=0, token_major=False, big=1.0, pad=0):
        rng = np.random.default_rng(seed)
        self.H, self.KVH, self.D, self.page, self.dtype = H, KVH, D, page, dtype
        self.B, self.lens, self.news = len(lens), np.array(lens), np.array(news)
        self.T = int(self.news.sum())
        per = max(1, -(-max(lens) // page)) + 1
        used = sum(-(-x // page) for x in lens)
        self.pages = used + 3
        order = rng.permutation(self.pages)
        self.table = np.full((self.B, per), 2 ** 31 - 1, np.int64)  # entries past the length: never read
        at = 0
        for b, x in enumerate(lens):
            n = -(-x // page)
            self.table[b, :n] = order[at:at + n]
            at += n
        self.q_start = np.concatenate([[0], np.cumsum(self.news)])
        dt = DT[dtype]
        shape = (self.pages, page, KVH, D + pad) if token_major else (self.pages, KVH, page, D + pad)

        def cache(x):
            t = torch.full(shape, float("nan"), dtype=dt, device=cuda)
            t = t.permute(0, 2, 1, 3) if token_major else t
            t = t[..., :D]
            for b, n in enumerate(lens):
                pg, row = opg.slots(self.table, b, n, page)
                t[torch.from_numpy(pg).to(cuda), :, torch.from_numpy(row).to(cuda)] = \
                    torch.from_numpy(rng.standard_normal((n, KVH, D)) * x).to(cuda).to(dt)
            return t

        self.k, self.v = cache(big), cache(1.0)
        self.q = torch.from_numpy(rng.standard_normal((self.T, H, D)) * 1.5).to(cuda).to(dt)
        self.kv = ops.PagedKV(self.k, self.v)

        def i32(a):
            return torch.from_numpy(np.asarray(a, np.int32)).to(cuda)

        self.i32, self.rng, self.cuda = i32, rng, cuda
        self.batch = ops.PagedBatch(i32(self.q_start), i32(self.lens), i32(self.table), max_q=max(max(news), 1),
                                    max_kv=max(max(lens), 1))

    def host(self, t):
        return t.float().cpu().numpy().astype(np.float64)

    def attention(self, gate=None, scale=None):
        return opg.attention(self.host(self.q), self.host(self.k), self.host(self.v), self.table, self.q_start, self.lens,
                             1 / np.sqrt(self.D) if scale is None else scale, gate)

    def check(self, o, lse, gate=None, scale=None, u=None):
        ro, rl = self.attention(gate, scale)
        u = U[self.dtype] if u is None else u
        vmax = np.nanmax(np.abs(self.host(self.v)))
        o, lse = self.host(o), self.host(lse)
        bad = np.abs(o - ro) > u * (vmax + np.abs(ro)) + 2e-5 * vmax
        assert not bad.any(), (bad.sum(), np.abs(o - ro).max())
        assert np.array_equal(np.isneginf(lse), np.isneginf(rl))
        f = np.isfinite(rl)
        assert np.all(np.abs(lse[f] - rl[f]) <= 1e-5 * (1 + np.abs(rl[f])))


HEADS = [(8, 2, 256), (32, 8, 128), (16, 1, 64), (4, 4, 128), (6, 2, 80), (5, 1, 192), (3, 3, 16), (24, 1, 96)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("H,KVH,D", HEADS)
@pytest.mark.parametrize("lens,news", [
    ([1], [1]), ([16], [1]), ([17], [17]), ([129], [1]), ([128], [128]), ([300, 1, 77], [40, 1, 3]),
    ([0, 5, 260], [0, 0, 131]), ([640, 33, 0, 127], [1, 1, 0, 1])])
def test_attention(cuda, lens, news, H, KVH, D, dtype):
    c = Case(cuda, lens, news, H, KVH, D, dtype, seed=len(lens) + D)
    o, lse = ops.attn_paged(c.q, c.kv, c.batch)
    c.check(o, lse)
    assert ops.device_error() == 0


@pytest.mark.parametrize("page", [16, 32, 48, 128, 400, 1024])
@pytest.mark.parametrize("token_major,pad", [(False, 0), (True, 0), (True, 24)])
def test_attention_pages_and_strides(cuda, page, token_major, pad):
    """Pages that end inside a tile, longer than one, and caches in other orders."""
    c = Case(cuda, [700, 131], [150, 2], 8, 2, 128, page=page, token_major=token_major, pad=pad, seed=page)
    c.check(*ops.attn_paged(c.q, c.kv, c.batch))


@pytest.mark.parametrize("H,KVH,D", [(8, 2, 256), (8, 2, 128), (16, 1, 64)])
def test_attention_more_tokens_than_slots(cuda, H, KVH, D):
    """The first new tokens of a sequence that is shorter than them see nothing: o = 0, lse = -inf."""
    c = Case(cuda, [5, 0, 140], [9, 4, 150], H, KVH, D, seed=3)
    o, lse = ops.attn_paged(c.q, c.kv, c.batch)
    c.check(o, lse)
    assert torch.isneginf(lse[:4]).all() and (o[:4] == 0).all() and (o[9:13] == 0).all()


@pytest.mark.parametrize("lens,news", [([5000], [1]), ([4100, 300], [2, 1]), ([2500], [700]), ([9000], [16])])
@pytest.mark.parametrize("H,KVH,D", [(8, 2, 256), (32, 8, 128), (16, 1, 64)])
def test_attention_long(cuda, lens, news, H, KVH, D):
    if sum(news) > 100:
        lens, news = [x // 2 for x in lens], [x // 4 for x in news]
    c = Case(cuda, lens, news, H, KVH, D, "bf16", page=64, seed=sum(lens))
    c.check(*ops.attn_paged(c.q, c.kv, c.batch))


def _dense(c, scale=None):
    """Float64 attention on the GPU, one sequence and head at a time, for sizes past the restatement's."""
    o = torch.zeros((c.T, c.H, c.D), dtype=torch.float64, device=c.cuda)
    lse = torch.full((c.T, c.H), -torch.inf, dtype=torch.float64, device=c.cuda)
    G = c.H // c.KVH
    for b in range(c.B):
        n, L = int(c.news[b]), int(c.lens[b])
        if not n or not L:
            continue
        pg, row = (torch.from_numpy(x).to(c.cuda) for x in opg.slots(c.table, b, L, c.page))
        k, v = c.k[pg, :, row].double(), c.v[pg, :, row].double()
        t = slice(int(c.q_start[b]), int(c.q_start[b]) + n)
        sees = torch.ones((n, L), dtype=torch.bool, device=c.cuda).tril(L - n)
        for h in range(c.H):
            s = (c.q[t, h].double() @ k[:, h // G].T / c.D ** 0.5).masked_fill(~sees, -torch.inf)
            lse[t, h] = s.logsumexp(1)
            o[t, h] = s.softmax(1).nan_to_num(0) @ v[:, h // G]
    return o, lse


@pytest.mark.parametrize("lens,news", [
    ([100003], [1]), ([60001, 7, 30000], [1, 1, 2]), ([4001], [4001]), ([9000, 300], [1500, 300]),
    ([100 + 37 * i for i in range(60)], [1] * 60), ([1 + i for i in range(300)], [1 + i % 3 for i in range(300)]),
    ([2000 + 13 * i for i in range(12)], [(0, 1, 700, 90)[i % 4] for i in range(12)])])
@pytest.mark.parametrize("H,KVH,D,dtype", [(8, 2, 256, "f16"), (32, 8, 128, "bf16"), (16, 1, 64, "f16"), (6, 2, 192, "bf16"),
                                           (32, 2, 64, "bf16")])
def test_attention_many_steps(cuda, lens, news, H, KVH, D, dtype):
    """Stretches of many kv steps, items of one step, items that several CTAs share; against float64
    on the same GPU, at the restatement's tolerances."""
    c = Case(cuda, lens, news, H, KVH, D, dtype, page=32, seed=len(lens))
    o, lse = ops.attn_paged(c.q, c.kv, c.batch)
    assert ops.device_error() == 0
    ro, rl = _dense(c)
    vmax = c.v.float().nan_to_num(0).abs().max().item()
    bad = (o.double() - ro).abs() > U[dtype] * (vmax + ro.abs()) + 2e-5 * vmax
    assert not bad.any(), (int(bad.sum()), (o.double() - ro).abs().max().item())
    assert torch.equal(torch.isneginf(lse), torch.isneginf(rl))
    f = torch.isfinite(rl)
    assert ((lse.double() - rl)[f].abs() <= 1e-5 * (1 + rl[f].abs())).all()
    again = ops.attn_paged(c.q, c.kv, c.batch)
    assert torch.equal(o, again[0]) and torch.equal(lse, again[1])


def test_attention_gate_strides_types(cuda):
    """A gate beside each head's query, q inside a wider row, f32 output, another scale."""
    c = Case(cuda, [333, 20], [30, 1], 8, 2, 256, seed=9)
    wide = torch.zeros((c.T, 8 * 256 + 64), dtype=torch.float16, device=cuda)
    wide[:, :8 * 256] = c.q.flatten(1)
    q = wide[:, :8 * 256].view(c.T, 8, 256)
    gate = torch.from_numpy(c.rng.standard_normal((c.T, 8, 512)).astype(np.float32)).to(cuda)[:, :, 256:]
    o = torch.empty((c.T, 8, 256), dtype=torch.float32, device=cuda)
    o, lse = ops.attn_paged(q, c.kv, c.batch, scale=0.11, gate=gate, o=o)
    c.check(o, lse, gate=gate.cpu().numpy(), scale=0.11)


@pytest.mark.parametrize("H,KVH,D", [(8, 2, 256), (8, 2, 128)])
def test_attention_large_scores(cuda, H, KVH, D):
    """Scores of some hundreds, the largest in a late tile: the running maximum moves far."""
    c = Case(cuda, [520], [70], H, KVH, D, seed=4)
    pg, row = opg.slots(c.table, 0, 520, c.page)
    grow = torch.linspace(0.1, 30, 520, device=cuda)[:, None, None]
    idx = torch.from_numpy(pg).to(cuda), torch.from_numpy(row).to(cuda)
    c.k[idx[0], :, idx[1]] = (c.k[idx[0], :, idx[1]].float() * grow).half()
    o, lse = ops.attn_paged(c.q, c.kv, c.batch)
    # scores of up to 300 carry f32 errors of 300 * 2^-23 * sqrt(D) terms: 1e-3 relative in a weight
    ro, rl = c.attention()
    vmax = np.nanmax(np.abs(c.host(c.v)))
    assert np.all(np.abs(c.host(o) - ro) <= (U["f16"] * 2 + 1e-3) * vmax)
    assert np.all(np.abs(c.host(lse) - rl) <= 1e-5 * (1 + np.abs(rl)))


def test_attention_other_stream_and_repeat(cuda):
    """On a stream of its own, twice: the same bits; and from a graph after the lengths moved."""
    c = Case(cuda, [900, 64], [1, 1], 8, 2, 256, seed=6)
    a = ops.attn_paged(c.q, c.kv, c.batch)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    ws = ops.attn_paged_workspace(c.batch, c.T, 8, 2, 256, cuda)
    o, lse = torch.empty_like(c.q), torch.empty((c.T, 8), device=cuda)
    with torch.cuda.stream(s):
        b = ops.attn_paged(c.q, c.kv, c.batch, workspace=ws)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            ops.attn_paged(c.q, c.kv, c.batch, o=o, lse=lse, workspace=ws)
    torch.cuda.synchronize()
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    for lens in ([900, 64], [130, 1], [513, 30]):
        c.batch.kv_len.copy_(c.i32(lens))
        c.lens = np.array(lens)
        g.replay()
        torch.cuda.synchronize()
        c.check(o, lse)
    del g


def test_attention_idle_step(cuda):
    c = Case(cuda, [10, 20], [0, 0], 8, 2, 128)
    o, lse = ops.attn_paged(c.q, c.kv, c.batch)
    assert o.shape == (0, 8, 128) and lse.shape == (0, 8)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("H,KVH,D", HEADS)
@pytest.mark.parametrize("lens,news", [([1], [1]), ([33], [33]), ([300, 1, 77, 12], [40, 1, 3, 0]), ([5, 140], [9, 150]),
                                       ([1030], [1])])
def test_weights(cuda, lens, news, H, KVH, D, dtype):
    c = Case(cuda, lens, news, H, KVH, D, dtype, seed=11)
    _, lse = c.attention()
    lse = torch.from_numpy(lse.astype(np.float32)).to(cuda)
    cap = c.batch.max_kv + 5
    acc0 = c.rng.random((c.B, KVH, cap)).astype(np.float32)
    acc = torch.from_numpy(acc0).to(cuda)
    out = ops.attn_weights(c.q, lse, c.kv, c.batch, acc)
    again = ops.attn_weights(c.q, lse, c.kv, c.batch, torch.from_numpy(acc0).to(cuda))
    assert out is acc and torch.equal(acc, again)
    ref = opg.weights(c.host(c.q), c.host(lse), c.host(c.k), c.table, c.q_start, c.lens, 1 / np.sqrt(D), acc0)
    assert np.all(np.abs(c.host(acc) - ref) <= 4e-5 * np.abs(ref) + 1e-6), np.abs(c.host(acc) - ref).max()
    for b, n in enumerate(lens):  # nothing past a sequence's slots
        assert np.array_equal(acc.cpu().numpy()[b, :, n:], acc0[b, :, n:])


@pytest.mark.parametrize("H,KVH,D", [(8, 2, 256), (32, 8, 128), (16, 1, 64)])
@pytest.mark.parametrize("page", [32, 48])
def test_weights_sum_to_rows(cuda, H, KVH, D, page):
    """With attn_paged's own lse the weights of a step sum to one for each row that sees anything."""
    c = Case(cuda, [1500, 640], [260, 1], H, KVH, D, "bf16", page=page, seed=12)
    _, lse = ops.attn_paged(c.q, c.kv, c.batch)
    acc = ops.attn_weights(c.q, lse, c.kv, c.batch, torch.zeros((2, KVH, 1500), device=cuda))
    got = acc.double().sum(2).cpu().numpy()
    assert np.allclose(got, np.array([[260.0], [1.0]]) * (H // KVH), rtol=4e-5)


def _rope_rows(c, qkv, gated, qn, kn, table, pos, interleaved):
    T, H, KVH, D = c.T, c.H, c.KVH, c.D
    x = qkv.reshape(T, -1, D).astype(np.float64)
    step = 2 if gated else 1
    cs = table[pos].astype(np.float64) if table is not None else np.zeros((T, 0))
    q = np.stack([opg.norm_rope(x[:, h * step], qn, 1e-6, cs, interleaved) for h in range(H)], 1)
    k = np.stack([opg.norm_rope(x[:, H * step + h], kn, 1e-6, cs, interleaved) for h in range(KVH)], 1)
    return q, k, x[:, H * step + KVH:]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("H,KVH,D,rot", [(8, 2, 256, 64), (32, 8, 128, 128), (16, 1, 64, 32), (6, 2, 80, 16), (3, 3, 16, 16),
                                         (5, 1, 192, 192), (4, 4, 128, 0)])
@pytest.mark.parametrize("gated,interleaved,norm", [(False, False, True), (True, True, True), (True, False, False)])
def test_norm_rope_append(cuda, H, KVH, D, rot, gated, interleaved, norm, dtype):
    lens, news = [40, 3, 1, 200, 9], [7, 0, 1, 33, 12]  # the last has more new tokens than slots
    c = Case(cuda, lens, news, H, KVH, D, dtype, seed=D + rot)
    rng = c.rng
    width = (H * (2 if gated else 1) + 2 * KVH) * D
    qkv = (rng.standard_normal((c.T, width)) * 2).astype(np.float32)
    qn, kn = (rng.standard_normal(D).astype(np.float32) for _ in range(2)) if norm else (None, None)
    table = rng.standard_normal((300, rot)).astype(np.float32) if rot else None
    pos = rng.integers(0, 300, c.T)
    dev = lambda a: None if a is None else torch.from_numpy(a).to(cuda)  # noqa: E731
    k0, v0 = c.k.clone(), c.v.clone()
    q = ops.qk_norm_rope_kv(dev(qkv), c.kv, c.batch, c.i32(pos), dev(table), H, q_norm=dev(qn), k_norm=dev(kn),
                            gated=gated, interleaved=interleaved)
    rq, rk, rv = _rope_rows(c, qkv, gated, qn, kn, table, pos, interleaved)

    def near(a, b):
        assert np.all(np.abs(a - b) <= U[dtype] * np.abs(b) + 1e-5 * np.abs(b).max()), np.abs(a - b).max()

    near(c.host(q), rq)
    k, v = c.host(c.k), c.host(c.v)
    untouched = np.ones((c.pages, c.page), bool)
    for b in range(c.B):
        pg, row = opg.slots(c.table, b, lens[b], c.page)
        for i in range(news[b]):
            j = lens[b] - news[b] + i
            if j >= 0:
                near(k[pg[j], :, row[j]], rk[c.q_start[b] + i])
                near(v[pg[j], :, row[j]], rv[c.q_start[b] + i])
                untouched[pg[j], row[j]] = False
    m = torch.from_numpy(untouched).to(cuda)[:, None, :, None].expand_as(c.k)
    same = (c.k.view(torch.int16) == k0.view(torch.int16)) & (c.v.view(torch.int16) == v0.view(torch.int16))
    assert same[m].all()


def test_norm_rope_saturates_and_clamps(cuda):
    """A value past f16's range becomes its largest one, NaN stays, a zero row stays zero, and a
    position past the table takes its last row."""
    c = Case(cuda, [4], [4], 2, 1, 64)
    qkv = np.zeros((4, 4 * 64), np.float32)
    qkv[0, 3 * 64] = 1e9
    qkv[1, 3 * 64 + 1] = -1e9
    qkv[2, 3 * 64 + 2] = np.nan
    qkv[3, :128] = 1.0
    table = np.random.default_rng(0).standard_normal((5, 32)).astype(np.float32)
    w = torch.ones(64, device=cuda)
    q = ops.qk_norm_rope_kv(torch.from_numpy(qkv).to(cuda), c.kv, c.batch, c.i32([0, 1, 2, 99]),
                            torch.from_numpy(table).to(cuda), 2, q_norm=w, k_norm=w)
    pg, row = opg.slots(c.table, 0, 4, c.page)
    v = c.v.float().cpu().numpy()[pg, 0, row]
    assert v[0, 0] == 65504 and v[1, 1] == -65504 and np.isnan(v[2, 2]) and np.isfinite(np.delete(v[2], 2)).all()
    assert (q[:3] == 0).all()
    ref = opg.norm_rope(qkv[3:4, :64], np.ones(64), 1e-6, table[4:5].astype(np.float64), False)
    assert np.allclose(q[3, 0].float().cpu().numpy(), ref[0], atol=2e-3)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("KVH,D,page", [(2, 256, 32), (8, 128, 48), (1, 80, 16)])
@pytest.mark.parametrize("lens,keep", [([1], [0]), ([1, 2], [1, 1]), ([100, 1025, 0, 37], [100, 1024, 5, 20]),
                                       ([5000, 2049], [700, 2000]), ([64], [32])])
@pytest.mark.parametrize("kind", ["spread", "ties", "odd"])
def test_evict(cuda, KVH, D, page, lens, keep, kind, dtype):
    B = len(lens)
    c = Case(cuda, lens, [0] * B, KVH, KVH, D, dtype, page=page, seed=sum(lens))
    rng, cap = c.rng, max(lens) + 3
    acc = np.exp(2 * rng.standard_normal((B, KVH, cap))).astype(np.float32)
    if kind == "ties":
        acc = rng.integers(0, 3, acc.shape).astype(np.float32)
    if kind == "odd":
        acc = np.where(rng.random(acc.shape) < 0.5, rng.choice([np.nan, np.inf, -np.inf, 0.0, -0.0, -1.0], acc.shape), acc)
        acc = acc.astype(np.float32)
    pos = np.stack([[rng.permutation(cap) for _ in range(KVH)] for _ in range(B)])
    low = np.array([max(lens) - (7 if kind != "odd" else 900)] * B).clip(0)
    k0, v0 = c.host(c.k), c.host(c.v)
    dacc, dpos = torch.from_numpy(acc).to(cuda), c.i32(pos)
    acc_out, pos_out = torch.full_like(dacc, -7), torch.full_like(dpos, -7)
    a, p, n = ops.kv_evict(c.kv, c.batch, dacc, dpos, c.i32(keep), c.i32(low), sink=2, acc_out=acc_out, pos_out=pos_out)
    rk, rv, ra, rp, rn = opg.evict(k0, v0, c.table, lens, acc, pos, keep, low, 2)
    assert n.cpu().tolist() == rn
    np.testing.assert_array_equal(c.host(c.k), rk)
    np.testing.assert_array_equal(c.host(c.v), rv)
    a, p = a.cpu().numpy(), p.cpu().numpy()
    for b in range(B):
        for h in range(KVH):
            np.testing.assert_array_equal(a[b, h, :rn[b]], ra[b, h])
            np.testing.assert_array_equal(p[b, h, :rn[b]], rp[b, h])
        assert (a[b, :, rn[b]:] == -7).all() and (p[b, :, rn[b]:] == -7).all()
    # in place, the same
    c.k.copy_(torch.from_numpy(k0).to(cuda))
    c.v.copy_(torch.from_numpy(v0).to(cuda))
    a2, p2, n2 = ops.kv_evict(c.kv, c.batch, dacc, dpos, c.i32(keep), c.i32(low), sink=2)
    assert a2 is dacc and torch.equal(n2, n)
    for b in range(B):
        assert np.array_equal(a2.cpu().numpy()[b, :, :rn[b]], a[b, :, :rn[b]], equal_nan=True)
        assert np.array_equal(p2.cpu().numpy()[b, :, :rn[b]], p[b, :, :rn[b]])
    np.testing.assert_array_equal(c.host(c.k), rk)


def test_evict_past_shared_memory(cuda):
    """More slots than a CTA keeps the keys of in shared memory, ties among them."""
    test_evict(cuda, 1, 80, 16, [60000, 52000], [20011, 51999], "ties", "f16")
    test_evict(cuda, 1, 80, 16, [60000, 51201], [59990, 7], "spread", "bf16")


def test_bad_indices_stay_in_range(cuda):
    """Lengths, starts and pages out of range are bounded by the kernels: values of no meaning, no
    access out of range, the context stays usable."""
    c = Case(cuda, [40, 40], [3, 1], 8, 2, 128)
    good = ops.attn_paged(c.q, c.kv, c.batch)[0].clone()
    bad = ops.PagedBatch(c.i32([0, 9, 2]), c.i32([10 ** 6, 39]), c.i32(np.full_like(c.table, 2 ** 31 - 1)), 3, 40)
    acc = torch.zeros((2, 2, 48), device=cuda)
    ops.attn_paged(c.q, c.kv, bad)
    ops.attn_weights(c.q, torch.zeros((4, 8), device=cuda), c.kv, bad, acc)
    ops.kv_evict(c.kv, bad, acc, torch.zeros_like(acc, dtype=torch.int32), c.i32([5, 10 ** 6]), c.i32([0, 0]))
    torch.cuda.synchronize()
    c2 = Case(cuda, [40, 40], [3, 1], 8, 2, 128)
    assert torch.equal(ops.attn_paged(c2.q, c2.kv, c2.batch)[0], good)


def test_refusals_on_tensors(cuda):
    c = Case(cuda, [40], [2], 8, 2, 128)
    f32 = torch.zeros((2, 8, 128), device=cuda)
    with pytest.raises(ValueError):
        ops.attn_paged(f32, c.kv, c.batch)  # q of another type
    with pytest.raises(ValueError):
        ops.attn_paged(c.q[:, :, :64], c.kv, c.batch)
    with pytest.raises(ValueError):
        ops.PagedKV(c.k, c.v.float())
    with pytest.raises(ValueError):
        ops.PagedBatch(c.batch.q_start.long(), c.batch.kv_len, c.batch.table, 1, 1)
    with pytest.raises(W4A8Error) as e:  # an output of a third type
        ops.attn_paged(c.q, c.kv, c.batch, o=torch.zeros((2, 8, 128), dtype=torch.bfloat16, device=cuda))
    assert e.value.status == 1
    with pytest.raises(W4A8Error):
        ops.attn_paged(c.q, c.kv, c.batch, workspace=torch.empty(1, dtype=torch.uint8, device=cuda))
    with pytest.raises(W4A8Error):  # 7 query heads over 2 kv heads
        ops.attn_paged(c.q[:, :7].contiguous(), c.kv, c.batch)
    acc = torch.zeros((1, 2, 40), device=cuda)
    pos = torch.zeros((1, 2, 40), dtype=torch.int32, device=cuda)
    one = c.i32([1])
    with pytest.raises(W4A8Error):  # the new length over the old one
        ops.kv_evict(c.kv, c.batch, acc, pos, one, one, len_out=c.batch.kv_len)
    with pytest.raises(ValueError):
        ops.kv_evict(c.kv, c.batch, acc[:, :, :30].contiguous(), pos[:, :, :30].contiguous(), one, one)
    with pytest.raises(ValueError):
        ops.qk_norm_rope_kv(torch.zeros((2, 13 * 128), device=cuda), c.kv, c.batch, c.i32([0, 1]), None, 8)
