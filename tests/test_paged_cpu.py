"""CPU: the paged operators' entry points refuse bad arguments before any launch, and the
float64 restatements they are tested against agree with the definitions worked out
another way."""

import ctypes
import math

import numpy as np
import pytest

from oracle import paged as opg
from webyiq_b200 import _lib

P = ctypes.c_void_p
CACHE = dict(k=256, v=256, dtype=0, pages=9, page=32, ps=2 * 32 * 128, hs=32 * 128, rs=128)
BATCH = dict(q_start=256, kv_len=512, table=256, batch=2, per=4, tokens=5, max_q=3, max_kv=100)


def _args(**kw):
    return {**CACHE, **BATCH, **dict(H=8, KVH=2, D=128, scale=0.1), **kw}


def _rope(**kw):
    a = _args(**{**dict(qkv=256, rows=12 * 128, qhs=128, rope=256, rot=64, rope_rows=10, pos=256, q=256), **kw})
    return _lib.load().w4a8_qk_norm_rope_kv(
        P(a["qkv"]), a["rows"], a["qhs"], a["H"], a["KVH"], a["D"], None, None, 1e-6, P(a["rope"]), a["rot"],
        a["rope_rows"], 0, P(a["pos"]), P(a["q_start"]), P(a["kv_len"]), P(a["table"]), a["batch"], a["per"], a["tokens"],
        P(a["q"]), P(a["k"]), P(a["v"]), a["dtype"], a["pages"], a["page"], a["ps"], a["hs"], a["rs"], None)


def _attn(**kw):
    a = _args(**{**dict(q=256, qrow=8 * 128, gate=0, gr=0, gh=0, o=256, otype=0, ws=256, wsn=1 << 30), **kw})
    return _lib.load().w4a8_attn_paged(
        P(a["q"]), a["qrow"], a["H"], a["KVH"], a["D"], a["scale"], P(a["gate"]), a["gr"], a["gh"], P(a["q_start"]),
        P(a["kv_len"]), P(a["table"]), a["batch"], a["per"], a["tokens"], a["max_q"], a["max_kv"], P(a["k"]), P(a["v"]),
        a["dtype"], a["pages"], a["page"], a["ps"], a["hs"], a["rs"], P(a["o"]), a["otype"], None, P(a["ws"]), a["wsn"],
        None)


def _weights(**kw):
    a = _args(**{**dict(q=256, qrow=8 * 128, lse=256, acc=256, stride=100, ws=0, wsn=0), **kw})
    return _lib.load().w4a8_attn_weights(
        P(a["q"]), a["qrow"], P(a["lse"]), a["H"], a["KVH"], a["D"], a["scale"], P(a["q_start"]), P(a["kv_len"]),
        P(a["table"]), a["batch"], a["per"], a["tokens"], a["max_q"], a["max_kv"], P(a["k"]), a["dtype"], a["pages"],
        a["page"], a["ps"], a["hs"], a["rs"], P(a["acc"]), a["stride"], P(a["ws"]), a["wsn"], None)


def _evict(**kw):
    a = _args(**{**dict(acc=256, pos=256, stride=100, keep=256, low=256, sink=0, acc_out=256, pos_out=256, len_out=256,
                        ws=256, wsn=1 << 30), **kw})
    return _lib.load().w4a8_kv_evict(
        P(a["k"]), P(a["v"]), a["dtype"], a["pages"], a["page"], a["ps"], a["hs"], a["rs"], a["KVH"], a["D"],
        P(a["kv_len"]), P(a["table"]), a["batch"], a["per"], P(a["acc"]), P(a["pos"]), a["stride"], P(a["keep"]),
        P(a["low"]), a["sink"], P(a["acc_out"]), P(a["pos_out"]), P(a["len_out"]), P(a["ws"]), a["wsn"], None)


SHARED = [dict(KVH=3), dict(KVH=0), dict(D=24), dict(D=272), dict(D=0), dict(k=0), dict(k=264), dict(dtype=2), dict(dtype=-1),
          dict(page=20), dict(page=0), dict(page=2048), dict(pages=0), dict(rs=64), dict(rs=132), dict(hs=8), dict(ps=8),
          dict(hs=100), dict(ps=1 << 40), dict(kv_len=0), dict(table=0), dict(batch=0), dict(batch=70000), dict(per=0),
          dict(per=1 << 21)]
STEP = [dict(q_start=0), dict(tokens=-1), dict(tokens=1 << 25), dict(H=7), dict(H=2 * 129)]


@pytest.mark.parametrize("call,cases", [
    (_rope, SHARED + STEP + [dict(v=0), dict(qkv=0), dict(q=0), dict(qkv=264), dict(q=264), dict(rows=11 * 128), dict(qhs=64),
                             dict(qhs=130), dict(rows=12 * 128 + 2), dict(rot=8), dict(rot=144), dict(rot=-16),
                             dict(rope=0), dict(pos=0), dict(rope_rows=0)]),
    (_attn, SHARED + STEP + [dict(v=0), dict(q=0), dict(o=0), dict(q=264), dict(o=264), dict(qrow=1000), dict(qrow=1028),
                             dict(otype=1), dict(otype=3), dict(gate=264, gr=4, gh=4), dict(gate=256, gr=6, gh=4),
                             dict(gate=256, gr=4, gh=-4), dict(max_q=-1), dict(max_kv=-1), dict(scale=math.nan),
                             dict(scale=-1.0), dict(ws=0), dict(wsn=0), dict(ws=260)]),
    (_weights, SHARED + STEP + [dict(q=0), dict(lse=0), dict(acc=0), dict(q=264), dict(acc=258), dict(qrow=1000),
                                dict(stride=99), dict(max_q=-1), dict(scale=math.nan), dict(max_q=40), dict(max_q=40, ws=264, wsn=1 << 20)]),
    (_evict, SHARED + [dict(v=0), dict(acc=0), dict(pos=0), dict(keep=0), dict(low=0), dict(acc_out=0), dict(pos_out=0),
                       dict(len_out=0), dict(len_out=512), dict(stride=0), dict(sink=-1), dict(ws=0), dict(wsn=0),
                       dict(batch=40000), dict(ws=260)])])
def test_refusals(call, cases):
    for kw in cases:
        if call is _evict and "KVH" in kw and kw["KVH"] == 3:
            continue  # any head count does there
        assert call(**kw) == _lib.EINVAL, kw
        assert _lib.load().w4a8_last_error(), kw


def test_no_tokens_is_a_no_op():
    """Nothing launched, so no GPU needed; null token arrays are fine then."""
    assert _rope(tokens=0, qkv=0, q=0, pos=0) == _lib.OK
    assert _attn(tokens=0, q=0, o=0) == _lib.OK
    assert _weights(tokens=0, q=0, lse=0, acc=0) == _lib.OK


def test_layouts_of_the_cache():
    """Any nested order of pages, heads and rows is taken; overlaps are not."""
    D = 128
    for kw in (dict(rs=2 * D, hs=D, ps=32 * 2 * D), dict(hs=9 * 32 * D, ps=32 * D, rs=D), dict(rs=D + 8, hs=32 * (D + 8), ps=2 * 32 * (D + 8)),
               dict(pages=1, ps=0), dict(KVH=1, H=8, hs=0, ps=32 * D)):
        assert _weights(tokens=0, **kw) == _lib.OK, (kw, _lib.load().w4a8_last_error())
    for kw in (dict(hs=31 * D), dict(rs=D, hs=D, ps=64 * D), dict(ps=2 * 32 * D - 8)):
        assert _weights(tokens=0, **kw) == _lib.EINVAL, kw


def test_workspace_sizes():
    L = _lib.load()
    assert L.w4a8_kv_evict_workspace_bytes(0, 1, 1) == 0
    assert L.w4a8_kv_evict_workspace_bytes(4, 8, 30016) >= 4 * 8 * 30016 // 2 * 8
    assert L.w4a8_attn_weights_workspace_bytes(8, 2, 32) == 0 < L.w4a8_attn_weights_workspace_bytes(8, 2, 33)
    assert L.w4a8_attn_paged_workspace_bytes(1, 8, 2, 256, 1, 1, 100000) >= 16


def test_restatements():
    """attention against one dense softmax; weights sum to one a row; eviction keeps the largest."""
    rng = np.random.default_rng(0)
    H, KVH, D, page, L, n = 4, 2, 16, 16, 41, 6
    k, v = rng.standard_normal((2, 5, KVH, page, D))
    table = np.array([[3, 0, 4]])
    q = rng.standard_normal((n, H, D))
    o, lse = opg.attention(q, k, v, table, np.array([0, n]), [L], 0.25)
    flat = [x[table[0]].transpose(1, 0, 2, 3).reshape(KVH, -1, D)[:, :L] for x in (k, v)]
    for h in range(H):
        s = q[:, h] @ flat[0][h // 2].T * 0.25
        s[np.arange(L)[None] > L - n + np.arange(n)[:, None]] = -np.inf
        p = np.exp(s)
        np.testing.assert_allclose(o[:, h], p / p.sum(1, keepdims=True) @ flat[1][h // 2], rtol=1e-12)
        np.testing.assert_allclose(lse[:, h], np.log(p.sum(1)), rtol=1e-12)
    acc = opg.weights(q, lse, k, table, np.array([0, n]), [L], 0.25, np.zeros((1, KVH, L)))
    np.testing.assert_allclose(acc.sum(2), n * H / KVH)
    assert np.all(opg.norm_rope(q[:, 0], None, 0, np.zeros((n, 0)), False) == q[:, 0])
    pos = np.tile(np.arange(L), (1, KVH, 1))
    k2, _, a, p, lens = opg.evict(k, v, table, [L], acc, pos, [20], [L - 5], 1)
    assert lens == [20]
    for h in range(KVH):
        kept = set(p[0, h])
        assert kept >= {0, *range(L - 5, L)} and len(kept) == 20
        rest = [j for j in range(1, L - 5) if j not in kept]
        assert acc[0, h, rest].max() <= min(acc[0, h, j] for j in kept if 1 <= j < L - 5)
        got = k2[table[0]].transpose(1, 0, 2, 3).reshape(KVH, -1, D)[h, :20]
        np.testing.assert_array_equal(got, flat[0][h][p[0, h]])
