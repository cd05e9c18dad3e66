"""The example's layer at its budget: every call of the accumulated weights and of the eviction that its steps make,
against the float64 restatements on what the call was given, so that what stays is worked out apart from the
kernels.  Tolerance of the weights as in test_gpu_paged.py; the eviction moves values: exact."""

import numpy as np
import pytest
import torch

from oracle import paged as opg

from test_gpu_paged_layer import _example

pytestmark = pytest.mark.gpu


def _host(t):
    return t.float().cpu().numpy().astype(np.float64)


@pytest.mark.parametrize("budget,recent,sink", [(48, 8, 2), (20, 32, 4)])  # the second: a window past the budget
def test_what_stays(cuda, monkeypatch, budget, recent, sink):
    ex = _example()
    torch.manual_seed(5)
    layer = ex.Layer(hidden=256, H=4, KVH=2, D=128, rot=64, max_pos=256)
    cache = ex.Cache(layer, 3, slots=128)
    cache.kv.k.fill_(float("nan"))
    cache.kv.v.fill_(float("nan"))
    weights, evict, seen = ex.ops.attn_weights, ex.ops.kv_evict, []

    def check_weights(q, lse, kv, batch, acc):
        before, table, lens = _host(acc), batch.table.cpu().numpy(), batch.kv_len.cpu().numpy()
        out = weights(q, lse, kv, batch, acc)
        ref = opg.weights(_host(q), _host(lse), _host(kv.k), table, batch.q_start.cpu().numpy(), lens, 128 ** -0.5, before)
        assert np.all(np.abs(_host(acc) - ref) <= 4e-5 * np.abs(ref) + 1e-6)
        return out

    def check_evict(kv, batch, acc, pos, keep, protect_from, sink):
        k, v, a, p = _host(kv.k), _host(kv.v), _host(acc), pos.cpu().numpy()
        table, lens = batch.table.cpu().numpy(), batch.kv_len.cpu().tolist()
        got = evict(kv, batch, acc, pos, keep, protect_from, sink=sink)
        rk, rv, ra, rp, rn = opg.evict(k, v, table, lens, a, p, keep.cpu().tolist(), protect_from.cpu().tolist(), sink)
        assert got[2].cpu().tolist() == rn == [min(n, budget) for n in lens]
        np.testing.assert_array_equal(_host(kv.k), rk)
        np.testing.assert_array_equal(_host(kv.v), rv)
        for b in range(3):
            for h in range(2):
                assert set(got[1][b, h, :rn[b]].cpu().tolist()) == set(rp[b, h].tolist())
                np.testing.assert_array_equal(got[1][b, h, :rn[b]].cpu().numpy(), rp[b, h])
                np.testing.assert_array_equal(_host(got[0][b, h, :rn[b]]), ra[b, h])
        seen.append(rn)
        return got

    monkeypatch.setattr(ex.ops, "attn_weights", check_weights)
    monkeypatch.setattr(ex.ops, "kv_evict", check_evict)
    for news in [[40, 1, 25], [30, 1, 0], [1, 1, 1], [1, 2, 33], [1, 1, 1], [1, 0, 1]]:
        due = any(n + m > budget for n, m in zip(cache.len, news))
        calls = len(seen)
        ex.step(layer, cache, torch.randn(sum(news), 256, device=cuda), news, budget=budget, recent=recent, sink=sink)
        assert len(seen) == calls + due
        if due:
            assert cache.len == seen[-1]
    assert len(seen) >= 4 and ex.ops.device_error() == 0
