"""The paged operators together, as examples/paged_attention_layer.py runs them: chunks of
prompts beside single tokens, against a dense float64 attention over the framework's own
projections; and with a budget, against the same over the slots that the eviction's rule
keeps.  Tolerance of o as in test_gpu_paged.py (f16 cache): weights rounded to 2^-11 and
cached rows to 2^-11 each, |err| <= 2^-11 (3 max|v| + ...) with the scores' error: a score
of size s moves by s 2^-10 from the rounding of q and k, so a weight by that factor; with
scores up to 8: 8e-3 max|v| bounds it."""

import importlib.util
import os

import numpy as np
import pytest
import torch

from oracle import paged as opg
from webyiq_b200 import ops

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "paged_attention_layer.py")


def _example():
    spec = importlib.util.spec_from_file_location("paged_attention_layer", PATH)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def _dense(layer, history, keep, b, out, rows):
    """o of new rows of sequence b over the kept positions [KVH][...] of its history of qkv rows."""
    H, KVH, D = layer.H, layer.KVH, layer.D
    x = history.reshape(len(history), -1, D)
    cs = layer.rope.double().cpu().numpy()
    qn, kn = (w.double().cpu().numpy() for w in (layer.q_norm, layer.k_norm))
    n = len(history)
    ref = np.zeros((len(rows), H, D))
    for h in range(H):
        kh = h // (H // KVH)
        k = opg.norm_rope(x[:, 2 * H + kh], kn, 1e-6, cs[:n], False)
        v = x[:, 2 * H + KVH + kh]
        for i, t in enumerate(rows):
            q = opg.norm_rope(x[t:t + 1, 2 * h], qn, 1e-6, cs[t:t + 1], False)[0]
            at = np.array([p for p in keep[kh] if p <= t])
            s = k[at] @ q / np.sqrt(D)
            e = np.exp(s - s.max())
            ref[i, h] = e @ v[at] / e.sum() / (1 + np.exp(-x[t, 2 * h + 1]))
    return ref


@pytest.mark.parametrize("budget", [None, 48])
def test_layer(cuda, budget):
    ex = _example()
    torch.manual_seed(3)
    layer = ex.Layer(hidden=256, H=4, KVH=2, D=128, rot=64, max_pos=256)
    plan = [[40, 1, 25], [30, 1, 0], [1, 1, 1], [1, 2, 33], [1, 1, 1], [1, 0, 1]]
    cache = ex.Cache(layer, 3, slots=128)
    cache.kv.k.fill_(float("nan"))
    cache.kv.v.fill_(float("nan"))
    history = [np.zeros((0, (2 * 4 + 2 * 2) * 128)) for _ in range(3)]
    kept = [[[] for _ in range(2)] for _ in range(3)]  # positions in the cache by sequence and head
    for news in plan:
        out = ex.step(layer, cache, torch.randn(sum(news), 256, device=cuda), news, budget=budget, recent=8, sink=2)
        qkv, o = out["qkv"].double().cpu().numpy(), out["o"].double().cpu().numpy()
        at = 0
        for b, m in enumerate(news):
            rows = range(len(history[b]), len(history[b]) + m)
            history[b] = np.concatenate([history[b], qkv[at:at + m]])
            for kh in range(2):
                kept[b][kh] += list(rows)
            if m:
                ref = _dense(layer, history[b], kept[b], b, out, list(rows))
                vmax = np.abs(history[b]).max()
                assert np.all(np.abs(o[at:at + m] - ref) <= 8e-3 * vmax), np.abs(o[at:at + m] - ref).max() / vmax
            at += m
            # after an eviction: the cache's own record of what stayed, which must hold the sinks and the latest
            n = cache.len[b]
            assert n == (min(len(kept[b][0]), budget) if budget and n != len(kept[b][0]) else len(kept[b][0]))
            for kh in range(2):
                now = cache.pos[b, kh, :n].cpu().tolist()
                assert set(now) <= set(kept[b][kh]) and len(set(now)) == n
                if n < len(kept[b][kh]):
                    seen = cache.seen[b]
                    assert {0, 1} <= set(now) and set(range(seen - 8, seen)) <= set(now)
                kept[b][kh] = now
        # weights of a step sum to the rows that gave them, over what is still cached or was before
        if budget is None:
            for b in range(3):
                total = cache.acc[b, :, :cache.len[b]].double().sum(1).cpu().numpy()
                assert np.allclose(total, cache.seen[b] * 2, rtol=1e-3)
    assert ops.device_error() == 0


def test_example_runs(cuda, capsys, monkeypatch):
    ex = _example()
    monkeypatch.setattr("sys.argv", ["x", "--steps", "6", "--budget", "64"])
    ex.main()
    assert "slots [64" in capsys.readouterr().out
