"""One attention layer of a W4A8 decoder over a paged KV cache, as a server would run it:
a batch of sequences of unlike lengths, prompts in chunks beside single tokens, and a
budget of slots a head held by eviction.

    python examples/paged_attention_layer.py [--steps 64] [--budget 256]

Each step: RMSNorm + quantization + qkv projection (ops.quant, ops.matmul), q/k norm,
rotation and append to the pages (ops.qk_norm_rope_kv), attention over the pages with the
gate (ops.attn_paged), the weight every cached slot received (ops.attn_weights), the o
projection, and, where a sequence passes the budget, eviction (ops.kv_evict).  Weights are
random."""

import argparse
import math
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from webyiq_b200 import ops  # noqa: E402


class Layer:
    """Gated attention: rows q | gate by head, then k, then v."""

    def __init__(self, hidden=2048, H=8, KVH=2, D=256, rot=64, max_pos=4096, device="cuda", seed=0):
        g = torch.Generator(device=device).manual_seed(seed)
        self.hidden, self.H, self.KVH, self.D = hidden, H, KVH, D

        def weight(n, k):
            q = torch.randint(-2 ** 31, 2 ** 31, (n, k // 8), generator=g, device=device, dtype=torch.int64).to(torch.int32)
            s = (torch.randn((n, k // 128), generator=g, device=device).abs() * (0.12 / math.sqrt(k))).half()
            return ops.QWeight(q, s, n, k, 128, False)

        self.qkv = weight((2 * H + 2 * KVH) * D, hidden)
        self.o = weight(hidden, H * D)
        self.norm = torch.ones(hidden, device=device)
        self.q_norm = 1 + 0.1 * torch.randn(D, generator=g, device=device)
        self.k_norm = 1 + 0.1 * torch.randn(D, generator=g, device=device)
        angle = torch.arange(max_pos, device=device)[:, None] * 1e6 ** (-torch.arange(rot // 2, device=device) * 2 / rot)
        self.rope = torch.cat([angle.cos(), angle.sin()], 1).float().contiguous()


class Cache:
    """Pages of B sequences, with what eviction goes by: each slot's weight and its token's position."""

    def __init__(self, layer, B, slots, page=32, dtype=torch.float16, device="cuda"):
        per = -(-slots // page)
        shape = (B * per, layer.KVH, page, layer.D)
        self.kv = ops.PagedKV(torch.empty(shape, dtype=dtype, device=device), torch.empty(shape, dtype=dtype, device=device))
        # the pages of a sequence lie anywhere
        self.table = torch.randperm(B * per, device=device).to(torch.int32).view(B, per)
        self.slots = per * page
        self.acc = torch.zeros((B, layer.KVH, self.slots), device=device)
        self.pos = torch.zeros((B, layer.KVH, self.slots), dtype=torch.int32, device=device)
        self.len = [0] * B   # slots in use
        self.seen = [0] * B  # tokens so far


def step(layer, cache, x, news, budget=None, recent=32, sink=4):
    """x f32 [tokens, hidden]: the rows of news[b] new tokens of each sequence.  Returns the layer's output
    (before the residual) and its inner values."""
    dev, B, T = x.device, len(news), x.shape[0]
    cache.len = [n + m for n, m in zip(cache.len, news)]

    def i32(values):
        return torch.tensor(values, dtype=torch.int32, device=dev)

    batch = ops.PagedBatch(i32([sum(news[:b]) for b in range(B + 1)]), i32(cache.len), cache.table, max_q=max(news),
                           max_kv=max(cache.len))
    pos = i32([cache.seen[b] + i for b in range(B) for i in range(news[b])])
    for b, m in enumerate(news):  # the new slots: no weight yet, their own positions
        new = slice(cache.len[b] - m, cache.len[b])
        cache.acc[b, :, new] = 0
        cache.pos[b, :, new] = torch.arange(cache.seen[b], cache.seen[b] + m, device=dev, dtype=torch.int32)
    cache.seen = [n + m for n, m in zip(cache.seen, news)]

    xq, xs = ops.quant(x, norm_w=layer.norm, act=ops.ACT_TOKEN)
    qkv = ops.matmul(layer.qkv, xq, xs, act=ops.ACT_TOKEN)
    q = ops.qk_norm_rope_kv(qkv, cache.kv, batch, pos, layer.rope, layer.H, q_norm=layer.q_norm, k_norm=layer.k_norm,
                            gated=True)
    gate = qkv.view(T, -1, layer.D)[:, 1:2 * layer.H:2]
    o = torch.empty((T, layer.H, layer.D), device=dev)  # f32: the o projection's quantizer takes it
    o, lse = ops.attn_paged(q, cache.kv, batch, gate=gate, o=o)
    ops.attn_weights(q, lse, cache.kv, batch, cache.acc)
    yq, ys = ops.quant(o.view(T, -1), act=ops.ACT_TOKEN)
    y = ops.matmul(layer.o, yq, ys, act=ops.ACT_TOKEN)

    if budget is not None and max(cache.len) > budget:
        ops.kv_evict(cache.kv, batch, cache.acc, cache.pos, i32([budget] * B), i32([n - recent for n in cache.seen]), sink=sink)
        cache.len = [min(n, budget) for n in cache.len]
    return {"y": y, "q": q, "qkv": qkv, "o": o, "lse": lse, "pos": pos}


def main():
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--steps", type=int, default=64)
    ap.add_argument("--budget", type=int, default=256)
    a = ap.parse_args()
    layer = Layer()
    prompts = [300, 40, 150]
    cache = Cache(layer, len(prompts), slots=a.budget + 300)
    left = list(prompts)
    gen = torch.Generator(device="cuda").manual_seed(1)
    for s in range(a.steps):
        news = [min(n, 128) if n else 1 for n in left]  # prompts in chunks of 128, then a token at a time
        left = [max(n - 128, 0) for n in left]
        out = step(layer, cache, torch.randn((sum(news), layer.hidden), generator=gen, device="cuda"), news, budget=a.budget)
        if s < 4 or s == a.steps - 1:
            print(f"step {s}: new tokens {news}, slots {cache.len}, |y| {out['y'].norm().item():.3f}")
    ops.device_error()


if __name__ == "__main__":
    main()
