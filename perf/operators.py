"""Measured cases of the paged-cache operators: q/k norm + rotation + cache append,
attention of new tokens over the pages, accumulated attention weights, eviction.

Sequence b of a batch has n_b new tokens (rows q_start[b] .. q_start[b+1]) and kv_len[b]
cached slots, the new tokens' own among them (the last n_b).  Slot j of the sequence is row
j % page of page table[b, j // page]; the cache is k, v [pages, KVH, page, D].  New token i
sees slots 0 .. kv_len[b] - n_b + i.

With `own` false every operator is computed by elementary torch operations in 32 bits;
with `own` true by webyiq_b200.ops."""

import math
import random

import torch

own = False

DT = {"f16": torch.float16, "bf16": torch.bfloat16}
OPS = ("rope", "attn", "weights", "evict")


def _case(name, op, batch, q, kv, H, KVH, D, dtype="f16", page=64, ragged=False, mix=0, **kw):
    return {"name": name, "op": op, "batch": batch, "q": q, "kv": kv, "H": H, "KVH": KVH, "D": D, "dtype": dtype,
            "page": page, "ragged": ragged, "mix": mix, **kw}


def listed():
    return [
        # one token of a decode step of a gated 8/2-head, 256-wide attention layer: latency
        _case("rope_token", "rope", 1, 1, 700, 8, 2, 256, page=32, rot=64, gated=True, pairs="half"),
        # prompts of a batch, three of unlike lengths, full rotation
        _case("rope_prompts", "rope", 3, 4000, 4000, 32, 8, 128, "bf16", ragged=True, mix=3, rot=128, gated=False,
              pairs="half"),
        # one token over a short cache: the smallest attention call of a decode step
        _case("attn_token", "attn", 1, 1, 777, 8, 2, 256, page=32, gated=True),
        # a decode batch of unlike lengths
        _case("attn_batch", "attn", 48, 1, 8191, 32, 8, 128, "bf16", ragged=True, mix=5, gated=False),
        # one token over a long cache
        _case("attn_long", "attn", 1, 1, 100003, 8, 2, 256, page=32, gated=True),
        # a chunk of a long prompt: new tokens over what earlier chunks left
        _case("attn_chunk", "attn", 1, 2048, 16384, 32, 8, 128, "bf16", gated=False),
        # the whole prompt in one chunk, gated 256-wide heads
        _case("attn_prompt", "attn", 1, 4001, 4001, 8, 2, 256, page=32, gated=True),
        # prompts, drafts to verify and single tokens in one step, many query heads on one kv head
        _case("attn_mixed", "attn", 9, 600, 5000, 16, 1, 64, page=16, ragged=True, mix=7, gated=False),
        # what a decode step adds to its slots' weights
        _case("weights_batch", "weights", 16, 1, 6007, 8, 2, 256, page=32, ragged=True, mix=9),
        # what a prompt chunk adds
        _case("weights_chunk", "weights", 1, 1500, 8200, 32, 8, 128, "bf16"),
        # a cache held at its budget: one slot a step goes
        _case("evict_step", "evict", 4, 1, 1025, 8, 2, 256, page=32, keep=1024, recent=32, sink=4),
        # after a prompt: long caches cut to the budget
        _case("evict_prompt", "evict", 4, 1, 30011, 32, 8, 128, "bf16", keep=4096, recent=256, sink=4, ragged=True,
              mix=11),
    ]


# query heads, kv heads, head size: the shapes of the attention tests, and 32/8 heads of 128
HEADS = ((8, 2, 256), (8, 2, 128), (16, 1, 64), (4, 4, 256), (32, 2, 64), (32, 8, 128))


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = {op: max((work(c) for c in listed() if c["op"] == op), key=lambda w: w["bytes"] + w["flops"]) for op in OPS}
    while True:
        H, KVH, D = rng.choice(HEADS)
        op = rng.choice(OPS)
        kind = rng.choice(("token", "chunk", "mixed"))
        batch = _log(rng, 1, 48) if kind == "token" else rng.randint(1, 8)
        kv = _log(rng, 33, 100003)
        q = 1 if kind == "token" else min(kv, _log(rng, 2, 4000))
        c = {"op": op, "batch": batch, "q": q, "kv": kv, "H": H, "KVH": KVH, "D": D,
             "dtype": rng.choice(("f16", "bf16")), "page": rng.choice((16, 32, 48, 64, 128)), "ragged": rng.random() < 0.7,
             "mix": rng.randrange(1 << 20)}
        if op in ("rope", "attn"):
            c["gated"] = rng.random() < 0.4
        if op == "rope":
            c["rot"], c["pairs"] = rng.choice((D, D // 4)), rng.choice(("half", "even"))
        if op == "evict":
            c["q"] = 1
            c["keep"] = max(1, int(kv * rng.uniform(0.05, 0.99)))
            c["recent"], c["sink"] = rng.choice((1, 32, 256)), rng.choice((0, 4))
        w, top = work(c), most[op]
        # the plain forms hold padded scores of every sequence: keep those, too, within the listed cases'
        if w["bytes"] <= top["bytes"] and w["flops"] <= max(top["flops"], 1) and batch * q * H * kv <= 2048 * 16384 * 32 \
                and batch * kv * KVH * D <= 48 * 8191 * 8 * 128 and 3072 not in (q, kv):
            return c


def _lens(c):
    """New tokens and cached slots of each sequence, from the case alone: the first has the
    full sizes; of the others, where they are ragged, some have one new token and one none."""
    n, kv = [c["q"]], [c["kv"]]
    r = random.Random(c["mix"])
    for b in range(1, c["batch"]):
        if not c["ragged"]:
            n.append(c["q"])
            kv.append(c["kv"])
            continue
        L = max(1, int(c["kv"] * r.uniform(0.1, 1.0)))
        m = 1 if r.random() < 0.4 else min(L, max(1, int(c["q"] * r.uniform(0.05, 1.0))))
        if b == c["batch"] - 1 and c["q"] > 1:
            m = 0  # a slot of the batch that is idle this step
        n.append(m)
        kv.append(L)
    return n, kv


def prepare(case, seed):
    c = dict(case)
    dev = "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, generator=g, device=dev)

    n, kv = _lens(c)
    B, T, H, KVH, D, page, dt = c["batch"], sum(n), c["H"], c["KVH"], c["D"], c["page"], DT[c["dtype"]]
    per = -(-max(kv) // page)
    pages = sum(-(-x // page) for x in kv) + 3
    order = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    table = torch.zeros((B, per), dtype=torch.int32, device=dev)
    at = 0
    for b in range(B):
        k = -(-kv[b] // page)
        table[b, :k] = order[at:at + k]
        at += k
    s = {"case": c, "table": table, "max_q": max(n), "max_kv": max(kv), "tokens": T,
         "q_start": torch.tensor([sum(n[:b]) for b in range(B + 1)], dtype=torch.int32, device=dev),
         "kv_len": torch.tensor(kv, dtype=torch.int32, device=dev),
         "k": randn(pages, KVH, page, D).to(dt), "v": randn(pages, KVH, page, D).to(dt)}
    if c["op"] == "rope":
        heads = H * (2 if c["gated"] else 1) + 2 * KVH
        s["qkv"] = randn(T, heads * D) * 1.5
        s["q_norm"], s["k_norm"] = 1 + 0.1 * randn(D), 1 + 0.1 * randn(D)
        R = c["rot"]
        angle = torch.arange(max(kv), device=dev, dtype=torch.float64)[:, None] * \
            1e6 ** (-torch.arange(R // 2, device=dev, dtype=torch.float64) * 2 / R)
        s["rope"] = torch.cat([angle.cos(), angle.sin()], 1).float()
        s["pos"] = torch.cat([torch.arange(x - m, x, dtype=torch.int32) for m, x in zip(n, kv)]).to(dev)
        s["q"] = torch.empty((T, H, D), dtype=dt, device=dev)
    if c["op"] in ("attn", "weights"):
        s["q"] = (1.5 * randn(T, H, D)).to(dt)  # normed queries times a learned weight
    if c["op"] == "attn":
        # the gate sits beside each head's query in the projection's row
        s["gate"] = randn(T, H, 2 * D)[:, :, D:] if c["gated"] else None
        s["o"] = torch.empty((T, H, D), dtype=dt, device=dev)
        s["lse"] = torch.empty((T, H), device=dev)
    if c["op"] == "weights":
        s["lse"] = _plain_attention(s)[1]
        s["acc"] = 3 * torch.rand((B, KVH, per * page), generator=g, device=dev)
    if c["op"] == "evict":
        cap = per * page
        # accumulated weights are heavy-tailed: a few slots hold most of the mass
        s["acc"] = torch.exp(2 * randn(B, KVH, cap))
        # earlier evictions left the slots out of order
        s["pos"] = torch.stack([torch.stack([torch.randperm(cap, generator=g, device=dev) for _ in range(KVH)])
                                for _ in range(B)]).to(torch.int32)
        s["protect_from"] = torch.full((B,), cap - c["recent"], dtype=torch.int32, device=dev)
        s["keep"] = torch.full((B,), c["keep"], dtype=torch.int32, device=dev)
        s["acc_out"], s["pos_out"] = torch.zeros_like(s["acc"]), torch.zeros_like(s["pos"])
        s["len_out"] = torch.zeros_like(s["kv_len"])
    if own:
        from webyiq_b200 import ops

        s["kv"] = ops.PagedKV(s["k"], s["v"])
        s["batch"] = ops.PagedBatch(s["q_start"], s["kv_len"], table, max_q=s["max_q"], max_kv=s["max_kv"])
        if c["op"] == "attn":
            s["ws"] = ops.attn_paged_workspace(s["batch"], T, H, KVH, D, dev)
        if c["op"] == "evict":
            s["ws"] = ops.kv_evict_workspace(s["batch"], KVH, dev)
    return s


def run(state):
    s, c = state, state["case"]
    if own:
        from webyiq_b200 import ops

        if c["op"] == "rope":
            q = ops.qk_norm_rope_kv(s["qkv"], s["kv"], s["batch"], s["pos"], s["rope"], c["H"], q_norm=s["q_norm"],
                                    k_norm=s["k_norm"], eps=1e-6, gated=c["gated"], interleaved=c["pairs"] == "even",
                                    q=s["q"])
            return {"q": q, "k": s["k"], "v": s["v"]}
        if c["op"] == "attn":
            o, lse = ops.attn_paged(s["q"], s["kv"], s["batch"], gate=s["gate"], o=s["o"], lse=s["lse"], workspace=s["ws"])
            return {"o": o, "lse": lse}
        if c["op"] == "weights":
            return {"acc": ops.attn_weights(s["q"], s["lse"], s["kv"], s["batch"], s["acc"])}
        ops.kv_evict(s["kv"], s["batch"], s["acc"], s["pos"], s["keep"], s["protect_from"], sink=c["sink"],
                     acc_out=s["acc_out"], pos_out=s["pos_out"], len_out=s["len_out"], workspace=s["ws"])
        return {"k": s["k"], "v": s["v"], "acc": s["acc_out"], "pos": s["pos_out"], "len": s["len_out"]}
    if c["op"] == "rope":
        return _plain_rope(s)
    if c["op"] == "attn":
        o, lse = _plain_attention(s)
        if s["gate"] is not None:
            o = o / (1 + torch.exp(-s["gate"]))
        return {"o": o.to(s["q"].dtype), "lse": lse}
    if c["op"] == "weights":
        return {"acc": _plain_weights(s)}
    return _plain_evict(s)


# ---------------------------------------------------------------------------
# The plain forms.  Sequences are padded to the longest; t_seq and t_i give the
# sequence of each new token and its place in it.


def _rows(s):
    t = torch.arange(s["tokens"], device="cuda")
    start = s["q_start"].long()
    t_seq = torch.searchsorted(start[1:].contiguous(), t, right=True)
    return t_seq, t - start[t_seq]


def _slots(s, seq, slot):
    """Page and row in the page of slots of sequences."""
    page = s["case"]["page"]
    return s["table"].long()[seq, slot // page], slot % page


def _plain_rope(s):
    c = s["case"]
    H, KVH, D, R = c["H"], c["KVH"], c["D"], c["rot"]
    T = s["tokens"]
    qh = H * (2 if c["gated"] else 1)
    x = s["qkv"].view(T, qh + 2 * KVH, D)
    q = x[:, :qh:2] if c["gated"] else x[:, :qh]

    def norm(y, w):
        return y * torch.rsqrt((y * y).mean(-1, keepdim=True) + 1e-6) * w

    cs = s["rope"][s["pos"].long()][:, None]
    cos, sin = cs[..., :R // 2], cs[..., R // 2:]

    def rotate(y):
        if c["pairs"] == "half":
            a, b = y[..., :R // 2], y[..., R // 2:R]
            return torch.cat([a * cos - b * sin, b * cos + a * sin, y[..., R:]], -1)
        a, b = y[..., 0:R:2], y[..., 1:R:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        return torch.cat([turned, y[..., R:]], -1)

    dt = s["k"].dtype
    t_seq, t_i = _rows(s)
    start = s["q_start"].long()
    slot = s["kv_len"].long()[t_seq] - (start[1:] - start[:-1])[t_seq] + t_i
    pg, row = _slots(s, t_seq, slot)
    s["k"][pg, :, row] = rotate(norm(x[:, qh:qh + KVH], s["k_norm"])).to(dt)
    s["v"][pg, :, row] = x[:, qh + KVH:].to(dt)
    s["q"].copy_(rotate(norm(q, s["q_norm"])))
    return {"q": s["q"], "k": s["k"], "v": s["v"]}


def _plain_scores(s):
    """Masked scores [B, KVH, G, Q, L] of padded batches, and the live slots [B, 1, L, 1]."""
    c = s["case"]
    B, H, KVH, D, Q, L = c["batch"], c["H"], c["KVH"], c["D"], s["max_q"], s["max_kv"]
    start, kv = s["q_start"].long(), s["kv_len"].long()
    n = start[1:] - start[:-1]
    i, j = torch.arange(Q, device="cuda"), torch.arange(L, device="cuda")
    qp = s["q"][(start[:-1, None] + i).clamp(max=s["tokens"] - 1)].float()  # [B, Q, H, D]
    qp = qp.view(B, Q, KVH, H // KVH, D).permute(0, 2, 3, 1, 4).reshape(B, KVH, (H // KVH) * Q, D)
    k = _gather(s, "k")
    scores = (qp @ k.transpose(-1, -2)).view(B, KVH, H // KVH, Q, L) * (1 / math.sqrt(D))
    sees = (j <= (kv - n)[:, None, None] + i[:, None]) & (i < n[:, None])[..., None]  # [B, Q, L]
    return scores.masked_fill_(~sees[:, None, None], float("-inf"))


def _gather(s, name):
    """Live rows of the cache in order, 32 bits [B, KVH, L, D]; zeros past each length."""
    L = s["max_kv"]
    x = s[name][s["table"].long()].permute(0, 2, 1, 3, 4).flatten(2, 3)[:, :, :L].float()
    live = torch.arange(L, device="cuda") < s["kv_len"][:, None]
    return x.masked_fill_(~live[:, None, :, None], 0)


def _plain_attention(s):
    c = s["case"]
    e = _plain_scores(s)
    m = e.amax(-1, keepdim=True)
    m = torch.where(torch.isinf(m), torch.zeros_like(m), m)
    e = e.sub_(m).exp_()
    total = e.sum(-1, keepdim=True)
    o = e.flatten(2, 3) @ _gather(s, "v")  # [B, KVH, G Q, D]
    o = o.view(*e.shape[:-1], c["D"]) / torch.where(total > 0, total, torch.ones_like(total))
    lse = (m + total.log())[..., 0]
    t_seq, t_i = _rows(s)
    o = o.permute(0, 3, 1, 2, 4)[t_seq, t_i].flatten(1, 2)
    return o, lse.permute(0, 3, 1, 2)[t_seq, t_i].flatten(1, 2).contiguous()


def _plain_weights(s):
    c = s["case"]
    B, KVH, Q = c["batch"], c["KVH"], s["max_q"]
    e = _plain_scores(s)
    at = (s["q_start"].long()[:-1, None] + torch.arange(Q, device="cuda")).clamp(max=s["tokens"] - 1)
    lse = s["lse"][at].view(B, Q, KVH, -1).permute(0, 2, 3, 1)[..., None]
    s["acc"][:, :, :s["max_kv"]] += e.sub_(lse).exp_().sum((2, 3))
    return s["acc"]


def _plain_evict(s):
    c = s["case"]
    B, KVH, cap = s["acc"].shape
    j = torch.arange(cap, device="cuda")
    inf = torch.full_like(s["acc"], float("inf"))
    kept_always = (s["pos"] < c["sink"]) | (s["pos"] >= s["protect_from"][:, None, None])
    live = j < s["kv_len"][:, None, None]
    key = torch.where(kept_always, inf, torch.where(torch.isnan(s["acc"]), -inf, s["acc"]))
    key = torch.where(live, key, -inf)
    order = key.sort(dim=-1, descending=True, stable=True).indices
    rank = torch.empty_like(order).scatter_(-1, order, j.expand_as(order))
    new_len = torch.minimum(s["kv_len"], s["keep"])
    nl = new_len[:, None, None]
    kept = rank < nl
    hole, source = ~kept & (j < nl), kept & (j >= nl)
    sources = torch.where(source, j, cap).sort(-1).values
    nth = (hole.cumsum(-1) - 1).clamp(min=0)
    came = torch.where(hole, sources.gather(-1, nth), j.expand_as(nth)).clamp(max=cap - 1)  # slot that each slot now holds
    s["acc_out"].copy_(torch.where(j < nl, s["acc"].gather(-1, came), s["acc_out"]))
    s["pos_out"].copy_(torch.where(j < nl, s["pos"].gather(-1, came), s["pos_out"]))
    s["len_out"].copy_(new_len)
    b, h, to = hole.nonzero(as_tuple=True)
    p0, r0 = _slots(s, b, came[b, h, to])
    p1, r1 = _slots(s, b, to)
    s["k"][p1, h, r1] = s["k"][p0, h, r0]
    s["v"][p1, h, r1] = s["v"][p0, h, r0]
    return {"k": s["k"], "v": s["v"], "acc": s["acc_out"], "pos": s["pos_out"], "len": s["len_out"]}


# ---------------------------------------------------------------------------


def work(case):
    c = case
    n, kv = _lens(c)
    T, H, KVH, D = sum(n), c["H"], c["KVH"], c["D"]
    live = sum(x for m, x in zip(n, kv) if m)  # slots that a pass reads
    seen = sum(m * (x - m) + m * (m + 1) // 2 for m, x in zip(n, kv))  # (new token, slot) pairs
    if c["op"] == "rope":
        return {"bytes": T * ((H + 2 * KVH) * D * 6 + c["rot"] * 4), "flops": T * (H + KVH) * D * 7}
    if c["op"] == "attn":
        return {"bytes": 2 * T * H * D * 2 + T * H * 4 + 2 * live * KVH * D * 2 + (T * H * D * 4 if c["gated"] else 0),
                "flops": 4 * D * H * seen}
    if c["op"] == "weights":
        return {"bytes": T * H * (D * 2 + 4) + live * KVH * (D * 2 + 8), "flops": 2 * D * H * seen}
    total = 0
    for x in kv:
        keep = min(x, c["keep"])
        moved = keep * (x - keep) / x  # kept slots that lie past the new length, when weights do not go by slot
        total += KVH * (x * 8 + keep * 8 + moved * 2 * D * 2 * 2)
    return {"bytes": total, "flops": 0}


def exact(case, seed):
    """From the definitions in 64 bits, one sequence at a time."""
    s = prepare(case, seed)
    c = s["case"]
    n, kv = _lens(c)
    H, KVH, D, page = c["H"], c["KVH"], c["D"], c["page"]
    G = H // KVH
    f64 = torch.float64

    def rows(name, b):
        """Slots 0 .. kv[b] of a sequence, [KVH, kv[b], D]."""
        ids = s["table"][b, :-(-kv[b] // page)].long()
        return s[name][ids].transpose(0, 1).reshape(KVH, -1, D)[:, :kv[b]].to(f64)

    first = [sum(n[:b]) for b in range(len(n))]
    if c["op"] == "rope":
        x = s["qkv"].to(f64)
        T, R = x.shape[0], c["rot"]
        step = 2 if c["gated"] else 1
        cs = s["rope"].to(f64)
        k_new, v_new = s["k"].to(f64), s["v"].to(f64)
        turn = torch.polar(torch.ones(cs.shape[0], R // 2, dtype=f64, device="cuda"),
                           torch.zeros(cs.shape[0], R // 2, dtype=f64, device="cuda"))
        turn = torch.complex(cs[:, :R // 2], cs[:, R // 2:]) * turn  # rotation as a complex product

        def head(at, w):
            y = x[:, at * D:(at + 1) * D]
            y = y / (y.pow(2).sum(1, keepdim=True) / D + 1e-6).sqrt() * w.to(f64)
            ia = torch.arange(R // 2, device="cuda") * (1 if c["pairs"] == "half" else 2)
            ib = ia + (R // 2 if c["pairs"] == "half" else 1)
            z = torch.complex(y[:, ia], y[:, ib]) * turn[s["pos"].long()]
            y = y.clone()
            y[:, ia], y[:, ib] = z.real, z.imag
            return y

        q = torch.stack([head(h * step, s["q_norm"]) for h in range(H)], 1)
        k = torch.stack([head(H * step + h, s["k_norm"]) for h in range(KVH)], 1)
        v = x[:, (H * step + KVH) * D:].view(T, KVH, D)
        for b in range(len(n)):
            slot = torch.arange(kv[b] - n[b], kv[b], device="cuda")
            ids = s["table"][b].long()[slot // page]
            k_new[ids, :, slot % page] = k[first[b]:first[b] + n[b]]
            v_new[ids, :, slot % page] = v[first[b]:first[b] + n[b]]
        return {"q": q, "k": k_new, "v": v_new}
    if c["op"] in ("attn", "weights"):
        o = torch.zeros((s["tokens"], H, D), dtype=f64, device="cuda")
        lse = torch.zeros((s["tokens"], H), dtype=f64, device="cuda")
        acc = s["acc"].to(f64) if c["op"] == "weights" else None
        for b in range(len(n)):
            if not n[b]:
                continue
            k, v = rows("k", b), rows("v", b)
            at = slice(first[b], first[b] + n[b])
            sees = torch.ones(n[b], kv[b], dtype=torch.bool, device="cuda").tril(kv[b] - n[b])
            for h in range(H):
                z = (s["q"][at, h].to(f64) @ k[h // G].T / D ** 0.5).masked_fill(~sees, -torch.inf)
                if c["op"] == "weights":
                    acc[b, h // G, :kv[b]] += (z - s["lse"][at, h, None].to(f64)).exp().sum(0)
                else:
                    lse[at, h] = z.logsumexp(1)
                    o[at, h] = z.softmax(1) @ v[h // G]
        if c["op"] == "weights":
            return {"acc": acc}
        if s["gate"] is not None:
            o = o * torch.sigmoid(s["gate"].to(f64))
        return {"o": o, "lse": lse}
    # eviction moves values: the kept set of one head at a time, on the host
    if sum(kv) * KVH > 2000000:
        return None
    k, v = s["k"].to(f64), s["v"].to(f64)
    acc_out, pos_out = torch.zeros_like(s["acc"], dtype=f64), torch.zeros_like(s["pos"])
    ids = s["table"].cpu()
    for b, L in enumerate(kv):
        new = min(L, c["keep"])
        low = s["protect_from"][b].item()
        for h in range(KVH):
            a, p = s["acc"][b, h, :L].cpu().tolist(), s["pos"][b, h, :L].cpu().tolist()
            w = [math.inf if x < c["sink"] or x >= low else y for x, y in zip(p, a)]
            kept = set(sorted(range(L), key=lambda i: (-w[i], i))[:new])
            came = list(range(new))
            late = sorted(i for i in kept if i >= new)
            gone = [i for i in range(new) if i not in kept]
            for i, m in zip(gone, late):
                came[i] = m
            acc_out[b, h, :new] = torch.tensor([a[i] for i in came], dtype=f64)
            pos_out[b, h, :new] = torch.tensor([p[i] for i in came], dtype=torch.int32)
            if gone:
                gone, late = torch.tensor(gone), torch.tensor(late)
                pg, pl = ids[b, gone // page].long().cuda(), ids[b, late // page].long().cuda()
                k[pg, h, (gone % page).cuda()] = k[pl, h, (late % page).cuda()]
                v[pg, h, (gone % page).cuda()] = v[pl, h, (late % page).cuda()]
    return {"k": k, "v": v, "acc": acc_out, "pos": pos_out,
            "len": torch.tensor([min(x, c["keep"]) for x in kv], dtype=torch.int32)}
