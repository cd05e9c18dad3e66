"""The engine's operator surface on torch CUDA tensors, over the C ABI.

Mirrors crates/engine/src/graph.rs: Builder::gemv (:190-198), Builder::gemm
(:200-205), Builder::matmul (:207-214), Builder::quant (:216-222) and the argmax op
of head_ops (:478-486), plus the fused lm_head argmax.  Every call launches on
torch's current CUDA stream and returns without synchronizing; arguments are
checked by the library (W4A8Error with status EINVAL before any launch).
"""

import ctypes
import math

import torch

from . import _lib
from ._lib import ACT_GROUP32, ACT_TOKEN, ADD, GEMV_MAX_M, STORE, SWIGLU  # noqa: F401


def _ptr(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def _stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def _need_cuda(*ts):
    for t in ts:
        if t is not None and (not t.is_cuda or not t.is_contiguous()):
            raise ValueError("webyiq_b200 ops take contiguous CUDA tensors")


class QWeight:
    """A quantized linear weight in device memory, in the reference's layout.

    q: int32/uint32 tensor [n, k/8] (the u32 words of `{w}.q`);
    s: has_min -> int32/uint32 [n, k/group] (`{w}.s`: f16 scale | f16 min << 16),
       else float16/int16 [n, k/group] (scale only, w = (q-8)*scale).
    """

    def __init__(self, q, s, n, k, group, has_min):
        _need_cuda(q, s)
        self.q, self.s = q, s
        self.n, self.k, self.group, self.has_min = int(n), int(k), int(group), int(bool(has_min))
        self.c = _lib.Weight()
        _lib.check(_lib.load().w4a8_weight_view(_ptr(q), _ptr(s), self.n, self.k, self.group, self.has_min,
                                                ctypes.byref(self.c)))

    def __repr__(self):
        return f"QWeight(n={self.n}, k={self.k}, group={self.group}, has_min={self.has_min})"


def xs_shape(m, k, act):
    return (m,) if act == ACT_TOKEN else (m, k // 32, 2)


def quant(x, norm_w=None, eps=1e-6, act=ACT_GROUP32, xq=None, xs=None):
    """int8 activation quantization of the rows of x f32 [m, k], optionally
    RMSNorm'ed with norm_w (quant.wgsl).  Returns (xq int8 [m, k], xs f32)."""
    _need_cuda(x, norm_w)
    m, k = x.shape
    if xq is None:
        xq = torch.empty((m, k), dtype=torch.int8, device=x.device)
    if xs is None:
        xs = torch.empty(xs_shape(m, k, act), dtype=torch.float32, device=x.device)
    _lib.check(_lib.load().w4a8_quant(_ptr(x), _ptr(norm_w), float(eps), m, k, act, _ptr(xq), _ptr(xs), _stream()))
    return xq, xs


def _out(w, m, mode, y, device):
    n_out = w.n // 2 if mode == SWIGLU else w.n
    if y is None:
        if mode == ADD:
            raise ValueError("mode ADD needs y")
        y = torch.empty((m, n_out), dtype=torch.float32, device=device)
    return y


def gemv(w, xq, xs, act=ACT_GROUP32, mode=STORE, y=None):
    """y (+)= W x for m <= 16 tokens (gemv_q4q8.wgsl)."""
    _need_cuda(xq, xs, y)
    m = xq.shape[0]
    y = _out(w, m, mode, y, xq.device)
    _lib.check(_lib.load().w4a8_gemv(ctypes.byref(w.c), _ptr(xq), _ptr(xs), act, m, mode, _ptr(y), _stream()))
    return y


def gemv_x(w, x, mode=STORE, y=None):
    """Per-token quant of f32 x [m, k] and the GEMV in one launch (group-128 weights);
    equal to quant(act=ACT_TOKEN) followed by gemv, bit for bit."""
    _need_cuda(x, y)
    m = x.shape[0]
    y = _out(w, m, mode, y, x.device)
    _lib.check(_lib.load().w4a8_gemv_x(ctypes.byref(w.c), _ptr(x), m, mode, _ptr(y), _stream()))
    return y


def gemv_xn(w, x, norm_w, eps, mode=STORE, y=None):
    """RMSNorm (norm_w f32 [k], eps), per-token quant and the GEMV in one launch, for
    one or two tokens; equal to quant(x, norm_w, eps, act=ACT_TOKEN) followed by gemv,
    bit for bit."""
    _need_cuda(x, norm_w, y)
    m = x.shape[0]
    y = _out(w, m, mode, y, x.device)
    _lib.check(_lib.load().w4a8_gemv_xn(ctypes.byref(w.c), _ptr(x), _ptr(norm_w), float(eps), m, mode, _ptr(y),
                                        _stream()))
    return y


def gemm(w, xq, xs, act=ACT_GROUP32, mode=STORE, y=None):
    """Y (+)= X W^T for any m (gemm_q4q8.wgsl)."""
    _need_cuda(xq, xs, y)
    m = xq.shape[0]
    y = _out(w, m, mode, y, xq.device)
    _lib.check(_lib.load().w4a8_gemm(ctypes.byref(w.c), _ptr(xq), _ptr(xs), act, m, mode, _ptr(y), _stream()))
    return y


def matmul(w, xq, xs, act=ACT_GROUP32, mode=STORE, y=None):
    """GEMV for m <= 16 tokens, GEMM above (Builder::matmul)."""
    _need_cuda(xq, xs, y)
    m = xq.shape[0]
    y = _out(w, m, mode, y, xq.device)
    _lib.check(_lib.load().w4a8_matmul(ctypes.byref(w.c), _ptr(xq), _ptr(xs), act, m, mode, _ptr(y), _stream()))
    return y


def argmax(logits, ids=None, out=None):
    """Greedy token of every row of logits f32 [m, v] (argmax.wgsl)."""
    _need_cuda(logits, ids, out)
    m, v = logits.shape
    if out is None:
        out = torch.empty(m, dtype=torch.int32, device=logits.device)
    _lib.check(_lib.load().w4a8_argmax(_ptr(logits), m, v, _ptr(ids), _ptr(out), _stream()))
    return out


def group_dots(w, xq):
    """Exact int32 dot of every (token, row, group): int32 [m, n, k/group]."""
    _need_cuda(xq)
    m = xq.shape[0]
    dots = torch.empty((m, w.n, w.k // w.group), dtype=torch.int32, device=xq.device)
    _lib.check(_lib.load().w4a8_group_dots(ctypes.byref(w.c), _ptr(xq), m, _ptr(dots), _stream()))
    return dots


def gemm_group_dots(w, xq):
    """The tcgen05 GEMM's int32 group dots (read back from tensor memory): int32 [m, n, k/128]."""
    _need_cuda(xq)
    m = xq.shape[0]
    dots = torch.empty((m, w.n, w.k // w.group), dtype=torch.int32, device=xq.device)
    _lib.check(_lib.load().w4a8_gemm_group_dots(ctypes.byref(w.c), _ptr(xq), m, _ptr(dots), _stream()))
    return dots


def lmhead_workspace(w, m, device):
    nbytes = _lib.load().w4a8_lmhead_workspace_bytes(w.n, m)
    return torch.zeros(nbytes, dtype=torch.uint8, device=device)


def lmhead_argmax(w, xq, xs, act=ACT_TOKEN, row_offset=0, logits=None, ids=None, workspace=None,
                  best_key=None, tok=None):
    """lm_head GEMV with fused argmax.  Returns (best_key int64 [m] (u64 bits), tok int32 [m])."""
    _need_cuda(xq, xs, logits, ids, workspace)
    m = xq.shape[0]
    dev = xq.device
    if workspace is None:
        workspace = lmhead_workspace(w, m, dev)
    if best_key is None:
        best_key = torch.empty(m, dtype=torch.int64, device=dev)
    if tok is None:
        tok = torch.empty(m, dtype=torch.int32, device=dev)
    _lib.check(_lib.load().w4a8_lmhead_argmax(ctypes.byref(w.c), int(row_offset), _ptr(xq), _ptr(xs), act, m,
                                              _ptr(logits), _ptr(best_key), _ptr(tok), _ptr(ids), _ptr(workspace),
                                              workspace.numel(), _stream()))
    return best_key, tok


def lmhead_argmax_noalloc(w, xq, xs, act=ACT_TOKEN, row_offset=0, logits=None, ids=None, best_key=None, tok=None):
    """lm_head GEMV with fused argmax, using the library's own scratch (no workspace,
    no device allocation; m <= 16).  Returns (best_key int64 [m], tok int32 [m])."""
    _need_cuda(xq, xs, logits, ids)
    m = xq.shape[0]
    dev = xq.device
    if best_key is None:
        best_key = torch.empty(m, dtype=torch.int64, device=dev)
    if tok is None:
        tok = torch.empty(m, dtype=torch.int32, device=dev)
    _lib.check(_lib.load().w4a8_lmhead_argmax_noalloc(ctypes.byref(w.c), int(row_offset), _ptr(xq), _ptr(xs), act, m,
                                                      _ptr(logits), _ptr(best_key), _ptr(tok), _ptr(ids), _stream()))
    return best_key, tok


# ---------------------------------------------------------------------------
# Column-split lm_head over GPUs (vocabulary rows sharded; one exchange of keys).

_SIGN = -(2 ** 63)


def merge_shard_keys(keys, group=None):
    """All-reduce (max) of packed argmax keys (int64 tensor holding u64 bits) over a
    torch.distributed group, in place.  Keys compare as unsigned integers; flipping
    the top bit makes the signed max agree, so any backend (NCCL, gloo) works."""
    import torch.distributed as dist

    keys ^= _SIGN
    dist.all_reduce(keys, op=dist.ReduceOp.MAX, group=group)
    keys ^= _SIGN
    return keys


def keys_to_tokens(keys, ids=None):
    """Token of every packed key (int64 u64 bits) on the keys' device: the index
    (~low word, 0 for the key 0), mapped through ids (int32 [vocab]) if given."""
    low = keys & 0xFFFFFFFF
    idx = torch.where(keys != 0, 0xFFFFFFFF - low, torch.zeros_like(low))
    if ids is not None:
        return ids.to(torch.int64)[idx].to(torch.int32)
    return idx.to(torch.int32)


def lmhead_argmax_sharded(w, xq, xs, row_offset, act=ACT_TOKEN, group=None, ids=None, workspace=None, logits=None):
    """This rank's vocabulary shard (global rows row_offset .. + w.n) through the
    fused lm_head argmax, then the keys merged over the torch.distributed group.
    Returns (best_key int64 [m], tok int32 [m]) of the global argmax on every rank."""
    best_key, _ = lmhead_argmax(w, xq, xs, act=act, row_offset=row_offset, logits=logits, workspace=workspace)
    merge_shard_keys(best_key, group)
    return best_key, keys_to_tokens(best_key, ids)


def gather_rows(w, ids):
    """The draft lm_head of an MTP step: rows ids (int32/uint32 [rows] on the device)
    of w's packed weights and scales, as a new QWeight (gather_rows.wgsl)."""
    _need_cuda(ids)
    rows = ids.numel()
    q = torch.empty((rows, w.k // 8), dtype=torch.int32, device=ids.device)
    sdt = torch.int32 if w.has_min else torch.int16
    s = torch.empty((rows, w.k // w.group), dtype=sdt, device=ids.device)
    _lib.check(_lib.load().w4a8_gather_rows(ctypes.byref(w.c), _ptr(ids), rows, _ptr(q), _ptr(s), _stream()))
    return QWeight(q, s, rows, w.k, w.group, w.has_min)


def spec_accept(tok, y, e, params, ctl, out=None):
    """End of a speculative step (spec_accept.wgsl), all int32 device tensors: tok [2]
    (rewritten), y [2], e [2], params [4] -> ctl [4] (may be params), out [5] or None."""
    _need_cuda(tok, y, e, params, ctl, out)
    _lib.check(_lib.load().w4a8_spec_accept(_ptr(tok), _ptr(y), _ptr(e), _ptr(params), _ptr(ctl), _ptr(out),
                                            _stream()))
    return tok, ctl, out


ATTN_CHUNK = 32


def attn_decode(qkv, kc, vc, H, KVH, D, params, m, chunks=None, part=None):
    """Flash-decoding partials (attn.wgsl): qkv f32 [m, (H + 2 KVH) D], kc / vc f16
    [KVH, maxctx, D], params int32 [4] on the device (pos first).  Returns part f32
    [m, H, maxctx / 32, D + 2]; chunks defaults to all of them."""
    _need_cuda(qkv, kc, vc, params, part)
    maxctx = kc.shape[1]
    nch = maxctx // ATTN_CHUNK
    if part is None:
        part = torch.empty((m, H, nch, D + 2), dtype=torch.float32, device=qkv.device)
    _lib.check(_lib.load().w4a8_attn_decode(_ptr(qkv), _ptr(kc), _ptr(vc), H, KVH, D, maxctx, _ptr(params), m,
                                            nch if chunks is None else chunks, _ptr(part), _stream()))
    return part


def attn_combine(part, H, KVH, D, maxctx, params, m, gsrc=None, want_o=False):
    """The chunks merged per head (attn_combine.wgsl), times sigmoid(gate) with gsrc,
    quantized per 32: -> (xq int8 [m, H D], xs f32 [m, H D / 32, 2], o f32 [m, H, D] or None)."""
    _need_cuda(part, params, gsrc)
    xq = torch.empty((m, H * D), dtype=torch.int8, device=part.device)
    xs = torch.empty((m, H * D // 32, 2), dtype=torch.float32, device=part.device)
    o = torch.empty((m, H, D), dtype=torch.float32, device=part.device) if want_o else None
    _lib.check(_lib.load().w4a8_attn_combine(_ptr(part), H, KVH, D, maxctx, _ptr(params), m, _ptr(gsrc), _ptr(xq),
                                             _ptr(xs), _ptr(o), _stream()))
    return xq, xs, o


def deltanet(proj, conv_w, conv_state, state, neg_a, dt_bias, gate_norm, params, nh, m, eps=1e-6, spec=False,
             out=None):
    """Gated DeltaNet mixer (deltanet.wgsl) on device f32 tensors; conv_state and state
    (three slots each) are updated in place.  Returns out f32 [m, nh * 128]."""
    _need_cuda(proj, conv_w, conv_state, state, neg_a, dt_bias, gate_norm, params, out)
    if out is None:
        out = torch.empty((m, nh * 128), dtype=torch.float32, device=proj.device)
    _lib.check(_lib.load().w4a8_deltanet(_ptr(proj), _ptr(conv_w), _ptr(conv_state), _ptr(state), _ptr(out),
                                         _ptr(neg_a), _ptr(dt_bias), _ptr(gate_norm), _ptr(params), nh, m, eps,
                                         1 if spec else 0, _stream()))
    return out


# ---------------------------------------------------------------------------
# A batch of sequences over a paged KV cache (w4a8.h: the paged operators).

_TYPES = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16, torch.float32: _lib.F32}


class _Fixed:
    """Attributes that hold for the object's life, but those of `free`, which every call reads anew."""

    free = ()

    def __setattr__(self, name, value):
        if name not in self.free:
            raise AttributeError(f"{type(self).__name__}.{name} is fixed: make a new {type(self).__name__}")
        self.__dict__[name] = value


class PagedKV(_Fixed):
    """A paged KV cache in device memory: k, v [pages, KVH, page, D], f16 or bf16, of the
    same strides.  Any order of the dimensions in memory does (a cache stored [pages, page,
    KVH, D] comes in as its permute(0, 2, 1, 3)); the inner stride is 1.  It holds the tensors'
    addresses: writing to them is fine, a tensor resized or set to other memory is refused."""

    free = ("scale",)

    def __init__(self, k, v):
        if not (k.is_cuda and v.is_cuda) or k.device != v.device:
            raise ValueError("PagedKV takes two tensors of one CUDA device")
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype or k.dtype not in (torch.float16, torch.bfloat16):
            raise ValueError("PagedKV takes k and v [pages, KVH, page, D] of one type, float16 or bfloat16")
        # (a dimension of one has no stride)
        strides, of_v = ([s if n > 1 else 0 for n, s in zip(k.shape[:3], x.stride())] for x in (k, v))
        if strides != of_v or k.stride(3) != 1 or v.stride(3) != 1:
            raise ValueError("PagedKV takes k and v of the same strides, with inner stride 1")
        if (strides[1] | strides[2]) >> 31:
            raise ValueError("PagedKV takes strides of heads and slots below 2^31 elements")
        pages, KVH, page, D = k.shape
        layout = (_TYPES[k.dtype], pages, page, *strides)
        # the library's arguments, converted once: a call of some thirty spends 3 us on that
        sizes = [ty(x) for ty, x in zip((ctypes.c_int32,) * 3 + (ctypes.c_size_t,) + (ctypes.c_int32,) * 2, layout)]
        pk, pv = _ptr(k), _ptr(v)
        self.__dict__.update(
            k=k, v=v, pages=pages, KVH=KVH, page=page, D=D, dtype=k.dtype, device=k.device, index=k.get_device(),
            scale=1.0 / math.sqrt(D),  # of the scores, where a call gives none
            layout=layout, c=(pk, pv, *sizes), c_k=(pk, *sizes), at=(k.data_ptr(), v.data_ptr()),
            now=(k.data_ptr, v.data_ptr))

    def __repr__(self):
        return f"PagedKV(pages={self.pages}, KVH={self.KVH}, page={self.page}, D={self.D}, {self.dtype})"


class PagedBatch(_Fixed):
    """A step's batch over a PagedKV: q_start int32 [B + 1] (first new token of each sequence,
    from 0), kv_len int32 [B] (slots, the new tokens' own among them), table int32 [B, pages a
    sequence]; sequences may share pages that a call only reads (kv_evict writes to all of its
    sequences' pages, qk_norm_rope_kv to those of the new slots).  max_q and max_kv bound the new tokens and the slots of any sequence (read on
    the device otherwise, so the arrays may be rewritten in place between calls); the two may
    be assigned anew.  Holds the arrays' addresses, as PagedKV does."""

    free = ("max_q", "max_kv")

    def __setattr__(self, name, value):
        super().__setattr__(name, self._bound(value) if name in self.free else value)

    @staticmethod
    def _bound(value):
        value = int(value)
        if value >> 31:
            raise ValueError(f"PagedBatch: a bound of {value}, not in 0 .. 2^31 - 1")
        return value

    def __init__(self, q_start, kv_len, table, max_q, max_kv):
        _need_cuda(q_start, kv_len, table)
        index, B = q_start.get_device(), kv_len.numel()
        if kv_len.get_device() != index or table.get_device() != index:
            raise ValueError("PagedBatch takes tensors of one device")
        if q_start.dtype != torch.int32 or kv_len.dtype != torch.int32 or table.dtype != torch.int32:
            raise ValueError("PagedBatch takes int32 tensors")
        if q_start.numel() != B + 1 or table.dim() != 2 or table.shape[0] != B:
            raise ValueError("PagedBatch takes q_start [B + 1], kv_len [B] and table [B, pages a sequence]")
        if table.shape[1] >> 31:
            raise ValueError("PagedBatch takes fewer than 2^31 pages a sequence")
        c = (_ptr(q_start), _ptr(kv_len), _ptr(table), ctypes.c_int32(B), ctypes.c_int32(table.shape[1]))
        self.__dict__.update(
            q_start=q_start, kv_len=kv_len, table=table, max_q=self._bound(max_q), max_kv=self._bound(max_kv), B=B,
            per=table.shape[1], index=index, c=c, c_slots=c[1:],
            at=(q_start.data_ptr(), kv_len.data_ptr(), table.data_ptr()),
            now=(q_start.data_ptr, kv_len.data_ptr, table.data_ptr))


# The paged operators are called once a layer and token, so their wrappers keep to cheap
# checks: each attribute of a tensor costs about a tenth of a microsecond.


def _raw_stream(index):
    """The current stream of a device as an integer (torch.cuda.current_stream builds an object: 3 us)."""
    return torch._C._cuda_getCurrentRawStream(index)


def _current_device():
    return torch._C._cuda_getDevice()


def _place(kv, batch):
    """Before a call: the library launches on the current device, so everything has to be there, and at the
    addresses that were taken."""
    k, v = kv.now
    q_start, kv_len, table = batch.now
    if (k(), v()) != kv.at or (q_start(), kv_len(), table()) != batch.at:
        raise ValueError("the cache's or the batch's tensors have moved since PagedKV or PagedBatch took them")
    if batch.index != kv.index:
        raise ValueError(f"a batch of cuda:{batch.index} with a cache of cuda:{kv.index}")
    if _current_device() != kv.index:
        raise ValueError(f"a cache of cuda:{kv.index}, which is not the current device")


def _is(t, dtype, index):
    return t.dtype is dtype and t.get_device() == index and t.is_contiguous()


def _opt(t, dtype, what, index):
    """Pointer of an optional contiguous tensor of a CUDA device (0 for None)."""
    if t is None:
        return 0
    if t.dtype is not dtype or t.get_device() != index or not t.is_contiguous():
        raise ValueError(f"{what}: a contiguous tensor of {dtype} on cuda:{index}")
    return t.data_ptr()


def _token_stride(name, t, kv):
    """Elements from token to token of a [tokens, heads, D] tensor of the cache's type, contiguous within a token."""
    if t.dtype is not kv.dtype or t.get_device() != kv.index or t.dim() != 3:
        raise ValueError(f"{name}: a [tokens, heads, D] tensor of {kv.dtype} on {kv.device}")
    T, H, D = t.shape
    if D != kv.D:
        raise ValueError(f"{name}: {D} dims, a cache of {kv.D}")
    s = t.stride()
    if T * H and (s[2] != 1 or (s[1] != D and H > 1)):
        raise ValueError(f"{name}: contiguous within a token")
    if T < 2:
        return H * D
    if s[0] >> 31:
        raise ValueError(f"{name}: {s[0]} elements from token to token, not below 2^31")
    return s[0]


def qk_norm_rope_kv(qkv, kv, batch, pos, rope, H, q_norm=None, k_norm=None, eps=1e-6, gated=False, interleaved=False,
                    q=None):
    """Norms of q and k per head, rotation, and append of k and v to the cache (w4a8.h).
    qkv f32 [tokens, (H + 2 KVH) D] (with gated, each query head followed by its gate: 2 H
    heads of D in their place); pos int32 [tokens]; rope f32 [rows, rot] (cosines, then
    sines) or None; q_norm, k_norm f32 [D] or None.  Returns q [tokens, H, D] of the
    cache's type."""
    _place(kv, batch)
    at = kv.index
    if qkv.dtype is not torch.float32 or qkv.get_device() != at or qkv.dim() != 2:
        raise ValueError(f"qk_norm_rope_kv: qkv f32 [tokens, heads * D] on {kv.device}")
    T, width = qkv.shape
    D = kv.D
    qhs = 2 * D if gated else D
    row, inner = qkv.stride()
    if width != H * qhs + 2 * kv.KVH * D or (inner != 1 and T):
        raise ValueError(f"qk_norm_rope_kv: rows of {width} for {H} query and {kv.KVH} kv heads of {D}, inner stride 1")
    if T < 2:
        row = width
    elif row >> 31:
        raise ValueError(f"qk_norm_rope_kv: {row} elements from row to row, not below 2^31")
    pqn, pkn = _opt(q_norm, torch.float32, "q_norm", at), _opt(k_norm, torch.float32, "k_norm", at)
    if (pqn and q_norm.numel() != D) or (pkn and k_norm.numel() != D):
        raise ValueError("qk_norm_rope_kv: norm weights f32 [D]")
    rot = rows = prope = ppos = 0
    if rope is not None:
        prope, ppos = _opt(rope, torch.float32, "rope", at), _opt(pos, torch.int32, "pos", at)
        if rope.dim() != 2 or not ppos and T or ppos and pos.numel() != T:
            raise ValueError("qk_norm_rope_kv: rope f32 [rows, rot] and pos int32 [tokens]")
        rows, rot = rope.shape
    if q is None:
        q = torch.empty((T, H, D), dtype=kv.dtype, device=qkv.device)
    elif q.shape != (T, H, D) or not _is(q, kv.dtype, at):
        raise ValueError("qk_norm_rope_kv: q [tokens, H, D] of the cache's type, contiguous")
    st = _lib.load().w4a8_qk_norm_rope_kv(
        qkv.data_ptr(), row, qhs, H, kv.KVH, D, pqn, pkn, eps, prope, rot, rows, interleaved, ppos,
        *batch.c, T, q.data_ptr(), *kv.c, _raw_stream(at))
    if st:
        _lib.check(st)
    return q


def attn_paged_workspace(batch, tokens, H, KVH, D, device):
    """Workspace of attn_paged for calls of this size (uint8; any contents)."""
    n = _lib.load().w4a8_attn_paged_workspace_bytes(tokens, H, KVH, D, batch.B, batch.max_q, batch.max_kv)
    return torch.empty(n, dtype=torch.uint8, device=device)


def attn_paged(q, kv, batch, scale=None, gate=None, o=None, lse=None, workspace=None):
    """Attention of the new tokens over the cache (w4a8.h): q [tokens, H, D] of the cache's
    type -> (o [tokens, H, D], lse f32 [tokens, H]); o of the cache's type, or f32 where
    an f32 o is given; gate f32 [tokens, H, D] (any token and head stride): o times
    sigmoid(gate).  scale defaults to 1 / sqrt(D)."""
    _place(kv, batch)
    at = kv.index
    row = _token_stride("attn_paged: q", q, kv)
    T, H, D = q.shape
    if o is None:
        o = torch.empty((T, H, D), dtype=kv.dtype, device=kv.device)
    elif o.shape != q.shape or not (o.get_device() == at and o.is_contiguous()):
        raise ValueError("attn_paged: o [tokens, H, D], contiguous")
    if lse is None:
        lse = torch.empty((T, H), dtype=torch.float32, device=kv.device)
    elif lse.numel() != T * H or not _is(lse, torch.float32, at):
        raise ValueError("attn_paged: lse f32 [tokens, H], contiguous")
    pg = gr = gh = 0
    if gate is not None:
        gs = gate.stride()
        if gate.dtype is not torch.float32 or gate.shape != q.shape or gate.get_device() != at or gs[2] != 1:
            raise ValueError("attn_paged: gate f32 [tokens, H, D] with inner stride 1")
        pg, gr, gh = gate.data_ptr(), gs[0] if T > 1 else 0, gs[1] if H > 1 else 0
        if (gr | gh) >> 31:
            raise ValueError("attn_paged: gate strides not below 2^31 elements")
    if workspace is None:
        workspace = attn_paged_workspace(batch, T, H, kv.KVH, D, kv.device)
    elif not _is(workspace, torch.uint8, at):
        raise ValueError("attn_paged: workspace uint8")
    st = _lib.load().w4a8_attn_paged(
        q.data_ptr(), row, H, kv.KVH, D, kv.scale if scale is None else scale, pg, gr, gh, *batch.c, T,
        batch.max_q, batch.max_kv, *kv.c, o.data_ptr(), _TYPES.get(o.dtype, -1),
        lse.data_ptr(), workspace.data_ptr(), workspace.numel(), _raw_stream(at))
    if st:
        _lib.check(st)
    return o, lse


def attn_weights_workspace(batch, H, KVH, device):
    """Workspace of attn_weights for calls of this size (uint8; any contents), or None where none is needed."""
    n = _lib.load().w4a8_attn_weights_workspace_bytes(H, KVH, batch.max_q)
    return torch.empty(n, dtype=torch.uint8, device=device) if n else None


def attn_weights(q, lse, kv, batch, acc, scale=None, workspace=None):
    """acc f32 [B, KVH, slots] += the attention weight each slot received from the new
    tokens (w4a8.h), with attn_paged's q, lse and scale.  Returns acc."""
    _place(kv, batch)
    at = kv.index
    row = _token_stride("attn_weights: q", q, kv)
    T, H, D = q.shape
    if lse.numel() != T * H or not (_is(lse, torch.float32, at) or not T):
        raise ValueError("attn_weights: lse f32 [tokens, H], contiguous")
    if acc.dim() != 3 or acc.shape[0] != batch.B or acc.shape[1] != kv.KVH or not _is(acc, torch.float32, at):
        raise ValueError("attn_weights: acc f32 [B, KVH, slots], contiguous")
    if acc.shape[2] >> 31:
        raise ValueError("attn_weights: fewer than 2^31 weights a head")
    if workspace is None:
        workspace = attn_weights_workspace(batch, H, kv.KVH, kv.device)
    st = _lib.load().w4a8_attn_weights(
        q.data_ptr(), row, lse.data_ptr(), H, kv.KVH, D, kv.scale if scale is None else scale, *batch.c, T,
        batch.max_q, batch.max_kv, *kv.c_k, acc.data_ptr(), acc.shape[2],
        _opt(workspace, torch.uint8, "workspace", at), 0 if workspace is None else workspace.numel(), _raw_stream(at))
    if st:
        _lib.check(st)
    return acc


def kv_evict_workspace(batch, KVH, device, slots=None):
    """Workspace of kv_evict (uint8; any contents) for acc and pos of `slots` entries a head;
    where not given, enough for batch.max_kv slots rounded up to whole pages."""
    n = _lib.load().w4a8_kv_evict_workspace_bytes(batch.B, KVH, batch.max_kv + 1024 if slots is None else slots)
    return torch.empty(n, dtype=torch.uint8, device=device)


def kv_evict(kv, batch, acc, pos, keep, protect_from, sink=0, acc_out=None, pos_out=None, len_out=None, workspace=None):
    """Eviction by accumulated weight (w4a8.h): of each sequence's slots keep[b] (int32) stay,
    in place in the cache; acc f32 and pos int32 [B, KVH, slots].  protect_from int32 [B]: the slots
    of positions from there on are protected (all where it is 0 or less).  Returns (acc_out, pos_out,
    len_out): acc_out and pos_out default to acc and pos themselves, len_out to a new tensor
    (it may not be batch.kv_len)."""
    _place(kv, batch)
    shape, at = acc.shape, kv.index
    if len(shape) != 3 or shape[0] != batch.B or shape[1] != kv.KVH:
        raise ValueError("kv_evict: acc f32 and pos int32 [B, KVH, slots], contiguous")
    slots = shape[2]
    if slots < batch.max_kv or slots >> 31:
        raise ValueError(f"kv_evict: {slots} weights a head for up to {batch.max_kv} slots (fewer than 2^31)")
    if acc_out is None:
        acc_out = acc
    if pos_out is None:
        pos_out = pos
    if len_out is None:
        len_out = torch.empty_like(batch.kv_len)
    for t, dtype in ((acc, torch.float32), (pos, torch.int32), (acc_out, torch.float32), (pos_out, torch.int32)):
        if t.dtype is not dtype or t.shape != shape or t.get_device() != at or not t.is_contiguous():
            raise ValueError("kv_evict: acc f32 and pos int32 [B, KVH, slots], contiguous; acc_out and pos_out as they")
    for t in (keep, protect_from, len_out):
        if t.dtype is not torch.int32 or t.numel() != batch.B or t.get_device() != at or not t.is_contiguous():
            raise ValueError("kv_evict: keep, protect_from and len_out int32 [B]")
    if workspace is None:
        workspace = kv_evict_workspace(batch, kv.KVH, kv.device, slots)
    elif not _is(workspace, torch.uint8, at):
        raise ValueError("kv_evict: workspace uint8")
    st = _lib.load().w4a8_kv_evict_signed(
        *kv.c, kv.KVH, kv.D, *batch.c_slots, acc.data_ptr(), pos.data_ptr(), slots, keep.data_ptr(), protect_from.data_ptr(),
        sink, acc_out.data_ptr(), pos_out.data_ptr(), len_out.data_ptr(), workspace.data_ptr(), workspace.numel(),
        _raw_stream(at))
    if st:
        _lib.check(st)
    return acc_out, pos_out, len_out


XCHG_HANDLE_BYTES = 64


class PeerExchange:
    """Peer-memory exchange buffers for w4a8_lmhead_argmax_xchg (one process per GPU
    of one node): this rank's buffer is made on the current device and its CUDA IPC
    handle is all-gathered over the torch.distributed group, then every peer's buffer
    is opened.  Every rank of the group must construct it (collective)."""

    def __init__(self, group=None):
        import torch.distributed as dist

        self.world = dist.get_world_size(group)
        self.rank = dist.get_rank(group)
        self.ptr = ctypes.c_void_p()
        handle = ctypes.create_string_buffer(XCHG_HANDLE_BYTES)
        _lib.check(_lib.load().w4a8_xchg_create(self.world, self.rank, handle, ctypes.byref(self.ptr)))
        handles = [None] * self.world
        dist.all_gather_object(handles, bytes(handle.raw), group=group)
        allh = ctypes.create_string_buffer(b"".join(handles), XCHG_HANDLE_BYTES * self.world)
        _lib.check(_lib.load().w4a8_xchg_open(self.ptr, allh))

    def close(self):
        if self.ptr:
            _lib.check(_lib.load().w4a8_xchg_destroy(self.ptr))
            self.ptr = ctypes.c_void_p()


def lmhead_argmax_xchg(w, xq, xs, xchg, act=ACT_TOKEN, row_offset=0, logits=None, ids=None, workspace=None,
                       best_key=None, tok=None, check=False):
    """Sharded lm_head with the key exchange over peer memory (PeerExchange) instead
    of NCCL.  Returns (best_key int64 [m], tok int32 [m]) of the global argmax.

    A peer that does not join within the exchange's bounded wait leaves this rank's
    own shard key in best_key, and only the device error word records it: with
    check=True the call synchronizes the stream and raises W4A8Error (ETIMEOUT) in
    that case; otherwise call device_error() before trusting the tokens (not inside
    a stream capture)."""
    _need_cuda(xq, xs, logits, ids, workspace)
    m = xq.shape[0]
    dev = xq.device
    if workspace is None:
        workspace = lmhead_workspace(w, m, dev)
    if best_key is None:
        best_key = torch.empty(m, dtype=torch.int64, device=dev)
    if tok is None:
        tok = torch.empty(m, dtype=torch.int32, device=dev)
    _lib.check(_lib.load().w4a8_lmhead_argmax_xchg(ctypes.byref(w.c), int(row_offset), _ptr(xq), _ptr(xs), act, m,
                                                   _ptr(logits), _ptr(best_key), _ptr(tok), _ptr(ids),
                                                   _ptr(workspace), workspace.numel(), xchg.ptr, _stream()))
    if check:
        device_error()
    return best_key, tok


def nccl_unique_id():
    """128-byte NCCL unique id (make it on one rank, give it to all)."""
    buf = ctypes.create_string_buffer(128)
    _lib.check(_lib.load().w4a8_nccl_get_unique_id(buf))
    return buf.raw


class NcclComm:
    """An NCCL communicator made by the library (for w4a8_lmhead_argmax_allreduce)."""

    def __init__(self, nranks, uid, rank):
        self.ptr = ctypes.c_void_p()
        buf = ctypes.create_string_buffer(bytes(uid), 128)
        _lib.check(_lib.load().w4a8_nccl_comm_init(int(nranks), buf, int(rank), ctypes.byref(self.ptr)))

    def close(self):
        if self.ptr:
            _lib.check(_lib.load().w4a8_nccl_comm_destroy(self.ptr))
            self.ptr = ctypes.c_void_p()


def lmhead_argmax_allreduce(w, xq, xs, comm, act=ACT_TOKEN, row_offset=0, logits=None, ids=None, workspace=None,
                            best_key=None, tok=None):
    """Sharded lm_head with the key exchange inside the library (NCCL all-reduce of
    the u64 keys over `comm`).  Returns (best_key int64 [m], tok int32 [m])."""
    _need_cuda(xq, xs, logits, ids, workspace)
    m = xq.shape[0]
    dev = xq.device
    if workspace is None:
        workspace = lmhead_workspace(w, m, dev)
    if best_key is None:
        best_key = torch.empty(m, dtype=torch.int64, device=dev)
    if tok is None:
        tok = torch.empty(m, dtype=torch.int32, device=dev)
    _lib.check(_lib.load().w4a8_lmhead_argmax_allreduce(ctypes.byref(w.c), int(row_offset), _ptr(xq), _ptr(xs), act, m,
                                                        _ptr(logits), _ptr(best_key), _ptr(tok), _ptr(ids),
                                                        _ptr(workspace), workspace.numel(), comm.ptr, _stream()))
    return best_key, tok


def key_index(key):
    """Index carried by a packed argmax key (python int, u64 bits)."""
    key &= (1 << 64) - 1
    return (~key) & 0xFFFFFFFF if key else 0


def set_pdl(enable):
    _lib.load().w4a8_set_pdl(1 if enable else 0)


def device_error():
    """Synchronize the current stream and raise W4A8Error(ETIMEOUT) if a kernel's
    bounded wait gave up since the last check."""
    code = ctypes.c_uint32(0)
    _lib.check(_lib.load().w4a8_device_error(ctypes.byref(code), _stream()))
    return code.value


def selftest_wait_timeout():
    """Launch the library's wait-timeout self test (see w4a8.h); read the result
    with device_error()."""
    _lib.check(_lib.load().w4a8_selftest_wait_timeout(_stream()))


def set_gemv_kernel(tensor_core):
    """Group-128 per-token GEMVs on the tensor-core kernel (True) or dp4a (False)."""
    _lib.load().w4a8_set_gemv_kernel(1 if tensor_core else 0)


def set_gemm_kernel(tensor_core):
    """GEMMs the tcgen05 kernel covers on it (True) or on GEMV token blocks (False)."""
    _lib.load().w4a8_set_gemm_kernel(1 if tensor_core else 0)
