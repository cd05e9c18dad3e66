"""CPU: what the paged operators' Python wrappers check before they call the library, on stand-ins for
CUDA tensors (a shape, strides, a type, a device and an address) and a library that only notes its calls."""

import math

import pytest
import torch

from webyiq_b200 import ops

F16, F32, I32, U8 = torch.float16, torch.float32, torch.int32, torch.uint8


class Fake:
    next_ptr = 1 << 20

    def __init__(self, shape, dtype, device=0, stride=None, ptr=None):
        self.shape, self.dtype, self.index = tuple(shape), dtype, device
        if stride is None:
            stride = [1] * len(shape)
            for i in range(len(shape) - 2, -1, -1):
                stride[i] = stride[i + 1] * shape[i + 1]
        self.strides = tuple(stride)
        Fake.next_ptr += 1 << 20
        self.ptr = Fake.next_ptr if ptr is None else ptr

    @property
    def device(self):
        return torch.device("cpu") if self.index < 0 else torch.device("cuda", self.index)

    @property
    def is_cuda(self):
        return self.index >= 0

    def get_device(self):
        return self.index

    def dim(self):
        return len(self.shape)

    def stride(self, i=None):
        return self.strides if i is None else self.strides[i]

    def numel(self):
        return math.prod(self.shape)

    def data_ptr(self):
        return self.ptr

    def is_contiguous(self):
        want = 1
        for n, s in zip(reversed(self.shape), reversed(self.strides)):
            if n != 1 and s != want:
                return False
            want *= n
        return True


class Library:
    """Notes each call's arguments."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, tuple(getattr(a, "value", a) for a in args)))
            return 0
        return call


@pytest.fixture
def lib(monkeypatch):
    lib = Library()
    lib.current = 0
    monkeypatch.setattr(ops._lib, "load", lambda: lib)
    monkeypatch.setattr(ops, "_current_device", lambda: lib.current)
    monkeypatch.setattr(ops, "_raw_stream", lambda index: 77 + index)
    return lib


T, H, KVH, D, B, PAGES, PAGE, PER, CAP = 5, 8, 2, 64, 2, 9, 16, 4, 64
SHAPES = {"k": ((PAGES, KVH, PAGE, D), F16), "q_start": ((B + 1,), I32), "kv_len": ((B,), I32), "table": ((B, PER), I32)}
OWN = {
    "rope": {"qkv": ((T, (H + 2 * KVH) * D), F32), "pos": ((T,), I32), "rope": ((100, 32), F32), "q_norm": ((D,), F32),
             "k_norm": ((D,), F32), "q": ((T, H, D), F16)},
    "attn": {"q": ((T, H, D), F16), "gate": ((T, H, D), F32), "o": ((T, H, D), F16), "lse": ((T, H), F32),
             "workspace": ((1 << 20,), U8)},
    "weights": {"q": ((T, H, D), F16), "lse": ((T, H), F32), "acc": ((B, KVH, CAP), F32), "workspace": ((1 << 20,), U8)},
    "evict": {"acc": ((B, KVH, CAP), F32), "pos": ((B, KVH, CAP), I32), "keep": ((B,), I32), "protect_from": ((B,), I32),
              "acc_out": ((B, KVH, CAP), F32), "pos_out": ((B, KVH, CAP), I32), "len_out": ((B,), I32),
              "workspace": ((1 << 20,), U8)}}
ENTRY = {"rope": "w4a8_qk_norm_rope_kv", "attn": "w4a8_attn_paged", "weights": "w4a8_attn_weights",
         "evict": "w4a8_kv_evict_signed"}


def tensors(op, **swap):
    t = {}
    for name, (shape, dtype) in {**SHAPES, **OWN[op]}.items():
        t[name] = Fake(shape, dtype)
    t["v"] = Fake(t["k"].shape, F16)
    t.update(swap)
    return t


def call(op, t):
    kv = ops.PagedKV(t["k"], t["v"])
    batch = ops.PagedBatch(t["q_start"], t["kv_len"], t["table"], 3, CAP)
    return invoke(op, t, kv, batch)


def invoke(op, t, kv, batch):
    if op == "rope":
        return ops.qk_norm_rope_kv(t["qkv"], kv, batch, t["pos"], t["rope"], H, t["q_norm"], t["k_norm"], q=t["q"])
    if op == "attn":
        return ops.attn_paged(t["q"], kv, batch, gate=t["gate"], o=t["o"], lse=t["lse"], workspace=t["workspace"])
    if op == "weights":
        return ops.attn_weights(t["q"], t["lse"], kv, batch, t["acc"], workspace=t["workspace"])
    return ops.kv_evict(kv, batch, t["acc"], t["pos"], t["keep"], t["protect_from"], 4, t["acc_out"], t["pos_out"],
                        t["len_out"], t["workspace"])


@pytest.mark.parametrize("op", OWN)
def test_calls_on_one_device(lib, op):
    """With everything on the current device: one call of the entry point, every tensor's address in it, on that
    device's stream."""
    for index in (0, 1):
        lib.current = index
        t = tensors(op)
        for x in t.values():
            x.index = index
        lib.calls.clear()
        call(op, t)
        (name, args), = lib.calls
        assert name == ENTRY[op] and args[-1] == 77 + index
        for key, x in t.items():
            if not (op == "weights" and key == "v" or op == "evict" and key == "q_start"):  # (not read)
                assert x.ptr in args, key


@pytest.mark.parametrize("op", OWN)
def test_refuses_another_device(lib, op):
    """A tensor of another GPU or of the host, or a current device that is not the tensors': the launch goes to the
    current device, so nothing is launched."""
    for name in tensors(op):
        for index in (1, -1):
            t = tensors(op)
            t[name].index = index
            with pytest.raises(ValueError):
                call(op, t)
    lib.current = 1
    with pytest.raises(ValueError, match="current device"):
        call(op, tensors(op))
    assert not [c for c in lib.calls if c[0] == ENTRY[op]]


@pytest.mark.parametrize("op", OWN)
@pytest.mark.parametrize("name", SHAPES)
def test_refuses_a_tensor_that_moved(lib, op, name):
    """PagedKV and PagedBatch hold addresses: a tensor that was resized or set to other memory after they were made
    leaves them behind, and nothing is launched on them."""
    for moved in (name, "v") if name == "k" else (name,):
        t = tensors(op)
        kv, batch = ops.PagedKV(t["k"], t["v"]), ops.PagedBatch(t["q_start"], t["kv_len"], t["table"], 3, CAP)
        invoke(op, t, kv, batch)
        lib.calls.clear()
        t[moved].ptr += 4096
        with pytest.raises(ValueError, match="moved"):
            invoke(op, t, kv, batch)
        assert not lib.calls


def test_attributes_that_are_fixed(lib):
    """What a call would not notice cannot be assigned; the bounds and the scale, which it reads, can."""
    t = tensors("attn")
    kv, batch = ops.PagedKV(t["k"], t["v"]), ops.PagedBatch(t["q_start"], t["kv_len"], t["table"], 3, CAP)
    for x, names in ((kv, ("k", "v", "pages", "page", "KVH", "D", "dtype", "device", "layout", "other")),
                     (batch, ("q_start", "kv_len", "table", "B", "per", "other"))):
        for name in names:
            with pytest.raises(AttributeError):
                setattr(x, name, getattr(x, name, 0))
    assert kv.k is t["k"] and batch.kv_len is t["kv_len"]
    batch.max_q, batch.max_kv, kv.scale = 7, 50, 0.25
    lib.calls.clear()
    invoke("attn", t, kv, batch)
    (_, args), = lib.calls
    assert args[5] == 0.25 and args[15:17] == (7, 50)


@pytest.mark.parametrize("op,name,stride", [
    ("attn", "k", (2 ** 33, 2 ** 31, D, 1)), ("attn", "k", (2 ** 40, 2 ** 33, 2 ** 32 + D, 1)),
    ("rope", "k", (PAGE * D, 2 ** 32 + PAGES * PAGE * D, D, 1)),  # heads outermost: cut to 32 bits it would still nest
    ("attn", "q", (2 ** 32 + H * D, D, 1)), ("weights", "q", (2 ** 31, D, 1)), ("rope", "qkv", (2 ** 32 + 1024, 1)),
    ("attn", "gate", (2 ** 32 + H * D, D, 1)), ("attn", "gate", (H * D, 2 ** 32 + D, 1))])
def test_refuses_strides_past_31_bits(lib, op, name, stride):
    """The library's strides but the pages' are 32-bit: a longer one would be cut to its low bits."""
    t = tensors(op)
    t[name].strides = stride
    if name == "k":
        t["v"].strides = stride
    with pytest.raises(ValueError, match="2\\^31"):
        call(op, t)
    assert not [c for c in lib.calls if c[0] == ENTRY[op]]


@pytest.mark.parametrize("bounds", [(2 ** 32, CAP), (2 ** 32 + 3, CAP), (3, 2 ** 32), (3, 2 ** 31), (-1, CAP)])
def test_refuses_bounds_past_31_bits(lib, bounds):
    """max_q = 2^32 would be 0 to the library: nothing computed and no error."""
    t = tensors("weights")
    with pytest.raises(ValueError, match="2\\^31"):
        ops.PagedBatch(t["q_start"], t["kv_len"], t["table"], *bounds)
    batch = ops.PagedBatch(t["q_start"], t["kv_len"], t["table"], 3, CAP)
    with pytest.raises(ValueError, match="2\\^31"):
        batch.max_q, batch.max_kv = bounds


def test_refuses_sizes_past_31_bits(lib):
    t = tensors("attn", table=Fake((B, 2 ** 32 + 4), I32))
    with pytest.raises(ValueError, match="2\\^31"):
        call("attn", t)
    long = (B, KVH, 2 ** 32 + CAP)
    with pytest.raises(ValueError, match="2\\^31"):
        call("weights", tensors("weights", acc=Fake(long, F32)))
    with pytest.raises(ValueError, match="2\\^31"):
        call("evict", tensors("evict", acc=Fake(long, F32), pos=Fake(long, I32), acc_out=Fake(long, F32), pos_out=Fake(long, I32)))
    assert not [c for c in lib.calls if not c[0].endswith("bytes")]


def test_dimensions_of_one_have_no_stride(lib):
    """What a tensor gives as the stride of a dimension of one is not looked at, nor has to fit."""
    t = tensors("attn", k=Fake((1, 1, PAGE, D), F16, stride=(3, 2 ** 40, D, 1)), v=Fake((1, 1, PAGE, D), F16, stride=(9, 5, D, 1)))
    t["q"], t["o"] = Fake((1, 1, D), F16, stride=(7, 2 ** 33, 1)), Fake((1, 1, D), F16)
    t["gate"], t["lse"] = Fake((1, 1, D), F32, stride=(3, 2 ** 35, 1)), Fake((1, 1), F32)
    call("attn", t)
    (_, args), = lib.calls
    assert args[7:9] == (0, 0) and args[1] == D  # gate strides, q's row
    assert args[22:25] == (0, 0, D)              # pages, heads, slots
