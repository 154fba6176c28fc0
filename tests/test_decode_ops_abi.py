"""Refusals of the decoding-step operators, without a GPU: validation runs
before any CUDA call, so a rejected request returns its status with a null
context, and an accepted one reports INVALID_ARGUMENT (18)."""

import ctypes

import numpy as np
import pytest

import decode_helpers as dh

B = ctypes.byref
OK = 18
VIEW, SHAPE, PARAMS, LAYOUT, CAPACITY = 1, 2, 3, 8, 14
FAR = 1 << 30  # addresses are never touched here; each view gets its own gigabyte


def view(emel, slot, ne, kind, nb=None, storage=None, data=None):
    v = emel.CView()
    size = dh.SIZE[kind]
    ne = list(ne) + [1] * (4 - len(ne))
    if nb is None:
        nb = [size]
        for d in range(1, 4):
            nb.append(nb[-1] * max(1, ne[d - 1]))
    v.data = FAR * (slot + 1) if data is None else data
    v.storage_bytes = sum((n - 1) * b for n, b in zip(ne, nb)) + size if storage is None else storage
    for d in range(4):
        v.ne[d], v.nb[d] = ne[d], nb[d]
    v.dtype = dh.CODES[kind]
    return v


def attn(emel, **change):
    a = {"q": ((64, 8, 3), "f32"), "k": ((64, 2, 16, 10), "f16"), "v": ((64, 2, 16, 10), "f16"), "table": ((5, 3), "i32"),
         "lengths": ((3,), "i32"), "out": ((64, 8, 3), "f32")}
    opts = change.pop("opts", None)
    views = []
    for slot, name in enumerate(a):
        c = change.get(name, a[name])
        views.append(c if c is None or isinstance(c, emel.CView) else view(emel, slot, *c[:2], **(c[2] if len(c) > 2 else {})))
    p = [None if v is None else B(v) for v in views]
    return emel.lib().emel_cuda_paged_attn(None, None, *p, None if opts is None else B(opts))


def test_attention(emel):
    assert attn(emel) == OK
    for name in ("q", "k", "v", "table", "lengths", "out"):
        assert attn(emel, **{name: None}) == VIEW, name
    q, kv = (64, 8, 3), (64, 2, 16, 10)
    assert attn(emel, q=(q, "f16"), out=(q, "f16")) == OK
    assert attn(emel, k=(kv, "bf16"), v=(kv, "bf16")) == OK
    assert attn(emel, q=(q, "bf16"), out=(q, "bf16")) == VIEW  # not the cache's type
    assert attn(emel, q=(q, "f16")) == VIEW
    assert attn(emel, v=(kv, "bf16")) == VIEW
    assert attn(emel, k=(kv, "f32"), v=(kv, "f32")) == VIEW
    assert attn(emel, table=((5, 3), "f32")) == VIEW
    assert attn(emel, k=(kv, "f16", {"storage": 100})) == VIEW
    assert attn(emel, k=(kv, "f16", {"data": 4097})) == VIEW
    assert attn(emel, k=((64, 2, 0, 10), "f16"), v=((64, 2, 0, 10), "f16")) == VIEW
    assert attn(emel, k=(kv, "f16", {"nb": [4, 256, 512, 8192]})) == LAYOUT
    assert attn(emel, q=(q, "f32", {"nb": [8, 512, 4096, 12288]})) == LAYOUT
    assert attn(emel, k=(kv, "f16", {"nb": [2, 2048, 128, 4096]}), v=(kv, "f16", {"nb": [2, 2048, 128, 4096]})) == OK
    assert attn(emel, q=((64, 7, 3), "f32"), out=((64, 7, 3), "f32")) == SHAPE  # 7 heads over 2
    assert attn(emel, q=((32, 8, 3), "f32"), out=((32, 8, 3), "f32")) == SHAPE
    assert attn(emel, q=((64, 8, 2), "f32"), out=((64, 8, 2), "f32")) == SHAPE
    assert attn(emel, lengths=((4,), "i32")) == SHAPE
    assert attn(emel, table=((5, 4), "i32")) == SHAPE
    assert attn(emel, table=((5, 3, 2), "i32")) == SHAPE
    assert attn(emel, v=((64, 2, 16, 11), "f16")) == SHAPE
    big = (257, 2, 16, 10)
    assert attn(emel, q=((257, 8, 3), "f32"), out=((257, 8, 3), "f32"), k=(big, "f16"), v=(big, "f16")) == SHAPE
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        assert attn(emel, opts=emel.CPagedAttnOptions(scale, 1, 0, 0)) == PARAMS
    assert attn(emel, opts=emel.CPagedAttnOptions(0.0, 0, 7, 0)) == OK
    assert attn(emel, opts=emel.CPagedAttnOptions(0.0, 0, 7, 1)) == PARAMS


def test_counts_that_would_wrap_are_refused(emel):
    """Sequences and ids of a history are walked with signed 32-bit counters, in steps of up to a few thousand."""
    for n, st in (((1 << 31) - (1 << 16), OK), ((1 << 31) - (1 << 16) + 1, SHAPE), ((1 << 31) - 1, SHAPE)):
        q = ((1, 1, n), "f16")
        cache = ((1, 1, 1, 1), "f16")
        assert attn(emel, q=q, out=(q[0], "f16", {"data": 1 << 46}), k=cache, v=cache, table=((1, n), "i32"),
                    lengths=((n,), "i32")) == st
        assert logits(emel, history=((n, 4), "i32")) == st


def test_events_take_views_and_keep_their_fields(emel):
    v = view(emel, 0, (64, 8, 3), "f32")
    with pytest.raises(TypeError):
        emel.OpLogitsAdjust(v, 7)
    event = emel.OpLogitsAdjust(v, v)
    with pytest.raises(Exception):
        event.src = v
    assert event.dispatch(type("Ctx", (), {"_lib": emel.lib(), "handle": None}), None) == SHAPE
    v.ne[2] = 1  # what a view holds may change
    assert event.dispatch(type("Ctx", (), {"_lib": emel.lib(), "handle": None}), None) == OK


def append(emel, **change):
    a = {"key": ((64, 2, 7), "f32"), "value": ((64, 2, 7), "f32"), "table": ((5, 3), "i32"), "seq": ((7,), "i32"),
         "pos": ((7,), "i32"), "k": ((64, 2, 16, 10), "f16"), "v": ((64, 2, 16, 10), "f16")}
    p = []
    for slot, name in enumerate(a):
        c = change.get(name, a[name])
        p.append(None if c is None else B(view(emel, slot, *c[:2], **(c[2] if len(c) > 2 else {}))))
    return emel.lib().emel_cuda_paged_kv_append(None, None, *p)


def test_append(emel):
    assert append(emel) == OK
    for name in ("key", "value", "table", "pos", "k", "v"):
        assert append(emel, **{name: None}) == VIEW, name
    assert append(emel, seq=None) == SHAPE  # 7 rows, 3 sequences
    assert append(emel, seq=None, key=((64, 2, 3), "f32"), value=((64, 2, 3), "f32"), pos=((3,), "i32")) == OK
    assert append(emel, key=((64, 2, 7), "f16"), value=((64, 2, 7), "f16")) == OK
    assert append(emel, key=((64, 2, 7), "bf16"), value=((64, 2, 7), "bf16")) == VIEW
    assert append(emel, key=((64, 2, 7), "f16")) == VIEW
    assert append(emel, pos=((7,), "f32")) == VIEW
    assert append(emel, key=((64, 2, 7), "f32", {"nb": [8, 512, 1024, 8192]})) == LAYOUT
    assert append(emel, v=((64, 2, 16, 10), "f16", {"nb": [4, 256, 512, 8192]})) == LAYOUT
    assert append(emel, key=((64, 3, 7), "f32"), value=((64, 3, 7), "f32")) == SHAPE
    assert append(emel, value=((64, 2, 8), "f32")) == SHAPE
    assert append(emel, pos=((8,), "i32")) == SHAPE
    assert append(emel, seq=((8,), "i32")) == SHAPE


@pytest.mark.parametrize("fmt", ["q4_0", "q4_1", "q4_k"])
def test_packed_bytes_and_pack(emel, fmt):
    lib = emel.lib()
    values, size = dh.BLOCK[fmt]
    n = ctypes.c_uint64()
    code = dh.CODES[fmt]
    per = {"q4_0": 256, "q4_1": 512, "q4_k": 320}[fmt]
    for k in (values, 3 * values, 4096):
        for rows in (1, 16, 17, 4096):
            assert lib.emel_cuda_q4_packed_bytes(code, k, rows, B(n)) == 0
            assert n.value == (rows + 15) // 16 * ((k + 63) // 64 * 512 + (k + 255) // 256 * per)
    for bad in ((code, values - 1, 4), (code, 0, 4), (code, values, 0), (8, 64, 4), (0, 64, 4), (code, 1 << 60, 1 << 40)):
        assert lib.emel_cuda_q4_packed_bytes(*bad, B(n)) == OK
    assert lib.emel_cuda_q4_packed_bytes(code, values, 4, None) == OK

    def pack(k=512, rows=20, data=4096, short=0, ne2=1, storage=None, dtype=code, out=True):
        v = emel.CView()
        row = k // values * size
        v.data, v.storage_bytes, v.dtype = FAR, row * rows * ne2 if storage is None else storage, dtype
        for d, (ne, nb) in enumerate(zip((k, rows, ne2, 1), (1, row, row * rows, row * rows * ne2))):
            v.ne[d], v.nb[d] = ne, nb
        lib.emel_cuda_q4_packed_bytes(code, 512, 20, B(n))
        w = emel.CQ4Weights()
        return lib.emel_cuda_q4_pack(None, None, B(v), ctypes.c_void_p(data), n.value - short, B(w) if out else None)

    assert pack() == OK
    assert pack(short=1) == CAPACITY
    assert pack(ne2=2) == SHAPE
    assert pack(storage=100) == VIEW
    assert pack(dtype=8) == VIEW
    assert lib.emel_cuda_q4_pack(None, None, None, ctypes.c_void_p(4096), 1 << 20, None) == VIEW


def test_product(emel):
    lib = emel.lib()

    def call(k=512, rows=20, n=3, x=None, y=None, **w):
        need = ctypes.c_uint64()
        lib.emel_cuda_q4_packed_bytes(2, k, rows, B(need))
        c = emel.CQ4Weights(w.get("data", FAR), w.get("bytes", need.value), w.get("k", k), rows, w.get("dtype", 2), w.get("reserved", 0))
        xv = view(emel, 1, (k, n), "f32") if x is None else view(emel, 1, *x[:2], **(x[2] if len(x) > 2 else {}))
        yv = view(emel, 2, (rows, n), "f32") if y is None else view(emel, 2, *y[:2], **(y[2] if len(y) > 2 else {}))
        return lib.emel_cuda_mul_mat_q4(None, None, B(c), B(xv), B(yv))

    assert call() == OK
    assert call(x=((512, 3), "f16"), y=((20, 3), "f16")) == OK
    assert call(data=None) == VIEW and call(data=4104) == VIEW and call(bytes=100) == VIEW
    assert call(dtype=8) == VIEW and call(reserved=1) == VIEW and call(k=500) == VIEW
    assert call(x=((512, 3), "bf16")) == VIEW and call(y=((20, 3), "i32")) == VIEW
    assert call(x=((512, 3), "f32", {"storage": 16})) == VIEW
    assert call(x=((512, 3), "f32", {"nb": [8, 4096, 12288, 12288]})) == LAYOUT
    assert call(y=((20, 3), "f32", {"nb": [8, 160, 480, 480]})) == LAYOUT
    assert call(x=((256, 3), "f32")) == SHAPE and call(x=((512, 4), "f32")) == SHAPE and call(y=((21, 3), "f32")) == SHAPE
    assert call(x=((512, 3, 2), "f32")) == SHAPE
    assert call(k=131072) == OK and call(k=131072 + 32) == SHAPE
    assert lib.emel_cuda_mul_mat_q4(None, None, None, None, None) == VIEW


def logits(emel, **change):
    a = {"src": ((100, 4), "f32"), "history": ((9, 4), "i32"), "used": ((4,), "i32"), "pen": ((3, 4), "f32"),
         "bias": ((100, 4), "f32"), "allowed": ((4, 4), "i32"), "dst": ((100, 4), "f32")}
    p = []
    for slot, name in enumerate(a):
        c = change.get(name, a[name])
        p.append(None if c is None else B(view(emel, slot, *c[:2], **(c[2] if len(c) > 2 else {}))))
    return emel.lib().emel_cuda_logits_adjust(None, None, *p)


def test_logits(emel):
    assert logits(emel) == OK
    assert logits(emel, history=None, used=None, pen=None, bias=None, allowed=None) == OK
    assert logits(emel, pen=((3, 1), "f32"), bias=((100, 1), "f32"), allowed=((4, 1), "i32")) == OK
    for name in ("src", "dst", "history", "used", "pen"):
        assert logits(emel, **{name: None}) == VIEW, name
    assert logits(emel, src=((100, 4), "f16")) == VIEW and logits(emel, src=((100, 4), "bf16")) == VIEW
    assert logits(emel, src=((100, 4), "f16"), dst=((100, 4), "f16")) == OK
    assert logits(emel, bias=((100, 4), "f16")) == VIEW and logits(emel, allowed=((4, 4), "f32")) == VIEW
    assert logits(emel, src=((100, 4), "f32", {"nb": [8, 800, 3200, 3200]})) == LAYOUT
    assert logits(emel, allowed=((4, 4), "i32", {"nb": [8, 32, 128, 128]})) == LAYOUT
    assert logits(emel, dst=((100, 3), "f32")) == SHAPE and logits(emel, history=((9, 3), "i32")) == SHAPE
    assert logits(emel, used=((3,), "i32")) == SHAPE and logits(emel, pen=((2, 4), "f32")) == SHAPE
    assert logits(emel, bias=((100, 3), "f32")) == SHAPE and logits(emel, allowed=((3, 4), "i32")) == SHAPE
    assert logits(emel, src=((100, 4, 2), "f32"), dst=((100, 4, 2), "f32")) == SHAPE


@pytest.mark.gpu
def test_overlaps_are_refused(emel):
    ctx = emel.Context(0)
    lib, h = ctx._lib, ctx.handle
    buf = emel.DeviceBuffer(ctx, 1 << 20)
    buf.upload(np.zeros(1 << 18, np.float32))
    at = lambda off, ne, kind: view(emel, 0, ne, kind, data=buf.ptr + off)  # noqa: E731
    x = at(0, (64, 2, 1), "f32")
    k, v = at(65536, (64, 2, 4, 2), "f16"), at(131072, (64, 2, 4, 2), "f16")
    table, n = at(4096, (1, 1), "i32"), at(8192, (1,), "i32")
    for out in (x, at(256, (64, 2, 1), "f32"), at(65536 + 100, (64, 2, 1), "f32"), at(4096, (64, 2, 1), "f32")):
        assert lib.emel_cuda_paged_attn(h, None, B(x), B(k), B(v), B(table), B(n), B(out), None) == OK
    src = at(0, (100, 4), "f32")
    assert lib.emel_cuda_logits_adjust(h, None, B(src), None, None, None, None, None, B(at(4, (100, 4), "f32"))) == OK
    assert lib.emel_cuda_logits_adjust(h, None, B(src), None, None, None, None, None, B(src)) == 0
    bias = at(0, (100, 1), "f32")
    assert lib.emel_cuda_logits_adjust(h, None, B(src), None, None, None, B(bias), None, B(src)) == OK
    ctx.synchronize()
    buf.free()


def test_windows_that_do_not_fit_are_refused(emel):
    """They would be taken modulo 2^32, and a window of 2^32 for none."""
    views = [view(emel, i, ne, kind) for i, (ne, kind) in enumerate(
        [((64, 8, 3), "f32"), ((64, 2, 16, 10), "f16"), ((64, 2, 16, 10), "f16"), ((5, 3), "i32"), ((3,), "i32"), ((64, 8, 3), "f32")])]
    ctx = type("Ctx", (), {"_lib": emel.lib(), "handle": None})
    for window in (-1, 1 << 32, -(1 << 40)):
        with pytest.raises(ValueError, match="window"):
            emel.OpPagedAttn(*views, window=window)
    with pytest.raises(TypeError):
        emel.OpPagedAttn(*views, window=1.5)
    for window in (0, 1, (1 << 32) - 1, np.int64(7)):
        assert emel.OpPagedAttn(*views, window=window).dispatch(ctx, None) == OK


@pytest.mark.parametrize("how", ["copy", "deepcopy", "pickle", "replace"])
def test_copies_of_an_event_stand_on_their_own(emel, how):
    """An event keeps the addresses of its options and views; a copy's are those of the copy's own."""
    import copy
    import dataclasses
    import pickle
    layout = lambda ne, kind: emel.Layout.contiguous(emel.DType(dh.CODES[kind]), list(ne) + [1] * (4 - len(ne)))  # noqa: E731
    views = [emel.TensorView(FAR * (i + 1), 1 << 20, layout(ne, kind)) for i, (ne, kind) in enumerate(
        [((64, 8, 3), "f32"), ((64, 2, 16, 10), "f16"), ((64, 2, 16, 10), "f16"), ((5, 3), "i32"), ((3,), "i32"), ((64, 8, 3), "f32")])]
    event = emel.OpPagedAttn(*views, scale=0.25, window=9)
    made = {"copy": copy.copy, "deepcopy": copy.deepcopy, "pickle": lambda e: pickle.loads(pickle.dumps(e)),
            "replace": lambda e: dataclasses.replace(e, window=9)}[how](event)
    assert made == event
    options, at = made._options
    assert at == ctypes.addressof(options) and (options.scale, options.window) == (0.25, 9)
    if how in ("deepcopy", "pickle", "replace"):
        assert options is not event._options[0]
    held = emel.OpLogitsAdjust(views[0].c(), views[5].c())
    if how in ("copy", "replace"):  # a CView is an address: Python does not copy it more deeply
        other = copy.copy(held) if how == "copy" else dataclasses.replace(held, dst=views[1].c())
        assert other._at == tuple(v and ctypes.addressof(v) for v in (getattr(other, n) for n in other.VIEWS))


class HostOnly:
    """A context whose memory and layout kernel are stand-ins: host logic without a GPU."""

    def __init__(self, emel):
        self.handle, self.freed, real = None, [], emel.lib()

        class Lib:
            def __getattr__(_, name):
                return getattr(real, name)

            def emel_cuda_malloc(_, ctx, n, out):
                out._obj.value = FAR
                return 0

            def emel_cuda_free(_, ctx, at):
                self.freed.append(at)
                return 0

            def emel_cuda_q4_pack(_, ctx, stream, src, data, n, out):
                w, v = out._obj, src._obj
                w.data, w.bytes, w.k, w.rows, w.dtype, w.reserved = data.value, n, v.ne[0], v.ne[1], v.dtype, 0
                return 0

        self._lib = Lib()


def test_weights_that_were_freed_are_refused(emel):
    """Their events keep the handle: it names no memory any more."""
    ctx = HostOnly(emel)
    src = view(emel, 3, (64, 16, 1, 1), "i32", nb=[1, 36, 576, 576], storage=576)
    src.dtype = dh.CODES["q4_0"]
    w = emel.Q4Weights(ctx, src)
    event = emel.OpMulMatQ4(w, view(emel, 1, (64, 2), "f32"), view(emel, 2, (16, 2), "f32"))
    assert event.dispatch(ctx, None) == OK
    w.free()
    assert ctx.freed == [FAR]
    assert event.dispatch(ctx, None) == VIEW
    w.free()
    assert ctx.freed == [FAR]
