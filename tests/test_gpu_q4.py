"""Matrix-vector products with 4-bit weights (emel_cuda_q4_pack,
emel_cuda_mul_mat_q4) against the formats' definitions in 64 bits.

With w = a (q - 8) + c per group of 32: products are exact or rounded once, a
group's 32 terms and then the k / 32 groups are added in binary32 (one extra
bit where an addition truncates), so |error| <= (64 + k / 32) 2^-23 sum (|a (q - 8)| + |c|) |x|.
A binary16 result adds its rounding, 2^-11 |y| (or 2^-25 where it is subnormal)."""

import numpy as np
import pytest

import decode_helpers as dh
import gguf_writer

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def kern(emel):
    return emel.Kernel(device=0, synchronize=True)


class Blocks:
    def __init__(self, emel, ctx, raw, fmt, skip=0):
        self.raw, self.fmt, self.emel = raw, fmt, emel
        host = np.concatenate([np.zeros(skip, np.uint8), raw.reshape(-1)])
        self.buf = emel.DeviceBuffer(ctx, max(16, host.nbytes))
        self.buf.upload(host)
        self.skip = skip

    def c(self):
        values, size = dh.BLOCK[self.fmt]
        v = self.emel.CView()
        rows, row = self.raw.shape
        v.data, v.storage_bytes, v.dtype = self.buf.ptr + self.skip, self.raw.size, dh.CODES[self.fmt]
        for d, (ne, nb) in enumerate(zip((row // size * values, rows, 1, 1), (1, row, row * rows, row * rows))):
            v.ne[d], v.nb[d] = ne, nb
        return v


def parts(raw, fmt):
    """|a (q - 8)| + |c| of every weight: the magnitude that the bar goes by."""
    w = dh.q4_values(raw, fmt)
    if fmt == "q4_0":
        return np.abs(w)
    mid = raw.copy().reshape(raw.shape[0], -1, dh.BLOCK[fmt][1])
    mid[:, :, 16 if fmt == "q4_k" else 4:] = 0x88  # quants of 8: what is left is c
    c = dh.q4_values(mid.reshape(raw.shape), fmt)
    return np.abs(w - c) + np.abs(c)


def check(emel, kern, fmt, k, rows, n, x="f32", out="f32", seed=0, pad=0, skip=0, values=None):
    rng = np.random.default_rng(seed + k + rows)
    raw = dh.q4_random(rng, fmt, rows, k)
    act = rng.standard_normal((n, k)) if values is None else values(rng, (n, k))
    act[:, ::41] *= 16
    xd = dh.Dev(emel, kern.ctx, act, x, pad=pad, skip=skip)
    yd = dh.Dev(emel, kern.ctx, np.full((n, rows), 7.0), out, pad=pad, skip=skip, fill=9.0)
    blocks = Blocks(emel, kern.ctx, raw, fmt, skip)
    w = emel.Q4Weights(kern.ctx, blocks.c())
    blocks.buf.free()
    assert kern.process_event(emel.OpMulMatQ4(w, xd.c(), yd.c())) == 0, kern.ctx.last_error
    got = yd.read()
    want = xd.values @ dh.q4_values(raw, fmt).T
    tol = (64 + k / 32) * 2.0 ** -23 * (np.abs(xd.values) @ parts(raw, fmt).T)
    if out == "f16":
        tol = tol + 2.0 ** -11 * np.abs(want) + 2.0 ** -25
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (int(bad.sum()), float(np.max(np.abs(got - want) / tol)), np.argwhere(bad)[:4])
    touched = np.zeros(yd.host.shape, bool)
    np.lib.stride_tricks.as_strided(touched[yd.skip:], yd.shape, list(yd.strides))[...] = True
    assert (yd.raw()[~touched] == 9.0).all()
    w.free()
    return got


FORMATS = ["q4_0", "q4_1", "q4_k"]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("x,out", [("f32", "f32"), ("f16", "f32"), ("f32", "f16"), ("f16", "f16")])
@pytest.mark.parametrize("n", [1, 2, 3, 5, 6, 8, 9, 17])
def test_tokens_and_types(emel, kern, fmt, x, out, n):
    check(emel, kern, fmt, 512, 100, n, x, out)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 33, 255, 2400, 5001])
@pytest.mark.parametrize("n", [1, 4])
def test_rows(emel, kern, fmt, rows, n):
    check(emel, kern, fmt, 768, rows, n)


@pytest.mark.parametrize("fmt,k", [("q4_0", 32), ("q4_0", 64), ("q4_0", 96), ("q4_0", 224), ("q4_0", 288), ("q4_0", 2848),
                                   ("q4_1", 32), ("q4_1", 160), ("q4_1", 4064), ("q4_k", 256), ("q4_k", 1280),
                                   ("q4_0", 8192), ("q4_1", 16384), ("q4_k", 20480), ("q4_0", 33568), ("q4_k", 70400)])
@pytest.mark.parametrize("x,n", [("f32", 1), ("f32", 8), ("f16", 1), ("f16", 8)])
def test_columns(emel, kern, fmt, k, x, n):
    check(emel, kern, fmt, k, 50, n, x)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("x,out", [("f32", "f32"), ("f16", "f16")])
@pytest.mark.parametrize("pad,skip", [(1, 0), (4, 2), (8, 8), (3, 1)])
def test_strides_and_alignment(emel, kern, fmt, x, out, pad, skip):
    check(emel, kern, fmt, 1024, 77, 3, x, out, pad=pad, skip=skip)


@pytest.mark.parametrize("size", [1e-30, 1e-12, 1e30])
def test_activations_of_any_size(emel, kern, size):
    check(emel, kern, "q4_0", 512, 40, 2, values=lambda rng, s: rng.standard_normal(s) * size)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("n", [1, 2, 3])
@pytest.mark.parametrize("size", [1e-32, 1e-34, 1e-37, 1e-40])
def test_activations_near_the_smallest_numbers(emel, kern, fmt, n, size):
    """Down to subnormal columns, which have fewer bits themselves, and subnormal results: every sum has 2^-23
    of its parts at least, far above half of 2^-149."""
    check(emel, kern, fmt, 512, 40, n, values=lambda rng, s: rng.standard_normal(s) * size)


def test_not_finite_activations_stay_in_their_column(emel, kern):
    rng = np.random.default_rng(3)
    raw = dh.q4_random(rng, "q4_1", 30, 256)
    act = rng.standard_normal((4, 256)).astype(np.float32)
    act[1, 7], act[2, 100], act[3, 9] = np.nan, np.inf, np.finfo(np.float32).max
    xd, yd = dh.Dev(emel, kern.ctx, act, "f32"), dh.Dev(emel, kern.ctx, np.zeros((4, 30)), "f32")
    blocks = Blocks(emel, kern.ctx, raw, "q4_1")
    w = emel.Q4Weights(kern.ctx, blocks.c())
    assert kern.process_event(emel.OpMulMatQ4(w, xd.c(), yd.c())) == 0
    got = yd.read()
    want = dh.q4_values(raw, "q4_1") @ act[0].astype(np.float64)
    assert np.abs(got[0] - want).max() < 1e-4
    assert np.isnan(got[1]).all() and not np.isfinite(got[2]).any()
    top = np.abs(got[3]) > 1e36  # the largest float: a sum near it, or past it
    assert top.sum() >= 20


@pytest.mark.parametrize("x", ["f32", "f16"])
def test_not_finite_activations_of_one_or_two_tokens(emel, kern, x):
    rng = np.random.default_rng(4)
    raw = dh.q4_random(rng, "q4_0", 40, 512)
    blocks = Blocks(emel, kern.ctx, raw, "q4_0")
    w = emel.Q4Weights(kern.ctx, blocks.c())
    for bad in (np.nan, np.inf, -np.inf):
        act = rng.standard_normal((2, 512)).astype(np.float32)
        act[0, 333] = bad
        xd, yd = dh.Dev(emel, kern.ctx, act, x), dh.Dev(emel, kern.ctx, np.zeros((2, 40)), "f32")
        assert kern.process_event(emel.OpMulMatQ4(w, xd.c(), yd.c())) == 0
        got = yd.read()
        assert not np.isfinite(got[0]).any()
        tol = (64 + 16) * 2.0 ** -23 * (np.abs(xd.values[1]) @ parts(raw, "q4_0").T)
        assert (np.abs(got[1] - xd.values[1] @ dh.q4_values(raw, "q4_0").T) <= tol).all()


def test_columns_of_zeros(emel, kern):
    rng = np.random.default_rng(14)
    raw = dh.q4_random(rng, "q4_1", 33, 320)
    blocks = Blocks(emel, kern.ctx, raw, "q4_1")
    w = emel.Q4Weights(kern.ctx, blocks.c())
    for n in (1, 2, 3, 8):
        xd, yd = dh.Dev(emel, kern.ctx, np.zeros((n, 320)), "f32"), dh.Dev(emel, kern.ctx, np.full((n, 33), 5.0), "f32")
        assert kern.process_event(emel.OpMulMatQ4(w, xd.c(), yd.c())) == 0
        assert (yd.read() == 0).all()


def test_the_same_call_gives_the_same_bits_on_another_stream(emel, kern):
    rng = np.random.default_rng(5)
    ctx = kern.ctx
    raw = dh.q4_random(rng, "q4_k", 3000, 4096)
    blocks = Blocks(emel, ctx, raw, "q4_k")
    w = emel.Q4Weights(ctx, blocks.c())
    xd, yd = dh.Dev(emel, ctx, rng.standard_normal((8, 4096)), "f32"), dh.Dev(emel, ctx, np.zeros((8, 3000)), "f32")
    event = emel.OpMulMatQ4(w, xd.c(), yd.c())
    assert kern.process_event(event) == 0
    first = yd.raw().copy()
    stream = emel.Stream(ctx)
    on = emel.Kernel(ctx=ctx, stream=stream.handle)
    with emel.Graph(ctx, stream) as graph:
        assert on.process_event(event) == 0
    for _ in range(10):
        yd.buf.upload(np.zeros_like(yd.host), stream.handle)
        graph.launch()
    stream.synchronize()
    assert (yd.raw() == first).all()
    graph.close()
    stream.close()


def test_weights_just_packed_are_read_whole(emel, kern):
    """Pack, product and a second product over its result, queued without a wait."""
    rng = np.random.default_rng(6)
    ctx = kern.ctx
    quiet = emel.Kernel(ctx=ctx)
    raw = dh.q4_random(rng, "q4_0", 1024, 1024)
    blocks = Blocks(emel, ctx, raw, "q4_0")
    x = dh.Dev(emel, ctx, rng.standard_normal((1, 1024)), "f32")
    mid, out = (dh.Dev(emel, ctx, np.zeros((1, 1024)), "f32") for _ in range(2))
    vals = dh.q4_values(raw, "q4_0")
    for _ in range(5):
        w = emel.Q4Weights(ctx, blocks.c())
        assert quiet.process_event(emel.OpMulMatQ4(w, x.c(), mid.c())) == 0
        assert quiet.process_event(emel.OpMulMatQ4(w, mid.c(), out.c())) == 0
        ctx.synchronize()
        mag = np.abs(x.values) @ np.abs(vals).T
        want = (x.values @ vals.T) @ vals.T
        tol = 2 * (64 + 32) * 2.0 ** -23 * (mag @ np.abs(vals).T)
        assert (np.abs(out.read() - want) <= tol).all()
        w.free()


def test_gguf_rows(emel, kern):
    """A Q4_K tensor of a GGUF image through the loader, the layout and a product."""
    rng = np.random.default_rng(8)
    raw = dh.q4_random(rng, "q4_k", 64, 512)
    image = gguf_writer.image([(b"w", [512, 64], 12, raw.tobytes())])
    buf, view = emel.GgufImage(image).upload(kern.ctx, "w")
    w = emel.Q4Weights(kern.ctx, view)
    x, y = dh.Dev(emel, kern.ctx, rng.standard_normal((1, 512)), "f32"), dh.Dev(emel, kern.ctx, np.zeros((1, 64)), "f32")
    assert kern.process_event(emel.OpMulMatQ4(w, x.c(), y.c())) == 0
    tol = (64 + 16) * 2.0 ** -23 * (np.abs(x.values) @ parts(raw, "q4_k").T)
    assert (np.abs(y.read() - x.values @ dh.q4_values(raw, "q4_k").T) <= tol).all()
    buf.free()
