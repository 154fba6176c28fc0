"""Penalties, biases and masks on logits (emel_cuda_logits_adjust) against the
formula in 64 bits.

At most five binary32 roundings of values no larger than |v| max(r, 1 / r) +
c |f| + |p| + |bias|: |error| <= 5 * 2^-24 of that sum; a binary16 result adds
its own rounding, 2^-11 |y| (or 2^-25 where it is subnormal)."""

import numpy as np
import pytest

import decode_helpers as dh

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def kern(emel):
    return emel.Kernel(device=0, synchronize=True)


def bits(mask):
    rows, vocab = mask.shape
    full = np.zeros((rows, (vocab + 31) // 32 * 32), bool)
    full[:, :vocab] = mask
    return np.packbits(full, axis=1, bitorder="little").view(np.int32)


def case(emel, ctx, seed, rows, vocab, hist=0, bias=0, allowed=0, kind="f32", pen_rows=None, pad=0, skip=0, special=False):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((rows, vocab)) * 4
    if special:
        x.reshape(-1)[rng.choice(x.size, 12, replace=False)] = [0.0, -0.0, np.inf, -np.inf, np.nan, 65504, -65504, 6e-8,
                                                                 -np.inf, np.nan, np.inf, 1.0]
    d = {"src": dh.Dev(emel, ctx, x, kind, pad=pad, skip=skip)}
    if hist:
        ids = (rng.random((rows, hist)) ** 3 * vocab).astype(int)
        ids[rng.random((rows, hist)) < 0.05] = -1
        ids[rng.random((rows, hist)) < 0.02] = vocab + 3
        n = rng.integers(0, hist + 1, rows)
        n[0] = hist
        d["history"], d["used"] = dh.Dev(emel, ctx, ids, "i32", pad=pad), dh.Dev(emel, ctx, n, "i32")
        pr = pen_rows or rows
        d["pen"] = dh.Dev(emel, ctx, np.stack([rng.uniform(0.8, 1.6, pr), rng.uniform(-0.5, 1, pr), rng.uniform(-0.5, 1, pr)], 1), "f32", pad=pad)
    if bias:
        d["bias"] = dh.Dev(emel, ctx, rng.standard_normal((bias, vocab)) * (rng.random((bias, vocab)) < 0.1), "f32", pad=pad, skip=skip)
    if allowed:
        d["mask"] = rng.random((allowed, vocab)) < 0.5
        if rows > 1 and allowed == rows:
            d["mask"][1] = False  # a row with nothing left
        d["allowed"] = dh.Dev(emel, ctx, bits(d["mask"]), "i32", pad=pad, skip=skip)
    return d


def run(emel, kern, d, kind, pad=0, skip=0, in_place=False):
    out = d["src"] if in_place else dh.Dev(emel, kern.ctx, np.full(d["src"].shape, 7.0), kind, pad=pad, skip=skip, fill=9.0)
    opt = lambda k: d[k].c() if k in d else None  # noqa: E731
    st = kern.process_event(emel.OpLogitsAdjust(d["src"].c(), out.c(), opt("history"), opt("used"), opt("pen"), opt("bias"), opt("allowed")))
    assert int(st) == 0, kern.ctx.last_error
    return out


def check(emel, kern, d, kind, out):
    val = lambda k: d[k].values if k in d else None  # noqa: E731
    x, got = d["src"].values, out.read()
    with np.errstate(invalid="ignore"):
        want = dh.adjusted(x, val("history"), val("used"), val("pen"), val("bias"), d.get("mask"))
        mag = np.abs(x)
        if "pen" in d:
            r, f, p = (np.abs(val("pen")[:, i: i + 1]) for i in range(3))
            mag = mag * np.maximum(r, 1 / r) + val("history").shape[1] * f + p
        if "bias" in d:
            mag = mag + np.abs(val("bias"))
        if kind == "f16":
            want = np.where(np.abs(want) >= 65520, np.sign(want) * np.inf, want)
        tol = 5 * 2.0 ** -24 * mag + (2.0 ** -11 * np.abs(want) + 2.0 ** -25 if kind == "f16" else 0.0)
        fine = np.isfinite(want)
        assert (np.isnan(got) == np.isnan(want)).all()
        assert (got[~fine & ~np.isnan(want)] == want[~fine & ~np.isnan(want)]).all()
        bad = fine & ~(np.abs(got - want) <= tol)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4])


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (1, 31), (3, 33), (2, 8191), (2, 8192), (5, 8193), (4, 32000), (3, 50257), (2, 151936)])
@pytest.mark.parametrize("what", ["nothing", "history", "bias", "mask", "all"])
def test_sizes(emel, kern, kind, rows, vocab, what):
    use = lambda k: what in (k, "all")  # noqa: E731
    d = case(emel, kern.ctx, vocab, rows, vocab, 60 if use("history") else 0, rows if use("bias") else 0, rows if use("mask") else 0, kind)
    check(emel, kern, d, kind, run(emel, kern, d, kind))


@pytest.mark.parametrize("hist", [1, 2, 255, 256, 1023, 5000, 100000])
def test_history_lengths(emel, kern, hist):
    d = case(emel, kern.ctx, hist, 3, 20000, hist)
    check(emel, kern, d, "f32", run(emel, kern, d, "f32"))


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("pad,skip", [(1, 0), (0, 1), (4, 4), (3, 2), (8, 8)])
def test_strides_alignment_and_shared_rows(emel, kern, kind, pad, skip):
    for vocab in (9000, 16384, 77):
        d = case(emel, kern.ctx, pad + skip, 4, vocab, 40, 1, 1, kind, pen_rows=1, pad=pad, skip=skip)
        out = run(emel, kern, d, kind, pad, skip)
        check(emel, kern, d, kind, out)
        touched = np.zeros(out.host.shape, bool)
        np.lib.stride_tricks.as_strided(touched[out.skip:], out.shape, list(out.strides))[...] = True
        assert (out.raw()[~touched] == 9.0).all()


@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_infinities_and_nan(emel, kern, kind):
    for seed in range(4):
        d = case(emel, kern.ctx, seed, 2, 3000, 50, 2, 2 if seed % 2 else 0, kind, special=True)
        check(emel, kern, d, kind, run(emel, kern, d, kind))


def test_in_place_and_then_the_argmax(emel, kern):
    d = case(emel, kern.ctx, 3, 4, 32000, 100, 1, 4)
    check(emel, kern, d, "f32", run(emel, kern, d, "f32", in_place=True))
    val = lambda k: d[k].values  # noqa: E731
    want = dh.adjusted(val("src"), val("history"), val("used"), val("pen"), val("bias"), d["mask"])
    idx = emel.DeviceBuffer(kern.ctx, 64)
    view = idx.view(emel.Layout.contiguous(emel.DType.I32, [1, 4, 1, 1]))
    src = d["src"].c()
    assert kern.process_event(emel.OpArgmaxRows(src, view)) == 0
    got = idx.download(np.zeros(16, np.int32))[:4]
    rows = [0, 2, 3]
    assert [int(got[r]) for r in rows] == [int(np.argmax(want[r])) for r in rows]


def test_lengths_are_held_to_the_capacity(emel, kern):
    d = case(emel, kern.ctx, 9, 2, 500, 20)
    want_used = d["used"].values.copy()
    d["used"] = dh.Dev(emel, kern.ctx, [1 << 30, -7], "i32")
    out = run(emel, kern, d, "f32")
    d["used"].values = np.array([20, 0])
    check(emel, kern, d, "f32", out)
    assert want_used[0] == 20


def test_many_rows(emel, kern):
    d = case(emel, kern.ctx, 11, 70000, 40, 3)
    check(emel, kern, d, "f32", run(emel, kern, d, "f32"))
