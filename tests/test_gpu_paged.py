"""Paged cache (emel_cuda_paged_kv_append, emel_cuda_paged_attn) against the
formulas in 64 bits.

Attention's bar per output, with S the largest sum |q_i k_i| * scale, V the
largest |v| and T the tokens: a score is off by at most (d + 16) 2^-23 S (d
binary32 additions, two splits of the query, the scale), which moves a weight
by that much; the weights' exponential, their sum and the sum over the values
add (T + 16) 2^-23.  So |error| <= V (2 (d + 16) 2^-23 S + (T + 16) 2^-23).  16-bit
queries round each weight (relative 2^-11 in binary16, where a weight under
2^-14 of the largest is off by 2^-25 of it; 2^-9 in bfloat16) and the result
(the same, of the result).  The append is exact."""

import numpy as np
import pytest

import decode_helpers as dh

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def kern(emel):
    return emel.Kernel(device=0, synchronize=True)


def bar(q, k, v, table, lengths, scale, window, want, qkind, kvkind):
    page = k.shape[1]
    tol = np.zeros(want.shape[:2])
    unit = 0.0 if qkind == "f32" else 2.0 ** -11 if kvkind == "f16" else 2.0 ** -9
    for b, n in enumerate(lengths):
        n = max(0, min(int(n), table.shape[1] * page))
        at = np.arange(max(0, n - window) if window else 0, n)
        if at.size == 0:
            continue
        kk, vv = k[table[b, at // page], at % page], v[table[b, at // page], at % page]
        for h in range(q.shape[1]):
            g = h // (q.shape[1] // k.shape[2])
            s = (np.abs(kk[:, g]) @ np.abs(q[b, h]) * scale).max()
            big = np.abs(vv[:, g]).max()
            tol[b, h] = big * (2 * (q.shape[2] + 16) * 2.0 ** -23 * s + (at.size + 16) * 2.0 ** -23 +
                               unit + (at.size * 2.0 ** -25 if unit else 0.0))
    return tol[:, :, None] + unit * np.abs(want) + (2.0 ** -24 if qkind == "f16" else 0.0)


def cache(emel, ctx, rng, pages, page, kvh, d, kind, layout, used, pad=0, skip=0, garbage=True):
    """A cache whose slots outside `used` (page, offset pairs) hold NaN and infinities."""
    x = rng.standard_normal((pages, page, kvh, d)).astype(np.float32)
    if garbage:
        free = np.ones((pages, page), bool)
        free[used] = False
        x[free] = rng.choice(np.array([np.nan, np.inf, -np.inf], np.float32), (int(free.sum()), kvh, d))
    return dh.Dev(emel, ctx, x, kind, order=(0, 1, 2, 3) if layout == "token" else (0, 2, 1, 3), pad=pad, skip=skip)


def setup(emel, ctx, seed, lengths, kvh, rep, d, page, qkind="f32", kvkind="f16", layout="token", pad=0, skip=0,
          window=0, spare=2, extra_entries=0):
    rng = np.random.default_rng(seed)
    lengths = np.asarray(lengths)
    counts = np.maximum(0, -(-lengths // page))
    pages = int(counts.sum()) + spare
    pool = rng.permutation(pages)
    table = np.full((len(lengths), max(1, int(counts.max())) + extra_entries), -1, np.int64)
    at = 0
    used = ([], [])
    for b, n in enumerate(lengths):
        table[b, :counts[b]] = pool[at: at + counts[b]]
        at += counts[b]
        t = np.arange(max(0, n - window) if window else 0, max(0, n))
        used[0].extend(table[b, t // page])
        used[1].extend(t % page)
    used = (np.array(used[0], int), np.array(used[1], int))
    q = dh.Dev(emel, ctx, rng.standard_normal((len(lengths), kvh * rep, d)), qkind, pad=pad, skip=skip)
    k = cache(emel, ctx, rng, pages, page, kvh, d, kvkind, layout, used, pad, skip)
    v = cache(emel, ctx, rng, pages, page, kvh, d, kvkind, layout, used, pad, skip)
    out = dh.Dev(emel, ctx, np.full((len(lengths), kvh * rep, d), 7.0), qkind, pad=pad, skip=skip, fill=9.0)
    return q, k, v, dh.Dev(emel, ctx, table, "i32"), dh.Dev(emel, ctx, lengths, "i32"), out


def check(emel, kern, devs, scale=None, window=0, status=0):
    q, k, v, table, lengths, out = devs
    st = kern.process_event(emel.OpPagedAttn(q.c(), k.c(), v.c(), table.c(), lengths.c(), out.c(), scale, window))
    assert int(st) == status, kern.ctx.last_error
    got = out.read()
    s = 1.0 / np.sqrt(q.shape[2]) if scale is None else scale
    want = dh.attention(q.values, k.values, v.values, table.values, lengths.values, s, window)
    with np.errstate(invalid="ignore"):
        tol = bar(q.values, k.values, v.values, table.values, lengths.values, s, window, want, q.kind, k.kind)
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (int(bad.sum()), float(np.nanmax(np.abs(got - want) / tol)), np.argwhere(bad)[:4])
    return got, want


TYPES = [("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")]


@pytest.mark.parametrize("qkind,kvkind", TYPES)
@pytest.mark.parametrize("kvh,rep,d,page", [(8, 4, 128, 16), (2, 1, 64, 1), (1, 8, 256, 64), (3, 5, 80, 7), (1, 16, 96, 100),
                                            (2, 17, 40, 16), (1, 33, 192, 5), (4, 2, 32, 16), (2, 3, 72, 33)])
def test_heads_and_types(emel, kern, qkind, kvkind, kvh, rep, d, page):
    lengths = [1, 0, 17, 64, 65, 130, 300, 16]
    check(emel, kern, setup(emel, kern.ctx, 1, lengths, kvh, rep, d, page, qkind, kvkind))


@pytest.mark.parametrize("qkind,kvkind", TYPES)
@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 63, 64, 127, 255, 1000, 4097, 20000])
def test_lengths_of_one_sequence(emel, kern, qkind, kvkind, n):
    check(emel, kern, setup(emel, kern.ctx, n, [n], 2, 4, 128, 16, qkind, kvkind))


@pytest.mark.parametrize("layout", ["token", "head"])
@pytest.mark.parametrize("d,pad,skip", [(1, 0, 0), (7, 1, 3), (33, 0, 0), (64, 8, 8), (64, 4, 0), (100, 0, 4), (128, 1, 0),
                                        (200, 8, 1), (255, 1, 0), (256, 16, 5)])
@pytest.mark.parametrize("qkind,kvkind", TYPES)
def test_columns_strides_and_alignment(emel, kern, layout, d, pad, skip, qkind, kvkind):
    check(emel, kern, setup(emel, kern.ctx, d, [3, 77, 200], 2, 3, d, 9, qkind, kvkind, layout, pad, skip))


@pytest.mark.parametrize("window", [1, 5, 16, 63, 64, 200, 5000])
@pytest.mark.parametrize("qkind,kvkind", TYPES)
def test_window(emel, kern, window, qkind, kvkind):
    check(emel, kern, setup(emel, kern.ctx, window, [1, 5, 64, 1000, 0, 201, 3333], 2, 4, 64, 16, qkind, kvkind,
                            window=window), window=window)


def test_many_ragged_sequences(emel, kern):
    rng = np.random.default_rng(5)
    lengths = np.where(rng.random(300) < 0.3, 0, rng.integers(1, 400, 300))
    check(emel, kern, setup(emel, kern.ctx, 6, lengths, 2, 4, 64, 16, "bf16", "bf16"))
    check(emel, kern, setup(emel, kern.ctx, 7, lengths[:150], 1, 2, 128, 10))


def test_one_long_among_short(emel, kern):
    check(emel, kern, setup(emel, kern.ctx, 8, [1] * 40 + [30011] + [2] * 40, 1, 8, 64, 32))


def test_only_empty_sequences(emel, kern):
    devs = setup(emel, kern.ctx, 9, [0, 0, 0], 2, 4, 64, 16)
    got, _ = check(emel, kern, devs)
    assert (got == 0).all()


def test_scale_and_sharp_scores(emel, kern):
    devs = setup(emel, kern.ctx, 10, [500, 33], 2, 4, 64, 16)
    for scale in (1e-3, 0.5, 4.0):
        check(emel, kern, devs, scale=scale)


@pytest.mark.parametrize("kvkind", ["f16", "bf16"])
@pytest.mark.parametrize("size", [1e-6, 1e4, 3e5])
def test_queries_far_from_one(emel, kern, kvkind, size):
    """A binary32 query keeps its precision whatever its size: the scale brings the scores back."""
    q, k, v, table, lengths, out = setup(emel, kern.ctx, 11, [700, 90], 1, 4, 128, 16, "f32", kvkind)
    q = dh.Dev(emel, kern.ctx, q.values * size, "f32")
    check(emel, kern, (q, k, v, table, lengths, out), scale=0.1 / size)


def test_infinite_scores(emel, kern):
    """Scores of -inf weigh nothing; where every score is -inf the row is zero; +inf gives NaN."""
    ctx = kern.ctx
    q = dh.Dev(emel, ctx, np.ones((3, 1, 16)), "f32")
    k = np.ones((3, 16, 1, 16), np.float32)
    k[0, 3, 0, 0], k[1, :, 0, 2], k[2, 5, 0, 1] = -np.inf, -np.inf, np.inf
    rng = np.random.default_rng(3)
    kd, vd = dh.Dev(emel, ctx, k, "f16"), dh.Dev(emel, ctx, rng.standard_normal(k.shape), "f16")
    table, lengths = dh.Dev(emel, ctx, [[0], [1], [2]], "i32"), dh.Dev(emel, ctx, [16, 16, 16], "i32")
    out = dh.Dev(emel, ctx, np.zeros((3, 1, 16)), "f32")
    assert kern.process_event(emel.OpPagedAttn(q.c(), kd.c(), vd.c(), table.c(), lengths.c(), out.c())) == 0
    got = out.read()
    keep = [t for t in range(16) if t != 3]
    assert np.abs(got[0, 0] - vd.values[0, keep, 0].mean(0)).max() <= 32 * 2.0 ** -23 * np.abs(vd.values).max()
    assert (got[1] == 0).all()
    assert np.isnan(got[2]).all()


@pytest.mark.parametrize("kvkind", ["f16", "bf16"])
@pytest.mark.parametrize("size,scale", [(1e-39, 2e38), (1e-36, 1e35), (1e-30, 1e29), (1e37, 1e-38)])
def test_queries_of_any_size(emel, kern, kvkind, size, scale):
    """From subnormal queries to the largest: the scale brings the scores back."""
    q, k, v, table, lengths, out = setup(emel, kern.ctx, 11, [70, 9], 1, 4, 32, 16, "f32", kvkind)
    q = dh.Dev(emel, kern.ctx, q.values * size, "f32")
    check(emel, kern, (q, k, v, table, lengths, out), scale=scale)


@pytest.mark.parametrize("kvkind", ["f16", "bf16"])
@pytest.mark.parametrize("q,k,scale", [
    ([1.0, 1e-9, 0.5], [1.0, -np.inf, 1.0], 0.5),     # too small for a 16-bit part, and its key is infinite: -inf, not NaN
    ([1.0, 1e-41, 0.5], [1.0, -np.inf, 1.0], 0.5),
    ([1e30, -1e-9, 0.5], [1.0, np.inf, 1.0], 1e-30),
    ([3.4e38, 0.0, 0.0], [-1e-30, 0.0, 0.0], 1e-38),  # above the largest bfloat16 number
    ([np.finfo(np.float32).max, 0.0, 0.0], [-1e-5, 0.0, 0.0], 1e-38),
    ([1e-3, 0.0, 0.0], [-65504.0, 0.0, 0.0], 0.1)])
def test_parts_of_queries_beside_infinities_and_at_the_ends(emel, kern, kvkind, q, k, scale):
    """One row of few products: off by (16 + 16) 2^-23 of its values, and by (3 + 16) 2^-23 of scores up to 1 twice."""
    ctx, d, page = kern.ctx, 16, 8
    qq, kk = np.zeros((1, 1, d)), np.zeros((1, page, 1, d))
    qq[0, 0, :3] = q
    kk[0, :, 0, :3] = [0.25 if x > 0 else 0.0 for x in q]
    kk[0, 3, 0, :3] = k
    qd, kd = dh.Dev(emel, ctx, qq, "f32"), dh.Dev(emel, ctx, kk, kvkind)
    vd = dh.Dev(emel, ctx, np.random.default_rng(1).standard_normal(kk.shape), kvkind)
    table, lengths, out = dh.Dev(emel, ctx, [[0]], "i32"), dh.Dev(emel, ctx, [page], "i32"), dh.Dev(emel, ctx, qq, "f32")
    assert kern.process_event(emel.OpPagedAttn(qd.c(), kd.c(), vd.c(), table.c(), lengths.c(), out.c(), scale)) == 0
    s = np.array([sum(a * b for a, b in zip(qd.values[0, 0], row) if a and b) for row in kd.values[0, :, 0]]) * scale
    p = np.exp(s - s.max())
    want = p @ vd.values[0, :, 0] / p.sum()
    most = np.abs(s[np.isfinite(s)]).max()
    assert np.abs(out.read()[0, 0] - want).max() <= np.abs(vd.values).max() * 2.0 ** -23 * (32 + 2 * 19 * most)


@pytest.mark.parametrize("kvkind", ["f16", "bf16"])
def test_infinite_queries(emel, kern, kvkind):
    """Every score is -inf, whatever large numbers stand beside the infinity: zeros."""
    ctx = kern.ctx
    q = np.zeros((1, 1, 16))
    q[0, 0, :3] = [np.inf, 1e6, -1e6]
    k = np.zeros((1, 8, 1, 16))
    k[..., :3] = [-0.5, 1.0, 1.0]
    k[..., 3:] = 1.0
    qd, kd, vd = dh.Dev(emel, ctx, q, "f32"), dh.Dev(emel, ctx, k, kvkind), dh.Dev(emel, ctx, k, kvkind)
    table, lengths, out = dh.Dev(emel, ctx, [[0]], "i32"), dh.Dev(emel, ctx, [8], "i32"), dh.Dev(emel, ctx, q + 7.0, "f32")
    assert kern.process_event(emel.OpPagedAttn(qd.c(), kd.c(), vd.c(), table.c(), lengths.c(), out.c())) == 0
    assert (out.read() == 0).all()


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("kvh,rep,d", [(2, 1, 8), (1, 4, 16), (1, 9, 8), (1, 17, 16)])
def test_16_bit_queries_round_only_the_result(emel, kern, kind, kvh, rep, d):
    """Before its rounding the result is within the binary32 bar (a score moves by (d + 16) 2^-23 S, sums over n
    tokens by (n + 16) 2^-23) and 2^-17 for weights in two parts: no room for 16-bit weights.  Rounding is
    monotone, so the result lies between the rounded ends."""
    q, k, v, table, lengths, out = setup(emel, kern.ctx, rep, [16] * 40 + [5, 30], kvh, rep, d, 7, kind, kind)
    assert kern.process_event(emel.OpPagedAttn(q.c(), k.c(), v.c(), table.c(), lengths.c(), out.c())) == 0
    got = out.read()
    want = dh.attention(q.values, k.values, v.values, table.values, lengths.values, 1 / np.sqrt(d))
    for b, n in enumerate(lengths.values):
        where = table.values[b, np.arange(n) // 7], np.arange(n) % 7
        for h in range(kvh * rep):
            s = (np.abs(k.values[where][:, h // rep]) @ np.abs(q.values[b, h])).max() / np.sqrt(d)
            tol = np.abs(v.values[where][:, h // rep]).max() * (2 * (d + 16) * 2.0 ** -23 * s + (n + 16) * 2.0 ** -23 + 2.0 ** -17)
            lo, hi = (dh.store(want[b, h] + e, kind)[1] for e in (-tol, tol))
            assert ((lo <= got[b, h]) & (got[b, h] <= hi)).all(), (b, h)


def test_padding_of_the_destination_is_not_written(emel, kern):
    devs = setup(emel, kern.ctx, 12, [40, 3], 2, 2, 40, 16, pad=5, skip=3)
    check(emel, kern, devs)
    out = devs[5]
    touched = np.zeros(out.host.shape, bool)
    np.lib.stride_tricks.as_strided(touched[out.skip:], out.shape, list(out.strides))[...] = True
    assert (out.raw()[~touched] == 9.0).all()


def test_pages_outside_the_cache_are_rejected(emel, kern):
    q, k, v, table, lengths, out = setup(emel, kern.ctx, 13, [100, 50], 1, 2, 64, 16)
    t = table.values.copy()
    keep = np.arange(100)
    keep = keep[(keep // 16 != 2) & (keep // 16 != 4)]
    t[0, 2], t[0, 4] = k.shape[0], -1
    bad = dh.Dev(emel, kern.ctx, t, "i32")
    quiet = emel.Kernel(ctx=kern.ctx)
    assert quiet.process_event(emel.OpPagedAttn(q.c(), k.c(), v.c(), bad.c(), lengths.c(), out.c())) == 0
    assert kern.ctx._lib.emel_cuda_stream_synchronize(kern.ctx.handle, None) == 9  # INDEX_OUT_OF_BOUNDS, once
    kern.ctx.synchronize()
    got = out.read()
    where = table.values[0, keep // 16], keep % 16
    for h in range(2):
        s = k.values[where][:, 0] @ q.values[0, h] / 8
        p = np.exp(s - s.max())
        assert np.abs(got[0, h] - p @ v.values[where][:, 0] / p.sum()).max() < 1e-5
    want = dh.attention(q.values, k.values, v.values, table.values, lengths.values, 1 / 8)
    assert np.abs(got[1] - want[1]).max() < 1e-5
    check(emel, kern, (q, k, v, table, lengths, out))  # nothing of the rejected call is left


@pytest.mark.parametrize("page", [-1, -2, -3, 1 << 20, 2 ** 31 - 1, -2 ** 31])
@pytest.mark.parametrize("pad", [0, 1])
def test_every_page_number_outside_the_cache_is_reported(emel, kern, page, pad):
    q, k, v, table, lengths, out = setup(emel, kern.ctx, 13, [100, 50], 1, 2, 64, 16, pad=pad)
    t = table.values.copy()
    t[0, 2] = page
    bad = dh.Dev(emel, kern.ctx, t, "i32")
    quiet = emel.Kernel(ctx=kern.ctx)
    assert quiet.process_event(emel.OpPagedAttn(q.c(), k.c(), v.c(), bad.c(), lengths.c(), out.c())) == 0
    assert kern.ctx._lib.emel_cuda_stream_synchronize(kern.ctx.handle, None) == 9


def test_lengths_outside_the_table_are_rejected(emel, kern):
    q, k, v, table, lengths, out = setup(emel, kern.ctx, 14, [32, 20], 1, 2, 64, 16)
    far = dh.Dev(emel, kern.ctx, [33, -5], "i32")
    quiet = emel.Kernel(ctx=kern.ctx)
    assert quiet.process_event(emel.OpPagedAttn(q.c(), k.c(), v.c(), table.c(), far.c(), out.c())) == 0
    assert kern.ctx._lib.emel_cuda_stream_synchronize(kern.ctx.handle, None) == 9
    got = out.read()
    want = dh.attention(q.values, k.values, v.values, table.values, [32, 0], 1 / 8)
    assert np.abs(got - want).max() < 1e-5


def test_negative_lengths_are_empty_sequences(emel, kern):
    """They give zeros and nothing to report: a padded row of a captured step beside the append's negative position."""
    q, k, v, table, lengths, out = setup(emel, kern.ctx, 14, [32, 20, 7], 1, 2, 64, 16)
    below = dh.Dev(emel, kern.ctx, [32, -5, -2 ** 31], "i32")
    check(emel, kern, (q, k, v, table, below, out))
    assert kern.ctx._lib.emel_cuda_stream_synchronize(kern.ctx.handle, None) == 0
    assert (out.read()[1:] == 0).all()


def test_replay_reads_new_lengths_and_the_same_inputs_give_the_same_bits(emel, kern):
    ctx = kern.ctx
    stream = emel.Stream(ctx)
    q, k, v, table, lengths, out = setup(emel, ctx, 15, [3000, 700, 1, 0], 2, 4, 128, 16, "f16", "f16")
    on = emel.Kernel(ctx=ctx, stream=stream.handle)
    event = emel.OpPagedAttn(q.c(), k.c(), v.c(), table.c(), lengths.c(), out.c())
    with emel.Graph(ctx, stream) as graph:
        assert on.process_event(event) == 0
    seen = []
    for n in ([3000, 700, 1, 0], [17, 0, 1, 0], [2999, 64, 0, 0], [3000, 700, 1, 0]):
        lengths.buf.upload(np.array(n, np.int32))
        graph.launch()
        stream.synchronize()
        got = out.read()
        want = dh.attention(q.values, k.values, v.values, table.values, n, 1 / np.sqrt(128))
        assert np.abs(got - want).max() < 6 * 2.0 ** -11
        seen.append(out.raw().copy())
    assert (seen[0] == seen[3]).all()
    for _ in range(20):  # the joined pieces keep their order
        graph.launch()
    stream.synchronize()
    assert (out.raw() == seen[0]).all()
    graph.close()
    stream.close()


def test_back_to_back_calls_share_the_workspace(emel, kern):
    """Calls of other shapes queued on one stream without a wait in between."""
    quiet = emel.Kernel(ctx=kern.ctx)
    sets = [setup(emel, kern.ctx, 20 + i, n, kvh, rep, d, 16) for i, (n, kvh, rep, d) in enumerate(
        [([9000], 1, 4, 64), ([5, 4000, 9], 2, 2, 128), ([1], 8, 4, 128), ([2000] * 9, 1, 8, 256)])]
    for _ in range(3):
        for q, k, v, table, lengths, out in sets:
            assert quiet.process_event(emel.OpPagedAttn(q.c(), k.c(), v.c(), table.c(), lengths.c(), out.c())) == 0
    kern.ctx.synchronize()
    for q, k, v, table, lengths, out in sets:
        want = dh.attention(q.values, k.values, v.values, table.values, lengths.values, 1 / np.sqrt(q.shape[2]))
        tol = bar(q.values, k.values, v.values, table.values, lengths.values, 1 / np.sqrt(q.shape[2]), 0, want, "f32", "f16")
        assert (np.abs(out.read() - want) <= tol).all()


def test_cache_beyond_32_bits(emel, kern):
    """Pages whose bytes lie past 4 GiB and whose elements lie past 2^31, with a wide page stride."""
    ctx = kern.ctx
    page, kvh, d, far = 16, 1, 64, 300
    step = 16 * 1024 * 1024  # bytes from page to page
    pages = far + 1
    buf = [emel.DeviceBuffer(ctx, pages * step) for _ in range(2)]
    rng = np.random.default_rng(1)
    table = np.array([[0, 299, 150], [300, 7, 290]])
    lengths = np.array([48, 40])
    q = dh.Dev(emel, ctx, rng.standard_normal((2, 2, d)), "f32")
    out = dh.Dev(emel, ctx, np.zeros((2, 2, d)), "f32")
    new = [dh.Dev(emel, ctx, rng.standard_normal((88, kvh, d)), "f32") for _ in range(2)]
    seq = np.repeat([0, 1], lengths)
    pos = np.concatenate([np.arange(n) for n in lengths])
    views = []
    for b in buf:
        v = emel.CView()
        v.data, v.storage_bytes, v.dtype = b.ptr, pages * step, 1
        for i, (ne, nb) in enumerate(zip((d, kvh, page, pages), (2, 2 * d, 2 * d * kvh, step))):
            v.ne[i], v.nb[i] = ne, nb
        views.append(v)
    t, n = dh.Dev(emel, ctx, table, "i32"), dh.Dev(emel, ctx, lengths, "i32")
    s, at = dh.Dev(emel, ctx, seq, "i32"), dh.Dev(emel, ctx, pos, "i32")
    assert kern.process_event(emel.OpPagedKvAppend(new[0].c(), new[1].c(), t.c(), s.c(), at.c(), *views)) == 0
    assert kern.process_event(emel.OpPagedAttn(q.c(), *views, t.c(), n.c(), out.c())) == 0
    got = out.read()
    for b in range(2):
        k, v = (x.values[seq == b][:, 0].astype(np.float16).astype(np.float64) for x in new)
        for h in range(2):
            p = np.exp(k @ q.values[b, h] / 8 - (k @ q.values[b, h] / 8).max())
            assert np.abs(got[b, h] - p @ v / p.sum()).max() < 1e-5
    for b in buf:
        b.free()


@pytest.mark.parametrize("src,kind", [("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("layout", ["token", "head"])
@pytest.mark.parametrize("kvh,d,page,pad,skip", [(8, 128, 16, 0, 0), (1, 1, 1, 0, 0), (3, 33, 7, 0, 0), (2, 64, 16, 8, 8),
                                                 (2, 40, 5, 4, 2), (4, 80, 100, 1, 1), (1, 256, 64, 0, 0)])
def test_append(emel, kern, src, kind, layout, kvh, d, page, pad, skip):
    rng = np.random.default_rng(d + page)
    past, counts = np.array([0, 3, 40, page, 1]), np.array([1, 70, 1, 5, 30])
    need = -(-(past + counts) // page)
    pages = int(need.sum()) + 1
    pool, table, at = rng.permutation(pages), np.full((5, int(need.max()) + 1), -1), 0
    for b in range(5):
        table[b, :need[b]] = pool[at: at + need[b]]
        at += need[b]
    seq = np.repeat(np.arange(5), counts)
    pos = np.concatenate([past[b] + np.arange(counts[b]) for b in range(5)])
    pos[[2, 50]] = -1  # padding rows
    mix = rng.permutation(seq.size)
    seq, pos = seq[mix], pos[mix]
    size = np.array([1.0, 1e-6, 1e5, 1e39, np.inf, np.nan, -0.0], np.float32)
    with np.errstate(over="ignore", invalid="ignore"):
        vals = [rng.standard_normal((seq.size, kvh, d)).astype(np.float32) *
                rng.choice(size, (seq.size, kvh, d), p=[.8, .1, .05, .02, .01, .01, .01]) for _ in range(2)]
        key, value = (dh.Dev(emel, kern.ctx, x, src, pad=pad, skip=skip) for x in vals)
        order = (0, 1, 2, 3) if layout == "token" else (0, 2, 1, 3)
        kc, vc = (dh.Dev(emel, kern.ctx, rng.standard_normal((pages, page, kvh, d)), kind, order=order, pad=pad, skip=skip,
                         fill=5.0) for _ in range(2))
        t, s, p = (dh.Dev(emel, kern.ctx, x, "i32") for x in (table, seq, pos))
        want = []
        for new, c in ((key, kc), (value, vc)):
            ok = pos >= 0
            raw = np.ascontiguousarray(new.spot())[ok] if src == kind else dh.store(new.values[ok], kind)[0]
            c.spot()[table[seq[ok], pos[ok] // page], pos[ok] % page] = raw
            want.append(c.host.copy())
    assert kern.process_event(emel.OpPagedKvAppend(key.c(), value.c(), t.c(), s.c(), p.c(), kc.c(), vc.c())) == 0
    for c, w in zip((kc, vc), want):
        got = c.raw()
        same = got == w if got.dtype != np.float16 else (got.view(np.uint16) == w.view(np.uint16)) | (np.isnan(got) & np.isnan(w))
        if kind == "bf16":
            same |= (got & 0x7FFF > 0x7F80) & (w & 0x7FFF > 0x7F80)
        assert same.all(), np.argwhere(~same)[:5]


def test_append_one_token_of_every_sequence(emel, kern):
    rng = np.random.default_rng(2)
    table, pos = np.arange(12).reshape(4, 3), np.array([0, 17, 47, 16])
    new = [dh.Dev(emel, kern.ctx, rng.standard_normal((4, 2, 64)), "f16") for _ in range(2)]
    cache = [dh.Dev(emel, kern.ctx, np.zeros((12, 16, 2, 64)), "f16") for _ in range(2)]
    t, p = dh.Dev(emel, kern.ctx, table, "i32"), dh.Dev(emel, kern.ctx, pos, "i32")
    assert kern.process_event(emel.OpPagedKvAppend(new[0].c(), new[1].c(), t.c(), None, p.c(), cache[0].c(), cache[1].c())) == 0
    for n, c in zip(new, cache):
        want = np.zeros((12, 16, 2, 64))
        want[table[np.arange(4), pos // 16], pos % 16] = n.values
        assert (c.read() == want).all()


def test_append_rejects_what_has_no_place(emel, kern):
    rng = np.random.default_rng(4)
    table = np.array([[0, 1], [5, -1]])
    seq, pos = np.array([0, 1, 1, 2, -1, 0, 0]), np.array([1, 2, 17, 0, 0, 32, 20])
    new = [dh.Dev(emel, kern.ctx, rng.standard_normal((7, 1, 8)), "f32") for _ in range(2)]
    cache = [dh.Dev(emel, kern.ctx, np.zeros((5, 16, 1, 8)), "f16") for _ in range(2)]
    t, s, p = (dh.Dev(emel, kern.ctx, x, "i32") for x in (table, seq, pos))
    quiet = emel.Kernel(ctx=kern.ctx)
    assert quiet.process_event(emel.OpPagedKvAppend(new[0].c(), new[1].c(), t.c(), s.c(), p.c(), cache[0].c(), cache[1].c())) == 0
    assert kern.ctx._lib.emel_cuda_stream_synchronize(kern.ctx.handle, None) == 9
    for n, c in zip(new, cache):
        want = np.zeros((5, 16, 1, 8))
        want[0, 1], want[1, 4] = n.values[0].astype(np.float16), n.values[6].astype(np.float16)
        assert (c.read() == want).all()
