"""Precision of the decoding-step operators where it rests on the lower parts of a split number: inputs
whose leading parts cancel or meet zeros, so that a lost part shows.  Each test also takes the same
answer without the part and asks that it misses the bar."""

import numpy as np
import pytest

import decode_helpers as dh
from test_gpu_paged import setup
from test_gpu_q4 import Blocks

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -23


@pytest.fixture(scope="module")
def kern(emel):
    return emel.Kernel(device=0, synchronize=True)


def part(x, kind):
    """The 16-bit number nearest to x."""
    return dh.store(np.asarray(x, np.float32), kind)[1]


def parts(x, kind, n):
    """The sum of the n leading 16-bit parts of x."""
    total = np.zeros_like(x)
    for _ in range(n):
        total = total + part(x - total, kind)
    return total


def attend(emel, kern, q, k, v, kind, scale):
    """q [batch, heads, d], k / v [batch, tokens, d]: a page for each sequence."""
    qd = dh.Dev(emel, kern.ctx, q, "f32")
    kd, vd = (dh.Dev(emel, kern.ctx, x[:, :, None], kind) for x in (k, v))
    table = dh.Dev(emel, kern.ctx, np.arange(len(q))[:, None], "i32")
    lengths = dh.Dev(emel, kern.ctx, np.full(len(q), k.shape[1]), "i32")
    out = dh.Dev(emel, kern.ctx, np.zeros(q.shape), "f32")
    assert kern.process_event(emel.OpPagedAttn(qd.c(), kd.c(), vd.c(), table.c(), lengths.c(), out.c(), scale)) == 0
    return out.read(), lambda q: dh.attention(q, kd.values, vd.values, table.values, lengths.values, scale)


@pytest.mark.parametrize("kind,kept", [("f16", 1), ("bf16", 1), ("bf16", 2)])
@pytest.mark.parametrize("heads", [1, 8, 11])
def test_lower_parts_of_the_query(emel, kern, kind, kept, heads):
    """Columns a and b = the leading parts of a, against keys K and -K, powers of two: a score is K (a - b), in
    each part a sum without rounding.  Two binary16 parts leave 2^-12 of a - b (22 bits of a), three bfloat16
    parts nothing; the rest of the bar is that of binary32 scores, weights and sums over T tokens."""
    rng = np.random.default_rng(heads)
    tokens, half = 48, 8
    a = rng.uniform(1, 2, (4, heads, half)).astype(np.float32).astype(np.float64)
    b = parts(a, kind, kept)
    q = np.concatenate([a, b], 2)
    size = 2.0 ** (10 if kind == "f16" else 7 if kept == 1 else 15)
    key = size * rng.choice([-1.0, 0.5, 1.0], (4, tokens, half))
    k, v = np.concatenate([key, -key], 2), rng.standard_normal((4, tokens, 2 * half))
    got, exact = attend(emel, kern, q, k, v, kind, 1.0)
    s = np.abs(a - b).sum(2).max() * size
    assert 0.2 < s < 20
    lost = s * (2.0 ** -12 if kind == "f16" else 0.0)
    tol = np.abs(v).max() * (2 * (s * 32 * EPS + lost) + (tokens + 16) * EPS)
    assert np.abs(got - exact(q)).max() <= tol
    assert np.abs(exact(np.concatenate([b, b], 2)) - exact(q)).max() > 4 * tol


@pytest.mark.parametrize("kind,kept", [("f16", 1), ("bf16", 1), ("bf16", 2)])
def test_lower_parts_of_the_weights(emel, kern, kind, kept):
    """Two tokens of scores x and 0, values 1 and -1: tanh(x / 2) for small x is what the weights' last bits
    say.  The weights stand near 2^8: the exponential is off by 2^-22, its argument near 8 by 2^-21 ln 2, sums
    and the division by less than 2^-22 together: 2^-20 in all."""
    rng = np.random.default_rng(7)
    x = (2.0 ** rng.uniform(-16, -8, 400)).astype(np.float32).astype(np.float64)
    q, k, v = np.zeros((400, 1, 8)), np.zeros((400, 2, 8)), np.zeros((400, 2, 8))
    q[:, 0, 0], k[:, 0, 0] = x, 1.0
    v[:, 0], v[:, 1] = 1.0, -1.0
    got, exact = attend(emel, kern, q, k, v, kind, 1.0)
    want = np.tanh(x / 2)
    assert np.abs(exact(q)[:, 0, 0] - want).max() < 1e-12
    assert np.abs(got[:, 0] - want[:, None]).max() <= 2.0 ** -20
    w = 256.0 * np.exp(-x)
    short = (256.0 - parts(w, kind, kept)) / (256.0 + w)
    assert np.abs(short - want).max() > 2.0 ** -20


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("tokens", [300, 5000, 20000])
def test_errors_of_binary32_queries_as_a_whole(emel, kern, kind, tokens):
    """Scores of size 1 are rounded once for every 16 columns, to 2^-23 at most, and results of values without a
    mean move by as much of themselves: (128 / 16 + 8) 2^-23 of the results' size, both as roots of mean
    squares, is ample, and 16-bit parts of one less (2^-18 and 2^-12 each way) are beyond it."""
    q, k, v, table, lengths, out = setup(emel, kern.ctx, tokens, [tokens], 1, 8, 128, 64, "f32", kind)
    assert kern.process_event(emel.OpPagedAttn(q.c(), k.c(), v.c(), table.c(), lengths.c(), out.c())) == 0
    rms = lambda x: np.sqrt((x * x).mean())  # noqa: E731
    at = lambda q: dh.attention(q, k.values, v.values, table.values, lengths.values, 1 / np.sqrt(128))  # noqa: E731
    want = at(q.values)
    assert rms(out.read() - want) <= 16 * EPS * rms(want)
    assert rms(at(parts(q.values, kind, 1 if kind == "f16" else 2)) - want) > 16 * EPS * rms(want)


def product(emel, kern, raw, fmt, x, kind="f32"):
    blocks = Blocks(emel, kern.ctx, raw, fmt)  # owns what the view names until the layout has run
    w = emel.Q4Weights(kern.ctx, blocks.c())
    xd, yd = dh.Dev(emel, kern.ctx, x, kind), dh.Dev(emel, kern.ctx, np.zeros((len(x), len(raw))), "f32")
    assert kern.process_event(emel.OpMulMatQ4(w, xd.c(), yd.c())) == 0
    assert (xd.values == x).all()
    return yd.read()


@pytest.mark.parametrize("n", [1, 2])
@pytest.mark.parametrize("k", [512, 2048, 8192])
def test_lowest_digit_of_the_activations(emel, kern, n, k):
    """The column's largest value meets weights of 0; the others, 2^-20 of it, stand in the two lowest digits.
    Each counts to 2^-30 of the largest, and sums are binary32."""
    rng = np.random.default_rng(k + n)
    raw = dh.q4_random(rng, "q4_0", 40, k).reshape(40, -1, 18)
    raw[:, ::16, 2] = raw[:, ::16, 2] & 0xF0 | 8  # weight 0 at every 512th column
    raw = raw.reshape(40, -1)
    x = (rng.standard_normal((n, k)) * 2.0 ** -20).astype(np.float32).astype(np.float64)
    x[:, ::512] = 1.0
    w = dh.q4_values(raw, "q4_0")
    assert (w[:, ::512] == 0).all()
    want = x @ w.T
    tol = np.abs(w).sum(1) * 2.0 ** -30 + (64 + k / 32) * EPS * ((np.abs(x) * (np.abs(x) < 0.5)) @ np.abs(w).T)
    assert (np.abs(product(emel, kern, raw, "q4_0", x) - want) <= tol).all()
    digits = np.rint(x * 2.0 ** 29)
    short = (digits - ((digits + 128) % 256 - 128)) * 2.0 ** -29
    assert (np.abs(short @ w.T - want) > tol).mean() > 0.5


@pytest.mark.parametrize("fmt", ["q4_0", "q4_1"])
@pytest.mark.parametrize("n", [3, 4, 5, 8])
@pytest.mark.parametrize("k", [512, 8192])
def test_second_part_of_the_activations(emel, kern, fmt, n, k):
    """Columns i and i + 16 of a group have one weight, and x there is a and the leading part of -a: the products
    are w (a - b).  Each value counts to 2^-23 of itself; the leading parts' sums are exact and cancel."""
    rng = np.random.default_rng(k + n)
    head = dh.BLOCK[fmt][1] - 16
    raw = dh.q4_random(rng, fmt, 40, k).reshape(40, -1, head + 16)
    raw[:, :, head:] = (raw[:, :, head:] & 15) * 17
    raw = raw.reshape(40, -1)
    a = rng.uniform(1, 2, (n, k // 32, 1, 16)).astype(np.float32).astype(np.float64)
    b = part(a, "f16")
    x = np.concatenate([a, -b], 2).reshape(n, k)
    w = dh.q4_values(raw, fmt)
    want = x @ w.T
    size = np.concatenate([np.abs(a - b), np.abs(a - b)], 2).reshape(n, k)
    most = 17 / 64  # |a (q - 8)| + |c|, with scales and minimums up to 1 / 64
    tol = EPS * (np.abs(x) @ np.abs(w).T) + (64 + k / 32) * EPS * most * size.sum(1)[:, None]
    assert (np.abs(product(emel, kern, raw, fmt, x) - want) <= tol).all()
    assert (np.abs(want) > tol).mean() > 0.5  # what the leading parts alone give is 0
