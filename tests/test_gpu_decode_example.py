"""examples/decode_step.py, its operators together, against the same decoder
in 64 bits: logits of every step, eagerly and as a replayed graph, across page
ends, with penalties, a mask and a sliding window.

The reference rounds only what the device keeps in binary16 (cached keys and
values).  A layer's binary32 operators are each within about 1e-6 of their inputs'
scale, and a cached value that falls on the other side of a binary16 rounding
boundary is off by 2^-11 of itself for one token among many: logits, of unit
size, are held to 5e-3."""

import sys
from pathlib import Path

import numpy as np
import pytest

import decode_helpers as dh

pytestmark = pytest.mark.gpu
sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "examples"))


class Plain:
    def __init__(self, c, weights, batch):
        self.c, self.batch = c, batch
        self.w = {n: dh.q4_values(a, "q4_0") if a.dtype == np.uint8 else a.astype(np.float64) for n, a in weights.items()}
        self.k = [[[] for _ in range(batch)] for _ in range(c.layers)]
        self.v = [[[] for _ in range(batch)] for _ in range(c.layers)]

    def norm(self, x, name):
        return x / np.sqrt((x * x).mean(-1, keepdims=True) + self.c.eps) * self.w[name]

    def rope(self, x, pos):
        half = self.c.head_dim // 2
        angle = pos * self.c.rope_base ** (-np.arange(half) / half)
        a, b = x[:, :half], x[:, half:]
        return np.concatenate([a * np.cos(angle) - b * np.sin(angle), a * np.sin(angle) + b * np.cos(angle)], 1)

    def step(self, tokens):
        c = self.c
        out = np.zeros((self.batch, c.vocab))
        for b, token in enumerate(tokens):
            x = self.w["embed"][token]
            for i in range(c.layers):
                h = self.norm(x, f"{i}.norm1")
                q, k, v = ((self.w[f"{i}.{n}"] @ h).reshape(-1, c.head_dim) for n in "qkv")
                pos = len(self.k[i][b])
                q, k = self.rope(q, pos), self.rope(k, pos)
                self.k[i][b].append(k.astype(np.float32).astype(np.float16).astype(np.float64))
                self.v[i][b].append(v.astype(np.float32).astype(np.float16).astype(np.float64))
                keys, values = np.array(self.k[i][b]), np.array(self.v[i][b])
                if c.window:
                    keys, values = keys[-c.window:], values[-c.window:]
                a = np.zeros_like(q)
                for n in range(c.heads):
                    s = keys[:, n * c.kv_heads // c.heads] @ q[n] / np.sqrt(c.head_dim)
                    p = np.exp(s - s.max())
                    a[n] = p @ values[:, n * c.kv_heads // c.heads] / p.sum()
                x = x + self.w[f"{i}.o"] @ a.reshape(-1)
                h = self.norm(x, f"{i}.norm2")
                gate = self.w[f"{i}.gate"] @ h
                x = x + self.w[f"{i}.down"] @ ((self.w[f"{i}.up"] @ h) * gate / (1 + np.exp(-gate)))
            out[b] = self.w["out"] @ self.norm(x, "norm")
        return out


@pytest.mark.parametrize("replay", [False, True])
@pytest.mark.parametrize("window", [0, 20])
def test_decoder_follows_the_plain_one(emel, replay, window):
    import decode_step as ex
    c = ex.Config(vocab=777, window=window)
    weights = ex.random_weights(c, 5)
    ctx = emel.Context(0)
    stream = emel.Stream(ctx)
    batch = 3
    model, plain = ex.Decoder(emel, c, weights, batch, stream.handle, ctx), Plain(c, weights, batch)
    pen = np.array([[1.3, 0.2, 0.1], [1.0, 0.0, 0.0], [0.9, 0.05, 0.3]], np.float32)
    model.put("penalties", pen)
    allowed = np.ones(c.vocab, bool)
    allowed[np.arange(0, c.vocab, 7)] = False
    bits = np.zeros((c.vocab + 31) // 32 * 32, bool)
    bits[:c.vocab] = allowed
    model.put("allowed", np.packbits(bits, bitorder="little").view(np.int32))
    graph = None
    if replay:
        with emel.Graph(ctx, stream) as graph:
            model.enqueue()
    tokens = np.array([1, 500, 3], np.int32)
    seen = [[] for _ in range(batch)]
    for _ in range(40):
        for b in range(batch):
            seen[b].append(int(tokens[b]))
        want = dh.adjusted(plain.step(tokens), np.array(seen), [len(s) for s in seen], pen.astype(np.float64), None, allowed[None])
        chosen = model.step(tokens, graph)
        got = model.adjusted_logits().astype(np.float64)
        assert np.isneginf(got[:, ~allowed]).all()
        assert np.abs(got[:, allowed] - want[:, allowed]).max() < 5e-3
        assert (chosen == got.argmax(1)).all()
        tokens = chosen
    assert sorted(model.free_pages + list(model.table[model.table >= 0])) == list(range(c.pages))
    if graph is not None:
        graph.close()


def test_the_example_runs(emel, capsys):
    import decode_step as ex
    ex.main()
    assert capsys.readouterr().out.count("sequence") == 3


def test_a_cache_without_pages_says_so(emel):
    import decode_step as ex
    c = ex.Config(pages=2)
    model = ex.Decoder(emel, c, ex.random_weights(c, 2), 2)
    for _ in range(16):
        model.step(np.zeros(2, np.int32))
    with pytest.raises(RuntimeError, match="no free page"):
        model.step(np.zeros(2, np.int32))


def state(model):
    return [x.copy() for x in (model.table, model.lengths, model.history)] + [sorted(model.free_pages)]


def test_a_refused_step_changes_nothing_and_loses_no_page(emel):
    import decode_step as ex
    c = ex.Config(pages=3)
    model = ex.Decoder(emel, c, ex.random_weights(c, 2), 2)
    for _ in range(16):
        model.step(np.zeros(2, np.int32))
    before = state(model)
    for _ in range(2):  # two pages are needed, one is free
        with pytest.raises(RuntimeError, match="no free page"):
            model.step(np.ones(2, np.int32))
        assert all(np.array_equal(a, b) for a, b in zip(before, state(model)))
    model.free_pages.append(int(model.table[0, 0]))  # the first sequence ends, another takes its place
    model.table[0], model.lengths[0] = -1, 0
    model.step(np.ones(2, np.int32))
    assert sorted(model.free_pages + list(model.table[model.table >= 0])) == [0, 1, 2]


def test_a_full_table_says_so(emel):
    import decode_step as ex
    c = ex.Config(capacity=32)
    model = ex.Decoder(emel, c, ex.random_weights(c, 2), 2)
    for _ in range(32):
        model.step(np.zeros(2, np.int32))
    before = state(model)
    with pytest.raises(RuntimeError, match="capacity"):
        model.step(np.zeros(2, np.int32))
    assert all(np.array_equal(a, b) for a, b in zip(before, state(model)))


def test_a_capacity_that_ends_inside_a_page(emel):
    import decode_step as ex
    c = ex.Config(capacity=20)
    model = ex.Decoder(emel, c, ex.random_weights(c, 2), 2)
    for _ in range(20):
        model.step(np.zeros(2, np.int32))
    with pytest.raises(RuntimeError, match="capacity"):
        model.step(np.zeros(2, np.int32))
