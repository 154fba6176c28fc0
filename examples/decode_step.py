"""A small decoder that generates tokens for a batch of sequences, on the
device's own operators: 4-bit projections, a paged key/value cache with its
append and attention, and adjusted logits, between the embedding, the norms, the
rotary positions, the gated unit and the argmax.

    python examples/decode_step.py            # on a B200: prints the tokens

Weights are random; the point is how the operators go together:

  * weights are laid out once (Q4Weights), the cache and every buffer are
    allocated once; a step only enqueues events on one stream;
  * sequences own pages, not ranges: a page is taken from a free list when a
    sequence's next token needs one, and the block table names it;
  * lengths and positions are device arrays, so a step can be captured into a
    graph and replayed while the sequences grow.
"""

import sys
from pathlib import Path

import numpy as np

ROOT = Path(__file__).resolve().parent.parent
if str(ROOT) not in sys.path:
    sys.path.insert(0, str(ROOT))

F32, I32 = np.float32, np.int32


class Config:
    def __init__(self, vocab=1000, hidden=256, heads=8, kv_heads=2, head_dim=32, ffn=512, layers=2, page=16, pages=32,
                 capacity=128, window=0, eps=1e-6, rope_base=10000.0):
        self.__dict__.update({k: v for k, v in locals().items() if k != "self"})


def random_q4_0(rng, rows, k):
    """Rows of Q4_0 blocks: binary16 scale, 32 quants."""
    raw = rng.integers(0, 256, (rows, k // 32, 18), dtype=np.uint8)
    d = (rng.uniform(0.5, 1.0, (rows, k // 32)) / (3.0 * np.sqrt(k))).astype(np.float16)
    raw[:, :, :2] = d.view(np.uint8).reshape(rows, k // 32, 2)
    return raw.reshape(rows, -1)


def random_weights(c, seed):
    """Host weights: names to arrays (Q4_0 rows as bytes, the rest binary32)."""
    rng = np.random.default_rng(seed)
    w = {"embed": rng.standard_normal((c.vocab, c.hidden)).astype(F32), "norm": rng.uniform(0.5, 1.5, c.hidden).astype(F32),
         "out": random_q4_0(rng, c.vocab, c.hidden)}
    for i in range(c.layers):
        w[f"{i}.norm1"] = rng.uniform(0.5, 1.5, c.hidden).astype(F32)
        w[f"{i}.norm2"] = rng.uniform(0.5, 1.5, c.hidden).astype(F32)
        for name, rows, k in (("q", c.heads * c.head_dim, c.hidden), ("k", c.kv_heads * c.head_dim, c.hidden),
                              ("v", c.kv_heads * c.head_dim, c.hidden), ("o", c.hidden, c.heads * c.head_dim),
                              ("up", c.ffn, c.hidden), ("gate", c.ffn, c.hidden), ("down", c.hidden, c.ffn)):
            w[f"{i}.{name}"] = random_q4_0(rng, rows, k)
    return w


class Decoder:
    """Greedy decoding of `batch` sequences side by side."""

    def __init__(self, emel, config, weights, batch, stream=None, ctx=None):
        self.emel, self.c, self.batch = emel, config, batch
        c = config
        self.kernel = emel.Kernel(ctx=ctx or emel.Context(0), stream=stream)
        self.ctx, self.stream = self.kernel.ctx, stream
        self.buffers = {}
        self.q4 = {}
        for name, a in weights.items():
            if a.dtype == np.uint8:
                rows, row = a.shape
                buf = emel.DeviceBuffer(self.ctx, a.nbytes)
                buf.upload(a, stream)
                layout = emel.Layout.new(emel.DType.Q4_0, [row // 18 * 32, rows, 1, 1], [1, row, row * rows, row * rows])
                self.q4[name] = emel.Q4Weights(self.ctx, emel.TensorView(buf.ptr, a.nbytes, layout), stream)
                self.ctx.synchronize(stream)
                buf.free()  # the packed form is all that is needed from here on
            else:
                self.put(name, a)
        b, hd = batch, c.head_dim
        for name, n in (("x", c.hidden), ("h", c.hidden), ("q", c.heads * hd), ("k", c.kv_heads * hd), ("v", c.kv_heads * hd),
                        ("a", c.heads * hd), ("ffn", 2 * c.ffn), ("g", c.ffn), ("logits", c.vocab), ("adjusted", c.vocab)):
            self.put(name, np.zeros(n * b, F32))
        for i in range(c.layers):
            for kv in "kv":
                self.put(f"cache.{kv}{i}", np.zeros(c.pages * c.page * c.kv_heads * hd, np.float16))
        self.columns = -(-c.capacity // c.page)
        self.table = np.full((b, self.columns), -1, I32)
        self.free_pages = list(range(c.pages))[::-1]
        self.lengths = np.zeros(b, I32)
        self.history = np.full((b, c.capacity), -1, I32)
        for name, a in (("table", self.table), ("lengths", self.lengths), ("positions", np.zeros(b, I32)),
                        ("tokens", np.zeros(b, I32)), ("history", self.history), ("used", np.zeros(b, I32)),
                        ("penalties", np.tile(np.array([1.0, 0.0, 0.0], F32), (b, 1))),
                        ("allowed", np.full((c.vocab + 31) // 32, -1, I32))):
            self.put(name, a)

    # -- device arrays ------------------------------------------------------
    def put(self, name, a):
        a = np.ascontiguousarray(a)
        if name not in self.buffers:
            self.buffers[name] = self.emel.DeviceBuffer(self.ctx, max(16, a.nbytes))
        self.buffers[name].upload(a, self.stream)

    def view(self, name, ne, dtype="F32", offset=0):
        e = self.emel
        dt = getattr(e.DType, dtype)
        layout = e.Layout.contiguous(dt, list(ne) + [1] * (4 - len(ne)))
        buf = self.buffers[name]
        return e.TensorView(buf.ptr + offset, buf.nbytes - offset, layout)

    def cache(self, kv, layer):
        c = self.c
        return self.view(f"cache.{kv}{layer}", [c.head_dim, c.kv_heads, c.page, c.pages], "F16")

    def run(self, event):
        status = self.kernel.process_event(event)
        if status != self.emel.Status.OK:
            raise RuntimeError(f"{type(event).__name__}: {status.name} ({self.ctx.last_error})")

    # -- one step -----------------------------------------------------------
    def beginning(self):
        """The sequences whose next token begins a page; raises, with nothing changed, when it has no place."""
        c = self.c
        if int(self.lengths.max()) >= c.capacity:
            raise RuntimeError("a sequence has reached the capacity of its table")
        begin = np.flatnonzero(self.lengths % c.page == 0)
        if len(begin) > len(self.free_pages):
            raise RuntimeError("the cache has no free page")
        return begin

    def reserve(self, begin):
        """Counts one more token for every sequence, and gives a page to those that begin one."""
        for b in begin:
            self.table[b, self.lengths[b] // self.c.page] = self.free_pages.pop()
        self.put("positions", self.lengths)
        self.lengths += 1
        self.put("lengths", self.lengths)
        self.put("table", self.table)

    def enqueue(self):
        """The events of one step: tokens in, the next tokens out in the same buffer."""
        e, c, b, hd = self.emel, self.c, self.batch, self.c.head_dim
        x, h = self.view("x", [c.hidden, b]), self.view("h", [c.hidden, b])
        norm = lambda name: self.view(name, [c.hidden])  # noqa: E731
        rope = {"n_dims": hd, "mode": 2, "freq_base": c.rope_base, "freq_scale": 1.0, "ext_factor": 0.0, "attn_factor": 1.0}
        positions = self.view("positions", [b], "I32")
        self.run(e.OpGetRows(self.view("embed", [c.hidden, c.vocab]), self.view("tokens", [b], "I32"), x))
        for i in range(c.layers):
            self.run(e.OpRmsNormMul(x, norm(f"{i}.norm1"), h, c.eps))
            for name, heads in (("q", c.heads), ("k", c.kv_heads), ("v", c.kv_heads)):
                self.run(e.OpMulMatQ4(self.q4[f"{i}.{name}"], h, self.view(name, [heads * hd, b])))
            for name, heads in (("q", c.heads), ("k", c.kv_heads)):
                rows = self.view(name, [hd, heads, b])
                self.run(e.OpRope(rows, positions, rows, rope))
            self.run(e.OpPagedKvAppend(self.view("k", [hd, c.kv_heads, b]), self.view("v", [hd, c.kv_heads, b]),
                                       self.view("table", [self.columns, b], "I32"), None, positions,
                                       self.cache("k", i), self.cache("v", i)))
            self.run(e.OpPagedAttn(self.view("q", [hd, c.heads, b]), self.cache("k", i), self.cache("v", i),
                                   self.view("table", [self.columns, b], "I32"), self.view("lengths", [b], "I32"),
                                   self.view("a", [hd, c.heads, b]), window=c.window))
            self.run(e.OpMulMatQ4(self.q4[f"{i}.o"], self.view("a", [c.heads * hd, b]), h))
            self.run(e.OpAdd(x, h, x))
            self.run(e.OpRmsNormMul(x, norm(f"{i}.norm2"), h, c.eps))
            half = c.ffn * b * 4
            self.run(e.OpMulMatQ4(self.q4[f"{i}.up"], h, self.view("ffn", [c.ffn, b])))
            self.run(e.OpMulMatQ4(self.q4[f"{i}.gate"], h, self.view("ffn", [c.ffn, b], offset=half)))
            self.run(e.OpGlu((self.buffers["ffn"].ptr, 2 * c.ffn * b), (self.buffers["g"].ptr, c.ffn * b), e.GluSubOp.SWIGLU))
            self.run(e.OpMulMatQ4(self.q4[f"{i}.down"], self.view("g", [c.ffn, b]), h))
            self.run(e.OpAdd(x, h, x))
        self.run(e.OpRmsNormMul(x, norm("norm"), h, c.eps))
        logits, adjusted = self.view("logits", [c.vocab, b]), self.view("adjusted", [c.vocab, b])
        self.run(e.OpMulMatQ4(self.q4["out"], h, logits))
        self.run(e.OpLogitsAdjust(logits, adjusted, self.view("history", [c.capacity, b], "I32"), self.view("used", [b], "I32"),
                                  self.view("penalties", [3, b]), None, self.view("allowed", [(c.vocab + 31) // 32, 1], "I32")))
        self.run(e.OpArgmaxRows(adjusted, self.view("tokens", [1, b], "I32")))

    def remember(self, tokens):
        """Puts the tokens that a step is about to read into the histories."""
        self.history[np.arange(self.batch), self.lengths] = tokens
        self.put("history", self.history)
        self.put("used", self.lengths + 1)

    def step(self, tokens, graph=None):
        """Feeds one token per sequence; returns the tokens chosen next."""
        tokens = np.ascontiguousarray(tokens, I32)
        begin = self.beginning()
        self.remember(tokens)
        self.reserve(begin)
        self.put("tokens", tokens)
        if graph is None:
            self.enqueue()
        else:
            graph.launch()
        self.ctx.synchronize(self.stream)
        return self.buffers["tokens"].download(np.empty(self.batch, I32), self.stream)

    def adjusted_logits(self):
        return self.buffers["adjusted"].download(np.empty((self.batch, self.c.vocab), F32), self.stream)


def main():
    from __graft_entry__ import load_package
    emel = load_package()
    config = Config()
    ctx = emel.Context(0)
    stream = emel.Stream(ctx)
    model = Decoder(emel, config, random_weights(config, 1), batch=3, stream=stream.handle, ctx=ctx)
    model.put("penalties", np.tile(np.array([1.2, 0.1, 0.2], F32), (3, 1)))
    with emel.Graph(ctx, stream) as graph:  # recorded once; every step replays it
        model.enqueue()
    tokens, said = np.array([1, 2, 3], I32), []
    for _ in range(24):
        tokens = model.step(tokens, graph)
        said.append(tokens)
    for b, row in enumerate(np.array(said).T):
        print(f"sequence {b}:", " ".join(str(t) for t in row))
    graph.close()


if __name__ == "__main__":
    main()
