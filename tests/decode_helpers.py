"""Plain 64-bit forms and device views for the tests of the decoding-step
operators (paged cache, 4-bit projections, logits)."""

import numpy as np

CODES = {"f32": 0, "f16": 1, "bf16": 30, "i32": 26, "q4_0": 2, "q4_1": 3, "q4_k": 12}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "i32": 4}
BLOCK = {"q4_0": (32, 18), "q4_1": (32, 20), "q4_k": (256, 144)}


def to_bf16(x):
    """float32 -> bfloat16 bits, to nearest even; a NaN stays one."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    r = ((u.astype(np.uint64) + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), ((u >> 16) | 0x40).astype(np.uint16), r)


def store(x, kind):
    """The values of x as they are held in `kind`: (raw array, float64 values)."""
    x = np.asarray(x)
    if kind == "i32":
        return np.ascontiguousarray(x, np.int32), x
    if kind == "bf16":
        raw = to_bf16(x.astype(np.float32))
        return raw, (raw.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    raw = np.ascontiguousarray(x, np.float16 if kind == "f16" else np.float32)
    return raw, raw.astype(np.float64)


def load(raw, kind):
    """float64 values of raw device bytes."""
    return (raw.astype(np.uint32) << 16).view(np.float32).astype(np.float64) if kind == "bf16" else raw.astype(np.float64)


class Dev:
    """A device array of shape `shape` (outermost first).  `order` is the order of its axes in
    memory, `pad` the elements added to the innermost stored row, `skip` the elements before it."""

    def __init__(self, emel, ctx, values, kind, order=None, pad=0, skip=0, fill=None):
        self.emel, self.kind = emel, kind
        raw, self.values = store(values, kind)
        self.shape = raw.shape
        axes = list(order) if order is not None else list(range(raw.ndim))
        inner = [raw.shape[a] for a in axes]
        row = inner[-1] + pad
        count = skip + int(np.prod(inner[:-1], dtype=np.int64)) * row
        self.host = np.full(count, 0 if fill is None else store(np.float32(fill), kind)[0], raw.dtype)
        at, step = [0] * raw.ndim, 1
        for k, a in reversed(list(enumerate(axes))):
            at[a] = step
            step *= row if k == len(axes) - 1 else inner[k]
        self.strides, self.skip = at, skip
        self.spot()[...] = raw
        self.buf = emel.DeviceBuffer(ctx, max(16, self.host.nbytes))
        self.buf.upload(self.host)

    def spot(self):
        size = self.host.itemsize
        return np.lib.stride_tricks.as_strided(self.host[self.skip:], self.shape, [s * size for s in self.strides])

    def c(self, **change):
        v = self.emel.CView()
        size = self.host.itemsize
        v.data = change.get("data", self.buf.ptr + self.skip * size)
        v.storage_bytes = change.get("storage", self.host.nbytes - self.skip * size)
        ne = list(self.shape)[::-1]
        nb = [s * size for s in self.strides][::-1]
        while len(ne) < 4:
            nb.append(nb[-1] * ne[-1])
            ne.append(1)
        ne, nb = change.get("ne", ne), change.get("nb", nb)
        for d in range(4):
            v.ne[d], v.nb[d] = ne[d], nb[d]
        v.dtype = change.get("dtype", CODES[self.kind])
        return v

    def read(self):
        """float64 values now on the device; self.host then holds the raw bytes."""
        self.buf.download(self.host)
        return load(np.ascontiguousarray(self.spot()), self.kind)

    def raw(self):
        self.buf.download(self.host)
        return self.host


def attention(q, k, v, table, lengths, scale, window=0):
    """q [batch, heads, d], k / v [page, token, kv head, d] -> [batch, heads, d], in 64 bits."""
    out = np.zeros_like(q, np.float64)
    page, rep = k.shape[1], q.shape[1] // k.shape[2]
    for b, n in enumerate(lengths):
        n = max(0, min(int(n), table.shape[1] * page))
        at = np.arange(max(0, n - window) if window else 0, n)
        if at.size == 0:
            continue
        where = table[b, at // page]
        kk, vv = k[where, at % page], v[where, at % page]
        for h in range(q.shape[1]):
            s = kk[:, h // rep] @ q[b, h] * scale
            p = np.exp(s - s.max())
            out[b, h] = p @ vv[:, h // rep] / p.sum()
    return out


def q4_random(rng, fmt, rows, k):
    """Rows of packed blocks as bytes [rows, row bytes]: random quants and scales of both signs."""
    values, size = BLOCK[fmt]
    raw = rng.integers(0, 256, (rows, k // values, size), dtype=np.uint8)
    heads = 1 if fmt == "q4_0" else 2
    d = (rng.uniform(0.2, 1.0, (rows, k // values, heads)) * rng.choice([-1.0, 1.0], (rows, k // values, heads)) / 64)
    raw[:, :, : 2 * heads] = d.astype(np.float16).view(np.uint8).reshape(rows, k // values, 2 * heads)
    return raw.reshape(rows, -1)


def q4_values(raw, fmt):
    """The blocks' weights in 64 bits, [rows, k], one value at a time from the format's definition."""
    values, size = BLOCK[fmt]
    rows, n = raw.shape[0], raw.shape[1] // size
    b = raw.reshape(rows, n, size)
    half = lambda at: np.ascontiguousarray(b[:, :, at: at + 2]).view(np.float16)[:, :, 0].astype(np.float64)  # noqa: E731
    w = np.zeros((rows, n, values))
    for i in range(values):
        if fmt == "q4_k":
            j, c = i // 32, b[:, :, 4:16].astype(int)
            s = c[:, :, j] & 63 if j < 4 else (c[:, :, j + 4] & 15) | ((c[:, :, j - 4] >> 6) << 4)
            e = c[:, :, j + 4] & 63 if j < 4 else (c[:, :, j + 4] >> 4) | ((c[:, :, j] >> 6) << 4)
            byte = b[:, :, 16 + 32 * (j // 2) + i % 32]
            q = (byte >> 4 if j % 2 else byte & 15).astype(np.float64)
            w[:, :, i] = half(0) * s * q - half(2) * e
        else:
            byte = b[:, :, size - 16 + i % 16]
            q = (byte & 15 if i < 16 else byte >> 4).astype(np.float64)
            w[:, :, i] = half(0) * (q - 8) if fmt == "q4_0" else half(0) * q + half(2)
    return w.reshape(rows, -1)


def adjusted(x, history=None, used=None, penalties=None, bias=None, allowed=None):
    """The logits' formula in 64 bits; x [rows, vocab], allowed as truth values."""
    x = np.array(x, np.float64)
    for row in range(x.shape[0]):
        if history is not None:
            r, f, p = penalties[row if len(penalties) > 1 else 0]
            ids = [int(t) for t in history[row][: max(0, min(int(used[row]), history.shape[1]))] if 0 <= t < x.shape[1]]
            for t in set(ids):
                v = x[row, t]
                x[row, t] = (v / r if v > 0 else v * r) - ids.count(t) * f - p
        if bias is not None:
            x[row] += bias[row if len(bias) > 1 else 0]
        if allowed is not None:
            x[row][~allowed[row if len(allowed) > 1 else 0]] = -np.inf
    return x
