"""The operators of one decoding step over a paged cache with 4-bit weights, as cases to time.

Four operators, each in its plain form (elementary torch operations in 32
bits) and through this repository's events:

  attn    one new token of every sequence attends over its pages of cached
          keys and values (OpPagedAttn)
  append  new keys and values go into their pages (OpPagedKvAppend)
  q4      a few activation rows times a matrix of 4-bit weights with one
          scale for each group (Q4Weights, OpMulMatQ4)
  logits  penalties for repeated tokens, biases and the mask of the tokens
          that a grammar allows (OpLogitsAdjust)

A case is a dict of plain values whose "op" names the operator.
"""

import importlib.util
import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
Q4_BLOCK = {"q4_0": (32, 18), "q4_1": (32, 20), "q4_k": (256, 144)}  # values and bytes of one block


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------

def _attn(batch, tokens, kv_heads, rep, d, page, q="f32", kv="f16", window=0, ragged=False, layout="token"):
    return {"op": "attn", "batch": batch, "tokens": tokens, "kv_heads": kv_heads, "rep": rep, "d": d, "page": page,
            "q": q, "kv": kv, "window": window, "ragged": ragged, "layout": layout}


def _append(n, sequences, past, kv_heads, d, page, src="f32", kv="f16", layout="token"):
    return {"op": "append", "n": n, "sequences": sequences, "past": past, "kv_heads": kv_heads, "d": d, "page": page,
            "src": src, "kv": kv, "layout": layout}


def _q4(fmt, k, rows, n=1, x="f32"):
    return {"op": "q4", "fmt": fmt, "k": k, "rows": rows, "n": n, "x": x}


def _logits(rows, vocab, history, bias="none", allowed="none", dtype="f32"):
    return {"op": "logits", "rows": rows, "vocab": vocab, "history": history, "bias": bias, "allowed": allowed,
            "dtype": dtype}


def listed():
    return [
        # the first tokens of one conversation: nothing but latency
        {"name": "attn one short", **_attn(1, 17, 8, 4, 128, 16)},
        # one conversation at the length and head shape of this repository's attention workload
        {"name": "attn one 32k", **_attn(1, 32768, 8, 4, 128, 64)},
        # a server's mixed batch, 16-bit activations, short and long sequences side by side
        {"name": "attn ragged batch", **_attn(64, 8191, 8, 4, 128, 16, "bf16", "bf16", ragged=True)},
        # heads of 80 columns in groups of five, pages of 24 tokens stored head by head, a sliding window
        {"name": "attn odd heads", **_attn(24, 5000, 4, 5, 80, 24, "f32", "bf16", window=4000, ragged=True, layout="head")},
        # one token of every sequence of a batch
        {"name": "append step", **_append(64, 64, 4000, 8, 128, 16)},
        # several prompts at once, already in the cache's type
        {"name": "append prompts", **_append(8191, 5, 100, 8, 128, 16, "bf16", "bf16", "head")},
        # a small model's projection for one token
        {"name": "q4 small", **_q4("q4_0", 1024, 1024)},
        # a projection of a large model for one token, super-blocks of 256 with 6-bit scales and minimums
        {"name": "q4 projection", **_q4("q4_k", 4096, 14336)},
        # the vocabulary of this repository's matvec workload, one token
        {"name": "q4 vocabulary", **_q4("q4_0", 4096, 151936)},
        # eight sequences at once, an odd number of rows, scales with a minimum
        {"name": "q4 eight tokens", **_q4("q4_1", 4096, 11007, 8)},
        # one sequence that has generated a short text, plain penalties
        {"name": "logits one", **_logits(1, 32000, 50)},
        # a server's batch over the vocabulary of configuration 4b, everything on
        {"name": "logits batch", **_logits(64, 151936, 4096, "rows", "rows")},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attn", "attn", "append", "q4", "q4", "logits"])
    if op == "attn":
        q, kv = rng.choice([("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")])
        batch, kv_heads = _log(rng, 1, 64), rng.choice([1, 2, 4, 8])
        d = rng.choice([40, 64, 72, 80, 96, 128, 192, 256])
        most = 64 * 8191 * 8 * 128 // 4 // (batch * kv_heads * d)
        tokens = _log(rng, 1, max(1, min(40000, most)))
        window = _log(rng, 1, tokens) if rng.random() < 0.3 else 0
        return _attn(batch, tokens, kv_heads, rng.choice([1, 2, 3, 4, 5, 7, 8, 16]), d, rng.choice([1, 7, 16, 32, 64, 100]),
                     q, kv, window, rng.random() < 0.6, rng.choice(["token", "head"]))
    if op == "append":
        sequences = _log(rng, 1, 64)
        src, kv = rng.choice([("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")])
        return _append(max(sequences, _log(rng, 1, 8191)), sequences, _log(rng, 1, 2000), rng.choice([1, 2, 4, 8]),
                       rng.choice([40, 64, 72, 80, 96, 128]), rng.choice([1, 7, 16, 32, 64, 100]), src, kv,
                       rng.choice(["token", "head"]))
    if op == "q4":
        fmt = rng.choice(["q4_0", "q4_1", "q4_k"])
        group = Q4_BLOCK[fmt][0]
        k = group * max(1, _log(rng, 32, 16384) // group)
        rows = _log(rng, 1, min(151936, 300_000_000 // k))
        return _q4(fmt, k, rows, rng.choice([1, 1, 1, 2, 3, 4, 5, 7, 8, 13]), rng.choice(["f32", "f16"]))
    kinds = ["none", "shared", "rows"]
    return _logits(_log(rng, 1, 64), _log(rng, 500, 151936), rng.choice([0, 1, _log(rng, 2, 4096)]), rng.choice(kinds),
                   rng.choice(kinds), rng.choice(["f32", "f16"]))


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def _spread(case):
    """Lengths of a batch, the same for every seed: half of them few, spread over their logarithm, half over the range."""
    top, batch = case["tokens"], case["batch"]
    if not case["ragged"]:
        return np.full(batch, top, np.int64)
    short = (batch + 1) // 2
    few = np.exp(np.log(top) * (np.arange(short) + 0.5) / short)
    many = top * (np.arange(batch - short) + 1.0) / max(1, batch - short)
    return np.clip(np.concatenate([few, many]).astype(np.int64), 1, top)


def _lengths(case, seed):
    return np.random.default_rng(seed).permutation(_spread(case)).astype(np.int32)


def _used(case):
    """How many ids of each row's history are in use: spread from few to all."""
    return case["history"] * (np.arange(case["rows"]) + 1) // case["rows"]


def _pages(need, page, seed):
    """A block table of one row for each sequence, -1 beyond its pages, over a shuffled pool."""
    rng = np.random.default_rng(seed + 1)
    counts = -(-need // page)
    total = int(need.sum()) // page + len(need) + 3  # a few pages belong to nobody
    pool = rng.permutation(total).astype(np.int32)
    table = np.full((len(need), max(1, int(counts.max()))), -1, np.int32)
    at = np.arange(table.shape[1])[None, :] < counts[:, None]
    table[at] = pool[: int(counts.sum())]
    return table, total


def _cache(pages, case, g):
    """A pool of pages as [page, token, kv head, d], stored in that order or head by head."""
    shape = (pages, case["page"], case["kv_heads"], case["d"])
    if case["layout"] == "head":
        stored = torch.randn((shape[0], shape[2], shape[1], shape[3]), generator=g, device="cuda", dtype=DTYPES[case["kv"]])
        return stored.permute(0, 2, 1, 3)
    return torch.randn(shape, generator=g, device="cuda", dtype=DTYPES[case["kv"]])


def _blocks(case, g):
    """Rows of packed 4-bit blocks as they stand in a model file: random quants, scales of usual size."""
    values, size = Q4_BLOCK[case["fmt"]]
    n = case["rows"] * (case["k"] // values)
    raw = torch.randint(0, 256, (n, size), generator=g, device="cuda", dtype=torch.uint8)
    if case["fmt"] == "q4_k":
        head = torch.rand((n, 2), generator=g, device="cuda") * torch.tensor([2e-4, 1e-3], device="cuda") + 1e-5
    elif case["fmt"] == "q4_1":
        d = torch.rand((n, 1), generator=g, device="cuda") * 0.01 + 1e-3
        head = torch.cat([d, -d * (7 + torch.rand((n, 1), generator=g, device="cuda"))], 1)
    else:
        head = (torch.rand((n, 1), generator=g, device="cuda") * 0.01 + 1e-3) * torch.where(
            torch.rand((n, 1), generator=g, device="cuda") < 0.5, -1.0, 1.0)
    head = head.to(torch.float16).contiguous().view(torch.uint8)
    raw[:, : head.shape[1]] = head
    return raw.view(case["rows"], -1)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = {"case": case}
    if case["op"] == "attn":
        need = _lengths(case, seed)
        table, pages = _pages(need, case["page"], seed)
        s["q"] = torch.randn((case["batch"], case["kv_heads"] * case["rep"], case["d"]), generator=g, device="cuda",
                             dtype=DTYPES[case["q"]])
        s["k"], s["v"] = _cache(pages, case, g), _cache(pages, case, g)
        s["table"], s["lengths"] = torch.from_numpy(table).cuda(), torch.from_numpy(need).cuda()
        if own:
            s["out"] = torch.empty_like(s["q"])
            p = _package()
            s["event"] = p.OpPagedAttn(_view(s["q"]), _view(s["k"]), _view(s["v"]), _view(s["table"]),
                                       _view(s["lengths"]), _view(s["out"]), window=case["window"])
    elif case["op"] == "append":
        rng = np.random.default_rng(seed)
        cut = np.sort(rng.choice(np.arange(1, case["n"]), case["sequences"] - 1, replace=False)) if case["sequences"] > 1 else []
        counts = np.diff(np.concatenate([[0], cut, [case["n"]]])).astype(np.int64)
        past = rng.permutation(case["past"] * np.arange(1, case["sequences"] + 1) // case["sequences"])
        table, pages = _pages(past + counts, case["page"], seed)
        of = np.repeat(np.arange(case["sequences"]), counts)
        first = np.concatenate([[0], np.cumsum(counts)[:-1]])
        at = past[of] + np.arange(case["n"]) - first[of]
        shape = (case["n"], case["kv_heads"], case["d"])
        s["key"] = torch.randn(shape, generator=g, device="cuda", dtype=DTYPES[case["src"]])
        s["value"] = torch.randn(shape, generator=g, device="cuda", dtype=DTYPES[case["src"]])
        s["k"], s["v"] = _cache(pages, case, g), _cache(pages, case, g)
        s["table"] = torch.from_numpy(table).cuda()
        s["sequence"] = torch.from_numpy(of.astype(np.int32)).cuda()
        s["position"] = torch.from_numpy(at.astype(np.int32)).cuda()
        if own:
            p = _package()
            s["event"] = p.OpPagedKvAppend(_view(s["key"]), _view(s["value"]), _view(s["table"]), _view(s["sequence"]),
                                           _view(s["position"]), _view(s["k"]), _view(s["v"]))
    elif case["op"] == "q4":
        s["blocks"] = _blocks(case, g)
        x = torch.randn((case["n"], case["k"]), generator=g, device="cuda")
        x[:, :: 97] *= 20.0  # a few columns of hidden states are far larger than the others
        s["x"] = x.to(DTYPES[case["x"]])
        if own:
            s["out"] = torch.empty((case["n"], case["rows"]), device="cuda")
            p = _package()
            kernel = _kernel()
            s["weights"] = p.Q4Weights(kernel.ctx, _packed_view(case, s["blocks"]), kernel.stream)
            s["event"] = p.OpMulMatQ4(s["weights"], _view(s["x"]), _view(s["out"]))
    else:
        rows, vocab = case["rows"], case["vocab"]
        rng = np.random.default_rng(seed)
        s["logits"] = (torch.randn((rows, vocab), generator=g, device="cuda") * 3.0).to(DTYPES[case["dtype"]])
        if case["history"]:
            # a text repeats its frequent tokens: ids fall off as a power of a uniform number
            u = torch.rand((rows, case["history"]), generator=g, device="cuda")
            s["history"] = (u.pow(4) * vocab).to(torch.int32).clamp_(0, vocab - 1)
            s["counts"] = torch.from_numpy(rng.permutation(_used(case)).astype(np.int32)).cuda()
            pen = np.stack([rng.uniform(1.0, 1.5, rows), rng.uniform(0.0, 1.0, rows), rng.uniform(0.0, 1.0, rows)], 1)
            s["penalties"] = torch.from_numpy(pen.astype(np.float32)).cuda()
        if case["bias"] != "none":
            n = rows if case["bias"] == "rows" else 1
            keep = torch.rand((n, vocab), generator=g, device="cuda") < 0.01
            s["bias"] = torch.randn((n, vocab), generator=g, device="cuda") * keep
        if case["allowed"] != "none":
            n = rows if case["allowed"] == "rows" else 1
            words = (vocab + 31) // 32
            s["allowed"] = torch.randint(-(1 << 31), 1 << 31, (n, words), generator=g, device="cuda").to(torch.int32)
        if own:
            s["out"] = torch.empty_like(s["logits"])
            p = _package()
            opt = lambda name: _view(s[name]) if name in s else None  # noqa: E731
            s["event"] = p.OpLogitsAdjust(_view(s["logits"]), _view(s["out"]), opt("history"), opt("counts"),
                                          opt("penalties"), opt("bias"), opt("allowed"))
    return s


# ---------------------------------------------------------------------------
# The framework's operators
# ---------------------------------------------------------------------------

_loaded = {}


def _package():
    if "package" not in _loaded:
        name = "emel_rs_b200"
        if name not in sys.modules:
            at = Path(__file__).resolve().parent.parent / "emel.rs_b200"
            spec = importlib.util.spec_from_file_location(name, at / "__init__.py", submodule_search_locations=[str(at)])
            sys.modules[name] = importlib.util.module_from_spec(spec)
            spec.loader.exec_module(sys.modules[name])
        _loaded["package"] = sys.modules[name]
    return _loaded["package"]


def _kernel():
    if "kernel" not in _loaded:
        _loaded["kernel"] = _package().Kernel(device=torch.cuda.current_device())
    return _loaded["kernel"]


def _view(t):
    """A torch tensor as the framework's device view: extents and byte strides, innermost first."""
    p = _package()
    code = {torch.float32: p.DType.F32, torch.float16: p.DType.F16, torch.bfloat16: p.DType.BF16, torch.int32: p.DType.I32}
    ne = list(t.shape)[::-1]
    nb = [x * t.element_size() for x in t.stride()][::-1]
    while len(ne) < 4:
        nb.append(nb[-1] * ne[-1])
        ne.append(1)
    reach = sum((n - 1) * b for n, b in zip(ne, nb)) + t.element_size()
    return p.TensorView(t.data_ptr(), reach, p.Layout.new(code[t.dtype], ne, nb)).c()


def _packed_view(case, blocks):
    p = _package()
    code = {"q4_0": p.DType.Q4_0, "q4_1": p.DType.Q4_1, "q4_k": p.DType.Q4_K}[case["fmt"]]
    row = blocks.shape[1]
    layout = p.Layout.new(code, [case["k"], case["rows"], 1, 1], [1, row, row * case["rows"], row * case["rows"]])
    return p.TensorView(blocks.data_ptr(), blocks.numel(), layout).c()


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------

def run(s):
    op = s["case"]["op"]
    if own:
        status = _kernel().process_event(s["event"])
        if status != 0:
            raise RuntimeError("%s: %s" % (op, status))
        return {"k": s["k"], "v": s["v"]} if op == "append" else s["out"]
    return {"attn": _plain_attn, "append": _plain_append, "q4": _plain_q4, "logits": _plain_logits}[op](s)


def _plain_attn(s):
    q, table = s["q"], s["table"].long().clamp(min=0)
    batch, heads, d = q.shape
    page, kv_heads = s["k"].shape[1], s["k"].shape[2]
    at = torch.arange(table.shape[1] * page, device=q.device)[None, :]
    n = s["lengths"].long()[:, None]
    seen = at < n
    if s["case"]["window"]:
        seen = seen & (at >= n - s["case"]["window"])
    k = s["k"][table].flatten(1, 2).float()  # [batch, token, kv head, d]
    v = s["v"][table].flatten(1, 2).float()
    v = torch.where(seen[:, :, None, None], v, torch.zeros((), device=q.device))
    x = q.float().view(batch, kv_heads, heads // kv_heads, d) * (1.0 / math.sqrt(d))
    score = torch.matmul(x, k.permute(0, 2, 3, 1))
    score = torch.where(seen[:, None, None, :], score, torch.full((), -math.inf, device=q.device))
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v.permute(0, 2, 1, 3)) / torch.where(total > 0, total, torch.ones_like(total))
    return out.reshape(batch, heads, d).to(q.dtype)


def _plain_append(s):
    page = s["k"].shape[1]
    at = s["position"].long()
    to = s["table"].long()[s["sequence"].long(), at // page]
    s["k"][to, at % page] = s["key"].to(s["k"].dtype)
    s["v"][to, at % page] = s["value"].to(s["v"].dtype)
    return {"k": s["k"], "v": s["v"]}


def _q4_weights(blocks, fmt, dtype):
    """The blocks' values as [rows, k]: d (q - 8), d q + m, or d s q - e m with 6-bit s and m."""
    values, size = Q4_BLOCK[fmt]
    rows = blocks.shape[0]
    b = blocks.view(rows, -1, size)
    if fmt == "q4_k":
        d, e = b[..., 0:4].contiguous().view(torch.float16).to(dtype).split(1, -1)
        c = b[..., 4:16]
        low, high, top = c[..., 0:4], c[..., 4:8], c[..., 8:12]
        scale = torch.cat([low & 63, (top & 15) | ((low >> 6) << 4)], -1).to(dtype)
        least = torch.cat([high & 63, (top >> 4) | ((high >> 6) << 4)], -1).to(dtype)
        q = b[..., 16:].reshape(rows, -1, 4, 1, 32)
        q = torch.cat([q & 15, q >> 4], -2).reshape(rows, -1, 8, 32).to(dtype)
        w = (d * scale)[..., None] * q - (e * least)[..., None]
        return w.reshape(rows, -1)
    head = b[..., : size - 16].contiguous().view(torch.float16).to(dtype)
    q = b[..., size - 16:]
    q = torch.cat([q & 15, q >> 4], -1).to(dtype)
    w = head[..., 0:1] * (q - 8) if fmt == "q4_0" else head[..., 0:1] * q + head[..., 1:2]
    return w.reshape(rows, -1)


def _plain_q4(s):
    return torch.matmul(s["x"].float(), _q4_weights(s["blocks"], s["case"]["fmt"], torch.float32).t())


def _plain_logits(s):
    x = s["logits"].float()
    rows, vocab = x.shape
    if "history" in s:
        h = s["history"]
        used = torch.arange(h.shape[1], device=x.device)[None, :] < s["counts"][:, None]
        count = torch.zeros((rows, vocab), device=x.device)
        count.scatter_add_(1, h.long(), used.float())
        r, f, p = s["penalties"].split(1, 1)
        changed = torch.where(x > 0, x / r, x * r) - count * f - p
        x = torch.where(count > 0, changed, x)
    if "bias" in s:
        x = x + s["bias"]
    if "allowed" in s:
        bit = torch.arange(vocab, device=x.device)
        ok = (s["allowed"][:, bit // 32] >> (bit % 32)) & 1
        x = torch.where(ok != 0, x, torch.full((), -math.inf, device=x.device))
    return x.to(s["logits"].dtype)


# ---------------------------------------------------------------------------
# What a pass cannot do without, and what it should give
# ---------------------------------------------------------------------------

def work(case):
    if case["op"] == "attn":
        n = _spread(case)
        tokens = int(np.minimum(n, case["window"]).sum() if case["window"] else n.sum())
        seen = tokens * case["kv_heads"] * case["d"]
        rows = case["batch"] * case["kv_heads"] * case["rep"] * case["d"]
        return {"bytes": 2 * seen * BYTES[case["kv"]] + 2 * rows * BYTES[case["q"]], "flops": 4 * seen * case["rep"]}
    if case["op"] == "append":
        values = 2 * case["n"] * case["kv_heads"] * case["d"]
        return {"bytes": values * (BYTES[case["src"]] + BYTES[case["kv"]]) + 12 * case["n"], "flops": 0}
    if case["op"] == "q4":
        values, size = Q4_BLOCK[case["fmt"]]
        weights = case["rows"] * case["k"]
        rest = case["n"] * case["k"] * BYTES[case["x"]] + case["n"] * case["rows"] * 4
        return {"bytes": weights // values * size + rest, "flops": 2 * weights * case["n"]}
    each = case["rows"] * case["vocab"]
    many = {"none": 0, "shared": 1, "rows": case["rows"]}
    moved = 2 * each * BYTES[case["dtype"]] + 4 * case["vocab"] * many[case["bias"]]
    moved += case["vocab"] * many[case["allowed"]] / 8 + 4 * int(_used(case).sum())
    return {"bytes": moved, "flops": 4 * each}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attn":
        q, page = s["q"].double(), case["page"]
        out = torch.zeros_like(q)
        for b, n in enumerate(s["lengths"].tolist()):
            first = max(0, n - case["window"]) if case["window"] else 0
            at = torch.arange(first, n, device=q.device)
            where = s["table"][b].long()[at // page]
            k, v = s["k"][where, at % page].double(), s["v"][where, at % page].double()
            for h in range(case["kv_heads"]):
                of = slice(h * case["rep"], (h + 1) * case["rep"])
                out[b, of] = torch.softmax(q[b, of] @ k[:, h].t() / math.sqrt(case["d"]), -1) @ v[:, h]
        return out
    if case["op"] == "append":
        k, v = s["k"].double(), s["v"].double()
        seq, at = s["sequence"].long(), s["position"].long()
        to = s["table"].long()[seq, torch.div(at, case["page"], rounding_mode="floor")]
        flat = to * case["page"] + at % case["page"]
        for cache, new in ((k, s["key"]), (v, s["value"])):
            where = flat[:, None, None] // case["page"], flat[:, None, None] % case["page"]
            cache.index_put_((where[0], where[1], torch.arange(case["kv_heads"], device="cuda")[None, :, None],
                              torch.arange(case["d"], device="cuda")[None, None, :]), new.double())
        return {"k": k, "v": v}
    if case["op"] == "q4":
        x, parts = s["x"].double(), []
        step = max(1, (1 << 26) // case["k"])
        for at in range(0, case["rows"], step):
            parts.append(x @ _exact_q4(s["blocks"][at: at + step], case["fmt"]).t())
        return torch.cat(parts, 1)
    x = s["logits"].double().cpu().numpy()
    if "history" in s:
        hist, used, pen = s["history"].cpu().numpy(), s["counts"].cpu().numpy(), s["penalties"].double().cpu().numpy()
        for row in range(case["rows"]):
            ids, many = np.unique(hist[row, : used[row]], return_counts=True)
            old, (r, f, p) = x[row, ids], pen[row]
            x[row, ids] = np.where(old > 0, old / r, old * r) - many * f - p
    if "bias" in s:
        x = x + s["bias"].double().cpu().numpy()
    if "allowed" in s:
        bits = np.unpackbits(s["allowed"].cpu().numpy().view(np.uint8), axis=1, bitorder="little")[:, : case["vocab"]]
        x = np.where(bits == 1, x, -np.inf)
    return torch.from_numpy(x).cuda()


def _exact_q4(blocks, fmt):
    """The values group by group, in 64 bits."""
    values, size = Q4_BLOCK[fmt]
    rows, n = blocks.shape[0], blocks.shape[1] // size
    b = blocks.view(rows, n, size)
    w = torch.empty((rows, n, values), device=blocks.device, dtype=torch.float64)
    half = lambda at: b[:, :, at: at + 2].contiguous().view(torch.float16).double()  # noqa: E731
    if fmt == "q4_k":
        for j in range(8):
            if j < 4:
                scale, least = b[:, :, 4 + j] & 63, b[:, :, 8 + j] & 63
            else:
                scale = (b[:, :, 8 + j] & 15) + 16 * (b[:, :, j] >> 6)
                least = (b[:, :, 8 + j] >> 4) + 16 * (b[:, :, 4 + j] >> 6)
            byte = b[:, :, 16 + 32 * (j // 2): 48 + 32 * (j // 2)]
            q = (byte >> 4 if j % 2 else byte & 15).double()
            w[:, :, 32 * j: 32 * j + 32] = half(0) * scale.double()[:, :, None] * q - half(2) * least.double()[:, :, None]
        return w.view(rows, -1)
    byte = b[:, :, size - 16:]
    w[:, :, :16], w[:, :, 16:] = (byte & 15).double(), (byte >> 4).double()
    w = (w - 8) * half(0) if fmt == "q4_0" else w * half(0) + half(2)
    return w.reshape(rows, -1)
