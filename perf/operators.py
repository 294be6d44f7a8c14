"""The row-table operators and how they are measured: cases, inputs, plain forms and 64-bit values.

Four operators on tables of learned rows (horizongs_amd/embedding.py, horizongs_amd/rowcache.py):

  lookup  out[i, :] = scale * weight[ids[i], :]; a row of zeros where ids[i] lies outside the table
  grad    dw[v, :]  = scale * sum over i with ids[i] = v of g[i, :]   (train: the lookup and this, by autograd)
  write   slot slots[i] of an 8-bit cache takes row i: one scale per `group` columns, one 8-bit code per value;
          the last row wins where a slot is named twice, a slot outside the cache takes nothing
  read    out[i, c] = codes[slots[i], c] * scales[slots[i], c // group], zeros for a slot outside the cache

`own` picks the framework's calls instead of the plain forms in run().
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2, "i32": 4, "i64": 8}
CODES = {"int8": (torch.int8, 127.0), "e4m3": (torch.float8_e4m3fn, 448.0)}
SCALE_FLOOR = 2.0 ** -100


def _rows(op, name, rows, dim, n, dtype, ids, idtype="i64", **more):
    c = {"name": name, "op": op, "rows": rows, "dim": dim, "n": n, "dtype": dtype, "ids": ids, "idtype": idtype,
         "scale": 1.0, "pad": False, "extra": 0, "out": dtype, "fmt": "", "group": 0}
    c.update(more)
    return c


def listed():
    return [
        # the appearance row of the one camera that a step renders, from a table of a 16-view set
        _rows("lookup", "lookup_view", 16, 32, 1, "f32", "one"),
        # the visible half of a million anchors' features, compacted before the heads (an ascending index)
        _rows("lookup", "lookup_anchors", 1_000_000, 32, 500_000, "f32", "sorted", "i32"),
        # a batch of tokens, ids as skewed as words are, rows scaled by the root of their width
        _rows("lookup", "lookup_tokens", 65_536, 2048, 16_384, "bf16", "zipf", scale=2048 ** 0.5),
        # odd sizes, a padded batch, a table that is a column range of a wider one
        _rows("lookup", "lookup_ragged", 10_007, 333, 4_099, "f16", "uniform", "i32", scale=0.5, pad=True, extra=3),
        # a training step on a few rows: each view of a batch looks its camera up, forward and backward
        _rows("train", "train_views", 1_600, 32, 24, "f32", "uniform", scale=0.25),
        # every anchor's share of the gradient of the appearance rows, 16 views of a batch joined
        _rows("grad", "grad_views", 16, 32, 500_000, "f32", "uniform"),
        # the gradient of the compacted features, back to every anchor (rows not visible get zeros)
        _rows("grad", "grad_anchors", 1_000_000, 32, 500_000, "f32", "sorted", "i32"),
        # the gradient of the batch of tokens: a few rows named thousands of times, most once or never
        _rows("grad", "grad_tokens", 65_536, 2048, 16_384, "bf16", "zipf", scale=2048 ** 0.5),
        # anchors' features go into an 8-bit cache of a million slots
        _rows("write", "write_anchors", 1_000_000, 32, 500_000, "f32", "sorted", "i32", fmt="int8", group=32),
        # one step's few new rows into a cache of wide rows
        _rows("write", "write_step", 65_536, 1024, 8, "bf16", "uniform", fmt="e4m3", group=128),
        # the visible half of the cached features, for a rendered view
        _rows("read", "read_anchors", 1_000_000, 32, 500_000, "f32", "sorted", "i32", fmt="int8", group=32),
        # wide cached rows in any order, some named twice, back to 16 bits
        _rows("read", "read_tokens", 65_536, 2048, 16_384, "bf16", "uniform", fmt="e4m3", group=64),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["lookup", "grad", "write", "read"])
    dim = rng.choice([_log(rng, 1, 2048), _log(rng, 8, 2048) // 8 * 8, 32])
    rows = _log(rng, 16, max(16, min(1_000_000, 33_000_000 // dim)))
    n = _log(rng, 1, max(1, min(500_000, 33_000_000 // dim)))
    kind = rng.choice(["uniform", "zipf", "sorted", "one"] if op in ("lookup", "grad") else ["uniform", "sorted"])
    if kind == "sorted":
        n = min(n, rows)
    dtype = rng.choice(["f32", "bf16", "f16"])
    more = {"scale": rng.choice([1.0, 0.5, round(math.sqrt(dim), 3)]), "pad": rng.random() < 0.3, "out": dtype}
    if op in ("lookup", "write"):
        more["extra"] = rng.choice([0, 0, 1, 8])
    if op == "grad":
        more["out"] = rng.choice([dtype, "f32"])
    if op in ("write", "read"):
        more.update(scale=1.0, fmt=rng.choice(["int8", "e4m3"]), group=rng.choice([16, 32, 64, 128]))
    c = _rows(op, "", rows, dim, n, dtype, kind, rng.choice(["i32", "i64"]), **more)
    del c["name"]
    return c


def _seeded(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _make_ids(c, g):
    V, n = c["rows"], c["n"]
    if c["ids"] == "one":
        ids = torch.randint(0, V, (1,), generator=g, device=DEV).expand(n).contiguous()
    elif c["ids"] == "sorted":
        ids = torch.randperm(V, generator=g, device=DEV)[:n].sort().values
    elif c["ids"] == "zipf":  # p(rank k) ~ 1/k, the ranks spread over the table
        u = torch.rand(n, generator=g, device=DEV, dtype=torch.float64)
        rank = (torch.exp(u * math.log(V + 1)) - 1).long().clamp_(0, V - 1)
        ids = torch.randperm(V, generator=g, device=DEV)[rank]
    else:
        ids = torch.randint(0, V, (n,), generator=g, device=DEV)
    if c["pad"]:
        ids = torch.where(torch.rand(n, generator=g, device=DEV) < 0.1, -1, ids)
    return ids.to(torch.int32 if c["idtype"] == "i32" else torch.int64)


def _normal(g, n, dim, extra, t):
    """[n, dim] normal values of type t, a column range of rows `extra` columns wider."""
    x = torch.randn(n, dim + extra, generator=g, device=DEV).to(t)
    return x[:, :dim]


def prepare(case, seed):
    c, g = case, _seeded(seed)
    t = TYPES[c["dtype"]]
    s = {"case": c, "ids": _make_ids(c, g)}
    if c["op"] in ("lookup", "train"):
        s["weight"] = _normal(g, c["rows"], c["dim"], c["extra"], t)
    if c["op"] == "train":
        s["weight"] = s["weight"].requires_grad_(True)
    if c["op"] in ("grad", "train"):
        s["g"] = _normal(g, c["n"], c["dim"], 0, t)
    if c["op"] == "write":
        # features as trained: most channels small, a few larger
        gain = torch.exp(torch.randn(c["dim"] + c["extra"], generator=g, device=DEV))
        x = torch.randn(c["n"], c["dim"] + c["extra"], generator=g, device=DEV) * gain
        s["x"] = x.to(t)[:, :c["dim"]]
    if c["op"] in ("write", "read"):  # what the cache holds already
        kind, top = CODES[c["fmt"]]
        q = torch.randn(c["rows"], c["dim"], generator=g, device=DEV) * (top / 3)
        q = q.clamp_(-top, top)
        codes = q.round_().to(kind) if c["fmt"] == "int8" else q.to(kind)
        groups = -(-c["dim"] // c["group"])
        scales = torch.exp(torch.randn(c["rows"], groups, generator=g, device=DEV)) / top
        s["cache"] = (codes, scales, c["group"])
    return s


# ---- the plain forms


def _plain_lookup(weight, ids, scale):
    V = weight.shape[0]
    inside = (ids >= 0) & (ids < V)
    out = weight[ids.clamp(0, V - 1).long()].float() * scale
    return torch.where(inside[:, None], out, 0.0).to(weight.dtype)


def _plain_grad(g, ids, V, scale, out_type, long):
    at = torch.where((ids >= 0) & (ids < V), ids, V).long()  # V: outside the table
    if long:  # few rows of many terms each: running sums of the sorted terms, in 64 bits, and their differences
        n, D = g.shape
        at, order = torch.sort(at)
        run = torch.zeros(D * n + 1, dtype=torch.float64, device=g.device)
        torch.cumsum(g.double()[order].t().reshape(-1), 0, out=run[1:])  # column after column
        v = torch.arange(V, device=g.device)
        col = torch.arange(D, device=g.device) * n
        first, end = torch.searchsorted(at, v), torch.searchsorted(at, v, right=True)
        return ((run[end[:, None] + col] - run[first[:, None] + col]) * scale).to(out_type)
    dw = torch.zeros(V + 1, g.shape[1], dtype=torch.float32, device=g.device).index_add_(0, at, g.float())
    return (dw[:V] * scale).to(out_type)


def _plain_group_scales(scales, group, dim):
    return scales[:, torch.arange(dim, device=scales.device) // group]


def _plain_write(cache, x, slots):
    codes, scales, group = cache
    cap, dim = codes.shape
    n, groups = x.shape[0], scales.shape[1]
    top = 127.0 if codes.dtype == torch.int8 else 448.0
    x = x.float()
    wide = torch.zeros(n, groups * group, device=x.device)
    wide[:, :dim] = x
    amax = wide.view(n, groups, group).abs().amax(2)  # a NaN stays one
    s = torch.where(amax.isfinite(), (amax / top).clamp_min(SCALE_FLOOR), math.nan)
    q = (x.double() / _plain_group_scales(s, group, dim).double()).nan_to_num(0.0)  # 64 bits: codes next to a border
    if codes.dtype == torch.int8:
        q = q.round().to(torch.int8)
    else:
        step = torch.exp2(torch.frexp(q).exponent.clamp_min(-5) - 4.0)  # 3 bits behind the leading one, 2^-9 below 2^-6
        q = ((q / step).round() * step).float().to(codes.dtype)
    # where a slot is named twice every one of its rows writes what the last one holds; a row whose slot
    # lies outside writes slot 0 as it is, or as its own last row makes it
    at = torch.where((slots >= 0) & (slots < cap), slots, cap).long()
    last = torch.full((cap + 1,), -1, device=x.device, dtype=torch.int64)
    last.scatter_reduce_(0, at, torch.arange(n, device=x.device), "amax")
    at = torch.where(at < cap, at, 0)
    src = last[at]
    wins = (src >= 0)[:, None]
    src = src.clamp_min(0)
    bits = codes.view(torch.uint8)
    bits.index_copy_(0, at, torch.where(wins, q.view(torch.uint8)[src], bits[at]))
    scales.index_copy_(0, at, torch.where(wins, s[src], scales[at]))
    return codes, scales


def _plain_read(cache, slots, out_type):
    codes, scales, group = cache
    cap, dim = codes.shape
    inside = (slots >= 0) & (slots < cap)
    at = slots.clamp(0, cap - 1).long()
    q = codes.view(torch.uint8)[at].view(codes.dtype).float()
    out = q * _plain_group_scales(scales[at], group, dim)
    return torch.where(inside[:, None], out, 0.0).to(out_type)


def run(state):
    s, c = state, state["case"]
    if own:
        from horizongs_amd import embedding as E
        from horizongs_amd import rowcache as R
        if c["op"] == "lookup":
            return E.embedding(s["weight"], s["ids"], c["scale"])
        if c["op"] == "train":
            out = E.embedding(s["weight"], s["ids"], c["scale"])
            return out.detach(), torch.autograd.grad(out, s["weight"], s["g"])[0]
        if c["op"] == "grad":
            return E.embedding_grad(s["g"], s["ids"], c["rows"], c["scale"], dtype=TYPES[c["out"]])
        if c["op"] == "write":
            R.rowcache_write(s["cache"], s["x"], s["ids"])
            return s["cache"][0], s["cache"][1]
        return R.rowcache_read(s["cache"], s["ids"], dtype=TYPES[c["dtype"]])
    long = c["ids"] == "one" or c["n"] > 64 * c["rows"]
    with torch.no_grad():
        if c["op"] == "lookup":
            return _plain_lookup(s["weight"], s["ids"], c["scale"])
        if c["op"] == "train":
            return (_plain_lookup(s["weight"], s["ids"], c["scale"]),
                    _plain_grad(s["g"], s["ids"], c["rows"], c["scale"], s["weight"].dtype, long))
        if c["op"] == "grad":
            return _plain_grad(s["g"], s["ids"], c["rows"], c["scale"], TYPES[c["out"]], long)
        if c["op"] == "write":
            return _plain_write(s["cache"], s["x"], s["ids"])
        return _plain_read(s["cache"], s["ids"], TYPES[c["dtype"]])


def _distinct(c):
    """Expected number of different rows that the ids name."""
    V, n = c["rows"], c["n"]
    if c["ids"] == "one":
        return 1
    if c["ids"] == "sorted":
        return n
    if c["ids"] == "zipf":
        k = np.arange(V, dtype=np.float64)
        p = np.log((k + 2) / (k + 1)) / math.log(V + 1)
        return float(np.sum(-np.expm1(n * np.log1p(-np.minimum(p, 1 - 1e-12)))))
    return V * -math.expm1(n * math.log1p(-1.0 / V)) if V > 1 else 1


def work(case):
    c = case
    n, V, D, sz, ids = c["n"], c["rows"], c["dim"], SIZE[c["dtype"]], c["n"] * SIZE[c["idtype"]]
    touched = _distinct(c)
    lookup = ids + touched * D * sz + n * D * sz
    grad = ids + n * D * sz + V * D * SIZE[c["out"]]
    if c["op"] == "lookup":
        return {"bytes": lookup, "flops": n * D}
    if c["op"] == "train":
        return {"bytes": lookup + grad - ids, "flops": 2 * n * D}
    if c["op"] == "grad":
        return {"bytes": grad, "flops": n * D}
    held = touched * (D + 4 * -(-D // c["group"]))  # the slots' codes and scales
    return {"bytes": ids + held + n * D * sz, "flops": n * D}


def _values_of_codes(codes):
    """The values of 8-bit codes, from the format's definition."""
    if codes.dtype == torch.int8:
        return codes.cpu().numpy().astype(np.float64)
    b = codes.view(torch.uint8).cpu().numpy().astype(np.int64)
    return _e4m3_table()[b & 127] * np.where(b > 127, -1.0, 1.0)


def _e4m3_table():
    k = np.arange(128)
    e, m = k >> 3, k & 7
    t = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0))
    t[127] = np.nan
    return t


def _nearest_e4m3(q):
    t = _e4m3_table()[:127]
    a = np.abs(q)
    hi = np.clip(np.searchsorted(t, a), 0, 126)
    lo = np.maximum(hi - 1, 0)
    down, up = a - t[lo], t[hi] - a
    k = np.where((down < up) | ((down == up) & (lo % 2 == 0)), lo, hi)
    return np.copysign(t[k], q)


def exact(case, seed):
    c = case
    s = prepare(case, seed)
    ids = s["ids"].cpu().numpy().astype(np.int64)
    V, D, n = c["rows"], c["dim"], c["n"]
    ok = np.flatnonzero((ids >= 0) & (ids < V))
    if c["op"] in ("lookup", "train"):
        out = np.zeros((n, D))
        out[ok] = s["weight"].detach().double().cpu().numpy()[ids[ok]] * c["scale"]
    if c["op"] in ("grad", "train"):
        order = ok[np.argsort(ids[ok], kind="stable")]
        dw = np.zeros((V, D))
        if order.size:
            first = np.flatnonzero(np.r_[True, np.diff(ids[order]) > 0])
            dw[ids[order][first]] = np.add.reduceat(s["g"].double().cpu().numpy()[order], first, axis=0) * c["scale"]
    if c["op"] == "lookup":
        return out
    if c["op"] == "train":
        return out, dw
    if c["op"] == "grad":
        return dw
    codes, scales, group = s["cache"]
    if c["op"] == "read":
        out = np.zeros((n, D))
        wide = np.repeat(scales.double().cpu().numpy(), group, axis=1)[:, :D]
        out[ok] = (_values_of_codes(codes) * wide)[ids[ok]]
        return out
    held_c, held_s = _values_of_codes(codes), scales.double().cpu().numpy()
    slot, last = np.unique(ids[ok][::-1], return_index=True)  # the last row of each slot
    x = s["x"].double().cpu().numpy()[ok[::-1][last]]
    wide = np.zeros((x.shape[0], held_s.shape[1] * group))
    wide[:, :D] = np.abs(x)
    top = CODES[c["fmt"]][1]
    sc = np.maximum(wide.reshape(x.shape[0], -1, group).max(2) / top, SCALE_FLOOR)
    q = x / np.repeat(sc.astype(np.float32).astype(np.float64), group, axis=1)[:, :D]  # the scale that is held
    held_c[slot] = np.rint(q) if c["fmt"] == "int8" else _nearest_e4m3(q)
    held_s[slot] = sc
    return (None if c["fmt"] == "int8" else held_c), held_s
