"""Cases, inputs and plain forms of the windowed, paged and shared-prefix attention operators.

Five operators, in the order in which a model meets them:

  prompt  attention of a whole sequence in which a token sees the `window` newest tokens up to
          itself and the `sinks` first ones (out)
  train   the same with its gradients (out, dq, dk, dv)
  cache   new tokens enter a paged key/value cache: block tables and slots from the request
          lengths, then the copy of k and v (block_table, slots, starts, used, k_cache, v_cache)
  decode  attention of one token for each request over the paged cache, all of it or a window
          with sinks (out)
  prefix  the same for a batch whose requests share a prefix, which is stored once (out)

`run` computes them in plain torch operations, or, where `own` is true, by the calls of
mini_flash_attention.
"""
import math
import sys
from pathlib import Path

import torch

own = False

_PACKAGE = str(Path(__file__).resolve().parents[1] / "mini-flash-attention_b200")
_TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _mfa():
    if _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)
    import mini_flash_attention

    return mini_flash_attention


# ------------------------------------------------------------------------------- the cases
def listed():
    return [
        # a short ragged batch of a small grouped-head model, odd length, one sink token
        {"name": "prompt_odd", "op": "prompt", "dtype": "bf16", "batch": 2, "kv_heads": 2,
         "group": 3, "n": 1000, "d": 128, "window": 256, "sinks": 1},
        # a long prompt, the benchmark's length, a window of a quarter of it
        {"name": "prompt_long", "op": "prompt", "dtype": "fp16", "batch": 1, "kv_heads": 4,
         "group": 4, "n": 8192, "d": 64, "window": 2048, "sinks": 64},
        # fine-tuning on short texts: few blocks, a window of one block
        {"name": "train_odd", "op": "train", "dtype": "fp16", "batch": 2, "kv_heads": 2,
         "group": 3, "n": 777, "d": 64, "window": 128, "sinks": 4},
        # training on long texts
        {"name": "train_long", "op": "train", "dtype": "bf16", "batch": 1, "kv_heads": 4,
         "group": 4, "n": 8192, "d": 64, "window": 2048, "sinks": 16},
        # one token for each of many requests enters the cache (one step of serving)
        {"name": "cache_step", "op": "cache", "dtype": "bf16", "batch": 256, "kv_heads": 8,
         "d": 128, "page": 16, "cached_min": 15, "cached_max": 2047, "added_min": 1,
         "added_max": 1, "spare": 0},
        # a batch of prompts enters it, padded to a fixed number of tokens
        {"name": "cache_prompts", "op": "cache", "dtype": "fp16", "batch": 33, "kv_heads": 8,
         "d": 64, "page": 64, "cached_min": 0, "cached_max": 500, "added_min": 17,
         "added_max": 8191, "spare": 1000},
        # one user, one token, a short context: latency counts
        {"name": "decode_one", "op": "decode", "dtype": "bf16", "batch": 1, "kv_heads": 8,
         "group": 4, "d": 128, "page": 16, "len_min": 1000, "len_max": 1000, "window": 0,
         "sinks": 0},
        # a full serving batch with contexts from a few tokens to long ones
        {"name": "decode_batch", "op": "decode", "dtype": "bf16", "batch": 64, "kv_heads": 8,
         "group": 4, "d": 128, "page": 32, "len_min": 100, "len_max": 16384, "window": 0,
         "sinks": 0},
        # streaming: very long contexts of which a window and the first tokens are read
        {"name": "decode_window", "op": "decode", "dtype": "fp16", "batch": 100, "kv_heads": 4,
         "group": 5, "d": 64, "page": 64, "len_min": 1, "len_max": 32768, "window": 1024,
         "sinks": 4},
        # a few answers to one short system prompt
        {"name": "prefix_few", "op": "prefix", "dtype": "fp16", "batch": 3, "kv_heads": 2,
         "group": 4, "d": 64, "page": 16, "prefix": 500, "len_min": 1, "len_max": 60},
        # a batch of questions about one long document
        {"name": "prefix_batch", "op": "prefix", "dtype": "bf16", "batch": 64, "kv_heads": 8,
         "group": 4, "d": 128, "page": 32, "prefix": 16001, "len_min": 16, "len_max": 1000},
        # many samples of one very long context, enough rows to be bound by arithmetic
        {"name": "prefix_many", "op": "prefix", "dtype": "fp16", "batch": 250, "kv_heads": 4,
         "group": 8, "d": 64, "page": 128, "prefix": 32768, "len_min": 1, "len_max": 300},
    ]


def _between(rng, low, high):
    """A whole number in [low, high], spread evenly over its logarithm."""
    return min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))


def draw(rng):
    op = rng.choice(("prompt", "train", "cache", "decode", "decode", "prefix"))
    c = {"op": op, "dtype": rng.choice(("fp16", "bf16"))}
    if op in ("prompt", "train"):
        n = _between(rng, 1, 8192)
        c |= {"n": n, "d": 64 if op == "train" else rng.choice((32, 64, 128)),
              "window": _between(rng, 1, 2048), "sinks": rng.choice((0, 1, 4, 16, 130, 300))}
        heads = min(64, 9 * 8192 * 8192 // (n * n))  # of all sequences together
        c["group"] = rng.choice([g for g in (1, 2, 3, 4, 5, 8) if g <= heads])
        c["kv_heads"] = rng.choice([h for h in (1, 2, 4, 8) if h * c["group"] <= heads])
        c["batch"] = rng.randint(1, max(1, min(4, heads // (c["group"] * c["kv_heads"]))))
    elif op == "cache":
        c |= {"kv_heads": rng.choice((1, 2, 3, 8)), "d": rng.choice((64, 128)),
              "page": rng.choice((16, 32, 64, 128)), "batch": _between(rng, 1, 300),
              "spare": rng.choice((0, 1, 100))}
        most = 23_000_000 // (c["batch"] * c["kv_heads"] * c["d"])
        c["added_max"] = _between(rng, 1, max(1, min(8191, most)))
        c["added_min"] = rng.choice((0, 1, c["added_max"]))
        c["cached_max"] = _between(rng, 1, 2047)
        c["cached_min"] = rng.choice((0, c["cached_max"]))
    else:
        c |= {"kv_heads": rng.choice((1, 2, 4, 8)), "d": rng.choice((64, 128)),
              "page": rng.choice((16, 32, 64, 128)),
              "group": rng.choice((1, 2, 3, 4, 5, 7, 8, 16)), "len_min": rng.choice((0, 1, 50))}
        if op == "decode":
            c["batch"] = _between(rng, 1, 200)
            most = 64 * 16384 * 8 * 128 // (c["batch"] * c["kv_heads"] * c["d"])
            c["len_max"] = _between(rng, 50, min(65536, most))
            c["window"] = rng.choice((0, _between(rng, 1, 8192)))
            c["sinks"] = rng.choice((0, 1, 4, 100)) if c["window"] else 0
        else:
            c["batch"] = _between(rng, 1, 250)
            rows = c["batch"] * c["kv_heads"] * c["group"]
            c["prefix"] = _between(rng, 16, min(32768, 250 * 32 * 32768 * 64 // (rows * c["d"])))
            c["len_max"] = _between(rng, 50, 1000)
    return c


# ------------------------------------------------------------------------------ the inputs
def _lengths(low, high, count):
    """`count` lengths from `low` to `high`, evenly spread over the logarithm: known from the
    case alone, whatever the seed."""
    if count == 1:
        return [high]
    a, b = math.log(low + 1), math.log(high + 1)
    return [min(high, max(low, round(math.exp(a + (b - a) * i / (count - 1)) - 1)))
            for i in range(count)]


def _random(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _shuffled(values, g):
    t = torch.tensor(values, dtype=torch.int32, device="cuda")
    return t[torch.randperm(len(values), generator=g, device="cuda")]


def _normal(shape, dtype, g):
    return torch.randn(shape, generator=g, device="cuda", dtype=dtype)


def _pages(lengths, page):
    return [-(-n // page) for n in lengths]


def _tables(counts, columns, pages):
    """A [requests, columns] table with the first counts[i] entries of row i taken from the
    shuffled pages, -1 behind them."""
    col = torch.arange(columns, device="cuda")[None, :]
    first = torch.cumsum(counts, 0) - counts
    at = (first[:, None] + col).clamp(max=max(0, len(pages) - 1))
    none = torch.full((), -1, dtype=torch.int32, device="cuda")
    return torch.where(col < counts[:, None], pages[at] if len(pages) else none, none)


def prepare(case, seed):
    c, g, dtype = case, _random(seed), _TYPES[case["dtype"]]
    if c["op"] in ("prompt", "train"):
        heads = c["kv_heads"] * c["group"]
        s = {"op": c["op"], "window": c["window"], "sinks": c["sinks"]}
        s["q"] = _normal((c["batch"], heads, c["n"], c["d"]), dtype, g)
        s["k"] = _normal((c["batch"], c["kv_heads"], c["n"], c["d"]), dtype, g)
        s["v"] = _normal((c["batch"], c["kv_heads"], c["n"], c["d"]), dtype, g)
        if c["op"] == "train":
            s["dout"] = _normal(s["q"].shape, dtype, g)
            for x in ("q", "k", "v"):
                s[x].requires_grad_()
        return s
    page, batch = c["page"], c["batch"]
    if c["op"] == "cache":
        cached, added = _cache_lengths(c)
        total, have = sum(added), _pages(cached, page)
        need = _pages([x + y for x, y in zip(cached, added)], page)
        order = torch.randperm(batch, generator=g, device="cuda")
        to_gpu = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")[order]  # noqa: E731
        pages = _shuffled(range(sum(need) + 8), g)
        shape = (len(pages), c["kv_heads"], page, c["d"])
        rows = (total + c["spare"], c["kv_heads"], c["d"])
        return {"op": "cache", "page": page, "cached": to_gpu(cached), "added": to_gpu(added),
                "block_table": _tables(to_gpu(have), max(1, max(need)), pages),
                "free_pages": pages[sum(have):].contiguous(), "capacity": rows[0],
                "k": _normal(rows, dtype, g), "v": _normal(rows, dtype, g),
                "k_cache": _normal(shape, dtype, g), "v_cache": _normal(shape, dtype, g)}
    lengths = _lengths(c["len_min"], c["len_max"], batch)
    shared = -(-c["prefix"] // page) if c["op"] == "prefix" else 0
    counts = _pages(lengths, page)
    pages = _shuffled(range(sum(counts) + shared), g)
    lengths = _shuffled(lengths, g)
    shape = (len(pages), c["kv_heads"], page, c["d"])
    s = {"op": c["op"], "lengths": lengths,
         "block_table": _tables((lengths + page - 1) // page, max(1, max(counts)), pages[shared:]),
         "q": _normal((batch, c["kv_heads"] * c["group"], c["d"]), dtype, g),
         "k_cache": _normal(shape, dtype, g), "v_cache": _normal(shape, dtype, g)}
    if c["op"] == "prefix":
        s |= {"prefix_pages": pages[:shared].contiguous(), "prefix_length": c["prefix"]}
    else:
        s |= {"window": c["window"], "sinks": c["sinks"]}
    return s


def _cache_lengths(c):
    cached = _lengths(c["cached_min"], c["cached_max"], c["batch"])
    added = _lengths(c["added_min"], c["added_max"], c["batch"])
    return cached, added[::2] + added[1::2]  # long and short ones meet


# ------------------------------------------------------------------------- the plain forms
def _attend(scores, seen, v):
    """Softmax over the seen places of the last axis, times v; 0 where nothing is seen. Also
    the weights."""
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top > -math.inf, top, 0.0))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, 1.0)
    return p @ v, p


def _plain_sequence(q, k, v, window, sinks, dout=None):
    b, h, n, d = q.shape
    hk, scale = k.shape[1], d ** -0.5
    qf = q.float().reshape(b, hk, h // hk, n, d)
    kf, vf = k.float()[:, :, None], v.float()[:, :, None]
    i = torch.arange(n, device=q.device)
    i, j = i[:, None], i[None, :]
    seen = (j <= i) & ((j > i - window) | (j < sinks))
    out, p = _attend(qf @ kf.transpose(-1, -2) * scale, seen, vf)
    if dout is None:
        return out.reshape(q.shape).to(q.dtype)
    do = dout.float().reshape(out.shape)
    dv = (p.transpose(-1, -2) @ do).sum(2)
    ds = p * (do @ vf.transpose(-1, -2) - (do * out).sum(-1, keepdim=True)) * scale
    dq, dk = ds @ kf, (ds.transpose(-1, -2) @ qf).sum(2)
    return [x.reshape(y.shape).to(q.dtype) for x, y in ((out, q), (dq, q), (dk, k), (dv, v))]


def _gathered(cache, table):
    """[requests, kv_heads, columns * page, d] in 32 bits: the pages of each table row."""
    x = cache[table.clamp(min=0).long()].float().transpose(1, 2)
    return x.reshape(x.shape[0], x.shape[1], -1, x.shape[-1])


def _plain_decode(q, k_cache, v_cache, table, lengths, window, sinks):
    b, h, d = q.shape
    hk = k_cache.shape[1]
    qf = q.float().reshape(b, hk, h // hk, d)
    k, v = _gathered(k_cache, table), _gathered(v_cache, table)
    j, n = torch.arange(k.shape[2], device=q.device)[None, :], lengths[:, None]
    seen = (j < n) & ((j >= n - window) | (j < sinks)) if window else j < n
    out, _ = _attend(qf @ k.transpose(-1, -2) * d ** -0.5, seen[:, None, None], v)
    return out.reshape(q.shape).to(q.dtype)


def _plain_prefix(q, k_cache, v_cache, prefix_pages, prefix, table, lengths):
    b, h, d = q.shape
    hk = k_cache.shape[1]
    qf = q.float().reshape(b, hk, h // hk, d)
    k0, v0 = (_gathered(x, prefix_pages[None])[0, :, :prefix] for x in (k_cache, v_cache))
    k1, v1 = _gathered(k_cache, table), _gathered(v_cache, table)
    rows = qf.transpose(0, 1).reshape(hk, -1, d)  # the prefix meets all rows at once
    s0 = (rows @ k0.transpose(-1, -2)).reshape(hk, b, -1, prefix).transpose(0, 1)
    s = torch.cat((s0, qf @ k1.transpose(-1, -2)), -1) * d ** -0.5
    j = torch.arange(s.shape[-1], device=q.device)[None, :]
    s = s.masked_fill(~(j < prefix + lengths[:, None])[:, None, None], -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    p0 = p[..., :prefix].transpose(0, 1).reshape(hk, -1, prefix)
    out = (p0 @ v0).reshape(hk, b, -1, d).transpose(0, 1) + p[..., prefix:] @ v1
    return out.reshape(q.shape).to(q.dtype)


def _plain_cache(s):
    page, table = s["page"], s["block_table"]
    cached, added = s["cached"].long(), s["added"].long()
    have, need = (cached + page - 1) // page, (cached + added + page - 1) // page
    ends, first = torch.cumsum(added, 0), torch.cumsum(need - have, 0) - (need - have)
    col = torch.arange(table.shape[1], device=table.device)[None, :]
    fresh = (col >= have[:, None]) & (col < need[:, None])
    at = (first[:, None] + col - have[:, None]).clamp(0, s["free_pages"].numel() - 1)
    table.copy_(torch.where(fresh, s["free_pages"][at], table))
    t = torch.arange(s["capacity"], device=table.device)
    b = torch.searchsorted(ends, t, right=True).clamp(max=len(cached) - 1)
    pos = cached[b] + t - (ends - added)[b]
    held = t < ends[-1]
    slots = table[b, (pos // page).clamp(max=table.shape[1] - 1)] * page + pos % page
    slots = torch.where(held, slots, -1).to(torch.int32)
    starts = torch.cat((ends[:1] * 0, ends)).to(torch.int32)
    used = (need - have).sum().to(torch.int32).reshape(1)
    to = slots[held].long()
    s["k_cache"][to // page, :, to % page] = s["k"][held]
    s["v_cache"][to // page, :, to % page] = s["v"][held]
    return [table, slots, starts, used, s["k_cache"], s["v_cache"]]


def run(state):
    s = state
    if own:
        return _run_own(s)
    with torch.no_grad():
        if s["op"] in ("prompt", "train"):
            return _plain_sequence(s["q"], s["k"], s["v"], s["window"], s["sinks"], s.get("dout"))
        if s["op"] == "cache":
            return _plain_cache(s)
        if s["op"] == "decode":
            return _plain_decode(s["q"], s["k_cache"], s["v_cache"], s["block_table"],
                                 s["lengths"], s["window"], s["sinks"])
        return _plain_prefix(s["q"], s["k_cache"], s["v_cache"], s["prefix_pages"],
                             s["prefix_length"], s["block_table"], s["lengths"])


def _run_own(s):
    mfa = _mfa()
    if s["op"] == "prompt":
        return mfa.forward_window(s["q"], s["k"], s["v"], s["window"], s["sinks"])
    if s["op"] == "train":
        leaves = (s["q"], s["k"], s["v"])
        out = mfa.window_attention(*leaves, s["window"], s["sinks"])
        return [out.detach(), *torch.autograd.grad(out, leaves, s["dout"])]
    if s["op"] == "cache":
        slots, starts, used = mfa.extend_block_tables(
            s["block_table"], s["cached"], s["added"], s["free_pages"], s["page"], s["capacity"])
        mfa.append_kv(s["k"], s["v"], s["k_cache"], s["v_cache"], slots)
        return [s["block_table"], slots, starts, used, s["k_cache"], s["v_cache"]]
    if s["op"] == "decode":
        return mfa.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["block_table"],
                                   s["lengths"], s["window"], s["sinks"])
    return mfa.shared_prefix_attention(s["q"], s["k_cache"], s["v_cache"], s["prefix_pages"],
                                       s["prefix_length"], s["block_table"], s["lengths"])


# ---------------------------------------------------------------------------- their work
def _seen_pairs(n, window, sinks):
    """(query, key) pairs of one sequence of n tokens."""
    total = 0
    for i in range(n):
        newest = min(window, i + 1)
        total += newest + min(sinks, i + 1 - newest)
    return total


def _seen_keys(n, window, sinks):
    return n if not window else min(n, window) + min(sinks, max(0, n - window))


def work(case):
    c = case
    if c["op"] in ("prompt", "train"):
        heads, row = c["kv_heads"] * c["group"], c["n"] * c["d"] * 2
        pairs = c["batch"] * heads * _seen_pairs(c["n"], c["window"], c["sinks"])
        q, kv = c["batch"] * heads * row, 2 * c["batch"] * c["kv_heads"] * row
        if c["op"] == "prompt":  # q, k, v in, out out; two products
            return {"bytes": 2 * q + kv, "flops": 4 * pairs * c["d"]}
        # q, k, v, dout in; out, dq, dk, dv out; two products and five more
        return {"bytes": 4 * q + 2 * kv, "flops": 14 * pairs * c["d"]}
    if c["op"] == "cache":
        cached, added = _cache_lengths(c)
        copied = 2 * 2 * 2 * sum(added) * c["kv_heads"] * c["d"]
        fresh = sum(_pages([x + y for x, y in zip(cached, added)], c["page"]))
        fresh -= sum(_pages(cached, c["page"]))
        whole = 4 * (3 * c["batch"] + 2 + 2 * fresh + sum(added) + c["spare"])
        return {"bytes": copied + whole, "flops": 0}
    lengths = _lengths(c["len_min"], c["len_max"], c["batch"])
    keys = sum(_seen_keys(n, c.get("window", 0), c.get("sinks", 0)) for n in lengths)
    shared, rows = c.get("prefix", 0), c["kv_heads"] * c["group"]
    moved = 4 * (keys + shared) * c["kv_heads"] * c["d"] + 4 * c["batch"] * rows * c["d"]
    return {"bytes": moved + 4 * (c["batch"] + (keys + shared) // c["page"]),
            "flops": 4 * (keys + shared * c["batch"]) * rows * c["d"]}


# ----------------------------------------------------------------------- in 64 bits, apart
def _exact_head(q, k, v, window, sinks, dout=None):
    """One head of one sequence, by torch's softmax and autograd in 64 bits."""
    n, d = q.shape
    age = torch.arange(n, device=q.device)[:, None] - torch.arange(n, device=q.device)[None, :]
    hidden = (age < 0) | (age >= window)
    hidden[:, :sinks] = age[:, :sinks] < 0
    x = [t.detach().double().requires_grad_(dout is not None) for t in (q, k, v)]
    w = torch.softmax((x[0] @ x[1].T / math.sqrt(d)).masked_fill(hidden, -math.inf), -1)
    out = w @ x[2]
    if dout is None:
        return (out,)
    return (out.detach(), *torch.autograd.grad(out, x, dout.double()))


def _exact_request(q, k, v):
    """[heads, d] of one request whose keys k and values v are [kv_heads, n, d]."""
    hk, n, d = k.shape
    if n == 0:
        return torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    group = q.shape[0] // hk
    w = torch.einsum("hgd,hnd->hgn", q.double().reshape(hk, group, d), k.double()) / math.sqrt(d)
    return torch.einsum("hgn,hnd->hgd", torch.softmax(w, -1), v.double()).reshape(q.shape)


def _exact_rows(cache, row, positions):
    """[kv_heads, len(positions), d] of the tokens at these positions of a request."""
    page = cache.shape[2]
    at = torch.tensor(positions, dtype=torch.long, device=cache.device)
    return cache[row.long()[at // page], :, at % page].transpose(0, 1)


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] in ("prompt", "train"):
        group = case["group"]
        outs = [[] for _ in range(4 if s["op"] == "train" else 1)]
        for b in range(case["batch"]):
            for h in range(case["kv_heads"]):
                parts = [_exact_head(s["q"][b, h * group + g], s["k"][b, h], s["v"][b, h],
                                     s["window"], s["sinks"],
                                     s["dout"][b, h * group + g] if "dout" in s else None)
                         for g in range(group)]
                for x, into in enumerate(outs):
                    per_head = torch.stack([p[x] for p in parts])
                    into.append(per_head if x < 2 else per_head.sum(0))
        shapes = [s["q"].shape, s["q"].shape, s["k"].shape, s["v"].shape]
        outs = [torch.stack(x).reshape(shape) for x, shape in zip(outs, shapes)]
        return outs if s["op"] == "train" else outs[0]
    if s["op"] == "cache":
        page, free = s["page"], s["free_pages"].tolist()
        table, cached, added = s["block_table"].tolist(), s["cached"].tolist(), s["added"].tolist()
        slots, starts, used = [], [0], 0
        for row, c, a in zip(table, cached, added):
            for p in range(c, c + a):
                if p % page == 0:  # a page begins
                    row[p // page] = free[used]
                    used += 1
                slots.append(row[p // page] * page + p % page)
            starts.append(len(slots))
        at = torch.tensor(slots, dtype=torch.long, device="cuda")
        for x in ("k", "v"):
            flat = s[x + "_cache"].transpose(1, 2).reshape(-1, case["kv_heads"], case["d"])
            flat = flat.index_copy(0, at, s[x][: len(slots)])
            s[x + "_cache"] = flat.reshape(-1, page, case["kv_heads"], case["d"]).transpose(1, 2)
        slots += [-1] * (s["capacity"] - len(slots))
        whole = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
        return [whole(table), whole(slots), whole(starts), whole([used]),
                s["k_cache"].contiguous(), s["v_cache"].contiguous()]
    outs = []
    for q, row, n in zip(s["q"], s["block_table"], s["lengths"].tolist()):
        window, sinks = s.get("window", 0), s.get("sinks", 0)
        seen = [j for j in range(n) if not window or n - j <= window or j < sinks]
        k, v = (_exact_rows(s[x], row, seen) for x in ("k_cache", "v_cache"))
        if s["op"] == "prefix":
            first = list(range(s["prefix_length"]))
            k, v = (torch.cat((_exact_rows(s[x], s["prefix_pages"], first), y), 1)
                    for x, y in (("k_cache", k), ("v_cache", v)))
        outs.append(_exact_request(q, k, v))
    return torch.stack(outs)
