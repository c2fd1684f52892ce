"""Measured cases of the operators on an 8-bit and on a windowed paged KV cache: writing it, reading it back, and
attending over it with single tokens and with chunks of new tokens.

Every operator has a plain form here (elementary torch operations in 32 bits, rounded once at the end), the call that
a user of the package makes instead of it, and its definition in 64 bits.

  write    ``reshape_and_cache_flash`` into a float8 cache: quantise each new K/V row as it is written
  gather   ``gather_cache_flash``: the rows of some sequences back out of the cache, packed and dequantised
  attend   ``flash_attn_varlen_func`` over a float8 cache (one new token, or a chunk of them, per sequence), and with
           a sliding window whose sequences keep their first tokens visible (float8 or 16-bit cache)

Lengths depend on the case alone (so that the work does too); values, page order and slots come from the seed.
"""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32,
         "e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
LARGEST = {torch.float8_e4m3fn: 448.0, torch.float8_e5m2: 57344.0}


def listed():
    return [
        # one decode step of 256 sequences writes one K/V row each, out of the fused projection's output
        dict(name="write step 256", op="write", tokens=256, kv_heads=8, dim=128, page=16, dtype="bf16", cache="e4m3",
             per_head=False, fused=True, spare=4096),
        # a mixed serving step: a few prompts and running sequences, odd row count, one scale for each head
        dict(name="write mixed 1355 e5m2", op="write", tokens=1355, kv_heads=4, dim=128, page=32, dtype="fp16",
             cache="e5m2", per_head=True, fused=False, spare=1024),
        # all prompt rows of a prefill batch of 16 sequences
        dict(name="write prompt 33355", op="write", tokens=33355, kv_heads=8, dim=128, page=16, dtype="bf16",
             cache="e4m3", per_head=True, fused=True, spare=2048),
        # a few cached prefixes read back for a short request
        dict(name="gather prefixes", op="gather", batch=5, shortest=1, longest=463, kv_heads=8, dim=128, page=16,
             dtype="bf16", cache="e4m3", per_head=False),
        # long cached contexts moved out of the cache in the type that the model computes in
        dict(name="gather contexts", op="gather", batch=16, shortest=512, longest=8192, kv_heads=8, dim=128, page=16,
             dtype="bf16", cache="e4m3", per_head=True),
        # single-token steps: a handful of chats (latency), and the full batch of the decode benchmark
        dict(name="decode chats", op="attend", batch=8, new_shortest=1, new_longest=1, shortest=18, longest=1328,
             heads=32, kv_heads=8, dim=128, page=16, dtype="bf16", cache="e4m3", window=-1, sinks=0),
        dict(name="decode batch 256", op="attend", batch=256, new_shortest=1, new_longest=1, shortest=512, longest=8192,
             heads=32, kv_heads=8, dim=128, page=16, dtype="bf16", cache="e4m3", window=-1, sinks=0),
        # a chunk of new tokens over the cached context: short continuations of a few long chats, and a prompt's chunk
        dict(name="chunk continuations", op="attend", batch=4, new_shortest=9, new_longest=33, shortest=1777,
             longest=16384, heads=32, kv_heads=8, dim=128, page=16, dtype="fp16", cache="e4m3", window=-1, sinks=0),
        dict(name="chunk prompt 2048", op="attend", batch=2, new_shortest=2000, new_longest=2048, shortest=4096,
             longest=8192, heads=32, kv_heads=8, dim=128, page=16, dtype="bf16", cache="e4m3", window=-1, sinks=0),
        # streaming chats far beyond the window: 4 first tokens and the last 1024 stay visible, 16-bit cache
        dict(name="sinks decode", op="attend", batch=64, new_shortest=1, new_longest=1, shortest=1000, longest=16384,
             heads=32, kv_heads=8, dim=128, page=16, dtype="bf16", cache="bf16", window=1023, sinks=4),
        # the same over an 8-bit cache with a longer window
        dict(name="sinks decode 8-bit", op="attend", batch=64, new_shortest=1, new_longest=1, shortest=5000,
             longest=16384, heads=32, kv_heads=8, dim=128, page=32, dtype="bf16", cache="e4m3", window=4095, sinks=4),
        # a prompt's chunk under the window
        dict(name="sinks chunk 1500", op="attend", batch=2, new_shortest=1100, new_longest=1500, shortest=2500,
             longest=12000, heads=32, kv_heads=8, dim=128, page=16, dtype="bf16", cache="bf16", window=2047, sinks=4),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kv_heads = rng.choice([1, 2, 4, 8])
    dim = rng.choice([128, 128, 128, 64, 256])
    page = rng.choice([16, 16, 32, 64, 128])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    cache = rng.choice(["e4m3", "e4m3", "e5m2"])
    kind = rng.choice(["write", "gather", "decode", "chunk", "sinks decode", "sinks chunk"])
    if kind == "write":
        return dict(op="write", tokens=spread(1, 33355), kv_heads=kv_heads, dim=dim, page=page,
                    dtype=rng.choice(["bf16", "fp16", "fp32"]), cache=cache, per_head=rng.random() < 0.5,
                    fused=rng.random() < 0.5, spare=spread(1, 4096))
    if kind == "gather":
        longest = spread(1, 8192)
        return dict(op="gather", batch=spread(1, 16), shortest=rng.randint(1, longest), longest=longest,
                    kv_heads=kv_heads, dim=dim, page=page, dtype=dtype, cache=cache, per_head=rng.random() < 0.5)
    group = rng.choice([1, 2, 4, 4, 7, 8, 16]) if kv_heads <= 4 else rng.choice([1, 2, 4, 4, 7, 8])
    c = dict(op="attend", heads=kv_heads * group, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype, cache=cache,
             window=-1, sinks=0)
    if kind.startswith("sinks"):
        c.update(window=spread(64, 4096) - 1, sinks=rng.choice([1, 4, 4, 16, 128]), cache=rng.choice([dtype, cache]))
    if kind.endswith("decode"):
        c.update(new_longest=1, longest=spread(32, 16384))
        held = 2 * c["longest"] * kv_heads * dim * (1 if c["cache"] in ("e4m3", "e5m2") else 2)
        c.update(batch=max(1, min(spread(1, 256), 2 * 10 ** 9 // held)))      # bytes of the cache
    else:
        c.update(new_longest=spread(2, 2048), longest=spread(32, 16384))
        c["longest"] = max(c["longest"], c["new_longest"])
        most = 2 ** 36 // (c["heads"] * c["new_longest"] * c["longest"] * dim)     # products of a head's rows
        c.update(batch=max(1, min(spread(1, 8), most)))
        c["longest"] = min(c["longest"], max(c["new_longest"], 2 ** 36 // (c["heads"] * c["new_longest"] * dim)))
    c.update(new_shortest=rng.randint(1, c["new_longest"]))
    c.update(shortest=rng.randint(c["new_longest"], c["longest"]))
    return c


def _lengths(n, lo, hi):
    """n lengths spread over [lo, hi], in no order; the longest is among them."""
    return [hi if i == n // 2 else lo + int(((i + 1) * 0.6180339887) % 1.0 * (hi - lo + 1)) for i in range(n)]


def _randn(gen, shape, spread=None):
    x = torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32)
    return x if spread is None else x.mul_(spread)


def _scales(gen, c):
    """A K and a V scale that put the largest values near the top of the type; one for all heads or one for each."""
    top = 6.0 / LARGEST[TYPES[c["cache"]]]
    n = c["kv_heads"] if c.get("per_head") else 1
    return tuple(top * (0.75 + 0.5 * torch.rand((n,), generator=gen, device=DEV)) for _ in range(2))


def _starts(lengths):
    cu = torch.zeros(len(lengths) + 1, dtype=torch.int32)
    cu[1:] = torch.tensor(lengths, dtype=torch.int32).cumsum(0)
    return cu.to(DEV)


def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)

    def fill(cache, scale):
        """Normal values with a spread for each head and channel, as the cache holds them, a few pages at a time."""
        step = max(1, (1 << 27) // max(1, cache[0].numel()))
        for i in range(0, cache.shape[0], step):
            x = _randn(gen, cache[i:i + step].shape, spread)
            if scale is not None:
                x = (x / scale.view(-1, 1)).clamp_(-LARGEST[cache.dtype], LARGEST[cache.dtype])
            cache[i:i + step] = x.to(cache.dtype)

    def paged(lengths):
        """A table of pages in a random order (entries behind a sequence's last page stay zero), and their number."""
        pages = [(n + page - 1) // page for n in lengths]
        order = torch.randperm(sum(pages), generator=gen, device=DEV).to(torch.int32)
        table = torch.zeros((len(lengths), max(pages)), dtype=torch.int32, device=DEV)
        at = 0
        for i, n in enumerate(pages):
            table[i, :n] = order[at:at + n]
            at += n
        return table, sum(pages)

    hk, d, page = c["kv_heads"], c["dim"], c["page"]
    cache_type, dtype = TYPES[c["cache"]], TYPES[c["dtype"]]
    eight = cache_type in LARGEST
    s = {"case": c, "k_scale": None, "v_scale": None}
    if eight:
        s["k_scale"], s["v_scale"] = _scales(gen, c)
    spread = (0.4 * _randn(gen, (hk, d))).exp()       # channels differ in size, as keys' channels do

    if c["op"] == "write":
        t = c["tokens"]
        rows = _randn(gen, (t, 6 if c["fused"] else 2, hk, d), spread).to(dtype)   # fused: 4 query heads per KV head
        s["key"], s["value"] = rows[:, -2], rows[:, -1]
        if not c["fused"]:
            s["key"], s["value"] = s["key"].contiguous(), s["value"].contiguous()
        blocks = (t + c["spare"] + page - 1) // page
        caches = []
        for scale in (s["k_scale"], s["v_scale"]):
            cache = torch.empty((blocks, page, hk, d), dtype=cache_type, device=DEV)
            fill(cache, scale)
            caches.append(cache)
        s["key_cache"], s["value_cache"] = caches
        s["slots"] = torch.randperm(blocks * page, generator=gen, device=DEV)[:t]
        return s

    lengths = _lengths(c["batch"], c["shortest"], c["longest"])
    s["table"], blocks = paged(lengths)
    for name in ("key_cache", "value_cache"):
        s[name] = torch.empty((blocks, page, hk, d), dtype=cache_type, device=DEV)
        fill(s[name], s["k_scale" if name == "key_cache" else "v_scale"])
    s["lens"] = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    s["max_k"] = max(lengths)

    if c["op"] == "gather":
        s["cu"], s["total"] = _starts(lengths), sum(lengths)
        s["key"] = torch.empty((s["total"], hk, d), dtype=dtype, device=DEV)
        s["value"] = torch.empty_like(s["key"])
        return s

    new = _lengths(c["batch"], c["new_shortest"], c["new_longest"])
    s["cu"], s["total"], s["max_q"] = _starts(new), sum(new), max(new)
    q = _randn(gen, (s["total"], c["heads"], d))
    if c["sinks"]:
        # the first tokens draw a good part of every query's attention, as they do in trained models
        u = _randn(gen, (hk, d))
        u /= u.norm(dim=-1, keepdim=True)
        q += 3.0 * u.repeat_interleave(c["heads"] // hk, 0)
        first = min(c["sinks"], min(lengths))
        at = torch.arange(first, device=DEV)
        rows = s["table"][:, at // page].long() * page + at % page
        k = (1.2 * math.sqrt(d) * u).expand(c["batch"], first, hk, d)
        if eight:
            k = (k / s["k_scale"].view(-1, 1)).clamp(-LARGEST[cache_type], LARGEST[cache_type])
        s["key_cache"].view(torch.uint8 if eight else cache_type).view(-1, hk, d)[rows] = \
            k.to(cache_type).view(torch.uint8) if eight else k.to(cache_type)
    s["q"] = q.to(dtype)
    s["scale"] = d ** -0.5
    return s


# ------------------------------------------------------------------------------------------------ the plain forms
def _as_float(rows, scale):
    """Cached rows [..., kv_heads, dim] in 32 bits; `scale` has one entry or one for each head."""
    return rows.float() if scale is None else rows.float() * scale.view(-1, 1)


def _pick(cache, index):
    """cache[index] for 8-bit types too."""
    return cache.view(torch.uint8)[index].view(cache.dtype) if cache.element_size() == 1 else cache[index]


def _plain_write(rows, cache, slots, scale):
    top = LARGEST[cache.dtype]
    q = (rows.float() / scale.view(-1, 1)).clamp(-top, top).to(cache.dtype)
    cache.view(torch.uint8).view(-1, *cache.shape[2:])[slots] = q.view(torch.uint8)


def _plain_gather(s):
    seq = torch.repeat_interleave(torch.arange(s["lens"].numel(), device=DEV), s["lens"], output_size=s["total"])
    pos = torch.arange(s["total"], device=DEV) - s["cu"][seq]
    page = s["key_cache"].shape[1]
    index = s["table"][seq, pos // page].long(), pos % page
    s["key"].copy_(_as_float(_pick(s["key_cache"], index), s["k_scale"]))
    s["value"].copy_(_as_float(_pick(s["value_cache"], index), s["v_scale"]))
    return s["key"], s["value"]


def _plain_attend(s):
    c, cu, lens = s["case"], s["cu"], s["lens"]
    b, h, hk, d = c["batch"], c["heads"], c["kv_heads"], c["dim"]
    new = cu[1:] - cu[:-1]
    i = torch.arange(s["max_q"], device=DEV)
    rows = (cu[:-1, None] + i).clamp(max=s["total"] - 1)
    q = s["q"][rows].float().view(b, -1, hk, h // hk, d).permute(0, 2, 3, 1, 4).reshape(b, hk, -1, d)
    table = s["table"].long()
    k = _as_float(_pick(s["key_cache"], table), s["k_scale"]).view(b, -1, hk, d).permute(0, 2, 3, 1)
    scores = (torch.matmul(q, k) * s["scale"]).view(b, hk, h // hk, s["max_q"], -1)
    del k
    j = torch.arange(scores.shape[-1], device=DEV)
    at = (i + (lens - new)[:, None])[:, :, None]             # the position of each new token in its sequence
    seen = (j <= at) & (j < lens[:, None, None])
    if c["window"] >= 0:
        seen &= (j >= at - c["window"]) | (j < c["sinks"])
    scores = scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = (scores - top.masked_fill(top == -math.inf, 0.0)).exp_()
    del scores
    total = p.sum(-1, keepdim=True)
    v = _as_float(_pick(s["value_cache"], table), s["v_scale"]).view(b, -1, hk, d).permute(0, 2, 1, 3)
    o = torch.matmul(p.view(b, hk, -1, p.shape[-1]), v).view(b, hk, h // hk, -1, d)
    o = o / total.masked_fill(total == 0, 1.0)
    seq = torch.repeat_interleave(torch.arange(b, device=DEV), new, output_size=s["total"])
    pos = torch.arange(s["total"], device=DEV) - cu[seq]
    return o.permute(0, 3, 1, 2, 4).reshape(b, -1, h, d)[seq, pos].to(s["q"].dtype)


# ------------------------------------------------------------------------------------------------ the calls
def _call(s):
    import flaggems_b200 as fg

    c = s["case"]
    kind = "fp8_" + c["cache"] if c["cache"] in ("e4m3", "e5m2") else "auto"
    if c["op"] == "write":
        fg.reshape_and_cache_flash(s["key"], s["value"], s["key_cache"], s["value_cache"], s["slots"], kind,
                                   s["k_scale"], s["v_scale"])
        return s["key_cache"], s["value_cache"]
    if c["op"] == "gather":
        fg.gather_cache_flash(s["key_cache"], s["value_cache"], s["key"], s["value"], s["table"], s["cu"], kind,
                              s["k_scale"], s["v_scale"])
        return s["key"], s["value"]
    return fg.flash_attn_varlen_func(
        s["q"], s["key_cache"], s["value_cache"], s["max_q"], s["cu"], s["max_k"], seqused_k=s["lens"],
        softmax_scale=s["scale"], causal=True, window_size=(c["window"], 0) if c["window"] >= 0 else (-1, -1),
        block_table=s["table"], k_descale=s["k_scale"], v_descale=s["v_scale"], sink_tokens=c["sinks"])


def run(state):
    if own:
        return _call(state)
    op = state["case"]["op"]
    if op == "write":
        _plain_write(state["key"], state["key_cache"], state["slots"], state["k_scale"])
        _plain_write(state["value"], state["value_cache"], state["slots"], state["v_scale"])
        return state["key_cache"], state["value_cache"]
    return _plain_gather(state) if op == "gather" else _plain_attend(state)


# ------------------------------------------------------------------------------------------------ the work
def work(case):
    c = case

    def visible(new, length):
        """(query, key) pairs that count, and keys that at least one new token sees."""
        first, window = length - new, c["window"]
        if window < 0:
            return sum(first + i + 1 for i in range(new)), length
        low = [max(0, first + i - window) for i in range(new)]
        return (sum(first + i + 1 - n + min(c["sinks"], n) for i, n in enumerate(low)),
                length - low[0] + min(c["sinks"], low[0]))

    size = {"bf16": 2, "fp16": 2, "fp32": 4, "e4m3": 1, "e5m2": 1}
    row = c["kv_heads"] * c["dim"]
    if c["op"] == "write":
        return {"bytes": 2 * c["tokens"] * row * (size[c["dtype"]] + size[c["cache"]]) + 8 * c["tokens"],
                "flops": 2 * c["tokens"] * row}
    lengths = _lengths(c["batch"], c["shortest"], c["longest"])
    table = sum((n + c["page"] - 1) // c["page"] for n in lengths) * 4
    if c["op"] == "gather":
        return {"bytes": 2 * sum(lengths) * row * (size[c["dtype"]] + size[c["cache"]]) + table,
                "flops": 2 * sum(lengths) * row}
    new = _lengths(c["batch"], c["new_shortest"], c["new_longest"])
    both = [visible(n, m) for n, m in zip(new, lengths)]
    return {"bytes": 2 * sum(k for _, k in both) * row * size[c["cache"]]
            + 2 * sum(new) * c["heads"] * c["dim"] * size[c["dtype"]],
            "flops": 4 * c["dim"] * c["heads"] * sum(p for p, _ in both)}


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    c, page = s["case"], case["page"]
    heads = range(c["kv_heads"])

    def scale_of(name, head):
        t = s[name]
        return 1.0 if t is None else float(t[head if t.numel() > 1 else 0].double())

    if c["op"] == "write":
        out = []
        for new, cache, scale in (("key", "key_cache", "k_scale"), ("value", "value_cache", "v_scale")):
            top = LARGEST[s[cache].dtype]
            values = s[cache].double()
            blocks, offsets = s["slots"] // page, s["slots"] % page
            for head in heads:
                x = s[new][:, head].double() / scale_of(scale, head)
                x = torch.minimum(torch.maximum(x, torch.tensor(-top, device=DEV)), torch.tensor(top, device=DEV))
                values[blocks, offsets, head] = x.to(s[cache].dtype).double()
            out.append(values)
        return tuple(out)

    def cached(name, which, b, length):
        """[length, kv_heads, dim] of sequence b in 64 bits."""
        pages = s["table"][b, :(length + page - 1) // page].tolist()
        raw = s[name].view(torch.uint8) if s[name].element_size() == 1 else s[name]
        rows = torch.cat([raw[p] for p in pages])[:length].view(s[name].dtype).double()
        return torch.stack([rows[:, head] * scale_of(which, head) for head in heads], 1)

    lengths = s["lens"].tolist()
    if c["op"] == "gather":
        return tuple(torch.cat([cached(n, w, b, m) for b, m in enumerate(lengths)])
                     for n, w in (("key_cache", "k_scale"), ("value_cache", "v_scale")))

    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    group = c["heads"] // c["kv_heads"]
    starts = s["cu"].tolist()
    for b, length in enumerate(lengths):
        begin, end = starts[b], starts[b + 1]
        k, v = cached("key_cache", "k_scale", b, length), cached("value_cache", "v_scale", b, length)
        where = torch.arange(length - (end - begin), length, device=DEV).view(-1, 1)
        key = torch.arange(length, device=DEV).view(1, -1)
        hidden = key > where
        if c["window"] >= 0:
            hidden |= (key + c["window"] < where) & (key >= c["sinks"])
        for head in range(c["heads"]):
            a = s["q"][begin:end, head].double() @ k[:, head // group].T * s["scale"]
            a[hidden] = -math.inf
            out[begin:end, head] = torch.softmax(a, -1) @ v[:, head // group]
    return out
