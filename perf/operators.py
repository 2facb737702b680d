"""Measured cases of the paged key/value cache and of sampling.

Three operators of a decoder's serving path:

* ``append``: the rows [q | k | v] of a QKV projection enter a paged cache.  Queries and keys are
  (optionally) RMS-normalised per head and rotated (rotate-half); the rotated queries come back, keys
  and values are stored as fp16 ("F16") or as 4-bit blocks ("Q4_0": 32 values x = d (c - 8) with an
  fp16 d and codes c in 0..15).  The stored keys and values of the new tokens are read back as values.
* ``attend``: causal grouped-query attention of the new tokens over the cache, optionally restricted
  to a sliding window plus the first ``sinks`` positions.
* ``sample``: one token per row of logits by temperature, top-k, top-p and min-p from given random
  numbers, with its log-probability.

``run`` computes them in plain torch where ``own`` is false and through the package where it is true.

A pool is a uint8 tensor [pages][kv heads][bytes of a page of one head].  With S tokens a page, D
values a head and n = D / 32 groups, those bytes are K then V; "F16": [S][D] halves each; "Q4_0":
[S][D / 2] bytes of codes, then [S][n] fp16 scales, each.  In a row of codes, nibble i of 32-bit word
p is value 32 (p % n) + 8 (p // n) + i of a key; nibble i of 16-bit word h is value
32 (h % n) + 4 (h // n) + i of a value.
"""

import torch

own = False

_DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------
def _append(name, **kw):
    c = {"op": "append", "name": name, "hq": 32, "hk": 8, "d": 128, "kv": "Q4_0", "page": 64, "type": "f32",
         "norm": False, "batch": 1, "new": 1, "past": 0, "theta": 5e5}
    c.update(kw)
    return c


def _attend(name, **kw):
    c = {"op": "attend", "name": name, "hq": 32, "hk": 8, "d": 128, "kv": "Q4_0", "page": 64, "type": "f16",
         "batch": 1, "new": 1, "past": 0, "window": 0, "sinks": 0}
    c.update(kw)
    return c


def _sample(name, **kw):
    c = {"op": "sample", "name": name, "batch": 1, "vocab": 32000, "type": "f32", "filters": "all"}
    c.update(kw)
    return c


def listed():
    return [
        # one decode step of the default decoder (32 query, 8 KV heads of 128), batch 1: latency
        _append("append_step_1", past=639),
        # a decode step of 64 sequences at mixed positions, normalised heads, 16-bit cache, small pages
        _append("append_step_64_norm_f16", kv="F16", type="bf16", norm=True, batch=64, past=4095, page=16),
        # eight prompts of mixed lengths up to 2048 entering a 4-bit cache, normalised heads
        _append("append_prompt_8x2048_norm", norm=True, batch=8, new=2048),
        # attention of a batch-1 decode step at the default context: latency
        _attend("attend_step_1x640", past=639),
        # decode step of 8 sequences, 16-bit cache, contexts up to 4096
        _attend("attend_step_8x4096_f16", kv="F16", type="bf16", batch=8, past=4095, page=16),
        # decode step of a full serving batch, mixed contexts up to 8192
        _attend("attend_step_64x8192", type="bf16", batch=64, past=8191),
        # one sequence with a very long context
        _attend("attend_step_1x131072", past=131071, page=128),
        # chunks of mixed lengths behind cached prefixes, sliding window and sinks, heads of 64 in groups of 7
        _attend("attend_chunk_4x1000_window", hq=28, hk=4, d=64, kv="F16", type="bf16", batch=4, new=1000, past=5000,
                window=1024, sinks=4, page=32),
        # a whole long prompt at once (the largest)
        _attend("attend_prompt_1x8192", new=8192),
        # one row of the default vocabulary, every filter
        _sample("sample_1x32000"),
        # a serving batch over a large vocabulary, every row its own filters
        _sample("sample_64x128000", batch=64, vocab=128000),
        # temperature alone over many rows of 16-bit logits
        _sample("sample_256x32000_bf16", batch=256, type="bf16", filters="temperature"),
    ]


def _log(rng, lo, hi):
    """A whole number, its logarithm uniform."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["append", "append", "step", "step", "chunk", "chunk", "sample", "sample"])
    hk = rng.choice([1, 2, 4, 8])
    g = rng.choice([1, 2, 4, 5, 7, 8])
    d = rng.choice([64, 128, 128])
    page = rng.choice([16, 32, 64, 128])
    kv = rng.choice(["F16", "Q4_0", "Q4_0"])
    if op == "append":
        batch = _log(rng, 1, 64)
        new = rng.choice([1, _log(rng, 1, max(1, 8192 // batch))])
        return {"op": "append", "hq": hk * g, "hk": hk, "d": d, "kv": kv, "page": page,
                "type": rng.choice(["f32", "f16", "bf16"]), "norm": rng.random() < 0.5, "batch": batch, "new": new,
                "past": _log(rng, 1, 8192) - 1, "theta": rng.choice([1e4, 5e5])}
    if op == "step":
        batch = _log(rng, 1, 64)
        return {"op": "attend", "hq": hk * g, "hk": hk, "d": d, "kv": kv, "page": page,
                "type": rng.choice(["f16", "bf16"]), "batch": batch, "new": 1,
                "past": _log(rng, 1, min(131072, 524288 // batch)) - 1, "window": rng.choice([0, 0, 500, 4096]),
                "sinks": rng.choice([0, 4])}
    if op == "chunk":
        batch = _log(rng, 1, 8)
        new = _log(rng, 2, 4096 // batch)
        return {"op": "attend", "hq": hk * min(g, 4), "hk": hk, "d": d, "kv": kv, "page": page,
                "type": rng.choice(["f16", "bf16"]), "batch": batch, "new": new,
                "past": rng.choice([0, _log(rng, 1, 4096)]), "window": rng.choice([0, 0, 300, 2000]),
                "sinks": rng.choice([0, 4])}
    batch = _log(rng, 1, 256)
    return {"op": "sample", "batch": batch, "vocab": _log(rng, 1000, min(200000, 16000000 // batch)),
            "type": rng.choice(["f32", "f16", "bf16"]), "filters": rng.choice(["all", "all", "temperature", "top_p"])}


# ---------------------------------------------------------------------------------------------
# the pool's 4-bit rows
# ---------------------------------------------------------------------------------------------
def _dims(d, part):
    """The value that each nibble of a row of codes holds (part "k" or "v")."""
    n, w = d // 32, 8 if part == "k" else 4
    i = torch.arange(d, device="cuda")
    p = i // w
    return 32 * (p % n) + w * (p // n) + i % w


def _quantise(x):
    """Codes and fp16 scales of rows x [..., D]: d = (the value of largest magnitude, the first of equals) / -8,
    codes floor(x / d + 8.5) in 0..15."""
    g = x.unflatten(-1, (-1, 32))
    mag = g.abs()
    at = torch.where(mag == mag.amax(-1, keepdim=True), torch.arange(32, device=x.device, dtype=torch.int8), 32)
    first = g.gather(-1, at.amin(-1, keepdim=True).clamp(max=31).long())
    d = (first.float() / -8).half()
    q = torch.floor(g / d.to(g.dtype) + 8.5).clamp(0, 15)
    codes = torch.where(d == 0, 8, q).to(torch.uint8)
    return codes.flatten(-2), d.squeeze(-1)


def _pack(codes, part):
    b = codes[..., _dims(codes.shape[-1], part)].unflatten(-1, (-1, 2))
    return b[..., 0] | (b[..., 1] << 4)


def _parts(pool, case):
    """Views of the pool: {"k": (codes, scales)} or {"k": (halves,)}, and "v"."""
    s, d = case["page"], case["d"]
    half = pool.shape[-1] // 2
    got = {}
    for part, o in (("k", 0), ("v", half)):
        if case["kv"] == "F16":
            got[part] = (pool[..., o:o + half].unflatten(-1, (s, 2 * d)),)
        else:
            c = s * d // 2
            got[part] = (pool[..., o:o + c].unflatten(-1, (s, d // 2)),
                         pool[..., o + c:o + half].unflatten(-1, (s, d // 16)))
    return got


def _values(rows, scales, part, d):
    """Rows of codes and the bytes of their scales as 32-bit values."""
    nib = torch.stack((rows & 15, rows >> 4), -1).flatten(-2)
    back = torch.empty(d, dtype=torch.long, device="cuda")
    back[_dims(d, part)] = torch.arange(d, device="cuda")
    c = nib[..., back].float().unflatten(-1, (-1, 32)) - 8
    return (c * scales.contiguous().view(torch.float16).float()[..., None]).flatten(-2)


def _head_bytes(case):
    s, d = case["page"], case["d"]
    return 2 * s * 2 * d if case["kv"] == "F16" else 2 * s * (d // 2 + d // 16)


# ---------------------------------------------------------------------------------------------
# prepare
# ---------------------------------------------------------------------------------------------
def _lengths(case):
    """(new tokens, tokens in the cache with them) of each sequence, the same in every seed."""
    b, new, past = case["batch"], case["new"], case["past"]
    ql = [new if i == 0 else 1 + (i * 7919 * 31) % new for i in range(b)]
    pl = [past if i == 0 else (i * 104729 * 17) % (past + 1) for i in range(b)]
    return ql, [q + p for q, p in zip(ql, pl)]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dev = dict(device="cuda")

    def normal(*shape):
        return torch.randn(*shape, generator=g, **dev)

    if case["op"] == "sample":
        b, v = case["batch"], case["vocab"]
        logits = normal(b, v) * 2.5                     # most of a vocabulary, and a few likely tokens
        hot = torch.randint(0, v, (b, 24), generator=g, **dev)
        logits.scatter_add_(1, hot, normal(b, 24).abs() * 4)
        s = {"case": case, "logits": logits.to(_DT[case["type"]]), "u": torch.rand(b, generator=g, **dev)}

        def uniform(lo, hi):
            return lo + (hi - lo) * torch.rand(b, generator=g, **dev)

        s["temperature"] = uniform(0.5, 1.3)
        s["top_k"] = torch.zeros(b, dtype=torch.int32, **dev)
        s["top_p"] = torch.ones(b, **dev)
        s["min_p"] = torch.zeros(b, **dev)
        if case["filters"] in ("all", "top_p"):
            s["top_p"] = uniform(0.7, 1.0)
        if case["filters"] == "all":                    # half of the rows each, and greedy rows among them
            s["top_k"] = torch.randint(1, 400, (b,), generator=g, **dev, dtype=torch.int32)
            s["top_k"][1::2] = 0
            s["min_p"] = uniform(0.0, 0.1)
            s["min_p"][2::3] = 0
            s["temperature"][5::9] = 0
        return s
    hq, hk, d, page = case["hq"], case["hk"], case["d"], case["page"]
    ql, kl = _lengths(case)
    width = -(-max(kl) // page)
    need = [-(-k // page) for k in kl]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, **dev).int()
    table = torch.zeros(case["batch"], width, dtype=torch.int32, **dev)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    total = sum(ql)
    s = {"case": case, "table": table, "lens": torch.tensor(kl, dtype=torch.int32, **dev), "tokens": total,
         "cu": None, "max_q": max(ql), "max_kv": max(kl),
         "pool": torch.zeros(pages, hk, _head_bytes(case), dtype=torch.uint8, **dev)}
    if case["new"] > 1:
        cu = [0]
        for q in ql:
            cu.append(cu[-1] + q)
        s["cu"] = torch.tensor(cu, dtype=torch.int32, **dev)
    if case["op"] == "append":
        s["qkv"] = normal(total, (hq + 2 * hk) * d).to(_DT[case["type"]])
        ang = torch.arange(max(kl), dtype=torch.float64, **dev)[:, None] / case["theta"] ** (
            torch.arange(0, d, 2, dtype=torch.float64, **dev) / d)
        s["rope"] = torch.stack((ang.cos(), ang.sin()), -1).float()
        s["q_norm"] = 1 + 0.1 * normal(d) if case["norm"] else None
        s["k_norm"] = 1 + 0.1 * normal(d) if case["norm"] else None
    else:
        s["q"] = (normal(total, hq, d) * 1.5).to(_DT[case["type"]])
        step = max(1, (1 << 26) // (hk * page * d))
        for p0 in range(0, pages, step):                # a cache that earlier tokens have filled
            v = _parts(s["pool"][p0:p0 + step], case)
            for part in ("k", "v"):
                x = normal(min(step, pages - p0), hk, page, d)
                if case["kv"] == "F16":
                    v[part][0].copy_(x.half().view(torch.uint8))
                else:
                    codes, scale = _quantise(x)
                    v[part][0].copy_(_pack(codes, part))
                    v[part][1].copy_(scale.contiguous().view(torch.uint8))
    if own:
        from xanosmerks_b200.kvcache import PagedKVCache
        s["cache"] = PagedKVCache(pages, hk, d, page, case["kv"], pool=s["pool"])
    return s


# ---------------------------------------------------------------------------------------------
# run
# ---------------------------------------------------------------------------------------------
def _where(s):
    """Sequence and position of each new token."""
    t = torch.arange(s["tokens"], device="cuda")
    if s["cu"] is None:
        return t, s["lens"].long() - 1
    seq = torch.bucketize(t, s["cu"][1:].long(), right=True)
    end = s["cu"][1:].long()[seq]
    return seq, s["lens"].long()[seq] - end + t


def _plain_append(s):
    case = s["case"]
    hq, hk, d, page = case["hq"], case["hk"], case["d"], case["page"]
    seq, pos = _where(s)
    # 64 bits for keys that become codes: a value next to a border between two codes goes one way
    wide = torch.float64 if case["kv"] == "Q4_0" else torch.float32

    def turned(x, w):
        if w is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-5) * w.to(x.dtype)
        cos, sin = s["rope"].to(x.dtype)[pos][:, None].unbind(-1)
        a, b = x[..., :d // 2], x[..., d // 2:]
        return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)

    rows = s["qkv"].unflatten(-1, (-1, d))
    q = turned(rows[:, :hq].float(), s["q_norm"]).to(torch.float16 if case["type"] == "f32" else _DT[case["type"]])
    new = {"k": turned(rows[:, hq:hq + hk].to(wide), s["k_norm"]).float(), "v": rows[:, hq + hk:].float()}
    at, slot = s["table"].long()[seq, pos // page], pos % page
    parts, got = _parts(s["pool"], case), {"q": q}
    for part, x in new.items():
        if case["kv"] == "F16":
            got[part] = x.half()
            parts[part][0][at, :, slot] = got[part].view(torch.uint8)
        else:
            codes, scale = _quantise(x.double())
            parts[part][0][at, :, slot] = _pack(codes, part)
            parts[part][1][at, :, slot] = scale.contiguous().view(torch.uint8)
            got[part] = ((codes.float().unflatten(-1, (-1, 32)) - 8) * scale.float()[..., None]).flatten(-2).half()
    return got


def _plain_attend(s):
    case = s["case"]
    hq, hk, d, page = case["hq"], case["hk"], case["d"], case["page"]
    seq, pos = _where(s)
    b, mq, g = case["batch"], s["max_q"], hq // hk
    parts = _parts(s["pool"], case)

    def cached(part):                                   # [batch][kv heads][keys][D]
        got = [x[s["table"].long()].transpose(1, 2).flatten(2, 3) for x in parts[part]]
        if case["kv"] == "F16":
            return got[0].contiguous().view(torch.float16).float()
        return _values(got[0], got[1], part, d)

    first = torch.arange(b, device="cuda") if s["cu"] is None else s["cu"][:-1].long()
    row = (first[:, None] + torch.arange(mq, device="cuda")).clamp(max=s["tokens"] - 1)
    q = s["q"][row].float().unflatten(2, (hk, g)).permute(0, 2, 3, 1, 4).flatten(2, 3)
    score = (q * d ** -0.5) @ cached("k").transpose(-1, -2)
    key = torch.arange(score.shape[-1], device="cuda")
    at = pos[row][:, None, None, :, None]
    seen = key <= at
    if case["window"]:
        seen = seen & ((key > at - case["window"]) | (key < case["sinks"]))
    score = score.unflatten(2, (g, mq)).masked_fill_(~seen, float("-inf"))
    top = score.amax(-1, keepdim=True)
    p = score.sub_(torch.where(top == float("-inf"), 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    o = (p.flatten(2, 3) @ cached("v")).unflatten(2, (g, mq)) / torch.where(total == 0, 1.0, total)
    o = o.permute(0, 3, 1, 2, 4).flatten(2, 3)          # [batch][row][query heads][D]
    return {"out": o[seq, torch.arange(s["tokens"], device="cuda") - first[seq]].to(s["q"].dtype)}


def _plain_sample(s):
    x = s["logits"].double()
    t = s["temperature"].double()[:, None]
    w = ((x - x.amax(-1, keepdim=True)) / torch.where(t == 0, 1.0, t)).exp()
    v = x.shape[-1]
    big, order = w.sort(dim=-1, descending=True, stable=True)
    rank = torch.arange(v, device="cuda")
    k = s["top_k"].long()[:, None]
    k = torch.where(k <= 0, v, k)
    k = torch.where(t == 0, 1, k)
    big = big * (rank < k)
    before = big.cumsum(-1) - big
    p = s["top_p"].double()[:, None]
    keep = (rank < k) & ((p >= 1) | (before < p * big.sum(-1, keepdim=True)) | (rank == 0))
    keep = keep & (big >= s["min_p"].double()[:, None] * big[:, :1])
    w = w * torch.zeros_like(w).scatter_(1, order, keep.double())
    c = w.cumsum(-1)
    ids = (c <= s["u"].double()[:, None] * c[:, -1:]).sum(-1, keepdim=True)
    logp = (w.gather(1, ids) / c[:, -1:]).log()
    return {"ids": ids[:, 0].int(), "logprob": logp[:, 0].float()}


def run(state):
    s = state
    case = s["case"]
    if not own:
        return {"append": _plain_append, "attend": _plain_attend, "sample": _plain_sample}[case["op"]](s)
    if case["op"] == "append":
        c = s["cache"]
        q = c.append(s["qkv"], case["hq"], s["table"], s["lens"], s["cu"], rope=s["rope"], q_norm=s["q_norm"],
                     k_norm=s["k_norm"], eps=1e-5)
        k, v = c.read(s["table"], s["lens"], s["cu"], num_tokens=s["tokens"])
        return {"q": q, "k": k, "v": v}
    if case["op"] == "attend":
        return {"out": s["cache"].attend(s["q"], s["table"], s["lens"], s["cu"], window=case["window"],
                                         sinks=case["sinks"])}
    from xanosmerks_b200.sampling import sample
    ids, logp = sample(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                       min_p=s["min_p"])
    return {"ids": ids, "logprob": logp}


# ---------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------
def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}
    if case["op"] == "sample":
        n = case["batch"] * case["vocab"]
        return {"bytes": n * size[case["type"]] + case["batch"] * 28, "flops": 3 * n}
    hq, hk, d = case["hq"], case["hk"], case["d"]
    ql, kl = _lengths(case)
    t = sum(ql)
    row = 2 * d if case["kv"] == "F16" else d // 2 + d // 16      # bytes of a key or value in the cache
    if case["op"] == "append":
        # rows in, rotated queries, stored rows, the stored rows read and returned as halves
        b = t * ((hq + 2 * hk) * d * size[case["type"]] + hq * d * 2 + 2 * hk * (2 * row + 2 * d) + 4 * d)
        return {"bytes": b, "flops": t * (hq + hk) * d * 3}
    keys = pairs = 0
    for q, k in zip(ql, kl):
        w = case["window"] or k + 1
        for j in range(q):                              # position k - q + j sees this many keys
            n = k - q + j + 1
            pairs += min(n, w + min(case["sinks"], max(0, n - w)))
        oldest = max(0, k - q + 1 - w)
        keys += k - oldest + min(case["sinks"], oldest)
    return {"bytes": keys * hk * 2 * row + 2 * t * hq * d * 2, "flops": 4 * pairs * hq * d}


# ---------------------------------------------------------------------------------------------
# the definitions in 64 bits, written apart
# ---------------------------------------------------------------------------------------------
def _exact_blocks(x):
    """What Q4_0 blocks stand for: the codes by counting the borders (j - 8.5) d that a value has passed."""
    rows = x.reshape(-1, 32)
    up, down = rows.max(-1).values, rows.min(-1).values
    big = torch.maximum(up, -down)
    both = (up == -down) & (up > 0)
    a = torch.where(up >= -down, up, down)
    if bool(both.any()):                                # equal magnitudes of both signs: the first one counts
        r = rows[both]
        lead = (r.abs() == big[both][:, None]).int().cumsum(-1).eq(0).sum(-1)
        a[both] = r[torch.arange(len(r), device=r.device), lead]
    d = (-a / 8).half().double()
    code = torch.zeros_like(rows)
    for j in range(1, 16):
        border = (j - 8.5) * d[:, None]
        code += torch.where(d[:, None] > 0, rows >= border, rows <= border).double()
    return torch.where(d[:, None] == 0, 0.0, (code - 8) * d[:, None]).reshape(x.shape)


def _exact_append(s, case):
    hq, hk, d = case["hq"], case["hk"], case["d"]
    ql, kl = _lengths(case)
    at = torch.cat([torch.arange(k - q, k, device="cuda") for q, k in zip(ql, kl)])
    turn = torch.view_as_complex(s["rope"].double())[at]
    x = s["qkv"].double().reshape(s["tokens"], hq + 2 * hk, d)

    def heads(y, w):
        if w is not None:
            y = y / torch.sqrt(y.square().sum(-1, keepdim=True) / d + 1e-5) * w.double()
        z = torch.complex(y[..., :d // 2], y[..., d // 2:]) * turn[:, None, :]
        return torch.cat((z.real, z.imag), -1)

    k, v = heads(x[:, hq:hq + hk], s["k_norm"]), x[:, hq + hk:]
    if case["kv"] == "Q4_0":
        k, v = _exact_blocks(k.float().double()), _exact_blocks(v)
    return {"q": heads(x[:, :hq], s["q_norm"]), "k": k, "v": v}


def _exact_rows(s, case, i, n, h):
    """Keys and values 0..n-1 of sequence i, KV head h, in 64 bits."""
    page, d = case["page"], case["d"]
    pages = s["table"][i, :-(-n // page)].long()
    raw = s["pool"][pages, h]
    half = raw.shape[1] // 2
    out = []
    for part, wide in ((0, 8), (1, 4)):
        b = raw[:, part * half:(part + 1) * half]
        if case["kv"] == "F16":
            out.append(b.contiguous().view(torch.float16).reshape(-1, d)[:n].double())
            continue
        word = b[:, :page * d // 2].contiguous().view(torch.int32 if wide == 8 else torch.int16).reshape(-1, d // wide)
        scale = b[:, page * d // 2:].contiguous().view(torch.float16).reshape(-1, d // 32).double()
        nib = torch.stack([(word >> (4 * e)) & 15 for e in range(wide)], -1).double() - 8    # [key][word][nibble]
        grouped = nib.reshape(nib.shape[0], -1, d // 32, wide).transpose(1, 2)               # [key][group][word][nibble]
        out.append((grouped.reshape(-1, d // 32, 32) * scale[..., None]).reshape(-1, d)[:n])
    return out


def _exact_attend(s, case):
    hq, hk, d = case["hq"], case["hk"], case["d"]
    ql, kl = _lengths(case)
    g, o, t0 = hq // hk, torch.zeros(s["tokens"], hq, d, dtype=torch.float64, device="cuda"), 0
    for i, (m, n) in enumerate(zip(ql, kl)):
        for h in range(hk):
            k, v = _exact_rows(s, case, i, n, h)
            for j0 in range(0, m, 1024):
                j1 = min(m, j0 + 1024)
                pos = torch.arange(n - m + j0, n - m + j1, device="cuda")[:, None]
                key = torch.arange(n, device="cuda")[None, :]
                hide = key > pos
                if case["window"]:
                    hide |= (key <= pos - case["window"]) & (key >= case["sinks"])
                for e in range(g):
                    q = s["q"][t0 + j0:t0 + j1, h * g + e].double()
                    z = torch.matmul(q, k.T) / d ** 0.5
                    o[t0 + j0:t0 + j1, h * g + e] = torch.softmax(z.masked_fill(hide, -torch.inf), -1) @ v
        t0 += m
    return {"out": o}


def _exact_sample(s, case):
    ids, logp = [], []
    for r in range(case["batch"]):
        x, t = s["logits"][r].double(), float(s["temperature"][r])
        if t == 0:
            ids.append(int((x == x.max()).nonzero()[0]))
            logp.append(0.0)
            continue
        l = torch.log_softmax(x / t, 0)
        order = torch.argsort(-l, stable=True)
        k = int(s["top_k"][r])
        n = min(k, len(order)) if k > 0 else len(order)
        pr = l[order[:n]].exp()
        c = pr.cumsum(0) / pr.sum()
        top_p = float(s["top_p"][r])
        if top_p < 1:
            n = min(n, 1 + int((c < top_p).sum()))
        n = min(n, int((l[order[:n]] - l[order[0]] >= torch.log(s["min_p"][r].double())).sum()))
        kept = order[:n].sort().values
        q = l[kept].exp()
        c = q.cumsum(0) / q.sum()
        i = min(int((c <= float(s["u"][r])).sum()), n - 1)
        ids.append(int(kept[i]))
        logp.append(float((q[i] / q.sum()).log()))
    return {"ids": torch.tensor(ids, dtype=torch.int32, device="cuda"),
            "logprob": torch.tensor(logp, dtype=torch.float64, device="cuda")}


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "sample": _exact_sample}[case["op"]](s, case)
