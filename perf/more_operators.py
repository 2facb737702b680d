"""Measured cases of a mixture-of-experts step, of block norms with their residual, and of token log-probabilities.

Three operators of a decoder's serving path:

* ``moe``: the whole mixture-of-experts layer for a few tokens.  Each row of x is (optionally) RMS-normalised, the router
  picks the k experts of the largest logits (equal logits: the lower expert), softmax over those logits gives their
  weights, and the result is the weighted sum of w2 (act(w1 x) * (w3 x)) over them, added to a residual if there is one.
  The experts' weights are GGUF blocks (Q4_K, Q5_K, Q6_K or Q8_0).
* ``norm``: what stands between two blocks: the output y of one is (optionally) RMS-normalised, gated, scaled and added to
  the residual stream, and the stream is (optionally) normalised for the next block.
* ``logp``: log-probability and rank of given tokens, the entropy of each row of logits, and its largest alternatives.

``run`` computes them in plain torch where ``own`` is false and through the package where it is true.

A weight of n rows of k values is n * k / QK records in the order of the rows.  "Q4_K" (256 values in 144 bytes): fp16 d
and dmin, twelve bytes with eight pairs (s, m) of 6 bits, 128 bytes of 4-bit codes; sub-block j of 32 values is
d s_j c - dmin m_j.  "Q5_K" (176 bytes): the same with a fifth bit of each code: bit l of the little-endian word j / 2 of
the 32 bytes before the codes.  "Q6_K" (210 bytes): 128 bytes of low nibbles, 64 bytes of high pairs of bits, sixteen int8
scales s, fp16 d; 16 values are d s_j (c - 32).  "Q8_0" (32 values in 34 bytes): fp16 d, 32 int8 codes; d c.
"""

import torch

own = False

_DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_RECORD = {"Q4_K": (256, 144), "Q5_K": (256, 176), "Q6_K": (256, 210), "Q8_0": (32, 34)}


# ---------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------
def _moe(name, **kw):
    c = {"op": "moe", "name": name, "tokens": 1, "experts": 8, "top": 2, "hidden": 4096, "inter": 14336, "kind": "Q4_K",
         "type": "f32", "act": "silu", "norm": True, "residual": True}
    c.update(kw)
    return c


def _norm(name, **kw):
    c = {"op": "norm", "name": name, "batch": 1, "rows": 1, "dim": 4096, "stream": "f32", "type": "f32", "post": True,
         "pre": True, "gate": "none", "scale": 1.0}
    c.update(kw)
    return c


def _logp(name, **kw):
    c = {"op": "logp", "name": name, "rows": 1, "vocab": 32000, "type": "f32", "top": 0, "masked": 0, "temperature": 1.0}
    c.update(kw)
    return c


def listed():
    return [
        # one decode step of the benchmark's block (8 experts, 2 of them a token), batch 1, on the residual stream
        _moe("moe_1x8"),
        # a small serving batch, seven sequences, on 16-bit rows that are already normalised
        _moe("moe_7x8_bf16", tokens=7, type="bf16", norm=False, residual=False),
        # many small experts, batch 1: little to read, latency
        _moe("moe_1x128_small", experts=128, top=8, hidden=2048, inter=768),
        # many small experts, a batch with an odd number of sequences, 6-bit weights: most experts are met
        _moe("moe_33x128_small_q6", tokens=33, experts=128, top=8, hidden=2048, inter=768, kind="Q6_K"),
        # between two blocks of a decode step
        _norm("norm_1"),
        # a serving batch of decode steps, a residual scale, a block output in 16 bits
        _norm("norm_64_scaled", rows=64, type="f16", scale=0.22),
        # a long prompt, the stream in fp32, block outputs in 16 bits
        _norm("norm_8192", rows=8192, type="bf16"),
        # image tokens: four sequences, each with its own gate, everything in 16 bits, an odd width
        _norm("norm_4x1111_gated", batch=4, rows=1111, dim=1154, stream="bf16", type="bf16", gate="sequence"),
        # one row of the default vocabulary with a few alternatives: latency
        _logp("logp_1x32000", top=5),
        # a serving batch over a large vocabulary with a masked tail, at a temperature
        _logp("logp_64x128000_bf16", rows=64, vocab=128000, type="bf16", top=20, masked=1000, temperature=0.7),
        # a prompt scored, fp32 logits, no alternatives
        _logp("logp_2048x32000", rows=2048),
        # a chunk of a corpus scored over an odd vocabulary (the largest)
        _logp("logp_2000x128001_f16", rows=2000, vocab=128001, type="f16", top=8),
    ]


def _log(rng, lo, hi):
    """A whole number, its logarithm uniform."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["moe", "norm", "logp"])
    if op == "moe":
        tokens = _log(rng, 1, 64)
        hidden = 256 * _log(rng, 1, 24)
        # as much to read as the largest listed case has, at most
        inter = 256 * _log(rng, 1, min(56, (4096 * 14336) // (256 * hidden)))
        experts = _log(rng, 2, max(2, min(160, 8 * 4096 * 14336 // (hidden * inter))))
        top = _log(rng, 1, min(experts, 8))
        return {"op": op, "tokens": tokens, "experts": experts, "top": top, "hidden": hidden, "inter": inter,
                "kind": rng.choice(["Q4_K", "Q4_K", "Q5_K", "Q6_K", "Q8_0"]), "type": rng.choice(["f32", "f16", "bf16"]),
                "act": rng.choice(["silu", "silu", "gelu", "relu"]), "norm": rng.random() < 0.6,
                "residual": rng.random() < 0.6}
    if op == "norm":
        batch, dim = _log(rng, 1, 16), _log(rng, 64, 16384)
        return {"op": op, "batch": batch, "rows": _log(rng, 1, max(1, min(8192, 33000000 // dim) // batch)), "dim": dim,
                "stream": rng.choice(["f32", "f32", "f16", "bf16"]), "type": rng.choice(["f32", "f16", "bf16"]),
                "post": rng.random() < 0.7, "pre": rng.random() < 0.8,
                "gate": rng.choice(["none", "none", "channel", "sequence", "row"]), "scale": rng.choice([1.0, 0.22, 1.4])}
    vocab = _log(rng, 500, 260000)
    return {"op": op, "rows": _log(rng, 1, min(4096, 120000000 // vocab)), "vocab": vocab,
            "type": rng.choice(["f32", "f16", "bf16"]), "top": rng.choice([0, 1, 5, _log(rng, 1, 64)]),
            "masked": rng.choice([0, 0, vocab // 10]), "temperature": rng.choice([1.0, 1.0, 0.6, 1.3])}


# ---------------------------------------------------------------------------------------------
# prepare
# ---------------------------------------------------------------------------------------------
def _weights(g, kind, n, count):
    """`count` weights of n values each as random blocks, values of a mean of zero and an rms near 0.02."""
    qk, rec = _RECORD[kind]
    blocks = count * n // qk
    b = torch.randint(0, 256, (blocks, rec), dtype=torch.uint8, device="cuda", generator=g)

    def put(at, v):
        b[:, at:at + 2] = v.half().view(torch.uint8).view(blocks, 2)

    size = 0.7 + 0.6 * torch.rand(blocks, 1, device="cuda", generator=g)
    if kind == "Q4_K":
        put(0, size * 9e-5)
        put(2, size * 7.5 * 9e-5)
    elif kind == "Q5_K":
        put(0, size * 4.5e-5)
        put(2, size * 15.5 * 4.5e-5)
    elif kind == "Q6_K":
        put(208, size * 1.5e-5)
    else:
        put(0, size * 2.7e-4)
    return b.view(count, -1)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dev = dict(device="cuda")

    def normal(*shape):
        return torch.randn(*shape, generator=g, **dev)

    s = {"case": case}
    if case["op"] == "moe":
        t, e, h, f = case["tokens"], case["experts"], case["hidden"], case["inter"]
        s["gate"] = normal(e, h) / h ** 0.5
        s["w1"], s["w3"], s["w2"] = (_weights(g, case["kind"], h * f, e) for _ in range(3))
        s["x"] = (normal(t, h) * (0.5 + torch.rand(t, 1, generator=g, **dev))).to(_DT[case["type"]])
        s["norm"] = 1 + 0.1 * normal(h) if case["norm"] else None
        s["residual"] = normal(t, h) if case["residual"] else None
        if own:
            from xanosmerks_b200.moe import MoELayer
            from xanosmerks_b200.ops import GGUFTensor
            shape = {"w1": (f, h), "w3": (f, h), "w2": (h, f)}
            s["layer"] = MoELayer(
                {"num_experts": e, "num_experts_per_tok": case["top"], "hidden_act": case["act"]},
                {"gate": {"weight": s["gate"]},
                 "experts": {str(i): {w: {"weight": GGUFTensor(s[w][i], case["kind"], shape[w])} for w in shape}
                             for i in range(e)}})
        return s
    if case["op"] == "norm":
        b, r, d = case["batch"], case["rows"], case["dim"]
        s["stream"] = (normal(b, r, d) * 2).to(_DT[case["stream"]])
        s["y"] = (normal(b, r, d) * (0.1 + torch.rand(b, r, 1, generator=g, **dev))).to(_DT[case["type"]])
        s["post"] = 1 + 0.1 * normal(d) if case["post"] else None
        s["pre"] = 1 + 0.1 * normal(d) if case["pre"] else None
        shape = {"none": None, "channel": (d,), "sequence": (b, 1, d), "row": (b, r, 1)}[case["gate"]]
        s["gate"] = None if shape is None else torch.tanh(normal(*shape)).to(_DT[case["type"]])
        return s
    r, v = case["rows"], case["vocab"]
    logits = normal(r, v) * 2.5                             # most of a vocabulary, and a few likely tokens
    hot = torch.randint(0, v, (r, 24), generator=g, **dev)
    logits.scatter_add_(1, hot, normal(r, 24).abs() * 4)
    if case["masked"]:
        logits[:, v - case["masked"]:] = float("-inf")
    s["logits"] = logits.to(_DT[case["type"]])
    some = torch.randint(0, v - case["masked"], (r,), generator=g, **dev)
    s["tokens"] = torch.where(torch.arange(r, **dev) % 3 == 0, some, hot[:, 0].clamp(max=v - case["masked"] - 1))
    return s


# ---------------------------------------------------------------------------------------------
# run
# ---------------------------------------------------------------------------------------------
def _halves(b, at):
    return b[..., at:at + 2].contiguous().view(torch.float16).float()


def _pairs(b):
    """The eight scales and eight minima of twelve bytes, as fp32 [..., 8]."""
    low, mid, top = b[..., 0:4], b[..., 4:8], b[..., 8:12]
    s = torch.cat((low & 63, (top & 15) | ((low >> 6) << 4)), -1)
    m = torch.cat((mid & 63, (top >> 4) | ((mid >> 6) << 4)), -1)
    return s.float(), m.float()


def _values(raw, kind, n, k):
    """Blocks [count, bytes] as fp32 values [count, n, k]."""
    qk, rec = _RECORD[kind]
    b = raw.view(raw.shape[0], n, k // qk, rec)
    if kind == "Q8_0":
        return (_halves(b, 0) * b[..., 2:].view(torch.int8).float()).flatten(-2)
    if kind == "Q6_K":
        low = b[..., :128].unflatten(-1, (2, 1, 2, 32))
        high = b[..., 128:192].unflatten(-1, (2, 1, 1, 32))
        c = torch.cat((low & 15, low >> 4), -3)             # [half][nibble][of two][32]
        turn = torch.tensor([[0, 2], [4, 6]], dtype=torch.uint8, device="cuda")[:, :, None]
        c = (c | (((high >> turn) & 3) << 4)).float() - 32
        scale = _halves(b, 208) * b[..., 192:208].view(torch.int8).float()
        return (c.flatten(-4).unflatten(-1, (16, 16)) * scale[..., None]).flatten(-3)
    s, m = _pairs(b[..., 4:16])
    at = 16 if kind == "Q4_K" else 48
    q = b[..., at:at + 128].unflatten(-1, (4, 1, 32))
    c = torch.cat((q & 15, q >> 4), -2)
    if kind == "Q5_K":
        bit = torch.arange(8, dtype=torch.uint8, device="cuda")
        fifth = (b[..., 16:32, None] >> bit) & 1            # bit l of word j
        c = c | (fifth.flatten(-2).unflatten(-1, (4, 1, 32)) << 4)
    c = c.flatten(-3, -2).float()
    return ((_halves(b, 0) * s)[..., None] * c - (_halves(b, 2) * m)[..., None]).flatten(-3)


def _act(name, x):
    if name == "gelu":
        return 0.5 * x * (1 + torch.tanh(0.7978845608 * (x + 0.044715 * x * x * x)))
    return x.clamp(min=0) if name == "relu" else x / (1 + (-x).exp())


def _plain_moe(s):
    case = s["case"]
    t, e, k, h, f = (case[n] for n in ("tokens", "experts", "top", "hidden", "inter"))
    x = s["x"].float()
    if s["norm"] is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-5) * s["norm"]
    # 64 bits for the logits: a tie of two experts goes one way
    logit, at = (x.double() @ s["gate"].double().T).sort(dim=-1, descending=True, stable=True)
    w = (logit[:, :k] - logit[:, :1]).exp()
    w, at = (w / w.sum(-1, keepdim=True)).float(), at[:, :k]
    if t * k < e:                                           # the chosen experts' weights, one product a pair
        rows, pick = x.repeat_interleave(k, 0)[:, None], at.flatten()
    else:                                                   # every expert on every row
        rows, pick = x.expand(e, t, h), torch.arange(e, device="cuda")
    a = _act(case["act"], rows @ _values(s["w1"][pick], case["kind"], f, h).transpose(1, 2))
    a = a * (rows @ _values(s["w3"][pick], case["kind"], f, h).transpose(1, 2))
    y = a @ _values(s["w2"][pick], case["kind"], h, f).transpose(1, 2)
    if t * k < e:
        out = (y.view(t, k, h) * w[..., None]).sum(1)
    else:
        share = torch.zeros(t, e, device="cuda").scatter_(1, at, w)
        out = (y * share.T[..., None]).sum(0)
    return {"out": out if s["residual"] is None else s["residual"] + out}


def _plain_norm(s):
    case = s["case"]
    y = s["y"].float()
    if s["post"] is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + 1e-5) * s["post"]
    if s["gate"] is not None:
        y = y * s["gate"].float()
    h = s["stream"].float() + case["scale"] * y
    got = {"stream": h.to(s["stream"].dtype)}
    if s["pre"] is not None:
        got["next"] = (h * torch.rsqrt((h * h).mean(-1, keepdim=True) + 1e-5) * s["pre"]).to(s["y"].dtype)
    return got


def _plain_logp(s):
    case = s["case"]
    raw = s["logits"].float()
    x = raw / case["temperature"]
    x = x - x.amax(-1, keepdim=True)
    w = x.exp()
    total = w.sum(-1, keepdim=True)
    log = total.log()
    got = {"entropy": (log - torch.where(w > 0, w * x, 0).sum(-1, keepdim=True) / total)[:, 0]}
    mine = s["tokens"][:, None]
    own_raw = raw.gather(1, mine)
    before = torch.arange(case["vocab"], device="cuda") < mine
    got["rank"] = ((raw > own_raw) | ((raw == own_raw) & before)).sum(-1).int()
    got["logprob"] = (x.gather(1, mine) - log)[:, 0]
    if case["top"]:
        at = raw.sort(dim=-1, descending=True, stable=True)[1][:, :case["top"]]
        got["top_ids"], got["top_logprobs"] = at.int(), x.gather(1, at) - log
    return got


def run(state):
    s = state
    case = s["case"]
    if not own:
        return {"moe": _plain_moe, "norm": _plain_norm, "logp": _plain_logp}[case["op"]](s)
    if case["op"] == "moe":
        return {"out": s["layer"].step(s["x"], norm_weight=s["norm"], eps=1e-5, residual=s["residual"])}
    if case["op"] == "norm":
        from xanosmerks_b200.ops import residual_norm
        stream, after = residual_norm(s["stream"], s["y"], post_weight=s["post"], gate=s["gate"], scale=case["scale"],
                                      pre_weight=s["pre"], eps=1e-5)
        return {"stream": stream} if after is None else {"stream": stream, "next": after}
    from xanosmerks_b200.sampling import logprobs
    r = logprobs(s["logits"], s["tokens"], temperature=case["temperature"], top=case["top"])
    got = {"entropy": r.entropy, "rank": r.rank, "logprob": r.logprob}
    if case["top"]:
        got["top_ids"], got["top_logprobs"] = r.top_ids, r.top_logprobs
    return got


# ---------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------
def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}
    if case["op"] == "moe":
        t, e, k, h, f = (case[n] for n in ("tokens", "experts", "top", "hidden", "inter"))
        qk, rec = _RECORD[case["kind"]]
        met = e * (1 - (1 - k / e) ** t)                    # experts that some token meets, on average
        b = met * 3 * h * f * rec / qk + 4 * e * h + t * h * (size[case["type"]] + 4 + 4 * case["residual"])
        return {"bytes": b, "flops": 6.0 * t * k * h * f + 2.0 * t * e * h}
    if case["op"] == "norm":
        n, d = case["batch"] * case["rows"], case["dim"]
        gate = {"none": 0, "channel": d, "sequence": case["batch"] * d, "row": n}[case["gate"]]
        b = n * d * (2 * size[case["stream"]] + (1 + case["pre"]) * size[case["type"]])
        return {"bytes": b + gate * size[case["type"]] + 4 * d * (case["post"] + case["pre"]), "flops": 10 * n * d}
    n = case["rows"] * case["vocab"]
    return {"bytes": n * size[case["type"]] + case["rows"] * (20 + 8 * case["top"]), "flops": 4 * n}


# ---------------------------------------------------------------------------------------------
# the definitions in 64 bits, written apart
# ---------------------------------------------------------------------------------------------
def _exact_rows(raw, kind, n, k):
    """One weight in 64 bits, value by value from the bytes that hold it."""
    qk, rec = _RECORD[kind]
    b = raw.view(n * (k // qk), rec).int()
    i = torch.arange(qk, device="cuda")

    def half(at):
        return (b[:, at] | (b[:, at + 1] << 8)).to(torch.int16).view(torch.float16).double()[:, None]

    def signed(v):
        return torch.where(v > 127, v - 256, v).double()

    if kind == "Q8_0":
        return (half(0) * signed(b[:, 2 + i])).view(n, k)
    if kind == "Q6_K":
        part, j, l = i // 128, i % 128 // 32, i % 32
        low = (b[:, 64 * part + 32 * (j % 2) + l] >> (4 * (j // 2))) & 15
        high = (b[:, 128 + 32 * part + l] >> (2 * j)) & 3
        return (half(208) * signed(b[:, 192 + i // 16]) * (low + 16 * high - 32)).view(n, k)
    j, l = i // 32, i % 32
    r = j % 4
    s = torch.where(j < 4, b[:, 4 + r] & 63, (b[:, 12 + r] & 15) + 16 * (b[:, 4 + r] >> 6))
    m = torch.where(j < 4, b[:, 8 + r] & 63, (b[:, 12 + r] >> 4) + 16 * (b[:, 8 + r] >> 6))
    c = (b[:, (16 if kind == "Q4_K" else 48) + 32 * (j // 2) + l] >> (4 * (j % 2))) & 15
    if kind == "Q5_K":
        c = c + 16 * ((b[:, 16 + 4 * (j // 2) + l // 8] >> (l % 8)) & 1)
    return (half(0) * s * c - half(2) * m).view(n, k)


def _exact_moe(s, case):
    e, k, h, f = (case[n] for n in ("experts", "top", "hidden", "inter"))
    x = s["x"].double()
    if s["norm"] is not None:
        x = x / torch.sqrt(x.square().sum(-1, keepdim=True) / h + 1e-5) * s["norm"].double()
    z = torch.matmul(x, s["gate"].double().T)
    order = torch.argsort(-z, stable=True, dim=-1)[:, :k]
    p = torch.softmax(z.gather(1, order), -1)
    out = torch.zeros_like(x) if s["residual"] is None else s["residual"].double()
    for i in torch.unique(order).tolist():
        t, j = (order == i).nonzero(as_tuple=True)
        g = x[t] @ _exact_rows(s["w1"][i], case["kind"], f, h).T
        u = x[t] @ _exact_rows(s["w3"][i], case["kind"], f, h).T
        if case["act"] == "gelu":
            g = g / (1 + torch.exp(-2 * 0.7978845608 * (g + 0.044715 * g ** 3)))
        elif case["act"] == "relu":
            g = torch.relu(g)
        else:
            g = g * torch.sigmoid(g)
        out.index_add_(0, t, ((g * u) @ _exact_rows(s["w2"][i], case["kind"], h, f).T) * p[t, j][:, None])
    return {"out": out}


def _exact_norm(s, case):
    def normed(v, w):
        return v / torch.sqrt(v.square().sum(-1, keepdim=True) / case["dim"] + 1e-5) * w.double()

    y = s["y"].double()
    if s["post"] is not None:
        y = normed(y, s["post"])
    if s["gate"] is not None:
        y = y * s["gate"].double()
    h = torch.add(s["stream"].double(), y, alpha=case["scale"])
    return {"stream": h} if s["pre"] is None else {"stream": h, "next": normed(h, s["pre"])}


def _exact_logp(s, case):
    parts = []
    for r in range(0, case["rows"], 64):                    # a few rows at a time
        x = s["logits"][r:r + 64].double()
        t = s["tokens"][r:r + 64]
        lp = torch.log_softmax(x / case["temperature"], -1)
        p = lp.exp()
        mine = x[torch.arange(len(t), device="cuda"), t][:, None]
        at = torch.arange(case["vocab"], device="cuda")
        got = {"entropy": -(p * torch.where(p > 0, lp, 0.0)).sum(-1),
               "rank": ((x > mine).sum(-1) + ((x == mine) & (at < t[:, None])).sum(-1)).int(),
               "logprob": lp[torch.arange(len(t), device="cuda"), t]}
        if case["top"]:
            ids = torch.argsort(-x, stable=True, dim=-1)[:, :case["top"]]
            got["top_ids"], got["top_logprobs"] = ids.int(), lp.gather(1, ids)
        parts.append(got)
    return {n: torch.cat([p[n] for p in parts]) for n in parts[0]}


def exact(case, seed):
    s = prepare(case, seed)
    return {"moe": _exact_moe, "norm": _exact_norm, "logp": _exact_logp}[case["op"]](s, case)
