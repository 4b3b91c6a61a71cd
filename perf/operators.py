"""Operator cases: 4-bit weights, the 4-bit key/value cache and token log probabilities, in plain
torch and through this package.

`listed()` names the fixed cases and `draw(rng)` gives more of the same ranges; `prepare` makes what
a program holds before the call, `run` is one pass through an operator (the package's entry point
where `own` is true, elementary 32-bit torch operations otherwise), `work` the bytes and operations
a pass cannot do without, and `exact` the result in 64 bits.

The kinds of case:
  w4       w4_linear: y = x W^T (+ residual) of 1 to 64 rows with 4-bit weights in groups of 32, 64
           or 128 along the input
  append   KV4Cache.append of new key and value rows, and KV4Cache.read of what the cache now holds
           for them (the values that later tokens attend over)
  attend   KV4Cache.attend: queries of the last positions of every sequence over its cached rows
  logprob  token_logprobs: log probability of a given token in every row of logits, the row's
           entropy and its most likely tokens

A weight or cache row is held as 4-bit codes u with a scale s per group and stands for s (u - z),
z = 8 where no zero points are given.
"""
from __future__ import annotations

import math

import torch

own = False

VOCAB = 151936


def listed():
    return [
        # the q|k|v projection of one token: the smallest product, host and launch count
        {"name": "w4_qkv", "kind": "w4", "m": 1, "n": 4096, "k": 1024, "group": 128,
         "dtype": "bf16", "out": "bf16", "zeros": False, "residual": False},
        # the vocabulary projection of one token, fp32 logits
        {"name": "w4_lm_head", "kind": "w4", "m": 1, "n": VOCAB, "k": 1024, "group": 128,
         "dtype": "bf16", "out": "fp32", "zeros": False, "residual": False},
        # the down projection and its residual for seven draft tokens checked at once
        {"name": "w4_down_draft", "kind": "w4", "m": 7, "n": 1024, "k": 3072, "group": 64,
         "dtype": "fp16", "out": "fp16", "zeros": True, "residual": True},
        # a wide layer for a batch of tokens, odd row counts, the finest groups
        {"name": "w4_wide_batch", "kind": "w4", "m": 33, "n": 16001, "k": 4096, "group": 32,
         "dtype": "bf16", "out": "bf16", "zeros": True, "residual": False},
        # one token's key and value rows
        {"name": "append_token", "kind": "append", "batch": 1, "t": 1, "heads": 8, "dim": 128,
         "group": 32, "cap": 4096, "max_len": 201, "dtype": "bf16"},
        # the rows of three prompts of different length, padded on the left
        {"name": "append_prompts", "kind": "append", "batch": 3, "t": 2731, "heads": 8, "dim": 128,
         "group": 64, "cap": 4096, "max_len": 2731, "dtype": "fp16"},
        # a token of a chat, at the start of a conversation
        {"name": "attend_chat", "kind": "attend", "batch": 1, "t": 1, "heads": 8, "ratio": 2,
         "dim": 128, "group": 32, "cap": 4096, "max_len": 201, "dtype": "bf16"},
        # a token at the end of the longest context the package's tests use
        {"name": "attend_32k", "kind": "attend", "batch": 1, "t": 1, "heads": 8, "ratio": 2,
         "dim": 128, "group": 32, "cap": 32768, "max_len": 32768, "dtype": "bf16"},
        # a batch of conversations of every length, an empty slot among them
        {"name": "attend_batch", "kind": "attend", "batch": 24, "t": 1, "heads": 8, "ratio": 4,
         "dim": 128, "group": 64, "cap": 8192, "max_len": 8191, "dtype": "fp16"},
        # a chunk of a long prompt over the rows before it and its own
        {"name": "attend_chunk", "kind": "attend", "batch": 1, "t": 509, "heads": 8, "ratio": 2,
         "dim": 128, "group": 128, "cap": 8192, "max_len": 6007, "dtype": "bf16"},
        # one decoded token's logits, as the decoder gives them
        {"name": "logprob_token", "kind": "logprob", "rows": 1, "vocab": VOCAB, "top": 20,
         "dtype": "fp32", "masked": False},
        # every position of a prompt that is scored
        {"name": "logprob_prompt", "kind": "logprob", "rows": 2047, "vocab": VOCAB, "top": 5,
         "dtype": "bf16", "masked": False},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["w4", "w4", "append", "attend", "attend", "attend", "logprob", "logprob"])
    if kind == "w4":
        group = rng.choice([32, 64, 128])
        m = rng.choice([1, 1, 2, rng.randint(3, 16), rng.randint(17, 64)])
        n = _log_int(rng, 500, 60000)
        k = group * _log_int(rng, 512 // group, 8192 // group)
        while n * k > (1 << 27):
            n //= 2
        dtype = rng.choice(["bf16", "fp16"])
        return {"kind": kind, "m": m, "n": n, "k": k, "group": group, "dtype": dtype,
                "out": rng.choice([dtype, dtype, "fp32"]), "zeros": rng.random() < 0.5,
                "residual": rng.random() < 0.3}
    if kind == "append":
        t = _log_int(rng, 1, 4000)
        return {"kind": kind, "batch": rng.randint(1, 3), "t": t, "heads": rng.choice([2, 4, 8]),
                "dim": rng.choice([64, 128, 128]), "group": rng.choice([32, 64]), "cap": 4096,
                "max_len": rng.randint(t, 4096), "dtype": rng.choice(["bf16", "fp16"])}
    if kind == "attend":
        dim = rng.choice([64, 128, 128])
        t = rng.choice([1, 1, 1, rng.randint(2, 16), rng.randint(17, 400)])
        batch = 1 if t > 16 else rng.choice([1, 1, 2, 5, 16])
        max_len = _log_int(rng, max(t, 40), 32768 if batch == 1 and t == 1 else 6000)
        heads, ratio = rng.choice([1, 4, 8]), rng.choice([1, 2, 4, 8])
        while batch * heads * ratio * t * max_len * 4 * dim > 20e9:
            max_len = max(t, max_len // 2)
            ratio = max(1, ratio // 2)
        return {"kind": kind, "batch": batch, "t": t, "heads": heads, "ratio": ratio, "dim": dim,
                "group": rng.choice([32, 64] if dim == 64 else [32, 64, 128]),
                "cap": max_len + rng.randint(0, 500), "max_len": max_len,
                "dtype": rng.choice(["bf16", "fp16"])}
    return {"kind": kind, "rows": _log_int(rng, 1, 600),
            "vocab": rng.choice([VOCAB, rng.randint(32000, 200000)]), "top": rng.choice([0, 1, 5, 20]),
            "dtype": rng.choice(["fp32", "bf16", "fp16"]), "masked": rng.random() < 0.3}


# ------------------------------------------------------------------------------ inputs
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _pack(u):
    """Codes 0..15 [..., n] as bytes [..., n / 2], the even element in the low nibble."""
    return (u[..., 0::2] | (u[..., 1::2] << 4)).to(torch.uint8)


def _unpack(packed):
    return torch.stack([packed & 15, packed >> 4], -1).flatten(-2)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))

    def randn(*shape, std=1.0):
        return torch.randn(*shape, generator=gen, device="cuda") * std

    s, kind, dtype = {"case": case}, case["kind"], DTYPES[case["dtype"]]
    if kind == "w4":
        m, n, k, g = case["m"], case["n"], case["k"], case["group"]
        # codes of normal weights: the scale covers about 2.6 deviations, the rest is clipped
        u = torch.empty(n, k, dtype=torch.uint8, device="cuda")
        for i in range(0, n, 16384):
            u[i:i + 16384] = (randn(min(16384, n - i), k, std=2.7).round() + 8).clamp(0, 15)
        s["qweight"] = _pack(u)
        s["scales"] = (0.0075 * (1 + 0.3 * torch.rand(n, k // g, generator=gen, device="cuda"))).to(dtype)
        s["zeros"] = None
        if case["zeros"]:
            s["zeros"] = torch.randint(5, 11, (n, k // g), generator=gen, device="cuda").to(torch.uint8)
        s["x"] = randn(m, k).to(dtype)
        s["out"] = DTYPES[case["out"]]
        s["residual"] = randn(m, n).to(s["out"]) if case["residual"] else None
        if own:
            from megaqwen_amd.w4 import w4_linear
            s["op"] = w4_linear
    elif kind in ("append", "attend"):
        b, t, hk, d, cap = (case[x] for x in ("batch", "t", "heads", "dim", "cap"))
        ng = d // case["group"]
        s["k_codes"] = torch.zeros(b, hk, cap, d // 2, dtype=torch.uint8, device="cuda")
        s["v_codes"] = torch.zeros_like(s["k_codes"])
        s["scales"] = torch.zeros(b, hk, cap, 2, ng, dtype=torch.bfloat16, device="cuda")
        lens = [case["max_len"]]
        for i in range(1, b):               # every length in between, an empty slot among many
            lens.append(0 if i == 7 else int(torch.randint(
                min(t, case["max_len"]), case["max_len"] + 1, (1,), generator=gen, device="cuda")))
        if kind == "append" and b > 1:      # prompts shorter than the padded rows
            lens = lens[:1] + [max(1, int(x * 0.6)) for x in lens[1:]]
        s["lengths"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        if kind == "append":
            s["k"], s["v"] = randn(b, t, hk, d).to(dtype), randn(b, t, hk, d, std=0.64).to(dtype)
        else:
            for i, x in enumerate((s["k_codes"], s["v_codes"])):
                for j in range(b):
                    u, sc = _quantize(randn(hk, cap, d, std=0.64 if i else 1.0), case["group"])
                    x[j] = _pack(u)
                    s["scales"][j, :, :, i] = sc
            s["q"] = randn(b, t, hk * case["ratio"], d).to(dtype)
        if own:
            from megaqwen_amd.kv4 import KV4Cache
            s["cache"] = KV4Cache.from_tensors(s["k_codes"], s["v_codes"], s["scales"])
    else:
        rows, v = case["rows"], case["vocab"]
        s["tokens"] = torch.randint(0, v, (rows,), generator=gen, device="cuda")
        x = torch.empty(rows, v, dtype=dtype, device="cuda")
        for i in range(0, rows, 256):
            c = randn(min(256, rows - i), v, std=2.5)
            if case["masked"]:               # a grammar that allows one token in twenty
                c.masked_fill_(torch.rand(c.shape, generator=gen, device="cuda") < 0.95, -math.inf)
            x[i:i + 256] = c
        at = torch.arange(rows, device="cuda")
        x[at, s["tokens"]] = (4.0 + 12.0 * torch.rand(rows, generator=gen, device="cuda")).to(dtype)
        s["logits"] = x
        if own:
            from megaqwen_amd.logprobs import token_logprobs
            s["op"] = token_logprobs
    torch.cuda.synchronize()
    return s


# ------------------------------------------------------------------------- plain forms
def _quantize(x, group):
    """Codes and bf16 scales of x [..., n] in groups: s = max|x| / 7, u = x / s + 8."""
    y = x.float().unflatten(-1, (-1, group))
    amax = y.abs().amax(-1)
    scale = torch.where(torch.isfinite(amax), amax / 7.0, math.nan).to(torch.bfloat16)
    sf = scale.float().unsqueeze(-1)
    q = torch.where(sf > 0, y / sf, torch.zeros_like(y)).round().clamp(-7, 7)
    return (q + 8).to(torch.uint8).flatten(-2), scale


def _values(codes, scales):
    """s (u - 8) of packed codes [..., n / 2] and scales [..., groups]."""
    u = _unpack(codes).float().unflatten(-1, (scales.shape[-1], -1)) - 8
    return (u * scales.float().unsqueeze(-1)).flatten(-2)


def _w4(s):
    ng = s["scales"].shape[1]
    u = _unpack(s["qweight"]).float().unflatten(-1, (ng, -1))
    z = 8 if s["zeros"] is None else s["zeros"].float().unsqueeze(-1)
    w = ((u - z) * s["scales"].float().unsqueeze(-1)).flatten(-2)
    y = s["x"].float() @ w.T
    return (y if s["residual"] is None else y + s["residual"].float()).to(s["out"])


def _append(s):
    """Row i of t goes to position length - t + i; what stands at a row that does not exist (a
    negative position, counted from the end here) is written back."""
    b, t = s["k"].shape[:2]
    pos = s["lengths"].long()[:, None] - t + torch.arange(t, device="cuda")
    there = (pos >= 0)[:, :, None, None]
    p, at, out = pos % s["k_codes"].shape[2], torch.arange(b, device="cuda")[:, None], []
    for i, (x, codes) in enumerate(((s["k"], s["k_codes"]), (s["v"], s["v_codes"]))):
        u, scale = _quantize(x, s["case"]["group"])
        codes[at, :, p] = torch.where(there, _pack(u), codes[at, :, p])
        s["scales"][at, :, p, i] = torch.where(there, scale, s["scales"][at, :, p, i])
        value = _values(codes[at, :, p], s["scales"][at, :, p, i])
        out.append(torch.where(there, value, 0).to(torch.bfloat16))
    return out


def _attend(s):
    """Scores, softmax and sum over every cached row up to the longest length, masked."""
    case, q = s["case"], s["q"].float()
    b, t, hq, d = q.shape
    hk, n = case["heads"], case["max_len"]
    k = _values(s["k_codes"][:, :, :n], s["scales"][:, :, :n, 0])
    q = q.unflatten(2, (hk, -1)).permute(0, 2, 1, 3, 4).reshape(b, hk, -1, d)
    scores = q @ k.transpose(-1, -2) / math.sqrt(d)                  # [b, hk, t * ratio, n]
    last = s["lengths"][:, None] - t + torch.arange(t, device="cuda")
    seen = torch.arange(n, device="cuda") <= last.repeat_interleave(hq // hk, 1)[..., None]
    scores = scores.masked_fill(~seen[:, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(torch.isfinite(top), top, 0))
    total = p.sum(-1, keepdim=True)
    v = _values(s["v_codes"][:, :, :n], s["scales"][:, :, :n, 1])
    o = torch.where(total > 0, (p @ v) / total, 0)
    return o.unflatten(2, (t, -1)).permute(0, 2, 1, 3, 4).reshape(b, t, hq, d).to(s["q"].dtype)


def _best(x, k):
    """The k largest of every row, equal values by their lowest index: the largest of whole numbers
    that rise with the value and fall with the index."""
    bits = (x + 0.0).view(torch.int32)
    rising = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
    key = rising * (1 << 32) - torch.arange(x.shape[-1], device=x.device)
    at = -torch.topk(key, k).values % (1 << 32)
    return x.gather(1, at), at.to(torch.int32)


def _logprob_rows(x, tokens, k):
    top = x.amax(-1, keepdim=True)
    d = x - top
    e = torch.exp(d)
    total = e.sum(-1)
    entropy = torch.log(total) - torch.where(e > 0, e * d, 0).sum(-1) / total
    d = d - torch.log(total)[:, None]
    got = [d.gather(1, tokens[:, None])[:, 0], entropy]
    if k:
        value, at = _best(x, k)
        got += [value - top - torch.log(total)[:, None], at]
    return got


def _logprob(s):
    got = [_logprob_rows(x.float(), t, s["case"]["top"])
           for x, t in zip(s["logits"].split(512), s["tokens"].split(512))]
    return [torch.cat(x) for x in zip(*got)]


def run(state):
    s, case = state, state["case"]
    kind = case["kind"]
    if kind == "w4":
        if own:
            return s["op"](s["x"], s["qweight"], s["scales"], s["zeros"], residual=s["residual"],
                           out_dtype=s["out"])
        return _w4(s)
    if kind == "append":
        if own:
            s["cache"].append(s["k"], s["v"], s["lengths"])
            return list(s["cache"].read(s["lengths"], case["t"]))
        return _append(s)
    if kind == "attend":
        if own:
            return s["cache"].attend(s["q"], s["lengths"], max_length=case["max_len"])
        return _attend(s)
    if own:
        return list(s["op"](s["logits"], s["tokens"], top_k=case["top"]))[:4 if case["top"] else 2]
    return _logprob(s)


# ------------------------------------------------------------------------------- floors
def work(case):
    kind = case["kind"]
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    if kind == "w4":
        m, n, k, groups = case["m"], case["n"], case["k"], case["n"] * case["k"] // case["group"]
        out = m * n * size[case["out"]]
        return {"bytes": n * k // 2 + groups * (3 if case["zeros"] else 2) + 2 * m * k
                + out * (2 if case["residual"] else 1), "flops": 2 * m * n * k}
    if kind in ("append", "attend"):
        b, t, hk, d = (case[x] for x in ("batch", "t", "heads", "dim"))
        row = hk * 2 * (d // 2 + 2 * (d // case["group"]))        # a position's codes and scales
        if kind == "append":                # rows read, codes written, and read again as values
            return {"bytes": b * t * (2 * hk * d * 2 + 2 * row + 2 * hk * d * 2),
                    "flops": 6 * b * t * hk * d}
        # lengths of a batch are uniform up to the longest
        n = case["max_len"] + (b - 1) * (case["max_len"] + t) // 2
        hq = hk * case["ratio"]
        pairs = t * n - b * t * (t - 1) // 2
        return {"bytes": n * row + 2 * b * t * hq * d * 2, "flops": 4 * d * hq * pairs}
    rows, v = case["rows"], case["vocab"]
    return {"bytes": rows * (v * size[case["dtype"]] + 16 + 8 * case["top"]), "flops": 5 * rows * v}


# --------------------------------------------------------------------------- 64-bit results
def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "w4":
        groups, out = case["k"] // case["group"], []
        x = s["x"].double().unflatten(1, (groups, -1)).transpose(0, 1)       # [groups, m, G]
        for i in range(0, case["n"], 8192):
            rows = slice(i, i + 8192)
            low, high = s["qweight"][rows] % 16, s["qweight"][rows] // 16
            u = torch.empty(low.shape[0], case["k"], dtype=torch.float64, device="cuda")
            u[:, ::2], u[:, 1::2] = low, high
            u = u.unflatten(1, (groups, -1)).permute(1, 2, 0).contiguous()   # [groups, G, rows]
            z = 8.0 if s["zeros"] is None else s["zeros"][rows].double().T[:, None]
            part = torch.bmm(x.contiguous(), u - z)                          # [groups, m, rows]
            out.append((part * s["scales"][rows].double().T[:, None]).sum(0))
        y = torch.cat(out, 1)
        return y if s["residual"] is None else y + s["residual"].double()
    if kind == "append":
        t, out = case["t"], []
        for x in (s["k"].double(), s["v"].double()):
            y = x.reshape(*x.shape[:-1], -1, case["group"])
            step = (y.abs().max(-1, keepdim=True).values / 7).to(torch.bfloat16).double()
            y = (torch.round(y / step) * step).reshape(x.shape)
            for j, n in enumerate(s["lengths"].tolist()):
                y[j, :max(0, t - n)] = 0
            out.append(y)
        return out
    if kind == "attend":
        q, t = s["q"].double(), case["t"]
        out = torch.zeros_like(q)
        for j, n in enumerate(s["lengths"].tolist()):
            for h in range(case["heads"] if n else 0):
                kv = []
                for i, codes in enumerate((s["k_codes"], s["v_codes"])):
                    c = codes[j, h, :n].long()
                    u = torch.stack([c % 16, c // 16], -1).reshape(n, -1, case["group"]).double() - 8
                    kv.append((u * s["scales"][j, h, :n, i].double()[..., None]).reshape(n, -1))
                ahead = torch.arange(n, device="cuda") > torch.arange(n - t, n, device="cuda")[:, None]
                for r in range(case["ratio"]):
                    z = q[j, :, h * case["ratio"] + r] @ kv[0].T / math.sqrt(case["dim"])
                    w = torch.softmax(z.masked_fill(ahead, -math.inf), -1).nan_to_num(0.0)
                    out[j, :, h * case["ratio"] + r] = w @ kv[1]
        return out
    parts = []
    for x, tok in zip(s["logits"].split(256), s["tokens"].split(256)):
        x = x.double()
        lse = torch.logsumexp(x, -1)
        p = torch.exp(x - lse[:, None])
        got = [x.gather(1, tok[:, None])[:, 0] - lse, lse - (p * x.clamp_min(-1e300)).sum(-1)]
        if case["top"]:
            got.append(torch.topk(x, case["top"]).values - lse[:, None])
        parts.append(got)
    out = [torch.cat(x) for x in zip(*parts)]
    return out + [None] if case["top"] else out
