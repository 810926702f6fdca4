"""What this library's serving operators are timed on: the calls that a program
makes between the projections of a decoder layer, and after the LM head, when it
serves several sequences from one paged KV cache.

Operators ("op" of a case):
  append  RMS norm of each query and key head (if the model has it), position
          rotation, and the store of the new keys and values into the cache's
          pages, fp16 or int8 with a scale per (position, KV head)
  attend  attention of each sequence's new tokens over its pages, causal; one new
          token is decoding, more are a prompt's chunk or a draft being checked
  sample  the next token of each row of logits: temperature, top-k, top-p, min-p
          and a given random number

Sequences: `seqs` of them have new tokens spread between new[0] and new[1] after
cached positions spread between past[0] and past[1] (evenly over the logarithm, in
a scattered order), and `decodes` more have one new token each.  Pages lie in the
pool in random order; table entries past a sequence's end are -1.  Queries, keys and
values are N(0, 1), int8 scales such that the values are.  Logits are N(0, 2) with
64 raised tokens a row.

`run` is the plain form (elementary operations, 32 bits, 64 for angles and for
probabilities' sums), or with `own` the library's entry points; a program builds
its cache and batch descriptors once, as the first pass does here.
"""
import math

import torch

own = False
DEV = "cuda"


# ------------------------------------------------------------------ the cases
def _attend(name, seqs, new, past, decodes=0, heads=(32, 8, 128), page=16, int8=False):
    return {"name": name, "op": "attend", "seqs": seqs, "new_lo": new[0], "new_hi": new[1], "past_lo": past[0],
            "past_hi": past[1], "decodes": decodes, "heads": heads[0], "kv": heads[1], "head_dim": heads[2],
            "page": page, "int8": int8}


def _append(name, seqs, new, past, decodes=0, heads=(32, 8, 128), page=16, int8=False, dtype="f16", norm=True,
            n_rot=128, interleaved=False):
    return {**_attend(name, seqs, new, past, decodes, heads, page, int8), "op": "append", "dtype": dtype, "norm": norm,
            "n_rot": n_rot, "interleaved": interleaved}


def listed():
    return [
        # one user's next token, 3B-class heads (16 / 2 of 128): the smallest call, latency
        _attend("decode_1x1000", 0, (1, 1), (1000, 1000), decodes=1, heads=(16, 2, 128)),
        # a full decode batch of 8B-class heads, conversations of every length
        _attend("decode_64_ragged", 0, (1, 1), (64, 8000), decodes=64),
        # long documents in an int8 cache
        _attend("decode_16_long_int8", 0, (1, 1), (20000, 40000), decodes=16, page=64, int8=True),
        # drafts of a few tokens being checked, groups of seven heads
        _attend("draft_12x5", 12, (3, 6), (500, 6000), heads=(28, 4, 128), page=32),
        # a usual prefill chunk deep in a long prompt
        _attend("chunk_512_at_7000", 1, (512, 512), (7000, 7000), heads=(16, 2, 128)),
        # four prompts prefilled together from an empty cache, odd lengths: the largest
        _attend("prefill_4_prompts", 4, (1000, 4000), (0, 0), page=64),
        # continuous batching: two chunks beside decoding sequences, heads of 80, small
        # pages, int8
        _attend("mixed_2_and_30", 2, (200, 500), (100, 3000), decodes=30, heads=(8, 4, 80), page=8, int8=True),
        # one user's next token
        _append("append_1", 0, (1, 1), (1000, 1000), decodes=1, heads=(16, 2, 128)),
        # a decode batch into an int8 cache; no head norms, neighbouring dims rotated
        _append("append_64_int8", 0, (1, 1), (64, 8000), decodes=64, int8=True, norm=False, interleaved=True),
        # prompts' chunks from bf16 projections
        _append("append_4_chunks_bf16", 4, (500, 1500), (0, 4000), dtype="bf16", page=64),
        # one user's next token from the 151936 logits of the LM head
        {"name": "sample_1", "op": "sample", "rows": 1, "vocab": 151936, "params": "chat"},
        # a full batch, every request with settings of its own
        {"name": "sample_128_mixed", "op": "sample", "rows": 128, "vocab": 151936, "params": "mixed"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "append", "sample"])
    if op == "sample":
        vocab = _log(rng, 1000, 160000)
        return {"op": op, "rows": _log(rng, 1, min(256, 128 * 151936 // vocab)), "vocab": vocab,
                "params": rng.choice(["chat", "mixed", "mixed", "plain", "nucleus"])}
    kv = rng.choice([1, 2, 4, 8])
    hd = rng.choice([128, 128, 128, 64, 80, 96, 256])
    c = {"op": op, "heads": kv * rng.choice([1, 2, 4, 4, 5, 7, 8]), "kv": kv, "head_dim": hd,
         "page": rng.choice([1, 4, 8, 16, 16, 32, 64, 128, 256]), "int8": rng.random() < 0.35}
    shape = rng.choice(["decode", "decode", "draft", "chunk", "mixed"])
    lo = _log(rng, 1, 8000)
    hi = max(lo, _log(rng, 100, 30000 if shape == "decode" else 12000))
    new = _log(rng, 2, 12) if shape == "draft" else _log(rng, 12, 2000)
    c |= {"seqs": 0 if shape == "decode" else _log(rng, 1, 32 if shape == "draft" else 4), "new_lo": max(1, new // 2),
          "new_hi": new, "past_lo": lo, "past_hi": hi,
          "decodes": _log(rng, 1, 64) if shape in ("decode", "mixed") else 0}
    if op == "append":
        c |= {"dtype": rng.choice(["f16", "f16", "bf16", "f32"]), "norm": rng.random() < 0.6,
              "n_rot": rng.choice([hd, hd, hd // 2]), "interleaved": rng.random() < 0.4}
    most = next(x for x in listed() if x["name"] == "prefill_4_prompts")
    while _cost(c) > _cost(most):  # fewer, shorter sequences until it costs no more than the largest listed one
        c |= {"decodes": c["decodes"] * 3 // 4, "seqs": max(c["seqs"] * 3 // 4, 1 if c["new_hi"] > 1 else 0)}
        c |= {"past_hi": max(c["past_hi"] * 3 // 4, 1), "past_lo": max(c["past_lo"] * 3 // 4, 1)}
        c |= {"new_hi": max(c["new_hi"] * 3 // 4, 1), "new_lo": max(c["new_lo"] * 3 // 4, 1)}
    return c


def _cost(c):
    """What a case takes in either form: its work, and the plain form's padded arrays."""
    new, lens = _lengths(c)
    s, q, n = len(new), max(new), max(lens)
    w = work(c)
    return max(w["bytes"] / 5e12, w["flops"] / 3e14, s * n * c["kv"] * c["head_dim"] / 2e13 + s * q * n * c["heads"] / 6e12)


def _spread(lo, hi, n):
    """n whole numbers between lo and hi, even over the logarithm, in a scattered order."""
    at = [((i + 0.5) * 0.6180339887498949) % 1.0 for i in range(n)]
    return [int(round((lo + 1) * ((hi + 1) / (lo + 1)) ** x)) - 1 for x in at]


def _lengths(c):
    """Each sequence's new tokens and its positions with them."""
    new = _spread(c["new_lo"], c["new_hi"], c["seqs"]) + [1] * c["decodes"]
    past = _spread(c["past_lo"], c["past_hi"], len(new))
    return new, [p + n for p, n in zip(past, new)]


def work(c):
    if c["op"] == "sample":
        n = c["rows"] * c["vocab"]
        return {"bytes": 4 * n + 24 * c["rows"], "flops": 4 * n}
    new, lens = _lengths(c)
    rows, kvd, esz = sum(new), c["kv"] * c["head_dim"], 1 if c["int8"] else 2
    position = 2 * (kvd * esz + (4 * c["kv"] if c["int8"] else 0))
    if c["op"] == "append":
        x = 4 if c["dtype"] == "f32" else 2
        return {"bytes": rows * ((c["heads"] * c["head_dim"] + 2 * kvd) * x + c["heads"] * c["head_dim"] * 2 + position),
                "flops": rows * (c["heads"] + c["kv"]) * c["head_dim"] * 8}
    seen = sum(n * (m - n) + n * (n + 1) // 2 for n, m in zip(new, lens))
    return {"bytes": sum(lens) * position + 4 * rows * c["heads"] * c["head_dim"],
            "flops": 4 * c["head_dim"] * c["heads"] * seen}


# ------------------------------------------------------------------ the inputs
def prepare(c, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device=DEV)

    if c["op"] == "sample":
        n, v = c["rows"], c["vocab"]
        logits = normal(n, v) * 2
        at = torch.randint(0, v, (n, 64), generator=g, device=DEV)
        logits.scatter_add_(1, at, torch.rand((n, 64), generator=g, device=DEV) * 10)
        s = {"op": "sample", "logits": logits, "u": torch.rand(n, generator=g, device=DEV),
             "ids": torch.empty(n, dtype=torch.int32, device=DEV)}
        if c["params"] == "mixed":
            def pick(values, dtype):
                i = torch.randint(0, len(values), (n,), generator=g, device=DEV)
                return torch.tensor(values, dtype=dtype, device=DEV)[i]
            s |= {"temperature": pick([0.0, 0.6, 0.7, 1.0, 1.3], torch.float32), "top_k": pick([0, 0, 20, 64, 500], torch.int32),
                  "top_p": pick([1.0, 0.95, 0.9, 0.8], torch.float32), "min_p": pick([0.0, 0.0, 0.05, 0.1], torch.float32)}
        else:
            def full(value, dtype=torch.float32):
                return torch.full((n,), value, dtype=dtype, device=DEV)
            s |= {"temperature": full(0.7 if c["params"] == "chat" else 1.0),
                  "top_k": full(50, torch.int32) if c["params"] == "chat" else None,
                  "top_p": None if c["params"] == "plain" else full(0.9), "min_p": None}
        return s

    new, lens = _lengths(c)
    S, rows, heads, kv, hd, page = len(new), sum(new), c["heads"], c["kv"], c["head_dim"], c["page"]
    used = [-(-n // page) for n in lens]
    width, pages = max(used), sum(used) + 3
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    cell = torch.arange(width, device=DEV)[None, :] < torch.tensor(used, device=DEV)[:, None]
    table = torch.full((S, width), -1, dtype=torch.int32, device=DEV)
    table[cell] = order[:sum(used)]
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    s = {"op": c["op"], "n_heads": heads, "page": page, "n_tokens": rows, "max_new": max(new), "max_len": max(lens),
         "table": table, "starts": torch.tensor(starts, dtype=torch.int32, device=DEV),
         "lens": torch.tensor(lens, dtype=torch.int32, device=DEV), "k_scales": None, "v_scales": None,
         "out": torch.empty((rows, heads, hd), dtype=torch.float16, device=DEV)}
    if c["int8"]:
        for x in "kv":
            s[x + "_cache"] = torch.randint(-127, 128, (pages, page, kv, hd), generator=g, device=DEV, dtype=torch.int8)
            s[x + "_scales"] = (torch.rand((pages, page, kv), generator=g, device=DEV) + 0.5) / 73
    else:
        for x in "kv":
            s[x + "_cache"] = normal(pages, page, kv, hd).half()
    if c["op"] == "attend":
        return s | {"q": normal(rows, heads, hd).half(), "scale": hd ** -0.5}
    # what the layer's fused projection left: one row a token, queries, keys, values
    dtype = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}[c["dtype"]]
    qkv = normal(rows, heads + 2 * kv, hd).to(dtype)
    s |= {"q": qkv[:, :heads], "k": qkv[:, heads:heads + kv], "v": qkv[:, heads + kv:], "interleaved": c["interleaved"],
          "q_weight": None, "k_weight": None, "eps": 1e-6,
          "inv_freq": (1e6 ** (-torch.arange(0, c["n_rot"], 2, device=DEV, dtype=torch.float64) / c["n_rot"])).float()}
    if c["norm"]:
        s |= {"q_weight": 1 + 0.2 * normal(hd), "k_weight": 1 + 0.2 * normal(hd)}
    if c["int8"]:
        s["slots"] = _slots(s)[0]
    return s


# ------------------------------------------------------------- the plain forms
def _slots(s):
    """Each token's place in the pool, and its position."""
    starts, page = s["starts"].long(), s["page"]
    token = torch.arange(s["n_tokens"], device=DEV)
    seq = (token[:, None] >= starts[None, 1:]).sum(1)
    pos = s["lens"].long()[seq] - starts[seq + 1] + token
    return s["table"].long()[seq, pos // page] * page + pos % page, pos


def _positions(s):
    """[sequence, position]: its place in the pool (0 past the end), and whether it is within the sequence."""
    pos, page = torch.arange(s["max_len"], device=DEV), s["page"]
    inside = pos[None, :] < s["lens"].long()[:, None]
    return (s["table"].long()[:, pos // page].clamp(min=0) * page + pos % page) * inside, inside


def _read(s, x, slots):
    """Keys or values at `slots` in 32 bits."""
    cache = s[x + "_cache"].flatten(0, 1)[slots].float()
    return cache if s[x + "_scales"] is None else cache * s[x + "_scales"].flatten(0, 1)[slots][..., None]


def _attend_plain(s):
    q, starts = s["q"].float(), s["starts"].long()
    rows, heads, hd = q.shape
    slots, inside = _positions(s)
    k = _read(s, "k", slots).permute(0, 2, 3, 1).contiguous()  # sequence, KV head, dim, position
    v = (_read(s, "v", slots) * inside[..., None, None]).transpose(1, 2).contiguous()
    S, kv, _, L = k.shape
    group, Q = heads // kv, s["max_new"]
    t = torch.arange(Q, device=DEV)
    n = starts[1:] - starts[:-1]
    real = t[None, :] < n[:, None]  # sequence, new token
    row = (starts[:-1, None] + t) * real
    qs = q[row].view(S, Q, kv, group, hd).permute(0, 2, 3, 1, 4).reshape(S, kv, group * Q, hd)
    score = (torch.matmul(qs, k) * s["scale"]).view(S, kv, group, Q, L)
    last = s["lens"].long()[:, None] - n[:, None] + t
    seen = (torch.arange(L, device=DEV) <= last[..., None])[:, None, None]
    score = score.masked_fill(~seen, -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-3e38)  # rows that see nothing: zeros
    e = (score - top).exp_()
    total = e.sum(-1, keepdim=True)
    o = torch.matmul(e.view(S, kv, group * Q, L), v).view(S, kv, group, Q, hd) / total.clamp(min=1e-30)
    return {"out": o.permute(0, 3, 1, 2, 4).reshape(S, Q, heads, hd)[real].half()}


def _normed(x, weight, eps):
    return x if weight is None else x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * weight


def _rotated(x, cos, sin, interleaved):
    r = 2 * cos.shape[-1]
    x, rest = x[..., :r], x[..., r:]
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :r // 2], x[..., r // 2:])
    a, b = a * cos - b * sin, b * cos + a * sin
    x = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((x, rest), -1)


def _append_plain(s):
    slots, pos = _slots(s)
    angle = pos.double()[:, None, None] * s["inv_freq"].double()
    cos, sin = angle.cos().float(), angle.sin().float()
    q = _rotated(_normed(s["q"].float(), s["q_weight"], s["eps"]), cos, sin, s["interleaved"])
    k = _rotated(_normed(s["k"].float(), s["k_weight"], s["eps"]), cos, sin, s["interleaved"])
    s["out"].copy_(q)
    for x, rows in (("k", k), ("v", s["v"].float())):
        if s[x + "_scales"] is None:
            s[x + "_cache"].flatten(0, 1)[slots] = rows.half()
        else:
            scale = rows.abs().amax(-1) / 127
            s[x + "_scales"].flatten(0, 1)[slots] = scale
            s[x + "_cache"].flatten(0, 1)[slots] = (rows / scale.clamp(min=1e-38)[..., None]).round().to(torch.int8)


def _sample_plain(s):
    logits = s["logits"]
    n, v = logits.shape
    order = torch.sort(logits, dim=1, descending=True, stable=True)
    t = s["temperature"].double()[:, None]
    z = order.values.double()
    w = ((z - z[:, :1]) / torch.where(t > 0, t, 1.0)).exp()
    rank = torch.arange(v, device=DEV)[None, :]
    if s["top_k"] is not None:
        k = s["top_k"].long()[:, None]
        w = w * ((k <= 0) | (rank < k))
    before = w.cumsum(1) - w
    keep = w > 0
    if s["top_p"] is not None:
        p = s["top_p"].double()[:, None]
        keep &= (p >= 1) | (before < p * w.sum(1, keepdim=True))
    if s["min_p"] is not None:
        keep &= w >= s["min_p"].double()[:, None]
    w = w * keep
    chosen = (w.cumsum(1) <= s["u"].double()[:, None] * w.sum(1, keepdim=True)).sum(1)
    chosen = torch.where(t[:, 0] > 0, torch.minimum(chosen, keep.sum(1) - 1), 0)
    return {"ids": order.indices.gather(1, chosen[:, None])[:, 0].int()}


# ---------------------------------------------------------------- one pass
def run(s):
    if own:
        _own(s)
    elif s["op"] == "append":
        _append_plain(s)
    else:
        return _attend_plain(s) if s["op"] == "attend" else _sample_plain(s)
    if s["op"] == "sample":
        return {"ids": s["ids"]}
    if s["op"] == "attend":
        return {"out": s["out"]}
    if s["k_scales"] is None:
        return {"q": s["out"], "k": s["k_cache"], "v": s["v_cache"]}
    # what the int8 rows stand for, read back from their slots
    return {"q": s["out"], "k": _read(s, "k", s["slots"]).half(), "v": _read(s, "v", s["slots"]).half()}


def _own(s):
    capi = s.get("capi") or _library(s)
    if s["op"] == "sample":
        capi.sample_f32(s["ids"], s["logits"], s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])
    elif s["op"] == "attend":
        capi.attention_paged_f16(s["out"], s["q"], s["batch"], s["cache"], s["scale"])
    else:
        capi.qk_norm_rope(s["out"], s["q"], s["k"], s["v"], s["batch"], s["cache"], s["inv_freq"], s["q_weight"],
                          s["k_weight"], s["eps"], s["interleaved"])


def _library(s):
    """The binding, and the descriptors that a program keeps beside its cache and its batch."""
    import os
    import sys
    package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "reflex-infer_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    from rxq4 import capi
    if s["op"] != "sample":
        s["cache"] = capi.PagedKV(s["k_cache"], s["v_cache"], s["table"], s["k_scales"], s["v_scales"])
        s["batch"] = capi.SeqBatch(s["starts"], s["lens"], s["n_tokens"], s["max_new"], s["max_len"])
    s["capi"] = capi
    return capi


# ------------------------------------------------------ the definitions in 64 bits
def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "sample":
        return None  # whole numbers
    new, lens = _lengths(c)
    kv, hd, page = c["kv"], c["head_dim"], c["page"]
    group = c["heads"] // kv
    if c["op"] == "attend":
        if work(c)["flops"] > 3e12:
            return None
        out = torch.empty(s["out"].shape, dtype=torch.float64, device=DEV)
        first = 0
        for i, (n, m) in enumerate(zip(new, lens)):
            pages = s["table"][i, :-(-m // page)].long()

            def values(x):
                y = s[x + "_cache"][pages].double()
                if c["int8"]:
                    y = y * s[x + "_scales"][pages].double().unsqueeze(-1)
                return y.reshape(-1, kv, hd)[:m]

            k, v = values("k"), values("v")
            hidden = torch.ones((n, m), dtype=torch.bool, device=DEV).triu(m - n + 1)
            for h in range(c["heads"]):
                x = s["q"][first:first + n, h].double() @ k[:, h // group].t().contiguous() * s["scale"]
                p = torch.exp(x.masked_fill(hidden, -math.inf) - x.max(dim=1, keepdim=True).values)
                out[first:first + n, h] = (p @ v[:, h // group].contiguous()) / p.sum(dim=1, keepdim=True)
            first += n
        return {"out": out}
    place = torch.cat([torch.arange(m - n, m, device=DEV) for n, m in zip(new, lens)])
    owner = torch.cat([torch.full((n,), i, device=DEV) for i, n in enumerate(new)])
    where = (s["table"][owner, place // page].long(), place % page)
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEV), place.double()[:, None] * s["inv_freq"].double())

    def turned(x, weight):
        y = x.double()
        if weight is not None:
            y = y / torch.sqrt(y.square().sum(-1, keepdim=True) / hd + s["eps"]) * weight.double()
        y = y.clone()
        r = c["n_rot"]
        pair = (y[..., 0:r:2], y[..., 1:r:2]) if c["interleaved"] else (y[..., :r // 2], y[..., r // 2:r])
        z = torch.complex(pair[0].contiguous(), pair[1].contiguous()) * turn[:, None]
        pair[0].copy_(z.real)
        pair[1].copy_(z.imag)
        return y

    q, k, v = turned(s["q"], s["q_weight"]), turned(s["k"], s["k_weight"]), s["v"].double()
    if c["int8"]:
        step = [x.abs().max(dim=-1, keepdim=True).values / 127 for x in (k, v)]
        return {"q": q, "k": torch.round(k / step[0]) * step[0], "v": torch.round(v / step[1]) * step[1]}
    whole = {"q": q}
    for name, rows in (("k", k), ("v", v)):
        whole[name] = s[name + "_cache"].double()
        whole[name][where] = rows
    return whole
