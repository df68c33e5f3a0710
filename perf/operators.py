"""The operators between a decoder layer's q/k/v projection and its output projection, as cases that can be timed.

A case is a plain dict; its field "op" names the operator:
  rope   capi.qk_norm_rotary_embedding        root-mean-square norm of every query and key head and the position
                                              rotation, in one pass over the rows of a fused q/k/v projection
  cache  ops.cache_write, ops.cache_read      keys and values of new tokens into a paged cache (as they are, or as
                                              8-bit e4m3 values with a power of two per token and head), and tokens
                                              read back from it
  attn   ops.paged_attention                  new tokens of several sequences over their paged caches

With `own` false, `run` computes the operator from elementary torch operations in 32 bits and rounds once at the end;
with `own` true it makes the package's calls.  `exact` states the same definitions in 64 bits.

An e4m3 cache holds, for every token and head, one exponent byte b: the value is code * 2^(b - 127), and b - 127 is the
smallest integer e with max |x| <= 448 * 2^e.

Ranges: 1 to 8192 tokens, 1 to 40 key heads with 1 to 8 query heads each, heads of 64 and 128, pages of 16 to 128 tokens,
1 to 64 sequences of up to 131072 tokens, fp16 and bf16, caches of the same type or e4m3.
"""
import math
import random

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # A decode step of seven requests: the least a call can be.
        {"name": "rope-7tok", "op": "rope", "T": 7, "Hq": 32, "Hkv": 8, "D": 128, "rot": 128, "neox": True, "dtype": "bf16", "table": "same"},
        # An odd-sized chunk, interleaved pairs, half of every head rotated, the position table in 32 bits.
        {"name": "rope-part", "op": "rope", "T": 1023, "Hq": 16, "Hkv": 4, "D": 64, "rot": 32, "neox": False, "dtype": "fp16", "table": "fp32"},
        # The prompts of a 13B-shaped model, 40 heads of queries and of keys.
        {"name": "rope-prompt", "op": "rope", "T": 8191, "Hq": 40, "Hkv": 40, "D": 128, "rot": 128, "neox": True, "dtype": "fp16", "table": "same"},
        # One decode step of 61 requests into an e4m3 cache, and those tokens back.
        {"name": "cache-decode", "op": "cache", "T": 61, "R": 61, "H": 8, "D": 128, "page": 16, "dtype": "bf16", "cache": "e4m3"},
        # A chunk of 1500 tokens into a cache of the same type, and a prefix of 4000 tokens back (handed to another worker).
        {"name": "cache-prefix", "op": "cache", "T": 1500, "R": 4000, "H": 8, "D": 128, "page": 64, "dtype": "bf16", "cache": "same"},
        # The prompts of a 13B-shaped model into an e4m3 cache, and all of it back.
        {"name": "cache-prompt", "op": "cache", "T": 8192, "R": 8192, "H": 40, "D": 128, "page": 32, "dtype": "fp16", "cache": "e4m3"},
        # One request of a 7B-shaped model, one token: the least an attention call can be.
        {"name": "attn-1tok", "op": "attn", "B": 1, "new": 1, "least": 700, "most": 700, "Hq": 32, "Hkv": 32, "D": 128, "page": 16,
         "dtype": "fp16", "cache": "same", "window": 0, "causal": True},
        # A decode step of 64 requests of very different lengths, shared key heads.
        {"name": "attn-decode", "op": "attn", "B": 64, "new": 1, "least": 100, "most": 8000, "Hq": 32, "Hkv": 8, "D": 128, "page": 16,
         "dtype": "bf16", "cache": "same", "window": 0, "causal": True},
        # Three requests deep in long documents, one token each, e4m3 cache.
        {"name": "attn-decode-long", "op": "attn", "B": 3, "new": 1, "least": 90000, "most": 131072, "Hq": 32, "Hkv": 8, "D": 128,
         "page": 64, "dtype": "bf16", "cache": "e4m3", "window": 0, "causal": True},
        # A mixed step: chunks of 1 to 700 new tokens of five requests behind histories of their own.
        {"name": "attn-chunk", "op": "attn", "B": 5, "new": 700, "least": 1000, "most": 6000, "Hq": 32, "Hkv": 8, "D": 128, "page": 16,
         "dtype": "bf16", "cache": "same", "window": 0, "causal": True},
        # Two chunks of up to 1024 tokens over long histories in an e4m3 cache.
        {"name": "attn-chunk-e4m3", "op": "attn", "B": 2, "new": 1024, "least": 8000, "most": 12000, "Hq": 32, "Hkv": 8, "D": 128,
         "page": 32, "dtype": "bf16", "cache": "e4m3", "window": 0, "causal": True},
        # The whole prompt of one request of a 7B-shaped model.
        {"name": "attn-prompt", "op": "attn", "B": 1, "new": 8192, "least": 8192, "most": 8192, "Hq": 32, "Hkv": 32, "D": 128, "page": 64,
         "dtype": "fp16", "cache": "same", "window": 0, "causal": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = [(32, 32), (40, 40), (32, 8), (8, 1), (16, 4), (40, 8), (12, 4), (8, 8)]    # (query heads, key heads)


def draw(rng):
    """One more case of the same ranges: sizes spread over their logarithm, odd ones among them."""
    op = rng.choice(["rope", "cache", "attn", "attn", "attn", "attn"])
    hq, hkv = rng.choice(HEADS)
    d, dtype = rng.choice([64, 128, 128]), rng.choice(["fp16", "bf16"])
    if op == "rope":
        return {"op": op, "T": _log_int(rng, 1, 8191), "Hq": hq, "Hkv": hkv, "D": d, "rot": rng.choice([d, d, d // 2]),
                "neox": rng.random() < 0.7, "dtype": dtype, "table": rng.choice(["same", "fp32"])}
    page = rng.choice([16, 16, 32, 48, 64, 128])
    cache = rng.choice(["same", "e4m3"])
    if op == "cache":
        t = _log_int(rng, 1, 8192)
        return {"op": op, "T": t, "R": min(8192, _log_int(rng, t, 4 * t)), "H": hkv, "D": d, "page": page, "dtype": dtype, "cache": cache}
    kind = rng.choice(["decode", "decode", "chunk", "chunk", "prompt"])
    case = {"op": op, "B": _log_int(rng, 1, 64), "new": 1, "Hq": hq, "Hkv": hkv, "D": d, "page": page, "dtype": dtype, "cache": cache,
            "window": 0, "causal": True}
    if kind == "decode":
        most = _log_int(rng, 64, 131072)
        case["B"] = max(1, min(case["B"], 400_000 * 8 // (most * hkv)))
        most = min(most, 400_000 * 8 // (case["B"] * hkv))
        case.update(most=most, least=max(1, int(most * rng.uniform(0.02, 1.0))))
    else:
        new = _log_int(rng, 2, 1500) if kind == "chunk" else _log_int(rng, 64, 8192)
        most = new if kind == "prompt" else new + _log_int(rng, 16, 12000)
        b = min(case["B"], 8)
        while b > 1 and b * new * most * hq * d > 6e10:
            b -= 1
        while new * most * hq * d > 1.3e11:
            new, most = max(1, new // 2), max(1, most // 2)
        case.update(B=b, new=new, most=most, least=max(new, int(most * rng.uniform(0.5, 1.0))))
        case["causal"] = kind == "prompt" or rng.random() < 0.8
    if case["causal"] and rng.random() < 0.2:
        case["window"] = _log_int(rng, 16, 4096)
    return case


# ------------------------------------------------------------------------------------------- inputs
def _plan(case):
    """(tokens in the cache, new tokens) of every sequence: the sizes of the case, whatever the seed of its values."""
    rng = random.Random("%(B)d %(new)d %(least)d %(most)d" % case)
    lengths = [rng.randint(case["least"], case["most"]) for _ in range(case["B"])]
    new = [case["new"] if case["new"] == 1 else rng.randint(1, case["new"]) for _ in range(case["B"])]
    lengths[-1], new[-1] = case["most"], case["new"]
    return lengths, [min(a, b) for a, b in zip(new, lengths)]


def _exponents(x):
    """Exponent byte of every row of x (its last axis): smallest e with max |x| <= 448 * 2^e, biased by 127."""
    m, e = torch.frexp(x.float().abs().amax(-1))
    e = torch.where(m == 0, torch.zeros_like(e), e - 9 + (m > 0.875).int())
    return (e.clamp(-126, 127) + 127).to(torch.uint8)


def _powers(b):
    return (b.int() << 23).view(torch.float32)        # 2^(b - 127) is the 32-bit number with this exponent field


def _encode(x):
    """(codes, exponent bytes) of the rows of x."""
    b = _exponents(x)
    return (x.float() / _powers(b)[..., None]).to(torch.float8_e4m3fn), b


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    dtype, dev = DTYPES[case["dtype"]], "cuda"
    D = case["D"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev, dtype=torch.float32).to(dtype)

    if case["op"] == "rope":
        T, Hq, Hkv, rot = case["T"], case["Hq"], case["Hkv"], case["rot"]
        qkv = normal(T, (Hq + 2 * Hkv) * D + 16) * 2                  # rows of a fused projection, padded
        angles = torch.outer(torch.arange(16384, dtype=torch.float64, device=dev),
                             10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=dev) / rot))
        table = torch.cat([angles.cos(), angles.sin()], 1)
        return {"case": case, "positions": torch.randint(0, 16384, (T,), generator=g, device=dev),
                "query": qkv[:, :Hq * D], "key": qkv[:, Hq * D:(Hq + Hkv) * D],
                "table": table.to(dtype if case["table"] == "same" else torch.float32),
                "query_weight": (1 + 0.1 * normal(D)).to(dtype), "key_weight": (1 + 0.1 * normal(D)).to(dtype), "eps": 1e-6,
                "query_out": torch.empty(T, Hq * D, dtype=dtype, device=dev), "key_out": torch.empty(T, Hkv * D, dtype=dtype, device=dev)}
    if case["op"] == "cache":
        T, R, H, page = case["T"], case["R"], case["H"], case["page"]
        pages = -(-max(T, R) // page) + 3
        x = normal(2, pages, page, H, D)
        if case["cache"] == "e4m3":
            (kc, ke), (vc, ve) = _encode(x[0]), _encode(x[1])
        else:
            (kc, ke), (vc, ve) = (x[0].clone(), None), (x[1].clone(), None)
        order = torch.randperm(pages, generator=g, device=dev)
        slots = (order[:, None] * page + torch.arange(page, device=dev)).reshape(-1)
        first = max(T, R) - T
        scale = torch.exp(0.5 * torch.randn(T, H, 1, generator=g, device=dev))     # heads of different magnitude
        qkv = (normal(T, 4, H, D) * scale[:, None]).to(dtype)
        return {"case": case, "key": qkv[:, 1], "value": qkv[:, 2], "key_cache": kc, "value_cache": vc, "key_exponents": ke,
                "value_exponents": ve, "write_slots": slots[first:first + T].clone(), "read_slots": slots[max(T, R) - R:max(T, R)].clone()}
    lengths, new = _plan(case)
    B, Hq, Hkv, page = case["B"], case["Hq"], case["Hkv"], case["page"]
    used = [-(-n // page) for n in lengths]
    pages = sum(used) + 2
    x = normal(pages, page, Hkv, D)
    kc, ke = _encode(x) if case["cache"] == "e4m3" else (x, None)
    x = normal(pages, page, Hkv, D)
    vc, ve = _encode(x) if case["cache"] == "e4m3" else (x, None)
    order = torch.randperm(pages, generator=g, device=dev).int()
    table = torch.zeros(B, max(used), dtype=torch.int32, device=dev)
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = order[at:at + n]
        at += n
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    return {"case": case, "query": normal(starts[-1], Hq + 1, D)[:, :Hq], "key_cache": kc, "value_cache": vc, "key_exponents": ke,
            "value_exponents": ve, "page_table": table, "lengths": torch.tensor(lengths, dtype=torch.int32, device=dev),
            "query_starts": None if case["new"] == 1 else torch.tensor(starts, dtype=torch.int32, device=dev),
            "scale": D ** -0.5, "longest": max(lengths), "most_new": max(new)}


# ------------------------------------------------------------------------------------------- plain forms
def _rope_plain(s):
    c = s["case"]
    T, D, rot = c["T"], c["D"], c["rot"]
    row = s["table"].float()[s["positions"]]
    cos, sin = row[:, None, :rot // 2], row[:, None, rot // 2:]

    def half(x, weight):
        x = x.reshape(T, -1, D).float()
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + s["eps"]) * weight.float()
        a, b = (x[..., :rot // 2], x[..., rot // 2:rot]) if c["neox"] else (x[..., 0:rot:2], x[..., 1:rot:2])
        a, b = a * cos - b * sin, b * cos + a * sin
        turned = torch.cat([a, b], -1) if c["neox"] else torch.stack([a, b], -1).flatten(-2)
        return torch.cat([turned, x[..., rot:]], -1).reshape(T, -1).to(DTYPES[c["dtype"]])

    return half(s["query"], s["query_weight"]), half(s["key"], s["key_weight"])


def _cache_plain(s):
    dtype = DTYPES[s["case"]["dtype"]]

    def half(x, cache, exponents):
        flat, w, r = cache.flatten(0, 1), s["write_slots"], s["read_slots"]
        if exponents is None:
            flat[w] = x
            return flat[r]
        codes, b = _encode(x)
        flat.view(torch.uint8)[w] = codes.view(torch.uint8)
        eflat = exponents.flatten(0, 1)
        eflat[w] = b
        return (flat.view(torch.uint8)[r].view(torch.float8_e4m3fn).float() * _powers(eflat[r])[..., None]).to(dtype)

    return half(s["key"], s["key_cache"], s["key_exponents"]), half(s["value"], s["value_cache"], s["value_exponents"])


def _gathered(cache, exponents, slots):
    """Keys or values [sequences, positions, heads, size] at the slots, in 32 bits."""
    if exponents is None:
        return cache.flatten(0, 1)[slots].float()
    x = cache.flatten(0, 1).view(torch.uint8)[slots].view(torch.float8_e4m3fn).float()
    return x * _powers(exponents.flatten(0, 1)[slots])[..., None]


def _attention_plain(s):
    c = s["case"]
    B, n, L, page, Hq, Hkv, D = c["B"], s["most_new"], s["longest"], c["page"], c["Hq"], c["Hkv"], c["D"]
    q, T, dev = s["query"], s["query"].shape[0], s["query"].device
    j = torch.arange(L, device=dev)
    slots = s["page_table"][:, j // page].long() * page + j % page
    k = _gathered(s["key_cache"], s["key_exponents"], slots)
    v = _gathered(s["value_cache"], s["value_exponents"], slots)
    starts = torch.arange(B + 1, device=dev) if s["query_starts"] is None else s["query_starts"].long()
    i = torch.arange(n, device=dev)
    rows, real = starts[:-1, None] + i, i < (starts[1:] - starts[:-1])[:, None]
    length = s["lengths"].long()[:, None]
    at = length - (starts[1:] - starts[:-1])[:, None] + i
    seen = (j < length)[:, None, :] & real[..., None]
    if c["causal"]:
        seen = seen & (j <= at[..., None])
    if c["window"]:
        seen = seen & (j > at[..., None] - c["window"])
    x = q[rows.clamp(max=T - 1)].float().view(B, n, Hkv, Hq // Hkv, D).permute(0, 2, 3, 1, 4)
    scores = (x.reshape(B, Hkv, -1, D) @ k.permute(0, 2, 3, 1)).view(B, Hkv, -1, n, L) * s["scale"]
    scores.masked_fill_(~seen[:, None, None], float("-inf"))
    p = torch.exp(scores - scores.amax(-1, keepdim=True).clamp(min=-1e30))
    o = (p.view(B, Hkv, -1, L) @ v.permute(0, 2, 1, 3)).view(B, Hkv, -1, n, D)
    o = o / p.sum(-1, keepdim=True).clamp(min=1e-30)
    out = torch.zeros(T + 1, Hq, D, dtype=q.dtype, device=dev)         # the last row takes what is padding
    out[torch.where(real, rows, T)] = o.permute(0, 3, 1, 2, 4).reshape(B, n, Hq, D).to(q.dtype)
    return out[:T]


# ------------------------------------------------------------------------------------------- one pass
def run(state):
    c = state["case"]
    if c["op"] == "rope":
        if not own:
            return _rope_plain(state)
        from triteia_b200 import capi
        capi.qk_norm_rotary_embedding(state["positions"], state["query"], state["key"], c["D"], state["table"], c["neox"],
                                      state["query_weight"], state["key_weight"], state["eps"], state["query_out"], state["key_out"])
        return state["query_out"], state["key_out"]
    if c["op"] == "cache":
        if not own:
            key, value = _cache_plain(state)
        else:
            from triteia_b200 import ops
            ops.cache_write(state["key"], state["value"], state["key_cache"], state["value_cache"], state["write_slots"],
                            state["key_exponents"], state["value_exponents"])
            key, value = ops.cache_read(state["key_cache"], state["value_cache"], state["read_slots"], state["key_exponents"],
                                        state["value_exponents"], dtype=DTYPES[c["dtype"]])
        out = {"key": key, "value": value}
        if c["cache"] == "e4m3":
            out.update(key_exponents=state["key_exponents"], value_exponents=state["value_exponents"])
        else:
            out.update(key_cache=state["key_cache"], value_cache=state["value_cache"])
        return out
    if not own:
        return _attention_plain(state)
    from triteia_b200 import ops
    return ops.paged_attention(state["query"], state["key_cache"], state["value_cache"], state["page_table"], state["lengths"],
                               state["query_starts"], scale=state["scale"], causal=c["causal"], window=c["window"] or None,
                               key_exponents=state["key_exponents"], value_exponents=state["value_exponents"])


# ------------------------------------------------------------------------------------------- what a pass needs
def _pairs(n, length, causal, window):
    """Number of (new token, visible position) pairs of a sequence."""
    if not causal:
        return n * length
    if not window:
        return n * (length - n) + n * (n + 1) // 2
    return sum(min(length - n + i + 1, window) for i in range(n))


def work(case):
    D = case["D"]
    if case["op"] == "rope":
        heads, esize = case["T"] * (case["Hq"] + case["Hkv"]), 2 if case["table"] == "same" else 4
        return {"bytes": 2 * heads * D * 2 + case["T"] * (case["rot"] * esize + 8), "flops": heads * (4 * D + 3 * case["rot"])}
    if case["op"] == "cache":
        H, T, R = case["H"], case["T"], case["R"]
        stored = H * (D + 1) if case["cache"] == "e4m3" else H * D * 2
        return {"bytes": 2 * (T + R) * (H * D * 2 + stored) + 8 * (T + R), "flops": 4 * (T + R) * H * D}
    lengths, new = _plan(case)
    stored = case["Hkv"] * (D + 1 if case["cache"] == "e4m3" else 2 * D)
    read = [min(a, case["window"] + n - 1) if case["window"] else a for a, n in zip(lengths, new)]
    pairs = sum(_pairs(n, a, case["causal"], case["window"]) for a, n in zip(lengths, new))
    return {"bytes": 2 * stored * sum(read) + 2 * sum(new) * case["Hq"] * D * 2, "flops": 4 * case["Hq"] * D * pairs}


# ------------------------------------------------------------------------------------------- in 64 bits
def _e4m3_nearest(x):
    """x rounded to the e4m3 grid: 4 significant bits, exponents from -6, ties to even, at most 448."""
    _, e = torch.frexp(x.abs())                      # x in [2^(e - 1), 2^e); a rounded logarithm would miss powers of two
    step = torch.exp2((e.double() - 1).clamp(min=-6) - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)


def _rope_exact(s):
    c = s["case"]
    D, rot = c["D"], c["rot"]
    row = s["table"].double()[s["positions"]]
    turn = torch.complex(row[:, :rot // 2], row[:, rot // 2:])[:, None]
    out = []
    for x, w in ((s["query"], s["query_weight"]), (s["key"], s["key_weight"])):
        x = x.double().reshape(c["T"], -1, D)
        x = x / (x.pow(2).sum(-1, keepdim=True) / D + s["eps"]).sqrt() * w.double()
        pair = x[..., :rot].reshape(c["T"], -1, 2, rot // 2).transpose(-1, -2) if c["neox"] else x[..., :rot].reshape(c["T"], -1, rot // 2, 2)
        z = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * turn)
        x[..., :rot] = (z.transpose(-1, -2) if c["neox"] else z).reshape(c["T"], -1, rot)
        out.append(x.reshape(c["T"], -1))
    return tuple(out)


def _cache_exact(s):
    c, out = s["case"], {}
    for name in ("key", "value"):
        x, cache, b = s[name].double(), s[name + "_cache"], s[name + "_exponents"]
        held = cache.flatten(0, 1).double()
        if c["cache"] == "e4m3":
            power = torch.exp2(b.flatten(0, 1).double() - 127)
            top = x.abs().amax(-1)
            e = torch.zeros_like(top)
            for k in range(-126, 128):                  # the smallest integer e with top <= 448 * 2^e
                e += (top > 448 * 2.0 ** (k - 1)) & (top > 0)
            e = torch.where(top > 0, e - 127, e).clamp(min=-126)
            held = held * power[..., None]
            held[s["write_slots"]] = _e4m3_nearest(x / torch.exp2(e)[..., None]) * torch.exp2(e)[..., None]
            b = b.clone()
            b.flatten(0, 1)[s["write_slots"]] = (e + 127).to(torch.uint8)
            out[name + "_exponents"] = b
        else:
            held[s["write_slots"]] = x
            out[name + "_cache"] = held.view(cache.shape)
        out[name] = held[s["read_slots"]]
    return out


def _attention_exact(s):
    c = s["case"]
    lengths, new = _plan(c)
    group, page, out, at = c["Hq"] // c["Hkv"], c["page"], [], 0
    for b, (length, n) in enumerate(zip(lengths, new)):
        used = s["page_table"][b, :-(-length // page)].long()
        place = torch.arange(n, device=used.device) + (length - n)
        j = torch.arange(length, device=used.device)
        hidden = torch.zeros(n, length, dtype=torch.bool, device=used.device)
        if c["causal"]:
            hidden |= j > place[:, None]
        if c["window"]:
            hidden |= j <= place[:, None] - c["window"]
        rows = torch.empty(n, c["Hq"], c["D"], dtype=torch.float64, device=used.device)
        for h in range(c["Hkv"]):
            kv = []
            for name in ("key", "value"):
                x = s[name + "_cache"][:, :, h].view(torch.uint8)[used] if c["cache"] == "e4m3" else s[name + "_cache"][:, :, h][used]
                if c["cache"] == "e4m3":
                    x = x.view(torch.float8_e4m3fn).double() * torch.exp2(s[name + "_exponents"][:, :, h][used].double() - 127)[..., None]
                kv.append(x.double().reshape(-1, c["D"])[:length])
            q = s["query"][at:at + n, h * group:(h + 1) * group].double()
            a = torch.einsum("nhd,ld->hnl", q, kv[0]).mul_(s["scale"]).masked_fill_(hidden, float("-inf"))
            rows[:, h * group:(h + 1) * group] = torch.einsum("hnl,ld->nhd", torch.softmax(a, -1), kv[1])
        out.append(rows)
        at += n
    return torch.cat(out)


def exact(case, seed):
    s = prepare(case, seed)
    return {"rope": _rope_exact, "cache": _cache_exact, "attn": _attention_exact}[case["op"]](s)
