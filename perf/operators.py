"""Operators for attention over prompts and over a key / value cache that is held in four bits, with what each of them costs at least.

Every case is one call, or the few calls that belong together, as a program that serves sequences makes them:

  prompt   attention of packed sequences of different lengths over their own keys: chunk-wise causal, with a window, heads shared in groups
  append   new keys and values rounded to four bits and put behind what a cache holds, then read back
  attend   the newest tokens of every row over the cached keys and values, with or without adding up the attention that each slot received
  evict    the slots that received most attention, and the newest ones, moved into a smaller cache

The four-bit format: 32 neighbouring channels of one token share a power of two, 2^(byte - 127), the smallest one (between bytes 16 and 252)
with which none of them is beyond 6; a channel is one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 or its negative, to nearest, ties to the even code
(sign in bit 3).  A group that holds an infinity or NaN gets byte 255 and reads as NaN.

`run` computes the operators with elementary torch operations where `own` is false, and calls the framework's where it is true."""
import math

import numpy as np
import torch

own = False

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# ---------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # the denoiser's own attention at base width: three guidance rows of one clip of 256 frames, a window of 8, chunks of 4
        dict(name="prompt_clip", op="prompt", type="fp32", seqs=3, low=256, high=256, heads=8, kv_heads=8, dim=64, window=8, chunk=4, prefix=0),
        # a handful of short requests of uneven length
        dict(name="prompt_short", op="prompt", type="bf16", seqs=5, low=17, high=211, heads=8, kv_heads=2, dim=64, window=0, chunk=1, prefix=0),
        # an ordinary batch of prompts, one token to two thousand, that continue a common prefix of 37 cached tokens
        dict(name="prompt_batch", op="prompt", type="fp16", seqs=16, low=1, high=2047, heads=32, kv_heads=8, dim=128, window=0, chunk=1, prefix=37),
        # one long prompt
        dict(name="prompt_long", op="prompt", type="bf16", seqs=1, low=16384, high=16384, heads=32, kv_heads=8, dim=128, window=0, chunk=1, prefix=0),
        # the keys and values of eight prompts enter empty rows
        dict(name="append_prompt", op="append", type="bf16", rows=8, low=1, high=4095, kv_heads=8, dim=128, capacity=4096, tokens=0),
        # one token for each of 64 rows that are filled to different lengths
        dict(name="append_token", op="append", type="fp16", rows=64, low=0, high=4095, kv_heads=8, dim=128, capacity=4096, tokens=1),
        # the smallest step: one row, one token, a few hundred slots
        dict(name="attend_small", op="attend", type="fp32", rows=1, low=300, high=300, heads=8, kv_heads=8, dim=64, capacity=512, tokens=1, count=False),
        # a step of a full batch
        dict(name="attend_batch", op="attend", type="bf16", rows=64, low=1, high=8192, heads=32, kv_heads=8, dim=128, capacity=8192, tokens=1, count=False),
        # two very long rows, with the attention of each slot added up
        dict(name="attend_long", op="attend", type="fp16", rows=2, low=131071, high=131071, heads=64, kv_heads=8, dim=128, capacity=131072, tokens=1, count=True),
        # the last 32 tokens of four prompts look at the whole prompt, to find out what of it is worth keeping
        dict(name="attend_observe", op="attend", type="bf16", rows=4, low=9001, high=16384, heads=32, kv_heads=8, dim=128, capacity=16384, tokens=32, count=True),
        # three short rows are halved
        dict(name="evict_small", op="evict", rows=3, low=400, high=1000, kv_heads=8, dim=64, capacity=1024, keep=509, recent=32),
        # eight long rows are cut to a quarter
        dict(name="evict_long", op="evict", rows=8, low=20001, high=32768, kv_heads=8, dim=128, capacity=32768, keep=8192, recent=1024),
    ]


def draw(rng):
    def log(a, b):
        return min(b, max(a, int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))))

    op = rng.choice(["prompt", "append", "attend", "attend", "evict"])
    dim, kv_heads, kind = rng.choice([64, 128]), rng.choice([1, 2, 4, 8]), rng.choice(["bf16", "fp16", "fp32"])
    if op == "prompt":
        seqs, group = log(1, 24), rng.choice([1, 2, 4, 8])
        high = log(1, max(1, 8192 // seqs)) if kind != "fp32" else log(1, max(1, 2048 // seqs))
        chunk = rng.choice([1, 1, 4])
        return dict(op=op, type=kind, seqs=seqs, low=log(1, high), high=high, heads=kv_heads * group, kv_heads=kv_heads, dim=dim,
                    window=rng.choice([0, 0, 8, 16, log(1, 1024)]), chunk=chunk, prefix=rng.choice([0, 0, log(1, 1000)]))
    rows = log(1, 64)
    high = log(33, max(64, min(65536, 2 ** 29 // (rows * kv_heads * dim))))
    capacity = -(-high // 32) * 32
    low = log(1, high)
    if op == "append":
        high = min(high, 16384)
        tokens = rng.choice([0, 1, log(1, 32)])
        return dict(op=op, type=kind, rows=rows, low=min(low, high), high=high, kv_heads=kv_heads, dim=dim, capacity=capacity + 32 * rng.choice([0, 1]), tokens=tokens)
    if op == "attend":
        tokens = rng.choice([1, 1, 2, log(1, 32)])
        return dict(op=op, type=kind, rows=rows, low=low, high=high, heads=kv_heads * rng.choice([1, 2, 4, 8]), kv_heads=kv_heads, dim=dim, capacity=capacity,
                    tokens=tokens, count=rng.random() < 0.5)
    keep = log(1, high)
    return dict(op=op, rows=rows, low=low, high=high, kv_heads=kv_heads, dim=dim, capacity=capacity, keep=keep, recent=rng.choice([0, log(1, keep)]))


def _lengths(case):
    """How long the sequences / rows of a case are: spread over [low, high], the longest among them."""
    n, low, high = case.get("seqs") or case["rows"], case["low"], case["high"]
    spread = [low + int((high - low) * math.modf((i + 1) * 0.6180339887498949)[0]) for i in range(n)]
    spread[n // 2] = high
    return spread


def _bounds(length, keys, window, chunk):
    """[first, last) of the keys that each query sees; the queries are the newest `length` of `keys` tokens."""
    at = np.arange(keys - length, keys)
    begin = at // chunk * chunk
    last = np.minimum(begin + chunk, keys)
    first = np.minimum(begin, np.maximum(0, at - window + 1)) if window else np.zeros_like(at)
    return first, last


def work(case):
    lens, dim, kv = _lengths(case), case["dim"], case["kv_heads"]
    token = kv * 2 * (dim // 2 + dim // 32)  # bytes of a cached token's keys and values
    if case["op"] == "prompt":
        pairs = 0
        for n in lens:
            first, last = _bounds(n, n + case["prefix"], case["window"], case["chunk"])
            pairs += int((last - first).sum())
        total, keys = sum(lens), sum(lens) + case["prefix"] * len(lens)
        return {"bytes": SIZE[case["type"]] * dim * (2 * total * case["heads"] + 2 * keys * kv), "flops": 4 * pairs * case["heads"] * dim}
    if case["op"] == "append":
        new = sum(lens) if not case["tokens"] else case["rows"] * case["tokens"]
        back = case["rows"] * (case["tokens"] or max(lens))
        return {"bytes": new * (token + 2 * kv * dim * SIZE[case["type"]]) + back * 2 * kv * dim * 2, "flops": 4 * new * kv * dim}
    if case["op"] == "attend":
        ends = case["rows"] * case["tokens"] * case["heads"] * dim * 2 * SIZE[case["type"]]
        return {"bytes": sum(lens) * token + ends + (8 * kv * sum(lens) if case["count"] else 0), "flops": 4 * sum(lens) * case["tokens"] * case["heads"] * dim}
    kept = sum(min(n, case["keep"]) for n in lens)
    return {"bytes": kv * 4 * sum(lens) + kept * (2 * token + 12 * kv) + case["rows"] * case["keep"] * 2 * kv * dim * 2, "flops": kv * sum(lens)}


# ---------------------------------------------------------------------------------------------------------------- four bits, in torch
def _round4(x):
    """[..., D] -> (codes [..., D], scale bytes [..., D / 32]), both uint8."""
    x = x.float().unflatten(-1, (-1, 32))
    top = x.abs().amax(-1)
    part, power = torch.frexp(top)  # top = part * 2^power, part in [0.5, 1): 6 * 2^e = 0.75 * 2^(e + 3)
    e = torch.where(part <= 0.75, power - 3, power - 2)
    e = torch.where(top > 0, e, -200).clamp(16 - 127, 252 - 127)
    bad = ~torch.isfinite(top)
    y = torch.ldexp(x, -e.unsqueeze(-1)).abs()
    code = (y > 0.25).to(torch.uint8) + (y >= 0.75) + (y > 1.25) + (y >= 1.75) + (y > 2.5) + (y >= 3.5) + (y > 5)
    code = code + 8 * torch.signbit(x)
    code = torch.where(bad.unsqueeze(-1), 0, code)
    return code.to(torch.uint8).flatten(-2), torch.where(bad, 255, e + 127).to(torch.uint8)


def _value4(code, scale):
    """The float32 values of codes [..., D] under scale bytes [..., D / 32]."""
    table = torch.tensor(GRID + tuple(-g for g in GRID), device=code.device)
    power = torch.where(scale == 255, math.nan, torch.ldexp(torch.ones((), device=code.device), scale.int() - 127))
    return (table[code.int()].unflatten(-1, (-1, 32)) * power.unsqueeze(-1)).flatten(-2)


def _pack(keys, values):
    """Codes [R, H, C, D] -> the cache's two buffers: keys two channels to a byte; values in blocks of eight tokens, two tokens to a byte,
    the channels of a block in the order [D / 2 % 16][D / 32][2]."""
    k = keys[..., 0::2] | keys[..., 1::2] << 4
    v = values.unflatten(2, (-1, 4, 2)).unflatten(-1, (-1, 16, 2))  # [R, H, C / 8, 4, 2, G, 16, 2]
    v = (v[:, :, :, :, 0] | v[:, :, :, :, 1] << 4).permute(0, 1, 2, 5, 4, 6, 3)  # [R, H, C / 8, 16, G, 2, 4]
    return k.contiguous(), v.reshape(*v.shape[:3], -1, 4).contiguous()


def _keys(c):
    k = torch.stack([c["keys"] & 15, c["keys"] >> 4], -1).flatten(-2)
    return _value4(k, c["key_scales"])


def _values(c):
    v = torch.stack([c["values"] & 15, c["values"] >> 4], -1).flatten(-2)  # [R, H, C / 8, D, 8]
    v = v.unflatten(3, (16, -1, 2)).permute(0, 1, 2, 6, 4, 3, 5)  # [R, H, C / 8, 8, G, 16, 2]
    return _value4(v.flatten(-3).flatten(2, 3), c["value_scales"])


# ---------------------------------------------------------------------------------------------------------------- inputs
def _tokens(g, *shape):
    """Keys or values as a trained layer makes them: a few channels carry much more than the others, and an offset."""
    dim = shape[-1]
    lift = 1 + 4 * (torch.rand(dim, generator=g, device="cuda") < 0.06)
    return torch.randn(*shape, generator=g, device="cuda") * lift + torch.randn(dim, generator=g, device="cuda") * 0.5


def _filled(case, g, lens):
    rows, kv, dim, cap = case["rows"], case["kv_heads"], case["dim"], case["capacity"]
    keys, key_scales = _round4(_tokens(g, rows, kv, cap, dim))
    values, value_scales = _round4(_tokens(g, rows, kv, cap, dim))
    keys, values = _pack(keys, values)
    lengths = torch.tensor(lens, dtype=torch.int32, device="cuda")
    held = torch.arange(cap, device="cuda") < lengths[:, None, None]
    weights = torch.where(held, torch.rand(rows, kv, cap, generator=g, device="cuda") ** 6, 0)
    # few slots receive most of the attention, and several exactly none or the same
    weights = torch.where(torch.rand(rows, kv, cap, generator=g, device="cuda") < 0.1, (weights * 8).floor() / 8, weights)
    return dict(keys=keys, key_scales=key_scales, values=values, value_scales=value_scales, weights=weights, lengths=lengths)


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    lens, dim, kv = _lengths(case), case["dim"], case["kv_heads"]
    s = dict(case=case, lens=lens)
    if case["op"] == "prompt":
        kind, heads, total = TYPES[case["type"]], case["heads"], sum(lens)
        keys = [n + case["prefix"] for n in lens]
        # one projection's output, as the three are cut from it
        fused = torch.cat([torch.randn(sum(keys), heads, dim, generator=g, device="cuda"), _tokens(g, sum(keys), 2 * kv, dim)], 1).to(kind)
        s["k"], s["v"] = fused[:, heads:heads + kv], fused[:, heads + kv:]
        s["q"] = fused[:total, :heads]
        s["starts"] = torch.tensor(np.cumsum([0] + lens), dtype=torch.int32, device="cuda")
        s["key_starts"] = torch.tensor(np.cumsum([0] + keys), dtype=torch.int32, device="cuda") if case["prefix"] else s["starts"]
        s["key_lens"] = keys
        return s
    if case["op"] == "append":
        kind, rows, tokens = TYPES[case["type"]], case["rows"], case["tokens"]
        shape = (rows * tokens if tokens else sum(lens), kv, dim)
        s["k"], s["v"] = _tokens(g, *shape).to(kind), _tokens(g, *shape).to(kind)
        counts = [tokens] * rows if tokens else lens
        s["starts"] = torch.tensor(np.cumsum([0] + counts), dtype=torch.int32, device="cuda")
        s["row"] = torch.repeat_interleave(torch.arange(rows, device="cuda"), torch.tensor(counts, device="cuda"))
        s["held"] = torch.tensor([min(n, case["capacity"] - tokens) if tokens else 0 for n in lens], dtype=torch.int32, device="cuda")
        s["back"] = tokens or max(lens)
        return s
    s["cache"] = _filled(case, g, lens)
    if case["op"] == "attend":
        s["q"] = (1.5 * torch.randn(case["rows"], case["tokens"], case["heads"], dim, generator=g, device="cuda")).to(TYPES[case["type"]])
        s["received"] = s["cache"]["weights"].clone()
    return s


# ---------------------------------------------------------------------------------------------------------------- the calls
def _prompt(s):
    c = s["case"]
    kind, dim, kv = s["q"].dtype, c["dim"], c["kv_heads"]
    out = torch.empty(*s["q"].shape, device="cuda", dtype=kind)
    b = a = 0
    for n, m in zip(s["lens"], s["key_lens"]):  # one sequence after the other: each has scores of its own shape
        q = s["q"][a:a + n].float().unflatten(1, (kv, -1)).permute(1, 2, 0, 3).flatten(1, 2) * (1 / math.sqrt(dim))  # [KV, G n, D]
        k, v = s["k"][b:b + m].float().transpose(0, 1), s["v"][b:b + m].float().transpose(0, 1)
        x = (q @ k.transpose(1, 2)).unflatten(1, (-1, n))
        at = torch.arange(m - n, m, device="cuda")
        begin = at // c["chunk"] * c["chunk"]
        first = torch.minimum(begin, (at - c["window"] + 1).clamp(min=0)) if c["window"] else torch.zeros_like(at)
        key = torch.arange(m, device="cuda")
        x.masked_fill_((key < first[:, None]) | (key >= (begin + c["chunk"])[:, None]), -math.inf)
        x = x.sub_(x.amax(-1, keepdim=True)).exp_()
        total = x.sum(-1, keepdim=True)
        y = (x.flatten(1, 2) @ v).unflatten(1, (-1, n)) / total
        out[a:a + n] = y.permute(2, 0, 1, 3).flatten(1, 2).to(kind)
        a, b = a + n, b + m
    return {"out": out}


def _append(s):
    c = s["case"]
    rows, kv, dim, back = c["rows"], c["kv_heads"], c["dim"], s["back"]
    at = torch.arange(len(s["row"]), device="cuda") - s["starts"][:-1].long()[s["row"]]
    k = _value4(*_round4(s["k"])).to(torch.bfloat16)
    v = _value4(*_round4(s["v"])).to(torch.bfloat16)
    found = []
    for x in (k, v):
        y = torch.zeros(rows, back, kv, dim, device="cuda", dtype=torch.bfloat16)
        y[s["row"], at] = x
        found.append(y.transpose(1, 2).contiguous())
    return {"keys": found[0], "values": found[1], "lengths": s["held"] + s["starts"].diff()}


def _attend(s):
    c, q, cache = s["case"], s["q"], s["cache"]
    k, v, lengths = _keys(cache), _values(cache), cache["lengths"]
    rows, tokens, heads, dim = q.shape
    x = q.float().unflatten(2, (c["kv_heads"], -1)).permute(0, 2, 3, 1, 4).flatten(2, 3) @ k.transpose(2, 3) * (1 / math.sqrt(dim))  # [R, KV, G T, C]
    x = x.unflatten(2, (-1, tokens))
    last = lengths[:, None] - tokens + 1 + torch.arange(tokens, device="cuda")  # [R, T]
    seen = torch.arange(k.shape[2], device="cuda") < last[:, None, None, :, None]
    x = x.masked_fill_(~seen, -math.inf)
    x = x.sub_(x.amax(-1, keepdim=True).clamp(min=-3e38)).exp_()
    x = x.div_(x.sum(-1, keepdim=True).clamp(min=1e-30))
    y = (x.flatten(2, 3) @ v).unflatten(2, (-1, tokens)).permute(0, 3, 1, 2, 4).flatten(2, 3).to(q.dtype)
    if not c["count"]:
        return {"out": y}
    return {"out": y, "weights": s["received"] + x.sum((2, 3))}


def _evict(s):
    c, cache = s["case"], s["cache"]
    lengths, weights = cache["lengths"], cache["weights"]
    slot = torch.arange(weights.shape[2], device="cuda")
    n = lengths[:, None, None]
    rank = torch.where(slot >= n - c["recent"], math.inf, weights)
    rank = torch.where(slot < n, rank, -math.inf)
    kept = rank.sort(dim=-1, descending=True, stable=True).indices[..., :c["keep"]].sort(-1).values
    new = lengths.clamp(max=c["keep"])
    alive = torch.arange(c["keep"], device="cuda") < new[:, None, None]
    kept = torch.where(alive, kept, 0)
    k, v = (torch.where(alive[..., None], x.gather(2, kept[..., None].expand(-1, -1, -1, c["dim"])), 0).to(torch.bfloat16) for x in (_keys(cache), _values(cache)))
    return {"slots": torch.where(alive, kept, -1).int(), "lengths": new, "keys": k, "values": v, "weights": torch.where(alive, weights.gather(2, kept), 0)}


def _cache(s, capacity):
    """The framework's cache of a case, made once, as a program that serves keeps it."""
    from after_amd import KVCache4
    c = s["case"]
    if "handle" not in s:
        s["handle"] = KVCache4(c["rows"], c["kv_heads"], c["dim"], c["capacity"], device="cuda", buffers=s.get("cache"))
        if c["op"] == "append":
            s["handle"].lengths.copy_(s["held"])  # its rows hold that many slots already
        if c["op"] == "evict":
            s["smaller"] = KVCache4(c["rows"], c["kv_heads"], c["dim"], capacity, device="cuda")
    return s["handle"]


def _own(s):
    c = s["case"]
    if c["op"] == "prompt":
        from after_amd import attend_packed
        return {"out": attend_packed(s["q"], s["k"], s["v"], s["starts"], s["key_starts"], window=c["window"] or None, chunk=c["chunk"])}
    cache = _cache(s, c.get("keep"))
    if c["op"] == "append":
        cache.truncate(s["held"])
        cache.append(s["k"], s["v"], s["starts"])
        k, v = cache.read(s["held"], s["back"])
        return {"keys": k, "values": v, "lengths": cache.lengths}
    if c["op"] == "attend":
        if not c["count"]:
            return {"out": cache.attend(s["q"])}
        cache.weights.copy_(s["received"])  # each pass adds to the same sums
        return {"out": cache.attend(s["q"], accumulate=True), "weights": cache.weights}
    slots = cache.evict(s["smaller"], c["keep"], c["recent"])
    k, v = s["smaller"].read(count=c["keep"])
    return {"slots": slots, "lengths": s["smaller"].lengths, "keys": k, "values": v, "weights": s["smaller"].weights[..., :c["keep"]]}


def run(state):
    if own:
        return _own(state)
    return {"prompt": _prompt, "append": _append, "attend": _attend, "evict": _evict}[state["case"]["op"]](state)


# ---------------------------------------------------------------------------------------------------------------- in 64 bits
def _exact_round(x):
    """Nearest of the fifteen multiples of each group's power of two, by distance."""
    g = x.double().unflatten(-1, (-1, 32))
    top = g.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(torch.where(top > 0, top, 1.0) / 6)).clamp(-111, 125)
    e = torch.where(6 * 2.0 ** (e - 1) >= top, e - 1, e)  # a logarithm next to a whole number may be off either way
    e = torch.where(6 * 2.0 ** e < top, e + 1, e).clamp(-111, 125)
    y = (g.abs() / 2.0 ** e).clamp(max=6)
    grid = torch.tensor([0, 1, 2, 4, 0.5, 1.5, 3, 6], dtype=torch.float64, device=x.device)  # the even codes first: they win a tie
    best, far = torch.zeros_like(y), torch.full_like(y, math.inf)
    for v in grid:
        d = (y - v).abs()
        best, far = torch.where(d < far, v, best), torch.minimum(d, far)
    return (torch.sign(g) * best * 2.0 ** e).flatten(-2)


def _exact_value(byte, scale):
    """One nibble each, as sign, two bits of exponent and one of fraction."""
    sign, ex, frac = 1 - 2 * (byte >> 3).double(), (byte >> 1 & 3).double(), (byte & 1).double()
    v = torch.where(ex > 0, (1 + frac / 2) * 2.0 ** (ex - 1), frac / 2)
    p = 2.0 ** (scale.double() - 127)
    return sign * v * p.masked_fill(scale == 255, math.nan).repeat_interleave(32, -1)


def _exact_row(cache, r):
    """(keys, values) of a row, [H, C, D]."""
    k, v = cache["keys"][r], cache["values"][r]
    H, C, half = k.shape
    out = torch.empty(H, C, 2 * half, dtype=torch.uint8, device="cuda")
    out[..., 0::2], out[..., 1::2] = k & 15, k >> 4
    val = torch.empty_like(out)
    channel = torch.arange(2 * half, device="cuda")
    place = channel // 2 % 16 * (2 * half // 16) + channel // 32 * 2 + channel % 2
    for t in range(8):
        val[:, t::8] = (v[..., place, t // 2] >> 4 * (t % 2)) & 15
    return _exact_value(out, cache["key_scales"][r]), _exact_value(val, cache["value_scales"][r])


def exact(case, seed):
    s = prepare(case, seed)
    dim, kv = case["dim"], case["kv_heads"]
    if case["op"] == "prompt":
        group = case["heads"] // kv
        out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
        a = b = 0
        for n, m in zip(s["lens"], s["key_lens"]):
            first, last = (torch.tensor(t, device="cuda")[:, None] for t in _bounds(n, m, case["window"], case["chunk"]))
            key = torch.arange(m, device="cuda")[None]
            seen = (key >= first) & (key < last)
            for h in range(case["heads"]):
                x = s["q"][a:a + n, h].double() @ s["k"][b:b + m, h // group].double().T / math.sqrt(dim)
                out[a:a + n, h] = torch.softmax(x.masked_fill_(~seen, -math.inf), -1) @ s["v"][b:b + m, h // group].double()
            a, b = a + n, b + m
        return {"out": out}
    if case["op"] == "append":
        found = {"lengths": s["held"].long() + s["starts"].long().diff()}
        cuts = s["starts"].tolist()
        for name, x in (("keys", s["k"]), ("values", s["v"])):
            y = torch.zeros(case["rows"], kv, s["back"], dim, dtype=torch.float64, device="cuda")
            for r in range(case["rows"]):
                y[r, :, :cuts[r + 1] - cuts[r]] = _exact_round(x[cuts[r]:cuts[r + 1]]).transpose(0, 1)
            found[name] = y
        return {"keys": found["keys"], "values": found["values"], "lengths": found["lengths"].int()}
    cache = s["cache"]
    if case["op"] == "attend":
        T, group = case["tokens"], case["heads"] // kv
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        got = s["received"].double()
        for r, n in enumerate(s["lens"]):
            k, v = _exact_row(cache, r)
            for t in range(max(0, T - n), T):
                m = n - T + t + 1
                p = torch.softmax(s["q"][r, t].double().view(kv, group, dim) @ k[:, :m].transpose(1, 2) / math.sqrt(dim), -1)
                out[r, t] = (p @ v[:, :m]).reshape(-1, dim)
                got[r, :, :m] += p.sum(1)
        return {"out": out, "weights": got} if case["count"] else {"out": out}
    keep, recent = case["keep"], case["recent"]
    slots = torch.full((case["rows"], kv, keep), -1, dtype=torch.int64)
    ks, vs = (torch.zeros(case["rows"], kv, keep, dim, dtype=torch.float64, device="cuda") for _ in range(2))
    weights = torch.zeros(case["rows"], kv, keep, dtype=torch.float64, device="cuda")
    w = cache["weights"].cpu().numpy()
    for r, n in enumerate(s["lens"]):
        k, v = _exact_row(cache, r)
        old, m = max(0, n - recent), min(n, keep)
        for h in range(kv):
            best = np.argsort(-w[r, h, :old], kind="stable")[:max(0, m - (n - old))] if m < n else np.arange(old)
            newest = np.arange(n - min(n - old, m), n) if m == n or recent <= keep else np.arange(n - keep, n)
            at = torch.tensor(np.sort(np.concatenate([best, newest])))
            slots[r, h, :m] = at
            ks[r, h, :m], vs[r, h, :m] = k[h, at.cuda()], v[h, at.cuda()]
            weights[r, h, :m] = cache["weights"][r, h, at.cuda()].double()
    return {"slots": slots.int(), "lengths": torch.tensor([min(n, keep) for n in s["lens"]], dtype=torch.int32), "keys": ks, "values": vs, "weights": weights}
