"""Cases of the 4-bit KV cache: quantising rows as they are written, reading them back, decode attention over the cache
(full layers, and sliding-window layers whose first tokens stay visible) and prefill attention into it.

A cache row (one token, one KV head, K or V) is 128 values x, rounded to half, in four groups of 32.  A group keeps
    lo = min x,  d = half((max x - lo) / 15),  code = round-half-even((x - lo) / d) limited to 0..15 (0 where d = 0)
and stands for lo + code * d.  Attention is the model's: 32 query heads over 4 KV heads of 128, RMSNorm with weight on q
and k, rotation by position on layers that have it, one learned sink per head in the denominator.  Tokens of a call are
attended at half precision, everything older as the cache holds it.
"""
import math

import torch

own = False

HEADS, KV_HEADS, DIM, GROUP = 32, 4, 128, 32
QKV = (HEADS + 2 * KV_HEADS) * DIM
WINDOW, RING = 513, 1024       # sliding-window layers: keys a query sees, itself included; rows their cache keeps
ROW_BYTES = 2 * (DIM // 2 + 4 * DIM // GROUP)  # K and V of one token and KV head: codes, and d and lo of each group
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def listed():
    return [
        # a serving step's rows written into the caches of its 64 sequences: latency
        {"name": "store_step", "op": "store", "n": 64, "rows": 1, "at": 4095, "type": "bfloat16", "paged": True},
        # a prompt of 16384 tokens prefilled elsewhere, brought into the cache
        {"name": "store_prompt", "op": "store", "n": 1, "rows": 16384, "at": 0, "type": "float16", "paged": False},
        # a few hundred rows of a few sequences, from the middle of a page on
        {"name": "load_ragged", "op": "load", "n": 7, "rows": 229, "at": 1001, "type": "bfloat16", "paged": True},
        # a long context read back whole, for a layer that wants it in half precision
        {"name": "load_long", "op": "load", "n": 1, "rows": 131071, "at": 0, "type": "float16", "paged": False},
        # one short conversation: latency
        {"name": "decode_short", "op": "decode", "n": 1, "shortest": 317, "longest": 317, "rope": True, "type": "float32", "paged": False},
        # a full batch of equal contexts: the benchmark's 64 x 8192
        {"name": "decode_batch", "op": "decode", "n": 64, "shortest": 8192, "longest": 8192, "rope": False, "type": "bfloat16", "paged": False},
        # a server's mix, from an empty cache to a long context, on pages
        {"name": "decode_ragged", "op": "decode", "n": 32, "shortest": 0, "longest": 32768, "rope": False, "type": "bfloat16", "paged": True},
        # one very long context
        {"name": "decode_long", "op": "decode", "n": 1, "shortest": 131072, "longest": 131072, "rope": False, "type": "bfloat16", "paged": False},
        # sliding-window layer, far positions, four first tokens that stay visible
        {"name": "window_far", "op": "window", "n": 32, "shortest": 9000, "longest": 100001, "first": 4, "rope": True, "type": "float32"},
        # a large mixed batch on a sliding-window layer: new sequences and old ones, a whole block of first tokens
        {"name": "window_batch", "op": "window", "n": 256, "shortest": 0, "longest": 40000, "first": 64, "rope": True, "type": "bfloat16"},
        # a chunk of a prompt behind a cached context, full layer
        {"name": "prefill_chunk", "op": "prefill", "tokens": 512, "past": 16384, "window": False, "first": 0, "rope": False, "type": "bfloat16"},
        # the benchmark's 4000-token prompt on a sliding-window layer, with first tokens
        {"name": "prefill_window", "op": "prefill", "tokens": 4000, "past": 0, "window": True, "first": 4, "rope": True, "type": "bfloat16"},
    ]


def _spread(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["store", "load", "decode", "window", "prefill"])
    kind = rng.choice(["float32", "bfloat16"])
    if op in ("store", "load"):
        n = _spread(rng, 1, 64)
        rows = _spread(rng, 1, (16384 if op == "store" else 131071) // n)
        return {"op": op, "n": n, "rows": rows, "at": rng.randrange(4096), "type": rng.choice(list(TYPES)),
                "paged": rng.random() < 0.5}
    if op == "decode":
        n = _spread(rng, 1, 64)
        longest = _spread(rng, 1, min(131072, 524288 // n))
        return {"op": op, "n": n, "shortest": longest if rng.random() < 0.3 else rng.randrange(longest), "longest": longest, "rope": rng.random() < 0.5,
                "type": kind, "paged": rng.random() < 0.5}
    if op == "window":
        longest = _spread(rng, 1, 120000)
        return {"op": op, "n": _spread(rng, 1, 256), "shortest": rng.randrange(longest), "longest": longest, "first": rng.choice([0, 1, 4, 16, 33, 64]),
                "rope": rng.random() < 0.7, "type": kind}
    if rng.random() < 0.5:  # sliding window: the ring keeps a call's history only while the call has at most 512 tokens
        tokens = _spread(rng, 1, 4000)
        return {"op": op, "tokens": tokens, "past": rng.randrange(20000) if tokens <= RING // 2 else 0, "window": True,
                "first": rng.choice([0, 1, 4, 16, 33, 64]), "rope": True, "type": kind}
    tokens = _spread(rng, 1, 2048)
    return {"op": op, "tokens": tokens, "past": rng.randrange(min(16384, 4000000 // tokens)), "window": False, "first": 0, "rope": rng.random() < 0.5,
            "type": kind}


def _positions(case):
    """Positions of the new tokens of a decode call: spread evenly over the logarithm, neighbours in the batch far apart."""
    n, lo, hi = case["n"], case["shortest"], case["longest"]
    at = [round(math.exp(math.log(lo + 1) + (math.log(hi + 1) - math.log(lo + 1)) * i / max(1, n - 1))) - 1 for i in range(n)]
    step = next(s for s in range(n // 2 + 1, 2 * n + 2) if math.gcd(s, n) == 1)
    return [at[i * step % n] for i in range(n)]


def _seen(pos, first):
    """Cached keys that a query at `pos` of a sliding-window layer sees."""
    old = max(0, pos - (WINDOW - 1))
    return pos - old + min(first, old)


def work(case):
    op, size = case["op"], {"float32": 4, "bfloat16": 2, "float16": 2}[case["type"]]
    if op in ("store", "load"):
        rows = case["n"] * case["rows"] * KV_HEADS
        if op == "store":  # the rows as they were given, the cache, and the values that the cache then stands for
            return {"bytes": rows * (2 * DIM * size + ROW_BYTES + 2 * DIM * 2), "flops": rows * 2 * DIM * 8}
        return {"bytes": rows * (2 * DIM * size + ROW_BYTES), "flops": rows * 2 * DIM * 2}
    if op in ("decode", "window"):
        keys = sum(p if op == "decode" else _seen(p, case["first"]) for p in _positions(case))
        new = case["n"]
        pairs = keys + new
    else:
        new, past = case["tokens"], case["past"]
        if case["window"]:
            pairs = sum(_seen(p, case["first"]) + 1 for p in range(past, past + new))
            keys = _seen(past, case["first"])
        else:
            pairs, keys = new * past + new * (new + 1) // 2, past
    kept = new if op != "prefill" or not case["window"] else min(new, RING)
    return {"bytes": new * (QKV * size + HEADS * DIM * 2) + (keys + kept) * KV_HEADS * ROW_BYTES + kept * KV_HEADS * 2 * DIM * 2,
            "flops": pairs * HEADS * DIM * 4}


# ---------------------------------------------------------------------------------------------- inputs
def _normal(gen, *shape):
    return torch.randn(*shape, device="cuda", generator=gen)


def _inputs(case, seed):
    """What the seed decides: raw q|k|v rows, norm weights, sinks, and the half-precision rows that the cache was written from."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    op, d = case["op"], {}
    if op in ("store", "load"):
        rows, per = case["rows"], (case["n"], KV_HEADS)
    elif op == "decode":
        rows, per = max(1, case["longest"]), (case["n"], KV_HEADS)
    elif op == "window":
        rows, per = RING, (case["n"], KV_HEADS)
    else:
        rows, per = (min(case["past"], WINDOW - 1) if case["window"] else case["past"]), (1, KV_HEADS)
    # keys have some channels larger than others, and values a mean
    d["k"] = (_normal(gen, *per, rows, DIM) * (0.7 + 0.6 * torch.rand(KV_HEADS, 1, DIM, device="cuda", generator=gen))).to(torch.float16)
    d["v"] = (_normal(gen, *per, rows, DIM) + 0.3 * _normal(gen, KV_HEADS, 1, DIM)).to(torch.float16)
    if op in ("store", "load"):
        return d
    # rows of the first tokens; those that the rows above hold too are the same there
    at = torch.tensor(_positions(case) if op == "window" else [case.get("past", 0)], device="cuda")
    j = torch.arange(64, device="cuda")
    for x in "kv":
        d[x + "_first"] = _normal(gen, *per, 64, DIM).to(torch.float16)
        if op == "window":  # slot j of the ring holds position j
            d[x + "_first"] = torch.where((j >= at[:, None] - RING)[:, None, :, None], d[x][:, :, :64], d[x + "_first"])
        elif op == "prefill" and case["window"]:
            start = case["past"] - rows
            d[x + "_first"][:, :, start:case["past"]] = d[x][:, :, :max(0, 64 - start)]
    n = case["tokens"] if op == "prefill" else case["n"]
    d["qkv"] = _normal(gen, n, QKV).to(TYPES[case["type"]])
    d["q_norm"], d["k_norm"] = (1 + 0.1 * _normal(gen, DIM) for _ in range(2))
    d["sinks"] = _normal(gen, HEADS)
    return d


def _quantise(x):
    """Codes, two to a byte, and d and lo of each group, of half-precision rows."""
    g = x.float().unflatten(-1, (DIM // GROUP, GROUP))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    d = ((hi - lo) / 15).to(torch.float16).float()
    code = torch.where(d > 0, ((g - lo) / d).round(), 0).clamp(0, 15).to(torch.uint8).flatten(-2)
    return code[..., 0::2] | code[..., 1::2] << 4, d.squeeze(-1).to(torch.float16), lo.squeeze(-1).to(torch.float16)


def _values(packed):
    """What the codes stand for, in 32 bits."""
    codes, d, lo = packed
    code = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float().unflatten(-1, (DIM // GROUP, GROUP))
    return (lo.float()[..., None] + code * d.float()[..., None]).flatten(-2)


def _ring_at(pos):
    """Positions that the slots of a ring hold in front of a token at `pos` (negative: none yet)."""
    slot = torch.arange(RING, device="cuda")
    return pos[:, None] - 1 - (pos[:, None] - 1 - slot) % RING


def prepare(case, seed):
    op, d = case["op"], _inputs(case, seed)
    s = {"case": case, "type": TYPES[case["type"]]}
    if op == "store":
        s["k"], s["v"] = d["k"].to(s["type"]), d["v"].to(s["type"])
    elif op != "load":
        s.update({k: d[k] for k in ("qkv", "q_norm", "k_norm", "sinks")})
        s["pos"] = torch.tensor(_positions(case) if op != "prefill" else [case["past"]], device="cuda")
    if own:
        _open(s, case, d)
        return s
    if op != "store":
        s["k"], s["v"] = _quantise(d["k"]), _quantise(d["v"])
    if op in ("window", "prefill"):
        s["k_first"], s["v_first"] = _quantise(d["k_first"]), _quantise(d["v_first"])
    return s


# ---------------------------------------------------------------------------------------------- plain form
def _norm_rope(x, weight, pos, rope):
    """x [tokens][heads][128] -> RMSNorm with weight, then dims i and i + 64 turned by pos * 10000^(-i / 64).  The model's
    angle is that product of two 32-bit numbers, rounded to 32 bits; its sine and cosine are taken in 64."""
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * weight
    if not rope:
        return x
    freq = (10000.0 ** (-torch.arange(DIM // 2, device="cuda", dtype=torch.float64) / (DIM // 2))).float()
    angle = (pos.float()[:, None] * freq).double()[:, None]
    cos, sin = angle.cos().float(), angle.sin().float()
    a, b = x[..., :DIM // 2], x[..., DIM // 2:]
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)


def _attend(q, k, v, seen, sinks):
    """q [..][rows][128], k and v [..][keys][128], seen [..][rows][keys], sinks [..][rows][1]."""
    score = (q @ k.transpose(-1, -2) / math.sqrt(DIM)).masked_fill(~seen, -math.inf)
    top = torch.maximum(score.amax(-1, keepdim=True), sinks)
    p = (score - top).exp()
    return p @ v / (p.sum(-1, keepdim=True) + (sinks - top).exp())


def _plain_decode(s, case):
    n, pos, window = case["n"], s["pos"], case["op"] == "window"
    x = s["qkv"].float().view(n, HEADS + 2 * KV_HEADS, DIM)
    rope = case["rope"]
    q = _norm_rope(x[:, :HEADS], s["q_norm"], pos, rope).view(n, KV_HEADS, HEADS // KV_HEADS, DIM)
    k_new = _norm_rope(x[:, HEADS:HEADS + KV_HEADS], s["k_norm"], pos, rope).to(torch.float16)
    v_new = x[:, HEADS + KV_HEADS:].to(torch.float16)
    k, v = [_values(s["k"])], [_values(s["v"])]
    if window:
        at = _ring_at(pos)
        seen = [(at >= 0) & (at > pos[:, None] - WINDOW)]
        k.append(_values(s["k_first"]))
        v.append(_values(s["v_first"]))
        j = torch.arange(64, device="cuda")
        seen.append((j < case["first"]) & (j < pos[:, None] - (WINDOW - 1)))
    else:
        seen = [torch.arange(k[0].shape[2], device="cuda") < pos[:, None]]
    k.append(k_new.float()[:, :, None])
    v.append(v_new.float()[:, :, None])
    seen.append(torch.ones(n, 1, dtype=torch.bool, device="cuda"))
    out = _attend(q, torch.cat(k, 2), torch.cat(v, 2), torch.cat(seen, 1)[:, None, None], s["sinks"].view(KV_HEADS, -1, 1))
    return {"out": out.reshape(n, HEADS * DIM).to(torch.bfloat16),
            "k": _values(_quantise(k_new[:, :, None])).to(torch.float16), "v": _values(_quantise(v_new[:, :, None])).to(torch.float16)}


def _plain_prefill(s, case):
    n, past, window, first = case["tokens"], case["past"], case["window"], case["first"]
    pos = torch.arange(past, past + n, device="cuda")
    x = s["qkv"].float().view(n, HEADS + 2 * KV_HEADS, DIM)
    q = _norm_rope(x[:, :HEADS], s["q_norm"], pos, case["rope"])
    q = q.view(n, KV_HEADS, HEADS // KV_HEADS, DIM).permute(1, 2, 0, 3).reshape(KV_HEADS, -1, DIM)
    k_new = _norm_rope(x[:, HEADS:HEADS + KV_HEADS], s["k_norm"], pos, case["rope"]).to(torch.float16).transpose(0, 1)
    v_new = x[:, HEADS + KV_HEADS:].to(torch.float16).transpose(0, 1)
    k, v, at = [_values(s["k"])[0]], [_values(s["v"])[0]], [torch.arange(past - s["k"][0].shape[2], past, device="cuda")]
    k.append(k_new.float())
    v.append(v_new.float())
    at.append(pos)
    seen = torch.cat(at) <= pos[:, None]
    if window:
        at = torch.cat(at)
        seen &= (at > pos[:, None] - WINDOW) | (at < first)
        # first tokens that neither the call nor the window's history brings along
        k.append(_values(s["k_first"])[0])
        v.append(_values(s["v_first"])[0])
        j = torch.arange(64, device="cuda")
        seen = torch.cat((seen, ((j < first) & (j < max(0, past - (WINDOW - 1)))).expand(n, 64)), 1)
    out = _attend(q, torch.cat(k, 1), torch.cat(v, 1), seen.repeat(HEADS // KV_HEADS, 1),
                  s["sinks"].view(KV_HEADS, -1, 1).repeat_interleave(n, 1))
    out = out.view(KV_HEADS, HEADS // KV_HEADS, n, DIM).permute(2, 0, 1, 3).reshape(n, HEADS * DIM)
    kept = min(n, RING) if window else n
    return {"out": out.to(torch.bfloat16), "k": _values(_quantise(k_new[:, n - kept:])).to(torch.float16),
            "v": _values(_quantise(v_new[:, n - kept:])).to(torch.float16)}


# ---------------------------------------------------------------------------------------------- the framework's calls
def _open(s, case, d):
    """A handle with one layer in the 4-bit format, its cache written from the half-precision rows."""
    import flint_mac_b200 as fa

    op = case["op"]
    ring = op == "window" or case.get("window", False)
    n = case.get("n", 1)
    if op in ("store", "load"):
        at = [case["at"] + 5 * i for i in range(n)]
        n_ctx = max(at) + case["rows"]
    else:
        at = [int(p) for p in s["pos"].tolist()]
        n_ctx = max(at) + max(RING, case.get("tokens", 1)) + 1
    pages = sum((p + (case["rows"] if op in ("store", "load") else 1) + 63) // 64 for p in at) if case.get("paged") else 0
    h = fa.Attn([ring], [case.get("rope", False)], n, n_ctx, kv_pages=pages, kv_format=fa.KV_INT4, first_tokens=case.get("first", 0))
    # the calls of one pass, with all but the rows settled, as a serving loop keeps them; results go to the program's buffers
    stream, kind = torch.cuda.current_stream().cuda_stream, {"float32": fa.F32, "bfloat16": fa.BF16, "float16": fa.F16}[case["type"]]
    seqs, rows = fa.i32_array(range(n)), case.get("rows", 1)
    if op == "prefill":
        rows = min(case["tokens"], RING) if ring else case["tokens"]
        back_at = [at[0] + case["tokens"] - rows]
    else:
        back_at = at
    dtype, back = (s["type"], kind) if op == "load" else (torch.float16, fa.F16)
    k, v = (torch.empty(n, KV_HEADS, rows, DIM, dtype=dtype, device="cuda") for _ in range(2))
    s["back"] = h.prepared_load_kv_dev(0, seqs, back_at, rows, k, v, back, stream)
    s["handle"], s["outputs"] = h, {"k": k, "v": v}
    if op == "load":
        h.store_kv_dev(0, seqs, at, rows, d["k"], d["v"], fa.F16)
        return
    if op == "store":
        s["call"] = h.prepared_store_kv_dev(0, seqs, at, rows, s["k"], s["v"], kind, stream)
        return
    s["outputs"]["out"] = out = torch.empty(len(s["qkv"]), HEADS * DIM, dtype=torch.bfloat16, device="cuda")
    if op == "prefill":
        s["call"] = lambda: h.prefill_dev(0, 0, case["tokens"], s["qkv"], kind, out, fa.BF16, stream)
        s["outputs"].update(k=k[0], v=v[0])
    else:
        decode = h.prepared_decode_dev(0, seqs, kind, out, fa.BF16, stream)
        s["call"] = lambda: decode(s["qkv"].data_ptr())
    h.set_layer(0, *(s[k].cpu().numpy() for k in ("q_norm", "k_norm", "sinks")))
    if op == "decode":
        by_length = {}
        for i, p in enumerate(at):
            by_length.setdefault(p, []).append(i)
        for p, who in by_length.items():
            if p:
                h.store_kv_dev(0, who, [0] * len(who), p, d["k"][who, :, :p].contiguous(), d["v"][who, :, :p].contiguous(), fa.F16)
    elif op == "window":
        start = (s["pos"] - RING).clamp(min=0)
        slot = ((start[:, None] + torch.arange(RING, device="cuda")) % RING)[:, None, :, None].expand(-1, KV_HEADS, -1, DIM)
        h.store_kv_dev(0, seqs, [0] * n, 64, d["k_first"], d["v_first"], fa.F16)
        h.store_kv_dev(0, seqs, start.tolist(), RING, d["k"].gather(2, slot), d["v"].gather(2, slot), fa.F16)
    elif at[0]:
        rows = d["k"].shape[2]
        if ring:
            h.store_kv_dev(0, [0], [0], 64, d["k_first"], d["v_first"], fa.F16)
        h.store_kv_dev(0, [0], [at[0] - rows], rows, d["k"], d["v"], fa.F16)
    for i, p in enumerate(at):
        h.set_pos(i, p)
    h.check()


def _ours(s, case):
    if case["op"] != "load":
        s["call"]()
    s["back"]()
    return s["outputs"]


def run(state):
    """One pass.  What a call wrote into the cache comes back as the values that it stands for."""
    case = state["case"]
    if own:
        return _ours(state, case)
    if case["op"] == "store":
        return {x: _values(_quantise(state[x].to(torch.float16))).to(torch.float16) for x in "kv"}
    if case["op"] == "load":
        return {x: _values(state[x]).to(state["type"]) for x in "kv"}
    return _plain_prefill(state, case) if case["op"] == "prefill" else _plain_decode(state, case)


# ---------------------------------------------------------------------------------------------- in 64 bits
def _kept64(x):
    """The values that a cache keeps of half-precision rows, in 64 bits."""
    x = x.double().reshape(*x.shape[:-1], DIM // GROUP, GROUP)
    lo = x.min(-1, keepdim=True).values
    step = ((x.max(-1, keepdim=True).values - lo) / 15.0).to(torch.float16).double()
    level = torch.nan_to_num((x - lo) / step, nan=0.0).round().clamp(max=15.0)
    return (lo + level * step).flatten(-2)


def _turned64(x, weight, at, rope):
    x = x * weight.double() / ((x ** 2).mean(-1, keepdim=True) + 1e-6).sqrt()
    if rope:
        freq = torch.tensor([math.pow(10000.0, -i / 64) for i in range(64)], dtype=torch.float64, device="cuda").float()
        z = torch.complex(x[..., :64], x[..., 64:]) * torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), (at.float()[:, None] * freq).double())[:, None]
        x = torch.cat((z.real, z.imag), -1)
    return x


def _softmax64(q, k, v, hidden, sinks):
    """q [heads][rows][128], k and v [heads][keys][128] -> [heads][rows][128]."""
    s = torch.einsum("hrd,hkd->hrk", q, k) / DIM ** 0.5
    s[hidden.expand_as(s)] = -math.inf
    s = torch.cat((s, sinks.double()[:, None, None].expand(-1, s.shape[1], 1)), 2).softmax(2)
    return torch.einsum("hrk,hkd->hrd", s[..., :-1], v)


def exact(case, seed):
    op, d = case["op"], _inputs(case, seed)
    if op in ("store", "load"):
        kind = torch.float16 if op == "load" else TYPES[case["type"]]
        return {x: _kept64(d[x].to(kind).to(torch.float16)) for x in "kv"}
    decode = op != "prefill"
    window, first, rope = op == "window" or case.get("window", False), case.get("first", 0), case.get("rope", False)
    x = d["qkv"].double().view(-1, HEADS + 2 * KV_HEADS, DIM)
    at = torch.tensor(_positions(case), device="cuda") if decode else torch.arange(case["past"], case["past"] + case["tokens"], device="cuda")
    q = _turned64(x[:, :HEADS], d["q_norm"], at, rope)
    k_new = _turned64(x[:, HEADS:HEADS + KV_HEADS], d["k_norm"], at, rope).to(torch.float16).double()
    v_new = x[:, HEADS + KV_HEADS:].to(torch.float16).double()
    group = HEADS // KV_HEADS
    wide = lambda t: t.repeat_interleave(group, 0)  # noqa: E731  a KV head serves its group of query heads
    outs = []
    for i in range(len(at) if decode else 1):
        me = slice(i, i + 1) if decode else slice(None)
        mine, start = at[me], int(at[i])
        if op == "window":  # the rows of the last positions, in order, out of the ring
            old = torch.arange(max(0, start - (WINDOW - 1)), start, device="cuda")
            k_old, v_old = (d[c][i, :, old % RING] for c in "kv")
        else:
            old = torch.arange(max(0, start - (WINDOW - 1)) if window else 0, start, device="cuda")
            k_old, v_old = (d[c][i, :, :len(old)] for c in "kv")
        ends = torch.arange(min(first, start - len(old)) if window else 0, device="cuda")
        k_end, v_end = (d[c + "_first"][i, :, :len(ends)] for c in "kv")
        key_at = torch.cat((ends, old, mine))
        k = torch.cat((_kept64(k_end), _kept64(k_old), k_new[me].transpose(0, 1)), 1)
        v = torch.cat((_kept64(v_end), _kept64(v_old), v_new[me].transpose(0, 1)), 1)
        hidden = key_at > mine[:, None]
        if window:
            hidden = hidden | ((key_at <= mine[:, None] - WINDOW) & (key_at >= first))
        outs.append(_softmax64(q[me].transpose(0, 1), wide(k), wide(v), hidden, d["sinks"]).transpose(0, 1))
    return {"out": torch.cat(outs).reshape(len(at), HEADS * DIM), "k": None, "v": None}
