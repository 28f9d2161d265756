"""Cases for the quantised serving operators: matrix products with 4-bit weights and group scales
(`quant.int4_linear`, `quant.int4_swiglu`), and the exchange with a store whose value rows are held in
8 or 4 bits (`LemaCache(quant=...)`). Each case runs in a plain form (elementary torch operations in
32 bits, or 64 next to a rounding border) or, with `own`, through the framework's entry points.

Sizes are those of the 834M-shaped and 309M-shaped models of the benchmark (dim 1536 and 1024, 64 heads
of 24 values, MLP width 4096 and 2816, vocabulary 50304), and odd ones."""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
STEPS = {"int8": 127.0, "int4": 7.0}   # largest code of the integer formats
ROW_GROUP = 32                         # values that share a scale in an int4 row


def _linear(name, m, n, k, group, dtype, residual):
    return {"name": name, "op": "linear", "m": m, "n": n, "k": k, "group": group, "dtype": dtype, "residual": residual}


def _swiglu(name, m, n, k, group, dtype):
    return {"name": name, "op": "swiglu", "m": m, "n": n, "k": k, "group": group, "dtype": dtype}


def _exchange(name, batch, heads, past, t, d_v, fmt, dtype):
    return {"name": name, "op": "exchange", "batch": batch, "heads": heads, "past": past, "t": t, "d_v": d_v, "fmt": fmt, "dtype": dtype}


def listed():
    return [
        # one token of one sequence: the output projection with the residual added
        _linear("o_proj token", 1, 1536, 1536, 128, "bf16", True),
        # the vocabulary head of eight sequences' newest tokens
        _linear("head batch 8", 8, 50304, 1536, 64, "bf16", False),
        # a batched decode step: the MLP's down projection for 256 sequences
        _linear("down batch 256", 256, 1536, 4096, 128, "bf16", True),
        # sizes that fill no tile: features, inputs, rows and the last group are all ragged
        _linear("odd fp16", 37, 1000, 1100, 32, "fp16", False),
        # a small model kept in fp32
        _linear("down fp32", 3, 1024, 2816, 64, "fp32", True),
        # a prompt of 16384 tokens through the down projection
        _linear("down prompt", 16384, 1536, 4096, 128, "bf16", True),
        # the gate and up projections with the activation: one token, a batch, a prompt
        _swiglu("mlp token", 1, 4096, 1536, 128, "bf16"),
        _swiglu("mlp batch 64", 64, 2816, 1024, 64, "fp16"),
        _swiglu("mlp prompt", 8192, 4096, 1536, 128, "bf16"),
        # two decode steps of one layer, the second reading back what the first wrote
        _exchange("step batch 1", 1, 64, 3000, 1, 24, "int8", "bf16"),
        _exchange("step batch 256", 256, 64, 512, 1, 24, "int4", "bf16"),
        # a prompt's chunk of one layer against the store
        _exchange("chunk", 16, 64, 1024, 1024, 24, "fp8", "bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["linear", "linear", "swiglu", "exchange", "exchange"])
    if op == "exchange":
        t = 1 if rng.random() < 0.5 else _log(rng, 2, 1024)
        d_v = rng.choice([8, 16, 24, 32, 48, 64, 96, 128, 40, 20, 33, 7])
        dtype = rng.choice(["bf16", "fp16", "fp32"])
        past = _log(rng, 16, 3000)
        most = (1 << 20) * 24 // max(24, d_v)
        batch, heads = _log(rng, 1, 256), rng.choice([1, 7, 16, 24, 64])
        rows = past + t if t > 1 else past // 4 + 1
        batch = max(1, min(batch, most // (heads * rows) or 1))
        return {"op": op, "batch": batch, "heads": heads, "past": past, "t": t, "d_v": d_v, "fmt": rng.choice(["int8", "fp8", "int4"]), "dtype": dtype}
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    m = _log(rng, 1, 16384 if dtype != "fp32" else 64)
    k = _log(rng, 64, 4096)
    n = _log(rng, 64, 50304 if op == "linear" else 4096)
    if rng.random() < 0.6:  # model widths are mostly whole tiles; the others stay odd
        n, k = -(-n // 64) * 64, -(-k // 64) * 64
    cols = n if op == "linear" else 2 * n
    m = max(1, min(m, 16384 * 1536 * 4096 // (cols * k)))
    case = {"op": op, "m": m, "n": n, "k": k, "group": rng.choice([32, 64, 128]), "dtype": dtype}
    if op == "linear":
        case["residual"] = rng.random() < 0.5
    return case


# ------------------------------------------------------------------ inputs
def _weight(g, n, k, group, dtype):
    """Codes and scales as a checkpoint holds them: int8 [n, k] in -8 .. 7, one scale per `group` inputs."""
    codes = (torch.randn(n, k, generator=g, device="cuda") * 2.5).round().clamp(-8, 7).to(torch.int8)
    scales = (0.5 + torch.rand(n, -(-k // group), generator=g, device="cuda")) / (2.5 * math.sqrt(k))
    return codes, scales.to(torch.float16 if dtype == "fp16" else torch.bfloat16)


def _codes(g, shape, low):
    """Random 32-bit codes whose two lowest bits are `low` (the pools below share no code)."""
    r = torch.randint(-(1 << 31), 1 << 31, shape, generator=g, device="cuda")
    return ((r & ~3) | low).to(torch.int32)


def _pick(g, pool, count):
    at = torch.randint(0, pool.shape[1], (pool.shape[0], count), generator=g, device="cuda")
    return pool.gather(1, at)


def _mix(g, a, b, share):
    return torch.where(torch.rand(a.shape, generator=g, device="cuda") < share, a, b)


def _values(g, p, t, d_v, dtype):
    """Value rows: each row has its own size, as projections of different tokens do."""
    v = torch.randn(p, t, d_v, generator=g, device="cuda") * torch.exp(torch.randn(p, t, 1, generator=g, device="cuda"))
    return v.to(TYPES[dtype])


def _streams(case, seed):
    """Keys of the past and new queries, keys and values, [partitions, positions]. A query asks for a key of the
    past that is not written anew, for an earlier key of this call, or for one that nobody wrote."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    p, s, t, d = case["batch"] * case["heads"], case["past"], case["t"], case["d_v"]
    read, written, late = (_codes(g, (p, max(1, s // 3)), low) for low in (0, 1, 3))
    past = _mix(g, _pick(g, read, s), _pick(g, written, s), 0.6)
    i = {"past": past, "past_v": _values(g, p, s, d, case["dtype"])}
    old = _mix(g, _pick(g, read, t), _codes(g, (p, t), 2), 0.75)
    i["k"] = [_mix(g, _pick(g, written, t), _codes(g, (p, t), 1), 0.5)]
    if t == 1:
        i["k"].append(_mix(g, _pick(g, late, 1), _codes(g, (p, 1), 3), 0.5))
        i["q"] = [old, _mix(g, i["k"][0], _pick(g, read, 1), 0.5)]
    else:
        before = (torch.rand(p, t, generator=g, device="cuda") * torch.arange(t, device="cuda")).long()
        inside = torch.rand(p, t, generator=g, device="cuda") < 0.3
        inside[:, 0] = False
        i["q"] = [torch.where(inside, i["k"][0].gather(1, before), old)]
    i["v"] = [_values(g, p, t, d, case["dtype"]) for _ in i["k"]]
    return i


def prepare(case, seed):
    if case["op"] == "exchange":
        s = {"case": case, **_streams(case, seed)}
        b, h, t, d = case["batch"], case["heads"], case["t"], case["d_v"]
        # what a layer hands to the cache: codes [B, H, T], values projected as [B, T, H, d_v] and seen as [B, H, T, d_v]
        s["new"] = [(q.view(b, h, t), k.view(b, h, t), v.view(b, h, t, d).transpose(1, 2).contiguous().transpose(1, 2))
                    for q, k, v in zip(s["q"], s["k"], s["v"])]
        if own:
            from latest_exact_match_attention_b200.cache import LemaCache
            from latest_exact_match_attention_b200.model import ModelConfig
            cfg = ModelConfig(vocab_size=128, depth=1, dim=h * d, num_heads=h, d_qk=32, d_v=d)
            past = case["past"]
            s["cache"] = LemaCache(cfg, dtype=TYPES[case["dtype"]], batch=b, max_cache_len=past + 2 * t, quant=case["fmt"])
            keys = s["past"].view(b, h, past)
            s["cache"].layer(0).exchange(keys, keys, s["past_v"].view(b, h, past, d))
        return s
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = TYPES[case["dtype"]]
    s = {"case": case, "x": torch.randn(case["m"], case["k"], generator=g, device="cuda").to(dt), "r": None}
    s["w"] = [_weight(g, case["n"], case["k"], case["group"], case["dtype"]) for _ in range(1 if case["op"] == "linear" else 2)]
    if case.get("residual"):
        s["r"] = torch.randn(case["m"], case["n"], generator=g, device="cuda").to(dt)
    if own:
        from latest_exact_match_attention_b200.quant import Int4Weight
        flat = [t for pair in s["w"] for t in pair]
        s["packed"] = (Int4Weight.pack if case["op"] == "linear" else Int4Weight.pack_gate_up)(*flat, group=case["group"])
    return s


# ------------------------------------------------------------------ one pass
def _held(v, fmt):
    """The values that the held codes of rows `v` [..., d] stand for, in 32 bits."""
    v = v.float()
    if fmt == "fp8":
        # the smallest power of two that brings the row within e4m3's +-448: the quotients are then exact
        m, e = torch.frexp(v.abs().amax(-1, keepdim=True).double() / 448)
        s = ((torch.where(m == 0.5, e - 1, e).clamp(min=-126) + 127) << 23).view(torch.float32)
        return (v / s).to(torch.float8_e4m3fn).float() * s
    d, top = v.shape[-1], STEPS[fmt]
    wide = ROW_GROUP if fmt == "int4" else d
    pad = -d % wide
    rows = torch.nn.functional.pad(v, (0, pad)).unflatten(-1, (-1, wide))
    s = (rows.abs().amax(-1, keepdim=True).double() / top).float()
    codes = torch.where(s > 0, rows.double() / s.double(), 0.0).round().clamp(-top, top)
    return (codes.float() * s).flatten(-2)[..., :d]


def _exchange_plain(s):
    case, out = s["case"], []
    b, h, t, d = case["batch"], case["heads"], case["t"], case["d_v"]
    keys, vals = s["past"], s["past_v"]
    if t == 1:
        q, k, v = (torch.cat(x, 1) for x in (s["q"], s["k"], s["v"]))
        at = torch.arange(1, keys.shape[1] + 1, device=keys.device)
        first = torch.where(keys == q[:, :1], at, 0).amax(1) - 1
        second = torch.where(keys == q[:, 1:], at, 0).amax(1) - 1
        got = torch.stack([vals.gather(1, x.clamp(min=0).view(-1, 1, 1).expand(-1, 1, d))[:, 0] for x in (first, second)], 1)
        back = (q[:, 1] == k[:, 0]).view(-1, 1)
        got = torch.stack([got[:, 0], torch.where(back, v[:, 0], got[:, 1])], 1)
        hit = torch.stack([first >= 0, (second >= 0) | back[:, 0]], 1)
        got = (_held(got, case["fmt"]) * hit[..., None]).to(vals.dtype)
        out = [got[:, 0].reshape(b, h, 1, d), got[:, 1].reshape(b, h, 1, d)]
        new = k
    else:
        q, new = s["q"][0], s["k"][0]
        n = keys.shape[1]
        allk = torch.cat([keys, new], 1)
        part = torch.arange(allk.shape[0], device=q.device).view(-1, 1) << 32
        keyed = (((part | (allk.long() & 0xFFFFFFFF)) << 16) | torch.arange(n + t, device=q.device)).flatten().sort().values
        want = ((part | (q.long() & 0xFFFFFFFF)) << 16) | torch.arange(n, n + t, device=q.device)
        at = torch.searchsorted(keyed, want) - 1
        found = keyed[at.clamp(min=0)]
        hit = (at >= 0) & ((found >> 16) == (want >> 16))
        rows = torch.cat([vals, s["v"][0]], 1).gather(1, torch.where(hit, found & 0xFFFF, 0)[..., None].expand(-1, -1, d))
        out = [(_held(rows, case["fmt"]) * hit[..., None]).to(vals.dtype).view(b, h, t, d)]
    # entries of each partition after the call: its distinct keys
    every = torch.cat([keys, new], 1).sort(1).values
    out.append((1 + (every[:, 1:] != every[:, :-1]).sum(1)).long())
    return out


def _dense(w, group):
    codes, scales = w
    return codes.float() * scales.float().repeat_interleave(group, 1)[:, :codes.shape[1]]


def run(state):
    case = state["case"]
    if case["op"] == "exchange":
        if not own:
            return _exchange_plain(state)
        cache = state["cache"]
        layer = cache.layer(0)
        return [layer.exchange(q, k, v, check=False) for q, k, v in state["new"]] + [cache.store.counts]
    if own:
        from latest_exact_match_attention_b200 import quant
        if case["op"] == "linear":
            return quant.int4_linear(state["x"], state["packed"], residual=state["r"])
        return quant.int4_swiglu(state["x"], state["packed"])
    x = state["x"].float()
    if case["op"] == "linear":
        y = x @ _dense(state["w"][0], case["group"]).t()
        return (y if state["r"] is None else y + state["r"].float()).to(state["x"].dtype)
    gate, up = (x @ _dense(w, case["group"]).t() for w in state["w"])
    return (gate / (1 + torch.exp(-gate)) * up).to(state["x"].dtype)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "exchange":
        calls = 2 if case["t"] == 1 else 1
        n, d = calls * case["batch"] * case["heads"] * case["t"], case["d_v"]
        held = d + 4 if case["fmt"] != "int4" else -(-d // 2) + 4 * -(-d // ROW_GROUP)
        # two codes; the value row in and the retrieved row out; a held row read and one written; the slot's key beside each
        return {"bytes": n * (8 + 2 * d * size + 2 * held + 2 * 16), "flops": n * 4 * d}
    m, n, k = case["m"], case["n"], case["k"]
    cols = n if case["op"] == "linear" else 2 * n
    outs = 2 if case.get("residual") else 1
    return {"bytes": cols * k / 2 + cols * -(-k // case["group"]) * 2 + size * (m * k + outs * m * n), "flops": 2 * m * cols * k}


# ------------------------------------------------------------------ the definition in 64 bits
def _power(p):
    """2 ** p of whole numbers, from the exponent's bits (a pow need not be exact)."""
    return ((p.long() + 1023) << 52).view(torch.float64)


def _code_values(v, fmt):
    """One scale group `v` [rows, values] in 64 bits: the numbers that its codes stand for. The scale is held in 32 bits."""
    peak = v.abs().max(1).values
    if fmt == "fp8":
        p = torch.ceil(torch.log2((peak / 448).clamp(min=2.0 ** -126)))
        p = torch.where(peak <= 448 * _power(p - 1), p - 1, p)
        p = torch.where(peak > 448 * _power(p), p + 1, p).clamp(min=-126)
        s = _power(p)[:, None]
        y = v / s
        # e4m3: four significant bits down to 2^-6, steps of 2^-9 below; ties to even
        step = _power(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
        return torch.round(y / step) * step * s
    top = STEPS[fmt]
    s = (peak / top).float().double()[:, None]
    return torch.round(v / s.clamp(min=2.0 ** -149)).clamp(-top, top) * s


def exact(case, seed):
    if case["op"] == "exchange":
        i = _streams(case, seed)
        b, h, t, d = case["batch"], case["heads"], case["t"], case["d_v"]
        keys, vals, outs = i["past"].long(), i["past_v"].double(), []
        for q, k, v in zip(i["q"], i["k"], i["v"]):
            got = torch.zeros(b * h, t, d, dtype=torch.float64, device="cuda")
            span = max(1, (1 << 27) // (b * h * (keys.shape[1] + t)))
            allk, allv = torch.cat([keys, k.long()], 1), torch.cat([vals, v.double()], 1)
            for t0 in range(0, t, span):
                n = min(span, t - t0)
                same = allk[:, None, :] == q[:, t0:t0 + n, None].long()
                same &= torch.arange(allk.shape[1], device="cuda") < keys.shape[1] + t0 + torch.arange(n, device="cuda")[:, None]
                last = allk.shape[1] - 1 - same.flip(2).int().argmax(2)
                rows = allv.gather(1, last[..., None].expand(-1, -1, d))
                got[:, t0:t0 + n] = rows * same.any(2)[..., None]
            wide = ROW_GROUP if case["fmt"] == "int4" else d
            flat = got.view(-1, d)
            held = torch.cat([_code_values(flat[:, c:c + wide], case["fmt"]) for c in range(0, d, wide)], 1)
            outs.append(held.view(b, h, t, d))
            keys, vals = allk, allv
        return outs + [None]
    i = prepare(case, seed)
    x, group = i["x"].double(), case["group"]
    sums = []
    for codes, scales in i["w"]:
        y = torch.zeros(case["m"], case["n"], dtype=torch.float64, device="cuda")
        for c in range(scales.shape[1]):
            cols = slice(c * group, (c + 1) * group)
            y += (x[:, cols] @ codes[:, cols].double().t()) * scales[:, c].double()
        sums.append(y)
    if case["op"] == "swiglu":
        return sums[0] * torch.sigmoid(sums[0]) * sums[1]
    return sums[0] if i["r"] is None else sums[0] + i["r"].double()
