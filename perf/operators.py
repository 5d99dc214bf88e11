"""Workloads of the cache-memory operators: a KV cache held in 4 bits (append, read-back, decode attention) and eviction
by accumulated attention weight (decode attention and prompt queries that accumulate the weights, selection and in-place
compaction of the ranges).  ``run`` computes a case either in plain torch (``own`` false) or through ``glake_b200.ops``.

The 4-bit row of one token: heads come in units of U (8, 4, 2 or 1: the largest that divides the kv heads); a unit is
U x 64 bytes of nibbles, then U x 4 bytes of group scales, zero-padded to a multiple of 16 bytes.  Inside a head's 64
bytes dim 32 G + 4 r + j lies in byte 8 r + 2 G + j // 2 (low nibble for even j), stored as value + 8 with the value in
-7 .. 7; group G (32 dims) has one e4m3 scale.  element = value * group scale * scale[kv head].
"""
import math

import torch

own = False

D = 128
_KINDS = ("write", "decode4", "scored", "prompt", "evict")


# ------------------------------------------------------------------ cases
def listed():
    return [
        # short prompts of a chat turn into a 2-kv-head rank's cache, one of them extending a cached prefix
        {"name": "write_small", "op": "write", "batch": 3, "h": 8, "kvh": 2, "lo": 1, "hi": 130, "prefix": 37},
        # eight 4k prompts, 8 kv heads: the prompt batch of the repository's prefill benchmark
        {"name": "write_8x4k", "op": "write", "batch": 8, "h": 32, "kvh": 8, "lo": 4096, "hi": 4096, "prefix": 0},
        # one user, one short context: latency
        {"name": "decode4_one", "op": "decode4", "batch": 1, "h": 32, "kvh": 8, "lo": 700, "hi": 700, "empty": 0},
        # the 7B shape's layer (32/32 heads) at batch 64, contexts 1k-4k
        {"name": "decode4_mha", "op": "decode4", "batch": 64, "h": 32, "kvh": 32, "lo": 1024, "hi": 4096, "empty": 0},
        # long contexts, grouped queries: 32/8 heads, 16k-32k
        {"name": "decode4_long", "op": "decode4", "batch": 32, "h": 32, "kvh": 8, "lo": 16384, "hi": 32768, "empty": 0},
        # bf16 cache, the small operator-level decode case (batch 8, 32/32 heads), weights accumulated
        {"name": "scored_bf16_mha", "op": "scored", "kv": "bf16", "batch": 8, "h": 32, "kvh": 32, "lo": 512, "hi": 2048, "empty": 0},
        # fp8 cache, batch 64, 32/8 heads, 2k-8k
        {"name": "scored_fp8", "op": "scored", "kv": "fp8", "batch": 64, "h": 32, "kvh": 8, "lo": 2048, "hi": 8192, "empty": 1},
        # one rank's share of a sharded 64/8-head model: 8 q heads on one kv head, long contexts
        {"name": "scored_bf16_share", "op": "scored", "kv": "bf16", "batch": 32, "h": 8, "kvh": 1, "lo": 4096, "hi": 16384, "empty": 0},
        # observation window of short prompts: odd lengths, fewer queries than the window
        {"name": "prompt_small", "op": "prompt", "batch": 4, "h": 8, "kvh": 2, "lo": 5, "hi": 1001, "window": 16},
        # four 16k prompts judged by their last 32 queries
        {"name": "prompt_16k", "op": "prompt", "batch": 4, "h": 32, "kvh": 8, "lo": 16384, "hi": 16384, "window": 32},
        # a single conversation cut from just over a thousand rows to 512
        {"name": "evict_one", "op": "evict", "kv": "bf16", "batch": 1, "h": 32, "kvh": 8, "lo": 1027, "hi": 1027, "budget": 512, "sink": 4, "recent": 64},
        # long contexts cut to 8k rows per head
        {"name": "evict_long", "op": "evict", "kv": "bf16", "batch": 16, "h": 32, "kvh": 8, "lo": 7000, "hi": 32768, "budget": 8192, "sink": 4, "recent": 512},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(_KINDS)
    h, kvh = rng.choice([(32, 8), (32, 32), (8, 1), (16, 2), (8, 8), (64, 8), (16, 16), (8, 2), (16, 1), (32, 4), (6, 3), (12, 12)])
    batch = _log(rng, 1, 64)
    most = {"write": 262144, "decode4": 4000000, "scored": 2500000, "prompt": 400000, "evict": 1500000}[op] // kvh
    hi = max(2, min(_log(rng, 2, 32768), most // batch))
    lo = max(1, int(hi * rng.uniform(0.1, 1.0)))
    case = {"op": op, "batch": batch, "h": h, "kvh": kvh, "lo": lo, "hi": hi}
    if op == "write":
        case["prefix"] = rng.choice([0, 0, 1, _log(rng, 2, 500)])
    elif op in ("decode4", "scored"):
        case["empty"] = rng.choice([0, 0, 1])
        if op == "scored":
            case["kv"] = rng.choice(["bf16", "fp8", "int4"])
    elif op == "prompt":
        case["window"] = _log(rng, 1, 64)
    else:
        case["kv"] = rng.choice(["bf16", "fp8"])
        case["budget"] = max(1, int(hi * rng.uniform(0.05, 0.9)))
        case["sink"] = min(rng.choice([0, 1, 4, 16]), case["budget"])
        case["recent"] = int((case["budget"] - case["sink"]) * rng.uniform(0, 1))
    return case


def _lens(case):
    """Context (or prompt) lengths of a case: spread over lo .. hi, ``empty`` sequences without a row at the end."""
    b, lo, hi = case["batch"], case["lo"], case["hi"]
    lens = [lo + int(round((hi - lo) * ((0.618034 * (i + 1)) % 1.0))) for i in range(b)]
    lens[0] = hi
    for i in range(1, 1 + min(case.get("empty", 0), b - 1)):
        lens[-i] = 0
    return lens


# ------------------------------------------------------------------ the 4-bit format
def _unit(kvh):
    return next(u for u in (8, 4, 2, 1) if kvh % u == 0)


def _unit_bytes(kvh):
    u = _unit(kvh)
    return 64 * u + (4 * u + 15) // 16 * 16


def _row_bytes(kvh):
    return kvh // _unit(kvh) * _unit_bytes(kvh)


def _pack4(x, scale):
    """Rows [n, kvh, 128] (any float type) -> uint8 [n, row bytes]; scale float32 [kvh]."""
    n, kvh, _ = x.shape
    u = _unit(kvh)
    g = torch.nan_to_num(x.float(), nan=0.0, posinf=math.inf, neginf=-math.inf).view(n, kvh, 4, 32)
    s8 = (g.abs().amax(-1) / (7.0 * scale)[:, None]).clamp(max=448.0).to(torch.float8_e4m3fn)
    step = (s8.float() * scale[:, None])[..., None]
    q = torch.where(step > 0, torch.round(g / step), torch.zeros_like(g)).clamp(-7, 7).to(torch.int16) + 8
    q = q.view(n, kvh, 4, 8, 2, 2)                                   # G, r, j // 2, j % 2
    byte = (q[..., 0] | (q[..., 1] << 4)).to(torch.uint8)            # G, r, j // 2
    nib = byte.permute(0, 1, 3, 2, 4).reshape(n, kvh // u, u * 64)   # r, G, j // 2
    sc = s8.view(torch.uint8).view(n, kvh // u, u * 4)
    pad = torch.zeros(n, kvh // u, _unit_bytes(kvh) - u * 68, dtype=torch.uint8, device=x.device)
    return torch.cat([nib, sc, pad], -1).view(n, _row_bytes(kvh))


def _unpack4(rows, kvh, scale):
    """uint8 [..., row bytes] -> float32 [..., kvh, 128]."""
    lead, u = rows.shape[:-1], _unit(kvh)
    rows = rows.reshape(-1, kvh // u, _unit_bytes(kvh))
    n = rows.shape[0]
    byte = rows[..., :u * 64].reshape(n, kvh, 8, 4, 2)               # r, G, j // 2
    q = torch.stack([byte & 15, byte >> 4], -1).permute(0, 1, 3, 2, 4, 5).reshape(n, kvh, 4, 32)
    s8 = rows[..., u * 64:u * 68].reshape(n, kvh, 4).view(torch.float8_e4m3fn).float()
    x = (q.float() - 8.0) * s8[..., None] * scale[:, None, None]
    return x.view(*lead, kvh, D)


# ------------------------------------------------------------------ inputs
def _values(n, kvh, gen, spread):
    """Rows as a model writes them: unit normals, a few loud channels per head."""
    x = torch.randn(n, kvh, D, generator=gen, device="cuda")
    return (x * spread).bfloat16()


def _spread(kvh, gen):
    loud = torch.rand(kvh, D, generator=gen, device="cuda") < 0.02
    return torch.where(loud, 4.0, 1.0)


def _amax_scale(spread, gen):
    """What the scale op makes of a first prompt: amax / 448 per kv head, of about 5 sigma."""
    return (spread.amax(-1) * (4.6 + 0.8 * torch.rand(spread.shape[0], generator=gen, device="cuda")) / 448.0).float()


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed) * 7919 + 17)
    op, b, h, kvh = case["op"], case["batch"], case["h"], case["kvh"]
    kv = "int4" if op in ("write", "decode4") else case.get("kv", "bf16")
    lens = _lens(case)
    prefix = case.get("prefix", 0)
    ctx = [n + prefix for n in lens]
    cap = max(ctx) + 9
    n_slots = b + 2
    dev = "cuda"
    row = {"bf16": kvh * D * 2, "fp8": kvh * D, "int4": _row_bytes(kvh)}[kv]
    order = torch.randperm(n_slots, generator=gen, device=dev)[:b]
    k_spread, v_spread = _spread(kvh, gen), torch.ones(kvh, D, device=dev)
    s = {"case": dict(case), "kv": kv, "kvh": kvh, "h": h, "cap": cap, "scale": D ** -0.5, "max_len": max(ctx),
         "k": torch.zeros(n_slots, cap, row, dtype=torch.uint8, device=dev), "v": torch.zeros(n_slots, cap, row, dtype=torch.uint8, device=dev),
         "k_scale": _amax_scale(k_spread, gen), "v_scale": _amax_scale(v_spread, gen),
         "slots": order.to(torch.int64), "seq_lens": torch.tensor(ctx, dtype=torch.int32, device=dev)}
    for name in ("k", "v"):
        base = s[name].data_ptr()
        s[name + "_table"] = torch.tensor([base + i * cap * row for i in range(n_slots)], dtype=torch.int64, device=dev)
    rows_now = [prefix] * b if op == "write" else ctx
    for i, slot in enumerate(order.tolist()):
        for name, spread, scale in (("k", k_spread, s["k_scale"]), ("v", v_spread, s["v_scale"])):
            n = rows_now[i]
            if op == "prompt" and name == "v" or n == 0:
                continue
            x = _values(n, kvh, gen, spread)
            if kv == "int4":
                s[name][slot, :n] = _pack4(x, scale)
            elif kv == "fp8":
                s[name][slot, :n] = (x.float() / scale[:, None]).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8).view(n, row)
            else:
                s[name][slot, :n] = x.view(torch.uint8).view(n, row)
    if op == "write":
        starts = [sum(lens[:i]) for i in range(b)]
        s["key"], s["value"] = _values(sum(lens), kvh, gen, k_spread), _values(sum(lens), kvh, gen, v_spread)
        s["rows"] = torch.tensor(lens, dtype=torch.int32, device=dev)
        s["starts"] = torch.tensor(starts, dtype=torch.int32, device=dev)
        s["slot_m"] = torch.full((b,), prefix * row, dtype=torch.int64, device=dev)
        s["max_rows"] = max(max(lens), 2)
        s["out_start"] = torch.tensor([sum(ctx[:i]) for i in range(b)], dtype=torch.int32, device=dev)
        s["k_out"], s["v_out"] = (torch.empty(sum(ctx), kvh, D, dtype=torch.bfloat16, device=dev) for _ in range(2))
    if op in ("decode4", "scored"):
        s["q"] = (1.5 * torch.randn(b, h, D, generator=gen, device=dev)).bfloat16()
    if op == "prompt":
        q_lens = [max(1, n - n // 3) for n in lens]      # the rest is a prefix that was in the cache already
        s["q"] = (1.5 * torch.randn(sum(q_lens), h, D, generator=gen, device=dev)).bfloat16()
        s["q_lens"] = torch.tensor(q_lens, dtype=torch.int32, device=dev)
        s["q_start"] = torch.tensor([sum(q_lens[:i]) for i in range(b)], dtype=torch.int32, device=dev)
    if op in ("scored", "prompt"):
        s["scores"] = _weights(n_slots, kvh, cap, gen) / cap     # of the size of what one pass adds
    if op == "evict":
        s["scores"] = _weights(n_slots, kvh, cap, gen)
        s["scores_out"] = torch.zeros_like(s["scores"])
    return s


def _weights(n_slots, kvh, cap, gen):
    """Accumulated weights as decoding leaves them: heavy-tailed, many small ones equal."""
    x = torch.exp(2.0 * torch.randn(n_slots, kvh, cap, generator=gen, device="cuda") - 4.0)
    return torch.where(x < 0.01, torch.round(x * 512.0) / 512.0, x)


# ------------------------------------------------------------------ plain forms
def _cache(s, name, n):
    """Rows 0 .. n of every sequence's range as float32 [B, n, kvh, 128]."""
    rows = s[name][s["slots"], :n]
    if s["kv"] == "int4":
        return _unpack4(rows, s["kvh"], s[name + "_scale"])
    if s["kv"] == "fp8":
        return rows.view(torch.float8_e4m3fn).view(*rows.shape[:2], s["kvh"], D).float() * s[name + "_scale"][:, None]
    return rows.view(torch.bfloat16).view(*rows.shape[:2], s["kvh"], D).float()


def _rows_of(starts, lens, most):
    """[B, most] row numbers of packed rows and which of them exist."""
    t = torch.arange(most, device=lens.device)
    return starts[:, None].long() + t, t < lens[:, None]


def _plain_write(s):
    kvh, row = s["kvh"], s["k"].shape[-1]
    src, valid = _rows_of(s["starts"], s["rows"], s["max_rows"])
    at = s["slot_m"][:, None] // row + torch.arange(s["max_rows"], device="cuda")
    slot = s["slots"][:, None].expand_as(at)
    out_at, there = _rows_of(s["out_start"], s["seq_lens"], s["max_len"])
    got = []
    for_k, for_v = (s["key"], "k", s["k_out"]), (s["value"], "v", s["v_out"])
    for new, name, out in (for_k, for_v):
        s[name][slot[valid], at[valid]] = _pack4(new[src[valid]], s[name + "_scale"])
        out[out_at[there]] = _cache(s, name, s["max_len"])[there].bfloat16()
        got.append(out)
    return {"k": got[0], "v": got[1]}


def _plain_decode(s):
    n, kvh = s["max_len"], s["kvh"]
    b, h, _ = s["q"].shape
    q = s["q"].float().view(b, kvh, h // kvh, D)
    logits = torch.matmul(q, _cache(s, "k", n).permute(0, 2, 3, 1)) * s["scale"]
    logits.masked_fill_((torch.arange(n, device="cuda") >= s["seq_lens"][:, None])[:, None, None], -math.inf)
    lse = torch.logsumexp(logits, -1)
    p = torch.exp(logits - torch.where(lse > -math.inf, lse, torch.zeros_like(lse))[..., None])
    out = torch.matmul(p, _cache(s, "v", n).permute(0, 2, 1, 3)).reshape(b, h, D).bfloat16()
    if s["case"]["op"] == "scored":
        s["scores"][s["slots"], :, :n] += p.sum(2)
    return out, lse.reshape(b, h)


def _plain_prompt(s):
    n, kvh, h, b = s["max_len"], s["kvh"], s["h"], s["slots"].numel()
    w = s["case"]["window"]
    used = s["q_lens"].clamp(max=w)
    src, there = _rows_of(s["q_start"] + s["q_lens"] - used, used, w)
    q = s["q"][torch.where(there, src, 0)].float().view(b, w, kvh, h // kvh, D).permute(0, 2, 3, 1, 4).reshape(b, kvh, -1, D)
    logits = torch.matmul(q, _cache(s, "k", n).permute(0, 2, 3, 1)).view(b, kvh, h // kvh, w, n) * s["scale"]
    sees = (s["seq_lens"] - used)[:, None] + torch.arange(w, device="cuda")           # last key of a query
    mask = (torch.arange(n, device="cuda") <= sees[..., None]) & there[..., None]
    logits.masked_fill_(~mask[:, None, None], -math.inf)
    p = torch.where(mask[:, None, None], torch.exp(logits - torch.logsumexp(logits, -1, keepdim=True)), 0.0)
    s["scores"][s["slots"], :, :n] += p.sum((2, 3))
    return {"scores": s["scores"]}


def _plain_evict(s):
    c, n, kvh, b = s["case"], s["max_len"], s["kvh"], s["slots"].numel()
    budget, lens = c["budget"], s["seq_lens"][:, None, None].long()
    t = torch.arange(n, device="cuda").expand(b, kvh, n)
    x = s["scores"][s["slots"], :, :n]
    x = torch.where(torch.isnan(x), -math.inf, x)
    key = torch.where((t < c["sink"]) | (t >= lens - c["recent"]), math.inf, x)
    key = torch.where(t < lens, key, -math.inf)
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :budget]
    most = order.shape[-1]
    kept = torch.where(torch.arange(most, device="cuda") < lens, order, n).sort(-1).values
    whole = torch.arange(most, device="cuda").expand_as(kept)
    kept = torch.where(lens <= budget, torch.where(whole < lens, whole, n), kept)
    here = kept < n
    at = torch.where(here, kept, whole)
    keep_n = here.sum(-1, keepdim=True)
    new = torch.zeros(b, kvh, n, device="cuda")
    new[..., :most] = torch.where(here, torch.gather(s["scores"][s["slots"], :, :n], 2, at), 0.0)
    old = s["scores_out"][s["slots"], :, :n]
    s["scores_out"][s["slots"], :, :n] = torch.where((t < lens) | (t < keep_n), new, old)
    moved = []
    for name in ("k", "v"):
        cells = s[name].view(torch.int64).view(s[name].shape[0], s["cap"], kvh, -1)
        idx = at.permute(0, 2, 1)[..., None].expand(-1, -1, -1, cells.shape[-1])
        cells[s["slots"], :most] = torch.gather(cells[s["slots"]], 1, idx)
        moved.append(_typed(s, name, most))
    full = torch.full((b, kvh, budget), -1, dtype=torch.int32, device="cuda")
    full[..., :most] = torch.where(here, kept, -1).int()
    return {"kept": full, "scores": s["scores_out"], "k": moved[0], "v": moved[1]}


def _typed(s, name, n):
    rows = s[name][:, :n]
    return rows.view(torch.bfloat16 if s["kv"] == "bf16" else torch.float8_e4m3fn)


# ------------------------------------------------------------------ one pass
def run(s):
    op = s["case"]["op"]
    if own:
        return _own(s, op)
    if op == "write":
        return _plain_write(s)
    if op in ("decode4", "scored"):
        out, lse = _plain_decode(s)
        return {"out": out, "lse": lse} if op == "decode4" else {"out": out, "lse": lse, "scores": s["scores"]}
    return _plain_prompt(s) if op == "prompt" else _plain_evict(s)


def _own(s, op):
    from glake_b200 import ops
    kt, vt = s["k_table"].data_ptr(), s["v_table"].data_ptr()
    dt = {"bf16": "auto", "fp8": "fp8_e4m3", "int4": "int4"}[s["kv"]]
    quant = {"kv_cache_dtype": dt, "k_scale": s["k_scale"], "v_scale": s["v_scale"]} if dt != "auto" else {}
    if op == "write":
        ops.reshape_and_cache(s["key"], s["value"], s["k_table"], s["v_table"], s["slot_m"], s["slots"], s["rows"],
                              s["starts"], s["max_rows"], s["kvh"], D, **quant)
        ops.dequantize_ranges(s["k_out"], s["v_out"], kt, vt, s["kvh"], s["slots"], s["seq_lens"], s["out_start"],
                              s["max_len"], **quant)
        return {"k": s["k_out"], "v": s["v_out"]}
    if op in ("decode4", "scored"):
        b, h, _ = s["q"].shape
        scores = {"scores": s["scores"]} if op == "scored" else {}
        out, lse = ops.fwd_kvcache(s["q"].view(b, 1, h, D), kt, vt, s["max_len"], s["kvh"], b, s["slots"], None, None,
                                   s["seq_lens"], None, None, None, None, None, None, s["scale"], True, -1, -1, None,
                                   0, **quant, **scores)
        got = {"out": out.view(b, h, D), "lse": lse.view(b, h)}
        return got if op == "decode4" else {**got, **scores}
    if op == "prompt":
        ops.prompt_scores(s["scores"], s["q"], kt, s["kvh"], s["scale"], s["slots"], s["seq_lens"], s["q_lens"],
                          s["q_start"], s["max_len"], s["case"]["window"])
        return {"scores": s["scores"]}
    c = s["case"]
    kept = ops.evict_rows(s["scores"], kt, vt, s["kvh"], s["slots"], s["seq_lens"], s["max_len"], c["budget"],
                          c["sink"], c["recent"], kv_cache_dtype=dt, scores_out=s["scores_out"])
    n = min(c["budget"], s["max_len"])
    return {"kept": kept, "scores": s["scores_out"], "k": _typed(s, "k", n), "v": _typed(s, "v", n)}


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    op, b, h, kvh = case["op"], case["batch"], case["h"], case["kvh"]
    lens = _lens(case)
    total = sum(lens)
    kv = "int4" if op in ("write", "decode4") else case.get("kv", "bf16")
    row = {"bf16": kvh * D * 2, "fp8": kvh * D, "int4": _row_bytes(kvh)}[kv]
    if op == "write":
        ctx = total + b * case["prefix"]
        return {"bytes": 2 * (total * kvh * D * 2 + total * row + ctx * row + ctx * kvh * D * 2), "flops": 4 * (total + ctx) * kvh * D}
    if op in ("decode4", "scored"):
        acc = 8 * kvh * total if op == "scored" else 0
        return {"bytes": 2 * total * row + 4 * b * h * D + 4 * b * h + acc, "flops": 4 * h * D * total}
    if op == "prompt":
        w = [min(case["window"], max(1, n - n // 3)) for n in lens]
        return {"bytes": total * row + sum(w) * h * D * 2 + 8 * kvh * total, "flops": 2 * h * D * sum(x * n for x, n in zip(w, lens))}
    cut = [n for n in lens if n > case["budget"]]
    return {"bytes": len(cut) * case["budget"] * row * 4 + kvh * (8 * total + 4 * len(cut) * case["budget"]), "flops": 8 * kvh * total}


# ------------------------------------------------------------------ 64 bits, from the definitions
def _row64(byte_row, kvh, scale):
    """One sequence's 4-bit rows uint8 [n, row bytes] -> float64 [n, kvh, 128], dim by dim from the format's definition."""
    u, ub = _unit(kvh), _unit_bytes(kvh)
    d = torch.arange(D, device=byte_row.device)
    grp, r, j = d // 32, d % 32 // 4, d % 4
    head = torch.arange(kvh, device=byte_row.device)[:, None]
    base = head // u * ub
    b = byte_row[:, (base + 64 * (head % u) + 8 * r + 2 * grp + j // 2).reshape(-1)].view(-1, kvh, D).to(torch.int64)
    nib = torch.where(j % 2 == 0, b % 16, b // 16) - 8
    e = byte_row[:, (base + 64 * u + 4 * (head % u) + grp).reshape(-1)].view(-1, kvh, D).to(torch.int64)
    exp, man = (e // 8) % 16, (e % 8).double()
    s8 = torch.where(exp > 0, torch.ldexp(1.0 + man / 8.0, exp - 7), torch.ldexp(man / 8.0, torch.full_like(exp, -6)))
    return nib.double() * s8 * scale.double()[:, None]


def _cache64(s, name, i):
    n, kvh = int(s["seq_lens"][i]), s["kvh"]
    rows = s[name][int(s["slots"][i]), :n]
    if s["kv"] == "int4":
        return _row64(rows, kvh, s[name + "_scale"])
    if s["kv"] == "fp8":
        return rows.contiguous().view(torch.float8_e4m3fn).view(n, kvh, D).double() * s[name + "_scale"].double()[:, None]
    return rows.contiguous().view(torch.bfloat16).view(n, kvh, D).double()


def _evict64(s):
    """Row by row of the definition: rank every row that may go by (weight, lower row first), keep what the budget holds."""
    c, kvh = s["case"], s["kvh"]
    most = min(c["budget"], s["max_len"])
    scores, moved = s["scores_out"].double(), {}
    picks = {}
    for i, slot in enumerate(s["slots"].tolist()):
        n = int(s["seq_lens"][i])
        if n <= c["budget"]:
            continue
        x = s["scores"][slot, :, :n].double()
        free = torch.arange(c["sink"], n - c["recent"], device="cuda")
        rank = torch.sort(-x[:, free], dim=-1, stable=True).indices[:, :c["budget"] - c["sink"] - c["recent"]]
        fixed = torch.cat([torch.arange(c["sink"], device="cuda"), torch.arange(n - c["recent"], n, device="cuda")])
        picks[slot] = torch.cat([free[rank], fixed.expand(kvh, -1)], -1).sort(-1).values
    for i, slot in enumerate(s["slots"].tolist()):
        n = int(s["seq_lens"][i])
        scores[slot, :, :n] = 0.0
        keep = picks.get(slot, torch.arange(n, device="cuda").expand(kvh, -1))
        scores[slot, :, :keep.shape[-1]] = s["scores"][slot].double().gather(1, keep)
    for name in ("k", "v"):
        rows = _typed(s, name, s["cap"])
        x = rows.view(*rows.shape[:2], kvh, D).double()
        for slot, keep in picks.items():
            x[slot, :c["budget"]] = x[slot].gather(0, keep.T[..., None].expand(-1, -1, D))
        moved[name] = x[:, :most].reshape(x.shape[0], most, -1)
    return {"kept": None, "scores": scores, "k": moved["k"], "v": moved["v"]}


def exact(case, seed):
    s = prepare(case, seed)
    op, kvh, h, b = case["op"], s["kvh"], s["h"], case["batch"]
    g = h // kvh
    if op == "evict":
        return _evict64(s)
    if op == "write":
        got = {"k": torch.zeros(s["k_out"].shape, dtype=torch.float64, device="cuda"), "v": torch.zeros(s["v_out"].shape, dtype=torch.float64, device="cuda")}
        row = s["k"].shape[-1]
        for i in range(b):
            o, n_old, n_new = int(s["out_start"][i]), int(s["slot_m"][i]) // row, int(s["rows"][i])
            for name, src in (("k", s["key"]), ("v", s["value"])):
                scale = s[name + "_scale"]
                x = src[int(s["starts"][i]):int(s["starts"][i]) + n_new].double().view(n_new, kvh, 4, 32)
                want = x.abs().amax(-1) / (7.0 * scale.double())[:, None]
                step = want.clamp(max=448.0).float().to(torch.float8_e4m3fn).double() * scale.double()[:, None]
                v = torch.where(step[..., None] > 0, torch.round(x / step[..., None]), 0.0).clamp(-7, 7) * step[..., None]
                got[name][o + n_old:o + n_old + n_new] = v.view(n_new, kvh, D)
                got[name][o:o + n_old] = _row64(s[name][int(s["slots"][i]), :n_old], kvh, scale)
        return got
    if op == "prompt":
        scores = s["scores"].double()
        for i in range(b):
            n, nq, w = int(s["seq_lens"][i]), int(s["q_lens"][i]), min(case["window"], int(s["q_lens"][i]))
            q = s["q"][int(s["q_start"][i]) + nq - w:int(s["q_start"][i]) + nq].double().view(w, kvh, g, D)
            x = torch.einsum("wkgd,nkd->kgwn", q, _cache64(s, "k", i)) * s["scale"]
            late = torch.arange(n, device="cuda") > (n - w + torch.arange(w, device="cuda"))[:, None]
            scores[int(s["slots"][i]), :, :n] += torch.softmax(x.masked_fill(late, -math.inf), -1).sum((1, 2))
        return {"scores": scores}
    out, lse = torch.zeros(b, h, D, dtype=torch.float64, device="cuda"), torch.full((b, h), -math.inf, dtype=torch.float64, device="cuda")
    scores = s["scores"].double() if op == "scored" else None
    for i in range(b):
        n = int(s["seq_lens"][i])
        if n == 0:
            continue
        x = torch.einsum("kgd,nkd->kgn", s["q"][i].double().view(kvh, g, D), _cache64(s, "k", i)) * s["scale"]
        p = torch.softmax(x, -1)
        out[i] = torch.einsum("kgn,nkd->kgd", p, _cache64(s, "v", i)).reshape(h, D)
        lse[i] = torch.logsumexp(x, -1).reshape(h)
        if scores is not None:
            scores[int(s["slots"][i]), :, :n] += p.sum(1)
    return {"out": out, "lse": lse} if op == "decode4" else {"out": out, "lse": lse, "scores": scores}
