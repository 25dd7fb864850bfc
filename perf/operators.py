"""The 8-bit KV cache and the attention over it, as measurable cases.

Three operators: `store` (rows are appended, each complete block of tokens is
quantised with one scale per KV head, and the blocks touched are read back),
`load` (rows of a filled cache are read back as fp16 or f32) and `attend`
(grouped-query attention of some query rows over a filled cache).

The cache's definition: rows are fp16 (f32 rows are rounded as they come). A
block of `block` tokens of one KV head, once complete, is held as codes and one
f32 scale, K and V apart; with a the largest magnitude of its block x d values,
    i8:    code = half-even rounding of 127 x / a,   value = code * (a / 127)
    e4m3:  code = e4m3 rounding of 448 x / a,        value = code * (a / 448)
and the tokens after the last complete block stay fp16.

Sizes: 32 query and 8 KV heads of 128 (the dense model of the benchmark),
head_dim 64 / 128 / 256 (the attention kernels' range), chunks of 1 to 256 rows
(the attention calls' range), 128-row micro-batches, contexts from one block to
131072 tokens.

Queries and values are normal; keys are normal with 1% of their channels 8 times
larger, as rotary keys have them.
"""
from __future__ import annotations

import math

import torch

own = False

TOP = {"i8": 127.0, "e4m3": 448.0}


# --- the cases ---------------------------------------------------------------

def listed():
    return [
        # a decode step's row that completes a block: two launches, latency
        store("store_decode_row", 991, 1, 8, 128, "i8", 32, "f16"),
        # a draft's rows from a token-major f32 projection, across a block end
        store("store_draft_rows", 1000, 37, 2, 256, "e4m3", 64, "f32"),
        # a whole prompt from a token-major f32 projection
        store("store_prompt", 0, 4096, 8, 128, "i8", 32, "f32"),
        # a prompt's prefix taken out of the cache, to keep or to share it
        load("load_prefix", 16384, 0, 16384, 8, 128, "i8", 32, "f16"),
        # a ragged piece, first and last row inside their blocks
        load("load_piece", 1030, 37, 977, 4, 64, "e4m3", 128, "f32"),
        # one decode step over a filled context of the dense model
        attend("decode", 1, 3980, 32, 8, 128, "i8", 32, True, "f16"),
        # the same over a very long context
        attend("decode_long", 1, 131071, 32, 8, 128, "e4m3", 64, True, "f32"),
        # few KV heads of 256, a long context
        attend("decode_d256", 1, 16000, 16, 2, 256, "i8", 32, True, "f32"),
        # bidirectional rows over narrow heads (no mask), ragged lengths
        attend("rows_d64", 19, 1981, 16, 8, 64, "e4m3", 128, False, "f16"),
        # a 128-token micro-batch at the end of a filled context
        attend("chunk", 128, 3968, 32, 8, 128, "i8", 32, True, "f16"),
        # the same with wide heads, f32 outputs
        attend("chunk_d256", 128, 1920, 16, 2, 256, "e4m3", 64, True, "f32"),
        # the largest: 256 rows at the end of a long context
        attend("chunk_long", 256, 32512, 32, 8, 128, "i8", 64, True, "f32"),
    ]


def store(name, start, rows, kh, d, fmt, block, dtype):
    return {"name": name, "kind": "store", "start": start, "rows": rows, "kh": kh, "d": d, "fmt": fmt,
            "block": block, "dtype": dtype}


def load(name, length, first, rows, kh, d, fmt, block, dtype):
    return {"name": name, "kind": "load", "length": length, "first": first, "rows": rows, "kh": kh, "d": d,
            "fmt": fmt, "block": block, "dtype": dtype}


def attend(name, rows, position, qh, kh, d, fmt, block, causal, dtype):
    return {"name": name, "kind": "attend", "rows": rows, "position": position, "qh": qh, "kh": kh, "d": d,
            "fmt": fmt, "block": block, "causal": causal, "dtype": dtype}


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["store", "load", "attend", "attend", "attend"])
    kh, d = rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 256])
    fmt, block, dtype = rng.choice(["i8", "e4m3"]), rng.choice([32, 64, 128]), rng.choice(["f16", "f32"])
    if kind == "store":
        case = store("", _log(rng, 1, 4096) - 1, _log(rng, 1, 4096), kh, d, fmt, block, dtype)
    elif kind == "load":
        rows = _log(rng, 1, 16384)
        first = _log(rng, 1, 4096) - 1
        case = load("", first + rows + rng.randrange(100), first, rows, kh, d, fmt, block, dtype)
    else:
        rows, qh = _log(rng, 1, 256), kh * rng.choice([1, 2, 4, 8])
        # (at most the keys of the longest listed context, and the products of the largest listed call)
        most = min(131072, 131072 * 1024 // (kh * d), 32768 * 256 * 4096 // (rows * qh * d)) - rows
        position = _log(rng, 1, most) - 1
        case = attend("", rows, position, qh, kh, d, fmt, block, rng.random() < 0.75, dtype)
    del case["name"]
    return case


# --- inputs ------------------------------------------------------------------

def _dtype(case):
    return torch.float16 if case["dtype"] == "f16" else torch.float32


def _heads(g, rows, heads, d, outliers):
    """[heads][rows][d] fp16 values."""
    x = torch.randn(heads, rows, d, generator=g, device="cuda")
    if outliers:
        wide = torch.randperm(heads * d, generator=g, device="cuda")[:math.ceil(0.01 * heads * d)]
        x *= torch.ones(heads * d, device="cuda").index_fill_(0, wide, 8.0).view(heads, 1, d)
    return x.half()


def _token_major(g, rows, kh, d):
    """A projection's f32 output [rows][k heads, v heads], as [kh][rows][d] views."""
    both = torch.randn(rows, 2 * kh, d, generator=g, device="cuda")
    return both[:, :kh].transpose(0, 1), both[:, kh:].transpose(0, 1)


def _inputs(case, seed):
    """The case's inputs, a function of the seed alone."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    kh, d, rows = case["kh"], case["d"], case["rows"]
    held = {"store": lambda: case["start"], "load": lambda: case["length"],
            "attend": lambda: case["position"] + rows}[case["kind"]]()
    x = {"k": _heads(g, held, kh, d, True), "v": _heads(g, held, kh, d, False)}
    if case["kind"] == "store":
        if case["dtype"] == "f16":
            x["new_k"], x["new_v"] = _heads(g, rows, kh, d, True), _heads(g, rows, kh, d, False)
        else:
            x["new_k"], x["new_v"] = _token_major(g, rows, kh, d)
    elif case["kind"] == "attend":
        x["q"] = _heads(g, rows, case["qh"], d, False)
    return x


# --- what a program holds, and one pass ----------------------------------------

def prepare(case, seed):
    x = _inputs(case, seed)
    kind, kh, d, rows = case["kind"], case["kh"], case["d"], case["rows"]
    state = {"case": case}
    if kind == "store":
        # (the blocks touched: from the first one's begin)
        first = case["start"] // case["block"] * case["block"]
        count = case["start"] + rows - first
        state.update(new_k=x["new_k"], new_v=x["new_v"], first=first)
        state.update({n: torch.empty(kh, count, d, device="cuda") for n in ("out_k", "out_v")})
    elif kind == "load":
        state.update({n: torch.empty(kh, rows, d, dtype=_dtype(case), device="cuda") for n in ("out_k", "out_v")})
    else:
        state.update(q=x["q"], out=torch.empty(case["qh"], rows, d, dtype=_dtype(case), device="cuda"))
    if own:
        from open_rknpu2_lm_infer_amd import device as D
        held = x["k"].shape[1]
        ctx = D.DeviceContext(0)
        cache = D.KvCacheQ8(ctx, case.get("qh", kh), kh, d, d ** -0.5, held + (rows if kind == "store" else 0),
                            fmt=case["fmt"], block=case["block"], causal=case.get("causal", True),
                            max_query_rows=rows if kind == "attend" else 1)
        if held:
            cache.append(x["k"], x["v"])
        state.update(ctx=ctx, cache=cache)
        if kind == "attend":
            state["ws"] = ctx.attention_workspace(cache)
        torch.cuda.synchronize()
    else:
        state.update(held_k=_held(x["k"], case), held_v=_held(x["v"], case))
    return state


def _held(x, case):
    """What a plain cache of x's rows holds: codes, scales, and the fp16 rows after them."""
    codes, scales = _quantised(x, case["fmt"], case["block"])
    return codes, scales, x[:, codes.shape[1] * case["block"]:].clone()


def _quantised(x, fmt, block):
    """Codes [kh][blocks][block][d] and scales [kh][blocks] of the complete blocks of x [kh][rows][d]."""
    kh, rows, d = x.shape
    blocks = x[:, :rows // block * block].float().reshape(kh, rows // block, block, d)
    top = blocks.abs().amax(dim=(2, 3))
    # (the quotient in 64 bits: many lie on a border of two codes)
    scaled = blocks.double() * TOP[fmt] / torch.where(top > 0, top, torch.ones_like(top))[:, :, None, None]
    codes = torch.round(scaled).to(torch.int8) if fmt == "i8" else scaled.to(torch.float8_e4m3fn)
    return codes, top / TOP[fmt]


def _values(codes, scales, tail):
    """The f32 values [kh][rows][d] that a plain cache stands for."""
    kh, blocks, block, d = codes.shape
    return torch.cat([(codes.float() * scales[:, :, None, None]).reshape(kh, blocks * block, d), tail.float()], dim=1)


def _store(held, new, fmt, block):
    rows = torch.cat([held[2], new.half()], dim=1)
    codes, scales = _quantised(rows, fmt, block)
    return _values(codes, scales, rows[:, codes.shape[1] * block:])


def _attend(q, k, v, scale, position, causal):
    """softmax(scale q k) v in f32; q [qh][rows][d], k and v [kh][keys][d]."""
    qh, rows, d = q.shape
    kh, keys, _ = k.shape
    s = torch.matmul(q.float().reshape(kh, qh // kh * rows, d), k.transpose(1, 2)) * scale
    s = s.view(kh, qh // kh, rows, keys)
    if causal:
        at = torch.arange(keys, device=q.device)
        seen = position + torch.arange(rows, device=q.device)
        s = torch.where(at[None, :] > seen[:, None], torch.full((), -math.inf, device=q.device), s)
    p = torch.exp(s - s.amax(dim=-1, keepdim=True))
    out = torch.matmul(p.view(kh, -1, keys), v) / p.sum(dim=-1).view(kh, -1, 1)
    return out.view(qh, rows, d)


def run(state):
    case = state["case"]
    kind = case["kind"]
    if own:
        cache = state["cache"]
        if kind == "store":
            cache.truncate(case["start"])
            cache.append(state["new_k"], state["new_v"])
            cache.read(state["first"], state["out_k"], state["out_v"])
            return state["out_k"], state["out_v"]
        if kind == "load":
            cache.read(case["first"], state["out_k"], state["out_v"])
            return state["out_k"], state["out_v"]
        from open_rknpu2_lm_infer_amd import device as D
        D.attention_q8(state["ctx"], cache, state["q"], state["out"], case["position"], ws=state["ws"])
        return state["out"]
    if kind == "store":
        return tuple(_store(state["held_" + n], state["new_" + n], case["fmt"], case["block"]) for n in ("k", "v"))
    k, v = _values(*state["held_k"]), _values(*state["held_v"])
    if kind == "load":
        piece = slice(case["first"], case["first"] + case["rows"])
        return k[:, piece].to(_dtype(case)), v[:, piece].to(_dtype(case))
    return _attend(state["q"], k, v, case["d"] ** -0.5, case["position"], case["causal"]).to(_dtype(case))


# --- what a pass cannot do without --------------------------------------------

def work(case):
    kind, kh, d, rows, block = case["kind"], case["kh"], case["d"], case["rows"], case["block"]
    esz = 2 if case["dtype"] == "f16" else 4
    if kind == "store":
        first = case["start"] // block * block
        count = case["start"] + rows - first
        coded = count // block * block
        # rows in, the open block's rows, codes and scales or fp16 tail out; the
        # same in again, f32 values out
        held = coded * d + 4 * (coded // block) + 2 * (count - coded) * d
        return {"bytes": 2 * kh * (rows * d * esz + 2 * (case["start"] - first) * d + 2 * held + 4 * count * d),
                "flops": 4 * kh * count * d}
    if kind == "load":
        coded = max(0, min(case["first"] + rows, case["length"] // block * block) - case["first"])
        return {"bytes": 2 * kh * (coded * d + 4 * (coded // block) + 2 * (rows - coded) * d + rows * d * esz),
                "flops": 2 * kh * rows * d}
    qh, pos = case["qh"], case["position"]
    keys = pos + rows
    coded = keys // block * block
    seen = rows * (pos + (rows + 1) / 2) if case["causal"] else rows * keys
    return {"bytes": 2 * kh * (coded * d + 4 * (coded // block) + 2 * (keys - coded) * d) + qh * rows * d * (2 + esz),
            "flops": int(4 * qh * d * seen)}


# --- the same in 64 bits -------------------------------------------------------

def _exact_values(x, fmt, block):
    """The values [kh][rows][d] of a cache of x's rows, in 64 bits, block by block from the definition."""
    y = x.to(torch.float16).double()
    whole = y.shape[1] - y.shape[1] % block
    body = y[:, :whole].unflatten(1, (-1, block)) if whole else y[:, :0].unsqueeze(2)
    if whole:
        largest = body.abs().flatten(2).max(dim=2).values[..., None, None]
        unit = largest / TOP[fmt]
        t = torch.where(largest > 0, body * TOP[fmt] / largest.clamp_min(1e-300), torch.zeros_like(body))
        if fmt == "i8":
            code = torch.round(t)
        else:
            # e4m3: 3 bits after the leading one, steps of 2^-9 below 2^-6
            steps = torch.tensor([2.0 ** n for n in range(-9, 6)], dtype=torch.float64, device=t.device)
            step = steps[torch.frexp(t)[1].clamp_min(-5).long() + 5]
            code = torch.round(t / step) * step
        y = torch.cat([(code * unit).flatten(1, 2), y[:, whole:]], dim=1)
    return y


def exact(case, seed):
    x = _inputs(case, seed)
    fmt, block = case["fmt"], case["block"]
    if case["kind"] == "store":
        first = case["start"] // block * block
        return tuple(_exact_values(torch.cat([x[n][:, first:].float(), x["new_" + n].float()], dim=1), fmt, block)
                     for n in ("k", "v"))
    k, v = _exact_values(x["k"], fmt, block), _exact_values(x["v"], fmt, block)
    if case["kind"] == "load":
        last = case["first"] + case["rows"]
        return k[:, case["first"]:last], v[:, case["first"]:last]
    rows, pos, group = case["rows"], case["position"], case["qh"] // case["kh"]
    out = torch.empty(case["qh"], rows, case["d"], dtype=torch.float64, device="cuda")
    # (the attention takes its scale as a 32-bit number)
    scale = float(torch.tensor(case["d"] ** -0.5, dtype=torch.float32))
    hidden = torch.ones(rows, pos + rows, dtype=torch.bool, device="cuda").triu_(pos + 1)
    for h in range(case["qh"]):
        s = (x["q"][h].double() @ k[h // group].t().contiguous()) * scale
        if case["causal"]:
            s.masked_fill_(hidden, -math.inf)
        out[h] = torch.softmax(s, dim=1) @ v[h // group]
    return out
