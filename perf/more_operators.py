"""The paged KV cache of a batch of sequences, as measurable cases.

Two operators: `append` (the batch's new K and V rows are rotated by their
positions and put into their sequences' pages, the query rows are rotated in the
same call, and the new rows are read back out of the pages) and `attend`
(grouped-query attention of each sequence's newest rows over its pages: one row
a sequence in a decode step, some for a draft's verification, many for a
prompt or a piece of one).

Definitions. A pool holds fp16 rows in pages of `page` tokens; token t of
sequence s lies in page table[s][t / page], at t % page. The batch's rows are
the sequences' newest tokens, the rows of one sequence after another: row i of
the n of a sequence of length L (these rows included) is token L - n + i.
Rotation: dims x[j], y[j] of pair j become x cos - y sin and y cos + x sin of
the angle position * theta^(-2 j / rotary); a pair is (j, j + rotary / 2), or
(2 j, 2 j + 1) where interleaved; dims from `rotary` on stay; K and V are rounded
to fp16 once, after it. Attention: softmax(scale q k) v over the tokens up to the
row's own, or over all L without a causal mask; a row that sees no token is 0.

Sizes: 32 query and 8 KV heads of 128 (the dense model of the benchmark),
head_dim 64 / 128 / 256 (the attention kernels' range), batches of 1 to 256
sequences, contexts up to 131072 tokens, prompts of 1 to 4096 rows, a rotation
of all dims or of the first quarter.
"""
from __future__ import annotations

import math

import torch

own = False


# --- the cases ---------------------------------------------------------------

def listed():
    return [
        # a decode step of a batch of conversations: latency
        append("append_decode", 64, 0, 4000, 1, 1, 32, 8, 128, 64, 128, False, 1e6, "f16"),
        # drafts from a token-major f32 projection, wide heads, a quarter of the dims rotated, far positions
        append("append_drafts", 7, 90000, 131000, 5, 5, 16, 2, 256, 16, 64, True, 1e7, "f32"),
        # a batch of whole prompts from a token-major f32 projection
        append("append_prompts", 6, 0, 0, 17, 1365, 32, 8, 128, 64, 128, False, 1e6, "f32"),
        # one conversation's decode step: latency
        attend("decode_one", 1, 3980, 3980, 1, 1, 0, 32, 8, 128, 64, True, "f16"),
        # many short ones over narrow heads in small pages, some places of the batch idle
        attend("decode_short", 240, 0, 700, 1, 1, 16, 16, 8, 64, 16, True, "f16"),
        # a server's batch, ragged lengths
        attend("decode_batch", 64, 60, 8100, 1, 1, 0, 32, 8, 128, 64, True, "f16"),
        # few very long ones
        attend("decode_long", 2, 131071, 131071, 1, 1, 0, 32, 8, 128, 256, True, "f32"),
        # few KV heads of 256
        attend("decode_d256", 16, 900, 16000, 1, 1, 0, 16, 2, 256, 32, True, "f32"),
        # verification of 5 drafted tokens a sequence
        attend("verify", 12, 500, 9000, 5, 5, 0, 32, 8, 128, 32, True, "f16"),
        # a batch of whole prompts
        attend("prompts", 6, 0, 0, 17, 1365, 0, 32, 8, 128, 64, True, "f16"),
        # pieces of prompts over wide heads, rows that see the whole of their sequence
        attend("chunk_d256", 3, 1000, 7000, 100, 200, 0, 16, 2, 256, 128, False, "f32"),
        # the largest: a piece of a prompt at the end of a long context
        attend("chunk_long", 1, 65000, 65000, 512, 512, 0, 32, 8, 128, 64, True, "f16"),
    ]


def append(name, sequences, ctx_lo, ctx_hi, rows_lo, rows_hi, qh, kh, d, page, rotary, interleaved, theta, dtype):
    return {"name": name, "kind": "append", "sequences": sequences, "ctx_lo": ctx_lo, "ctx_hi": ctx_hi,
            "rows_lo": rows_lo, "rows_hi": rows_hi, "idle": 0, "qh": qh, "kh": kh, "d": d, "page": page,
            "rotary": rotary, "interleaved": interleaved, "theta": theta, "dtype": dtype}


def attend(name, sequences, ctx_lo, ctx_hi, rows_lo, rows_hi, idle, qh, kh, d, page, causal, dtype):
    return {"name": name, "kind": "attend", "sequences": sequences, "ctx_lo": ctx_lo, "ctx_hi": ctx_hi,
            "rows_lo": rows_lo, "rows_hi": rows_hi, "idle": idle, "qh": qh, "kh": kh, "d": d, "page": page,
            "causal": causal, "dtype": dtype}


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "decode", "decode", "verify", "rows"])
    kh, d = rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 256])
    qh, page, dtype = kh * rng.choice([1, 2, 4, 8]), rng.choice([16, 32, 64, 128, 256]), rng.choice(["f16", "f32"])
    sequences = _log(rng, 1, 256)
    if kind == "append":
        rows = _log(rng, 1, max(1, 4096 // sequences))
        ctx = _log(rng, 1, max(1, 1048576 // sequences))
        case = append("", sequences, rng.randrange(ctx), ctx, rng.randint(1, rows), rows, qh, kh, d, page,
                      rng.choice([d, d // 4]), rng.random() < 0.5, rng.choice([1e4, 1e6, 1e7]), dtype)
    elif kind == "decode":
        # (a GB of fp16 rows at most)
        ctx = _log(rng, 1, min(131072, 262144 * 1024 // (sequences * kh * d)))
        case = attend("", sequences, rng.randrange(ctx), ctx, 1, 1, rng.choice([0, 0, sequences // 8]), qh, kh, d, page,
                      True, dtype)
    else:
        if kind == "verify":
            sequences = min(sequences, 32)
            rows = rng.randint(2, 8)
        else:
            sequences = _log(rng, 1, 16)
            rows = _log(rng, 9, 4096 // sequences)
        # (the bytes of the decode steps, the products of the largest listed call)
        most = min(262144 * 1024 // (sequences * kh * d), 65000 * 512 * 4096 // (rows * sequences * qh * d)) - rows
        ctx = _log(rng, 1, min(131072 - rows, max(2, most))) - 1
        case = attend("", sequences, rng.randint(0, ctx), ctx, rng.randint(max(1, rows // 4), rows), rows, 0, qh, kh, d,
                      page, rng.random() < 0.75, dtype)
    del case["name"]
    return case


def _spread(n, lo, hi):
    """n sizes over lo..hi, both among them, in no order."""
    return [hi if i == 0 else lo if i == 1 else lo + int((hi - lo + 1) * (i * 0.6180339887498949 % 1.0)) for i in range(n)]


def _sizes(case):
    """The sequences' lengths with the call's rows, and their rows; idle places have no tokens and a row each."""
    n, idle = case["sequences"], case["idle"]
    ctx, rows = _spread(n, case["ctx_lo"], case["ctx_hi"]), _spread(n, case["rows_lo"], case["rows_hi"])
    return [c + r for c, r in zip(ctx, rows)] + [0] * idle, rows + [1] * idle


# --- inputs ------------------------------------------------------------------

def _dtype(case):
    return torch.float16 if case["dtype"] == "f16" else torch.float32


def _heads(g, rows, heads, d, outliers):
    """[heads][rows][d] fp16 values; keys have 1% of their channels 8 times larger, as rotary keys do."""
    x = torch.randn(heads, rows, d, generator=g, device="cuda")
    if outliers:
        wide = torch.randperm(heads * d, generator=g, device="cuda")[:math.ceil(0.01 * heads * d)]
        x *= torch.ones(heads * d, device="cuda").index_fill_(0, wide, 8.0).view(heads, 1, d)
    return x.half()


def _inputs(case, seed):
    """The case's inputs, a function of the seed alone."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    qh, kh, d, page = case["qh"], case["kh"], case["d"], case["page"]
    lengths, rows = _sizes(case)
    # every sequence's pages, from all over the pool
    counts = [-(-n // page) for n in lengths]
    order = torch.randperm(sum(counts), generator=g, device="cuda").int()
    table = torch.zeros(len(lengths), max(counts), dtype=torch.int32, device="cuda")
    at = 0
    for s, n in enumerate(counts):
        table[s, :n] = order[at:at + n]
        at += n
    x = {"table": table, "pages": at}
    if case["kind"] == "append":
        # one projection's output [rows][q heads, k heads, v heads], as [heads][rows][d] views
        every = torch.randn(sum(rows), qh + 2 * kh, d, generator=g, device="cuda").to(_dtype(case)).transpose(0, 1)
        x.update(new_q=every[:qh], new_k=every[qh:qh + kh], new_v=every[qh + kh:])
    else:
        # the sequences' tokens, one sequence after another
        x.update(k=_heads(g, sum(lengths), kh, d, True), v=_heads(g, sum(lengths), kh, d, False),
                 q=_heads(g, sum(rows), qh, d, False))
    return x


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _offsets(sizes):
    out = [0]
    for n in sizes:
        out.append(out[-1] + n)
    return out


def _slots(case, table, sizes):
    """Where the last sizes[s] tokens of each sequence lie, as page * page_tokens + place, one sequence after another."""
    lengths = _sizes(case)[0]
    page = case["page"]
    slots = []
    for s, n in enumerate(sizes):
        t = torch.arange(max(0, lengths[s] - n), lengths[s], device="cuda")
        slots.append(table[s, t // page].long() * page + t % page)
    return torch.cat(slots)


# --- what a program holds, and one pass ----------------------------------------

def prepare(case, seed):
    x = _inputs(case, seed)
    qh, kh, d, page = case["qh"], case["kh"], case["d"], case["page"]
    lengths, rows = _sizes(case)
    state = {"case": case}
    if own:
        from open_rknpu2_lm_infer_amd import device as D
        ctx = D.DeviceContext(0)
        pages = D.KvPages(ctx, qh, kh, d, d ** -0.5, pages=x["pages"], page=page, capacity=max(lengths),
                          causal=case.get("causal", True), rotary_dim=case.get("rotary", 0),
                          interleaved=case.get("interleaved", False), rope_theta=case.get("theta", 1e4))
        step = D.PagedBatch(x["table"], _ints(lengths), None if max(rows) == 1 else _ints(_offsets(rows)),
                            max_rows=max(rows), max_tokens=max(lengths))
        state.update(ctx=ctx, pages=pages, batch=step)
        if case["kind"] == "attend":
            held = D.PagedBatch(x["table"], _ints(lengths), _ints(_offsets(lengths)), max_rows=max(lengths),
                                max_tokens=max(lengths))
            pages.append(held, x["k"], x["v"])
            state["ws"] = ctx.attention_workspace(pages)
        torch.cuda.synchronize()
    elif case["kind"] == "attend":
        state.update({n: torch.zeros(x["pages"] * page, kh, d, dtype=torch.float16, device="cuda") for n in ("pool_k", "pool_v")})
        every = _slots(case, x["table"], lengths)
        for n in ("k", "v"):
            state["pool_" + n][every] = x[n].transpose(0, 1)
        state["slots"] = every
    else:
        state.update({n: torch.zeros(x["pages"] * page, kh, d, dtype=torch.float16, device="cuda") for n in ("pool_k", "pool_v")})
        state["slots"] = _slots(case, x["table"], rows)
    if case["kind"] == "append":
        state.update(new_q=x["new_q"], new_k=x["new_k"], new_v=x["new_v"],
                     out_q=torch.empty(qh, sum(rows), d, dtype=torch.float16, device="cuda"))
        state.update({n: torch.empty(kh, sum(rows), d, dtype=torch.float16, device="cuda") for n in ("out_k", "out_v")})
        state["positions"] = _ints([lengths[s] - n + i for s, n in enumerate(rows) for i in range(n)])
        # angle of pair j at position p: p * frequency[j]
        half = case["rotary"] // 2
        state["frequencies"] = case["theta"] ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)
    else:
        state.update(q=x["q"], out=torch.empty(qh, sum(rows), d, dtype=_dtype(case), device="cuda"))
    return state


def _rotated(x, positions, frequencies, interleaved):
    """x [heads][rows][d] in f32, its first dims rotated."""
    rotary = 2 * frequencies.numel()
    angle = positions.double()[:, None] * frequencies
    c, s = torch.cos(angle).float(), torch.sin(angle).float()
    x = x.float()
    head, rest = x[..., :rotary], x[..., rotary:]
    if interleaved:
        a, b = head[..., 0::2], head[..., 1::2]
        turned = torch.stack([a * c - b * s, b * c + a * s], dim=-1).flatten(-2)
    else:
        a, b = head[..., :rotary // 2], head[..., rotary // 2:]
        turned = torch.cat([a * c - b * s, b * c + a * s], dim=-1)
    return torch.cat([turned, rest], dim=-1)


def _append(state):
    case, slots = state["case"], state["slots"]
    turn = (state["positions"], state["frequencies"], case["interleaved"])
    state["pool_k"][slots] = _rotated(state["new_k"], *turn).half().transpose(0, 1)
    state["pool_v"][slots] = state["new_v"].half().transpose(0, 1)
    q = _rotated(state["new_q"], *turn).half()
    return q, state["pool_k"][slots].transpose(0, 1), state["pool_v"][slots].transpose(0, 1)


def _attend(q, k, v, scale, first, causal):
    """softmax(scale q k) v in f32; q [qh][rows][d], row i is token first + i; k and v [tokens][kh][d]."""
    qh, rows, d = q.shape
    tokens, kh, _ = k.shape
    k, v = k.float().transpose(0, 1), v.float().transpose(0, 1)
    s = torch.matmul(q.float().reshape(kh, qh // kh * rows, d), k.transpose(1, 2)) * scale
    s = s.view(kh, qh // kh, rows, tokens)
    if causal:
        seen = first + torch.arange(rows, device=q.device)
        s = torch.where(torch.arange(tokens, device=q.device)[None, :] > seen[:, None],
                        torch.full((), -math.inf, device=q.device), s)
    p = torch.exp(s - s.amax(dim=-1, keepdim=True))
    out = torch.matmul(p.view(kh, -1, tokens), v) / p.sum(dim=-1).view(kh, -1, 1)
    return out.view(qh, rows, d)


def run(state):
    case = state["case"]
    if own:
        pages, batch = state["pages"], state["batch"]
        if case["kind"] == "append":
            pages.append(batch, state["new_k"], state["new_v"], q=state["new_q"], q_out=state["out_q"])
            pages.read(batch, state["out_k"], state["out_v"])
            return state["out_q"], state["out_k"], state["out_v"]
        from open_rknpu2_lm_infer_amd import device as D
        D.attention_paged(state["ctx"], pages, batch, state["q"], state["out"], ws=state["ws"])
        return state["out"]
    if case["kind"] == "append":
        return _append(state)
    lengths, rows = _sizes(case)
    tokens, begins = _offsets(lengths), _offsets(rows)
    out = torch.zeros(case["qh"], sum(rows), case["d"], device="cuda")
    for s in range(case["sequences"]):
        at, mine = state["slots"][tokens[s]:tokens[s + 1]], slice(begins[s], begins[s + 1])
        out[:, mine] = _attend(state["q"][:, mine], state["pool_k"][at], state["pool_v"][at], case["d"] ** -0.5,
                               lengths[s] - rows[s], case["causal"])
    return out.to(_dtype(case))


# --- what a pass cannot do without --------------------------------------------

def work(case):
    qh, kh, d = case["qh"], case["kh"], case["d"]
    lengths, rows = _sizes(case)
    total = sum(rows)
    esz = 2 if case["dtype"] == "f16" else 4
    if case["kind"] == "append":
        # rows in; q and fp16 K and V out; K and V in again and out
        return {"bytes": total * d * ((qh + 2 * kh) * esz + 2 * qh + 3 * 2 * 2 * kh) + 4 * len(lengths),
                "flops": 3 * total * (qh + kh) * case["rotary"]}
    pages = sum(-(-n // case["page"]) for n in lengths)
    seen = 0
    for n, r in zip(lengths, rows):
        if n:
            seen += r * (n - r) + r * (r + 1) // 2 if case["causal"] else r * n
    return {"bytes": 2 * 2 * kh * d * sum(lengths) + qh * total * d * (2 + esz) + 4 * pages + 4 * len(lengths),
            "flops": 4 * qh * d * seen}


# --- the same in 64 bits -------------------------------------------------------

def exact(case, seed):
    x = _inputs(case, seed)
    lengths, rows = _sizes(case)
    qh, kh, d = case["qh"], case["kh"], case["d"]
    if case["kind"] == "append":
        n = case["rotary"]
        where = torch.cat([torch.arange(end - r, end, dtype=torch.float64, device="cuda") for end, r in zip(lengths, rows)])
        pair = torch.arange(n // 2, dtype=torch.float64, device="cuda")
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                           where[:, None] * torch.exp(-2.0 * pair / n * math.log(case["theta"])))
        first = 2 * pair.long() if case["interleaved"] else pair.long()
        second = first + (1 if case["interleaved"] else n // 2)

        def rotated(y):
            y = y.double().clone()
            z = torch.complex(y[..., first], y[..., second]) * turn
            y[..., first], y[..., second] = z.real, z.imag
            return y
        return rotated(x["new_q"]), rotated(x["new_k"]), x["new_v"].double()
    group = qh // kh
    out = torch.zeros(qh, sum(rows), d, dtype=torch.float64, device="cuda")
    # (the attention takes its scale as a 32-bit number)
    scale = float(torch.tensor(d ** -0.5, dtype=torch.float32))
    token, row = 0, 0
    for n, r in zip(lengths, rows):
        for g in range(kh if n else 0):
            k, v = x["k"][g, token:token + n].double(), x["v"][g, token:token + n].double()
            for h in range(g * group, (g + 1) * group):
                s = (x["q"][h, row:row + r].double() @ k.t().contiguous()) * scale
                if case["causal"]:
                    s.masked_fill_(torch.ones(r, n, dtype=torch.bool, device="cuda").triu_(n - r + 1), -math.inf)
                out[h, row:row + r] = torch.softmax(s, dim=1) @ v
        token, row = token + n, row + r
    return out
