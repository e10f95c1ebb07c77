"""The operators of the decoder layer's attention over a paged cache, as timed cases: each in its plain form and as the
framework's own call.

* ``step``    page tables, positions and cache slots of a step's new tokens, from the requests' lengths;
* ``cache``   a fused qkv projection's rows: RMSNorm and rotation of the heads, keys and values into the cache;
* ``decode``  attention of one new token a request over its cached tokens, with or without a sliding window and first
              tokens that stay visible;
* ``prompt``  the same of many new tokens a request, causal among themselves.

The heads are the talker's and the predictor's (16 query heads and 8 key-value heads of 128, which make their qkv width of
2048 + 1024 + 1024); ``draw`` adds others.  A page holds ``[kv heads, page size, head size]`` keys and
``[kv heads, head size, page size]`` values.
"""

import os
import random
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "tts-inference_amd"))

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-6
THETA = 1e6  # the base of the rotation's angles
TALKER = {"heads": 16, "kv_heads": 8, "head_dim": 128}


def listed():
    return [
        # A full decode batch grows by a token each: latency alone counts.
        {"name": "step_64requests", "kind": "step", "requests": 64, "rows": 64, "cached": 4096, "page": 64},
        # A burst of ragged prompts and chunks of prompts, small pages, a few requests denied for want of them.
        {"name": "step_prompts_49152rows", "kind": "step", "requests": 200, "rows": 49152, "cached": 512, "page": 16},
        # One stream's decode step: one row, latency alone.
        {"name": "cache_1row", "kind": "cache", "requests": 1, "rows": 1, "cached": 900, "page": 64, "dtype": "bf16", **TALKER,
         "norm": True, "rope": True},
        # Prompts of seven requests in one batch with a few padding rows: bandwidth.
        {"name": "cache_2048rows", "kind": "cache", "requests": 7, "rows": 2048, "cached": 200, "page": 64, "dtype": "bf16",
         **TALKER, "norm": True, "rope": True},
        # One stream of speech a few seconds in: the smallest call, latency alone.
        {"name": "decode_1x300", "kind": "decode", "requests": 1, "cached": 300, "ragged": False, "page": 64, "dtype": "bf16",
         **TALKER, "window": 0, "sinks": 0},
        # A busy server's streams of ragged lengths, a window of the last tokens and the first four, small pages.
        {"name": "decode_27x4001_window", "kind": "decode", "requests": 27, "cached": 4001, "ragged": True, "page": 16,
         "dtype": "bf16", **TALKER, "window": 512, "sinks": 4},
        # A full batch of long conversations in fp16: the cache's bytes bound it.
        {"name": "decode_64x8192", "kind": "decode", "requests": 64, "cached": 8192, "ragged": True, "page": 64,
         "dtype": "fp16", **TALKER, "window": 0, "sinks": 0},
        # One very long document: the length has to be split to fill the card.
        {"name": "decode_1x65536", "kind": "decode", "requests": 1, "cached": 65536, "ragged": False, "page": 64,
         "dtype": "bf16", **TALKER, "window": 0, "sinks": 0},
        # The first text of three streams: few rows, latency.
        {"name": "prompt_3x37", "kind": "prompt", "requests": 3, "new": 37, "cached": 0, "page": 64, "dtype": "bf16", **TALKER,
         "window": 0, "sinks": 0},
        # Chunks of four long prompts, behind what is cached of each, in fp16.
        {"name": "prompt_4x1003_cached", "kind": "prompt", "requests": 4, "new": 1003, "cached": 2500, "page": 32,
         "dtype": "fp16", **TALKER, "window": 0, "sinks": 0},
        # One long prompt: the matrix cores bound it.
        {"name": "prompt_1x8192", "kind": "prompt", "requests": 1, "new": 8192, "cached": 0, "page": 64, "dtype": "bf16",
         **TALKER, "window": 0, "sinks": 0},
        # A prompt of twice that length under a window with the first four tokens.
        {"name": "prompt_1x16384_window", "kind": "prompt", "requests": 1, "new": 16384, "cached": 0, "page": 64,
         "dtype": "bf16", **TALKER, "window": 1024, "sinks": 4},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    kind = rng.choice(["step", "cache", "decode", "decode", "prompt", "prompt"])
    case = {"kind": kind, "page": rng.choice([16, 32, 64, 64, 128])}
    if kind == "step":
        requests = _log(rng, 1, 500)
        return dict(case, requests=requests, rows=_log(rng, requests, 49152), cached=_log(rng, 1, 8192))
    heads = rng.choice([(16, 8), (16, 8), (32, 8), (8, 8), (16, 1), (12, 4), (28, 4)])
    case |= {"heads": heads[0], "kv_heads": heads[1], "head_dim": rng.choice([64, 80, 128, 128, 128, 256]),
             "dtype": rng.choice(["bf16", "bf16", "fp16"])}
    if kind == "cache":
        rows = _log(rng, 1, 2048 * 4096 // ((heads[0] + 2 * heads[1]) * case["head_dim"]))
        return dict(case, rows=rows, requests=min(rows, _log(rng, 1, 40)), cached=_log(rng, 1, 4096),
                    norm=rng.random() < 0.7, rope=rng.random() < 0.8)
    windowed = rng.random() < 0.4
    case |= {"window": _log(rng, 16, 4096) if windowed else 0, "sinks": rng.choice([0, 1, 4, 4, 100]) if windowed else 0}
    width = heads[1] * case["head_dim"] / 1024
    if kind == "decode":
        requests = _log(rng, 1, 64)
        return dict(case, requests=requests, cached=_log(rng, 1, int(min(65536, 64 * 4096 / requests / width))),
                    ragged=rng.random() < 0.7)
    requests = _log(rng, 1, 8)
    new = _log(rng, 2, int(8192 / requests ** 0.5 / max(1, heads[0] / 16)))
    return dict(case, requests=requests, new=new, cached=rng.choice([0, 0, _log(rng, 1, new)]))


# ---- inputs --------------------------------------------------------------------------------


def _randn(seed, index, *shape):
    g = torch.Generator(device="cuda").manual_seed(seed * 1000 + index)
    return torch.randn(*shape, generator=g, device="cuda")


def _lengths(case, seed):
    """Tokens that each request holds before the step, and how many join it: the same ones for every seed, dealt anew."""
    rng, n, cached = random.Random(case["requests"] * 8209 + case["cached"]), case["requests"], case["cached"]
    new = [1] * n
    if case["kind"] == "decode":
        held = [cached - 1] + [rng.randint(max(1, cached // 8), cached) - 1 if case["ragged"] else cached - 1 for _ in range(n - 1)]
    elif case["kind"] == "prompt":
        held = [rng.randint(cached // 2, cached) for _ in range(n)]
        new = [case["new"]] + [rng.randint(max(1, case["new"] // 2), case["new"]) for _ in range(n - 1)]
    else:
        held = [rng.randint(0, cached) for _ in range(n)]
        if case["rows"] > n:
            share = [rng.random() + 0.05 for _ in range(n)]
            live = case["rows"] - case["rows"] // 50  # the rest are padding rows
            new = [max(1, int(live * s / sum(share))) for s in share]
    rng = random.Random(seed)
    rng.shuffle(held)
    rng.shuffle(new)
    return held, new


def _pages(case, held, new):
    """Columns of the page table and pages of the pool, however the lengths are dealt."""
    page = case["page"]
    return -(-(max(held) + max(new)) // page), sum(-(-n // page) for n in held + new)


def prepare(case, seed):
    case = dict(case)
    held, new = _lengths(case, seed)
    width, total = _pages(case, held, new)
    page, requests = case["page"], case["requests"]
    rng = random.Random(seed + 1)
    pool = list(range(total + 8))
    rng.shuffle(pool)
    cuda = lambda values: torch.tensor(values, dtype=torch.int32).cuda()  # noqa: E731
    if case["kind"] == "step":
        taken, table = 0, torch.full((requests, width), -1, dtype=torch.int32)
        for r, n in enumerate(held):
            have = -(-n // page)
            table[r, :have] = torch.tensor(pool[taken:taken + have], dtype=torch.int32)
            taken += have
        if requests >= 100:  # the last requests find no page left
            pool = pool[:taken + (total - taken) * 15 // 16]
        return {"case": case, "new": cuda(new), "lengths": cuda(held), "table": table.cuda(), "free": cuda(pool),
                "taken": cuda([taken])}
    # a step's batch as page tables and slot maps give it
    rows = case["rows"] if case["kind"] == "cache" else sum(new)
    table = torch.zeros(requests, width, dtype=torch.int32)
    positions, slots = torch.full((rows,), -1, dtype=torch.int32), torch.full((rows,), -1, dtype=torch.int32)
    taken, starts = 0, [0]
    for r, (a, b) in enumerate(zip(held, new)):
        have = -(-(a + b) // page)
        table[r, :have] = torch.tensor(pool[taken:taken + have], dtype=torch.int32)
        taken += have
        at = torch.arange(a, a + b)
        positions[starts[-1]:starts[-1] + b] = at.int()
        slots[starts[-1]:starts[-1] + b] = table[r, at // page] * page + (at % page).int()
        starts.append(starts[-1] + b)
    heads, kv, d, dtype = case["heads"], case["kv_heads"], case["head_dim"], DTYPES[case["dtype"]]
    state = {"case": case, "table": table.cuda(), "positions": positions.cuda(), "slots": slots.cuda(), "starts": cuda(starts),
             "counts": cuda(new), "lengths": cuda([a + b for a, b in zip(held, new)]), "max_new": max(new), "min_new": min(new)}
    state["k"] = _randn(seed, 1, len(pool), kv, page, d).to(dtype)
    state["v"] = _randn(seed, 2, len(pool), kv, d, page).to(dtype)
    if case["kind"] != "cache":
        # scores of unit spread and a few keys that stand out, as trained heads have them
        state["q"] = (_randn(seed, 3, rows, heads, d) * 1.5).to(dtype)
        return state
    state["qkv"] = (_randn(seed, 3, rows, (heads + 2 * kv) * d) * 2).to(dtype)
    if case["norm"]:
        state["q_norm"], state["k_norm"] = ((1 + 0.2 * _randn(seed, i, d)).to(dtype) for i in (4, 5))
    if case["rope"]:
        at = torch.arange(width * page, dtype=torch.float64, device="cuda")
        angle = at[:, None] * THETA ** (-torch.arange(0, d, 2, dtype=torch.float64, device="cuda") / d)
        state["cos"], state["sin"] = angle.cos().float(), angle.sin().float()
    return state


# ---- a pass --------------------------------------------------------------------------------


def _plain_step(state):
    page, rows = state["case"]["page"], state["case"]["rows"]
    new, lengths, table, free, taken = (state[k] for k in ("new", "lengths", "table", "free", "taken"))
    new = new.long().clamp_min(0)
    ends = new.cumsum(0)
    starts, held = ends - new, (lengths + page - 1) // page
    fits = (lengths + new <= table.shape[1] * page) & (ends <= rows)
    need = torch.where(fits, (lengths + new + page - 1) // page - held, 0)
    upto = need.cumsum(0)
    ok = fits & ((need == 0) | (upto <= free.shape[0] - taken))
    counts = torch.where(ok, new, 0)
    # a row's request, position and page: an old one by the table, a new one by the free list
    row = torch.arange(rows, device=new.device)
    request = torch.searchsorted(ends, row, right=True).clamp_max(new.shape[0] - 1)
    live = (row < ends[-1]) & ok[request]
    position = lengths[request] + row - starts[request]
    column = torch.where(live, position // page, 0)
    fresh = live & (column >= held[request])
    source = torch.where(fresh, taken + upto[request] - need[request] + column - held[request], 0)
    found = torch.where(fresh, free[source], table[request, column])
    out = torch.cat([table.flatten(), table.new_zeros(1)])  # the rows without a new page write behind the end
    out[torch.where(fresh, request * table.shape[1] + column, table.numel())] = found
    table.copy_(out[:-1].view_as(table))
    slots = torch.where(live, found * page + position % page, -1)
    total = torch.cat([starts.new_zeros(1), ends])
    return [total.int(), counts.int(), (lengths + counts).int(), torch.where(live, position, -1).int(), slots.int(), table,
            (taken + torch.where(ok, need, 0).sum()).int()]


def _rotated(state, x, position):
    if "cos" not in state:
        return x
    cos, sin = state["cos"][position].unsqueeze(1), state["sin"][position].unsqueeze(1)
    lo, hi = x.chunk(2, -1)
    return torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1)


def _plain_cache(state):
    case, qkv, page = state["case"], state["qkv"], state["case"]["page"]
    heads, kv, d = case["heads"], case["kv_heads"], case["head_dim"]
    live, position = state["slots"] >= 0, state["positions"].clamp_min(0).long()
    q, k, v = qkv.view(qkv.shape[0], -1, d).split([heads, kv, kv], 1)
    q, k = q.float(), k.float()
    if case["norm"]:
        q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + EPS) * state["q_norm"].float()
        k = k * torch.rsqrt(k.square().mean(-1, keepdim=True) + EPS) * state["k_norm"].float()
    q, k = (_rotated(state, x, position) for x in (q, k))
    slot = state["slots"][live].long()
    state["k"][slot // page, :, slot % page] = k[live].to(qkv.dtype)
    state["v"][slot // page, :, :, slot % page] = v[live]
    return [torch.where(live[:, None, None], q, 0.0).to(qkv.dtype), state["k"], state["v"]]


def _plain_attention(state):
    """Every request against its pages, new rows and pages padded to the longest's."""
    case, q = state["case"], state["q"]
    heads, kv, d, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    table, starts, counts, lengths, new = (state[k] for k in ("table", "starts", "counts", "lengths", "max_new"))
    requests, reach = table.shape[0], table.shape[1] * page
    k = state["k"][table].float().transpose(1, 2).reshape(requests, kv, reach, d)
    v = state["v"][table].float().permute(0, 2, 1, 4, 3).reshape(requests, kv, reach, d)
    key = torch.arange(reach, device=q.device)
    held = (key < lengths[:, None]).view(requests, 1, reach, 1)
    k, v = torch.where(held, k, 0.0), torch.where(held, v, 0.0)
    nth = torch.arange(new, device=q.device)
    row = (starts[:-1, None] + nth).clamp_max(q.shape[0] - 1).long()  # [requests, new]
    rows = q[row].float().view(requests, new, kv, heads // kv, d).permute(0, 2, 3, 1, 4).reshape(requests, kv, -1, d)
    score = torch.matmul(rows, k.transpose(2, 3).contiguous()).mul_(d ** -0.5).view(requests, kv, heads // kv, new, reach)
    at = (lengths - counts)[:, None] + nth  # [requests, new], the rows' positions
    seen = (key <= at[..., None]) & (nth < counts[:, None])[..., None]
    if case["window"]:
        seen &= (key > at[..., None] - case["window"]) | (key < case["sinks"])
    score.masked_fill_(~seen[:, None, None], float("-inf"))
    score.sub_(score.amax(-1, keepdim=True).clamp_min(-1e30)).exp_()
    out = torch.matmul(score.view(requests, kv, -1, reach), v).view(requests, kv, heads // kv, new, d)
    out = out / score.sum(-1, keepdim=True)
    request = torch.searchsorted(starts[1:].contiguous(), torch.arange(q.shape[0], device=q.device, dtype=torch.int32), right=True)
    nth = torch.arange(q.shape[0], device=q.device) - starts[request]
    return out.permute(0, 3, 1, 2, 4).reshape(requests, new, heads, d)[request, nth].to(q.dtype)


def run(state):
    case = state["case"]
    if own:
        from qtts_amd import ops

        if case["kind"] == "step":
            batch = ops.paged_step(state["new"], state["lengths"], state["table"], state["free"], state["taken"], case["page"],
                                   case["rows"])
            return [batch.starts, batch.counts, batch.lengths, batch.positions, batch.slots, batch.table, batch.taken]
        batch = ops.PagedBatch(state["table"], state["starts"], state["counts"], state["lengths"], state["positions"],
                               state["slots"], case["page"], max_new=state["max_new"], min_new=state["min_new"])
        if case["kind"] == "cache":
            rope = (state["cos"], state["sin"]) if case["rope"] else None
            q = ops.qkv_to_cache(state["qkv"], state["k"], state["v"], batch, case["heads"], state.get("q_norm"),
                                 state.get("k_norm"), EPS, rope)
            return [q, state["k"], state["v"]]
        return [ops.paged_attention(state["q"], state["k"], state["v"], batch, window=case["window"], sinks=case["sinks"])]
    if case["kind"] == "step":
        return _plain_step(state)
    return _plain_cache(state) if case["kind"] == "cache" else [_plain_attention(state)]


# ---- what a pass cannot do without ---------------------------------------------------------


def _visible(case, held, new):
    """Pairs of a query and a key that it sees, and keys that some query sees, over all requests."""
    pairs = keys = 0
    window, sinks = case["window"], case["sinks"]
    for a, b in zip(held, new):
        if not window:
            pairs += b * a + b * (b + 1) // 2
            keys += a + b
            continue
        for p in range(a, a + b):
            low = max(0, p - window + 1)
            pairs += p + 1 - low + min(sinks, low)
        low = max(0, a - window + 1)
        keys += a + b - low + min(sinks, low)
    return pairs, keys


def work(case):
    held, new = _lengths(case, 1)  # another seed has them in another order
    requests, page = case["requests"], case["page"]
    if case["kind"] == "step":
        fresh = sum(-(-(a + b) // page) - -(-a // page) for a, b in zip(held, new))
        return {"bytes": 4 * (4 * requests + 2 * fresh + 2 * case["rows"]), "flops": 0}
    heads, kv, d = case["heads"], case["kv_heads"], case["head_dim"]
    if case["kind"] == "cache":
        live = min(case["rows"], sum(new))
        return {"bytes": live * 4 * (heads + 2 * kv) * d + 8 * live + (4 * live * d if case["rope"] else 0),
                "flops": live * (heads + kv) * d * 8}
    pairs, keys = _visible(case, held, new)
    return {"bytes": 4 * keys * kv * d + 4 * sum(new) * heads * d, "flops": 4 * pairs * heads * d}


# ---- the same in 64 bits -------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "step":
        return None  # whole numbers
    page, d, kv, heads = case["page"], case["head_dim"], case["kv_heads"], case["heads"]
    if case["kind"] == "cache":
        slot = s["slots"].cpu().tolist()
        x = s["qkv"].double().view(len(slot), heads + 2 * kv, d)
        q, k, v = x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:]
        if case["norm"]:
            q, k = ((h / ((h * h).sum(2, keepdim=True) / d + EPS) ** 0.5) * s[w].double()
                    for h, w in ((q, "q_norm"), (k, "k_norm")))
        if case["rope"]:
            at = s["positions"].long().clamp(0)
            turn = torch.complex(s["cos"].double()[at], s["sin"].double()[at])[:, None]  # as complex numbers
            turned = [torch.complex(h[..., :d // 2].contiguous(), h[..., d // 2:].contiguous()) * turn for h in (q, k)]
            q, k = (torch.cat([z.real, z.imag], 2) for z in turned)
        keys, values = s["k"].double(), s["v"].double()
        q = q.clone()
        for t, at in enumerate(slot):
            if at < 0:
                q[t] = 0
            else:
                keys[at // page, :, at % page] = k[t]
                values[at // page, :, :, at % page] = v[t]
        return [q, keys, values]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for r in range(case["requests"]):
        length, count, start = int(s["lengths"][r]), int(s["counts"][r]), int(s["starts"][r])
        held = s["table"][r, :-(-length // page)].long()
        for h in range(kv):
            k = s["k"][held, h].double().reshape(-1, d)[:length]
            v = s["v"][held, h].double().transpose(1, 2).reshape(-1, d)[:length]
            for lo in range(0, count, 4096):
                hi = min(count, lo + 4096)
                at = torch.arange(length - count + lo, length - count + hi, device="cuda")[:, None]
                key = torch.arange(length, device="cuda")[None]
                hidden = key > at
                if case["window"]:
                    hidden |= (key <= at - case["window"]) & (key >= case["sinks"])
                for g in range(heads // kv):
                    q = s["q"][start + lo:start + hi, h * (heads // kv) + g].double()
                    p = torch.softmax((q @ k.t() / d ** 0.5).masked_fill(hidden, -torch.inf), 1)
                    out[start + lo:start + hi, h * (heads // kv) + g] = p @ v
    return [out]
