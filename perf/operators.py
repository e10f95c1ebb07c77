"""The operators around the quantized linears, as timed cases: each in its plain form and as the
framework's own call.

* ``norm``  residual addition, RMSNorm and the per-token 8-bit codes that a W8A8 linear multiplies;
* ``silu``  GatedMLP's activation straight to the per-token codes of a W8A8 down projection;
* ``lora``  low-rank adapters of many requests at once, added to a shared projection's output (one
            projection, or the four of a decoder layer under one routing of the rows).

The hidden, qkv and MLP widths are the talker's (hidden 2048, qkv 2048 + 1024 + 1024, MLP 6144) or the
predictor's (hidden 1024), which bench.py and the tests use; ``draw`` adds ragged ones.  e4m3 codes are
returned as they are, int8 codes as the values they stand for.
"""

import os
import random
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "tts-inference_amd"))

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
LIMIT = {"fp8": 448.0, "int8": 127.0}
EPS = 1e-6
FLOOR = 1e-6  # the least row maximum that a scale is made from
#: output partitions and input width of a decoder layer's linears
PROJECTIONS = {"qkv": ((2048, 1024, 1024), 2048), "o": ((2048,), 2048), "gate_up": ((6144, 6144), 2048),
               "down": ((2048,), 6144)}


def listed():
    return [
        # One stream's decode step into a W8A8 projection: latency alone counts.
        {"name": "norm_fp8_1row", "kind": "norm", "rows": 1, "k": 2048, "dtype": "bf16", "codes": "fp8",
         "residual": True, "normed": False},
        # A busy server's step of the predictor, with the 16-bit rows that its adapters read.
        {"name": "norm_int8_27rows", "kind": "norm", "rows": 27, "k": 1024, "dtype": "bf16", "codes": "int8",
         "residual": True, "normed": True},
        # A prompt of odd length in fp16, the first layer's norm (nothing to add yet).
        {"name": "norm_fp8_1003rows", "kind": "norm", "rows": 1003, "k": 2048, "dtype": "fp16", "codes": "fp8",
         "residual": False, "normed": False},
        # Many long prompts at once, rows of twice the width: bandwidth.
        {"name": "norm_fp8_8192rows", "kind": "norm", "rows": 8192, "k": 4096, "dtype": "bf16", "codes": "fp8",
         "residual": True, "normed": False},
        # A few streams' MLP between two W8A8 linears.
        {"name": "silu_fp8_5rows", "kind": "silu", "rows": 5, "k": 6144, "dtype": "bf16", "codes": "fp8", "act": False},
        # Prompts through the int8 method, an odd number of rows.
        {"name": "silu_int8_1501rows", "kind": "silu", "rows": 1501, "k": 6144, "dtype": "bf16", "codes": "int8",
         "act": False},
        # The largest prompt batch, with the 16-bit rows that down_proj's adapters read.
        {"name": "silu_fp8_4096rows", "kind": "silu", "rows": 4096, "k": 6144, "dtype": "fp16", "codes": "fp8",
         "act": True},
        # One request with one small adapter: the smallest call, latency alone.
        {"name": "lora_o_1row", "kind": "lora", "projection": "o", "rows": 1, "slots": 4, "rank": 16, "dtype": "bf16",
         "prompts": 0},
        # A decode step of 27 requests over 9 adapters, in the order in which they came, all four projections.
        {"name": "lora_layer_27rows", "kind": "lora", "projection": "layer", "rows": 27, "slots": 9, "rank": 16,
         "dtype": "bf16", "prompts": 0},
        # A full decode batch over many large adapters: the adapters' own bytes bound it.
        {"name": "lora_gate_up_64rows", "kind": "lora", "projection": "gate_up", "rows": 64, "slots": 32, "rank": 64,
         "dtype": "bf16", "prompts": 0},
        # Five prompts of ragged lengths in fp16, the widest input.
        {"name": "lora_down_1003rows", "kind": "lora", "projection": "down", "rows": 1003, "slots": 5, "rank": 32,
         "dtype": "fp16", "prompts": 5},
        # Many prompts through all four projections: the output's rows bound it.
        {"name": "lora_layer_2048rows", "kind": "lora", "projection": "layer", "rows": 2048, "slots": 8, "rank": 16,
         "dtype": "bf16", "prompts": 11},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    kind = rng.choice(["norm", "silu", "lora", "lora"])
    if kind == "lora":
        rows = _log(rng, 1, 2048)
        return {"kind": kind, "projection": rng.choice(["qkv", "o", "gate_up", "down", "layer", "free"]), "rows": rows,
                "slots": _log(rng, 1, 32), "rank": rng.choice([4, 8, 16, 16, 24, 32, 64]),
                "dtype": rng.choice(["bf16", "bf16", "fp16"]), "prompts": 0 if rows <= 64 else rng.randint(0, 20),
                "n": 8 * _log(rng, 8, 800), "k": 8 * _log(rng, 8, 800)}
    k = _log(rng, 33, 8192)
    case = {"kind": kind, "rows": min(_log(rng, 1, 8192), (8192 * 4096 if kind == "norm" else 4096 * 6144) // k),
            "k": k if rng.random() < 0.3 else k // 8 * 8,
            "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "codes": rng.choice(["fp8", "int8"])}
    if kind == "norm":
        return dict(case, residual=rng.random() < 0.7, normed=rng.random() < 0.3)
    return dict(case, act=rng.random() < 0.3)


# ---- inputs --------------------------------------------------------------------------------


def _randn(seed, index, *shape):
    g = torch.Generator(device="cuda").manual_seed(seed * 1000 + index)
    return torch.randn(*shape, generator=g, device="cuda")


def _shapes(case):
    """(output partitions, input width) of the projections that a lora case passes through."""
    if case["projection"] == "free":
        return [((case["n"],), case["k"])]
    names = PROJECTIONS if case["projection"] == "layer" else (case["projection"],)
    return [PROJECTIONS[name] for name in names]


def _routing(case, seed):
    """The adapter slot of each row (-1: none) and each slot's rank: one request a row in decode, runs of rows of
    ragged lengths where there are prompts; about one request in eight has no adapter."""
    rng = random.Random(seed)
    pick = lambda: -1 if rng.random() < 0.125 else rng.randrange(case["slots"])  # noqa: E731
    rows, prompts = case["rows"], case["prompts"]
    if prompts:
        cuts = [0, *sorted(rng.randint(0, rows) for _ in range(prompts - 1)), rows]
        index = [s for lo, hi in zip(cuts, cuts[1:]) for s in [pick()] * (hi - lo)]
    else:
        index = [pick() for _ in range(rows)]
    index[0] = max(index[0], 0)
    ranks = [rng.choice([case["rank"], case["rank"], max(1, case["rank"] // 2)]) for _ in range(case["slots"])]
    return index, ranks


def prepare(case, seed):
    case, dtype = dict(case), DTYPES[case["dtype"]]
    state = {"case": case}
    if case["kind"] == "lora":
        index, ranks = _routing(case, seed)
        state["index"] = torch.tensor(index, dtype=torch.int32).cuda()
        state["ranks"] = torch.tensor(ranks, dtype=torch.int32).cuda()
        state["scaling"] = _randn(seed, 0, case["slots"]).abs() + 0.5
        state["calls"] = []
        for i, (parts, k) in enumerate(_shapes(case)):
            state["calls"].append({
                "parts": list(parts),
                "base": _randn(seed, 10 * i + 1, case["rows"], sum(parts)).to(dtype),
                "x": _randn(seed, 10 * i + 2, case["rows"], k).to(dtype),
                "a": (_randn(seed, 10 * i + 3, case["slots"], len(parts) * case["rank"], k) / k ** 0.5).to(dtype),
                "b": (_randn(seed, 10 * i + 4, case["slots"], sum(parts), case["rank"]) * 0.1).to(dtype)})
        return state
    rows, k = case["rows"], case["k"]
    width = 2 * k if case["kind"] == "silu" else k
    x = _randn(seed, 1, rows, width) * (1 + 4 * (_randn(seed, 2, width).abs() > 2.5))  # a few outlier channels
    if rows > 4:
        x[rows - 1] = 0  # a padded row
    state["x"] = x.to(dtype)
    if case["kind"] == "norm":
        state["weight"] = (1 + 0.1 * _randn(seed, 3, k)).to(dtype)
        if case["residual"]:
            residual = 2 * _randn(seed, 4, rows, k)
            if rows > 4:
                residual[rows - 1] = 0
            state["residual"] = residual.to(dtype)
    if case["codes"] == "int8":  # the values of int8 codes are written here
        state["values"] = torch.empty(rows, k, dtype=torch.bfloat16 if case["dtype"] == "fp32" else dtype, device="cuda")
    return state


# ---- a pass --------------------------------------------------------------------------------


def _values(state, q, scale):
    """e4m3 codes as they are; int8 codes as what they stand for."""
    return torch.mul(q, scale.unsqueeze(1), out=state["values"]) if state["case"]["codes"] == "int8" else q


def _codes(case, v):
    """Codes and scales of fp32 rows: the scale is the row's largest magnitude over the code range."""
    scale = v.abs().amax(1).clamp_min(FLOOR) / LIMIT[case["codes"]]
    q = v / scale.unsqueeze(1)
    if case["codes"] == "int8":
        return q.round_().clamp_(-127.0, 127.0), scale
    return q.to(torch.float8_e4m3fn), scale


def _plain_norm(state):
    case, h, hidden = state["case"], state["x"], None
    if case["residual"]:
        h = hidden = (h.float() + state["residual"].float()).to(h.dtype)
    f = h.float()
    v = f * torch.rsqrt(f.square().mean(1, keepdim=True) + EPS) * state["weight"].float()
    q, scale = _codes(case, v)
    return [_values(state, q, scale), scale, hidden, v.to(h.dtype) if case["normed"] else None]


def _plain_silu(state):
    case = state["case"]
    gate, up = state["x"].float().split(case["k"], 1)
    v = gate / (1.0 + torch.exp(-gate)) * up
    q, scale = _codes(case, v)
    return [_values(state, q, scale), scale, v.to(state["x"].dtype) if case["act"] else None]


def _plain_lora(state, call):
    """Every row against every adapter, its own kept, then one product over all (adapter, rank) pairs a partition."""
    rows, slots = call["x"].shape[0], state["case"]["slots"]
    parts, rank = call["parts"], state["case"]["rank"]
    t = (call["x"].float() @ call["a"].float().reshape(-1, call["x"].shape[1]).t()).view(rows, slots, len(parts), rank)
    mine = state["index"].unsqueeze(1) == torch.arange(slots, device="cuda")
    live = torch.arange(rank, device="cuda") < state["ranks"].unsqueeze(1)
    keep = mine[:, :, None, None] & live[None, :, None, :]
    t = torch.where(keep, t * state["scaling"].view(1, -1, 1, 1), torch.zeros((), device="cuda"))
    columns = call["b"].float().split(parts, 1)
    delta = [t[:, :, p].reshape(rows, -1) @ b.transpose(1, 2).reshape(slots * rank, -1) for p, b in enumerate(columns)]
    return (call["base"].float() + torch.cat(delta, 1)).to(call["base"].dtype)


def run(state):
    case = state["case"]
    if own:
        from qtts_amd import ops

        if case["kind"] == "lora":
            batch = ops.lora_batch(state["index"], case["slots"])
            return [ops.lora_add(c["base"], c["x"], batch, c["a"], c["b"], state["scaling"], state["ranks"], c["parts"])
                    for c in state["calls"]]
        codes = ops.CODE_INT8 if case["codes"] == "int8" else ops.CODE_E4M3
        if case["kind"] == "norm":
            q, scale, *more = ops.rms_norm_quant(state["x"], state["weight"], EPS, state.get("residual"), codes,
                                                 want_normed=case["normed"])
        else:
            q, scale, *more = ops.silu_mul_quant(state["x"], codes, want_act=case["act"])
        return [_values(state, q, scale), scale, *more]
    if case["kind"] == "lora":
        return [_plain_lora(state, c) for c in state["calls"]]
    return _plain_norm(state) if case["kind"] == "norm" else _plain_silu(state)


# ---- what a pass cannot do without ---------------------------------------------------------


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "lora":
        index, ranks = _routing(case, 1)  # another seed routes alike
        used = {s for s in index if s >= 0}
        mean = sum(ranks[s] for s in used) / len(used)
        live = sum(s >= 0 for s in index)
        out = {"bytes": 4 * case["rows"], "flops": 0}
        for parts, k in _shapes(case):
            n = sum(parts)
            out["bytes"] += size * (live * k + 2 * case["rows"] * n + len(used) * mean * (len(parts) * k + n))
            out["flops"] += 2 * live * mean * (len(parts) * k + n)
        return out
    rows, k = case["rows"], case["k"]
    if case["kind"] == "norm":
        moved = rows * k * size * (1 + 2 * case["residual"] + case["normed"]) + k * size
        return {"bytes": moved + rows * (k + 4), "flops": 6 * rows * k}
    return {"bytes": rows * k * size * (2 + case["act"]) + rows * (k + 4), "flops": 8 * rows * k}


# ---- the same in 64 bits -------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "lora":
        outs = []
        for c in s["calls"]:
            y, ends = c["base"].double(), [sum(c["parts"][:i + 1]) for i in range(len(c["parts"]))]
            for slot in range(case["slots"]):
                rows = (s["index"] == slot).nonzero().flatten()
                r, scale = int(s["ranks"][slot]), float(s["scaling"][slot])
                for p, (hi, width) in enumerate(zip(ends, c["parts"])):
                    down = c["a"][slot, p * case["rank"]:p * case["rank"] + r].double()
                    up = c["b"][slot, hi - width:hi, :r].double()
                    y[rows, hi - width:hi] += scale * (c["x"][rows].double() @ down.t() @ up.t())
            outs.append(y)
        return outs
    if case["kind"] == "norm":
        h, hidden = s["x"].double(), None
        if case["residual"]:  # the sum is kept in the activations' type
            hidden = h + s["residual"].double()
            h = hidden.to(s["x"].dtype).double()
        v = h / (h.pow(2).sum(1, keepdim=True) / case["k"] + EPS).sqrt() * s["weight"].double()
        more = [hidden, v if case["normed"] else None]
    else:
        gate, up = s["x"][:, :case["k"]].double(), s["x"][:, case["k"]:].double()
        v = gate * torch.sigmoid(gate) * up
        more = [v if case["act"] else None]
    scale = torch.maximum(v.abs().max(1).values, torch.tensor(FLOOR, dtype=torch.float64, device="cuda")) / LIMIT[case["codes"]]
    q = v / scale[:, None]
    return [q if case["codes"] == "fp8" else q.round() * scale[:, None], scale, *more]
