"""Low-rank adapters of many requests beside a shared projection (ops.lora_batch, ops.lora_add) against 64 bits.

Tolerance of an output element, from the arithmetic (u = 2^-24): half a step of the output's type relative to the
result (eps / 2), plus the fp32 sums: K + R products each off by at most u of the sum of their magnitudes, twice
(rounding of the product's addition, and the order), and the first product's result carried to the second as two 16-bit
halves (2^-16 of it in bf16, the coarser of the two types)."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.fixture(scope="module")
def ops():
    from qtts_amd import ops as _ops
    assert _ops.device_supported(), "GPU is not a gfx950"
    _ops.reserve_workspace(torch.device("cuda"), 64 << 20)
    return _ops


def _rand(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _case(m, k, parts, slots, rank, dtype, seed, index=None, mixed=True):
    n = sum(parts)
    g = torch.Generator().manual_seed(seed)
    if index is None:
        index = torch.randint(-1, slots, (m,), generator=g, dtype=torch.int32)
    ranks = torch.randint(0, rank + 1, (slots,), generator=g, dtype=torch.int32) if mixed else None
    if ranks is not None and slots > 1:
        ranks[0] = rank
    return {"base": _rand((m, n), dtype, seed), "x": _rand((m, k), dtype, seed + 1), "index": index.cuda(),
            "a": _rand((slots, len(parts) * rank, k), dtype, seed + 2, max(k, 1) ** -0.5),
            "b": _rand((slots, n, rank), dtype, seed + 3, 0.2), "scaling": _rand((slots,), torch.float32, seed + 4) + 2,
            "ranks": None if ranks is None else ranks.cuda(), "parts": parts, "slots": slots, "rank": rank}


def _exact(c):
    """(result, error bound without the output's rounding), in 64 bits on the CPU."""
    y = c["base"].double().cpu()
    bound = y.abs() * U
    x, index, rank = c["x"].double().cpu(), c["index"].cpu(), c["rank"]
    lo = 0
    for p, width in enumerate(c["parts"]):
        for s in range(c["slots"]):
            rows = (index == s).nonzero().flatten()
            r = rank if c["ranks"] is None else int(c["ranks"][s].clamp(0, rank))
            if not len(rows) or not r:
                continue
            a = c["a"][s, p * rank:p * rank + r].double().cpu()
            b = c["b"][s, lo:lo + width, :r].double().cpu()
            scale = float(c["scaling"][s])
            y[rows, lo:lo + width] += scale * (x[rows] @ a.t() @ b.t())
            mags = abs(scale) * (x[rows].abs() @ a.abs().t() @ b.abs().t())
            carried = abs(scale) * ((x[rows] @ a.t()).abs() @ b.abs().t())
            bound[rows, lo:lo + width] += 2 * (x.shape[1] + r + 8) * U * mags + 2.0 ** -16 * carried
        lo += width
    return y, bound


def _check(out, c, what=""):
    y, bound = _exact(c)
    tiny = torch.finfo(out.dtype).smallest_normal * torch.finfo(out.dtype).eps / 2
    err = (out.double().cpu() - y).abs()
    ok = err <= bound + torch.finfo(out.dtype).eps / 2 * (y.abs() + bound) + tiny
    assert ok.all(), f"{what}: {int((~ok).sum())} of {ok.numel()} off, first at {(~ok).nonzero()[0].tolist()}"
    none = ((c["index"] < 0) | (c["index"] >= c["slots"])).nonzero().flatten()
    assert torch.equal(out[none], c["base"][none]), f"{what}: a row without an adapter changed"


def _run(ops, c, out=None):
    return ops.lora_add(c["base"], c["x"], ops.lora_batch(c["index"], c["slots"]), c["a"], c["b"], c["scaling"], c["ranks"],
                        c["parts"], out=out)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("m,k,parts,slots,rank", [
    (1, 2048, [2048], 4, 16), (1, 64, [64], 1, 8), (2, 1024, [2048, 1024, 1024], 3, 16), (16, 256, [512], 1, 16),
    (17, 256, [520], 1, 32), (27, 2048, [2048, 1024, 1024], 9, 16), (33, 128, [64, 72], 40, 24), (64, 512, [640], 32, 64),
    (65, 512, [640], 3, 16), (130, 256, [256, 256], 7, 128), (200, 96, [136], 150, 8), (1003, 64, [48], 5, 16),
    (64, 64, [64], 1, 128), (300, 2048, [80], 2, 40)])
def test_lora(ops, m, k, parts, slots, rank, dtype):
    for mixed in (True, False):
        c = _case(m, k, parts, slots, rank, dtype, seed=m + k + rank, mixed=mixed)
        _check(_run(ops, c), c, f"{m}x{k} parts {parts} slots {slots} rank {rank} {dtype}")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("rank", [8, 16, 24, 40, 64, 72, 100])
@pytest.mark.parametrize("m,parts,slots", [(2061, [4096, 4104], 3), (1100, [8000], 30), (66, [520, 24], 40)])
def test_wide_outputs(ops, m, parts, slots, rank, dtype):
    """The second product's 256, 128 and 64 columns a workgroup, with whole and broken tiles of rows."""
    c = _case(m, 64, parts, slots, rank, dtype, seed=m + rank)
    _check(_run(ops, c), c, f"{m} rows parts {parts} rank {rank} {dtype}")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("rank", [1, 2, 3, 4, 5, 7, 9, 12, 15, 17, 20, 31, 33, 50, 63, 65, 90, 100, 127])
def test_ranks_off_eight(ops, rank, dtype):
    """B's rows start anywhere: every slot's last columns, the last slot's among them, with values behind B that are no part of it."""
    for m, k, parts, slots in ((1, 64, [8], 1), (7, 256, [24, 8], 3), (60, 512, [2048, 72], 33), (150, 128, [264, 520], 4)):
        index = torch.arange(m, dtype=torch.int32) % (slots + 1)
        index[index == slots] = slots - 1
        c = _case(m, k, parts, slots, rank, dtype, seed=m + rank, index=index, mixed=False)
        room = torch.full((c["b"].numel() + 64,), float("nan"), dtype=dtype, device="cuda")
        room[:c["b"].numel()] = c["b"].flatten()
        c["b"] = room[:c["b"].numel()].view(c["b"].shape)
        _check(_run(ops, c), c, f"m={m}")
        c["ranks"] = torch.full((slots,), max(1, rank - 1), dtype=torch.int32, device="cuda")
        _check(_run(ops, c), c, f"m={m}, ranks short by one")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("k", [2048, 2056, 2104, 6144])
@pytest.mark.parametrize("m,parts,slots,rank", [
    (60, [4096], 30, 16), (60, [1024], 40, 64), (63, [520, 264], 63, 24), (70, [1024], 3, 8), (300, [520, 264], 4, 40),
    (1003, [1024], 30, 16), (130, [64] * 5, 2, 16)])
def test_long_k_in_parts(ops, m, parts, slots, rank, k, dtype):
    """Few groups and a long K: the first product in two parts of K, which the second adds.  Each part's sum is carried in 2^-17 of
    its own magnitude, which is at most that of all of K's products: within the bound's fp32 term, 2 K u >= 2^-12 of those."""
    c = _case(m, k, parts, slots, rank, dtype, seed=m + k + rank)
    _check(_run(ops, c), c)


@pytest.mark.parametrize("m", [1, 5, 40, 100])
@pytest.mark.parametrize("k,parts,rank", [(33, [17], 3), (65, [40, 1, 23], 4), (100, [13, 64], 12), (8, [8], 1),
                                          (2047, [31], 16), (64, [100], 17), (24, [7], 127), (16, [0, 24, 0], 8)])
def test_odd_sizes(ops, m, k, parts, rank):
    c = _case(m, k, parts, 3, rank, torch.bfloat16, seed=m + k)
    _check(_run(ops, c), c, f"{m}x{k} parts {parts} rank {rank}")


@pytest.mark.parametrize("m", [6, 70])
def test_strides_offsets_and_in_place(ops, m):
    """Rows of wider buffers, starts off 16 bytes, out the base itself, rows of another buffer left alone."""
    k, n = 128, 96
    for off in (0, 8, 1):
        c = _case(m, k, [64, 32], 4, 16, torch.bfloat16, seed=5 + off)
        wide_x = torch.zeros(m, k + 40, dtype=torch.bfloat16, device="cuda")
        wide_b = torch.full((m + 2, n + 48), 7.0, dtype=torch.bfloat16, device="cuda")
        wide_x[:, off:off + k] = c["x"]
        wide_b[1:m + 1, off:off + n] = c["base"]
        view = wide_b[1:m + 1, off:off + n]
        batch = ops.lora_batch(c["index"], 4)
        out = ops.lora_add(view, wide_x[:, off:off + k], batch, c["a"], c["b"], c["scaling"], c["ranks"], c["parts"])
        _check(out, c, f"offset {off}")
        got = ops.lora_add(view, wide_x[:, off:off + k], batch, c["a"], c["b"], c["scaling"], c["ranks"], c["parts"], out=view)
        assert got.data_ptr() == view.data_ptr()
        assert torch.equal(view, out), "in place"
        wide_b[1:m + 1, off:off + n] = 7.0
        assert (wide_b == 7.0).all(), "written outside its rows or columns"
    x3, b3 = c["x"].view(2, m // 2, k), c["base"].view(2, m // 2, n)
    y3 = ops.lora_add(b3, x3, batch, c["a"], c["b"], c["scaling"], c["ranks"], c["parts"])
    assert y3.shape == b3.shape and torch.equal(y3.view(m, n), out)


@pytest.mark.parametrize("m", [3, 64, 90])
def test_routing_edges(ops, m):
    """No row with an adapter, every row with one, one adapter a row, indices out of range, no slots at all."""
    for name, index in {"none": torch.full((m,), -1), "one": torch.full((m,), 2), "each": torch.arange(m) % 7,
                        "range": torch.arange(m) * 1000 - 5, "extremes": torch.tensor([2 ** 31 - 1, -2 ** 31, 0] * 30)[:m],
                        "last": torch.tensor([-1] * (m - 1) + [6])}.items():
        c = _case(m, 64, [48], 7, 16, torch.bfloat16, seed=3, index=index.to(torch.int32))
        _check(_run(ops, c), c, f"{name} {m}")
    e = torch.empty
    kw = dict(dtype=torch.bfloat16, device="cuda")
    out = ops.lora_add(c["base"], c["x"], ops.lora_batch(c["index"], 0), e(0, 16, 64, **kw), e(0, 48, 16, **kw),
                       e(0, device="cuda"))
    assert torch.equal(out, c["base"])


@pytest.mark.parametrize("m", [4, 80])
def test_ranks_hide_what_is_past_them(ops, m):
    """Entries past a slot's rank may hold anything, NaN and infinities among it; so may slots that no row takes,
    and rows without an adapter."""
    c = _case(m, 64, [32, 40], 5, 24, torch.float16, seed=9, mixed=False)
    c["index"] = (torch.arange(m) % 4 - 1).to(torch.int32).cuda()
    c["ranks"] = torch.tensor([5, 0, 24, 3, 9], dtype=torch.int32).cuda()
    want = _run(ops, c)
    _check(want, c)
    for s, r in enumerate(c["ranks"].tolist()):
        c["b"][s, :, r:] = float("nan")
        c["a"][s].view(2, 24, 64)[:, r:] = float("inf")
    c["a"][3:] = float("nan")
    c["b"][3:] = float("inf")
    c["scaling"][3:] = float("nan")
    c["x"][c["index"] < 0] = float("nan")
    got = _run(ops, c)
    assert torch.equal(got, want)
    c["ranks"] = torch.tensor([5, -3, 99, 3, 9], dtype=torch.int32).cuda()  # taken into 0..rank
    assert torch.isfinite(_run(ops, c)).all()


@pytest.mark.parametrize("m", [6, 100])
def test_values_stay_in_their_rows(ops, m):
    """NaN and infinity in one row's activations reach that row alone."""
    c = _case(m, 128, [64], 3, 16, torch.bfloat16, seed=21, index=torch.zeros(m, dtype=torch.int32), mixed=False)
    want = _run(ops, c)
    c["x"][2, 5] = float("nan")
    c["x"][4, 0] = float("inf")
    got = _run(ops, c)
    rest = [r for r in range(m) if r not in (2, 4)]
    assert torch.equal(got[rest], want[rest]) and torch.isnan(got[2]).all() and not torch.isfinite(got[4]).any()


def test_fp16_range(ops):
    """The first product's sums may pass fp16's range (65504): they are kept in fp32 or scaled."""
    c = _case(5, 512, [64], 2, 16, torch.float16, seed=23, mixed=False, index=torch.tensor([0, 1, 0, -1, 1], dtype=torch.int32))
    c["x"] *= 1000
    c["a"] *= 500
    c["b"] *= 1e-5
    _check(_run(ops, c), c)
    c["x"] *= 1e-6  # and far below its smallest normal
    c["a"] *= 1e-5
    c["b"] = (c["b"].float() * 1e5).half()
    _check(_run(ops, c), c)


@pytest.mark.parametrize("m", [1, 48, 100])
def test_graph_follows_the_index(ops, m):
    """A captured call reads index, activations and adapters anew on every replay, whatever ran in between."""
    c = _case(m, 256, [128, 64], 6, 16, torch.bfloat16, seed=31)
    other = _case(70, 256, [512], 2, 32, torch.bfloat16, seed=32)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _run(ops, c)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        batch = ops.lora_batch(c["index"], 6)
        out = ops.lora_add(c["base"], c["x"], batch, c["a"], c["b"], c["scaling"], c["ranks"], c["parts"])
        again = ops.lora_add(out, c["x"], batch, c["a"], c["b"], c["scaling"], c["ranks"], c["parts"])
    for i in range(3):
        fresh = _case(m, 256, [128, 64], 6, 16, torch.bfloat16, seed=40 + i)
        for key in ("index", "x", "base", "a", "ranks"):
            c[key].copy_(fresh[key])
        graph.replay()
        _check(_run(ops, other), other, "eager between")
        torch.cuda.synchronize()
        want = _run(ops, c)
        assert torch.equal(out, want), f"replay {i}"
        assert torch.equal(again, _run(ops, dict(c, base=want))), f"replay {i}"
        _check(out, c, f"replay {i}")


@pytest.mark.parametrize("m,slots", [(65, 1), (100, 3), (1000, 7), (4097, 768), (5000, 40), (70000, 500), (64 * 1024, 1)])
def test_plan(ops, m, slots):
    """The plan holds every row once, stably sorted by slot, in groups of at most 16 rows of one slot."""
    g = torch.Generator().manual_seed(m)
    index = torch.randint(-2, slots + 1, (m,), generator=g, dtype=torch.int32)
    plan = ops.lora_batch(index.cuda(), slots).plan.cpu()
    slot = torch.where((index < 0) | (index >= slots), slots, index)
    want = torch.argsort(slot, stable=True)
    count = int(plan[0])
    most = (m + 15) // 16 + min(m, slots + 1)
    groups = plan[4:4 + 2 * count].view(-1, 2)
    order = plan[4 + (2 * most + 3) // 4 * 4:][:16 * count].view(-1, 16)
    assert plan[1] == m and plan[2] == slots
    at = 0
    for (s, n), rows in zip(groups.tolist(), order):
        assert 0 < n <= 16 and torch.equal(rows[:n].long(), want[at:at + n])
        here = slots if s < 0 else s
        assert (slot[want[at:at + n]] == here).all()
        at += n
        assert n == 16 or at == m or slot[want[at]] != here
    assert at == m


def test_many_adapters(ops):
    """Past the slots that a plan takes, and past 64 rows, the rows are grouped window by window."""
    c = _case(150, 64, [40, 24], 900, 16, torch.bfloat16, seed=61)
    assert ops.lora_batch(c["index"], 900).plan is None
    _check(_run(ops, c), c)
    c["index"] = (torch.arange(150) % 2 * 800).to(torch.int32).cuda()
    _check(_run(ops, c), c)


def test_a_plan_of_another_batch_writes_nothing(ops):
    c = _case(100, 64, [40], 5, 16, torch.bfloat16, seed=62)
    plan = ops.lora_plan_buffer(100, 5, c["x"].device)
    batch = ops.lora_batch(c["index"], 5, plan)
    ops.lora_batch(c["index"][:90].contiguous(), 5, plan)  # the buffer now holds another batch's
    out = torch.full((100, 40), 3.0, dtype=torch.bfloat16, device="cuda")
    ops.lora_add(c["base"], c["x"], batch, c["a"], c["b"], c["scaling"], c["ranks"], c["parts"], out=out)
    assert (out == 3.0).all()
    ops.lora_batch(c["index"], 5, plan)
    _check(ops.lora_add(c["base"], c["x"], batch, c["a"], c["b"], c["scaling"], c["ranks"], c["parts"]), c)
    for bad in (plan[:100], plan.long(), plan.cpu(), plan[::2]):  # too short for the rows, or no plan buffer here
        with pytest.raises(ValueError, match="plan must hold"):
            ops.lora_batch(c["index"], 5, bad)
        with pytest.raises(ValueError, match="plan must hold"):
            torch.ops.qtts.lora_add(c["base"], c["x"], c["index"], bad, 5, c["a"], c["b"], c["scaling"], c["ranks"], c["parts"])


def test_repeats_give_the_same_bits(ops):
    for m in (30, 500):
        c = _case(m, 1024, [512], 8, 16, torch.bfloat16, seed=51)
        first = _run(ops, c)
        for _ in range(3):
            assert torch.equal(_run(ops, c), first)


def test_a_row_does_not_depend_on_its_batch(ops):
    """Within one kernel's range, a row's result is the same bits alone among others or in another order."""
    c = _case(40, 512, [256], 5, 16, torch.bfloat16, seed=53)
    want = _run(ops, c)
    perm = torch.randperm(40, generator=torch.Generator().manual_seed(1)).cuda()
    d = dict(c, x=c["x"][perm], base=c["base"][perm], index=c["index"][perm])
    assert torch.equal(_run(ops, d), want[perm])


def test_first_calls_of_a_process(ops, monkeypatch):
    """Without a workspace yet: a call of no rows or no columns needs none, any other reserves its own."""
    monkeypatch.setattr(ops, "_workspaces", {})
    for shape in ((0, 40), (2, 0, 40), (3, 0)):
        base = torch.empty(shape, dtype=torch.bfloat16, device="cuda")
        m, n = base.numel() // shape[-1] if shape[-1] else 3, shape[-1]
        batch = ops.lora_batch(torch.zeros(m, dtype=torch.int32, device="cuda"), 2)
        a, b = (torch.zeros(2, *s, dtype=torch.bfloat16, device="cuda") for s in ((8, 64), (n, 8)))
        x = torch.zeros((*shape[:-1], 64), dtype=torch.bfloat16, device="cuda")
        y = ops.lora_add(base, x, batch, a, b, torch.ones(2, device="cuda"))
        assert y.shape == base.shape and not ops._workspaces
        assert ops.lora_add(base, x, batch, a, b, torch.ones(2, device="cuda"), out=base) is base
    c = _case(5, 64, [40], 2, 8, torch.bfloat16, seed=71)
    _check(_run(ops, c), c)
    assert len(ops._workspaces) == 1


@pytest.mark.parametrize("m", [6, 70])
@pytest.mark.parametrize("k,parts,slots,rank", [(4096, [64] * 8, 540, 128), (64, [65536], 300, 128)], ids=["a", "b"])
def test_adapters_past_32_bits(ops, k, parts, slots, rank, m):
    """Adapters whose bytes pass 2^32: rows of the first slots, the last and those on either side of that offset."""
    n = sum(parts)
    shapes = (slots, len(parts) * rank, k), (slots, n, rank)
    used = sorted({0, 1, slots - 1} | {min(slots - 1, (1 << sh) // (2 * s[1] * s[2]) + d) for s in shapes for sh in (31, 32)
                                       for d in (0, 1)})
    a, b = (torch.empty(s, dtype=torch.bfloat16, device="cuda") for s in shapes)
    assert max(a.numel(), b.numel()) * 2 > 1 << 32
    for i, slot in enumerate(used):
        a[slot], b[slot] = _rand(shapes[0][1:], torch.bfloat16, i, k ** -0.5), _rand(shapes[1][1:], torch.bfloat16, 50 + i, 0.2)
    index = torch.tensor([used[i % len(used)] for i in range(m)], dtype=torch.int32)
    c = {"base": _rand((m, n), torch.bfloat16, 1), "x": _rand((m, k), torch.bfloat16, 2), "index": index.cuda(), "a": a, "b": b,
         "scaling": torch.full((slots,), 0.5, device="cuda"), "ranks": None, "parts": parts, "slots": slots, "rank": rank}
    _check(_run(ops, c), c)


@pytest.mark.parametrize("m", [50, 70])
def test_rows_past_32_bits(ops, m):
    """x, base and out with rows so far apart that their offsets pass 2^32 elements' bytes; what lies between stays as it was."""
    pitch = (1 << 26) + 8
    wide = [torch.empty((m - 1) * pitch + 64, dtype=torch.bfloat16, device="cuda") for _ in range(3)]
    x, base, out = (w.as_strided((m, 64), (pitch, 1)) for w in wide)
    c = _case(m, 64, [40, 24], 5, 16, torch.bfloat16, seed=81)
    x.copy_(c["x"]), base.copy_(c["base"])
    edges = wide[2].as_strided((m - 1, 64), (pitch, 1), 64)
    edges.fill_(3.0)
    ops.lora_add(base, x, ops.lora_batch(c["index"], 5), c["a"], c["b"], c["scaling"], c["ranks"], c["parts"], out=out)
    _check(out.contiguous(), c)
    assert (edges == 3.0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("m,k,parts,slots,rank", [(100, 64, [40], 5, 16), (1003, 128, [64, 72], 1, 24), (70, 2048, [264], 30, 16),
                                                  (3000, 64, [520, 16], 2, 64), (130, 96, [136], 150, 100), (300, 33, [17, 4], 6, 3)])
def test_a_fresh_output_is_whole_whatever_the_plan(ops, m, k, parts, slots, rank, dtype):
    """With a plan of another batch a fresh output has every row, by the index, also through the custom op and a captured call."""
    c = _case(m, k, parts, slots, rank, dtype, seed=m + rank)
    index, n = c["index"], sum(parts)
    plan = ops.lora_plan_buffer(m + 64, max(slots, 2), index.device)
    batch = ops.lora_batch(index, slots, plan)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = ops.lora_add(c["base"], c["x"], batch, c["a"], c["b"], c["scaling"], c["ranks"], c["parts"])
    for rows, of in ((m - 5, slots), (m + 33, slots), (m, 1 if slots > 1 else 2)):
        other = torch.zeros(rows, dtype=torch.int32, device="cuda")
        ops.lora_batch(other, of, plan)  # the buffer now holds another batch's
        torch.full((m, n), float("nan"), dtype=dtype, device="cuda")  # what torch.empty finds
        _check(ops.lora_add(c["base"], c["x"], batch, c["a"], c["b"], c["scaling"], c["ranks"], c["parts"]), c, f"plan of {rows}, {of}")
        torch.full((m, n), float("nan"), dtype=dtype, device="cuda")
        _check(torch.ops.qtts.lora_add(c["base"], c["x"], index, plan, slots, c["a"], c["b"], c["scaling"], c["ranks"], c["parts"]), c)
        held.fill_(float("nan"))
        graph.replay()
        _check(held, c, f"replay with a plan of {rows}, {of}")
    ops.lora_batch(index, slots, plan)
    graph.replay()
    assert torch.equal(held, ops.lora_add(c["base"], c["x"], batch, c["a"], c["b"], c["scaling"], c["ranks"], c["parts"]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("cancels", ["entries", "halves"])
@pytest.mark.parametrize("m,k,parts,slots,rank", [
    (1, 2048, [512], 2, 16), (16, 64, [72], 1, 8), (27, 2048, [256, 128, 128], 9, 16), (16, 2048, [512], 4, 32), (8, 2048, [264], 3, 64),
    (60, 2048, [512], 30, 16), (63, 6144, [264], 40, 24), (64, 6144, [520], 64, 64), (64, 1024, [136], 64, 100), (70, 2048, [264], 3, 8),
    (300, 6144, [520, 264], 4, 40), (300, 2048, [520], 4, 64), (1003, 6144, [72], 30, 16), (2100, 2048, [520], 8, 32), (130, 512, [264], 7, 128),
    (5000, 64, [4096], 5, 72), (40, 1003, [17, 40], 3, 12), (200, 333, [41], 5, 36), (100, 2040, [64], 2, 7)])
def test_what_cancels_is_exact(ops, m, k, parts, slots, rank, cancels, dtype):
    """The first product's sums keep fp32's 24 bits to the second: whole numbers of up to 2^21 whose terms cancel to fewer than 2^8,
    between neighbouring entries of the rank or between the two halves of K.  Every product, every partial sum in any order (8 terms of
    2^21, below 2^24) and the result are whole numbers that fp32, and the output's type, hold exactly, so the result is exact too."""
    g = torch.Generator().manual_seed(m + k + rank)
    most = max(1, min(200, (1 << 20) // (k * 100)))

    def whole(lo, hi, *shape):
        return torch.randint(lo, hi + 1, shape, generator=g).double()

    n, pairs = sum(parts), rank // 2
    x = whole(1, most, m, k)
    if cancels == "entries":  # rows of A in pairs that differ by one in a few places, B + and - of them
        a = whole(40, 200, slots, len(parts) * rank, k)
        for p in range(len(parts)):
            even = a[:, p * rank:p * rank + 2 * pairs:2]
            a[:, p * rank + 1:p * rank + 2 * pairs:2] = even + (torch.arange(k) == 0).double() - (torch.arange(k) == k - 1).double()
        b = torch.zeros(slots, n, rank, dtype=torch.float64)
        used = torch.randperm(pairs, generator=g)[:4]
        sign = whole(0, 1, slots, n, len(used)) * 2 - 1
        b[:, :, 2 * used], b[:, :, 2 * used + 1] = sign, -sign
        if most > 40:  # four of x's first and last, within 2^8
            x[:, 0], x[:, -1] = x[:, 0] % 20, x[:, -1] % 20
    else:  # the second half of K takes the first away, but for one place
        half = k // 2
        a = whole(40, 200, slots, len(parts) * rank, k)
        a[:, :, half:2 * half], x[:, half:2 * half] = -a[:, :, :half], x[:, :half]
        a[:, :, k - 1] = a[:, :, k - 1] + 1 if k % 2 == 0 else 1
        if most > 40:
            x[:, k - 1] = x[:, k - 1] % 30
            x[:, half - 1] = x[:, k - 1] if k % 2 == 0 else x[:, half - 1]
        b = torch.zeros(slots, n, rank, dtype=torch.float64)
        used = torch.randperm(rank, generator=g)[:2]
        b[:, :, used] = whole(0, 1, slots, n, len(used)) * 2 - 1
    base = whole(-20, 20, m, n)
    index = torch.randint(-1, slots, (m,), generator=g, dtype=torch.int32)
    scaling = whole(0, 1, slots) * 2 - 1
    want, lo = base.clone(), 0
    for p, width in enumerate(parts):
        for s in range(slots):
            rows = (index == s).nonzero().flatten()
            t = x[rows] @ a[s, p * rank:(p + 1) * rank].t()
            assert t.numel() == 0 or (t.abs().max() < 1 << 21 and (x[rows].abs() @ a[s, p * rank].abs()).max() < 1 << 21)
            want[rows, lo:lo + width] += scaling[s] * (t @ b[s, lo:lo + width].t())
        lo += width
    assert want.abs().max() <= 256 and torch.equal(want.to(dtype).double(), want)
    c = [v.to(dtype).cuda() for v in (base, x, a, b)]
    assert all(torch.equal(v.double().cpu(), w) for v, w in zip(c, (base, x, a, b)))
    out = ops.lora_add(c[0], c[1], ops.lora_batch(index.cuda(), slots), c[2], c[3], scaling.float().cuda(), None, parts)
    wrong = out.double().cpu() != want
    assert not wrong.any(), f"{int(wrong.sum())} of {wrong.numel()}, the first {float(out.double().cpu()[wrong][0])} for {float(want[wrong][0])}"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("m,k,parts,slots,rank", [(1, 256, [72], 1, 16), (20, 2048, [264], 3, 16), (30, 512, [512], 8, 32),
                                                  (64, 2048, [264, 8], 20, 64), (100, 2048, [72], 3, 40), (900, 320, [520], 4, 24)])
def test_large_entries_leave_the_small_ones_their_bits(ops, m, k, parts, slots, rank, dtype):
    """Entries of t 2^18 to 2^26 apart in one row, the large ones with a B of zero: the small ones' sums are exact, and so is the
    result (one product of the type's full mantissa)."""
    g = torch.Generator().manual_seed(m + rank)
    n, one = sum(parts), 1 + torch.finfo(dtype).eps
    x = torch.ones(m, k, dtype=torch.float64)
    a = torch.zeros(slots, len(parts) * rank, k, dtype=torch.float64)
    b = torch.zeros(slots, n, rank, dtype=torch.float64)
    small = torch.randint(0, rank, (slots,), generator=g)
    for s in range(slots):
        for p in range(len(parts)):
            rows = a[s, p * rank:(p + 1) * rank]
            rows[:] = (1 << 15) // (1 << s % 6)  # t: k times as much
            rows[small[s]] = 0
            rows[small[s], s % k] = one  # t: that value alone
        b[s, :, small[s]] = 1
    index = torch.randint(0, slots, (m,), generator=g, dtype=torch.int32)
    scaling = 2.0 ** torch.randint(-3, 4, (slots,), generator=g).double()
    want = (scaling[index.long()] * one)[:, None].expand(m, n)
    c = [v.to(dtype).cuda() for v in (torch.zeros(m, n), x, a, b)]
    out = ops.lora_add(c[0], c[1], ops.lora_batch(index.cuda(), slots), c[2], c[3], scaling.float().cuda(), None, parts)
    assert torch.equal(out.double().cpu(), want), f"{float(out.double().cpu()[0, 0])} for {float(want[0, 0])}"
