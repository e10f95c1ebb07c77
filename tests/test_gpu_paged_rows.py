"""Rows at the edges of a paged batch: rows of no request, rows whose slots and counts disagree, rows that a captured step was not
made for."""

from __future__ import annotations

import pytest
import torch

from test_gpu_paged import U, _batch, _exact, _i32, _inputs, _near

pytestmark = pytest.mark.gpu

DTYPES = pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])


@pytest.fixture(scope="module")
def ops():
    from qtts_amd import ops as _ops
    assert _ops.device_supported(), "GPU is not a gfx950"
    _ops.reserve_workspace(torch.device("cuda"), 64 << 20)
    return _ops


@DTYPES
@pytest.mark.parametrize("rope", [False, True])
@pytest.mark.parametrize("weight,eps", [(1.0, 0.0), (float("inf"), 1e-6), (float("nan"), 1e-6), (float("inf"), 0.0)])
def test_padding_rows_are_zeros_whatever_the_norm(ops, weight, eps, rope, dtype):
    """Rows of no request, few and many: their queries are zeros where the norm of zeros is none."""
    for rows, padding in ((3, 2), (2500, 37)):
        heads, kv, d = 16, 8, 64
        batch, pages = _batch(ops, [(0, rows)], 64, padding=padding)
        g = torch.Generator(device="cuda").manual_seed(rows)
        qkv = torch.randn(rows + padding, (heads + 2 * kv) * d, generator=g, device="cuda").to(dtype)
        k, v = torch.zeros(pages, kv, 64, d, dtype=dtype, device="cuda"), torch.zeros(pages, kv, d, 64, dtype=dtype, device="cuda")
        w = torch.full((d,), weight, dtype=dtype, device="cuda")
        turns = torch.zeros(batch.cols * 64, d // 2, device="cuda")
        q = ops.qkv_to_cache(qkv, k, v, batch, heads, w, w, eps, (turns + 1, turns) if rope else None)
        assert not q[rows:].any()
        if weight == 1.0:
            x = qkv[:rows].double().view(rows, -1, d)[:, :heads]
            want = x / x.square().mean(-1, keepdim=True).sqrt()
            _near(q[:rows], want, want.abs() * U * (d / 2 + 11), "q")


def _poisoned(shape, dtype):
    """What the next tensor of this size is likely to find in its memory."""
    torch.full(shape, float("nan"), dtype=dtype, device="cuda")


@DTYPES
@pytest.mark.parametrize("counts,heads,kv", [([1] * 9, 16, 8), ([1, 3, 60, 1, 0, 200], 8, 4)])
def test_rows_go_by_starts_and_counts(ops, counts, heads, kv, dtype):
    """Slots that disagree: every row of a request is computed and every other one zero, once each."""
    q, k, v, batch = _inputs(ops, [(30 + 7 * i, n) for i, n in enumerate(counts)], 16, heads, kv, 64, dtype, seed=4, padding=6)
    want = ops.paged_attention(q, k, v, batch)
    off, slots = torch.full_like(batch.slots, -1), batch.slots.clone()
    slots[-6:] = 5  # rows of no request
    slots[0] = -1
    for other in (off, slots, torch.zeros_like(off)):
        odd = ops.PagedBatch(batch.table, batch.starts, batch.counts, batch.lengths, batch.positions, other, 16, max_new=batch.max_new)
        for _ in range(3):
            _poisoned(q.shape, dtype)
            assert torch.equal(ops.paged_attention(q, k, v, odd), want)


@DTYPES
def test_gaps_between_requests(ops, dtype):
    """Requests with rows of none between and behind them, more than a workgroup's share of rows (its span of 1024 several times)."""
    at, counts = [3, 1030, 1100, 2047, 250000, 300000 - 41], [1, 70, 0, 2, 40, 41]
    rows, n = 300000, 100
    table = _i32([[i * 7 + j for j in range(7)] for i in range(6)])
    lengths = [n if c else 0 for c in counts]
    batch = ops.PagedBatch(table, _i32(at + [rows]), _i32(counts), _i32(lengths), _i32([-1] * rows), _i32([-1] * rows), 16, max_new=70)
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = (torch.randn(s, generator=g, device="cuda").to(dtype) for s in ((rows, 1, 16), (42, 1, 16, 16), (42, 1, 16, 16)))
    _poisoned(q.shape, dtype)
    out = ops.paged_attention(q, k, v, batch)
    live = torch.zeros(rows, dtype=torch.bool, device="cuda")
    for a, c in zip(at, counts):
        live[a:a + c] = True
    assert not out[~live].any()
    want, off = _exact(q, k, v, batch, 0, 0, 0.25)
    _near(out[live], want[live], off[live], "rows of requests")
    bad = [a if i != 1 else -5 for i, a in enumerate(at)]  # and where one of them is nothing that a step makes
    odd = ops.PagedBatch(table, _i32(bad + [rows]), batch.counts, batch.lengths, batch.positions, batch.slots, 16, max_new=70)
    _poisoned(q.shape, dtype)
    again = ops.paged_attention(q, k, v, odd)
    out[at[1]:at[1] + counts[1]] = 0
    assert torch.equal(again, out)


@DTYPES
@pytest.mark.parametrize("captured,later", [([1, 1], [3, 4]), ([0, 0, 0], [5, 0, 1]), ([2, 1], [1, 0, 7]), ([1] * 8, [8])])
def test_a_graph_of_a_step_without_max_new(ops, captured, later, dtype):
    """A step's own largest count bounds that step alone: a graph captured after it replays for counts up to its rows."""
    from qtts_amd import PagedCache, attend
    g = torch.Generator(device="cuda").manual_seed(3)
    attn = torch.nn.Module()
    caches = [PagedCache(1, 9, 40, 4, 1, 64, page_size=16, max_rows=64, dtype=dtype, rope_theta=1e4) for _ in range(2)]
    prompt = torch.randn(40, 6 * 64, generator=g, device="cuda").to(dtype)
    for c in caches:
        c.k[0].zero_(), c.v[0].zero_()
        c.step([20, 15, 5])
        attend(attn, prompt, c, 0)
    x = torch.randn(8, 6 * 64, generator=g, device="cuda").to(dtype)
    for c in caches:
        c.step(captured, rows=8)
        attend(attn, x, c, 0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = attend(attn, x, caches[1], 0)
    for n, new in enumerate((later, captured, later, [1, 2, 3])):
        x.copy_(torch.randn(8, 6 * 64, generator=g, device="cuda").to(dtype))
        for c in caches:
            c.step(new, rows=8)
        want = attend(attn, x, caches[0], 0)
        graph.replay()
        # of runs of one kernel or the other: within two steps of the largest value
        assert ((out.double() - want.double()).abs() <= 2 * torch.finfo(dtype).eps * x.abs().max()).all(), n
        assert torch.equal(out.any(1), want.any(1)) and int(want.any(1).sum()) == sum(new)
    # a bound that the caller gives stands for the graph as well: more tokens than it are zeros
    for c in caches:
        c.step([1, 1], rows=8, max_new=1)
    tight = torch.cuda.CUDAGraph()
    with torch.cuda.graph(tight):
        out = attend(attn, x, caches[1], 0)
    caches[1].step([1, 3], rows=8)
    tight.replay()
    assert out[0].any() and not out[1:].any()


def test_bounds_that_out_does_not_have(ops):
    """A step into a batch takes the batch's bounds: other ones beside it are refused, not left aside."""
    table, lengths, free, taken = _i32([[-1] * 4] * 2), _i32([0, 0]), _i32(list(range(8))), _i32([0])
    out = ops.paged_step(_i32([0, 0]), lengths, table, free, taken, 16, 9, max_new=5, min_new=1)
    args = (_i32([4, 2]), lengths, table, free, taken, 16, 9)
    for kw in ({"max_new": 3}, {"max_new": 9}, {"min_new": 2}):
        with pytest.raises(ValueError, match="new"):
            ops.paged_step(*args, out=out, **kw)
    for kw in ({}, {"max_new": 5}, {"min_new": 1}, {"max_new": 5, "min_new": 1}):
        assert ops.paged_step(*args, out=out, **kw).counts.tolist() == [4, 2]


@DTYPES
def test_head_norms_of_another_type(ops, dtype):
    """A norm whose weight is in 32 bits runs as the module it is (in 16 its weight would be rounded), and so does one that
    returns 32 bits."""
    from qtts_amd import PagedCache, attend
    from test_gpu_w8a8_layer import Norm
    d, heads, kv, rows = 64, 4, 2, 40

    class Wide(Norm):
        def forward(self, x):
            return super().forward(x.float())

    g = torch.Generator(device="cuda").manual_seed(6)
    qkv = torch.randn(rows, (heads + 2 * kv) * d, generator=g, device="cuda").to(dtype)
    attn = torch.nn.Module()
    for kind, weight in ((Norm, torch.float32), (Wide, torch.float32), (Wide, dtype), (Norm, dtype)):
        attn.q_norm, attn.k_norm = kind(d, weight), kind(d, weight)
        cache = PagedCache(1, 1, 4, heads, kv, d, page_size=16, max_rows=rows, dtype=dtype)
        batch = cache.step([rows])
        attend(attn, qkv, cache, 0)
        slot = batch.slots.long()
        got = cache.k[0][slot // 16, :, slot % 16]
        x = qkv.view(rows, -1, d)[:, heads:heads + kv].double()
        want = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * attn.k_norm.weight.double()
        # the module in fp32: half of the sum's relative error, then a root, a division, two products
        _near(got, want, want.abs() * U * (d / 2 + 11), kind.__name__)


@DTYPES
@pytest.mark.parametrize("heads,kv,d", [(200, 1, 16), (512, 2, 64), (129, 1, 128), (1024, 1024, 16), (1000, 8, 32)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (20, 3)])
def test_many_query_heads(ops, heads, kv, d, window, sinks, dtype):
    """A token's query heads past a run's rows, and so many key-value heads that nothing is cut."""
    q, k, v, batch = _inputs(ops, [(70, 1), (0, 3), (33, 2), None], 16, heads, kv, d, dtype, seed=heads, padding=2)
    want, off = _exact(q, k, v, batch, window, sinks, d ** -0.5)
    _near(ops.paged_attention(q, k, v, batch, window, sinks), want, off, "rows")
