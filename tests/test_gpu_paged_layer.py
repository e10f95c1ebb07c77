"""A model's layers over a paged cache, as a serving loop runs them: prompts, chunks of prompts and single tokens of several
requests in one cache, requests that end and pages that are used again, captured decode steps at several padded row counts,
on linears of several methods.

What attend computes is held against 64 bits on the cache's own contents (tolerances as derived in test_gpu_paged.py),
and the contents against 64 bits on qkv_proj's output; steps that differ only in how they are run, bit for bit."""

from __future__ import annotations

import pytest
import torch
from torch import nn

from test_gpu_paged import _exact, _near, _qkv_exact
from test_gpu_w8a8_layer import Norm

pytestmark = pytest.mark.gpu

HIDDEN, INTER, HEADS, KV, D = 256, 384, 4, 2, 64
THETA = 1e4


@pytest.fixture(scope="module")
def ops():
    from qtts_amd import ops as _ops
    assert _ops.device_supported(), "GPU is not a gfx950"
    return _ops


class Attention(nn.Module):
    def __init__(self, dtype):
        super().__init__()
        from qtts_amd.layers import LinearBase, MergedLinear
        self.qkv_proj = MergedLinear(HIDDEN, [HEADS * D, KV * D, KV * D], bias=True, dtype=dtype, device="cuda")
        self.q_norm, self.k_norm = Norm(D, dtype), Norm(D, dtype)
        self.o_proj = LinearBase(HEADS * D, HIDDEN, dtype=dtype, device="cuda")


class Layer(nn.Module):
    def __init__(self, dtype):
        super().__init__()
        from qtts_amd.layers import GatedMLP
        self.input_layernorm, self.post_attention_layernorm = Norm(HIDDEN, dtype), Norm(HIDDEN, dtype)
        self.attn = Attention(dtype)
        self.mlp = GatedMLP(HIDDEN, INTER, fuse=True, dtype=dtype, device="cuda")


def _model(method, dtype, layers=2, seed=3):
    from qtts_amd import QuantConfig
    from qtts_amd.quant.base import build_method, quantize_module
    model = nn.ModuleList([Layer(dtype) for _ in range(layers)])
    g = torch.Generator(device="cuda").manual_seed(seed)
    for name, p in model.named_parameters():
        if "norm" not in name:
            p.data.copy_((torch.randn(p.shape, device="cuda", generator=g) * 0.06).to(dtype))
    if method != "none":
        config = QuantConfig(method=method, calibrate=False)
        assert quantize_module(model, build_method(config), config, "talker")["converted"] == 4 * layers
    return model


def _cache(dtype, requests=6, layers=2, page=16, pages=80, rows=200, **kw):
    from qtts_amd import PagedCache
    return PagedCache(layers, requests, pages, HEADS, KV, D, page, max_rows=rows, dtype=dtype, rope_theta=THETA, **kw)


def _rows(m, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(m, HIDDEN, device="cuda", generator=g).to(dtype)


def _forward(model, cache, x, method, window=0, sinks=0):
    from qtts_amd.layers.decoder import paged_layer, paged_layer_w8a8
    if method in ("fp8", "int8"):
        delta, hidden = x, None
        for i, layer in enumerate(model):
            delta, hidden = paged_layer_w8a8(layer, delta, hidden, cache, i, window, sinks)
        return hidden + delta
    for i, layer in enumerate(model):
        x = paged_layer(layer, x, cache, i, window, sinks)
    return x


DTYPES = pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])


@DTYPES
@pytest.mark.parametrize("window,sinks", [(0, 0), (24, 3)])
def test_attend_over_steps(ops, window, sinks, dtype):
    """Prompts, decode, a chunk, a release and a new request on the freed pages: every step's cache contents and outputs."""
    from qtts_amd import attend
    model, cache = _model("none", dtype, layers=1), _cache(dtype, layers=1, pages=16)
    attn = model[0].attn
    steps = [[37, 5, 0, 1], [1, 1, 0, 1], [0, 40, 60], [1, 1, 1, 1], "release 1 0", [3, 90, 1, 1], [1, 1, 1, 1], "release 2", [1, 0, 0, 100, 64],
             [0, 0, 0, 0, 0, 0]]
    held, denied = [0] * 6, 0
    for n, new in enumerate(steps):
        if isinstance(new, str):
            gone = [int(r) for r in new.split()[1:]]
            cache.release(gone)
            held = [0 if r in gone else h for r, h in enumerate(held)]
            continue
        rows = sum(new) + n % 3
        batch = cache.step(new, rows=rows)
        qkv = attn.qkv_proj(_rows(rows, dtype, n)) * 4
        out = attend(attn, qkv, cache, 0, window, sinks)
        counts = batch.counts.tolist()
        held = [h + c for h, c in zip(held, counts)]
        denied += sum(c != w for c, w in zip(counts, new + [0] * 6))
        assert cache.lengths.tolist() == held
        assert all(c in (0, w) for c, w in zip(counts, new + [0] * 6))
        k, v = cache.k[0], cache.v[0]
        q, ek, ev, oq, ok = _qkv_exact(qkv, HEADS, KV, D, attn.q_norm.weight, attn.k_norm.weight, 1e-6, cache.rope, batch.positions)
        live = batch.slots >= 0
        slot = batch.slots[live].long()
        _near(k[slot // 16, :, slot % 16], ek[live], ok[live], f"k of step {n}")
        assert torch.equal(v[slot // 16, :, :, slot % 16].double(), ev[live])
        mine = ops.qkv_to_cache(qkv, k.clone(), v.clone(), batch, HEADS, attn.q_norm.weight, attn.k_norm.weight, 1e-6, cache.rope)
        _near(mine[live], q[live], oq[live], f"q of step {n}")
        want, off = _exact(mine, k, v, batch, window, sinks, D ** -0.5)
        _near(out.view(rows, HEADS, D), want, off, f"step {n}")
        assert not out[~live].any()
    assert denied == 1  # the last request of that step: 14 of 16 pages are held then, and its 64 tokens want 4
    used = sum(-(-h // 16) for h in held)
    assert int(cache.taken) == used


@DTYPES
@pytest.mark.parametrize("method", ["none", "int8_weight_only", "fp8", "int8", "fp8_weight_only"])
def test_captured_steps(ops, method, dtype):
    """Decode steps at three padded row counts, captured once each: every replay has the eager step's bits, on one cache and
    workspace, between prompts that run eagerly."""
    from qtts_amd.graphs import PaddedGraphs
    model = _model(method, dtype)
    eager, cache = _cache(dtype, requests=8, pages=120), _cache(dtype, requests=8, pages=120)
    for i in range(2):  # rows of padding may read nothing else
        for c in (eager, cache):
            c.k[i].fill_(float("nan")), c.v[i].fill_(float("nan"))
    graphs = PaddedGraphs(lambda x: _forward(model, cache, x, method), (HIDDEN,), dtype, batch_sizes=(1, 4, 8))
    plans = [[9, 30], [1], [1, 1], [1, 1, 1, 1, 0, 1], [0, 0, 50, 0, 17], [0, 1, 1, 1], [1] * 8, [1], [1, 0, 1], [1] * 8, [1, 1, 1, 1], [1] * 8]
    for n, new in enumerate(plans):
        total = sum(new)
        if max(new) > 1:
            x = _rows(total, dtype, n)
            outs = []
            for c in (eager, cache):
                c.step(new)
                outs.append(_forward(model, c, x, method))
        else:
            padded = graphs.padded_rows(total)
            x = _rows(total, dtype, n)
            eager.step(new, rows=padded, max_new=1)
            full = torch.zeros(padded, HIDDEN, dtype=dtype, device="cuda")
            full[:total] = x
            want = _forward(model, eager, full, method)[:total]
            cache.step(new, rows=padded, max_new=1)
            outs = [want, graphs.run(x).clone()]
        assert torch.equal(outs[0], outs[1]), f"step {n}"
        assert outs[0].isfinite().all()
        assert torch.equal(eager.lengths, cache.lengths) and torch.equal(eager.taken, cache.taken)
    assert len(graphs.graphs) == 3
    torch.cuda.synchronize()


def test_a_replay_without_its_step(ops):
    """A graph of more rows than the last step had: its further rows have no request, write nothing and get zeros."""
    from qtts_amd import attend
    dtype = torch.bfloat16
    model, cache = _model("none", dtype, layers=1), _cache(dtype, layers=1)
    cache.k[0].zero_(), cache.v[0].zero_()  # values that compare, where fresh memory may hold NaN
    x = _rows(6, dtype, 1)
    qkv = model[0].attn.qkv_proj(x)
    cache.step([1] * 6, max_new=1)
    attend(model[0].attn, qkv, cache, 0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = attend(model[0].attn, qkv, cache, 0)
    cache.step([1, 1], rows=3, max_new=1)
    before = cache.k[0].clone()
    out.fill_(7.0)
    graph.replay()
    assert not out[2:].any() and out[:2].any(1).all()
    slots = cache.batch.slots[:2].long()
    changed = (cache.k[0] != before).any(3).any(1).nonzero()
    assert sorted((changed[:, 0] * 16 + changed[:, 1]).tolist()) == sorted(slots.tolist())
    cache.step([30, 2], max_new=30)  # a step that the graph's kernels were not captured for
    graph.replay()
    assert out.isfinite().all()


@DTYPES
def test_chunks_make_the_same_cache(ops, dtype):
    """A prompt in one step, in chunks and token by token: the same keys and values, and outputs within two roundings."""
    from qtts_amd import attend
    model = _model("none", dtype, layers=1)
    x = _rows(70, dtype, 2)
    outs, caches = [], []
    for cuts in ([70], [16, 1, 33, 20], [1] * 70):
        cache, parts, at = _cache(dtype, layers=1), [], 0
        qkv = model[0].attn.qkv_proj(x)
        for n in cuts:
            cache.step([0, n])
            parts.append(attend(model[0].attn, qkv[at:at + n], cache, 0))
            at += n
        outs.append(torch.cat(parts))
        at = torch.arange(70, device="cuda")
        slot = cache.table[1].long()[at // 16] * 16 + at % 16
        caches.append((cache.k[0][slot // 16, :, slot % 16], cache.v[0][slot // 16, :, :, slot % 16]))
    for out, (k, v) in zip(outs[1:], caches[1:]):
        assert torch.equal(k, caches[0][0]) and torch.equal(v, caches[0][1])
        # half a step each of both results and of the weights', of values up to the largest
        off = 4 * torch.finfo(dtype).eps * v.abs().max().double()
        assert ((out.double() - outs[0].double()).abs() <= off).all()


def test_counts_on_the_gpu(ops):
    """A captured step of its own: the counts live on the GPU, the tables follow them at every replay, and what does not fit is denied."""
    dtype = torch.bfloat16
    cache = _cache(dtype, requests=4, pages=9, max_length=64)
    new = torch.zeros(4, dtype=torch.int32, device="cuda")
    cache.step(new, rows=12, max_new=10)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        batch = cache.step(new, rows=12, max_new=10)
    cache.release([0, 1, 2, 3])
    want = [0] * 4
    for values, counts in (([3, 0, 9, 0], [3, 0, 9, 0]), ([11, 1, 0, 0], [0, 1, 0, 0]), ([6, 6, 1, 0], [6, 6, 0, 0]), ([0, 0, 10, 2], [0, 0, 10, 2]),
                           ([-4, 1, 1, 1], [0, 1, 1, 1])):
        new.copy_(torch.tensor(values, dtype=torch.int32))
        graph.replay()
        want = [w + c for w, c in zip(want, counts)]
        assert batch.counts.tolist() == counts and cache.lengths.tolist() == want
        assert int(cache.taken) == sum(-(-w // 16) for w in want)
    with pytest.raises(ValueError, match="rows must be given"):
        cache.step(new)
    cache.release(torch.tensor([1, 900, -3, 1, 2 ** 40], device="cuda"))  # the same twice, and numbers of no request
    want[1] = 0
    assert cache.lengths.tolist() == want and int(cache.taken) == sum(-(-w // 16) for w in want)
    cache.release([3, 3])
    want[3] = 0
    assert cache.lengths.tolist() == want


def test_attend_with_other_norms(ops):
    """Heads whose norm is no RMSNorm of one weight run it as the module it is; none at all is none."""
    from qtts_amd import attend
    dtype = torch.bfloat16

    class Shifted(Norm):
        def forward(self, x):
            return super().forward(x) + 0.25

    model = _model("none", dtype, layers=1)
    attn = model[0].attn
    x = _rows(20, dtype, 5)
    qkv = attn.qkv_proj(x)
    results = {}
    for name in ("rms", "shifted", "none"):
        if name == "shifted":
            attn.q_norm = Shifted(D, dtype)
        if name == "none":
            attn.q_norm = attn.k_norm = None
        cache = _cache(dtype, layers=1)
        batch = cache.step([20])
        out = attend(attn, qkv.view(1, 20, -1), cache, 0)
        assert out.shape == (1, 20, HEADS * D)
        parts = qkv.view(20, HEADS + 2 * KV, D).split([HEADS, KV, KV], 1)
        if name != "none":
            parts = [attn.q_norm(parts[0]), attn.k_norm(parts[1]), parts[2]]
        k, v = torch.zeros_like(cache.k[0]), torch.zeros_like(cache.v[0])
        q = ops.qkv_to_cache(torch.cat(list(parts), 1).view(20, -1), k, v, batch, HEADS, rope=cache.rope)
        want, off = _exact(q, k, v, batch, 0, 0, D ** -0.5)
        results[name] = out.view(20, HEADS, D)
        if name == "rms":  # the kernel does not round between norm and rotation
            assert ((results[name].double() - want).abs() <= off + 0.05).all()
        else:
            _near(results[name], want, off, name)
    assert not torch.equal(results["rms"], results["shifted"])
    with pytest.raises(ValueError, match="set for 20 rows"):
        attend(attn, qkv[:3], cache, 0)
    with pytest.raises(ValueError, match="heads"):
        attend(attn, qkv[:, :64], cache, 0)


def test_streams_and_a_second_cache(ops):
    """Steps of two caches on two streams, each in its order on its own stream, one after the other on the shared workspace."""
    from qtts_amd import attend
    dtype = torch.bfloat16
    model = _model("none", dtype, layers=1)
    side = torch.cuda.Stream()
    outs = []
    for stream in (torch.cuda.current_stream(), side):
        cache = _cache(dtype, layers=1, requests=2, pages=700)
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            for n in (150, 200, 200):
                cache.step([n, 0])
                attend(model[0].attn, model[0].attn.qkv_proj(_rows(n, dtype, n)), cache, 0)
            cache.step([1, 1])
            outs.append(attend(model[0].attn, model[0].attn.qkv_proj(_rows(2, dtype, 9)), cache, 0))
        torch.cuda.current_stream().wait_stream(stream)
        torch.cuda.synchronize()
    assert torch.equal(outs[0], outs[1])
