"""The softmax's weights on their way through ops.paged_attention: what they keep of their bits where sums cancel, in long tails
far below the largest weight, and at scores whose own steps pass the weights' range.

Scores are exact here: a query has one nonzero entry, so a score is one product of two 16-bit numbers.  Tolerances, with
u = 2^-24 and e = eps / 2 of the type, for out = sum w_j v_j / sum w_j and A = sum w_j |v_j| / sum w_j:

* a weight's exponent is off by 4 u (|s_j| + |max|) and the exponential by 2^-22: with the largest of these, r, 2 r A;
* a weight goes to the second product in two parts of the type, the second one the first one's error: e^2 A (in one part, e A);
* fp16 holds nothing under 2^-25; of a tile's keys (64, the larger of the kernels') the largest weight is 1 or more
  before it is cut off, so that each key loses at most 2^-25 of the tile's largest weight;
* fp32's normal numbers end at 2^-126: a weight that is smaller beside the row's largest is zero (the exponential's, and the factor of
  a part that is joined), 2^-125 for both;
* n terms summed in fp32 in any order, and rescaled: 4 (n + 64) u A;
* the result is rounded once: e |out|.
"""

from __future__ import annotations

import pytest
import torch

from test_gpu_paged import U, _batch, _inputs, _near
from test_gpu_paged import _exact as _exact_rounded

pytestmark = pytest.mark.gpu

DTYPES = pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])


@pytest.fixture(scope="module")
def ops():
    from qtts_amd import ops as _ops
    assert _ops.device_supported(), "GPU is not a gfx950"
    _ops.reserve_workspace(torch.device("cuda"), 64 << 20)
    return _ops


def _call(ops, keys, values, count, dtype, heads=1, kv=1, page=64, window=0, sinks=0, scale=1.0, query=1.0, weights16=False):
    """One request whose key j has entry keys[j] and value values[j] ([n, d]), its last `count` tokens the rows, each of whose
    queries has one entry.  Returns the output [count, heads, d] and the batch."""
    n, d = values.shape
    batch, pages = _batch(ops, [(n - count, count)], page, seed=n)
    at = torch.arange(n, device="cuda")
    slot = batch.table[0].long()[at // page] * page + at % page
    k = torch.zeros(pages, kv, page, d, dtype=dtype, device="cuda")
    v = torch.zeros(pages, kv, d, page, dtype=dtype, device="cuda")
    k[slot // page, :, slot % page, 5] = keys.to(dtype)[:, None]
    v[slot // page, :, :, slot % page] = values.to(dtype)[:, None]
    q = torch.zeros(count, heads, d, dtype=dtype, device="cuda")
    q[:, :, 5] = query
    return ops.paged_attention(q, k, v, batch, window, sinks, scale, weights16)


def _exact(keys, values, count, dtype, window=0, sinks=0, weights16=False):
    """(result [count, d], bound without its rounding) in 64 bits, a row at a time."""
    n = values.shape[0]
    s, v = keys.to(dtype).double(), values.to(dtype).double()
    key = torch.arange(n, device="cuda")
    e = torch.finfo(dtype).eps / 2
    out, off, size = [], [], v.abs()
    dot = lambda x, y: (x[:, None] * y).sum(0)  # noqa: E731
    for p in range(n - count, n):
        seen = key <= p
        if window:
            seen &= (key > p - window) | (key < sinks)
        top = s[seen].max()
        w = torch.where(seen, (s - top).exp(), 0.0)
        total = w.sum()
        y, mags = dot(w, v) / total, dot(w, size) / total
        rel = 4 * U * (s[seen].abs().max() + top.abs()) + 2.0 ** -22
        bound = mags * (2 * rel + (e if weights16 else e * e) + 4 * (n + 64) * U) + 2.0 ** -125 * dot(seen, size) / total
        if dtype == torch.float16:
            tail = -n % 64
            tops = torch.nn.functional.pad(w, (0, tail)).view(-1, 64).amax(1).repeat_interleave(64)[:n]
            bound = bound + 2.0 ** -25 * dot(tops * seen, size) / total
        out.append(y)
        off.append(bound)
    return torch.stack(out), torch.stack(off)


def _check(ops, keys, values, count, dtype, heads=1, what="", window=0, sinks=0, weights16=False, **kw):
    out = _call(ops, keys, values, count, dtype, heads, window=window, sinks=sinks, weights16=weights16, **kw)
    want, off = _exact(keys, values, count, dtype, window, sinks, weights16)
    _near(out, want[:, None].expand_as(out), off[:, None].expand_as(out), what)


@DTYPES
@pytest.mark.parametrize("held,count,heads", [(63, 1, 1), (60, 1, 16), (0, 40, 1), (20, 44, 1), (0, 24, 8), (40, 17, 2), (100, 30, 4)])
@pytest.mark.parametrize("d", [16, 64, 128, 256])
def test_sums_that_cancel(ops, held, count, heads, d, dtype):
    """Values of both signs: the sum is far smaller than its terms, and no term loses what its rounding to 16 bits would take."""
    g = torch.Generator(device="cuda").manual_seed(held + count)
    n = held + count
    for spread in (128, 512):  # weights down to e^-1 and e^-4, in steps of 2^-7
        keys = -torch.randint(0, spread, (n,), generator=g, device="cuda") / 128.0
        keys = keys.to(dtype).float()
        values = torch.randn(n, d, generator=g, device="cuda")
        _check(ops, keys, values, count, dtype, heads)
        _check(ops, keys, values, count, dtype, heads, window=25, sinks=3)


@DTYPES
def test_a_chunk_whose_keys_are_split(ops, dtype):
    """The same where several workgroups share the keys: the chunk's rows see few of them but the first tokens."""
    g = torch.Generator(device="cuda").manual_seed(3)
    n, count = 3000, 70
    keys = (-torch.randint(0, 128, (n,), generator=g, device="cuda") / 128.0).to(dtype).float()
    keys[64:2900] -= 16  # (hardly any weight)
    values = torch.randn(n, 64, generator=g, device="cuda")
    _check(ops, keys, values, count, dtype)


@DTYPES
@pytest.mark.parametrize("heads,kv,d,page", [(16, 8, 128, 64), (4, 4, 64, 16), (4, 1, 256, 32), (12, 4, 80, 128)])
@pytest.mark.parametrize("requests,window,sinks", [([(0, 37), (300, 130), (9, 1)], 0, 0), ([(40, 1), (5000, 60), (0, 200)], 0, 0),
                                                   ([(500, 150), None, (3, 2)], 70, 4)])
def test_weights_of_16_bits(ops, requests, window, sinks, heads, kv, d, page, dtype):
    """Where a caller asks for them: prompts within half a step of each weight, requests of up to 16 rows as without."""
    q, k, v, batch = _inputs(ops, requests, page, heads, kv, d, dtype, seed=d, padding=2)
    full = ops.paged_attention(q, k, v, batch, window, sinks)
    out = ops.paged_attention(q, k, v, batch, window, sinks, weights16=True)
    want, off = _exact_rounded(q, k, v, batch, window, sinks, d ** -0.5)
    _near(out, want, off, "16 bits")
    at = 0
    for r in requests:
        new = 3 if r is None else r[1]
        same = torch.equal(out[at:at + new], full[at:at + new])
        assert same == (r is None or new * heads // kv <= 16)
        at += new
    assert not out[batch.slots < 0].any()


def test_weights_of_16_bits_in_a_layer(ops):
    """The switch's way through the cache's layer."""
    from qtts_amd import PagedCache, attend
    cache = PagedCache(1, 2, 8, 4, 2, 64, max_rows=64, rope_theta=1e4)
    g = torch.Generator(device="cuda").manual_seed(1)
    qkv = torch.randn(50, 8 * 64, generator=g, device="cuda").to(torch.bfloat16)
    cache.step([50])
    attn = torch.nn.Module()
    outs = [attend(attn, qkv, cache, 0, weights16=w) for w in (False, True, False)]
    assert torch.equal(outs[0], outs[2]) and not torch.equal(outs[0], outs[1])
    # half a step of each weight, and of either result
    assert (outs[1].double() - outs[0].double()).abs().max() < 2.0 ** -6 * qkv.abs().max()


@DTYPES
@pytest.mark.parametrize("count", [1, 5, 40])
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_past_the_weights_range(ops, count, sign, dtype):
    """Scores whose own fp32 steps are many powers of two: the largest one's key has all the weight (the next one is a
    thousand steps below), and rounding the maximum makes no weight infinite.  The result is that key's value, up to its weight's
    two parts (e^2), the sum's and the quotient's roundings (4 u) and its own."""
    g = torch.Generator(device="cuda").manual_seed(11)
    n, e = 100, torch.finfo(dtype).eps / 2
    for case in range(12):
        keys = sign * (1 + torch.randperm(n, generator=g, device="cuda") / 128.0)
        values = torch.randn(n, 64, generator=g, device="cuda").to(dtype)
        for power in (20, 24, 26, 27, 28, 30, 33, 36, 50, 100):
            out = _call(ops, keys, values, count, dtype, scale=2.0 ** power, query=1 + case / 16)
            for i in range(count):
                best = int(keys[:n - count + i + 1].argmax())
                v = values[best].double()
                err = (out[i, 0].double() - v).abs()
                assert (err <= (e + e * e + 4 * U) * v.abs()).all(), (case, power, i, float(err.max()))


def _tail(n, where, far, spread, g):
    """Scores of one key at 0 and the others `far` below it, give or take; values: 0 and 1, and the other way round."""
    keys = -far - torch.rand(n, generator=g, device="cuda") * spread
    at = {"first": 0, "middle": n // 2 + 3, "last": n - 41}[where]
    keys[at] = 0.0
    values = torch.ones(n, 16, device="cuda")
    values[:, 8:] = 0.0
    values[at] = 1 - values[at]
    return keys, values


@DTYPES
@pytest.mark.parametrize("count", [1, 40])
@pytest.mark.parametrize("where", ["first", "middle", "last"])
@pytest.mark.parametrize("far,spread", [(11.0, 0.0), (15.5, 3.0), (17.5, 0.0), (17.5, 4.0), (24.0, 0.0), (40.0, 0.0)])
def test_long_tails(ops, far, spread, where, count, dtype):
    """One key far above tens of thousands of others: their share of the result is theirs, however small each one's weight."""
    g = torch.Generator(device="cuda").manual_seed(7)
    keys, values = _tail(65536, where, far, spread, g)
    _check(ops, keys, values, count, dtype)
    if count > 1:
        _check(ops, keys, values, count, dtype, weights16=True)


@pytest.mark.parametrize("count", [1, 17])
def test_a_million_keys_behind_one(ops, count):
    """Lengths at which weights of 2^-25 outweigh the key that stands out."""
    for far in (14.0, 17.375, 19.0):
        keys, values = _tail(1 << 20, "first", far, 0.0, torch.Generator(device="cuda").manual_seed(1))
        _check(ops, keys, values, count, torch.float16, page=1024)


@DTYPES
@pytest.mark.parametrize("count", [1, 30])
def test_falling_and_rising_scores(ops, count, dtype):
    """Scores along a slope of hundreds of powers of two either way, and up and down again: the tiles' largest weights are anywhere
    below the row's."""
    n = 4000
    at = torch.arange(n, device="cuda")
    for keys in (-at / 32.0, (at - n) / 32.0, -(at - n / 2).abs() / 64.0, (at - n / 2).abs() / 64.0 - 40, -(at % 700) / 8.0):
        keys = keys.to(dtype).float()
        for low in (-3.0, -12.0, -25.0):
            below = keys - keys.max() < low  # of the sum, what lies under e^low alone
            values = below.float()[:, None].expand(n, 16)
            _check(ops, keys, values, count, dtype)
            _check(ops, keys, values, count, dtype, window=1000, sinks=70)


@DTYPES
@pytest.mark.parametrize("n,heads", [(20000, 1), (4096, 1024)])
@pytest.mark.parametrize("count", [1, 3, 20])
@pytest.mark.parametrize("value", [0.0, float("inf"), float("nan")])
def test_tails_around_a_value_that_is_not_finite(ops, value, count, n, heads, dtype):
    """Sums that are formed key by key keep the tail and the key before it as well: of the rows before the last one, which alone sees an
    infinity or NaN."""
    keys, v = _tail(n, "first", 17.5, 0.0, torch.Generator(device="cuda").manual_seed(2))
    v[n - 1] = value
    out = _call(ops, keys, v, count, dtype, heads=heads, kv=heads)
    want, off = _exact(keys, torch.nan_to_num(v, 0.0, 0.0, 0.0), count, dtype)
    last = count if value == 0.0 else count - 1
    _near(out[:last], want[:last, None].expand(last, heads, 16), off[:last, None].expand(last, heads, 16), "rows")
    if last < count:
        assert not out[-1].isfinite().any()


@DTYPES
@pytest.mark.parametrize("count", [1, 20])
def test_tails_of_many_heads(ops, count, dtype):
    """So many heads that each one's keys stay with a few waves, whose own keys are a tail behind the one that stands out."""
    keys, values = _tail(4096, "first", 17.5, 0.0, torch.Generator(device="cuda").manual_seed(5))
    _check(ops, keys, values, count, dtype, heads=1024, kv=1024)


@pytest.mark.parametrize("method", ["none", "fp8"])
def test_weights_of_16_bits_in_whole_layers(ops, method):
    from qtts_amd.layers.decoder import paged_layer, paged_layer_w8a8
    from test_gpu_paged_layer import _cache, _model, _rows
    dtype = torch.bfloat16
    layer, x = _model(method, dtype, layers=1)[0], _rows(50, torch.bfloat16, 1)
    outs = []
    for w in (False, True, False):
        cache = _cache(dtype, layers=1)
        cache.step([50])
        if method == "none":
            outs.append(paged_layer(layer, x, cache, 0, weights16=w))
        else:
            delta, hidden = paged_layer_w8a8(layer, x, None, cache, 0, weights16=w)
            outs.append(hidden + delta)
    assert torch.equal(outs[0], outs[2]) and not torch.equal(outs[0], outs[1])
    assert outs[1].isfinite().all()
