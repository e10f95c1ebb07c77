"""Calls over a paged cache without a GPU: what the entries and the cache refuse and how they pass on what they are given."""

from __future__ import annotations

import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import qtts_amd  # noqa: F401
from qtts_amd import _lib, ops

BUF = ctypes.create_string_buffer(1 << 20)
AT = (ctypes.addressof(BUF) + 255) & ~255


def _at(v):
    return None if v is None else AT + v


def _passes(status):
    """Past every check: no device here, or the call ran nothing."""
    assert status == 0 or (status == -2 and not torch.cuda.is_available()), _lib.last_error()


def _i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def _attention(entry, q=0, dt=1, rows=2, ldq=64, heads=4, kv=2, d=16, k=65536, v=131072, pages=8, page=16, table=4096, requests=2, cols=3,
               starts=5120, counts=5184, lengths=5248, slots=5312, least=1, most=1, window=0, sinks=0, scale=0.25, out=8192, ldo=64,
               ws=262144, ws_n=1 << 62):
    return entry(_at(q), dt, rows, ldq, heads, kv, d, _at(k), _at(v), pages, page, _at(table), requests, cols, _at(starts), _at(counts),
                 _at(lengths), _at(slots), least, most, window, sinks, scale, _at(out), ldo, _at(ws), ws_n, None)


def test_attention_with_weights_of_16_bits():
    """Its entry checks what the other one checks, and the op has it as its last argument."""
    entry = _lib.load().qtts_paged_attention_w16
    for kw, text in (({"dt": 0}, "bf16 or fp16"), ({"rows": -1}, "negative size"), ({"heads": 5}, "query heads"), ({"ldo": 56}, "leading dimension"),
                     ({"scale": 0.0}, "scale"), ({"out": 64}, "out overlaps q"), ({"ws": None}, "workspace"), ({"table": None}, "null pointer")):
        status = _attention(entry, **kw)
        assert status in (-1, -5) and text in _lib.last_error(), (kw, status, _lib.last_error())
    assert _attention(entry, rows=0) == 0
    if not torch.cuda.is_available():
        _passes(_attention(entry))
    with FakeTensorMode():
        bf = torch.bfloat16
        k, v = torch.empty(9, 2, 16, 32, dtype=bf, device="cuda"), torch.empty(9, 2, 32, 16, dtype=bf, device="cuda")
        state = [torch.empty(*s, dtype=torch.int32, device="cuda") for s in ((3, 4), (4,), (3,), (3,), (5,), (5,))]
        q = torch.empty(5, 4, 32, dtype=bf, device="cuda")
        assert torch.ops.qtts.paged_attention(q, k, v, state, [16, 5, 0], 0, 0, 0.1, True).shape == (5, 4, 32)
    batch = ops.PagedBatch(_i32(3, 4), _i32(4), _i32(3), _i32(3), _i32(5), _i32(5), 16)
    bf = torch.bfloat16
    with pytest.raises(ValueError, match="GPU tensor"):
        ops.paged_attention(torch.zeros(5, 4, 32, dtype=bf), torch.zeros(9, 2, 16, 32, dtype=bf), torch.zeros(9, 2, 32, 16, dtype=bf), batch,
                            weights16=True)


def test_an_eps_that_no_norm_has():
    entry = _lib.load().qtts_qkv_to_cache

    def call(eps, qn=8320, kn=8384):
        return entry(_at(0), 1, 2, 128, 4, 2, 16, _at(8192), _at(8256), _at(qn), _at(kn), eps, _at(8448), _at(12544), 32, _at(65536),
                     _at(131072), 8, 16, _at(16384), None)

    for eps in (-1e-6, float("nan"), float("inf"), -float("inf")):
        for norms in ({}, {"qn": None}, {"kn": None}):
            assert call(eps, **norms) == -1 and "eps" in _lib.last_error(), (eps, norms)
    if not torch.cuda.is_available():
        for eps in (0.0, 1e-6, 1.0):
            _passes(call(eps))
        _passes(call(-1.0, qn=None, kn=None))  # no norm, no eps


def test_rows_times_heads_past_32_bits():
    """A request's rows of one key-value head are counted in 32 bits and make a grid of fewer than 2^32 threads."""
    for entry in (_lib.load().qtts_paged_attention, _lib.load().qtts_paged_attention_w16):
        for rows, heads, kv in ((1 << 20, 2048, 1), ((1 << 24) - 1, 4096, 4), ((1 << 24) - 1, 129, 129)):
            # (q and out: any addresses that do not overlap; nothing is read)
            status = _attention(entry, rows=rows, heads=heads, kv=kv, ldq=heads * 16, ldo=heads * 16, q=0, out=1 << 45, k=1 << 50, v=1 << 51)
            assert status == -1 and "too large" in _lib.last_error(), (rows, heads, status, _lib.last_error())
        if not torch.cuda.is_available():
            _passes(_attention(entry, rows=(1 << 20) - 1, heads=2048, kv=1, ldq=2048 * 16, ldo=2048 * 16, q=0, out=1 << 45, k=1 << 50, v=1 << 51))
