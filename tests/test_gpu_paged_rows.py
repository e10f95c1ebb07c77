"""Rows at the edges of a paged batch: rows of no request, rows whose slots and counts disagree, rows that a captured step was not
made for."""

from __future__ import annotations

import pytest
import torch

from test_gpu_paged import U, _batch, _near

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
