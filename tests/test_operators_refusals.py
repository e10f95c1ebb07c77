"""What the operators around the quantized linears refuse (8-bit activations from their producers, low-rank adapters),
without a GPU: the C entries check every argument before any device use, the wrappers shapes and types before the call."""

from __future__ import annotations

import ctypes

import pytest
import torch

from qtts_amd import _lib, ops

P = ctypes.c_void_p


def _buf(n=1 << 16):
    return ctypes.create_string_buffer(n)


def _at(buf, off=0):
    return ctypes.addressof(buf) + off


def _refused(status, text):
    assert status == -1 and text in _lib.last_error(), (status, _lib.last_error())


def test_norm_quant_entry():
    L = _lib.load()
    b = _buf()
    at = lambda off: _at(b, off)  # noqa: E731

    def call(x=0, dt=1, m=2, k=64, ldx=64, res=4096, ldr=64, w=8192, codes=1, q=12288, sx=16384, hid=20480, ldh=64, nrm=24576,
             ldn=64):
        ptr = lambda v: None if v is None else at(v)  # noqa: E731
        return L.qtts_rms_norm_quant(ptr(x), dt, m, k, ldx, ptr(res), ldr, ptr(w), 1e-6, codes, ptr(q), ptr(sx), ptr(hid), ldh,
                                     ptr(nrm), ldn, None)

    _refused(call(m=-1), "negative size")
    _refused(call(m=1 << 31), "too large")
    _refused(call(k=1 << 31, ldx=1 << 31), "too large")
    _refused(call(dt=3), "dtype")
    _refused(call(codes=2), "code kind")
    for ld in ({"ldx": 63}, {"ldr": 63}, {"ldh": 63}, {"ldn": 63}):
        _refused(call(**ld), "leading dimension")
    for null in ("x", "w", "q", "sx"):
        _refused(call(**{null: None}), "null pointer")
    _refused(call(q=0), "qx overlaps")
    _refused(call(q=4096 + 64), "qx overlaps")
    _refused(call(hid=2), "hidden overlaps x")
    _refused(call(hid=4096, ldh=72), "hidden overlaps the residual")
    _refused(call(nrm=20480 + 100), "normed overlaps")
    _refused(call(nrm=0), "normed overlaps")
    assert call(m=0) == 0  # empty: no device needed
    if not torch.cuda.is_available():
        for fine in ({"hid": 0}, {"hid": 4096}, {"res": None, "hid": None, "nrm": None}, {}):
            assert call(**fine) == -2, _lib.last_error()  # past the checks: no device here


def test_silu_quant_entry():
    L = _lib.load()
    b = _buf()

    def call(x=0, dt=1, m=2, k=64, ld=128, codes=0, q=8192, sx=16384, act=20480, lda=64):
        ptr = lambda v: None if v is None else _at(b, v)  # noqa: E731
        return L.qtts_silu_mul_quant(ptr(x), dt, m, k, ld, codes, ptr(q), ptr(sx), ptr(act), lda, None)

    _refused(call(k=-1), "negative size")
    _refused(call(k=1 << 30, ld=1 << 31), "too large")
    _refused(call(dt=-1), "dtype")
    _refused(call(codes=7), "code kind")
    _refused(call(ld=127), "leading dimension")
    _refused(call(lda=63), "leading dimension")
    for null in ("x", "q", "sx"):
        _refused(call(**{null: None}), "null pointer")
    _refused(call(q=100), "qx overlaps")
    _refused(call(act=128), "act overlaps")
    assert call(m=0) == 0


def test_lora_entry():
    L = _lib.load()
    b = _buf(1 << 20)
    need = L.qtts_workspace_bytes(_lib.OP_LORA, 4, 1, 16, 0)
    assert need >= 4 * 16 * 4
    assert L.qtts_workspace_bytes(_lib.OP_LORA, 4, 9, 16, 0) == -1 and L.qtts_workspace_bytes(_lib.OP_LORA, 4, 1, 129, 0) == -1

    def call(x=0, dt=1, m=4, k=64, ldx=64, index=4096, slots=3, a=8192, bb=65536, rank=16, ranks=131072, scaling=131200,
             ends=(96,), base=140000, ldb=96, out=160000, n=96, ldo=96, ws=262144, ws_n=None, parts=None):
        ptr = lambda v: None if v is None else _at(b, v)  # noqa: E731
        arr = None if ends is None else (ctypes.c_int64 * max(1, len(ends)))(*ends)
        return L.qtts_lora_add(ptr(x), dt, m, k, ldx, ptr(index), None, slots, ptr(a), ptr(bb), rank, ptr(ranks), ptr(scaling),
                               arr, len(ends or ()) if parts is None else parts, ptr(base), ldb, ptr(out), n, ldo, ptr(ws),
                               need if ws_n is None else ws_n, None)

    _refused(call(m=-1), "negative size")
    _refused(call(slots=-1), "negative size")
    _refused(call(n=1 << 30, ldb=1 << 30, ldo=1 << 30), "too large")
    _refused(call(dt=0), "bf16 or fp16")
    _refused(call(rank=0), "rank")
    _refused(call(rank=129), "rank")
    _refused(call(ends=()), "partitions")
    _refused(call(ends=None, parts=1), "partitions")
    _refused(call(ends=(8,) * 8 + (96,)), "partitions")
    _refused(call(ends=(64, 32, 96)), "ascend")
    _refused(call(ends=(-1, 96)), "ascend")
    _refused(call(ends=(64,)), "the partitions end")
    _refused(call(ldx=63), "leading dimension")
    _refused(call(ldo=95), "leading dimension")
    for null in ("x", "index", "a", "bb", "scaling", "base", "out"):
        _refused(call(**{null: None}), "null pointer")
    _refused(call(out=140002), "out overlaps base")
    _refused(call(out=140000, ldo=104), "out overlaps base")
    _refused(call(out=64, ldo=96), "out overlaps x")
    for ws in ({"ws": None}, {"ws_n": need - 1}):
        assert call(**ws) == -5 and "workspace" in _lib.last_error()
    assert call(m=0) == 0 and call(n=0, ends=(0,)) == 0
    if not torch.cuda.is_available():
        assert call() == -2 and call(out=140000) == -2 and call(ranks=None) == -2 and call(ends=(0, 32, 32, 96), rank=4, ws_n=1 << 17) == -2


def test_lora_plan_entry():
    L = _lib.load()
    b = _buf()
    at = (_at(b) + 15) & ~15
    need = L.qtts_lora_plan_bytes(100, 4)
    assert need >= 4 * 100 and L.qtts_lora_plan_bytes(0, 0) > 0
    assert L.qtts_lora_plan_bytes(100, 769) == 0  # more than a plan takes
    for m, slots in ((-1, 4), (100, -1), (1 << 31, 4), (100, 1 << 30)):
        assert L.qtts_lora_plan_bytes(m, slots) == -1 and L.qtts_lora_plan(at, m, slots, at, 1 << 40, None) == -1
    _refused(L.qtts_lora_plan(at, 100, 769, at, 1 << 20, None), "slots")
    _refused(L.qtts_lora_plan(None, 100, 4, at, need, None), "null")
    _refused(L.qtts_lora_plan(at, 100, 4, None, need, None), "null")
    _refused(L.qtts_lora_plan(at, 100, 4, at + 4, need, None), "unaligned")
    _refused(L.qtts_lora_plan(at, 100, 4, at, need - 1, None), "needed")


def test_wrappers_check_shapes_and_types():
    bf, f32, i32 = torch.bfloat16, torch.float32, torch.int32
    x, w = torch.zeros(2, 64, dtype=bf), torch.ones(64, dtype=bf)
    with pytest.raises(ValueError, match="GPU tensor"):
        ops.rms_norm_quant(x, w)
    with pytest.raises(ValueError, match="norm weight"):
        ops.rms_norm_quant(x, w[:32])
    with pytest.raises(ValueError, match="residual"):
        ops.rms_norm_quant(x, w, residual=x[:, :32])
    with pytest.raises(ValueError, match="residual"):
        ops.rms_norm_quant(x, w, residual=x.float())
    with pytest.raises(ValueError, match="odd last dimension"):
        ops.silu_mul_quant(torch.zeros(2, 63, dtype=bf))
    with pytest.raises(ValueError, match="GPU tensor"):
        ops.silu_mul_quant(x)
    index = torch.zeros(2, dtype=i32)
    for bad in (index.long(), index.view(1, 2), torch.zeros(4, dtype=i32)[::2]):
        with pytest.raises(ValueError, match="index"):
            ops.lora_batch(bad, 3)
    with pytest.raises(ValueError, match="negative"):
        ops.lora_batch(index, -1)
    with pytest.raises(ValueError, match="GPU tensor"):
        ops.lora_batch(index, 3)
    batch = ops.LoraBatch(index, 3)
    a, b, s = torch.zeros(3, 32, 64, dtype=bf), torch.zeros(3, 96, 16, dtype=bf), torch.ones(3)
    base = torch.zeros(2, 96, dtype=bf)

    def call(base=base, x=x, batch=batch, a=a, b=b, s=s, ranks=None, parts=(64, 32)):
        return ops.lora_add(base, x, batch, a, b, s, ranks, parts)

    for match, kw in (("rows", {"base": base[:1]}), ("rows", {"batch": ops.LoraBatch(index[:1], 3)}),
                      ("one dtype", {"x": x.half()}), ("one dtype", {"a": a.float()}),
                      ("contiguous", {"a": a.transpose(1, 2)}), ("do not fit", {"b": b[0]}), ("do not fit", {"parts": (96,)}),
                      ("do not fit", {"parts": (64, 31)}), ("do not fit", {"a": a[:, :16].contiguous()}),
                      ("do not fit", {"b": b[:2]}),
                      ("partition of", {"parts": (100, -4)}),
                      ("at most", {"a": torch.zeros(3, 258, 64, dtype=bf), "b": torch.zeros(3, 96, 129, dtype=bf)}), ("scaling", {"s": s.to(bf)}), ("scaling", {"s": s[:2]}),
                      ("ranks", {"ranks": torch.zeros(3)}), ("ranks", {"ranks": torch.zeros(2, dtype=i32)}),
                      ("GPU tensor", {})):
        with pytest.raises(ValueError, match=match):
            call(**kw)


def test_a_torch_without_gpu_bindings_imports_and_refuses():
    """A CPU build of torch has no device and stream calls in its bindings: the package imports there (its checkers, packers' formats
    and configuration need no GPU) and an operator refuses the CPU tensor."""
    import os
    import subprocess
    import sys

    code = """
import torch
for name in ("_cuda_getDevice", "_cuda_getCurrentRawStream"):
    if hasattr(torch._C, name):
        delattr(torch._C, name)
from qtts_amd import ops
for call in (lambda: ops.rms_norm_quant(torch.zeros(2, 64), torch.ones(64)), lambda: ops.silu_mul_quant(torch.zeros(2, 64)),
             lambda: ops.lora_batch(torch.zeros(2, dtype=torch.int32), 3)):
    try:
        call()
    except ValueError as e:
        assert "GPU tensor" in str(e), e
    else:
        raise AssertionError("ran on the CPU")
print("refused")
"""
    env = dict(os.environ, PYTHONPATH=os.pathsep.join(sys.path))
    done = subprocess.run([sys.executable, "-c", code], env=env, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "refused" in done.stdout, done.stderr


def test_lora_add_fresh_entry_checks_as_lora_add_does():
    L = _lib.load()
    b = _buf(1 << 20)
    ends = (ctypes.c_int64 * 1)(96)
    for m, rank, out, ws_n, text in ((-1, 16, 160000, 1 << 18, "negative"), (4, 129, 160000, 1 << 18, "rank"),
                                     (4, 16, 140002, 1 << 18, "out overlaps base"), (4, 16, 160000, 8, "workspace")):
        status = [add(_at(b), 1, m, 64, 64, _at(b, 4096), None, 3, _at(b, 8192), _at(b, 65536), rank, None, _at(b, 131200), ends, 1,
                      _at(b, 140000), 96, _at(b, out), 96, 96, _at(b, 262144), ws_n, None)
                  for add in (L.qtts_lora_add, L.qtts_lora_add_fresh)]
        assert status[0] == status[1] < 0 and text in _lib.last_error()
