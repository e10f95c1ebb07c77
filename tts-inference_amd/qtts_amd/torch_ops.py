"""The quantized-linear entry points as torch custom ops (``torch.ops.qtts.*``).

The quant methods' ``apply`` and the decoder-layer helpers call these, so graph capture,
``torch.compile`` and ``torch._dynamo`` see each quantized linear as one opaque op with a
known output shape instead of a ctypes call they cannot trace (the reference compiles the
code predictor's prefix forward with ``torch.compile(dynamic=True)``,
qtts/models/code_predictor.py:186-192).  Each op's real implementation is the ``ops``
wrapper of the same name (one C-ABI call on torch's current stream); its fake
implementation only computes the output's shape and dtype, so tracing never touches a
device.  The ops are functional: every output is a fresh tensor.
"""

from __future__ import annotations

from typing import Optional

import torch
import torch.nn.functional as F

from . import ops

_LIB = "qtts"


def _rows_shape(x: torch.Tensor, n) -> tuple:
    return (*x.shape[:-1], n)


# ---- int8 weight-only (W8A16), qtts/quant/kernels.py:138-178 -------------------------------

@torch.library.custom_op(f"{_LIB}::w8a16_gemm", mutates_args=())
def w8a16_gemm(x: torch.Tensor, q: torch.Tensor, scale: torch.Tensor, bias: Optional[torch.Tensor],
               algo: int) -> torch.Tensor:
    return ops.w8a16_gemm(x, q, scale, bias, algo)


@w8a16_gemm.register_fake
def _(x, q, scale, bias, algo):
    return x.new_empty(_rows_shape(x, q.shape[0]))


@torch.library.custom_op(f"{_LIB}::w8a16_gemm_strips", mutates_args=())
def w8a16_gemm_strips(x: torch.Tensor, qs: torch.Tensor, n: int, scale: torch.Tensor, bias: Optional[torch.Tensor],
                      algo: int) -> torch.Tensor:
    return ops.w8a16_gemm_strips(x, qs, n, scale, bias, algo)


@w8a16_gemm_strips.register_fake
def _(x, qs, n, scale, bias, algo):
    return x.new_empty(_rows_shape(x, n))


# ---- fp8 W8A8 (Fp8Method.apply, qtts/quant/fp8.py:72-89) ------------------------------------

@torch.library.custom_op(f"{_LIB}::fp8_linear", mutates_args=())
def fp8_linear(x: torch.Tensor, qw: torch.Tensor, sw: torch.Tensor, bias: Optional[torch.Tensor], div_mode: int,
               algo: int) -> torch.Tensor:
    return ops.fp8_linear(x, qw, sw, bias, div_mode, algo)


@fp8_linear.register_fake
def _(x, qw, sw, bias, div_mode, algo):
    return x.new_empty(_rows_shape(x, qw.shape[0]))


@torch.library.custom_op(f"{_LIB}::fp8_linear_strips", mutates_args=())
def fp8_linear_strips(x: torch.Tensor, qws: torch.Tensor, n: int, sw: torch.Tensor, bias: Optional[torch.Tensor],
                      div_mode: int, algo: int) -> torch.Tensor:
    return ops.fp8_linear_strips(x, qws, n, sw, bias, div_mode, algo)


@fp8_linear_strips.register_fake
def _(x, qws, n, sw, bias, div_mode, algo):
    return x.new_empty(_rows_shape(x, n))


# ---- int8 W8A8 (Int8Method.apply, qtts/quant/int8.py:145-160) -------------------------------

@torch.library.custom_op(f"{_LIB}::int8_linear", mutates_args=())
def int8_linear(x: torch.Tensor, qw: torch.Tensor, sw: torch.Tensor, bias: Optional[torch.Tensor], div_mode: int,
                algo: int) -> torch.Tensor:
    return ops.int8_linear(x, qw, sw, bias, div_mode, algo)


@int8_linear.register_fake
def _(x, qw, sw, bias, div_mode, algo):
    return x.new_empty(_rows_shape(x, qw.shape[0]))


@torch.library.custom_op(f"{_LIB}::int8_linear_strips", mutates_args=())
def int8_linear_strips(x: torch.Tensor, qws: torch.Tensor, n: int, sw: torch.Tensor, bias: Optional[torch.Tensor],
                       div_mode: int, algo: int) -> torch.Tensor:
    return ops.int8_linear_strips(x, qws, n, sw, bias, div_mode, algo)


@int8_linear_strips.register_fake
def _(x, qws, n, sw, bias, div_mode, algo):
    return x.new_empty(_rows_shape(x, n))


# ---- fp8 weight-only (Fp8WeightOnlyMethod, qtts/quant/fp8.py:92-123) ------------------------

@torch.library.custom_op(f"{_LIB}::fp8w_gemm_strips", mutates_args=())
def fp8w_gemm_strips(x: torch.Tensor, qs: torch.Tensor, n: int, scale: torch.Tensor, bias: Optional[torch.Tensor],
                     algo: int) -> torch.Tensor:
    return ops.fp8w_gemm_strips(x, qs, n, scale, bias, algo)


@fp8w_gemm_strips.register_fake
def _(x, qs, n, scale, bias, algo):
    return x.new_empty(_rows_shape(x, n))


# ---- the weight-only methods' prefill route (quant/prefill.py) ------------------------------

@torch.library.custom_op(f"{_LIB}::dequant_linear", mutates_args=())
def dequant_linear(x: torch.Tensor, qs: torch.Tensor, codes: int, n: int, k: int, scale: torch.Tensor,
                   bias: Optional[torch.Tensor]) -> torch.Tensor:
    """``F.linear(x, dtype(codes * scale[:, None]), bias)``: the codes dequantized into the device's
    scratch buffer, then the library GEMM."""
    w = ops.dequant_scratch(x.device, n, k, x.dtype)
    ops.dequant_strips(qs, n, k, scale, x.dtype, codes, out=w)
    return F.linear(x, w, bias)


@dequant_linear.register_fake
def _(x, qs, codes, n, k, scale, bias):
    return x.new_empty(_rows_shape(x, n))


# ---- decoder-layer neighbours (qtts/layers/norm.py, activation.py; talker.py:246-271) -------

@torch.library.custom_op(f"{_LIB}::rms_norm", mutates_args=())
def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float) -> torch.Tensor:
    return ops.rms_norm(x, weight, eps)


@rms_norm.register_fake
def _(x, weight, eps):
    return torch.empty_like(x)


@torch.library.custom_op(f"{_LIB}::silu_mul", mutates_args=())
def silu_mul(gate_up: torch.Tensor) -> torch.Tensor:
    return ops.silu_mul(gate_up)


@silu_mul.register_fake
def _(gate_up):
    return gate_up.new_empty(_rows_shape(gate_up, gate_up.shape[-1] // 2))


@torch.library.custom_op(f"{_LIB}::w8a16_silu_mul_gemm_strips", mutates_args=())
def w8a16_silu_mul_gemm_strips(gate_up: torch.Tensor, qs: torch.Tensor, n: int, scale: torch.Tensor,
                               bias: Optional[torch.Tensor], algo: int) -> torch.Tensor:
    return ops.w8a16_silu_mul_gemm_strips(gate_up, qs, n, scale, bias, algo)


@w8a16_silu_mul_gemm_strips.register_fake
def _(gate_up, qs, n, scale, bias, algo):
    return gate_up.new_empty(_rows_shape(gate_up, n))


@torch.library.custom_op(f"{_LIB}::w8a16_fused_gemm_strips", mutates_args=())
def w8a16_fused_gemm_strips(x: torch.Tensor, qs: torch.Tensor, n: int, scale: torch.Tensor,
                            bias: Optional[torch.Tensor], prologue: int, norm_weight: Optional[torch.Tensor],
                            eps: float, residual: Optional[torch.Tensor], algo: int) -> torch.Tensor:
    return ops.w8a16_fused_gemm_strips(x, qs, n, scale, bias, prologue=prologue, norm_weight=norm_weight, eps=eps,
                                       residual=residual, algo=algo)


@w8a16_fused_gemm_strips.register_fake
def _(x, qs, n, scale, bias, prologue, norm_weight, eps, residual, algo):
    return x.new_empty(_rows_shape(x, n))


@torch.library.custom_op(f"{_LIB}::w8a16_gate_up_silu_strips", mutates_args=())
def w8a16_gate_up_silu_strips(x: torch.Tensor, qs: torch.Tensor, n: int, scale: torch.Tensor,
                              bias: Optional[torch.Tensor], prologue: int, norm_weight: Optional[torch.Tensor],
                              eps: float, algo: int) -> torch.Tensor:
    return ops.w8a16_gate_up_silu_strips(x, qs, n, scale, bias, prologue=prologue, norm_weight=norm_weight, eps=eps,
                                         algo=algo)


@w8a16_gate_up_silu_strips.register_fake
def _(x, qs, n, scale, bias, prologue, norm_weight, eps, algo):
    return x.new_empty(_rows_shape(x, n // 2))


# ---- the W8A8 GEMMs on given codes, and the codes' producers --------------------------------

def _reserve(op: int, qx: torch.Tensor, n: int, algo: int) -> None:
    """Workspace for rows past what the quant method reserved at load time."""
    rows, k = qx.shape
    ops._ensure_workspace(qx.device, ops.workspace_bytes(op, rows, n, k, algo), "w8a8_gemm_strips")


@torch.library.custom_op(f"{_LIB}::w8a8_fp8_gemm_strips", mutates_args=())
def w8a8_fp8_gemm_strips(qx: torch.Tensor, sx: torch.Tensor, qws: torch.Tensor, n: int, sw: torch.Tensor,
                         bias: Optional[torch.Tensor], out_dtype: torch.dtype, algo: int) -> torch.Tensor:
    _reserve(ops.OP_W8A8_FP8, qx, n, algo)
    return ops.w8a8_fp8_gemm_strips(qx, sx, qws, n, sw, bias, out_dtype, algo)


@torch.library.custom_op(f"{_LIB}::w8a8_int8_gemm_strips", mutates_args=())
def w8a8_int8_gemm_strips(qx: torch.Tensor, sx: torch.Tensor, qws: torch.Tensor, n: int, sw: torch.Tensor,
                          bias: Optional[torch.Tensor], out_dtype: torch.dtype, algo: int) -> torch.Tensor:
    _reserve(ops.OP_W8A8_INT8, qx, n, algo)
    return ops.w8a8_int8_gemm_strips(qx, sx, qws, n, sw, bias, out_dtype, algo)


@w8a8_fp8_gemm_strips.register_fake
@w8a8_int8_gemm_strips.register_fake
def _(qx, sx, qws, n, sw, bias, out_dtype, algo):
    return qx.new_empty((qx.shape[0], n), dtype=out_dtype)


_CODES = {ops.CODE_INT8: torch.int8, ops.CODE_E4M3: torch.float8_e4m3fn}


def _fake_codes(x, k, codes):
    rows = 1
    for d in x.shape[:-1]:
        rows = rows * d
    return x.new_empty((rows, k), dtype=_CODES[codes]), x.new_empty((rows,), dtype=torch.float32)


def _or_empty(t: Optional[torch.Tensor], x: torch.Tensor) -> torch.Tensor:
    return x.new_empty(0) if t is None else t


@torch.library.custom_op(f"{_LIB}::rms_norm_quant", mutates_args=())
def rms_norm_quant(x: torch.Tensor, weight: torch.Tensor, eps: float, residual: Optional[torch.Tensor], codes: int,
                   want_normed: bool) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """``ops.rms_norm_quant``; an output that was not asked for is an empty tensor."""
    qx, sx, hidden, normed = ops.rms_norm_quant(x, weight, eps, residual, codes, want_normed)
    return qx, sx, _or_empty(hidden, x), _or_empty(normed, x)


@rms_norm_quant.register_fake
def _(x, weight, eps, residual, codes, want_normed):
    qx, sx = _fake_codes(x, x.shape[-1], codes)
    return qx, sx, x.new_empty(x.shape if residual is not None else 0), x.new_empty(x.shape if want_normed else 0)


@torch.library.custom_op(f"{_LIB}::silu_mul_quant", mutates_args=())
def silu_mul_quant(gate_up: torch.Tensor, codes: int, want_act: bool) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``ops.silu_mul_quant``; the 16-bit value is an empty tensor unless asked for."""
    qx, sx, act = ops.silu_mul_quant(gate_up, codes, want_act)
    return qx, sx, _or_empty(act, gate_up)


@silu_mul_quant.register_fake
def _(gate_up, codes, want_act):
    k = gate_up.shape[-1] // 2
    qx, sx = _fake_codes(gate_up, k, codes)
    return qx, sx, gate_up.new_empty(_rows_shape(gate_up, k) if want_act else 0)


# ---- low-rank adapters (layers/adapters.py) ---------------------------------------------------

@torch.library.custom_op(f"{_LIB}::lora_add", mutates_args=())
def lora_add(base: torch.Tensor, x: torch.Tensor, index: torch.Tensor, plan: Optional[torch.Tensor], slots: int,
             a: torch.Tensor, b: torch.Tensor, scaling: torch.Tensor, ranks: Optional[torch.Tensor],
             partitions: list[int]) -> torch.Tensor:
    return ops.lora_add(base, x, ops.LoraBatch(index, slots, plan), a, b, scaling, ranks, partitions)


@lora_add.register_fake
def _(base, x, index, plan, slots, a, b, scaling, ranks, partitions):
    return base.new_empty(base.shape)


# ---- attention over a paged cache (layers/attention.py) ---------------------------------------

def _batch(state: list[torch.Tensor], bounds: list[int]) -> "ops.PagedBatch":
    """A step's batch from its tensors (table, starts, counts, lengths, positions, slots) and page size, max_new, min_new and
    whether max_new is of this step alone (no, where it is left out)."""
    return ops.PagedBatch(*state, bounds[0], max_new=bounds[1], min_new=bounds[2], this_step=any(bounds[3:]))


@torch.library.custom_op(f"{_LIB}::qkv_to_cache", mutates_args=("k", "v"))
def qkv_to_cache(qkv: torch.Tensor, k: torch.Tensor, v: torch.Tensor, state: list[torch.Tensor], bounds: list[int], heads: int,
                 q_norm: Optional[torch.Tensor], k_norm: Optional[torch.Tensor], eps: float, cos: Optional[torch.Tensor],
                 sin: Optional[torch.Tensor]) -> torch.Tensor:
    return ops.qkv_to_cache(qkv, k, v, _batch(state, bounds), heads, q_norm, k_norm, eps, None if cos is None else (cos, sin))


@qkv_to_cache.register_fake
def _(qkv, k, v, state, bounds, heads, q_norm, k_norm, eps, cos, sin):
    return qkv.new_empty((state[4].shape[0], heads, k.shape[3]))


@torch.library.custom_op(f"{_LIB}::paged_attention", mutates_args=())
def paged_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, state: list[torch.Tensor], bounds: list[int], window: int,
                    sinks: int, scale: float, weights16: bool = False) -> torch.Tensor:
    return ops.paged_attention(q, k, v, _batch(state, bounds), window, sinks, scale, weights16)


@paged_attention.register_fake
def _(q, k, v, state, bounds, window, sinks, scale, weights16=False):
    return q.new_empty(q.shape)


#: Every op this module registers, by name (``torch.ops.qtts.<name>``).
OPS = ("w8a16_gemm", "w8a16_gemm_strips", "fp8_linear", "fp8_linear_strips", "int8_linear", "int8_linear_strips",
       "fp8w_gemm_strips", "dequant_linear", "rms_norm", "silu_mul", "w8a16_silu_mul_gemm_strips",
       "w8a16_fused_gemm_strips", "w8a16_gate_up_silu_strips", "w8a8_fp8_gemm_strips", "w8a8_int8_gemm_strips",
       "rms_norm_quant", "silu_mul_quant", "lora_add", "qkv_to_cache", "paged_attention")
