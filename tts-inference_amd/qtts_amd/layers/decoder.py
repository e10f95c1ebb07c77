"""The talker decoder layer's linears with their neighbours fused (qtts/models/talker.py:246-271).

The reference's decode loop runs, per layer::

    q, k, v = attn.project(layer.input_layernorm(hidden))         # norm, qkv_proj
    ...attention...
    hidden = residual + attn.o_proj(out)                           # o_proj, add
    hidden = hidden + layer.mlp(layer.post_attention_layernorm(hidden))   # norm, MLP, add

Each helper here computes one of those lines from the reference's own modules (anything
with the same attributes): ``norm_linear`` is ``linear(norm(x))``, ``linear_residual`` is
``residual + linear(x)`` and ``norm_mlp_residual`` is ``hidden + mlp(norm(hidden))``.  When
the linears carry the int8 weight-only method on strip weights, the norm runs inside the
GEMM that follows it, the residual add in the GEMM's epilogue and GatedMLP's activation in
the gate_up GEMM's epilogue, so a layer is four launches.  Anything else computes the
reference's composition unchanged, so a caller can switch its loop over unconditionally.

``add_norm_linear`` and ``add_norm_mlp`` are for W8A8 linears (fp8 or int8, with or without adapters),
whose inputs are 8-bit codes: they carry the residual beside the hidden state, so that one kernel adds it,
normalizes the sum and quantizes the result::

    qkv, hidden = add_norm_linear(layer.input_layernorm, attn.qkv_proj, delta, hidden)
    ...attention...
    delta, hidden = add_norm_mlp(layer.post_attention_layernorm, layer.mlp, attn.o_proj(out), hidden)

``...attention...`` is ``out = attend(attn, qkv, cache, layer_index)`` over a :class:`~.attention.PagedCache`; :func:`paged_layer`
and :func:`paged_layer_w8a8` are a whole layer with it.
"""

from __future__ import annotations

import torch
import torch.nn.functional as F
from torch import nn

from .. import ops, torch_ops  # noqa: F401  (torch_ops registers torch.ops.qtts)
from ..quant.base import weight_flags
from .adapters import AdapterMethod
from .attention import PagedCache, attend
from .norm import is_rms_norm, norm_eps


def _int8_strips(linear: nn.Module, x: torch.Tensor) -> bool:
    """Whether ``linear`` runs x through the int8 weight-only strip kernels: its method, layout and
    x's dtype allow it, and its calibration routed x's row bucket to a kernel (not to F.linear on
    the kept weight, nor to the prefill route)."""
    method = getattr(linear, "quant_method", None)
    if not (getattr(method, "name", None) == "int8_weight_only" and getattr(linear, "int8_weight", None) is not None
            and getattr(linear, "int8_layout", None) == "strips" and x.is_cuda
            and x.dtype in (torch.bfloat16, torch.float16) and linear.in_features % 64 == 0):
        return False
    routed = getattr(method, "routes_to_kernel", None)
    return routed is None or routed(linear, x)


def _rms_norm_of(norm: nn.Module, x: torch.Tensor) -> bool:
    """Whether the kernels compute what ``norm`` does to x's rows: an RMSNorm of their width."""
    weight = getattr(norm, "weight", None)
    return weight is not None and weight.dim() == 1 and weight.shape[0] == x.shape[-1] and is_rms_norm(norm)


def norm_linear(norm: nn.Module, linear: nn.Module, x: torch.Tensor) -> torch.Tensor:
    """``linear(norm(x))``: input_layernorm + qkv_proj (talker.py:249), with the RMSNorm computed
    inside the int8 weight-only GEMM's prologue."""
    if _int8_strips(linear, x) and _rms_norm_of(norm, x):
        return torch.ops.qtts.w8a16_fused_gemm_strips(x, linear.int8_weight, linear.out_features, linear.int8_scale,
                                                      linear.bias, ops.PRO_RMS_NORM, norm.weight, norm_eps(norm),
                                                      None, ops.ALGO_AUTO | weight_flags(linear))
    return linear(norm(x))


def linear_residual(linear: nn.Module, x: torch.Tensor, residual: torch.Tensor) -> torch.Tensor:
    """``residual + linear(x)``: o_proj and the residual add (talker.py:270), the add in the GEMM's
    epilogue (the linear's output rounded to the activation dtype first, as torch adds two tensors)."""
    if _int8_strips(linear, x) and residual.shape[:-1] == x.shape[:-1] and residual.dtype == x.dtype:
        return torch.ops.qtts.w8a16_fused_gemm_strips(x, linear.int8_weight, linear.out_features, linear.int8_scale,
                                                      linear.bias, ops.PRO_NONE, None, 1e-6, residual,
                                                      ops.ALGO_AUTO | weight_flags(linear))
    return residual + linear(x)


def norm_mlp_residual(norm: nn.Module, mlp: nn.Module, hidden: torch.Tensor) -> torch.Tensor:
    """``hidden + mlp(norm(hidden))`` for a GatedMLP (talker.py:271; activation.py:142-147): the norm
    in the gate_up GEMM's prologue, ``silu(gate) * up`` in its epilogue, the residual add in the
    down GEMM's epilogue: two launches."""
    fused = getattr(mlp, "fuse", False)
    if (fused and _int8_strips(mlp.gate_up_proj, hidden) and mlp.gate_up_proj.out_features % 2 == 0
            and _rms_norm_of(norm, hidden)):
        up = mlp.gate_up_proj
        act = torch.ops.qtts.w8a16_gate_up_silu_strips(hidden, up.int8_weight, up.out_features, up.int8_scale,
                                                       up.bias, ops.PRO_RMS_NORM, norm.weight, norm_eps(norm),
                                                       ops.ALGO_AUTO | weight_flags(up))
        return linear_residual(mlp.down_proj, act, hidden)
    if fused:
        gate, up = mlp.gate_up_proj.split(mlp.gate_up_proj(norm(hidden)))
    else:
        h = norm(hidden)
        gate, up = mlp.gate_proj(h), mlp.up_proj(h)
    return hidden + mlp.down_proj(F.silu(gate) * up)


def _w8a8(linear: nn.Module, x: torch.Tensor):
    """``(method, codes)`` of a W8A8 linear on strip weights (its own method, or what its adapters stand on) that
    can take x as codes; None for any other."""
    method = getattr(linear, "quant_method", None)
    inner = method.inner if isinstance(method, AdapterMethod) else method
    name = getattr(inner, "name", None)
    if not x.is_cuda or x.dtype not in (torch.bfloat16, torch.float16):
        return None
    if name == "fp8" and getattr(linear, "fp8_layout", None) == "strips":
        return method, ops.CODE_E4M3
    if name == "int8" and getattr(linear, "int8_layout", None) == "strips":
        return method, ops.CODE_INT8
    return None


def _w8a8_linear(linear: nn.Module, method, codes: int, qx: torch.Tensor, sx: torch.Tensor, x: torch.Tensor | None,
                 shape: torch.Size, dtype: torch.dtype) -> torch.Tensor:
    """The linear on given codes; x: the 16-bit rows that its adapters read (None without adapters)."""
    algo = ops.ALGO_AUTO | weight_flags(linear)
    n = linear.out_features
    if codes == ops.CODE_E4M3:
        y = torch.ops.qtts.w8a8_fp8_gemm_strips(qx, sx, linear.fp8_weight, n, linear.fp8_scale.reshape(-1), linear.bias,
                                                dtype, algo)
    else:
        y = torch.ops.qtts.w8a8_int8_gemm_strips(qx, sx, linear.int8_weight, n, linear.int8_scale, linear.bias, dtype, algo)
    y = y.reshape(*shape[:-1], n)
    return y if x is None else linear.adapters.add(y, x, method.batch_for(linear, x))


def _add_norm_w8a8(norm: nn.Module, linear: nn.Module, found, x: torch.Tensor, residual: torch.Tensor | None):
    method, codes = found
    adapted = isinstance(method, AdapterMethod)
    qx, sx, hidden, normed = torch.ops.qtts.rms_norm_quant(x, norm.weight, norm_eps(norm), residual, codes, adapted)
    y = _w8a8_linear(linear, method, codes, qx, sx, normed if adapted else None, x.shape, x.dtype)
    return y, x if residual is None else hidden


def _norm_fits(norm: nn.Module, x: torch.Tensor, residual: torch.Tensor | None) -> bool:
    """Whether the kernel computes what ``norm`` does: an RMSNorm in x's type, of a residual like x."""
    return (_rms_norm_of(norm, x) and norm.weight.dtype == x.dtype
            and (residual is None or (residual.shape == x.shape and residual.dtype == x.dtype)))


def add_norm_linear(norm: nn.Module, linear: nn.Module, x: torch.Tensor, residual: torch.Tensor | None = None):
    """``hidden = residual + x`` (x without a residual) and ``linear(norm(hidden))``, as ``(output, hidden)``: for a W8A8
    linear one kernel up to its input's codes, then the GEMM on them.  The codes are made of the norm's fp32 value, which the
    linear's own quantizer would see rounded to 16 bits (int8: and with its scale in 16 bits): the output differs from
    ``linear(norm(hidden))`` by that rounding."""
    found = _w8a8(linear, x)
    if found is not None and _norm_fits(norm, x, residual):
        return _add_norm_w8a8(norm, linear, found, x, residual)
    hidden = x if residual is None else residual + x
    return linear(norm(hidden)), hidden


def add_norm_mlp(norm: nn.Module, mlp: nn.Module, x: torch.Tensor, residual: torch.Tensor | None = None):
    """``hidden = residual + x`` and ``mlp(norm(hidden))`` of a GatedMLP, as ``(output, hidden)``: with W8A8 linears both GEMMs
    take codes straight from their producers, the norm and ``silu(gate) * up``."""
    if getattr(mlp, "fuse", False):
        up, down = _w8a8(mlp.gate_up_proj, x), _w8a8(mlp.down_proj, x)
        if up is not None and down is not None and _norm_fits(norm, x, residual):
            gate_up, hidden = _add_norm_w8a8(norm, mlp.gate_up_proj, up, x, residual)
            method, codes = down
            adapted = isinstance(method, AdapterMethod)
            qx, sx, act = torch.ops.qtts.silu_mul_quant(gate_up, codes, adapted)
            y = _w8a8_linear(mlp.down_proj, method, codes, qx, sx, act if adapted else None, x.shape, x.dtype)
            return y, hidden
    hidden = x if residual is None else residual + x
    return mlp(norm(hidden)), hidden


def paged_layer(layer: nn.Module, hidden: torch.Tensor, cache: PagedCache, index: int, window: int = 0, sinks: int = 0,
                weights16: bool = False) -> torch.Tensor:
    """One decoder layer (talker.py:246-271) of the cache's step: ``layer.input_layernorm``, ``layer.attn`` (qkv_proj, q_norm, k_norm,
    o_proj), ``layer.post_attention_layernorm`` and ``layer.mlp``, with the neighbours inside int8 weight-only linears.  weights16:
    as in :func:`attend`."""
    attn = layer.attn
    out = attend(attn, norm_linear(layer.input_layernorm, attn.qkv_proj, hidden), cache, index, window, sinks, weights16=weights16)
    return norm_mlp_residual(layer.post_attention_layernorm, layer.mlp, linear_residual(attn.o_proj, out, hidden))


def paged_layer_w8a8(layer: nn.Module, delta: torch.Tensor, hidden: torch.Tensor | None, cache: PagedCache, index: int, window: int = 0,
                     sinks: int = 0, weights16: bool = False):
    """The same as ``(delta, hidden)`` for W8A8 linears, the residual beside the hidden state as in :func:`add_norm_linear`."""
    attn = layer.attn
    qkv, hidden = add_norm_linear(layer.input_layernorm, attn.qkv_proj, delta, hidden)
    out = attend(attn, qkv, cache, index, window, sinks, weights16=weights16)
    return add_norm_mlp(layer.post_attention_layernorm, layer.mlp, attn.o_proj(out), hidden)
