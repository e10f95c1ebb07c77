"""Which modules are RMSNorms that the fused kernels compute (qtts/layers/norm.py:50-93).

The decoder helpers take a model's own norm modules, known by their attributes alone, and run the kernels' formula
``x / sqrt(mean(x^2) + eps) * weight`` in their place.  Attributes do not tell that formula from ``1 + weight``, a mean taken
off or another place of eps, so each module is asked once, with a weight and rows of its width: on the CPU, or on its GPU
where it runs there alone.
"""

from __future__ import annotations

import copy

import torch
from torch import nn

#: The answer, kept on the module.
_ANSWER = "_is_rms_norm"


def norm_eps(norm: nn.Module) -> float | None:
    """The norm's eps, under the names that RMSNorms give it; None where it has none."""
    for attr in ("eps", "variance_epsilon"):
        if hasattr(norm, attr):
            eps = getattr(norm, attr)
            return None if eps is None else float(eps)
    return None


def _holds(norm: nn.Module, eps: float, device: torch.device, dtype: torch.dtype) -> bool:
    """Whether ``norm``, with a weight of this device and type in its own's place, gives the formula's rows."""
    k = norm.weight.shape[0]
    g = torch.Generator(device="cpu").manual_seed(k)
    weight = (torch.rand(k, generator=g, dtype=torch.float32, device="cpu") * 2 - 0.5).to(dtype)
    # an ordinary row, one whose square is about eps, a large one, each off centre
    x = torch.randn(3, k, generator=g, dtype=torch.float32, device="cpu") + 0.5
    x = (x * torch.tensor([[1.0], [max(eps, 1e-12) ** 0.5], [50.0]], device="cpu")).to(dtype)
    twin = copy.copy(norm)  # shares the module's attributes, but for the weight
    twin._parameters, twin._buffers = dict(norm._parameters), dict(norm._buffers)
    if "weight" in twin._parameters:
        twin._parameters["weight"] = nn.Parameter(weight.to(device), requires_grad=False)
    else:
        twin._buffers["weight"] = weight.to(device)
    with torch.no_grad():
        y = twin(x.to(device))
    x, weight = x.float(), weight.float()
    want = x * torch.rsqrt(x.square().mean(1, keepdim=True) + eps) * weight
    if not torch.is_tensor(y) or y.shape != want.shape:
        return False
    # 2^-6 of the row's largest: past the roundings to 16 bits on the way, far below another formula
    return bool(((y.float().cpu() - want).abs() <= 2.0 ** -6 * want.abs().amax(1, keepdim=True)).all())


def _ask(norm: nn.Module) -> bool | None:
    """Whether ``norm`` computes RMSNorm; None where it cannot be asked now."""
    held = {name: t for name, t in (*norm.named_parameters(), *norm.named_buffers())}
    eps = norm_eps(norm)
    if set(held) != {"weight"} or held["weight"].dim() != 1 or not held["weight"].numel() or eps is None:
        return False
    if type(torch.empty(0)) is not torch.Tensor:  # under fake tensors
        return None
    try:
        return _holds(norm, eps, torch.device("cpu"), torch.float32)
    except Exception:  # a norm of a GPU kernel alone is asked there, in its own type
        weight = held["weight"]
        if not weight.is_cuda:
            return False
        if torch.cuda.is_current_stream_capturing():
            return None
        try:
            return _holds(norm, eps, weight.device, weight.dtype)
        except Exception:
            return False


def is_rms_norm(norm: nn.Module) -> bool:
    """Whether ``norm`` is an RMSNorm of one weight, as :func:`mark_rms_norms` or its first eager call found."""
    answer = norm.__dict__.get(_ANSWER)
    if answer is None:
        if torch.compiler.is_compiling():  # nothing to ask while tracing: the norm itself is traced
            return False
        answer = _ask(norm)
        if answer is None:
            return False
        norm.__dict__[_ANSWER] = answer
    return answer


def mark_rms_norms(module: nn.Module) -> int:
    """Ask every norm under ``module`` ahead of its first call (a traced or captured one then knows); returns how many are RMSNorms."""
    return sum(is_rms_norm(m) for m in module.modules()
               if getattr(m, "weight", None) is not None and (hasattr(m, "eps") or hasattr(m, "variance_epsilon")))
