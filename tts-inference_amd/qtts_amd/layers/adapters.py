"""Low-rank adapters of many requests on a model's linears.

A served batch mixes requests of different fine-tunings: every row may carry its own adapter, a low-rank
``scaling * (x A^T) B^T`` beside the projection that all rows share.  The reference has no adapters; this
hangs them on the same hook its quant methods use, so the model code does not change:

* :class:`LinearAdapters` holds the adapters of one linear, ``slots`` of them of up to ``rank``, on
  whatever the linear runs (any quant method, or F.linear).  A merged qkv or gate_up has an A and a B for
  each of its partitions;
* :class:`AdapterRouting` says which slot each row of the step takes, for every linear of the model;
* :class:`AdapterMethod` is the quant method that adds the one to the other;
* :func:`attach_adapters` puts them on a model, before or after ``apply_quantization``.

Per step, a serving loop sets the routing, then runs the model::

    routing = AdapterRouting(slots=32, max_rows=64, device="cuda")
    banks = attach_adapters(talker, slots=32, rank=16, routing=routing)
    banks["layers.0.attn.qkv_proj"].load(3, [a_q, a_k, a_v], [b_q, b_k, b_v], scaling=alpha / r)
    ...
    routing.set([3, 3, -1, 7], rows=8)      # four requests padded to the captured batch of 8
    graph.replay()                           # reads the routing's buffers
"""

from __future__ import annotations

from typing import Sequence

import torch
import torch.nn.functional as F
from torch import nn

from .. import ops, torch_ops  # noqa: F401  (torch_ops registers torch.ops.qtts)
from ..quant.base import QuantMethodBase
from .linear import iter_linears


class AdapterRouting:
    """Which adapter slot each row takes (-1: none), in buffers that keep their addresses: a graph captured while the
    routing was set reads, on every replay, what the last :meth:`set` wrote.  A graph of another row count than that one's
    takes its rows' slots from it all the same, and no adapter for rows that it does not have."""

    def __init__(self, slots: int, max_rows: int, device: torch.device | str = "cuda") -> None:
        if slots < 1 or max_rows < 1:
            raise ValueError(f"an adapter routing needs slots and rows, got {slots} and {max_rows}")
        self.slots, self.max_rows = int(slots), int(max_rows)
        # One buffer, the index (as far as 16 bytes go), then the plan: one write clears the index's end and the plan's head.
        words, at = ops.lora_plan_buffer(self.max_rows, self.slots, torch.device("meta")).numel(), (self.max_rows + 3) // 4 * 4
        buffer = torch.full((at + words,), -1, dtype=torch.int32, device=device)
        self.index, self._plan = buffer[:self.max_rows], buffer[at:]
        self._live = buffer[:at + min(words, 4)]  # what a set writes
        self.batch: ops.LoraBatch | None = None

    def set(self, index: torch.Tensor | Sequence[int], rows: int | None = None) -> ops.LoraBatch:
        """The slots of the step's rows, ``rows`` of them with padding rows (no adapter) behind ``index``."""
        index = torch.as_tensor(index)
        if index.dim() != 1:
            raise ValueError(f"index must be 1-D, got shape {tuple(index.shape)}")
        given = index.shape[0]
        if given and (index.dtype == torch.bool or index.is_floating_point() or index.is_complex()):
            raise ValueError(f"index must hold whole numbers, got {index.dtype}")
        rows = given if rows is None else int(rows)
        if not given <= rows <= self.max_rows:
            raise ValueError(f"{given} rows padded to {rows} do not fit a routing of {self.max_rows}")
        if index.dtype != torch.int32:  # what int32 cannot hold is no slot either
            index = index.to(torch.int64).clamp(-1, self.slots).to(torch.int32)
        self.batch = None  # nothing stands if what follows fails
        # The rows behind the given ones have no adapter and the plan is of no batch, also for captured steps of other row counts.
        if index.device == self._live.device:
            self._live[:given].copy_(index)
            self._live[given:].fill_(-1)
        else:
            self._live.copy_(F.pad(index, (0, self._live.shape[0] - given), value=-1))
        self.batch = ops.lora_batch(self.index[:rows], self.slots, self._plan)
        return self.batch


class LinearAdapters(nn.Module):
    """``slots`` adapters of rank up to ``rank`` (kept as a multiple of 8) for one linear."""

    def __init__(self, in_features: int, partitions: Sequence[int], slots: int, rank: int, dtype: torch.dtype,
                 device: torch.device | str) -> None:
        super().__init__()
        if not 1 <= rank <= ops.LORA_MAX_RANK or slots < 1:
            raise ValueError(f"{slots} adapters of rank {rank}: at least one, of rank 1 to {ops.LORA_MAX_RANK}")
        if len(partitions) > ops.LORA_MAX_PARTS:
            raise ValueError(f"{len(partitions)} partitions, at most {ops.LORA_MAX_PARTS}")
        self.in_features, self.partitions, self.slots, self.max_rank = in_features, list(partitions), slots, rank
        self.rank = (rank + 7) // 8 * 8  # rows of B on 16 bytes
        parts, n = len(self.partitions), sum(self.partitions)
        kw = {"dtype": dtype, "device": device}
        self.register_buffer("lora_a", torch.zeros(slots, parts * self.rank, in_features, **kw), persistent=False)
        self.register_buffer("lora_b", torch.zeros(slots, n, self.rank, **kw), persistent=False)
        self.register_buffer("lora_scaling", torch.zeros(slots, dtype=torch.float32, device=device), persistent=False)
        self.register_buffer("lora_ranks", torch.zeros(slots, dtype=torch.int32, device=device), persistent=False)

    @torch.no_grad()  # the values alone: a's and b's graph does not become the bank's
    def load(self, slot: int, a, b, scaling: float = 1.0) -> None:
        """Adapter ``slot``: A ``[r, K]`` and B ``[N, r]``, or lists of one of each a partition (None: that partition
        has none).  One A serves every partition, and one B of all output channels is cut by partition."""
        if not 0 <= slot < self.slots:
            raise ValueError(f"slot {slot} of {self.slots}")
        if torch.is_tensor(b):
            if b.dim() != 2 or b.shape[0] != sum(self.partitions):
                raise ValueError(f"B is {tuple(b.shape)} for {sum(self.partitions)} output channels")
            b = list(b.split(self.partitions, 0))
        if torch.is_tensor(a):
            a = [a] * len(self.partitions)
        if len(a) != len(self.partitions) or len(b) != len(self.partitions):
            raise ValueError(f"{len(a)} A and {len(b)} B for {len(self.partitions)} partitions")
        for ap, bp, width in zip(a, b, self.partitions):
            if (ap is None) != (bp is None):
                raise ValueError("a partition has an A without a B, or a B without an A")
            if ap is not None and (ap.dim() != 2 or bp.dim() != 2 or ap.shape[1] != self.in_features or bp.shape != (width, ap.shape[0])
                                   or ap.shape[0] > self.max_rank):
                raise ValueError(f"A {tuple(ap.shape)} and B {tuple(bp.shape)} do not fit a [{width}, {self.in_features}] "
                                 f"partition with adapters of rank up to {self.max_rank}")
        own = {t.untyped_storage().data_ptr() for t in (self.lora_a, self.lora_b)}  # the bank's own, which clear zeroes
        a, b = ([t.clone() if t is not None and t.untyped_storage().data_ptr() in own else t for t in ts] for ts in (a, b))
        self.clear(slot)
        lo = 0
        for p, (ap, bp, width) in enumerate(zip(a, b, self.partitions)):
            if ap is not None:
                r = ap.shape[0]
                self.lora_a[slot, p * self.rank:p * self.rank + r].copy_(ap)
                self.lora_b[slot, lo:lo + width, :r].copy_(bp)
            lo += width
        self.lora_scaling[slot] = float(scaling)
        self.lora_ranks[slot] = max((ap.shape[0] for ap in a if ap is not None), default=0)

    @torch.no_grad()
    def clear(self, slot: int) -> None:
        """Slot ``slot`` without an adapter: its rows get the shared projection alone."""
        self.lora_a[slot].zero_()
        self.lora_b[slot].zero_()
        self.lora_scaling[slot] = 0.0
        self.lora_ranks[slot] = 0

    def add(self, base: torch.Tensor, x: torch.Tensor, batch: ops.LoraBatch) -> torch.Tensor:
        """``base`` (the shared projection of x) plus each row's adapter of x."""
        return torch.ops.qtts.lora_add(base, x, batch.index, batch.plan, batch.slots, self.lora_a, self.lora_b,
                                       self.lora_scaling, self.lora_ranks, self.partitions)


class AdapterMethod(QuantMethodBase):
    """A linear's own method (or F.linear) and, on top, its rows' adapters."""

    name = "adapters"

    def __init__(self, inner, routing: AdapterRouting) -> None:
        self.inner, self.routing = inner, routing

    def over(self, method) -> AdapterMethod:
        """These adapters on top of ``method`` (a linear that is quantized after its adapters were attached)."""
        return AdapterMethod(method, self.routing)

    def applies_to(self, layer) -> bool:
        return getattr(layer, "adapters", None) is not None

    def batch_for(self, layer, x: torch.Tensor) -> ops.LoraBatch:
        """The step's routing, which must be of x's rows."""
        rows = x.numel() // layer.in_features if layer.in_features else 0
        batch = self.routing.batch
        if batch is None or batch.rows != rows:
            raise ValueError(f"the adapter routing is set for {'no' if batch is None else batch.rows} rows, the call has {rows}")
        return batch

    def apply(self, layer, x: torch.Tensor, bias: torch.Tensor | None) -> torch.Tensor:
        batch = self.batch_for(layer, x)  # before the projection: a routing of other rows runs nothing
        base = self.inner.apply(layer, x, bias) if self.inner is not None else F.linear(x, layer.weight, bias)
        return layer.adapters.add(base, x, batch)


def attach_adapters(module: nn.Module, slots: int, rank: int, routing: AdapterRouting, targets: Sequence[str] = (),
                    dtype: torch.dtype | None = None) -> dict[str, LinearAdapters]:
    """Give every linear under ``module`` whose name holds one of ``targets`` (none: every linear) room for ``slots``
    adapters of rank up to ``rank``; returns them by name.  ``dtype``: the activations' (default: the weight's)."""
    if routing.slots != slots:
        raise ValueError(f"the routing has {routing.slots} slots, the adapters {slots}")
    layers = {name: layer for name, layer in iter_linears(module) if not targets or any(t in name for t in targets)}
    banks = {}
    for name, layer in layers.items():  # all of them before any layer changes: a refusal leaves the module as it was
        if isinstance(layer.quant_method, AdapterMethod):
            raise ValueError(f"{name} has adapters already")
        parts, device = getattr(layer, "partitions", None) or [layer.out_features], layer.weight.device
        bank = banks[name] = LinearAdapters(layer.in_features, parts, slots, rank, dtype or layer.weight.dtype, device)
        if device.type == "cuda":  # a captured call allocates no workspace
            ops.reserve_for_rows(device, ops.OP_LORA, len(parts), bank.rank, max(ops.WORKSPACE_ROWS, routing.max_rows))
    for name, layer in layers.items():
        layer.adapters = banks[name]
        layer.quant_method = AdapterMethod(layer.quant_method, routing)
    return banks
