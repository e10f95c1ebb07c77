"""A model's paged key-value cache and the attention that reads it (qtts/models/talker.py:47-136).

The reference's talker keeps a fixed slice of one tensor a request (talker.py:47-91) and runs torch's attention over it.
Here every request has pages of a pool that all requests and all layers' numbering share: a page table per request, the
lengths and the free list live on the GPU, and one kernel a step (:meth:`PagedCache.step`) turns the requests' new tokens
into positions and cache slots for every layer.  Per layer, :func:`attend` is two kernels: head norms, rotation and the
cache's writes, then attention.

Per step, a serving loop says how many tokens join each request, then runs the model::

    cache = PagedCache(layers=28, requests=64, pages=4096, heads=16, kv_heads=8, head_dim=128, rope_theta=1e6)
    cache.step([37, 12])                     # two prompts, 49 rows
    ...
    cache.step([1, 1, 0, 1], rows=8, max_new=1)   # decode: requests 0, 1 and 3, padded to the captured batch of 8
    graph.replay()                           # captured after such a step; reads the cache's buffers
    cache.release([1])                       # its pages are free again

A request is a row of the table; its number is the caller's.  Rows of the batch lie in the order of the requests.
"""

from __future__ import annotations

from typing import Sequence

import torch
from torch import nn

from .. import ops, torch_ops  # noqa: F401  (torch_ops registers torch.ops.qtts)
from .norm import is_rms_norm, norm_eps


def rope_tables(length: int, head_dim: int, theta: float = 1e6, device: torch.device | str = "cuda"):
    """fp32 ``(cos, sin)`` ``[length, head_dim / 2]`` of position times ``theta ** (-2 i / head_dim)`` (qtts/layers/rope.py:23-72):
    angles in 64 bits, since 32 lose the far positions'."""
    at = torch.arange(length, dtype=torch.float64, device=device)
    turn = float(theta) ** (-torch.arange(0, head_dim, 2, dtype=torch.float64, device=device) / head_dim)
    angle = at[:, None] * turn
    return angle.cos().float(), angle.sin().float()


class PagedCache:
    """Keys and values of up to ``requests`` requests in ``pages`` pages of ``page_size`` tokens, for ``layers`` layers, in
    buffers that keep their addresses: a graph captured after one :meth:`step` reads, on every replay, what the last one
    wrote (positions -1, and no attention, for rows that it does not have).  The graph has that step's ``rows`` and, where it was
    given, its ``max_new``: requests with more new tokens, or rows past those, get zeros.

    ``max_length``: tokens a request can have (None: as many as the pool holds); ``max_rows``: rows of a step.  ``rope_theta``:
    the base of the rotation's angles (None: no rotation; ``rope`` takes tables of the caller's own)."""

    def __init__(self, layers: int, requests: int, pages: int, heads: int, kv_heads: int, head_dim: int, page_size: int = 64,
                 max_length: int | None = None, max_rows: int = ops.WORKSPACE_ROWS, dtype: torch.dtype = torch.bfloat16,
                 device: torch.device | str = "cuda", rope_theta: float | None = None) -> None:
        if min(layers, requests, pages, kv_heads, head_dim, page_size, max_rows) < 1 or heads < kv_heads or heads % kv_heads:
            raise ValueError(f"a cache of {layers} layers, {requests} requests, {pages} pages of {page_size} tokens, {heads} and "
                             f"{kv_heads} heads of {head_dim}, {max_rows} rows a step")
        if requests > ops.PAGED_MAX_REQUESTS:
            raise ValueError(f"{requests} requests, at most {ops.PAGED_MAX_REQUESTS}")
        if dtype not in (torch.bfloat16, torch.float16):
            raise ValueError(f"a cache holds bfloat16 or float16, not {dtype}")
        self.heads, self.kv_heads, self.head_dim, self.page_size = heads, kv_heads, head_dim, page_size
        self.requests, self.pages, self.max_rows = requests, pages, int(max_rows)
        cols = pages if max_length is None else min(pages, -(-int(max_length) // page_size))
        if cols < 1:
            raise ValueError(f"requests of up to {max_length} tokens")
        kw = {"dtype": dtype, "device": device}
        self.k = [torch.empty(pages, kv_heads, page_size, head_dim, **kw) for _ in range(layers)]
        self.v = [torch.empty(pages, kv_heads, head_dim, page_size, **kw) for _ in range(layers)]
        kw = {"dtype": torch.int32, "device": device}
        self.lengths, self.table = torch.zeros(requests, **kw), torch.zeros(requests, cols, **kw)
        self.free, self.taken = torch.arange(pages, **kw), torch.zeros(1, **kw)
        self._new, self._which, self._numbers = torch.zeros(requests, **kw), torch.zeros(requests, **kw), torch.arange(requests, **kw)
        self._starts, self._counts = torch.zeros(requests + 1, **kw), torch.zeros(requests, **kw)
        self._positions, self._slots = torch.full((self.max_rows,), -1, **kw), torch.full((self.max_rows,), -1, **kw)
        self.rope = None if rope_theta is None else rope_tables(cols * page_size, head_dim, rope_theta, device)
        self.batch: ops.PagedBatch | None = None
        if self.table.is_cuda:  # a captured call allocates no workspace
            ops.reserve_workspace(self.table.device, ops.attention_bytes(self.max_rows * (heads // kv_heads), head_dim))

    def _whole(self, values, name: str) -> torch.Tensor:
        values = torch.as_tensor(values)
        if values.dim() != 1:
            raise ValueError(f"{name} must be 1-D, got shape {tuple(values.shape)}")
        if values.numel() and (values.dtype == torch.bool or values.is_floating_point() or values.is_complex()):
            raise ValueError(f"{name} must hold whole numbers, got {values.dtype}")
        return values

    def step(self, new: torch.Tensor | Sequence[int], rows: int | None = None, max_new: int | None = None,
             min_new: int = 0) -> ops.PagedBatch:
        """``new[r]`` tokens join request r (requests past the end of ``new``: none), in a batch of ``rows`` rows with padding
        rows behind.  Numbers on the host are checked here.  A tensor on the GPU is not read: ``rows`` is then required,
        ``max_new`` bounds its entries (None: ``rows``), and what does not fit is denied (``batch.counts`` 0).  Requests whose pages are not left
        are denied in either case.

        ``min_new``: tokens that a request has at least, if any; past 16 rows a key-value head the kernel of few rows is left out.
        A captured call keeps ``max_new`` (1: the decode step's kernel alone); without it, it is made for up to ``rows`` tokens a request,
        whatever this step's are."""
        new, this_step = self._whole(new, "new"), False
        if new.shape[0] > self.requests:
            raise ValueError(f"new must have up to {self.requests} entries, got {new.shape[0]}")
        if new.device.type == "cpu":
            given = new.tolist()
            if any(n < 0 for n in given):
                raise ValueError(f"new must not be negative: {given}")
            total, most, this_step = sum(given), max(given, default=0), max_new is None
            rows = total if rows is None else int(rows)
            if total > rows:
                raise ValueError(f"{total} new tokens do not fit a batch of {rows} rows")
            if max_new is None:
                max_new = most
            elif most > max_new:
                raise ValueError(f"{most} new tokens of a request, bounded by max_new = {max_new}")
            if min_new > min((n for n in given if n), default=min_new):
                raise ValueError(f"a request has fewer than min_new = {min_new} new tokens")
        elif rows is None:
            raise ValueError("rows must be given for counts on the GPU")
        if not 0 <= int(rows) <= self.max_rows:
            raise ValueError(f"a batch of {rows} rows in a cache for {self.max_rows}")
        rows = int(rows)
        self.batch = None  # nothing stands if what follows fails
        given = new.shape[0]
        if new.dtype != torch.int32:  # what int32 cannot hold fits no batch either
            new = new.to(torch.int64).clamp(-1, 2 ** 31 - 1).to(torch.int32)
        self._new[:given].copy_(new)
        if given < self.requests:
            self._new[given:].zero_()
        batch = ops.PagedBatch(self.table, self._starts, self._counts, self.lengths, self._positions[:rows], self._slots[:rows],
                               self.page_size, max_new, min_new, self.taken, this_step)
        ops.paged_step(self._new, self.lengths, self.table, self.free, self.taken, self.page_size, rows, out=batch, room=self.max_rows)
        self.batch = batch
        return batch

    def release(self, requests: torch.Tensor | Sequence[int]) -> None:
        """The requests (their numbers; on the GPU, others than the cache's are left aside) hold nothing from here on; their
        pages are free again."""
        requests = self._whole(requests, "requests")
        if requests.device.type == "cpu" and any(not 0 <= r < self.requests for r in requests.tolist()):
            raise ValueError(f"requests {requests.tolist()} of {self.requests}")
        if not requests.numel():
            return
        requests = requests.to(device=self._which.device, dtype=torch.int64)
        self._which.copy_((self._numbers[:, None] == requests).any(1))  # (an index out of range would end the process)
        ops.paged_release(self._which, self.lengths, self.table, self.free, self.taken, self.page_size)

    def batch_for(self, rows: int) -> ops.PagedBatch:
        """The step's batch, which must be of this many rows."""
        if self.batch is None or self.batch.rows != rows:
            raise ValueError(f"the cache is set for {'no' if self.batch is None else self.batch.rows} rows, the call has {rows}")
        return self.batch


def attend(attn: nn.Module, qkv: torch.Tensor, cache: PagedCache, layer: int, window: int = 0, sinks: int = 0,
           scale: float | None = None, weights16: bool = False) -> torch.Tensor:
    """The attention between qkv_proj and o_proj (talker.py:249-270) for the rows of the cache's step: head norms
    (``attn.q_norm``, ``attn.k_norm``, None or missing: none), rotation, this layer's cache, attention.  qkv
    ``[..., (Hq + 2 H) D]`` is qkv_proj's output; returns ``[..., Hq D]``, o_proj's input.  Norms that are no RMSNorm of one weight
    in qkv's type run as the modules they are.  weights16: :func:`~qtts_amd.ops.paged_attention`'s, for prompts whose time counts more than their
    last bits."""
    d, kv = cache.head_dim, cache.kv_heads
    shape, width = qkv.shape, (cache.heads + 2 * kv) * d
    rows = qkv.numel() // width
    if shape[-1] != width:
        raise ValueError(f"qkv is {tuple(shape)} for {cache.heads} + 2 x {kv} heads of {d}")
    batch = cache.batch_for(rows)
    norms = [getattr(attn, name, None) for name in ("q_norm", "k_norm")]
    eps = {norm_eps(n) for n in norms if n is not None}
    if all(n is None or (is_rms_norm(n) and n.weight.shape == (d,) and n.weight.dtype == qkv.dtype) for n in norms) and len(eps) <= 1:
        weights = [None if n is None else n.weight for n in norms]
        eps = next(iter(eps), 1e-6)
    else:
        x = qkv.reshape(rows, cache.heads + 2 * kv, d)
        q, k, v = x.split([cache.heads, kv, kv], 1)
        q, k = (t if n is None else n(t).to(qkv.dtype) for n, t in zip(norms, (q, k)))
        qkv, weights, eps = torch.cat([q, k, v], 1), [None, None], 1e-6
    cos, sin = cache.rope if cache.rope is not None else (None, None)
    state = [batch.table, batch.starts, batch.counts, batch.lengths, batch.positions, batch.slots]
    bounds = [batch.page_size, batch.max_new, batch.min_new, int(batch.this_step)]
    q = torch.ops.qtts.qkv_to_cache(qkv.reshape(rows, width), cache.k[layer], cache.v[layer], state, bounds, cache.heads, weights[0],
                                    weights[1], eps, cos, sin)
    out = torch.ops.qtts.paged_attention(q, cache.k[layer], cache.v[layer], state, bounds, window, sinks,
                                         d ** -0.5 if scale is None else scale, weights16)
    return out.view(*shape[:-1], cache.heads * d)
