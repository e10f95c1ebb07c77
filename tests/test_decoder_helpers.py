"""The decoder-layer helpers (qtts_amd.layers.decoder) on layers that are not int8 weight-only:
each returns the reference's composition (qtts/models/talker.py:249-271) unchanged.  CPU only."""

from __future__ import annotations

import torch
import torch.nn.functional as F
from torch import nn

from qtts_amd.layers import GatedMLP, LinearBase
from qtts_amd.layers.decoder import linear_residual, norm_linear, norm_mlp_residual


class Norm(nn.Module):
    """The reference RMSNorm's attributes (qtts/layers/norm.py:82-93) and eager formula."""

    def __init__(self, n: int, eps: float = 1e-6) -> None:
        super().__init__()
        self.weight = nn.Parameter(1 + 0.1 * torch.randn(n), requires_grad=False)
        self.eps = eps

    def forward(self, x):
        v = x.float().pow(2).mean(-1, keepdim=True)
        return (x.float() * torch.rsqrt(v + self.eps) * self.weight.float()).to(x.dtype)


def test_fallbacks_are_the_reference_composition():
    torch.manual_seed(0)
    norm = Norm(64)
    lin = LinearBase(64, 96)
    with torch.no_grad():
        lin.weight.normal_(0, 0.05)
    x = torch.randn(3, 1, 64)
    assert torch.equal(norm_linear(norm, lin, x), lin(norm(x)))
    o = LinearBase(64, 64, bias=True)
    with torch.no_grad():
        o.weight.normal_(0, 0.05)
        o.bias.normal_(0, 0.1)
    r = torch.randn(3, 1, 64)
    assert torch.equal(linear_residual(o, x, r), r + o(x))
    for fuse in (True, False):
        mlp = GatedMLP(64, 128, fuse=fuse)
        with torch.no_grad():
            for p in mlp.parameters():
                p.normal_(0, 0.05)
        h = norm(x)
        if fuse:
            gate, up = mlp.gate_up_proj.split(mlp.gate_up_proj(h))
        else:
            gate, up = mlp.gate_proj(h), mlp.up_proj(h)
        want = x + mlp.down_proj(F.silu(gate) * up)
        assert torch.equal(norm_mlp_residual(norm, mlp, x), want)


class ShiftedNorm(Norm):
    """``1 + weight`` in the weight's place."""

    def forward(self, x):
        v = x.float().pow(2).mean(-1, keepdim=True)
        return (x.float() * torch.rsqrt(v + self.eps) * (1 + self.weight.float())).to(x.dtype)


class BiasNorm(Norm):
    def __init__(self, n: int) -> None:
        super().__init__(n)
        self.bias = nn.Parameter(torch.zeros(n), requires_grad=False)

    def forward(self, x):
        return super().forward(x) + self.bias


class CenteredNorm(Norm):
    def forward(self, x):
        return super().forward(x - x.mean(-1, keepdim=True))


class OuterEpsNorm(Norm):
    def forward(self, x):
        return x / (x.pow(2).mean(-1, keepdim=True).sqrt() + self.eps) * self.weight


class NamedNorm(nn.Module):
    """Another name for eps, the weight multiplied in the rows' own type."""

    def __init__(self, n: int) -> None:
        super().__init__()
        self.weight = nn.Parameter(torch.ones(n))
        self.variance_epsilon = 1e-5

    def forward(self, x):
        h = x.float()
        return self.weight * (h * torch.rsqrt(h.pow(2).mean(-1, keepdim=True) + self.variance_epsilon)).to(torch.bfloat16).to(x.dtype)


class GpuNorm(Norm):
    def forward(self, x):
        if not x.is_cuda:
            raise RuntimeError("runs on a GPU alone")
        return super().forward(x)


def test_which_norms_the_kernels_take():
    """By what a norm computes, not by its attributes: once a module, without the global random state or the weight's values."""
    from qtts_amd.layers.norm import is_rms_norm, mark_rms_norms

    state = torch.random.get_rng_state()
    zero = Norm(64)
    zero.weight.data.zero_()
    for norm in (Norm(64), Norm(7, eps=0.0), zero, NamedNorm(33), nn.RMSNorm(64, eps=1e-6), Norm(64).to(torch.bfloat16), Norm(64).to("meta")):
        kept = None if norm.weight.is_meta else norm.weight.clone()
        assert is_rms_norm(norm) and is_rms_norm(norm), norm
        assert kept is None or torch.equal(norm.weight, kept)
    others = [ShiftedNorm(64), BiasNorm(64), CenteredNorm(64), OuterEpsNorm(64), GpuNorm(64), nn.LayerNorm(64), nn.LayerNorm(64, bias=False),
              nn.GroupNorm(4, 64), nn.BatchNorm1d(64), nn.RMSNorm(64), nn.RMSNorm((8, 8), eps=1e-6), nn.RMSNorm(64, eps=1e-6, elementwise_affine=False)]
    for norm in others:
        assert not is_rms_norm(norm), norm
    torch.random.set_rng_state(state)
    model = nn.ModuleList([Norm(64), ShiftedNorm(64), nn.Linear(64, 64), NamedNorm(16)])
    before = torch.random.get_rng_state()
    assert mark_rms_norms(model) == 2 and torch.equal(before, torch.random.get_rng_state())


def test_a_marked_norm_is_known_while_tracing():
    """Dynamo traces the question without a break: the answer of a marked norm, the composition for one that was never asked."""
    import torch._dynamo

    from qtts_amd.layers.norm import is_rms_norm

    class Step(nn.Module):
        def __init__(self) -> None:
            super().__init__()
            self.norm = Norm(64)

        def forward(self, x):
            return x + 1 if is_rms_norm(self.norm) else x - 1

    for marked in (False, True):
        torch._dynamo.reset()
        step, x = Step(), torch.zeros(2, 64)
        if marked:
            assert is_rms_norm(step.norm)
        assert torch.equal(torch.compile(step, fullgraph=True, backend="eager")(x), x + 1 if marked else x - 1)
