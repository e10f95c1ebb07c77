"""W8A8 decoder layers with their inputs' codes from the norm and the activation, and low-rank adapters of many requests
on top, as a serving step runs them: eager, captured, and several captured row counts on the shared workspace.

Each stage of a layer is held against 64 bits on the stage's own inputs.  Bound of a linear's output, from the arithmetic
(u = 2^-24): base is rounded once (half a step of its type; fp8 with a bias twice, since the fp8 GEMM's contract is
cast(cast(product) + bias): the product's own half step comes first), its K products are summed in fp32 (int8: exactly, then two
scale products), the adapter's part is off as derived for lora_add (fp32 sums of K and R products, the first product carried
in 2^-16), and the sum is rounded once more."""

from __future__ import annotations

import pytest
import torch
from torch import nn

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HIDDEN, INTER, SLOTS, RANK = 512, 1152, 6, 12


@pytest.fixture(scope="module")
def ops():
    from qtts_amd import ops as _ops
    assert _ops.device_supported(), "GPU is not a gfx950"
    return _ops


class Norm(nn.Module):
    """The reference RMSNorm's attributes (qtts/layers/norm.py:82-93) and eager formula."""

    def __init__(self, n: int, dtype: torch.dtype, eps: float = 1e-6) -> None:
        super().__init__()
        g = torch.Generator(device="cuda").manual_seed(n)
        self.weight = nn.Parameter((1 + 0.1 * torch.randn(n, device="cuda", generator=g)).to(dtype), requires_grad=False)
        self.eps = eps

    def forward(self, x):
        v = x.float().pow(2).mean(-1, keepdim=True)
        return (x.float() * torch.rsqrt(v + self.eps) * self.weight.float()).to(x.dtype)


class Block(nn.Module):
    def __init__(self, dtype: torch.dtype, seed: int) -> None:
        super().__init__()
        from qtts_amd.layers import GatedMLP, LinearBase, MergedLinear
        self.norm1, self.norm2 = Norm(HIDDEN, dtype), Norm(HIDDEN, dtype)
        self.qkv = MergedLinear(HIDDEN, [HIDDEN, HIDDEN // 2, HIDDEN // 2], bias=True, dtype=dtype, device="cuda")
        self.o = LinearBase(HIDDEN, HIDDEN, dtype=dtype, device="cuda")
        self.mlp = GatedMLP(HIDDEN, INTER, fuse=True, dtype=dtype, device="cuda")
        g = torch.Generator(device="cuda").manual_seed(seed)
        for name, p in self.named_parameters():
            if "norm" not in name:
                p.data.copy_((torch.randn(p.shape, device="cuda", generator=g) * 0.03).to(dtype))

    def forward(self, delta, hidden):
        from qtts_amd.layers.decoder import add_norm_linear, add_norm_mlp
        y, hidden = add_norm_linear(self.norm1, self.qkv, delta, hidden)
        q, _, _ = self.qkv.split(y)
        return add_norm_mlp(self.norm2, self.mlp, self.o(q), hidden)


def _block(method, dtype, seed=5, adapters=True, max_rows=256):
    from qtts_amd import AdapterRouting, QuantConfig, apply_quantization, attach_adapters
    from qtts_amd.quant.base import quantize_module, build_method
    block = Block(dtype, seed)
    if method != "none":
        config = QuantConfig(method=method, calibrate=False)
        assert quantize_module(block, build_method(config), config, "talker")["converted"] == 4
    routing = AdapterRouting(SLOTS, max_rows)
    if adapters:
        banks = attach_adapters(block, SLOTS, RANK, routing)
        assert len(banks) == 4
        g = torch.Generator().manual_seed(seed)
        for bank in banks.values():
            for slot in range(SLOTS - 1):  # the last slot holds none
                r = int(torch.randint(1, RANK + 1, (1,), generator=g))
                a = [torch.randn(r, bank.in_features, generator=g) * bank.in_features ** -0.5 for _ in bank.partitions]
                b = [torch.randn(w, r, generator=g) * 0.2 for w in bank.partitions]
                bank.load(slot, a, b, scaling=float(torch.rand(1, generator=g)) + 0.5)
    return block, routing


def _rows(m, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(m, HIDDEN, device="cuda", generator=g).to(dtype)


def _index(m, seed):
    return torch.randint(-1, SLOTS, (m,), generator=torch.Generator().manual_seed(seed), dtype=torch.int32)


def _weight(layer):
    from qtts_amd.quant.fp8 import fp8_weight_rowmajor
    from qtts_amd.quant.int8 import int8_weight_rowmajor
    if getattr(layer, "fp8_weight", None) is not None:
        return fp8_weight_rowmajor(layer).float().double().cpu(), layer.fp8_scale.reshape(-1).double().cpu()
    return int8_weight_rowmajor(layer).double().cpu(), layer.int8_scale.double().cpu()


def _hold(layer, y, qx, sx, x, index, adapters):
    """y against the linear on codes (qx, sx) plus the adapters on the 16-bit rows x, in 64 bits."""
    w, sw = _weight(layer)
    eps = torch.finfo(y.dtype).eps
    q, s = qx.float().double().cpu(), sx.double().cpu()[:, None]
    base = (q @ w.t()) * s * sw
    sums = (q.abs() @ w.abs().t()) * s * sw
    k = q.shape[1]
    bound = 2 * (k + 8) * U * sums + 4 * U * base.abs()
    if layer.bias is not None:
        if getattr(layer, "fp8_weight", None) is not None:
            bound = bound + eps / 2 * (base.abs() + bound)
        base = base + layer.bias.double().cpu()
        bound = bound + U * base.abs()
    bound = bound + eps / 2 * (base.abs() + bound)  # base stored in 16 bits
    want = base.clone()
    if adapters:
        bank, xd = layer.adapters, x.double().cpu()
        a, b, r = bank.lora_a.double().cpu(), bank.lora_b.double().cpu(), bank.rank
        lo = 0
        for p, width in enumerate(bank.partitions):
            for slot in range(SLOTS):
                rows = (index == slot).nonzero().flatten()
                scale = float(bank.lora_scaling[slot])
                ap, bp = a[slot, p * r:(p + 1) * r], b[slot, lo:lo + width]
                t = xd[rows] @ ap.t()
                want[rows, lo:lo + width] += scale * (t @ bp.t())
                bound[rows, lo:lo + width] += (2 * (k + r + 8) * U * scale * (xd[rows].abs() @ ap.abs().t() @ bp.abs().t())
                                               + 2.0 ** -16 * scale * (t.abs() @ bp.abs().t()))
            lo += width
        bound = bound + eps / 2 * (want.abs() + bound)
    tiny = torch.finfo(y.dtype).smallest_normal * eps
    err = (y.double().cpu() - want).abs()
    assert (err <= bound + tiny).all(), float((err / (bound + tiny)).max())


@pytest.mark.parametrize("adapters", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("method", ["fp8", "int8"])
@pytest.mark.parametrize("m", [0, 1, 7, 64, 131])
def test_layer_stages(ops, method, dtype, adapters, m):
    from qtts_amd.layers.decoder import add_norm_linear, add_norm_mlp
    block, routing = _block(method, dtype, adapters=adapters)
    index = _index(m, m)
    routing.set(index)
    codes = ops.CODE_E4M3 if method == "fp8" else ops.CODE_INT8
    x, res = _rows(m, dtype, m + 1), _rows(m, dtype, m + 2)
    y, hidden = add_norm_linear(block.norm1, block.qkv, x, res)
    qx, sx, want_hidden, normed = ops.rms_norm_quant(x, block.norm1.weight, 1e-6, res, codes, True)
    assert torch.equal(hidden, want_hidden) and torch.equal(hidden, (x.double() + res.double()).to(dtype))
    _hold(block.qkv, y, qx, sx, normed, index, adapters)
    out, again = add_norm_mlp(block.norm2, block.mlp, x, res)
    assert torch.equal(again, hidden)
    gate_up, _ = add_norm_linear(block.norm2, block.mlp.gate_up_proj, x, res)
    qx, sx, _, normed = ops.rms_norm_quant(x, block.norm2.weight, 1e-6, res, codes, True)
    _hold(block.mlp.gate_up_proj, gate_up, qx, sx, normed, index, adapters)
    qx, sx, act = ops.silu_mul_quant(gate_up, codes, True)
    _hold(block.mlp.down_proj, out, qx, sx, act, index, adapters)
    y3, h3 = add_norm_linear(block.norm1, block.qkv, x.view(m, 1, HIDDEN), res.view(m, 1, HIDDEN))  # a batch of one token
    assert y3.shape == (m, 1, 2 * HIDDEN) and torch.equal(y3.view_as(y), y) and torch.equal(h3.view_as(hidden), hidden)
    y1, h1 = add_norm_linear(block.norm1, block.qkv, hidden)  # nothing to add: the same row through the norm
    assert h1 is hidden and torch.equal(
        y1, add_norm_linear(block.norm1, block.qkv, hidden, torch.zeros_like(hidden))[0])


@pytest.mark.parametrize("method", ["fp8", "int8", "int8_weight_only", "fp8_weight_only", "none"])
def test_adapters_on_every_method(ops, method):
    """Rows without an adapter keep the bits of the linear's own method; the others add theirs to them."""
    block, routing = _block(method, torch.bfloat16)
    plain, _ = _block(method, torch.bfloat16, adapters=False)
    for m in (5, 70):
        x, index = _rows(m, torch.bfloat16, m), _index(m, m + 3)
        routing.set([-1] * m)
        base = block.qkv(x)
        assert torch.equal(base, plain.qkv(x))
        routing.set(index)
        y = block.qkv(x)
        free = ((index < 0) | (index == SLOTS - 1)).nonzero().flatten().cuda()
        assert torch.equal(y[free], base[free])
        batch = ops.lora_batch(index.cuda(), SLOTS)
        bank = block.qkv.adapters
        assert torch.equal(y, ops.lora_add(base, x, batch, bank.lora_a, bank.lora_b, bank.lora_scaling, bank.lora_ranks,
                                           bank.partitions))
        assert not torch.equal(y, base)


@pytest.mark.parametrize("method", ["fp8", "int8"])
def test_captured_steps_follow_the_routing(ops, method):
    """Two layers with adapters in captured graphs of three padded row counts: all on one workspace and one routing, replayed
    in turn with eager work between, each replay bit for bit the eager step of its rows and adapters."""
    from qtts_amd.graphs import PaddedGraphs
    layers, routings = zip(*[_block(method, torch.bfloat16, seed=20 + i) for i in range(2)])
    routing = routings[0]
    for block in layers[1:]:
        for linear in (block.qkv, block.o, block.mlp.gate_up_proj, block.mlp.down_proj):
            linear.quant_method.routing = routing

    def step(x):
        delta, hidden = x, None
        for block in layers:
            delta, hidden = block(delta, hidden)
        return hidden + delta

    graphs = PaddedGraphs(step, (HIDDEN,), torch.bfloat16, batch_sizes=(4, 48, 160))
    for turn in range(3):
        for rows in (3, 131, 40, 4, 160):
            x, index = _rows(rows, torch.bfloat16, 7 * rows + turn), _index(rows, rows + turn)
            padded = graphs.padded_rows(rows)
            routing.set(index, rows=padded)
            got = graphs.run(x).clone()
            routing.set(index, rows=padded)
            whole = torch.zeros(padded, HIDDEN, dtype=torch.bfloat16, device="cuda")
            whole[:rows] = x
            assert torch.equal(got, step(whole)[:rows]), (turn, rows)
    assert graphs.replays == 15


def test_other_stream_and_slot_changes(ops):
    """A slot loaded anew is what the next replay of a captured call adds, on a stream of its own."""
    block, routing = _block("fp8", torch.bfloat16)
    m = 9
    x, index = _rows(m, torch.bfloat16, 1), _index(m, 2)
    index[0], index[1] = 2, SLOTS - 1
    routing.set(index)
    block.qkv(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = block.qkv(x)
    bank = block.qkv.adapters
    side = torch.cuda.Stream()
    for turn in range(3):
        g = torch.Generator().manual_seed(turn)
        bank.clear(2)
        bank.load(SLOTS - 1, torch.randn(3, HIDDEN, generator=g), torch.randn(2 * HIDDEN, 3, generator=g) * 0.1)
        want = block.qkv(x)
        out.zero_()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graph.replay()
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(out, want)


def test_what_the_helpers_leave_to_the_linear(ops):
    """A norm that is no RMSNorm in x's type, another residual type and weight-only linears keep the composition's bits."""
    from qtts_amd.layers.decoder import add_norm_linear, add_norm_mlp
    block, _ = _block("fp8", torch.bfloat16, adapters=False)
    x, res = _rows(5, torch.bfloat16, 1), _rows(5, torch.bfloat16, 2)
    layer_norm = nn.LayerNorm(HIDDEN, device="cuda", dtype=torch.bfloat16)
    fp32_norm = Norm(HIDDEN, torch.float32)
    for norm, r in ((layer_norm, res), (fp32_norm, res), (block.norm1, res.float()[:1].to(torch.bfloat16))):
        h = r + x
        y, hidden = add_norm_linear(norm, block.qkv, x, r)
        assert torch.equal(hidden, h) and torch.equal(y, block.qkv(norm(h)))
        y, hidden = add_norm_mlp(norm, block.mlp, x, r)
        assert torch.equal(hidden, h) and torch.equal(y, block.mlp(norm(h)))
    weight_only, _ = _block("int8_weight_only", torch.bfloat16, adapters=False)
    y, hidden = add_norm_linear(weight_only.norm1, weight_only.qkv, x, res)
    assert torch.equal(y, weight_only.qkv(weight_only.norm1(res + x))) and torch.equal(hidden, res + x)


@pytest.mark.parametrize("method", ["fp8", "int8_weight_only"])
def test_quantizing_before_or_after_attaching(ops, method):
    """The order of attach_adapters and quantization is the caller's: the same bits either way."""
    from qtts_amd import QuantConfig
    from qtts_amd.quant.base import build_method, quantize_module
    before, first = _block(method, torch.bfloat16)
    after, second = _block("none", torch.bfloat16)
    config = QuantConfig(method=method, calibrate=False)
    assert quantize_module(after, build_method(config), config, "talker")["converted"] == 4
    x, index = _rows(9, torch.bfloat16, 3), _index(9, 4)
    first.set(index), second.set(index)
    want = before.qkv(x)
    first.set([-1] * 9)
    assert not torch.equal(want, before.qkv(x)) and torch.equal(after.qkv(x), want)


@pytest.mark.parametrize("captured", [100, 48])
def test_a_replay_after_a_routing_of_other_rows(ops, captured):
    """A captured step's rows take the last routing's slots, and none where it has no row, whatever its row count."""
    block, routing = _block("fp8", torch.bfloat16)
    x = _rows(captured, torch.bfloat16, 1)
    routing.set(_index(captured, 2))
    block.qkv(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = block.qkv(x)
    bank = block.qkv.adapters
    routing.set([-1] * captured)
    base = block.qkv(x)
    for turn, rows in enumerate((20, captured, 131, 66, 5, captured - 1, 200)):
        index = _index(rows, 30 + turn)
        routing.set([SLOTS - 2] * 256), routing.set(index if turn % 2 else index.cuda())
        graph.replay()
        mine = torch.full((captured,), -1, dtype=torch.int32)
        mine[:min(rows, captured)] = index[:captured]
        want = ops.lora_add(base, x, ops.lora_batch(mine.cuda(), SLOTS), bank.lora_a, bank.lora_b, bank.lora_scaling, bank.lora_ranks,
                            bank.partitions)
        # a call without this batch's plan sums in another order: at most a step of the output apart, and fp32's K + R roundings
        step = torch.finfo(out.dtype).eps * want.abs() + 2 * (HIDDEN + 16) * U * (want - base).abs().amax()
        assert ((out.float() - want.float()).abs() <= step.float()).all(), rows
        none = (mine < 0).nonzero().flatten().cuda()
        assert torch.equal(out[none], base[none]), rows


@pytest.mark.parametrize("kind", ["ShiftedNorm", "BiasNorm", "CenteredNorm", "OuterEpsNorm"])
def test_norms_that_only_look_like_rms_norm(ops, kind):
    """A norm of another formula with RMSNorm's attributes keeps the composition's bits in every helper."""
    import test_decoder_helpers as helpers
    from qtts_amd.layers.decoder import add_norm_linear, add_norm_mlp, norm_linear, norm_mlp_residual
    norm = getattr(helpers, kind)(HIDDEN).cuda().to(torch.bfloat16)
    if kind == "BiasNorm":
        norm.bias.data.fill_(0.5)
    x, res = _rows(5, torch.bfloat16, 1) + 0.25, _rows(5, torch.bfloat16, 2)
    block, _ = _block("fp8", torch.bfloat16, adapters=False)
    y, hidden = add_norm_linear(norm, block.qkv, x, res)
    assert torch.equal(hidden, res + x) and torch.equal(y, block.qkv(norm(res + x)))
    y, hidden = add_norm_mlp(norm, block.mlp, x, res)
    assert torch.equal(y, block.mlp(norm(res + x)))
    block, _ = _block("int8_weight_only", torch.bfloat16, adapters=False)
    assert torch.equal(norm_linear(norm, block.qkv, x), block.qkv(norm(x)))
    gate, up = block.mlp.gate_up_proj.split(block.mlp.gate_up_proj(norm(x)))
    assert torch.equal(norm_mlp_residual(norm, block.mlp, x), x + block.mlp.down_proj(torch.nn.functional.silu(gate) * up))


def test_a_norm_of_a_gpu_kernel_alone(ops):
    """It is asked on its own device, in its own type; a captured step that meets it first runs the norm itself."""
    import test_decoder_helpers as helpers
    from qtts_amd.layers.norm import is_rms_norm

    class KernelNorm(Norm):
        def forward(self, x):
            return ops.rms_norm(x, self.weight, self.eps)

    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        assert is_rms_norm(KernelNorm(HIDDEN, dtype)) and is_rms_norm(helpers.GpuNorm(HIDDEN).cuda().to(dtype))

    class ShiftedKernelNorm(Norm):
        def forward(self, x):
            return ops.rms_norm(x, 1 + self.weight, self.eps)

    assert not is_rms_norm(ShiftedKernelNorm(HIDDEN, torch.bfloat16))
    norm, x = KernelNorm(HIDDEN, torch.bfloat16), _rows(3, torch.bfloat16, 1)
    want = norm(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        assert not is_rms_norm(norm)
        out = norm(x)
    graph.replay()
    assert torch.equal(out, want) and is_rms_norm(norm)
