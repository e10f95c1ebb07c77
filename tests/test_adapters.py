"""Low-rank adapters on the linears' hook (qtts_amd.layers.adapters), the decoder helpers for W8A8 layers, their custom
ops' fakes and the dispatch rules of the kernels behind them, all without a GPU."""

from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F
from torch import nn
from torch._subclasses.fake_tensor import FakeTensorMode

from qtts_amd import AdapterRouting, attach_adapters, ops, torch_ops
from qtts_amd.layers import GatedMLP, LinearBase, MergedLinear
from qtts_amd.layers.adapters import AdapterMethod, LinearAdapters
from qtts_amd.layers.decoder import add_norm_linear, add_norm_mlp
from test_decoder_helpers import Norm
from test_dispatch_rules import _run


def _fill(m: nn.Module) -> nn.Module:
    with torch.no_grad():
        for p in m.parameters():
            p.normal_(0, 0.05)
    return m


@pytest.mark.parametrize("with_residual", [False, True])
def test_add_norm_fallbacks_are_the_composition(with_residual):
    torch.manual_seed(1)
    norm, lin = Norm(64), _fill(LinearBase(64, 96, bias=True))
    x = torch.randn(3, 2, 64)
    r = torch.randn(3, 2, 64) if with_residual else None
    h = x if r is None else r + x
    y, hidden = add_norm_linear(norm, lin, x, r)
    assert torch.equal(hidden, h) and torch.equal(y, lin(norm(h)))
    for fuse in (True, False):
        mlp = _fill(GatedMLP(64, 128, fuse=fuse))
        y, hidden = add_norm_mlp(norm, mlp, x, r)
        assert torch.equal(hidden, h) and torch.equal(y, mlp(norm(h)))


class Block(nn.Module):
    def __init__(self) -> None:
        super().__init__()
        self.qkv_proj = MergedLinear(64, [32, 16, 16])
        self.o_proj = LinearBase(32, 64)
        self.mlp = GatedMLP(64, 128)


def test_attach_finds_the_named_linears_and_their_partitions():
    block = _fill(Block())
    routing = AdapterRouting(4, 32, device="cpu")
    banks = attach_adapters(block, slots=4, rank=12, routing=routing, targets=("qkv", "down"))
    assert sorted(banks) == ["mlp.down_proj", "qkv_proj"]
    q = banks["qkv_proj"]
    assert q.lora_a.shape == (4, 3 * 16, 64) and q.lora_b.shape == (4, 64, 16) and q.rank == 16
    assert banks["mlp.down_proj"].lora_a.shape == (4, 16, 128)
    assert isinstance(block.qkv_proj.quant_method, AdapterMethod) and block.o_proj.quant_method is None
    assert block.qkv_proj.quant_method.applies_to(block.qkv_proj)
    assert not list(q.state_dict())  # adapters are loaded by slot, not from the checkpoint
    with pytest.raises(ValueError, match="has adapters already"):
        attach_adapters(block, slots=4, rank=12, routing=routing)
    with pytest.raises(ValueError, match="mlp.down_proj has adapters already"):  # after layers without any
        attach_adapters(block, slots=4, rank=12, routing=routing, targets=("o_proj", "mlp"))
    assert block.o_proj.quant_method is None and not hasattr(block.mlp.gate_up_proj, "adapters")
    with pytest.raises(ValueError, match="routing has 4 slots"):
        attach_adapters(_fill(Block()), slots=5, rank=12, routing=routing)
    for bad in ({"slots": 0}, {"rank": 0}, {"rank": 129}):
        kw = {"slots": 4, "rank": 8, **bad}
        with pytest.raises(ValueError):
            attach_adapters(_fill(Block()), routing=AdapterRouting(4, 8, device="cpu"), **kw)


def test_load_lays_adapters_out_by_partition():
    bank = LinearAdapters(8, [6, 4], 3, 5, torch.float32, "cpu")
    assert bank.rank == 8
    a0, a1, b0, b1 = torch.randn(5, 8), torch.randn(2, 8), torch.randn(6, 5), torch.randn(4, 2)
    bank.load(1, [a0, a1], [b0, b1], scaling=0.5)
    assert torch.equal(bank.lora_a[1, :5], a0) and torch.equal(bank.lora_a[1, 8:10], a1)
    assert torch.equal(bank.lora_b[1, :6, :5], b0) and torch.equal(bank.lora_b[1, 6:, :2], b1)
    assert not bank.lora_a[1, 5:8].any() and not bank.lora_a[1, 10:].any() and not bank.lora_b[1, 6:, 2:].any()
    assert bank.lora_ranks.tolist() == [0, 5, 0] and bank.lora_scaling.tolist() == [0.0, 0.5, 0.0]
    bank.load(1, a1, torch.cat([b0[:, :2], b1]))  # one A and one B for the whole linear
    assert torch.equal(bank.lora_a[1, :2], a1) and torch.equal(bank.lora_a[1, 8:10], a1) and not bank.lora_a[1, 2:8].any()
    assert bank.lora_ranks[1] == 2 and bank.lora_scaling[1] == 1
    bank.load(2, [None, a1], [None, b1])
    assert not bank.lora_a[2, :8].any() and bank.lora_ranks[2] == 2
    bank.clear(1)
    assert not bank.lora_a[1].any() and not bank.lora_b[1].any() and bank.lora_ranks.tolist() == [0, 0, 2]


def test_load_takes_a_training_modules_parameters():
    """The bank holds values: loading tensors that require grad leaves no graph behind, however often a slot is reloaded."""
    import copy

    bank = LinearAdapters(8, [6, 4], 3, 5, torch.float32, "cpu")
    a, b = nn.Parameter(torch.randn(5, 8)), nn.Parameter(torch.randn(10, 5))
    for _ in range(3):
        bank.load(1, a, b)
        assert not any(t.requires_grad or t.grad_fn is not None for t in bank.buffers())
    assert torch.equal(bank.lora_a[1, :5], a.detach()) and torch.equal(bank.lora_b[1, 6:, :5], b.detach()[6:])
    assert torch.equal(copy.deepcopy(bank).lora_a, bank.lora_a)
    bank.clear(1)
    assert not any(t.requires_grad for t in bank.buffers()) and a.grad is None


def test_load_from_the_bank_itself():
    """Adapters taken from the bank's own tensors, the slot's own among them (another scaling, a swap of partitions)."""
    bank = LinearAdapters(8, [6, 6], 3, 5, torch.float32, "cpu")
    a0, a1, b0, b1 = torch.randn(5, 8), torch.randn(5, 8), torch.randn(6, 5), torch.randn(6, 5)
    bank.load(1, [a0, a1], [b0, b1])
    held = [bank.lora_a[1, :5], bank.lora_a[1, 8:13]], [bank.lora_b[1, :6, :5], bank.lora_b[1, 6:, :5]]
    bank.load(1, *held, scaling=0.5)
    assert torch.equal(bank.lora_a[1, :5], a0) and torch.equal(bank.lora_b[1, 6:, :5], b1) and bank.lora_scaling[1] == 0.5
    bank.load(1, held[0][::-1], held[1][::-1])
    assert torch.equal(bank.lora_a[1, :5], a1) and torch.equal(bank.lora_a[1, 8:13], a0)
    assert torch.equal(bank.lora_b[1, :6, :5], b1) and torch.equal(bank.lora_b[1, 6:, :5], b0)
    bank.load(2, bank.lora_a[1, :5], bank.lora_b[1, :, :5])
    assert torch.equal(bank.lora_a[2, 8:13], a1) and torch.equal(bank.lora_b[2], bank.lora_b[1])


def test_load_refusals_leave_the_slot():
    bank = LinearAdapters(8, [6, 4], 3, 5, torch.float32, "cpu")
    a, b0, b1 = torch.randn(5, 8), torch.randn(6, 5), torch.randn(4, 5)
    bank.load(0, [a, a], [b0, b1])
    kept = bank.lora_a.clone(), bank.lora_b.clone()
    for slot, la, lb in ((3, [a, a], [b0, b1]), (-1, [a, a], [b0, b1]), (0, [a], [b0]), (0, [a, a], [b1, b0]),
                         (0, [a, None], [b0, b1]), (0, [torch.randn(6, 8)] * 2, [torch.randn(6, 6), torch.randn(4, 6)]),
                         (0, [a[:, :7]] * 2, [b0, b1]), (0, [a, a], [b0, b1[0]]), (0, a, b0), (0, a[0], torch.cat([b0, b1]))):
        with pytest.raises(ValueError):
            bank.load(slot, la, lb)
    assert torch.equal(bank.lora_a, kept[0]) and torch.equal(bank.lora_b, kept[1])


def test_routing_refusals():
    for bad in ((0, 8), (4, 0)):
        with pytest.raises(ValueError):
            AdapterRouting(*bad, device="cpu")
    routing = AdapterRouting(4, 8, device="cpu")
    for index, rows in (([0] * 9, None), ([0, 1], 1), ([0, 1], 9), ([[0, 1]], None)):
        with pytest.raises(ValueError):
            routing.set(index, rows)
    if not torch.cuda.is_available():
        with pytest.raises(ValueError):  # the kernels need a GPU, and no batch stands after a failed set
            routing.set([0, 1])
    assert routing.batch is None
    layer = _fill(LinearBase(64, 32))
    attach_adapters(layer, slots=4, rank=8, routing=routing)
    with pytest.raises(ValueError, match="set for no rows, the call has 3"):
        layer(torch.randn(3, 64))


def test_fakes():
    bf = torch.bfloat16
    assert {"rms_norm_quant", "silu_mul_quant", "lora_add"} <= set(torch_ops.OPS)
    with FakeTensorMode():
        x = torch.empty(3, 5, 1024, dtype=bf, device="cuda")
        w = torch.empty(1024, dtype=bf, device="cuda")
        q = torch.ops.qtts
        for codes, dtype in ((ops.CODE_E4M3, torch.float8_e4m3fn), (ops.CODE_INT8, torch.int8)):
            for res, want in ((x, True), (None, False)):
                qx, sx, hidden, normed = q.rms_norm_quant(x, w, 1e-6, res, codes, want)
                assert qx.shape == (15, 1024) and qx.dtype == dtype and sx.shape == (15,) and sx.dtype == torch.float32
                assert hidden.shape == (x.shape if want else (0,)) == normed.shape and normed.dtype == bf
                qx, sx, act = q.silu_mul_quant(x, codes, want)
                assert qx.shape == (15, 512) and qx.dtype == dtype and sx.shape == (15,)
                assert act.shape == ((3, 5, 512) if want else (0,)) and act.dtype == bf
        sw = torch.empty(96, device="cuda")
        bias = torch.empty(96, dtype=bf, device="cuda")
        ws = torch.empty(96 * 512, dtype=torch.int8, device="cuda")
        for gemm in (q.w8a8_fp8_gemm_strips, q.w8a8_int8_gemm_strips):
            y = gemm(qx, sx, ws, 96, sw, bias, torch.float16, 0)
            assert y.shape == (15, 96) and y.dtype == torch.float16
        base = torch.empty(3, 5, 96, dtype=bf, device="cuda")
        index = torch.empty(15, dtype=torch.int32, device="cuda")
        y = q.lora_add(base, x, index, None, 4, torch.empty(4, 16, 1024, dtype=bf, device="cuda"),
                       torch.empty(4, 96, 16, dtype=bf, device="cuda"), torch.empty(4, device="cuda"), None, [96])
        assert y.shape == base.shape and y.dtype == bf


def test_dynamo_traces_a_layer_with_adapters():
    """A linear with adapters is its own method's op and lora_add, without a graph break."""
    import torch._dynamo
    layer = MergedLinear(64, [32, 32], dtype=torch.bfloat16, device="meta")
    routing = AdapterRouting(4, 8, device="meta")
    attach_adapters(layer, slots=4, rank=8, routing=routing)
    routing.batch = ops.LoraBatch(routing.index[:3], 4)
    torch._dynamo.reset()
    report = torch._dynamo.explain(lambda x: layer(x) + 1)(torch.empty(3, 64, dtype=torch.bfloat16, device="meta"))
    assert report.graph_break_count == 0, report.break_reasons


def test_row_forms_hold_the_row(tmp_path):
    """Rows of 8-bit codes: in registers up to 16384 columns, and a grid whose threads fit 32 bits; read twice past that."""
    rows = _run(tmp_path, """
#include <stdio.h>
#include "quant_rows_rule.h"
int main() {
  const long long ms[] = {1, 1003, 1 << 22, (1 << 22) + 1, 1 << 25};
  for (long long m : ms) {
    for (long long k = 0; k <= 16500; ++k) {
      auto f = qtts::row_form(m, k);
      printf("%lld %lld %d %d\\n", m, k, f.threads, f.vectors);
    }
    auto f = qtts::row_form(m, 1 << 20); printf("%lld %d %d %d\\n", m, 1 << 20, f.threads, f.vectors);
  }
}
""")
    assert len(rows) == 5 * 16502
    forms = set()
    for m, k, threads, vectors in rows:
        if 0 < k <= 16384 and m <= 1 << 22:
            assert threads * vectors * 8 >= k and threads * m < 1 << 32, (m, k)
            forms.add((threads, vectors))
        else:
            assert threads == 0, (m, k)
    assert forms == {(64, 1), (128, 1), (256, 1), (256, 2), (256, 3), (256, 4), (512, 3), (512, 4)}  # the kernels that are built


def test_adapter_launches_cover_their_work(tmp_path):
    """Every rank has its blocks, every group of rows a workgroup, and one launch is taken only where it is allowed."""
    rows = _run(tmp_path, """
#include <stdio.h>
#include "lora_rule.h"
using namespace qtts;
int main() {
  for (int rank = 1; rank <= 128; ++rank) printf("0 %d %d\\n", rank, lora_blocks(rank));
  for (int m = 1; m <= 64; ++m)
    for (int slots = 0; slots <= 80; ++slots) printf("1 %d %d %lld\\n", m, slots, (long long)lora_groups(m, slots));
  const int ms[] = {1, 5, 64, 65, 1003, 2048, 8192, 1 << 20}, ns[] = {1, 64, 256, 2048, 4096, 12288};
  for (int m : ms) for (int n : ns) printf("2 %d %d %d\\n", m, n, lora_up_cols(m, n));
  for (int groups = 1; groups <= 700; groups += 9)
    for (int tiles = 1; tiles <= 64; ++tiles)
      for (int pack = 0; pack < 2; ++pack)
        if (pack || tiles % 2 == 0) {
          const int t = lora_down_tiles(groups, tiles, pack);
          printf("4 %d %d %d %d %d %d\\n", groups, tiles, pack, t, lora_splits(64, 6144, 16, groups * ((tiles + t - 1) / t)),
                 lora_splits(64, 1024, 16, 1));
        }
  for (int m = 1; m < 5000; m += 7)
    for (int rank = 8; rank <= 128; rank += 8)
      printf("5 %d %d %d %d\\n", m, rank, (int)lora_max_splits(m, rank), lora_splits(m, 6144, rank, (m + 15) / 16));
  for (int rank = 1; rank <= 128; ++rank)
    for (int chunks = 1; chunks <= 48; ++chunks)
      for (int m = 1; m <= 64; m += 7)
        printf("3 %d %d %d %d %d\\n", rank, chunks, m, (int)lora_one_launch(false, m, 2048, rank, 8, chunks, chunks < 8 ? chunks : 8),
               (int)lora_one_launch(true, m, 2048, rank, 8, chunks, 1));
}
""")
    one = two = 0
    seen = set()
    for kind, *v in rows:
        if kind == 0:
            rank, blocks = v
            assert blocks * (16 if rank <= 16 else 32) >= rank and blocks <= 4
        elif kind == 1:
            m, slots, groups = v
            # the rows of at most slots adapters and of none, in groups of up to 16, fit the workgroups
            assert groups >= min(m, min(m, slots + 1) + m // 16) or groups == m, (m, slots)
        elif kind == 2:
            assert v[2] in (64, 128, 256)
        elif kind == 4:
            groups, tiles, pack, t, splits, short = v
            assert t in ((1, 2, 3, 4) if pack else (2, 4)), v  # the kernels that are built
            assert splits == (2 if groups * -(-tiles // t) <= 128 else 1) and short == 1, v
            seen.add((pack, t))
        elif kind == 5:
            m, rank, most, splits = v
            assert 1 <= splits <= most <= 2 and (rank <= 64 or most == 1), v  # within the workspace
        else:
            rank, chunks, m, free, plan = v
            assert not plan and (not free or rank <= 64)
            one, two = one + free, two + (not free)
    assert one and two
    assert seen == {(1, 1), (1, 2), (1, 3), (1, 4), (0, 2), (0, 4)}


def test_quantizing_after_attaching_keeps_the_adapters():
    """quantize_module puts its method under a linear's adapters, as attaching afterwards would; excluded and declined linears keep
    what they had."""
    from qtts_amd import QuantConfig, quantize_module
    from qtts_amd.quant.base import QuantMethodBase

    class Method(QuantMethodBase):
        name = "marked"

        def process_weights(self, layer):
            layer.marked = layer.out_features != 32  # declines o_proj's width below

        def applies_to(self, layer):
            return layer.marked

    block = _fill(Block())
    block.o_proj = LinearBase(32, 32)
    routing = AdapterRouting(4, 32, device="cpu")
    attach_adapters(block, slots=4, rank=8, routing=routing, targets=("qkv", "o_proj", "down"))
    method = Method()
    report = quantize_module(block, method, QuantConfig(method="int8", exclude_substrings=("down_proj",)), "talker")
    assert report["converted"] == 2 and report["declined"] == 1 and report["excluded"] == 1
    qkv = block.qkv_proj.quant_method
    assert isinstance(qkv, AdapterMethod) and qkv.inner is method and qkv.routing is routing
    assert block.mlp.gate_up_proj.quant_method is method
    for linear in (block.o_proj, block.mlp.down_proj):
        assert isinstance(linear.quant_method, AdapterMethod) and linear.quant_method.inner is None
    again = Method()
    quantize_module(block, again, QuantConfig(method="int8"), "talker")  # another method: under the same adapters
    assert block.qkv_proj.quant_method.inner is again and block.qkv_proj.quant_method.routing is routing


@pytest.mark.parametrize("max_rows", [8, 200])
def test_a_routing_holds_its_last_index_alone(max_rows):
    """Behind the rows of the last set there is no adapter and no plan: a captured step of more rows, or of a plan's, finds nothing of
    an earlier one.  (The kernels need a GPU: set writes its buffers, then refuses here.)"""
    routing = AdapterRouting(4, max_rows, device="cpu")

    def held(index, rows=None):
        with pytest.raises(ValueError, match="GPU tensor"):
            routing.set(index, rows)
        n = len(index)
        assert routing.index[:n].tolist() == [int(i) for i in index] and (routing.index[n:] == -1).all()
        if max_rows > 64:
            assert routing._plan.data_ptr() % 16 == 0 and routing._plan.numel() * 4 >= ops._plan_bytes(max_rows, 4)
            assert (routing._plan[:4] == -1).all()  # of no row count

    if not torch.cuda.is_available():
        address = routing.index.data_ptr()
        held([3, 2, 1, 0, 3, 2, 1, 0])
        if max_rows > 64:
            routing._plan[:4] = torch.tensor([9, 100, 4, 0], dtype=torch.int32)
        held([1, 2], 7)
        held(torch.tensor([3] * max_rows))
        held([])
        assert routing.index.data_ptr() == address


def test_a_routing_takes_whole_numbers():
    """Values that int32 cannot hold are no slot; what is no whole number is refused, not cut."""
    routing = AdapterRouting(4, 8, device="cpu")
    for bad in ([0.5, 1.0], torch.zeros(2), torch.tensor([True, False])):
        with pytest.raises(ValueError, match="whole numbers"):
            routing.set(bad)
    if not torch.cuda.is_available():
        for dtype in (torch.int64, torch.uint8, torch.int16):
            given = torch.tensor([2, 3, 1], dtype=dtype)
            with pytest.raises(ValueError, match="GPU tensor"):
                routing.set(given)
            assert routing.index[:3].tolist() == [2, 3, 1]
        given = torch.tensor([1, 2 ** 32, 2 ** 32 + 3, -2 ** 40])
        kept = given.clone()
        with pytest.raises(ValueError, match="GPU tensor"):
            routing.set(given)
        index = routing.index[:4]
        assert index[0] == 1 and not ((index[1:] >= 0) & (index[1:] < 4)).any() and torch.equal(given, kept)


def test_places_for_every_routing(tmp_path):
    """lora_groups against the most groups of 16 rows of one slot that any routing of m rows over the slots and none makes, counted
    apart: most[c][r], of r rows in up to c classes, by trying every size of the last class."""
    rows = _run(tmp_path, """
#include <stdio.h>
#include "lora_rule.h"
int main() {
  for (int m = 1; m <= 64; ++m)
    for (int slots = 0; slots <= 80; ++slots) printf("%d %d %lld\\n", m, slots, (long long)qtts::lora_groups(m, slots));
}
""")
    most = [[0] + [-1] * 64]
    for _ in range(81):
        last = most[-1]
        most.append([max(last[r], max((last[r - c] - (-c // 16) for c in range(1, r + 1) if last[r - c] >= 0), default=-1))
                     for r in range(65)])
    assert most[1][33] == 3 and most[2][34] == 4 and most[81][64] == 64
    for m, slots, groups in rows:
        assert groups >= most[slots + 1][m], (m, slots, groups, most[slots + 1][m])


def test_parts_of_k_stay_in_their_workspace(tmp_path):
    """The workspace holds each row's sums for every part of K that a call may take, whatever the workgroups are."""
    from qtts_amd import _lib

    rows = _run(tmp_path, """
#include <stdio.h>
#include "lora_rule.h"
int main() {
  const int ks[] = {1, 2040, 2048, 6144, 1 << 20}, ws[] = {1, 128, 129, 5000};
  for (int m = 1; m <= 4100; m += 41)
    for (int rank = 1; rank <= 128; rank += 7)
      for (int k : ks) for (int w : ws) printf("%d %d %d\\n", m, rank, qtts::lora_splits(m, k, rank, w));
}
""")
    L = _lib.load()
    for m, rank, splits in {tuple(r) for r in rows}:
        # a row's block: three 16-bit parts of the rank's entries (fp16: two and an exponent) in a multiple of 16 or 32
        entries = 16 if rank <= 16 else -(-rank // 32) * 32
        need = splits * m * entries * 6
        assert L.qtts_workspace_bytes(_lib.OP_LORA, m, 1, rank, 0) >= need, (m, rank, splits)
