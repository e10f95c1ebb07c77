"""RMSNorm with the residual's addition and GatedMLP's activation, straight to 8-bit codes and their scales
(ops.rms_norm_quant, ops.silu_mul_quant), against 64-bit evaluations.

Tolerances, from the arithmetic (u = 2^-24, one fp32 rounding):

* the row's scale and its values v: the sum of squares adds up to K / 64 squares a lane and then 64 lanes and at most
  16 waves, each addition off by u, halved by the square root; a handful of roundings follow (the root, its
  reciprocal, the products, silu's exponential and quotient: 16 u covers them, and an exponential's argument g
  carries |g| u more, |g| <= 64 before the result vanishes).  REL(k) below;
* a code: half a step of its grid about v / scale (e4m3: relative 2^-4, absolute 2^-10 under 2^-6; int8: 1/2), plus
  v's own error;
* 16-bit outputs: half a step of the type, eps / 2 relative, plus v's own error.
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
LIMIT = {0: 127.0, 1: 448.0}


def rel(k: int) -> float:
    return (k / 128 + 48 + 64 + 16) * U


@pytest.fixture(scope="module")
def ops():
    from qtts_amd import ops as _ops
    assert _ops.device_supported(), "GPU is not a gfx950"
    return _ops


def _rand(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _check_codes(q, s, v, codes, tol, what):
    """q and s against the 64-bit rows v."""
    amax = v.abs().amax(1).clamp_min(1e-6) if v.shape[1] else torch.full((v.shape[0],), 1e-6, dtype=torch.float64)
    want = amax / LIMIT[codes]
    assert s.dtype == torch.float32 and s.shape == want.shape
    s = s.double().cpu()
    # 1e-6 itself is rounded to fp32
    assert ((s - want).abs() <= (tol + U) * want).all(), f"{what}: scale off by {((s - want).abs() / want).max()}"
    x, got = v / want[:, None], q.cpu().double()
    half = torch.full_like(x, 0.5) if codes == 0 else torch.maximum(x.abs() * 2.0 ** -4, torch.tensor(2.0 ** -10).double())
    err = (got - x).abs()
    assert (err <= half * (1 + 4 * tol) + 2 * tol * x.abs()).all(), f"{what}: code off by {(err / half).max()} half steps"
    assert got.abs().max() <= LIMIT[codes] if got.numel() else True


def _check_16bit(y, v, tol, what):
    """y against v: one rounding to y's type (fp32: none beyond v's own error)."""
    step = torch.finfo(y.dtype).eps / 2 if y.dtype != torch.float32 else 0.0
    tiny = torch.finfo(y.dtype).smallest_normal * torch.finfo(y.dtype).eps / 2
    err = (y.double().cpu() - v).abs()
    assert (err <= (step + 2 * tol) * v.abs() + tiny).all(), f"{what}: off by {(err / v.abs().clamp_min(1e-30)).max()}"


def _norm64(h, w, eps):
    h, w = h.double().cpu(), w.double().cpu()
    return h / (h.pow(2).mean(1, keepdim=True) + eps).sqrt() * w


def _silu64(gu):
    g, u = gu.double().cpu().chunk(2, 1)
    return g * torch.sigmoid(g) * u


SHAPES = [(1, 8), (1, 2048), (3, 100), (5, 1003), (17, 1024), (9, 520), (2, 6144), (3, 7), (70, 1), (4, 8192), (2, 9001),
          (2, 12296), (2, 16384), (3, 16385), (1, 33000), (2000, 72)]


@pytest.mark.parametrize("codes", [1, 0], ids=["e4m3", "int8"])
@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("m,k", SHAPES)
def test_norm(ops, m, k, dtype, codes):
    w = 1 + _rand((k,), torch.float32, 1, 0.1)
    w = w.to(dtype)
    x = _rand((m, k), dtype, 2)
    for residual in (None, _rand((m, k), dtype, 3, 2.0)):
        for want in (False, True):
            q, s, hidden, normed = ops.rms_norm_quant(x, w, 1e-6, residual, codes, want_normed=want)
            what = f"{m}x{k} {dtype} codes {codes} residual {residual is not None}"
            h = x if residual is None else x + residual
            if residual is None:
                assert hidden is None
            else:
                assert torch.equal(hidden, h), what
            v = _norm64(h, w, 1e-6)
            _check_codes(q, s, v, codes, rel(k), what)
            assert (normed is not None) == want
            if want:
                _check_16bit(normed, v, rel(k), what)


@pytest.mark.parametrize("codes", [1, 0], ids=["e4m3", "int8"])
@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("m,k", SHAPES)
def test_silu(ops, m, k, dtype, codes):
    gu = _rand((m, 2 * k), dtype, 5, 3.0)
    for want in (False, True):
        q, s, act = ops.silu_mul_quant(gu, codes, want_act=want)
        v = _silu64(gu)
        _check_codes(q, s, v, codes, rel(0), f"{m}x{k} {dtype} {codes}")
        assert (act is not None) == want
        if want:
            _check_16bit(act, v, rel(0), f"{m}x{k} {dtype} {codes}")


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "fp16", "fp32"])
def test_strided_and_shaped(ops, dtype):
    """Rows of a wider buffer, rows that start off 16 bytes, and leading dimensions."""
    k, m = 264, 6
    wide = _rand((m, 3 * k + 9), dtype, 7)
    w = (1 + _rand((k,), torch.float32, 8, 0.1)).to(dtype)
    for off in (0, 8, 1, 3):
        x, r = wide[:, off:off + k], wide[:, off + k + 1:off + 2 * k + 1]
        q, s, hidden, normed = ops.rms_norm_quant(x, w, 1e-5, r, want_normed=True)
        qc, sc, hc, nc = ops.rms_norm_quant(x.contiguous(), w, 1e-5, r.contiguous(), want_normed=True)
        assert torch.equal(hidden, x + r) and torch.equal(hc, hidden)
        v = _norm64(x + r, w, 1e-5)
        for a, b in ((q, s), (qc, sc)):
            _check_codes(a, b, v, 1, rel(k), f"offset {off}")
        _check_16bit(normed, v, rel(k), f"offset {off}")
        gu = wide[:, off:off + 2 * k]
        q, s, act = ops.silu_mul_quant(gu, 0, want_act=True)
        _check_codes(q, s, _silu64(gu), 0, rel(0), f"offset {off}")
    x3 = _rand((2, 3, k), dtype, 9)
    q, s, hidden, normed = ops.rms_norm_quant(x3, w, 1e-5, x3, want_normed=True)
    assert hidden.shape == normed.shape == x3.shape and q.shape == (6, k) and s.shape == (6,)
    q, s, act = ops.silu_mul_quant(x3, want_act=True)
    assert act.shape == (2, 3, k // 2) and q.shape == (6, k // 2)


def test_empty(ops):
    x = torch.empty(0, 64, dtype=torch.bfloat16, device="cuda")
    w = torch.ones(64, dtype=torch.bfloat16, device="cuda")
    q, s, hidden, normed = ops.rms_norm_quant(x, w, 1e-6, x, want_normed=True)
    assert q.shape == (0, 64) and s.shape == (0,) and hidden.shape == normed.shape == (0, 64)
    q, s, act = ops.silu_mul_quant(x, want_act=True)
    assert q.shape == (0, 32) and s.shape == (0,) and act.shape == (0, 32)
    q, s, _, _ = ops.rms_norm_quant(torch.empty(3, 0, device="cuda"), torch.empty(0, device="cuda"))
    assert q.shape == (3, 0) and torch.allclose(s, torch.full_like(s, 1e-6 / 448), rtol=1e-6)
    q, s, _ = ops.silu_mul_quant(torch.empty(3, 0, device="cuda"), 0)
    assert q.shape == (3, 0) and torch.allclose(s, torch.full_like(s, 1e-6 / 127), rtol=1e-6)


@pytest.mark.parametrize("codes", [1, 0], ids=["e4m3", "int8"])
@pytest.mark.parametrize("k", [64, 2048, 2049, 12296])
def test_odd_rows_leave_the_others_alone(ops, k, codes):
    """A zero row, a row under the scale's floor, and rows of infinities and NaN among ordinary ones."""
    x = _rand((9, k), torch.bfloat16, 11)
    w = (1 + _rand((k,), torch.float32, 12, 0.1)).to(torch.bfloat16)
    plain = ops.rms_norm_quant(x, w, 1e-6, None, codes)
    odd = x.clone()
    odd[1] = 0
    odd[2, k // 2] = float("nan")
    odd[4, 3] = float("inf")
    odd[6, k - 1] = float("-inf")
    q, s, _, _ = ops.rms_norm_quant(odd, w, 1e-6, None, codes)
    for r in (0, 3, 5, 7, 8):
        assert torch.equal(q[r].view(torch.uint8), plain[0][r].view(torch.uint8)) and s[r] == plain[1][r]
    assert (q[1].float() == 0).all() and abs(s[1].item() / (1e-6 / LIMIT[codes]) - 1) < 4 * U
    for r in (2, 4, 6):
        assert torch.isnan(s[r]), "a NaN among the values makes the scale NaN"
        assert (q[r] == 0).all() if codes == 0 else torch.isnan(q[r].float()).all()
    gu = torch.cat([x, x.roll(1, 0)], 1)
    plain = ops.silu_mul_quant(gu, codes)
    gu[2, k // 2] = float("nan")
    gu[4, 3] = float("inf")
    gu[6, k + 2] = 1e-30
    gu[7] = 0
    gu[8] = gu[8] * 1e-6
    q, s, _ = ops.silu_mul_quant(gu, codes)
    for r in (0, 1, 3, 5):
        assert torch.equal(q[r].view(torch.uint8), plain[0][r].view(torch.uint8)) and s[r] == plain[1][r]
    assert torch.isnan(s[2]) and torch.isinf(s[4]) and (q[7].float() == 0).all()
    _check_codes(q[7:], s[7:], _silu64(gu[7:]), codes, rel(0), "rows under the floor")


def test_in_place_hidden(ops):
    """hidden may be x or the residual (the C entry; the wrapper always returns a fresh one)."""
    from qtts_amd import _lib
    L = _lib.load()
    for k in (2048, 1001, 12296):
        w = torch.ones(k, dtype=torch.bfloat16, device="cuda")
        for which in (0, 1):
            x, r = _rand((5, k), torch.bfloat16, 13), _rand((5, k), torch.bfloat16, 14)
            want = ops.rms_norm_quant(x, w, 1e-6, r)
            q, s = torch.empty_like(want[0]), torch.empty_like(want[1])
            target = (x, r)[which]
            st = L.qtts_rms_norm_quant(x.data_ptr(), 1, 5, k, k, r.data_ptr(), k, w.data_ptr(), 1e-6, 1, q.data_ptr(),
                                       s.data_ptr(), target.data_ptr(), k, None, k, torch.cuda.current_stream().cuda_stream)
            assert st == 0, _lib.last_error()
            torch.cuda.synchronize()
            assert torch.equal(target, want[2]) and torch.equal(s, want[1])
            assert torch.equal(q.view(torch.uint8), want[0].view(torch.uint8))


@pytest.mark.parametrize("codes", [1, 0], ids=["e4m3", "int8"])
def test_feeds_the_w8a8_gemm(ops, codes):
    """The codes and scales are what the W8A8 GEMMs take: norm, gate_up, activation, down against 64 bits."""
    m, k, inter = 5, 512, 256
    x, r = _rand((m, k), torch.bfloat16, 15), _rand((m, k), torch.bfloat16, 16)
    w = (1 + _rand((k,), torch.float32, 17, 0.1)).to(torch.bfloat16)
    pack = ops.pack_fp8 if codes else ops.pack_int8
    gemm = ops.w8a8_fp8_gemm_strips if codes else ops.w8a8_int8_gemm_strips
    up_q, up_s = pack(_rand((2 * inter, k), torch.float32, 18, 0.05))
    down_q, down_s = pack(_rand((k, inter), torch.float32, 19, 0.05))
    q, s, hidden, _ = ops.rms_norm_quant(x, w, 1e-6, r, codes)
    gu = gemm(q, s, ops.to_strips(up_q), 2 * inter, up_s)
    ref = (q.double() * s.double()[:, None]) @ (up_q.double() * up_s.double()[:, None]).t()
    rms = ref.square().mean().sqrt()
    assert ((gu.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 1e-3 * rms).all()
    q, s, _ = ops.silu_mul_quant(gu, codes)
    y = gemm(q, s, ops.to_strips(down_q), k, down_s)
    ref = (q.double() * s.double()[:, None]) @ (down_q.double() * down_s.double()[:, None]).t()
    rms = ref.square().mean().sqrt()
    assert ((y.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 1e-3 * rms).all()


def test_graph_and_stream(ops):
    """Captured once and replayed on changing inputs, with eager calls between, and on a stream of its own."""
    x, r = _rand((6, 2048), torch.bfloat16, 21), _rand((6, 2048), torch.bfloat16, 22)
    w = (1 + _rand((2048,), torch.float32, 23, 0.1)).to(torch.bfloat16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        mine = ops.rms_norm_quant(x, w, 1e-6, r, 0, True)
        mine_act = ops.silu_mul_quant(x, 0, True)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.rms_norm_quant(x, w, 1e-6, r, 0, True)
        act = ops.silu_mul_quant(out[2], 0, True)
    for i in range(3):
        x.copy_(_rand((6, 2048), torch.bfloat16, 21 + 100 * i))
        graph.replay()
        want = ops.rms_norm_quant(x, w, 1e-6, r, 0, True)
        want_act = ops.silu_mul_quant(want[2], 0, True)
        torch.cuda.synchronize()
        for a, b in zip((*out, *act), (*want, *want_act)):
            assert torch.equal(a, b), f"replay {i}"
        if i == 0:
            assert all(torch.equal(a, b) for a, b in zip(mine, want))
            assert torch.equal(mine_act[0], ops.silu_mul_quant(x, 0, True)[0])


def test_more_rows_than_workgroups(ops):
    """Past 2^20 rows a workgroup takes several."""
    m, k = (1 << 20) + 77, 16
    x = _rand((m, k), torch.bfloat16, 31)
    w = torch.ones(k, dtype=torch.bfloat16, device="cuda")
    q, s, _, _ = ops.rms_norm_quant(x, w, 1e-6, None, 0)
    pick = torch.tensor([0, 1, 12345, 1 << 19, (1 << 20) - 1, 1 << 20, m - 2, m - 1], device="cuda")
    _check_codes(q[pick], s[pick], _norm64(x[pick], w, 1e-6), 0, rel(k), "many rows")
    q, s, _ = ops.silu_mul_quant(x, 1)
    _check_codes(q[pick], s[pick], _silu64(x[pick]), 1, rel(0), "many rows")


@pytest.mark.parametrize("k", [64, 63])
def test_rows_past_32_bits(ops, k):
    """Rows so far apart that their offsets pass 2^32 elements' bytes give what the same rows do side by side."""
    m, pitch = 40, (1 << 26) + 8
    wide = [torch.empty((m - 1) * pitch + 2 * k, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    x, res, gu = (w.as_strided((m, c), (pitch, 1)) for w, c in zip(wide + wide[:1], (k, k, 2 * k)))
    g = torch.Generator(device="cuda").manual_seed(k)
    gu.copy_(torch.randn(m, 2 * k, generator=g, device="cuda")), res.copy_(torch.randn(m, k, generator=g, device="cuda"))
    w = torch.ones(k, dtype=torch.bfloat16, device="cuda")
    near = ops.rms_norm_quant(x.contiguous(), w, 1e-6, res.contiguous(), 1, True)
    for got, want in ((ops.rms_norm_quant(x, w, 1e-6, res, 1, True), near),
                      (ops.silu_mul_quant(gu, 0, True), ops.silu_mul_quant(gu.contiguous(), 0, True))):
        assert all(torch.equal(p.view(torch.uint8), q.view(torch.uint8)) for p, q in zip(got, want))


@pytest.mark.parametrize("codes", [1, 0], ids=["e4m3", "int8"])
@pytest.mark.parametrize("dtype", DTYPES[:2], ids=["bf16", "fp16"])
@pytest.mark.parametrize("m,k", [(1, 8), (64, 2048), (33, 4095), (5, 16386), (700, 1024)])
def test_norm_codes_are_the_nearest(ops, m, k, dtype, codes):
    """v / sx = h w L / max |h w| has ties, as h w and its maximum have few bits: each code is the nearest of that quotient, a tie's
    the even one.  64 bits hold h w L exactly (16 or 22 bits by 9) and the division hits every tie; no other quotient of bf16 rows
    is within 2^-24 of one, so their codes are equal.  fp16 (h w of 22 bits): quotients that are no tie but round to one in fp32, of
    a relative distance under 2^-24 and of the other parity, are one code off; a hit needs a / b within 2^-24 of one of 127 ties,
    for which no more than 1 in 2^10 of all quotients can be counted (each tie's interval is 2^-23 of its own size, 2^-8 or more
    apart: 2^-14, and room for a row of few values)."""
    w = (1 + _rand((k,), torch.float32, 41, 0.1)).to(dtype)
    x, res = _rand((m, k), dtype, 42), _rand((m, k), dtype, 43, 2.0)
    x[0], res[0], w[:8] = torch.arange(k, device="cuda") % 17 - 8, 0, 1  # whole numbers: ties in plenty
    for r in (None, res):
        q, s, _, _ = ops.rms_norm_quant(x, w, 1e-6, r, codes)
        h = x if r is None else x + r
        hw = h.double() * w.double()
        want = hw * LIMIT[codes] / hw.abs().amax(1, keepdim=True)
        want = want.round() if codes == 0 else want.to(torch.float32).to(torch.float8_e4m3fn).double()
        off = int((q.double() != want).sum())
        assert off == 0 if dtype == torch.bfloat16 else off <= want.numel() >> 10, f"{off} of {want.numel()} codes"


@pytest.mark.parametrize("codes", [1, 0], ids=["e4m3", "int8"])
def test_norm_codes_at_the_ends_of_the_range(ops, codes):
    """Values whose product with the code range passes fp32, rows at and under the scale's floor, and eps of zero."""
    k = 64
    x = _rand((6, k), torch.float32, 44)
    w = torch.ones(k, device="cuda")
    w[5], w[9] = 1e20, -7e19
    x[0] *= 1e18  # h w of 1e38 (and |x| < 3.4 of these few), h w L past fp32
    x[1] *= 1e-30  # under eps: v of 1e-27
    x[2] *= 1e-18
    x[3] = 0
    for eps in (1e-6, 0.0):
        rows = [0, 1, 2, 3, 4, 5] if eps else [0, 2, 4, 5]  # (squares of 1e-30 vanish in fp32: without eps there is no norm)
        q, s, _, _ = ops.rms_norm_quant(x[rows], w, eps, None, codes)
        _check_codes(q, s, _norm64(x[rows], w, eps), codes, rel(k), f"eps {eps}")


@pytest.mark.parametrize("codes", [1, 0], ids=["e4m3", "int8"])
@pytest.mark.parametrize("k", [16, 15])
def test_rows_that_share_a_workgroup(ops, k, codes):
    """Past 2^22 rows the long kernels take a call, 2^20 workgroups of every 2^20-th row each: rows on both sides of every multiple,
    and all rows of a few workgroups, hold to 64 bits with and without a residual and the 16-bit outputs."""
    m, step = (1 << 22) + 77, 1 << 20
    x = torch.empty(m, 2 * k, dtype=torch.bfloat16, device="cuda").normal_(generator=torch.Generator(device="cuda").manual_seed(k))
    x[3 * step + 5] = 0
    x[2 * step + 6, 1] = float("nan")  # its workgroup's other rows are 6, step + 6, 3 step + 6 and 4 step + 6
    w = (1 + _rand((k,), torch.float32, 51, 0.1)).to(torch.bfloat16)
    near = {r + d for r in range(0, m, step) for d in range(-3, 12)}
    pick = torch.tensor(sorted(r for r in near | {m - 1, m - 2} if 0 <= r < m and r != 2 * step + 6), device="cuda")
    rows, res = x[:, :k], x[:, k:]
    for residual in (None, res):
        q, s, hidden, normed = ops.rms_norm_quant(rows, w, 1e-6, residual, codes, True)
        h = rows[pick] if residual is None else rows[pick] + res[pick]
        v = _norm64(h, w, 1e-6)
        _check_codes(q[pick], s[pick], v, codes, rel(k), "norm")
        _check_16bit(normed[pick], v, rel(k), "normed")
        assert hidden is None or torch.equal(hidden[pick], h)
        assert torch.isnan(s).nonzero().flatten().tolist() == [2 * step + 6]
        del q, s, hidden, normed
    q, s, act = ops.silu_mul_quant(x, codes, want_act=True)
    v = _silu64(x[pick])
    _check_codes(q[pick], s[pick], v, codes, rel(0), "silu")
    _check_16bit(act[pick], v, rel(0), "act")
    assert torch.isnan(s).nonzero().flatten().tolist() == [2 * step + 6]


@pytest.mark.parametrize("k", [1040, 1037, 16400])
@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "fp16", "fp32"])
def test_far_gates(ops, dtype, k):
    """Gates from where e^-g nears fp32's range (silu of -1e-36, a normal number) to that range's ends: what torch's fp32 gives, within
    two roundings of the exponent's argument (2 |g| u) and 16 u more, and the type's own."""
    g = torch.linspace(-88.7, -60, k).to(dtype)
    g[:4] = torch.tensor([-1000.0, -90.0, 60000.0, 0.0]).to(dtype)
    up = torch.full((k,), 2.0 ** 14).to(dtype)
    q, s, act = ops.silu_mul_quant(torch.cat([g, up])[None].cuda(), 0, want_act=True)
    v = g.double() * torch.sigmoid(g.double()) * up.double()
    far = g.double() < -88.7228  # e^-g past fp32: zero, as torch's
    tol = (2 * g.double().abs().clamp_max(89) + 16) * U
    step = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    err = (act[0].double().cpu() - v).abs()
    assert (act[0].cpu()[far] == 0).all() and far.any()
    assert (err <= (step + tol) * v.abs() + tiny)[~far].all() if dtype != torch.float16 else torch.isfinite(act[0, 3:]).all()
