"""Attention over a paged cache (ops.paged_step, ops.paged_release, ops.qkv_to_cache, ops.paged_attention) against plain
Python integers and 64-bit arithmetic.

Tolerances, from the arithmetic (u = 2^-24, e = eps / 2 of the 16-bit type, half a step).  qkv_to_cache: e relative to the
result, plus fp32 steps of the norm (a sum of d squares, a square root, a division, two products) and of the rotation (two
products and a sum).  paged_attention, for out = sum w_j v_j / sum w_j with A = sum w_j |v_j| / sum w_j:

* a score is off by 2 (d + 4) u scale sum |q_i k_i| (products exact in fp32, sums rounded, any order) and its place under
  the maximum by 4 u (|s_j| + |max|) plus the exponential's own 2^-22: with the largest of these, r, the weights move out by at most 2 r A;
* the weights enter the second product in 16 bits: e A, and where they are below fp16's normal numbers 2^-25 each;
* n terms summed in fp32 in any order, and rescaled: 4 (n + 64) u A;
* the result is rounded once: e |out|.
"""

from __future__ import annotations

import random

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DTYPES = pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])


@pytest.fixture(scope="module")
def ops():
    from qtts_amd import ops as _ops
    assert _ops.device_supported(), "GPU is not a gfx950"
    _ops.reserve_workspace(torch.device("cuda"), 64 << 20)
    return _ops


def _rand(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32).cuda()


# ---- the step -----------------------------------------------------------------------------------


def _step_plain(new, lengths, table, free, taken, page, rows, max_new):
    """The same on lists; `table` is changed.  Returns starts, counts, lengths, positions, slots, taken."""
    starts, counts, after = [0], [], []
    positions, slots = [-1] * rows, [-1] * rows
    needed, got = 0, 0
    for r, (n, have) in enumerate(zip(new, lengths)):
        n = max(n, 0)
        at = starts[-1]
        starts.append(at + n)
        want = -(-(have + n) // page) - -(-have // page)
        ok = have >= 0 and have + n <= len(table[r]) * page and at + n <= rows and n <= max_new
        if ok:
            needed += want
            ok = want == 0 or needed <= len(free) - taken
        counts.append(n if ok else 0)
        after.append(have + (n if ok else 0))
        if not ok:
            continue
        for j in range(want):
            table[r][-(-have // page) + j] = free[taken + got + j]
        got += want
        for i in range(n):
            p = have + i
            positions[at + i] = p
            slots[at + i] = table[r][p // page] * page + p % page
    return starts, counts, after, positions, slots, taken + got


def _state(requests, page, cols, seed, held=None, spare=40):
    rng = random.Random(seed)
    held = [rng.randint(0, cols * page) for _ in range(requests)] if held is None else held
    pool = list(range(sum(-(-h // page) for h in held) + spare))
    rng.shuffle(pool)
    table, taken = [[-7] * cols for _ in range(requests)], 0
    for r, h in enumerate(held):
        for j in range(-(-h // page)):
            table[r][j] = pool[taken]
            taken += 1
    return held, table, pool, taken


def _check_step(ops, new, held, table, pool, taken, page, rows, max_new=None, in_place=False):
    dev = [_i32(new), _i32(held), _i32(table).view(len(held), -1), _i32(pool), _i32([taken])]
    out = None
    if in_place:
        fresh = [torch.full((n,), -9, dtype=torch.int32, device="cuda") for n in (len(held) + 1, len(held), rows, rows)]
        out = ops.PagedBatch(dev[2], fresh[0], fresh[1], dev[1], fresh[2], fresh[3], page, max_new=max_new, taken=dev[4])
    b = ops.paged_step(*dev, page, rows, max_new, out=out)
    want = _step_plain(new, held, table, pool, taken, page, rows, rows if max_new is None else min(max_new, rows))
    for name, got, ref in zip(("starts", "counts", "lengths", "positions", "slots"),
                              (b.starts, b.counts, b.lengths, b.positions, b.slots), want):
        assert got.tolist() == ref, name
    assert b.taken.tolist() == [want[5]] and b.table.tolist() == table
    if not in_place:
        assert dev[1].tolist() == held and dev[4].tolist() == [taken] and dev[3].tolist() == pool
    return b


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("requests,page,cols,most,rows", [
    (1, 16, 1, 1, 1), (1, 64, 40, 300, 400), (3, 16, 5, 2, 9), (64, 64, 20, 1, 64), (65, 16, 9, 1, 70), (64, 16, 9, 3, 200),
    (200, 32, 30, 90, 9000), (257, 128, 4, 60, 5000), (1000, 16, 3, 1, 1000), (2048, 16, 2, 20, 30000), (5, 1024, 3, 700, 4097)])
def test_step(ops, requests, page, cols, most, rows, in_place):
    rng = random.Random(requests + page)
    for case in range(4):
        held, table, pool, taken = _state(requests, page, cols, case, spare=rng.choice([0, 3, requests, 40 * requests]))
        held = [max(0, h - rng.randint(0, most)) for h in held]  # some pages are held ahead of the tokens: written again
        new = [rng.choice([-1, 0, 1, most, rng.randint(0, most)]) for _ in range(requests)]
        _check_step(ops, new, held, table, pool, taken, page, rows, in_place=in_place)
        _check_step(ops, new, held, table, pool, taken, page, rows, max_new=max(1, most // 2), in_place=in_place)


def test_step_edges(ops):
    # no requests; no rows; a page ends with the last token; one token past the table; exactly the pages that are left
    assert ops.paged_step(_i32([]), _i32([]), _i32([]).view(0, 4), _i32([1, 2]), _i32([0]), 16, 3).slots.tolist() == [-1] * 3
    assert ops.paged_step(_i32([2]), _i32([0]), _i32([[-1]]), _i32([5]), _i32([0]), 16, 0).counts.tolist() == [0]
    _check_step(ops, [16, 1], [0, 16], [[-1, -1], [0, -1]], [0, 2, 1], 1, 16, 17)
    _check_step(ops, [1, 1], [32, 31], [[1, 2], [3, 0]], [1, 2, 3, 0, 4], 4, 16, 2)
    for left in (2, 3, 4):  # requests that need none pass even behind one that is denied
        _check_step(ops, [40, 20, 3, 17], [0, 0, 5, 0], [[-1] * 3, [-1] * 3, [0, 0, 0], [-1] * 3], list(range(left + 1)), 1, 16, 90)
    # lengths, a count of taken pages and pages that no step makes: denied, and no slot that int32 does not hold
    b = ops.paged_step(_i32([1, 1, 1]), _i32([-5, 3, 3]), _i32([[0], [-1], [1 << 27]]), _i32([0, 1]), _i32([0]), 16, 3)
    assert b.counts.tolist() == [0, 1, 1] and b.slots.tolist() == [-1, -1, -1] and b.positions.tolist() == [-1, 3, 3]
    # a free list shorter than the cache
    _check_step(ops, [20, 3], [0, 0], [[-1, -1], [-1, -1]], [900, 70, 5], 0, 16, 23)
    for taken in (-1, 3):
        assert ops.paged_step(_i32([1]), _i32([0]), _i32([[0]]), _i32([0, 1]), _i32([taken]), 16, 1).counts.tolist() == [0]


def test_step_far_counts(ops):
    """Sums of rows past 32 bits deny what does not fit and nothing else."""
    big = 2 ** 31 - 1
    b = ops.paged_step(_i32([3, big, big, big, 2]), _i32([0] * 5), _i32([[-1]] * 5), _i32([1, 2, 3]), _i32([0]), 16, 50)
    assert b.counts.tolist() == [3, 0, 0, 0, 0] and b.positions.tolist() == [0, 1, 2] + [-1] * 47
    assert b.starts.tolist() == [0, 3, big, big, big, big] and b.taken.tolist() == [1]


def test_steps_and_releases(ops):
    """A cache in use: requests grow, finish and are replaced; no page is in two places and none is lost."""
    rng = random.Random(3)
    requests, page, cols, pages, rows = 12, 16, 8, 50, 120
    lengths, table, free, taken = _i32([0] * requests), _i32([[-1] * cols] * requests), _i32(list(range(pages))), _i32([0])
    state = ops.paged_step(_i32([0] * requests), lengths, table, free, taken, page, rows)
    state = ops.PagedBatch(table, state.starts, state.counts, lengths, state.positions, state.slots, page, taken=taken)
    for _ in range(60):
        new = [rng.choice([0, 1, 1, rng.randint(0, 40)]) for _ in range(requests)]
        want_table, want_free = table.tolist(), free.tolist()
        want = _step_plain(new, lengths.tolist(), want_table, want_free, int(taken), page, rows, rows)
        ops.paged_step(_i32(new), lengths, table, free, taken, page, rows, out=state)
        assert (state.counts.tolist(), lengths.tolist(), state.slots.tolist(), int(taken)) == (want[1], want[2], want[4], want[5])
        assert table.tolist() == want_table
        which = [rng.choice([0, 0, 0, 1, 5]) for _ in range(requests)]
        back = [p for r in range(requests) if which[r] for p in want_table[r][:-(-want[2][r] // page)]]
        ops.paged_release(_i32(which), lengths, table, free, taken, page)
        assert int(taken) == want[5] - len(back) and free.tolist()[int(taken):want[5]] == back
        assert lengths.tolist() == [0 if w else n for w, n in zip(which, want[2])]
        held = [p for r in range(requests) for p in table.tolist()[r][:-(-int(lengths[r]) // page)]]
        assert sorted(held + free.tolist()[int(taken):]) == list(range(pages))
    ops.paged_release(_i32([1] * requests), lengths, table, free, taken, page)
    ops.paged_release(_i32([1] * requests), lengths, table, free, taken, page)  # nothing left to return
    assert int(taken) == 0 and sorted(free.tolist()) == list(range(pages))


@pytest.mark.parametrize("requests,cols", [(300, 70), (2048, 3)])
def test_release_of_many(ops, requests, cols):
    held, table, pool, taken = _state(requests, 16, cols, 5)
    which = [r % 3 != 1 for r in range(requests)]
    dev = [_i32([int(w) for w in which]), _i32(held), _i32(table), _i32(pool), _i32([taken])]
    ops.paged_release(*dev, 16)
    back = [p for r in range(requests) if which[r] for p in table[r][:-(-held[r] // 16)]]
    assert int(dev[4]) == taken - len(back) and dev[3].tolist() == pool[:taken - len(back)] + back + pool[taken:]
    assert dev[1].tolist() == [0 if w else h for w, h in zip(which, held)]
    # a count of taken pages that does not hold what comes back: left as it was
    dev = [_i32([1] * requests), _i32(held), _i32(table), _i32(pool), _i32([taken - 1])]
    ops.paged_release(*dev, 16)
    assert dev[1].tolist() == held and int(dev[4]) == taken - 1 and dev[3].tolist() == pool


# ---- batches made by hand ---------------------------------------------------------------------------


def _batch(ops, requests, page, seed=0, padding=0, spare_cols=1, spare_pages=3, **bounds):
    """A batch of (held, new) requests; None: a denied request of 3 rows.  Pages in random order."""
    rng = random.Random(seed)
    lengths = [0 if r is None else r[0] + r[1] for r in requests]
    each = [-(-n // page) for n in lengths]
    pool = list(range(sum(each) + spare_pages))
    rng.shuffle(pool)
    cols = max(each, default=0) + spare_cols
    table, starts, counts, positions, slots, at = [], [0], [], [], [], 0
    for r, n, have in zip(requests, lengths, each):
        table.append(pool[at:at + have] + [2 ** 31 - 1] * (cols - have))  # what lies behind is no page
        at += have
        new = 3 if r is None else r[1]
        starts.append(starts[-1] + new)
        counts.append(0 if r is None else new)
        for p in range(n - new, n) if r is not None else [None] * 3:
            positions.append(-1 if p is None else p)
            slots.append(-1 if p is None else table[-1][p // page] * page + p % page)
    positions += [-1] * padding
    slots += [-1] * padding
    bounds.setdefault("max_new", max([c for c in counts], default=0))
    return ops.PagedBatch(_i32(table).view(len(requests), cols), _i32(starts), _i32(counts), _i32(lengths), _i32(positions), _i32(slots), page,
                          **bounds), len(pool)


# ---- keys and values into the cache -------------------------------------------------------------------


def _qkv_exact(qkv, heads, kv, d, q_norm, k_norm, eps, rope, positions):
    """(q, k, v, bounds of q and k without the last rounding), in 64 bits."""
    x = qkv.double().view(qkv.shape[0], heads + 2 * kv, d)
    out = []
    for h, w in ((x[:, :heads], q_norm), (x[:, heads:heads + kv], k_norm)):
        off = torch.zeros_like(h)
        if w is not None:
            h = h / (h.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
            off = h.abs() * U * (d / 2 + 8)  # half of the sum's relative error, then sqrt, division, two products
        if rope is not None:
            c, s = (t.double()[positions.long().clamp_min(0)].unsqueeze(1) for t in rope)
            (a, b), (ea, eb) = h.chunk(2, -1), off.chunk(2, -1)
            h = torch.cat([a * c - b * s, b * c + a * s], -1)
            mags = torch.cat([(a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()], -1)
            off = torch.cat([ea * c.abs() + eb * s.abs(), eb * c.abs() + ea * s.abs()], -1) + 3 * U * mags
        out.append((h, off))
    return out[0][0], out[1][0], x[:, heads + kv:], out[0][1], out[1][1]


def _near(got, want, off, what):
    fi = torch.finfo(got.dtype)
    tiny = fi.smallest_normal * fi.eps / 2
    err = (got.double() - want).abs()
    ok = err <= off + fi.eps / 2 * (want.abs() + off) + tiny
    assert ok.all(), f"{what}: {int((~ok).sum())} of {ok.numel()} off, first at {(~ok).nonzero()[0].tolist()}"


def _check_cache(ops, requests, page, heads, kv, d, dtype, norm=True, rope=True, seed=0, padding=0, stride=0, lead=()):
    batch, pages = _batch(ops, requests, page, seed, padding)
    rows, width = batch.rows, (heads + 2 * kv) * d
    wide = _rand((rows, width + stride), dtype, seed + 1, 2.0)
    qkv = wide[:, :width]
    q_norm, k_norm = ((_rand((d,), dtype, seed + i, 0.2) + 1) if norm else None for i in (2, 3))
    tables = None
    if rope:
        at = torch.arange(batch.table.shape[1] * page, dtype=torch.float64, device="cuda")
        angle = at[:, None] * 1e4 ** (-torch.arange(0, d, 2, dtype=torch.float64, device="cuda") / d)
        tables = angle.cos().float(), angle.sin().float()
    before = [_rand((pages, kv, page, d), dtype, seed + 4), _rand((pages, kv, d, page), dtype, seed + 5)]
    k, v = (t.clone() for t in before)
    q = ops.qkv_to_cache(qkv.view(*lead, rows, width) if lead else qkv, k, v, batch, heads, q_norm, k_norm, 1e-6, tables)
    eq, ek, ev, oq, ok = _qkv_exact(qkv, heads, kv, d, q_norm, k_norm, 1e-6, tables, batch.positions)
    live = batch.slots >= 0
    _near(q[live], eq[live], oq[live], "q")
    assert not q[~live].any()
    slot = batch.slots[live].long()
    _near(k[slot // page, :, slot % page], ek[live], ok[live], "k")
    assert torch.equal(v[slot // page, :, :, slot % page].double(), ev[live])
    k[slot // page, :, slot % page] = before[0][slot // page, :, slot % page]  # nothing else was written
    v[slot // page, :, :, slot % page] = before[1][slot // page, :, :, slot % page]
    assert torch.equal(k, before[0]) and torch.equal(v, before[1])


@DTYPES
@pytest.mark.parametrize("norm,rope", [(True, True), (False, True), (True, False), (False, False)])
@pytest.mark.parametrize("requests,page,heads,kv,d,padding", [
    ([(0, 1)], 64, 16, 8, 128, 0), ([(900, 1)], 16, 16, 8, 128, 0), ([(5, 1)] * 27, 64, 16, 8, 128, 5),
    ([(0, 300), (7, 1), (64, 64), (63, 66)], 64, 16, 8, 128, 3), ([(0, 130), None, (31, 33)], 32, 4, 2, 64, 0),
    ([(15, 18), (16, 16)], 16, 3, 1, 80, 1), ([(0, 70)], 128, 2, 2, 256, 0), ([(1, 9)], 16, 1, 1, 16, 0),
    ([(0, 40), (3, 3)], 1024, 8, 8, 48, 2), ([(100, 129)], 256, 6, 2, 112, 0)])
def test_qkv_to_cache(ops, requests, page, heads, kv, d, padding, norm, rope, dtype):
    _check_cache(ops, requests, page, heads, kv, d, dtype, norm, rope, seed=d + page, padding=padding)


@DTYPES
def test_qkv_rows_apart(ops, dtype):
    _check_cache(ops, [(3, 70), (0, 1)], 16, 4, 2, 64, dtype, stride=24)
    _check_cache(ops, [(3, 70), (0, 1)], 16, 4, 2, 64, dtype, stride=3)  # rows off 16 bytes: copied first
    _check_cache(ops, [(3, 5), (0, 1)], 16, 4, 2, 64, dtype, lead=(1,))
    _check_cache(ops, [(0, 0), None], 16, 4, 2, 64, dtype)  # no live row at all


def test_qkv_large_and_bad_values(ops):
    """A row of infinities or NaN reaches its own query, key and value alone; large rows do not overflow the norm's sum."""
    batch, pages = _batch(ops, [(0, 40)], 16)
    qkv = _rand((40, 8 * 64), torch.bfloat16, 1)
    k, v = torch.zeros(pages, 2, 16, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(pages, 2, 64, 16, dtype=torch.bfloat16, device="cuda")
    w = torch.ones(64, dtype=torch.bfloat16, device="cuda")
    clean = ops.qkv_to_cache(qkv, k, v, batch, 4, w, w).clone()
    kc, vc = k.clone(), v.clone()
    bad = qkv.clone()
    bad[7, 0], bad[9, 4 * 64 + 3], bad[11, 6 * 64 + 5] = float("nan"), float("inf"), float("-inf")
    q = ops.qkv_to_cache(bad, k, v, batch, 4, w, w)
    assert q[7, 0].isnan().all() and torch.equal(q[7, 1:], clean[7, 1:]) and torch.equal(q[8:], clean[8:])
    slot = batch.slots.long()
    assert not k[slot[9] // 16, 0, slot[9] % 16].isfinite().all()
    same = [i for i in range(40) if i != 9]
    assert torch.equal(k[slot[same] // 16, :, slot[same] % 16], kc[slot[same] // 16, :, slot[same] % 16])
    assert v[slot[11] // 16, 0, 5, slot[11] % 16] == float("-inf")
    assert int((v != vc).sum()) == 1


# ---- attention -----------------------------------------------------------------------------------------


def _exact(q, k, v, batch, window, sinks, scale):
    """(result, bound without the result's rounding) in 64 bits, request by request."""
    rows, heads, d = q.shape
    kv, page = k.shape[1], batch.page_size
    e = torch.finfo(q.dtype).eps / 2
    out, off = (torch.zeros(rows, heads, d, dtype=torch.float64, device="cuda") for _ in range(2))
    for r in range(batch.requests):
        n, count, start = int(batch.lengths[r]), int(batch.counts[r]), int(batch.starts[r])
        if not count or count > batch.max_new:
            continue
        held = batch.table[r, :-(-n // page)].long()
        at = torch.arange(n - count, n, device="cuda")[:, None]
        key = torch.arange(n, device="cuda")[None]
        seen = key <= at
        if window:
            seen &= (key > at - window) | (key < sinks)
        for h in range(kv):
            kr = k[held, h].double().reshape(-1, d)[:n]
            vr = v[held, h].double().transpose(1, 2).reshape(-1, d)[:n]
            for g in range(heads // kv):
                x = q[start:start + count, h * (heads // kv) + g].double()
                s = torch.where(seen, scale * (x @ kr.t()), -torch.inf)
                m = s.amax(1, keepdim=True)
                w = torch.where(seen, torch.exp(s - m), 0.0)
                total = w.sum(1, keepdim=True)
                # what no row sees (it may be NaN) out of the products
                any_seen = seen.any(0)[:, None]
                vs, ks = torch.where(any_seen, vr, 0.0), torch.where(any_seen, kr, 0.0)
                y = w @ vs / total
                mags = w @ vs.abs() / total
                rel = 2 * (d + 4) * U * scale * (x.abs() @ ks.abs().t()) + 4 * U * (s.abs() + m.abs())
                rel = torch.where(seen, rel, 0.0).amax(1, keepdim=True) + 2.0 ** -22
                bound = mags * (2 * rel + e + 4 * (n + 64) * U)
                if q.dtype == torch.float16:
                    bound = bound + 2.0 ** -25 * (seen.double() @ vs.abs()) / total
                out[start:start + count, h * (heads // kv) + g], off[start:start + count, h * (heads // kv) + g] = y, bound
    return out, off


def _inputs(ops, requests, page, heads, kv, d, dtype, seed=0, padding=0, **bounds):
    """Rows, a cache that is NaN wherever no token of a request is, and the batch."""
    batch, pages = _batch(ops, requests, page, seed, padding, **bounds)
    k = torch.full((pages, kv, page, d), float("nan"), dtype=dtype, device="cuda")
    v = torch.full((pages, kv, d, page), float("nan"), dtype=dtype, device="cuda")
    for r in range(batch.requests):
        at = torch.arange(int(batch.lengths[r]), device="cuda")
        slot = batch.table[r].long()[at // page] * page + at % page if len(at) else at
        k[slot // page, :, slot % page] = _rand((len(at), kv, d), dtype, seed + 10 * r + 1)
        v[slot // page, :, :, slot % page] = _rand((len(at), kv, d), dtype, seed + 10 * r + 2)
    return _rand((batch.rows, heads, d), dtype, seed + 3, 1.5), k, v, batch


def _check(ops, q, k, v, batch, window=0, sinks=0, scale=None, what=""):
    out = ops.paged_attention(q, k, v, batch, window, sinks, scale)
    want, off = _exact(q, k, v, batch, window, sinks, q.shape[2] ** -0.5 if scale is None else scale)
    _near(out, want, off, what)
    assert not out[batch.slots < 0].any()
    return out


WINDOWS = [(0, 0), (1, 0), (7, 2), (100, 4), (33, 40)]


@DTYPES
@pytest.mark.parametrize("window,sinks", WINDOWS)
@pytest.mark.parametrize("held,page,heads,kv,d", [
    ([0], 64, 16, 8, 128), ([0, 1, 14, 15, 16, 30, 31, 32, 33, 62, 63, 64, 65, 127, 128], 16, 16, 8, 128), ([299, 2], 64, 16, 8, 128),
    ([1000, 0, 3000, 77, 513], 32, 16, 8, 128), ([5, 700], 128, 8, 8, 128), ([40, 257], 16, 16, 1, 64), ([90, 255, 256], 256, 4, 1, 256),
    ([33, 500], 64, 12, 4, 80), ([1, 100], 16, 14, 2, 112), ([65, 66], 16, 2, 1, 16), ([129], 1024, 28, 4, 96), ([50, 640], 64, 32, 1, 128)])
def test_single_tokens(ops, held, page, heads, kv, d, window, sinks, dtype):
    q, k, v, batch = _inputs(ops, [(h, 1) for h in held], page, heads, kv, d, dtype, seed=d + len(held))
    _check(ops, q, k, v, batch, window, sinks)


@DTYPES
@pytest.mark.parametrize("window,sinks", WINDOWS)
@pytest.mark.parametrize("requests,page,heads,kv,d,padding", [
    ([(0, 2)], 64, 16, 8, 128, 0), ([(0, 37), (0, 12), (0, 1)], 64, 16, 8, 128, 3), ([(0, 64)], 16, 16, 8, 128, 0),
    ([(0, 65), None, (100, 63)], 32, 16, 8, 128, 1), ([(0, 300), (299, 130)], 64, 16, 8, 128, 0), ([(31, 129), (1, 128)], 16, 4, 4, 128, 0),
    ([(0, 100), (70, 40)], 64, 16, 1, 64, 0), ([(10, 70)], 128, 4, 1, 256, 2), ([(0, 90), (33, 33)], 16, 12, 4, 80, 0), ([(5, 50)], 256, 3, 1, 16, 0),
    ([(700, 8), (3, 9), (0, 0), (800, 1)], 64, 16, 8, 128, 0), ([(1000, 200)], 64, 8, 2, 112, 0), ([(0, 600)], 1024, 2, 1, 128, 0)])
def test_many_tokens(ops, requests, page, heads, kv, d, padding, window, sinks, dtype):
    q, k, v, batch = _inputs(ops, requests, page, heads, kv, d, dtype, seed=d + len(requests), padding=padding)
    _check(ops, q, k, v, batch, window, sinks)


@DTYPES
@pytest.mark.parametrize("heads,kv,d,page", [(16, 8, 128, 64), (16, 8, 128, 16), (8, 8, 64, 32), (16, 1, 256, 64), (28, 4, 80, 128)])
@pytest.mark.parametrize("held,window,sinks", [([9000], 0, 0), ([20000, 3, 700], 0, 0), ([6000] * 5, 3000, 4), ([4095, 12345, 1], 0, 0),
                                               ([8000, 100], 5000, 300)])
def test_split_lengths(ops, held, window, sinks, heads, kv, d, page, dtype):
    """Lengths that several workgroups share, next to short ones; again on the workspace that the first call left."""
    q, k, v, batch = _inputs(ops, [(h, 1) for h in held], page, heads, kv, d, dtype, seed=len(held), padding=1)
    first = _check(ops, q, k, v, batch, window, sinks)
    for _ in range(2):
        assert torch.equal(ops.paged_attention(q, k, v, batch, window, sinks), first)


@DTYPES
@pytest.mark.parametrize("heads,kv,d,page", [(16, 8, 128, 64), (16, 8, 128, 16), (8, 8, 64, 32), (16, 1, 256, 64), (28, 4, 80, 128), (6, 2, 16, 16)])
@pytest.mark.parametrize("requests,window,sinks", [([(9000, 20)], 0, 0), ([(20000, 100), (3, 5), (700, 40)], 0, 0), ([(6000, 30)] * 3, 3000, 4),
                                                   ([(4095, 300), (1, 1)], 0, 0), ([(8000, 129)], 5000, 300)])
def test_split_runs(ops, requests, window, sinks, heads, kv, d, page, dtype):
    """Runs of many rows whose keys several workgroups share."""
    q, k, v, batch = _inputs(ops, requests, page, heads, kv, d, dtype, seed=len(requests), padding=1)
    first = _check(ops, q, k, v, batch, window, sinks)
    for _ in range(2):
        assert torch.equal(ops.paged_attention(q, k, v, batch, window, sinks), first)


@DTYPES
@pytest.mark.parametrize("requests,heads,kv", [([(50, 3), (0, 8), (1000, 1), (5000, 5)], 16, 8), ([(40, 4), (33, 2)], 4, 1), ([(100, 16)], 2, 2)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (20, 3)])
def test_drafted_tokens(ops, requests, heads, kv, window, sinks, dtype):
    """A few tokens a request (rows of a run at several positions), as when drafts are verified."""
    q, k, v, batch = _inputs(ops, requests, 32, heads, kv, 128, dtype, seed=5)
    _check(ops, q, k, v, batch, window, sinks)


def _poison(k, v, batch, r, positions, value, where):
    at = torch.tensor(positions, device="cuda")
    slot = batch.table[r].long()[at // batch.page_size] * batch.page_size + at % batch.page_size
    if "k" in where:
        k[slot // batch.page_size, :, slot % batch.page_size] = value
    if "v" in where:
        v[slot // batch.page_size, :, :, slot % batch.page_size] = value


@DTYPES
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("heads,kv,d", [(16, 8, 128), (4, 4, 64), (8, 1, 256), (4, 2, 80)])
@pytest.mark.parametrize("count", [1, 2, 7, 60, 150])
def test_what_a_row_does_not_see(ops, count, heads, kv, d, value, dtype):
    """Infinities and NaN in tokens behind a row, or outside its window, do not reach it; those it sees do."""
    requests = [(200, count), (3, 1)]
    q, k, v, batch = _inputs(ops, requests, 16, heads, kv, d, dtype, seed=7)
    clean = [_check(ops, q, k, v, batch, w, s) for w, s in ((0, 0), (50, 4))]
    if count > 1:  # the last token's: the rows before it do not see it
        kk, vv = k.clone(), v.clone()
        _poison(kk, vv, batch, 0, [200 + count - 1], value, "kv")
        for (w, s), want in zip(((0, 0), (50, 4)), clean):
            out = ops.paged_attention(q, kk, vv, batch, w, s)
            _check_rows(out, want, [r for r in range(count + 1) if r != count - 1])
    kk, vv = k.clone(), v.clone()
    _poison(kk, vv, batch, 0, list(range(4, 151)), value, "kv")  # outside the window, but of 50 keys in front of the first row
    out = ops.paged_attention(q, kk, vv, batch, 50, 4)
    _check_rows(out, clean[1], list(range(count + 1)))
    kk, vv = k.clone(), v.clone()  # seen by all rows, values alone: infinities come out as they are
    _poison(kk, vv, batch, 0, [199], value, "v")
    out = ops.paged_attention(q, kk, vv, batch)
    assert not out[:count].isfinite().any() and out[count:].isfinite().all()
    if value == value:
        assert (out[:count] == value).all()


def _check_rows(out, want, rows):
    """The rows as they are without the bad values (bit for bit up to the join of other tiles: within two steps)."""
    fi = torch.finfo(out.dtype)
    err = (out[rows].double() - want[rows].double()).abs()
    assert (err <= 2 * fi.eps * want[rows].double().abs().amax(-1, keepdim=True) + fi.tiny).all()


@DTYPES
@pytest.mark.parametrize("count,most,mixed", [(64, 40, False), (65, 200, False), (130, 90, True), (500, 300, False), (2048, 40, True)])
def test_many_requests(ops, count, most, mixed, dtype):
    """More requests than a wave has lanes: single tokens alone, and between prompts and drafts; a few denied ones."""
    rng = random.Random(count)
    requests = [None if rng.random() < 0.03 else (rng.randint(0, most), rng.choice([1, 1, 1, 3, 9, rng.randint(1, 40)]) if mixed else 1)
                for _ in range(count)]
    q, k, v, batch = _inputs(ops, requests, 16, 4, 2, 64, dtype, seed=count, padding=5)
    _check(ops, q, k, v, batch)
    _check(ops, q, k, v, batch, 20, 3)


@DTYPES
def test_one_long_among_short(ops, dtype):
    """A chunk behind a long cache, whose keys are split, next to prompts, drafts and single tokens."""
    requests = [(9000, 70), (0, 5), (100, 1), (3000, 1), (40, 200), (0, 1), (12000, 1)]
    q, k, v, batch = _inputs(ops, requests, 64, 8, 4, 128, dtype, seed=2, padding=2)
    first = _check(ops, q, k, v, batch)
    _check(ops, q, k, v, batch, 4000, 5)
    for _ in range(2):
        assert torch.equal(ops.paged_attention(q, k, v, batch), first)


def test_rows_apart_and_bounds(ops):
    """Query rows out of a wider tensor, off 16 bytes too; requests past max_new and lengths that no step makes get zeros."""
    requests = [(40, 1), (0, 30), (5, 2), (100, 1)]
    q, k, v, batch = _inputs(ops, requests, 16, 4, 2, 64, torch.bfloat16, seed=3, padding=3)
    want = _check(ops, q, k, v, batch)
    for width, lead in ((4 * 64 + 128, 64), (4 * 64 + 5, 3)):
        wide = torch.full((batch.rows, width), float("nan"), dtype=q.dtype, device="cuda")
        wide[:, lead:lead + 256] = q.view(batch.rows, 256)
        view = wide[:, lead:lead + 256].unflatten(1, (4, 64))
        assert torch.equal(ops.paged_attention(view, k, v, batch), want)
    assert torch.equal(ops.paged_attention(q.transpose(0, 1).contiguous().transpose(0, 1), k, v, batch), want)
    few = ops.PagedBatch(batch.table, batch.starts, batch.counts, batch.lengths, batch.positions, batch.slots, 16, max_new=2)
    out = ops.paged_attention(q, k, v, few)
    kept = [0, *range(31, 34)]
    assert not out[1:31].any() and torch.equal(out[34:], want[34:])
    _check_rows(out, want, kept)
    for field, value in (("lengths", 1 << 20), ("lengths", 0), ("lengths", -7), ("counts", 500), ("starts", -3), ("starts", 1 << 30)):
        parts = {n: getattr(batch, n).clone() for n in ("table", "starts", "counts", "lengths", "positions", "slots")}
        parts[field][1] = value
        odd = ops.PagedBatch(**parts, page_size=16, max_new=30)
        out = ops.paged_attention(q, k, v, odd)
        _check_rows(out, want, [0, 31, 32, 33] if field != "starts" else [31, 32, 33])
        if field == "lengths":
            assert not out[1:31].any()
    parts = {n: getattr(batch, n).clone() for n in ("table", "starts", "counts", "lengths", "positions", "slots")}
    parts["table"][1] = torch.tensor([-1, 2 ** 31 - 1, 10 ** 6], device="cuda")[torch.arange(parts["table"].shape[1], device="cuda") % 3]
    out = ops.paged_attention(q, k, v, ops.PagedBatch(**parts, page_size=16, max_new=30))  # entries that are no page: a page all the same
    _check_rows(out, want, [0, 31, 32, 33])
    slots = batch.slots.clone()
    slots[2], slots[5], slots[7] = 2 ** 31 - 1, -2 ** 31, k.shape[0] * 16  # slots outside the cache: nothing is written
    kc, vc = torch.zeros_like(k), torch.zeros_like(v)
    qkv = _rand((batch.rows, 8 * 64), torch.bfloat16, 4)
    out = ops.qkv_to_cache(qkv, kc, vc, ops.PagedBatch(batch.table, batch.starts, batch.counts, batch.lengths, batch.positions, slots, 16), 4)
    live = [i for i in range(34) if i not in (2, 5, 7)]
    assert not out[[2, 5, 7, 34, 35, 36]].any() and (out[live] != 0).any(-1).all()
    assert int((kc != 0).any(-1).sum()) == 2 * len(live)


@pytest.mark.parametrize("new", [1, 80])
def test_caches_past_32_bits(ops, new):
    """Pages whose bytes and elements pass 2^32, on either side of those offsets."""
    pages, kv, d, page = 70000, 8, 128, 64
    k, v = (torch.empty(shape, dtype=torch.bfloat16, device="cuda") for shape in ((pages, kv, page, d), (pages, kv, d, page)))
    assert k.numel() > 1 << 32
    used = [0, 32767, 32768, 65535, 65536, pages - 1, 1, 16384, 49152]
    table = _i32([used[:5], used[5:] + [7]])
    lengths = [5 * 64 - 3, 4 * 64]
    for i, p in enumerate(used + [7]):
        k[p], v[p] = _rand((kv, page, d), torch.bfloat16, i), _rand((kv, d, page), torch.bfloat16, 50 + i)
    at = [list(range(n - new, n)) for n in lengths]
    slots = [[table.tolist()[r][p // page] * page + p % page for p in at[r]] for r in range(2)]
    batch = ops.PagedBatch(table, _i32([0, new, 2 * new]), _i32([new, new]), _i32(lengths), _i32(at[0] + at[1]), _i32(slots[0] + slots[1]), page,
                           max_new=new)
    qkv = _rand((2 * new, 32 * d), torch.bfloat16, 3)
    q = ops.qkv_to_cache(qkv, k, v, batch, 16)
    slot = batch.slots.long()
    assert torch.equal(k[slot // page, :, slot % page], qkv.view(2 * new, 32, d)[:, 16:24])
    assert torch.equal(v[slot // page, :, :, slot % page], qkv.view(2 * new, 32, d)[:, 24:])
    _check(ops, q, k, v, batch)
    _check(ops, q, k, v, batch, 100, 70)


def test_first_calls_of_a_process(ops, monkeypatch):
    """Without a workspace yet: a call of no rows needs none, any other reserves its own; a captured one says what is missing."""
    monkeypatch.setattr(ops, "_workspaces", {})
    q, k, v, batch = _inputs(ops, [(0, 0)], 16, 4, 2, 64, torch.bfloat16)
    assert ops.paged_attention(q, k, v, batch).shape == (0, 4, 64)
    assert ops.qkv_to_cache(torch.empty(0, 8 * 64, dtype=torch.bfloat16, device="cuda"), k, v, batch, 4).shape == (0, 4, 64)
    assert not ops._workspaces
    q, k, v, batch = _inputs(ops, [(30, 1)], 16, 4, 2, 64, torch.bfloat16)
    _check(ops, q, k, v, batch)
    assert len(ops._workspaces) == 1
    monkeypatch.setattr(ops, "_workspaces", {})
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(ValueError, match="reserve_workspace"):
        with torch.cuda.graph(graph):
            ops.paged_attention(q, k, v, batch)


def test_large_scores(ops):
    """Scores of hundreds, rising and falling along the keys (the running maximum moves on every tile), and one that
    leaves all others without weight."""
    for dtype in (torch.bfloat16, torch.float16):
        for requests in ([(700, 1), (2000, 1)], [(100, 150), (1500, 70)]):
            q, k, v, batch = _inputs(ops, requests, 64, 8, 4, 128, dtype, seed=6)
            for ramp in (0.02, -0.02):
                kk = k.clone()
                for r in range(2):
                    at = torch.arange(int(batch.lengths[r]), device="cuda")
                    slot = batch.table[r].long()[at // 64] * 64 + at % 64
                    kk[slot // 64, :, slot % 64] = (kk[slot // 64, :, slot % 64].float() + ramp * at[:, None, None]).to(dtype)
                qq = (q.float() + 1).to(dtype)
                _check(ops, qq, kk, v, batch)
                _check(ops, qq, kk, v, batch, 130, 4)
            _check(ops, q, k, v, batch, scale=2.0)
            _check(ops, q, k, v, batch, scale=1e-3)


@DTYPES
@pytest.mark.parametrize("count", [1, 5, 70])
def test_unwritten_memory_of_any_bits(ops, count, dtype):
    """What lies behind a request's tokens on its last page may hold any bits, signalling NaN among them."""
    q, k, v, batch = _inputs(ops, [(33, count), (0, count)], 64, 8, 4, 128, dtype, seed=count)
    want = _check(ops, q, k, v, batch, 30, 2)
    exponent = 0x7f80 if dtype == torch.bfloat16 else 0x7c00
    for bits in (exponent + 1, exponent + 0x8001 - 0x10000, exponent, exponent + 0x8000 - 0x10000):
        for t in (k, v):
            t.view(torch.int16)[t.isnan()] = bits
        assert torch.equal(ops.paged_attention(q, k, v, batch, 30, 2), want)
        for t in (k, v):
            t[~t.isfinite()] = float("nan")
