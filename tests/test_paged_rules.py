"""Attention over a paged cache without a GPU: the rules that the kernels and their launcher share (csrc/paged_rule.h,
compiled alone), what the C entries and the wrappers refuse, the cache's host side and the custom ops' fakes."""

from __future__ import annotations

import ctypes
import os
import shutil
import subprocess

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from qtts_amd import PagedCache, _lib, ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "tts-inference_amd", "csrc")


# ---- the rules ------------------------------------------------------------------------------------


def _run(tmp_path, source: str) -> str:
    cxx = shutil.which("g++") or shutil.which("clang++")
    if not cxx:
        pytest.skip("no C++ compiler")
    src, exe = tmp_path / "rule.cpp", tmp_path / "rule"
    src.write_text('#include <initializer_list>\n#include <stdio.h>\n#include <stdlib.h>\n#include "paged_rule.h"\nusing namespace qtts;\n' + source)
    subprocess.run([cxx, "-std=c++17", "-O1", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover=undefined", "-I", CSRC,
                    str(src), "-o", str(exe)], check=True)
    return subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout


def test_key_tiles_hold_every_visible_key_once(tmp_path):
    """Every key that some row of a run sees is in exactly one tile of the list, the tiles ascend and none is without one; and
    no list is longer than most_tiles says."""
    assert _run(tmp_path, """
template <int T> long long check(int lo, int hi, int window, int sinks) {
  const KeyTiles t = key_tiles<T>(lo, hi, window, sinks);
  if (t.count < 1 || key_tile(t, t.count - 1) != hi / T) abort();
  for (int i = 1; i < t.count; ++i) if (key_tile(t, i) <= key_tile(t, i - 1)) abort();
  for (int k = 0, i = 0; k <= hi; ++k) {
    bool seen = false;
    for (int p = lo; p <= hi; ++p) seen |= k <= p && (!window || k > p - window || k < sinks);
    while (i < t.count && key_tile(t, i) < k / T) ++i;
    if (seen && (i >= t.count || key_tile(t, i) != k / T)) abort();
  }
  for (int i = 0; i < t.count; ++i) {
    bool any = false;
    for (int k = key_tile(t, i) * T; k < key_tile(t, i) * T + T && k <= hi; ++k) any |= !window || k > lo - window || k < sinks;
    if (!any) abort();
  }
  for (int later = 0; later < 2 * T; later += 7) if (t.count > most_tiles<T>(hi + 1 + later, hi - lo + 1, window, sinks)) abort();
  return 1;
}
int main() {
  long long n = 0;
  const int windows[] = {0, 1, 2, 31, 32, 33, 64, 100, 1000, 2147483647}, kept[] = {0, 1, 4, 32, 33, 200, 2147483647};
  for (int lo : {0, 1, 30, 31, 32, 63, 64, 200, 333})
    for (int span : {1, 2, 3, 16, 64, 65})
      for (int w : windows)
        for (int s : kept) n += check<32>(lo, lo + span - 1, w, s) + check<64>(lo, lo + span - 1, w, s);
  printf("%lld", n);
}
""") == str(9 * 6 * 10 * 7 * 2)


def test_splits_stay_within_their_slots_and_counters(tmp_path):
    """For calls of all kinds of lengths: the splits of the runs that are split have slots, counters are enough for them, and equal
    splits cover every tile."""
    assert _run(tmp_path, """
int main() {
  unsigned seed = 1;
  auto rnd = [&](int n) { seed = seed * 1664525u + 1013904223u; return (int)((seed >> 8) % (unsigned)n); };
  for (int call = 0; call < 200000; ++call) {
    const int kv = 1 << rnd(9), runs = 1 + rnd(1 << rnd(11)), longest = 1 + rnd(1 << rnd(21)), many = rnd(2);
    const PagedCut cut = many ? many_cut((long long)runs * kv) : small_cut((long long)runs * kv);
    if (cut.groups > kCutGroups || split_slots(cut.groups) > 16384 || cut.least < 1) abort();
    const int groups = cut.groups / kv;
    if (!groups) continue;
    unsigned long long total = 0;
    const unsigned first = seed;
    for (int r = 0; r < runs; ++r) total += 1 + rnd(longest);
    seed = first;
    const unsigned share = tiles_a_split(total, groups, cut.least);
    long long slots = 0, items = 0;
    for (int r = 0; r < runs; ++r) {
      const int tiles = 1 + rnd(longest);
      const unsigned mine = joined_share(tiles, share, many ? 1.0f : (1 + r * 97 % 4096) * kPartCost);
      const int n = splits_of(tiles, mine), chunk = (tiles + n - 1) / n;
      if (mine < share) abort();
      if ((tiles + chunk - 1) / chunk > n || n > splits_of(longest, cut.least)) abort();
      items += n;
      if (n > 1) slots += n;
    }
    if (slots > split_slots(groups) || slots * kv > split_slots(cut.groups) || items > (long long)runs + groups) abort();
  }
  // totals past 32 bits and the largest sizes
  for (unsigned long long total : {0ull, 1ull, 4294967295ull, 4294967296ull, 1ull << 40, 1ull << 60})
    for (int groups : {1, 7, 512, 4096}) {
      const unsigned long long c = (total + groups - 1) / groups, want = c < 8 ? 8 : c > 0x40000000 ? 0x40000000 : c;
      if (tiles_a_split(total, groups, 8) != want) abort();
    }
  for (int tiles : {0, 1, (1 << 27) - 1})
    for (unsigned share : {8u, 9u, 1u << 27, 0x40000000u}) {
      const long long n = (2ll * tiles + share) / (2ll * share);
      if (splits_of(tiles, share) != (n > 1 ? n : 1)) abort();
    }
  printf("fine");
}
""") == "fine"


def test_requests_and_pages_that_no_step_makes(tmp_path):
    """Rows outside the batch, more rows than tokens, tokens past the table, more rows than the bound: a request of none; any
    entry of a page table is a page of the cache."""
    assert _run(tmp_path, """
int main() {
  const int big = 2147483647;
  struct { int start, count, length, rows; long long capacity; int most, want; } cases[] = {
    {0, 1, 1, 1, 16, 1, 1}, {3, 5, 20, 8, 32, 5, 5}, {3, 6, 20, 8, 32, 6, 0}, {-1, 2, 20, 8, 32, 6, 0}, {0, 5, 4, 8, 32, 6, 0},
    {0, 5, 33, 8, 32, 6, 0}, {0, 5, 32, 8, 32, 4, 0}, {0, 0, 4, 8, 32, 6, 0}, {0, -3, 4, 8, 32, 6, 0}, {big, big, big, 8, 1ll << 40, big, 0},
    {0, 1, -5, 8, 32, 6, 0}, {0, big, big, big, 1ll << 31, big, big}};
  for (auto& c : cases) {
    const PagedRequest r = paged_request(c.start, c.count, c.length, c.rows, c.capacity, c.most);
    if (r.count != c.want || (c.want && (r.start != c.start || r.length != c.length))) abort();
  }
  for (int pages : {1, 7, big})
    for (int page : {0, 1, 6, 7, -1, -big - 1, big}) {
      const unsigned p = paged_page(page, pages);
      if (p >= (unsigned)pages || (page >= 0 && page < pages && p != (unsigned)page)) abort();
    }
  printf("fine");
}
""") == "fine"


# ---- refusals ---------------------------------------------------------------------------------------


BUF = ctypes.create_string_buffer(1 << 20)
AT = (ctypes.addressof(BUF) + 255) & ~255


def _at(v):
    return None if v is None else AT + v


def _refused(status, text):
    assert status in (-1, -5) and text in _lib.last_error(), (status, _lib.last_error())


def _passes(status):
    """Past every check: no device here, or the call ran nothing."""
    assert status == 0 or (status == -2 and not torch.cuda.is_available()), _lib.last_error()


def test_step_entry():
    L = _lib.load()

    def call(added=0, requests=4, lengths=64, table=128, cols=3, free=1024, pages=8, taken=2048, page=16, rows=10, room=10, most=5,
             starts=2112, counts=2176, after=64, left=2048, positions=4096, slots=8192, ws=16384, ws_n=65536):
        return L.qtts_paged_step(_at(added), requests, _at(lengths), _at(table), cols, _at(free), pages, _at(taken), page, rows, room, most,
                                 _at(starts), _at(counts), _at(after), _at(left), _at(positions), _at(slots), _at(ws), ws_n, None)

    for kw in ({"requests": -1}, {"cols": -1}, {"pages": -1}, {"rows": -1, "room": 0}, {"most": -1}):
        _refused(call(**kw), "negative size")
    for page in (0, 1, 8, 17, 48, 2048, -16):
        _refused(call(page=page), "power of two")
    _refused(call(requests=2049), "at most 2048")
    for kw in ({"pages": 1 << 27}, {"cols": 1 << 27}, {"rows": 1 << 31, "room": 1 << 31}, {"pages": 1 << 21, "page": 1024}):
        _refused(call(**kw), "too large")
    _refused(call(room=9), "room for 9 of 10")
    for null in ("added", "lengths", "table", "free", "taken", "starts", "counts", "after", "left", "positions", "slots"):
        _refused(call(**{null: None}), "null pointer")
    _refused(call(ws=None), "workspace")
    _refused(call(ws_n=65535), "workspace")
    if not torch.cuda.is_available():
        _passes(call())
        _passes(call(requests=0, added=None, lengths=None, counts=None, after=None, table=None))
        _passes(call(rows=0, room=0, positions=None, slots=None))
    assert ops.PAGED_MAX_REQUESTS == 2048


def test_release_entry():
    L = _lib.load()

    def call(which=0, requests=4, lengths=64, table=128, cols=3, free=1024, pages=8, taken=2048, page=16):
        return L.qtts_paged_release(_at(which), requests, _at(lengths), _at(table), cols, _at(free), pages, _at(taken), page, None)

    _refused(call(requests=-1), "negative size")
    _refused(call(page=24), "power of two")
    _refused(call(requests=4000), "at most")
    for null in ("which", "lengths", "table", "free", "taken"):
        _refused(call(**{null: None}), "null pointer")
    for none in ({"requests": 0}, {"cols": 0}, {"pages": 0}):
        assert call(**none) == 0
    if not torch.cuda.is_available():
        _passes(call())


def test_qkv_entry():
    L = _lib.load()

    def call(qkv=0, dt=1, rows=2, ld=128, heads=4, kv=2, d=16, positions=8192, slots=8256, qn=8320, kn=8384, cos=8448, sin=12544,
             turns=32, k=65536, v=131072, pages=8, page=16, q=16384):
        return L.qtts_qkv_to_cache(_at(qkv), dt, rows, ld, heads, kv, d, _at(positions), _at(slots), _at(qn), _at(kn), 1e-6, _at(cos),
                                   _at(sin), turns, _at(k), _at(v), pages, page, _at(q), None)

    for dt in (0, 3, -1):
        _refused(call(dt=dt), "bf16 or fp16")
    for kw in ({"heads": 3}, {"heads": 0}, {"kv": 0}, {"heads": 8192}):
        _refused(call(**kw), "query heads")
    for d in (0, 8, 24, 272, -16):
        _refused(call(d=d), "heads of")
    _refused(call(rows=-1), "negative size")
    _refused(call(rows=1 << 24), "too large")
    _refused(call(ld=127), "leading dimension")
    _refused(call(ld=1 << 40), "too large")
    _refused(call(sin=None), "half a rotation table")
    _refused(call(turns=0), "half a rotation table")
    for null in ("qkv", "slots", "q", "positions", "k", "v"):
        _refused(call(**{null: None}), "null pointer")
    for off in ({"qkv": 2}, {"q": 16386}, {"ld": 132}, {"qn": 8328}, {"cos": 8452}, {"k": 65544}):
        with_off = call(**off)
        assert with_off == -1 and ("16 bytes" in _lib.last_error() or "unaligned" in _lib.last_error())
    _refused(call(q=128), "q overlaps qkv")
    _refused(call(q=65600), "the cache overlaps")
    _refused(call(qkv=131072 + 4096), "the cache overlaps")
    assert call(rows=0) == 0
    if not torch.cuda.is_available():
        for fine in ({}, {"qn": None, "kn": None}, {"cos": None, "sin": None, "positions": None}):
            _passes(call(**fine))


def test_attention_entry():
    L = _lib.load()

    def call(q=0, dt=1, rows=2, ldq=64, heads=4, kv=2, d=16, k=65536, v=131072, pages=8, page=16, table=4096, requests=2, cols=3,
             starts=5120, counts=5184, lengths=5248, slots=5312, least=1, most=1, window=0, sinks=0, scale=0.25, out=8192, ldo=64,
             ws=262144, ws_n=1 << 62):
        return L.qtts_paged_attention(_at(q), dt, rows, ldq, heads, kv, d, _at(k), _at(v), pages, page, _at(table), requests, cols,
                                      _at(starts), _at(counts), _at(lengths), _at(slots), least, most, window, sinks, scale, _at(out), ldo,
                                      _at(ws), ws_n, None)

    _refused(call(dt=0), "bf16 or fp16")
    for kw in ({"rows": -1}, {"least": -1}, {"most": -1}, {"window": -1}, {"sinks": -1}, {"requests": -1}):
        _refused(call(**kw), "negative size")
    _refused(call(page=100), "power of two")
    _refused(call(heads=5), "query heads")
    _refused(call(d=20), "heads of")
    _refused(call(ldq=63), "leading dimension")
    _refused(call(ldo=56), "leading dimension")
    _refused(call(ldo=1 << 40), "too large")
    for scale in (0.0, -1.0, float("nan"), float("inf"), 3e38):
        _refused(call(scale=scale), "scale")
    for null in ("q", "out", "slots", "table", "starts", "counts", "lengths", "k", "v"):
        _refused(call(**{null: None}), "null pointer")
    for off in ({"q": 2}, {"out": 8194}, {"ldq": 68}, {"ldo": 68}):
        _refused(call(**off), "16 bytes")
    _refused(call(out=64), "out overlaps q")
    _refused(call(out=131072 + 512), "out overlaps the cache")
    _refused(call(ws=None), "workspace")
    need = L.qtts_workspace_bytes(_lib.OP_PAGED_ATTENTION, 2, 1, 16, 0)
    _refused(call(ws_n=need - 1), "workspace")
    assert call(rows=0) == 0
    if not torch.cuda.is_available():
        for fine in ({"ws_n": need}, {"window": 1 << 40, "sinks": 1 << 40}, {"requests": 0, "starts": None, "counts": None, "lengths": None},
                     {"least": 5, "most": 1 << 40}):
            _passes(call(**fine))


def test_workspace_query():
    L = _lib.load()
    small, more, many = (L.qtts_workspace_bytes(_lib.OP_PAGED_ATTENTION, m, 1, 128, 0) for m in (2, 16, 17))
    assert 65536 < small < more <= many < 1 << 28
    assert L.qtts_workspace_bytes(_lib.OP_PAGED_ATTENTION, 2, 1, 257, 0) == -1
    assert L.qtts_workspace_bytes(_lib.OP_PAGED_ATTENTION, (1 << 31) - 1, 1, 256, 0) > 0


def _i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def test_wrappers():
    table, lengths, free, taken, new = _i32(3, 4), _i32(3), _i32(9), _i32(1), _i32(3)

    def step(new=new, lengths=lengths, table=table, free=free, taken=taken, page=16, rows=5, **kw):
        return ops.paged_step(new, lengths, table, free, taken, page, rows, **kw)

    with pytest.raises(ValueError, match="GPU tensor"):
        step()
    for match, kw in (("page table", {"table": table[0]}), ("page table", {"table": table.long()}), ("page table", {"table": table.t()}),
                      ("rows", {"rows": -1})):
        with pytest.raises(ValueError, match=match):
            step(**kw)
    fields = {"table": table, "starts": _i32(4), "counts": _i32(3), "lengths": lengths, "positions": _i32(5), "slots": _i32(5)}
    batch = ops.PagedBatch(**fields, page_size=16)
    assert (batch.requests, batch.rows, batch.cols, batch.max_new, batch.min_new) == (3, 5, 4, 5, 0)
    for name, bad in (("starts", _i32(3)), ("counts", _i32(4)), ("lengths", lengths.float()), ("slots", _i32(6)), ("positions", _i32(10)[::2]),
                      ("taken", _i32(2)), ("page table", None)):
        with pytest.raises(ValueError, match=name):
            if bad is None:
                ops.PagedBatch(**dict(fields, table=_i32(12)), page_size=16)
            else:
                ops.PagedBatch(**dict(fields, **{name: bad}), page_size=16)
    bf = torch.bfloat16
    k, v, q = torch.zeros(9, 2, 16, 32, dtype=bf), torch.zeros(9, 2, 32, 16, dtype=bf), torch.zeros(5, 4, 32, dtype=bf)

    def attention(q=q, k=k, v=v, batch=batch, **kw):
        return ops.paged_attention(q, k, v, batch, **kw)

    for match, kw in (("GPU tensor", {}), ("head size", {"q": q[0]}), ("rows", {"q": q[:4]}), ("key-value heads", {"q": q[:, :3]}),
                      ("the rows are", {"q": q.half()}), ("the cache holds", {"v": v.half()}), ("page size", {"v": k}), ("page size", {"k": k[0]}),
                      ("pages of 32", {"batch": ops.PagedBatch(**fields, page_size=32)}), ("negative", {"window": -1}),
                      ("negative", {"sinks": -2}), ("contiguous", {"k": torch.zeros(9, 2, 32, 32, dtype=bf)[:, :, ::2]})):
        with pytest.raises(ValueError, match=match):
            attention(**kw)
    qkv, norm = torch.zeros(5, 8 * 32, dtype=bf), torch.ones(32, dtype=bf)
    turns = torch.zeros(64, 16)

    def fill(qkv=qkv, k=k, v=v, batch=batch, heads=4, q_norm=norm, k_norm=norm, rope=(turns, turns)):
        return ops.qkv_to_cache(qkv, k, v, batch, heads, q_norm, k_norm, 1e-6, rope)

    for match, kw in (("GPU tensor", {}), ("rows", {"qkv": qkv[:3]}), ("rows", {"heads": 5}), ("norm weight", {"k_norm": norm[:16]}),
                      ("rope", {"rope": (turns[:63], turns[:63])}), ("rope", {"rope": (turns, turns[:, :8])}), ("rope", {"rope": (turns.double(), turns)}),
                      ("rope", {"rope": (turns, torch.zeros(65, 16))}), ("the rows are", {"qkv": qkv.half()})):
        with pytest.raises(ValueError, match=match):
            fill(**kw)


# ---- the cache's host side ----------------------------------------------------------------------------


def _cache(**kw):
    args = {"layers": 1, "requests": 3, "pages": 10, "heads": 4, "kv_heads": 2, "head_dim": 32, "page_size": 16, "max_rows": 20,
            "device": "cpu"}
    return PagedCache(**dict(args, **kw))


def test_cache_sizes():
    c = _cache(max_length=40, rope_theta=1e4)
    assert c.table.shape == (3, 3) and c.rope[0].shape == (48, 16) and c.free.tolist() == list(range(10))
    assert c.k[0].shape == (10, 2, 16, 32) and c.v[0].shape == (10, 2, 32, 16)
    assert _cache().table.shape == (3, 10)
    for bad in ({"layers": 0}, {"requests": 0}, {"pages": 0}, {"heads": 3}, {"heads": 1}, {"max_rows": 0}, {"requests": 2049},
                {"dtype": torch.float32}, {"max_length": 0}):
        with pytest.raises(ValueError):
            _cache(**bad)


def test_cache_refuses_steps():
    c = _cache()
    for match, args in (("up to 3 entries", ([1] * 4,)), ("1-D", (torch.zeros(1, 2, dtype=torch.int64),)), ("whole numbers", ([1.0],)),
                        ("whole numbers", ([True],)), ("negative", ([1, -1],)), ("do not fit", ([5, 6], 10)), ("max_new", ([5, 6], 12, 5)),
                        ("min_new", ([5, 1], 12, 5, 2)), ("rows in a cache", ([15, 6],)), ("rows in a cache", ([1], 21)),
                        ("do not fit", ([], -1))):
        with pytest.raises(ValueError, match=match):
            c.step(*args)
    with pytest.raises(ValueError, match="no rows"):
        c.batch_for(1)
    for bad in ([3], [-1], [0.5], [[0]]):
        with pytest.raises(ValueError):
            c.release(bad)
    with pytest.raises(ValueError, match="GPU tensor"):  # past the checks: no CPU path
        c.step([1, 2])
    assert c.batch is None


def test_fakes():
    with FakeTensorMode():
        bf = torch.bfloat16
        k, v = torch.empty(9, 2, 16, 32, dtype=bf, device="cuda"), torch.empty(9, 2, 32, 16, dtype=bf, device="cuda")
        i32 = lambda *s: torch.empty(*s, dtype=torch.int32, device="cuda")  # noqa: E731
        state = [i32(3, 4), i32(4), i32(3), i32(3), i32(5), i32(5)]
        q = torch.ops.qtts.qkv_to_cache(torch.empty(5, 256, dtype=bf, device="cuda"), k, v, state, [16, 5, 0], 4, None, None, 1e-6, None, None)
        assert q.shape == (5, 4, 32) and q.dtype == bf
        assert torch.ops.qtts.paged_attention(q, k, v, state, [16, 5, 0], 0, 0, 0.1).shape == (5, 4, 32)
