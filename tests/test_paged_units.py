"""Host functions of the paged operators' sources, compiled by themselves and called without a GPU."""
import ctypes
import os
import random
import subprocess

import pytest

from conftest import REPO
from fftsparse_b200 import build

SOURCE = r"""
#include "paged_common.cuh"

namespace ffts { void set_error(int, const char *, ...) {} }

extern "C" int unit_rows_apart(const long long *sizes, const long long *strides, int n, long long inner) {
  int64_t a[3], b[3];
  for (int i = 0; i < n; ++i) { a[i] = sizes[i]; b[i] = strides[i]; }
  return ffts::rows_apart(a, b, n, inner);
}

using namespace ffts::paged;

// q tiles (tok0, pos0, ntok) of the batch as build_schedule lays them out; every share's segments, nine numbers each:
// share, q tile, head, j0, j1, key tiles, opens, the share that ends it, turn.  Returns how many there are.
template <int BN>
static long long walk(const long long *tiles, int n, int Hkv, int window, int sinks, int ctas, int overhead,
                      long long *out, long long room) {
  Params p{};
  p.Hkv = Hkv;
  p.window = window;
  p.sinks = sinks;
  p.ctas = ctas;
  p.overhead = overhead;
  p.max_tiles = n;
  Tile *t = new Tile[n];
  long long *cum = new long long[n + 1], found = 0;
  cum[0] = 0;
  for (int i = 0; i < n; ++i) {
    t[i] = Tile{int(tiles[3 * i]), int(tiles[3 * i + 1]), int(tiles[3 * i + 2]), 0};
    cum[i + 1] = cum[i] + keys_of<BN>(t[i].pos0, t[i].ntok, window, sinks).n + overhead;
  }
  const long long length = cum[n] * Hkv, per = share_of(p, length);
  for (int c = 0, at = 0; c < ctas; ++c) {
    const long long u0 = per * c, u1 = u0 + per < length ? u0 + per : length;
    if (u0 >= u1) break;
    while (cum[at + 1] * Hkv <= u0) ++at;
    Walk<BN> w(p, t, cum);
    w.start(u0, u1, at);
    while (w.segment()) {
      if (found == room) return -1;
      const long long row[9] = {c, w.x, w.h, w.j0, w.j1, w.g.n, w.opens, w.last_share(u0, per), w.turn};
      for (int i = 0; i < 9; ++i) out[9 * found + i] = row[i];
      ++found;
    }
  }
  delete[] t;
  delete[] cum;
  return found;
}

extern "C" long long unit_walk(int bn, const long long *tiles, int n, int Hkv, int window, int sinks, int ctas, int overhead,
                               long long *out, long long room) {
  return bn == 64 ? walk<64>(tiles, n, Hkv, window, sinks, ctas, overhead, out, room)
                  : walk<128>(tiles, n, Hkv, window, sinks, ctas, overhead, out, room);
}

// Whether keys [c0, c0 + bn) hold some that no row sees (bit 0), and some that rows may differ in (bit 1).
extern "C" int unit_differ(int bn, int pos0, int ntok, int window, int sinks, int c0) {
  return bn == 64 ? has_unseen<64>(keys_of<64>(pos0, ntok, window, sinks), sinks, c0) +
                        2 * rows_differ<64>(pos0, ntok, window, sinks, c0)
                  : has_unseen<128>(keys_of<128>(pos0, ntok, window, sinks), sinks, c0) +
                        2 * rows_differ<128>(pos0, ntok, window, sinks, c0);
}

// The key tiles of a q tile in the order in which a whole one with this turn visits them; *bounds its hi, lo.
extern "C" int unit_keys(int bn, int pos0, int ntok, int window, int sinks, int turn, int *out, int *bounds) {
  Params p{};
  Walk<64> a(p, nullptr, nullptr);
  Walk<128> b(p, nullptr, nullptr);
  a.g = keys_of<64>(pos0, ntok, window, sinks);
  b.g = keys_of<128>(pos0, ntok, window, sinks);
  const Keys g = bn == 64 ? a.g : b.g;
  a.j1 = b.j1 = g.n;
  a.turn = b.turn = turn;
  for (int j = 0; j < g.n; ++j) out[j] = bn == 64 ? a.key(j) : b.key(j);
  bounds[0] = g.hi;
  bounds[1] = g.lo;
  return g.n;
}
"""


@pytest.fixture(scope="module")
def units(tmp_path_factory):
    d = tmp_path_factory.mktemp("units")
    src, lib = d / "units.cu", d / "units.so"
    src.write_text(SOURCE)
    flags = [f for f in build.NVCC_FLAGS if f not in ("-Xcompiler", "-fvisibility=hidden", "-fPIC", "-O3")]
    subprocess.run([build.nvcc(), *flags, "-O1", "-Xcompiler", "-fPIC", "-shared", "-I", build.INCLUDE, "-I", build.CSRC,
                    str(src), "-o", str(lib)], check=True, cwd=REPO)
    return ctypes.CDLL(os.fspath(lib))


def longs(values):
    return (ctypes.c_longlong * len(values))(*values)


# ------------------------------------------------------------------ rows of a written tensor
def apart(units, sizes, strides, inner):
    return bool(units.unit_rows_apart(longs(sizes), longs(strides), len(sizes), ctypes.c_longlong(inner)))


@pytest.mark.parametrize("sizes,strides,inner,want", [
    ((3, 4), (256, 64), 64, True), ((3, 4), (64, 192), 64, True), ((3, 4), (72, 288), 64, True),
    ((3, 4), (0, 64), 64, False), ((1, 4), (0, 64), 64, True), ((3, 4), (256, 0), 64, False), ((3, 1), (64, 0), 64, True),
    ((3, 4), (248, 64), 64, False), ((3, 4), (256, 56), 64, False), ((1, 1), (0, 0), 64, True), ((0, 4), (0, 64), 64, True),
    ((2, 2, 16), (2048, 1024, 64), 64, True), ((2, 2, 16), (2048, 64, 128), 64, True), ((2, 2, 16), (1024, 1024, 64), 64, False),
    ((2, 2, 16), (2048, 0, 128), 64, False), ((2, 2, 16), (0, 64, 128), 64, False),
    ((40000, 8, 64), (65536, 8192, 128), 128, True), ((1 << 30, 8, 2), (2048, 256, 128), 128, True)])
def test_rows_apart(units, sizes, strides, inner, want):
    assert apart(units, sizes, strides, inner) is want


def test_rows_apart_never_passes_rows_that_overlap(units):
    rng = random.Random(1)
    passed = 0
    for _ in range(20000):
        sizes = [rng.randrange(1, 4) for _ in range(3)]
        strides = [rng.randrange(0, 20) for _ in range(3)]
        inner = rng.randrange(1, 4)
        if apart(units, sizes, strides, inner):
            seen = [i * strides[0] + j * strides[1] + k * strides[2] + e for i in range(sizes[0]) for j in range(sizes[1])
                    for k in range(sizes[2]) for e in range(inner)]
            assert len(set(seen)) == len(seen), (sizes, strides, inner)
            passed += 1
    assert passed > 1000


# ------------------------------------------------------------------ shares of the attention's line
OVERHEAD = 3


def walk(units, bn, tiles, Hkv, window, sinks, ctas, room=200000):
    out = (ctypes.c_longlong * (9 * room))()
    flat = longs([x for t in tiles for x in t])
    units.unit_walk.restype = ctypes.c_longlong
    n = units.unit_walk(bn, flat, len(tiles), Hkv, window, sinks, ctas, OVERHEAD, out, ctypes.c_longlong(room))
    assert n >= 0
    return [tuple(out[9 * i:9 * i + 9]) for i in range(n)]


def keys(units, bn, pos0, ntok, window, sinks, turn=0):
    out, bounds = (ctypes.c_int * (max(0, pos0 + ntok) // bn + 2))(), (ctypes.c_int * 2)()
    n = units.unit_keys(bn, pos0, ntok, window, sinks, turn, out, bounds)
    return list(out[:n]), bounds[0], bounds[1]


@pytest.mark.parametrize("bm,bn", [(128, 64), (256, 128)])
@pytest.mark.parametrize("seed", range(25))
def test_shares_hold_every_key_tile_once_and_cuts_name_their_shares(units, bm, bn, seed):
    """Every key that a token sees lies in one visited tile; every (q tile, head)'s tiles lie in one share or in
    neighbouring ones, of which the first knows the last; at most a share's first and last pieces are cut."""
    rng = random.Random(seed)
    G = rng.choice([1, 2, 4, 7, 8, 16, 128])
    Hkv, ctas = rng.choice([1, 2, 8]), rng.choice([1, 3, 8, 148, 296])
    window = rng.choice([0, 0, 1, 50, 700])
    sinks = rng.choice([0, 4, 130]) if window else 0
    tpt, tiles, tok = bm // 128 * (128 // G), [], 0
    for _ in range(rng.randrange(1, 12)):
        n = rng.choice([0, 1, 1, rng.randrange(1, 300)])
        kv = rng.choice([0, n, n + rng.randrange(0, 3000), rng.randrange(0, n + 1)])
        tiles += [(tok + i, kv - n + i, min(tpt, n - i)) for i in range(0, n, tpt)]
        tok += n
    if not tiles:
        return
    size = []
    for _, pos0, ntok in tiles:
        visited, hi, lo = keys(units, bn, pos0, ntok, window, sinks)
        size.append(len(visited))
        for turn in {0, 1 % len(visited), len(visited) - 1, rng.randrange(len(visited))}:
            turned = keys(units, bn, pos0, ntok, window, sinks, turn)[0]
            assert turned == visited[turn:] + visited[:turn] and len(set(visited)) == len(visited)
        for pos in range(max(0, pos0), pos0 + ntok):
            seen = [c for c in range(pos + 1) if not window or c > pos - window or c < sinks]
            assert {c // bn for c in seen} <= set(visited)
            assert all(c < hi and (c >= lo or c < sinks) for c in seen)
    segments = walk(units, bn, tiles, Hkv, window, sinks, ctas)
    parts, inside = {}, {}
    for c, x, h, j0, j1, n, opens, last, turn in segments:
        assert n == size[x] and 0 <= j0 < j1 <= n and (turn == 0 or (j0, j1) == (0, n)) and 0 <= turn < n
        parts.setdefault((x, h), []).append((c, j0, j1, opens, last))
        inside.setdefault(c, []).append((x, h, j1 - j0 == n))
    assert set(parts) == {(x, h) for x in range(len(tiles)) for h in range(Hkv)}
    for (x, h), ps in parts.items():
        at = size[x]  # the first share has the last key tiles
        for i, (c, j0, j1, opens, last) in enumerate(ps):
            assert j1 == at and c == ps[0][0] + i and bool(opens) == (i == 0)
            assert last == ps[-1][0] or not opens
            at = j0
        assert at == 0
    for c, ss in inside.items():
        assert all(whole for _, _, whole in ss[1:-1])  # the join looks in a share's first and last pieces only


def test_lines_longer_than_31_bits(units):
    """A share may be longer than 2^31 key tiles (requests that share pages), and so may what lies before it."""
    for ctas, heads, n in ((1, 8, 40), (3, 8, 200), (2, 16, 300)):
        tiles = [(i, (1 << 30) - 2, 1) for i in range(n)]
        per_head = (1 << 30) // 64
        assert n * heads * (per_head + OVERHEAD) // ctas > 2 ** 31
        segments = walk(units, 64, tiles, heads, 0, 0, ctas)
        total = {}
        for c, x, h, j0, j1, size, opens, last, turn in segments:
            assert size == per_head and 0 <= turn < size and c <= last < ctas
            total[x, h] = total.get((x, h), 0) + j1 - j0
        assert total == {(x, h): per_head for x in range(n) for h in range(heads)}
        for c in range(ctas):  # equal shares
            got = sum(j1 - j0 for s, _, _, j0, j1, *_ in segments if s == c)
            assert abs(got - n * heads * per_head // ctas) <= n * heads * OVERHEAD


@pytest.mark.parametrize("bn", [64, 128])
def test_tiles_whose_values_need_care(units, bn):
    """A visited tile with a key that no row sees, or one that some rows see and others do not, is known as such."""
    rng = random.Random(bn)
    for _ in range(1500):
        window = rng.choice([0, 0, 1, 3, 64, 100, 400])
        sinks = rng.choice([0, 4, 64, 130]) if window else 0
        pos0, ntok = rng.randrange(-20, 700), rng.choice([1, 2, 18, 32, 128, 256])
        rows = [{c for c in range(max(0, p + 1)) if not window or c > p - window or c < sinks} for p in range(pos0, pos0 + ntok)]
        some, every = set.union(*rows), set.intersection(*rows)
        for tile in keys(units, bn, pos0, ntok, window, sinks)[0]:
            c0 = tile * bn
            here = set(range(c0, c0 + bn))
            flags = units.unit_differ(bn, pos0, ntok, window, sinks, c0)
            if here - some:
                assert flags & 1, (pos0, ntok, window, sinks, c0)
            if here & some - every:
                assert flags & 2, (pos0, ntok, window, sinks, c0)
            if ntok == 1:
                assert not flags & 2  # decoding rows share what they see
