"""Which pieces of a cache the new rows of a decode step read (csrc/piece_range.h),
compiled for the host, against the mask's definition."""
import ctypes
import os
import random
import shutil
import subprocess

import numpy as np
import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                    "tagseq2tagseq_amd", "csrc")
SOURCE = """
#include "piece_range.h"
template <int kPiece>
static int pieces(const int32_t* pos, const int32_t* start, int rows, int keys, int window,
                  int sinks, int32_t* out) {
  const t2t::PieceRange<kPiece> r(pos, start, rows, keys, window, sinks);
  for (int i = 0; i < r.count; ++i) out[i] = r.at(i);
  return r.count;
}
extern "C" int pieces64(const int32_t* p, const int32_t* s, int r, int k, int w, int n, int32_t* o) {
  return pieces<64>(p, s, r, k, w, n, o);
}
extern "C" int pieces256(const int32_t* p, const int32_t* s, int r, int k, int w, int n, int32_t* o) {
  return pieces<256>(p, s, r, k, w, n, o);
}
"""


@pytest.fixture(scope="module")
def pieces(tmp_path_factory):
    d = tmp_path_factory.mktemp("piece_range")
    src, lib = d / "pieces.cpp", d / "pieces.so"
    src.write_text(SOURCE)
    subprocess.run([shutil.which("g++") or "c++", "-std=c++17", "-O1", "-fsanitize=undefined",
                    "-fno-sanitize-recover=all", "-shared", "-fPIC", f"-I{CSRC}", str(src), "-o",
                    str(lib)], check=True)
    L = ctypes.CDLL(str(lib))

    def call(size, pos, start, keys, window, sinks):
        p, s = np.asarray(pos, np.int32), np.asarray(start, np.int32)
        out = np.full(-(-keys // size) + 1, -1, np.int32)
        # as the launchers have it: no starts without sinks
        n = getattr(L, f"pieces{size}")(p.ctypes.data_as(ctypes.c_void_p),
                                        s.ctypes.data_as(ctypes.c_void_p) if sinks else None,
                                        len(p), keys, window, sinks,
                                        out.ctypes.data_as(ctypes.c_void_p))
        return out[:n].tolist()
    return call


def _read(size, pos, start, keys, window, sinks):
    """Pieces with a key that some row may read."""
    j = np.arange(keys, dtype=np.int64)
    ok = np.zeros(keys, bool)
    for p, s in zip(pos, start):
        near = p - j < window if window else np.ones(keys, bool)
        ok |= (j <= p) & (near | ((j >= s) & (j - s < sinks)))
    return set((j[ok] // size).tolist())


def _check(pieces, size, pos, start, keys, window, sinks):
    got = pieces(size, pos, start, keys, window, sinks)
    what = f"{size} {pos} {start} of {keys}, window {window}, {sinks} sinks: {got}"
    assert len(set(got)) == len(got) <= -(-keys // size), what
    assert all(0 <= x < -(-keys // size) for x in got), what
    assert _read(size, pos, start, keys, window, sinks) <= set(got), what
    return got


@pytest.mark.parametrize("size", [64, 256])
def test_rows_past_the_cache_keep_their_sinks(pieces, size):
    """Their windows hold no key of the cache, their sinks may lie behind the
    windows of the other rows."""
    for pos, start, keys, window, sinks in [
            ((100, 5200), (0, 4300), 5000, 40, 4), ((10, 10000), (0, 4000), 5000, 4, 4),
            ((5200, 100), (4300, 0), 5000, 40, 4), ((10000, 10), (4000, 0), 5000, 4, 300),
            ((3, 9, 2 ** 31 - 1), (0, 0, 2000), 2100, 1, 2 ** 31 - 1)]:
        _check(pieces, size, pos, start, keys, window, sinks)
        for p, s in zip(pos, start):
            _check(pieces, size, (p,), (s,), keys, window, sinks)


@pytest.mark.parametrize("size", [64, 256])
def test_neighbours_read_their_windows_and_sinks_alone(pieces, size):
    got = pieces(size, (30000, 30001), (9000, 9000), 32768, 700, 4)
    assert set(got) == _read(size, (30000, 30001), (9000, 9000), 32768, 700, 4)
    assert pieces(size, (5,), (0,), 0, 3, 2) == [] and pieces(size, (-1,), (0,), 90, 3, 2) == []


def test_any_rows(pieces):
    rng = random.Random(0)
    for _ in range(4000):
        keys = rng.choice([1, 63, 64, 700, 5000])
        n = rng.randrange(1, 9)
        far = rng.choice([keys, keys, 2 * keys + 50])  # (a third of them past the cache too)
        pos = [rng.randrange(-2, far) for _ in range(n)]
        start = [rng.randrange(0, max(1, p + 1)) if rng.random() < 0.9 else rng.randrange(-5, far)
                 for p in pos]
        window = rng.choice([0, 1, 4, 40, 300, 2 * keys])
        sinks = rng.choice([0, 1, 4, 200])
        for size in (64, 256):
            _check(pieces, size, pos, start, keys, window, sinks)
