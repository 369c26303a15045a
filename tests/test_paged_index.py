"""The paged cache's index arithmetic (csrc/paged.h), compiled for the host and swept.

The kernels index with nothing else, so what holds here -- every result inside
its bounds whatever the device arrays hold, every token in exactly one tile --
is what keeps bad tables, positions and cu from being followed.
"""

from __future__ import annotations

import ctypes
import os
import subprocess

import numpy as np
import pytest

from tests.paged_ref import key_range

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SHIM = r"""
#include "%s"
using namespace altxs_paged;
extern "C" {
unsigned t_div(unsigned n, unsigned d) { return div_by(n, fast_div(d)); }
long long t_first(long long start, int g, int br, long long b) { return first_slot(start, g, br, b); }
long long t_slots(long long T, int g, int br, long long B) { return slot_count(T, g, br, B); }
void t_segment(int c0, int c1, int pos, long long T, int cap, int* out) {
  Segment s = segment_of(c0, c1, pos, T, cap);
  out[0] = s.t0; out[1] = s.n; out[2] = s.pos; out[3] = s.ok;
}
void t_range(int p, int len, int window, int start, int prefix, int* out) {
  Range r = keys_seen(p, len, window, start, prefix);
  out[0] = r.lo; out[1] = r.hi;
}
int t_page(const int* row, int width, int shift, long long n_pages, int t) { return page_of(row, width, shift, n_pages, t); }
// the block that block_with_first() ends with, when a wave's ballots are `later`
void t_block(int B, const unsigned char* later, int* out) {
  Block b = {0, B};
  out[2] = 0;
  while (b.n > 64) {
    unsigned long long m = 0;
    for (int l = 0; l < 64; ++l) m |= (unsigned long long)later[part_end(b, l)] << l;
    b = part_of(b, m);
    ++out[2];
  }
  out[0] = b.lo; out[1] = b.n;
}
int t_part(int n, unsigned long long bits, int lane, int* out) {
  const Block b = part_of(Block{0, n}, bits);
  out[0] = b.lo; out[1] = b.n;
  return part_end(Block{0, n}, lane);
}
}
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("paged")
    src = d / "shim.cpp"
    src.write_text(SHIM % os.path.join(ROOT, "altxs_amd", "csrc", "paged.h"))
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-shared", "-fPIC",
                    str(src), "-o", str(d / "shim.so")], check=True)
    L = ctypes.CDLL(str(d / "shim.so"))
    L.t_first.restype = L.t_slots.restype = ctypes.c_longlong
    L.t_first.argtypes = [ctypes.c_longlong, ctypes.c_int, ctypes.c_int, ctypes.c_longlong]
    L.t_slots.argtypes = [ctypes.c_longlong, ctypes.c_int, ctypes.c_int, ctypes.c_longlong]
    L.t_segment.argtypes = [ctypes.c_int] * 3 + [ctypes.c_longlong, ctypes.c_int, ctypes.POINTER(ctypes.c_int)]
    L.t_page.argtypes = [ctypes.POINTER(ctypes.c_int), ctypes.c_int, ctypes.c_int, ctypes.c_longlong, ctypes.c_int]
    L.t_div.restype = ctypes.c_uint
    L.t_div.argtypes = [ctypes.c_uint, ctypes.c_uint]
    return L


def test_division(lib):
    r = np.random.RandomState(0)
    for d in [1, 2, 3, 5, 7, 12, 15, 24, 64, 100, 1000, 65537, (1 << 31) - 1] + r.randint(1, 1 << 20, 30).tolist():
        ns = np.concatenate([np.arange(0, 70), r.randint(0, (1 << 31) - 1, 200), [(1 << 31) - 1]])
        ns = np.concatenate([ns, ns // d * d, np.maximum(ns // d * d - 1, 0)])
        for n in ns.tolist():
            assert lib.t_div(n, d) == n // d, (n, d)


@pytest.mark.parametrize("g,br", [(1, 16), (2, 16), (8, 16), (3, 128), (1, 128), (16, 128), (64, 16)])
def test_slots_cover_every_row_once(lib, g, br):
    r = np.random.RandomState(g * 1000 + br)
    for _ in range(30):
        B = int(r.randint(1, 12))
        lens = r.randint(0, 90, B) * (r.rand(B) > 0.3)
        cu = np.concatenate([[0], np.cumsum(lens)])
        T = int(cu[-1] + r.randint(0, 5))  # rows behind the last segment
        first = [lib.t_first(int(c), g, br, b) for b, c in enumerate(cu)]
        assert first[0] == 0 and all(a < b for a, b in zip(first, first[1:]))
        assert first[-1] <= lib.t_slots(T, g, br, B)
        for b in range(B):
            assert first[b + 1] - first[b] >= -(-int(lens[b]) * g // br)


@pytest.mark.parametrize("B", [1, 2, 63, 64, 65, 127, 128, 129, 200, 4095, 4096, 4097, 10000, 300000])
def test_search_finds_the_first(lib, B):
    r = np.random.RandomState(B)
    out = (ctypes.c_int * 3)()
    for first in sorted({0, 1, 63, 64, 65, B // 2, B - 2, B - 1, *r.randint(0, B, 20).tolist()}):
        if not 0 <= first < B:
            continue
        later = (np.arange(B) >= first).astype(np.uint8)
        lib.t_block(B, later.ctypes.data_as(ctypes.c_char_p), out)
        assert 1 <= out[1] <= 64 and 0 <= out[0] <= first < out[0] + out[1] <= B
        assert 64 ** (out[2] + 1) < 64 * B + 64 * 64
    for later in (np.zeros(B, np.uint8), (r.rand(B) > 0.5).astype(np.uint8)):  # nobody; no order at all
        lib.t_block(B, later.ctypes.data_as(ctypes.c_char_p), out)
        assert 1 <= out[1] <= 64 and 0 <= out[0] and out[0] + out[1] <= B
    for n in (65, B + 64, (1 << 31) - 1):
        for lane in (0, 1, 62, 63):
            end = lib.t_part(n, ctypes.c_ulonglong(1 << lane), lane, out)
            assert 0 <= end < n
            if lane * ((n - 1) // 64 + 1) < n:
                assert out[0] + out[1] - 1 == end and out[1] >= 1


def test_segments_stay_in_bounds(lib):
    r = np.random.RandomState(1)
    out = (ctypes.c_int * 4)()
    lim = (1 << 31) - 1
    for _ in range(4000):
        T, cap = int(r.randint(0, 200)), int(r.choice([0, 1, 64, 1000, lim]))
        c0, c1, pos = (int(r.choice([r.randint(-5, 210), -lim - 1, lim, 0])) for _ in range(3))
        lib.t_segment(c0, c1, pos, T, cap, out)
        t0, n, p, ok = out[:]
        assert 0 <= t0 <= T and 0 <= n <= T - t0
        good = 0 <= c0 <= c1 <= T and pos >= 0 and pos + c1 - c0 <= cap
        assert ok == int(good)
        if good:
            assert (t0, n, p) == (c0, c1 - c0, pos)


def test_ranges(lib):
    r = np.random.RandomState(2)
    out = (ctypes.c_int * 2)()
    lim = (1 << 31) - 1
    for _ in range(4000):
        length = int(r.choice([1, 5, 64, 1000, lim]))
        p = int(r.randint(0, min(length, 1 << 30)))
        window = int(r.choice([0, 1, 7, 100, lim]))
        start = int(r.choice([0, -3, p, p + 1, r.randint(0, 1 << 20), lim, -lim - 1]))
        prefix = int(r.choice([0, -1, 3, p + 2, length, lim, -lim - 1]))
        lib.t_range(p, length, window, start, prefix, out)
        assert tuple(out[:]) == key_range(p, length, window, start, prefix)
        assert 0 <= out[0] <= out[1] <= length


def test_pages(lib):
    row = (ctypes.c_int * 4)(3, -1, 9, 10)
    for shift in (4, 6):
        for t in (-1, 0, 15, 16, 47, 63, 64, 130, 200, 255, 256, 1 << 30, (1 << 31) - 1, -(1 << 31)):
            want = -1
            if t >= 0 and (t >> shift) < 4:
                want = [3, -1, 9, 10][t >> shift]
                want = want if 0 <= want < 10 else -1
            assert lib.t_page(row, 4, shift, 10, t) == want
    assert lib.t_page(row, 0, 4, 10, 0) == -1 and lib.t_page(row, 4, 4, 0, 0) == -1
