"""Host: the chunk attention's division of a call into segments (``csrc/chunk_walk.cuh``), compiled for the host.

A warp is 32 calls of each warp function, one lane after the other: an order that independent thread scheduling allows, and
under which a walk that more than one lane moves goes wrong."""

from __future__ import annotations

import ctypes
import subprocess
from pathlib import Path

import numpy as np
import pytest

CSRC = Path(__file__).resolve().parents[1] / "unlimited-ocr-max_b200" / "csrc"
CUDA = Path("/usr/local/cuda/include")

CODE = r"""
#include <algorithm>
#include <stdint.h>
using std::max;
using std::min;
#define UOCR_DEV inline
template <typename T> inline T __ldg(const T* p) { return *p; }
static struct { unsigned x; } lane_id;
#define threadIdx lane_id
inline void __syncwarp() {}
static int from_lane_0;
inline int __shfl_sync(unsigned, int v, int) {
    if (threadIdx.x == 0) from_lane_0 = v;
    return from_lane_0;
}
#include "chunk_walk.cuh"
using namespace uocr;

static ChunkArgs args(int T, int B, int g, int kv, int cols, int window, const int32_t* off, const int32_t* start, const int32_t* prefix) {
    ChunkArgs a{};
    a.T = T, a.B = B, a.heads = g * kv, a.kv_heads = kv, a.pass_heads = kv, a.lut_cols = cols, a.window = window;
    a.offsets = off, a.start = start, a.prefix = prefix;
    a.group_shift = 32;
    while (g >> (a.group_shift - 31)) ++a.group_shift;
    a.group_mul = ((1ull << a.group_shift) + g - 1) / g;
    return a;
}

// Segments of all CTAs in their order: (CTA, request, tile, head, first page of the tile's, pages); -1: lanes disagree.
extern "C" int segments(int T, int B, int g, int kv, int cols, int window, const int32_t* off, const int32_t* start,
                        const int32_t* prefix, int tile, int lead, int ctas, int* out, int most) {
    const ChunkArgs a = args(T, B, g, kv, cols, window, off, start, prefix);
    uint32_t total = 0;
    for (int b = 0; b < B; ++b) {
        const Request r = request_at(a, b);
        for (int qt = 0; qt * tile < r.n * g; ++qt) total += (tile_at(a, r, qt, tile).count + lead) * kv;
    }
    ctas = std::min<uint32_t>(ctas, total);
    int found = 0;
    for (int c = 0; c < ctas; ++c) {
        const uint32_t each = total / ctas, rest = total - each * ctas;
        const uint32_t u0 = each * c + std::min<uint32_t>(c, rest), u1 = u0 + each + ((uint32_t)c < rest ? 1 : 0);
        Run run{};
        uint32_t before = 0;
        for (int b = 0; b < B; ++b) {  // where unit u0 lies
            const Request r = request_at(a, b);
            for (int qt = 0; qt * tile < r.n * g; ++qt) {
                const uint32_t count = tile_at(a, r, qt, tile).count + lead;
                if (u0 >= before && u0 < before + count * kv) {
                    Walk w{};
                    w.left = u1 - u0, w.b = b, w.qt = qt, w.head = (u0 - before) / count, w.r = r, w.tiles = (r.n * g + tile - 1) / tile;
                    run.some = w.enter(a, tile, lead, (u0 - before) % count);
                    run.first = w;
                }
                before += count * kv;
            }
        }
        Walk w{};
        for (bool begin = true;; begin = false) {
            bool more = false;
            for (threadIdx.x = 0; threadIdx.x < 32; ++threadIdx.x) {
                const bool mine = begin ? warp_first(w, run) : warp_next(w, a, g, tile, lead);
                if (threadIdx.x && mine != more) return -1;
                more = mine;
            }
            if (!more) break;
            if (found == most) return -2;
            const int v[] = {c, w.b, w.qt, w.head, w.j, w.n};
            std::copy(v, v + 6, out + 6 * found++);
        }
    }
    return found;
}

extern "C" void tile_pages(int T, int B, int g, int kv, int cols, int window, const int32_t* off, const int32_t* start,
                           const int32_t* prefix, int tile, int b, int qt, int* count, int* pages) {
    const ChunkArgs a = args(T, B, g, kv, cols, window, off, start, prefix);
    const Tile t = tile_at(a, request_at(a, b), qt, tile);
    *count = t.count;
    for (int j = 0; j < t.count; ++j) pages[j] = t.page(j);
}

extern "C" void request(int T, int B, int cols, const int32_t* off, const int32_t* start, const int32_t* prefix, int b, int* out) {
    const Request r = request_at(args(T, B, 1, 1, cols, 0, off, start, prefix), b);
    out[0] = r.lo, out[1] = r.n, out[2] = r.start, out[3] = r.prefix;
}
"""


@pytest.fixture(scope="module")
def walk(tmp_path_factory):
    d = tmp_path_factory.mktemp("walk")
    (d / "walk.cpp").write_text(CODE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-fwrapv", "-w", "-shared", "-fPIC", "-I", str(CSRC), "-I", str(CUDA), str(d / "walk.cpp"),
                    "-o", str(d / "walk.so")], check=True)
    return ctypes.CDLL(str(d / "walk.so"))


def _i32(v):
    return None if v is None else (ctypes.c_int32 * len(v))(*v)


@pytest.mark.parametrize("n,start,g,kv,window,prefix,tile,lead,ctas", [
    ([300, 1, 0, 77], [517, 640, 3, 0], 1, 10, 0, None, 128, 3, 148), ([700] * 3, [1500, 0, 200], 4, 2, 128, [512, 0, 90], 128, 3, 148),
    ([5, 1, 0, 3], [250, 0, 40, 126], 1, 2, 0, None, 3, 1, 148), ([1] * 40, [37 * i for i in range(40)], 1, 3, 0, None, 1, 1, 7),
    ([2, 257, 0, 64, 31], [383, 0, 5, 129, 1000], 7, 1, 1, [0] * 5, 128, 3, 20), ([9, 30], [2500, 100], 3, 5, 40, [300, 10 ** 9], 8, 1, 1),
    ([0, 0, 4], [5, 5, 900], 3, 3, 2 ** 31 - 1, [1, 1, 2 ** 31 - 1], 6, 1, 148),
])
def test_every_page_of_every_tile_once(walk, n, start, g, kv, window, prefix, tile, lead, ctas):
    off = [sum(n[:b]) for b in range(len(n) + 1)]
    cols = max((a + b + 127) // 128 for a, b in zip(n, start)) + 1
    call = (off[-1], len(n), g, kv, cols, window, _i32(off), _i32(start), _i32(prefix))
    out = (ctypes.c_int * 600000)()
    found = walk.segments(*call, tile, lead, ctas, out, 100000)
    assert found > 0
    segments = np.asarray(out[: 6 * found]).reshape(-1, 6).tolist()
    want = []  # (request, tile, head, page of the tile's) in order
    for b in range(len(n)):
        for qt in range(-(-n[b] * g // tile)):
            count, pages = ctypes.c_int(), (ctypes.c_int * (cols + 1))()
            walk.tile_pages(*call, tile, b, qt, ctypes.byref(count), pages)
            mine = pages[: count.value]
            assert sorted(set(mine)) == mine  # ascending, none twice
            for token in range(qt * tile // g, min(n[b], -(-(qt + 1) * tile // g))):
                p = start[b] + token
                seen = set(range(max(0, p - window + 1) // 128 if window else 0, p // 128 + 1))
                if window and prefix and prefix[b]:
                    seen |= set(range((min(prefix[b], p + 1) - 1) // 128 + 1))
                assert seen <= set(mine)
            want += [(b, qt, h, j) for h in range(kv) for j in range(count.value)]
    assert [(b, qt, h, j + i) for _, b, qt, h, j, k in segments for i in range(k)] == want
    assert [s[0] for s in segments] == sorted(s[0] for s in segments)


def test_requests_stay_inside_whatever_the_lengths_say(walk):
    low, high = -2 ** 31, 2 ** 31 - 1
    odd = [low, low + 1, -7, -1, 0, 1, 5, 99, 100, 101, 640, high - 1, high]
    out = (ctypes.c_int * 4)()
    for a in odd:
        for b in odd:
            for s in odd:
                walk.request(100, 1, 5, _i32([a, b]), _i32([s]), _i32([b]), 0, out)
                lo, n, start, prefix = out
                assert 0 <= lo <= lo + n <= 100 and 0 <= start <= start + n <= 640 and prefix >= 0, (a, b, s, out[:])
                if 0 <= a <= b <= 100 and 0 <= s <= 640:
                    assert (lo, n, start) == (a, min(b - a, 640 - s), s)
