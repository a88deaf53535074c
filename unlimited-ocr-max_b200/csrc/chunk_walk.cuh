// The chunk attention's requests, query tiles, and the walk over them (device code without inline PTX, so that a host test can
// compile it).
#pragma once

#include "kernels.h"

namespace uocr {
namespace {

constexpr int kPageRows = 128;  // rows of a page, and of a unit

struct Request {
    int lo, n, start, prefix;
};

UOCR_DEV Request request_at(const ChunkArgs& a, int b) {
    Request r;
    r.lo = min(max(__ldg(a.offsets + b), 0), a.T);
    r.start = min(max(__ldg(a.start + b), 0), a.lut_cols * kPageRows);
    const int hi = min(max(__ldg(a.offsets + b + 1), 0), a.T);  // (from 0 on: a difference with INT_MIN would wrap)
    r.n = max(min(hi - r.lo, a.lut_cols * kPageRows - r.start), 0);
    r.prefix = a.prefix ? max(__ldg(a.prefix + b), 0) : 0;
    return r;
}

// n / g for 0 <= n < 2^31 and g = heads / kv_heads: group_mul = 2^s / g rounded up, off by less than 1, so that the quotient is
// off by less than n / 2^s < 1 / g with s = group_shift > 31 + log2(g). (A division by a variable is 20 instructions, and
// the walks' code is fetched anew for every tile.)
UOCR_DEV int token_of(const ChunkArgs& a, int n) { return (int)((unsigned long long)(uint32_t)n * a.group_mul >> a.group_shift); }

// A query tile is `tile` (token, query head of the KV head) rows of a request. Its pages: columns [0, head_pages) and
// [tail_page, ...) of its lookup row, `count` in all.
struct Tile {
    int first_pos, last_pos;  // logical rows of its first and last token
    int head_pages, tail_page, count;
    UOCR_DEV int page(int j) const { return j < head_pages ? j : j - head_pages + tail_page; }
};

UOCR_DEV Tile tile_at(const ChunkArgs& a, const Request& r, int qt, int tile) {
    Tile t;
    const int r0 = qt * tile;
    t.first_pos = r.start + token_of(a, r0);
    t.last_pos = r.start + min(r.n - 1, token_of(a, r0 + tile - 1));
    t.head_pages = t.tail_page = 0;
    if (a.window > 0) {
        t.tail_page = max(0, t.first_pos - a.window + 1) / kPageRows;
        t.head_pages = min((min(r.prefix, t.last_pos + 1) + kPageRows - 1) / kPageRows, t.tail_page);
    }
    t.count = t.head_pages + t.last_pos / kPageRows + 1 - t.tail_page;
    return t;
}

// A CTA's run of the call's work. Work is counted in pages; a tile and head counts `lead` more in front of its pages, for what
// a CTA does once for it (its queries, its results), so that a run of many short tiles takes no longer than one of a few long
// ones.
// The walk over a CTA's units, a segment (pages of one tile and head) at a time; every warp has one of its own in shared
// memory, and one lane moves it.
struct Walk {
    int b, qt, head, j, n, tiles;  // segment: pages j .. j + n - 1 of the tile's
    int left;                      // of the run, behind this segment
    Request r;
    Tile t;
    // at x of the segment's tile and head; false: the run ends in front of its pages
    UOCR_DEV bool enter(const ChunkArgs& a, int tile, int lead, int x) {
        t = tile_at(a, r, qt, tile);
        const int end = min(x + left, t.count + lead);
        j = max(x - lead, 0);
        n = max(end - lead, 0) - j;
        left -= end - x;
        return n > 0;
    }
    UOCR_DEV bool next(const ChunkArgs& a, int g, int tile, int lead) {
        if (left <= 0) return false;
        if (++head == a.pass_heads) {
            head = 0;
            if (++qt >= tiles) {
                qt = 0;
                do {  // left > 0: another request with rows follows (unless offsets that do not ascend overflowed the count)
                    if (++b >= a.B) {
                        left = 0;
                        return false;
                    }
                    r = request_at(a, b);
                } while (r.n == 0);
                tiles = (r.n * g + tile - 1) / tile;
            }
        }
        return enter(a, tile, lead, 0);
    }
    UOCR_DEV bool whole() const { return j == 0 && n == t.count; }
};

// A CTA's run: its first segment, if it has one (heads are counted from the pass's first).
struct Run {
    Walk first;
    int some;
};

// A whole warp's: at the run's first segment; on to the next one. All lanes have read the walk before it moves, and see it moved.
UOCR_DEV bool warp_first(Walk& w, const Run& run) {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) w = run.first;
    __syncwarp();
    return run.some;
}
UOCR_DEV bool warp_next(Walk& w, const ChunkArgs& a, int g, int tile, int lead) {
    __syncwarp();
    int more = 0;
    if ((threadIdx.x & 31) == 0) more = w.next(a, g, tile, lead);
    more = __shfl_sync(0xffffffffu, more, 0);
    __syncwarp();
    return more;
}

}  // namespace
}  // namespace uocr
