// What the two forms of the chunk attention share: the division of a call's work over the CTAs, and the parts
// that they leave for the joining launch.
#pragma once

#include <algorithm>

#include "common.cuh"
#include "kernels.h"
#include "sm100.cuh"

namespace uocr {

// Parts of query tiles that were cut: per CTA two slots of [128 columns][tile rows] sums, m [tile], l [tile], and
// what the joining launch needs to know.
struct ChunkParts {
    float* slots;
    int* info;     // [CTAs][kInfoInts]: states of the two slots, then the place of the tile that slot 1 begins
    int ctas, tile;
};
cudaError_t launch_chunk_join(const ChunkArgs& a, const ChunkParts& p, cudaStream_t st);
cudaError_t launch_chunk_rows(const ChunkArgs& a, const ChunkParts& p, cudaStream_t st);

namespace {

constexpr int kPageRows = 128;  // rows of a page, and of a unit
constexpr int kDim = 128;
constexpr int kInfoInts = 8;
constexpr float kLog2e = 1.44269504088896341f;

UOCR_DEV size_t slot_floats(int tile) { return (size_t)tile * (kDim + 2); }

struct Request {
    int lo, n, start, prefix;
};

UOCR_DEV Request request_at(const ChunkArgs& a, int b) {
    Request r;
    r.lo = min(max(__ldg(a.offsets + b), 0), a.T);
    r.start = min(max(__ldg(a.start + b), 0), a.lut_cols * kPageRows);
    r.n = max(min(min(__ldg(a.offsets + b + 1), a.T) - r.lo, a.lut_cols * kPageRows - r.start), 0);
    r.prefix = a.prefix ? max(__ldg(a.prefix + b), 0) : 0;
    return r;
}

// n / g for 0 <= n < 2^31 and g = heads / kv_heads: group_mul = 2^s / g rounded up, off by less than 1, so that the quotient is
// off by less than n / 2^s < 1 / g with s = group_shift > 31 + log2(g). (A division by a variable is 20 instructions, and
// the walks' code is fetched anew for every tile.)
UOCR_DEV int token_of(const ChunkArgs& a, int n) { return (int)((unsigned long long)(uint32_t)n * a.group_mul >> a.group_shift); }

// A query tile is `tile` (token, query head of the KV head) rows of a request. Its pages: columns [0, head_pages) and [tail_page, ...) of its lookup row, `count` in all.
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
// The walk over a CTA's units, a segment (pages of one tile and head) at a time; every warp walks by
// itself.
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

template <typename T>
UOCR_DEV T warp_scan(T v, int lane) {  // inclusive
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const T u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
    }
    return v;
}

// All threads: this CTA's run of units. scratch: B words of shared memory. A call has less than 2^32 units, counted with the
// tiles' leads: the entry point sees to it. (Offsets that do not ascend may reach that many: the run then is some run,
// within the call's requests, tiles and heads.)
UOCR_DEV void find_run(const ChunkArgs& a, Run& run, uint32_t* scratch, int g, int tile, int lead) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // A warp's requests, one in each lane, then one after the other with the lanes on its tiles. (The loops stay rolled: run
    // once, short code is fetched sooner.)
    const int warps = blockDim.x / 32;
#pragma unroll 1
    for (int b0 = warp; b0 < a.B; b0 += 32 * warps) {
        const Request mine = request_at(a, min(b0 + lane * warps, a.B - 1));
#pragma unroll 1
        for (int i = 0, b = b0; i < 32 && b < a.B; ++i, b += warps) {
            Request r;
            r.lo = 0, r.n = __shfl_sync(0xffffffffu, mine.n, i), r.start = __shfl_sync(0xffffffffu, mine.start, i);
            r.prefix = __shfl_sync(0xffffffffu, mine.prefix, i);
            const int tiles = (r.n * g + tile - 1) / tile;
            uint32_t sum = 0;
#pragma unroll 1
            for (int qt = lane; qt < tiles; qt += 32) sum += tile_at(a, r, qt, tile).count + lead;
            sum = __reduce_add_sync(0xffffffffu, sum);
            if (lane == 0) scratch[b] = sum * a.pass_heads;
        }
    }
    __syncthreads();
    if (warp == 0) {
        uint32_t total = 0;
#pragma unroll 1
        for (int b = lane; b < a.B; b += 32) total += scratch[b];
        total = __reduce_add_sync(0xffffffffu, total);
        const uint32_t ctas = min(gridDim.x, total);
        uint32_t u0 = 0, u1 = 0;
        if (blockIdx.x < ctas) {  // runs of two lengths, the longer ones first
            const uint32_t each = total / ctas, rest = total - each * ctas;
            u0 = each * blockIdx.x + min(blockIdx.x, rest);
            u1 = u0 + each + (blockIdx.x < rest ? 1 : 0);
        }
        if (lane == 0) run.some = 0;
        __syncwarp();
        if (u1 > u0) {
            int b = 0;
            uint32_t before = 0;  // units in front of request b
#pragma unroll 1
            for (int b0 = 0; b0 < a.B; b0 += 32) {
                const uint32_t mine = b0 + lane < a.B ? scratch[b0 + lane] : 0;
                const uint32_t upto = before + warp_scan(mine, lane);
                const uint32_t hit = __ballot_sync(0xffffffffu, upto > u0);
                if (hit) {
                    const int f = __ffs(hit) - 1;
                    b = b0 + f;
                    before = __shfl_sync(0xffffffffu, upto - mine, f);
                    break;
                }
                before = __shfl_sync(0xffffffffu, upto, 31);
            }
            const Request r = request_at(a, b);
            const int tiles = (r.n * g + tile - 1) / tile;
#pragma unroll 1
            for (int q0 = 0; q0 < tiles; q0 += 32) {
                const uint32_t count = q0 + lane < tiles ? tile_at(a, r, q0 + lane, tile).count + lead : 0;
                const uint32_t upto = before + warp_scan(count * a.pass_heads, lane);
                const uint32_t hit = __ballot_sync(0xffffffffu, upto > u0);
                if (hit) {
                    if (lane == __ffs(hit) - 1) {
                        const uint32_t in = u0 - (upto - count * a.pass_heads);
                        Walk w;
                        w.left = (int)(u1 - u0), w.b = b, w.qt = q0 + lane, w.head = (int)min(in / count, a.pass_heads - 1u);
                        w.r = r, w.tiles = tiles;
                        run.some = w.enter(a, tile, lead, (int)(in % count));
                        run.first = w;
                    }
                    break;
                }
                before = __shfl_sync(0xffffffffu, upto, 31);
            }
        }
    }
    __syncthreads();
}

UOCR_DEV uint32_t pack_f16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
UOCR_DEV uint32_t pack_bf16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
UOCR_DEV float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Two fp32 operations an instruction (each rounded as its scalar form).
UOCR_DEV uint64_t pair(uint32_t x, uint32_t y) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(x), "r"(y));
    return r;
}
UOCR_DEV uint64_t pair(float x, float y) { return pair(__float_as_uint(x), __float_as_uint(y)); }
UOCR_DEV void unpair(uint64_t v, uint32_t& x, uint32_t& y) { asm("mov.b64 {%0, %1}, %2;" : "=r"(x), "=r"(y) : "l"(v)); }
UOCR_DEV uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
UOCR_DEV uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
UOCR_DEV uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

}  // namespace
}  // namespace uocr
