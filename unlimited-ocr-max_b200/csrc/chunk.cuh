// What the two forms of the chunk attention share: the division of a call's work over the CTAs, and the parts
// that they leave for the joining launch.
#pragma once

#include <algorithm>

#include "common.cuh"
#include "chunk_walk.cuh"
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

constexpr int kDim = 128;
constexpr int kInfoInts = 8;
constexpr float kLog2e = 1.44269504088896341f;

UOCR_DEV size_t slot_floats(int tile) { return (size_t)tile * (kDim + 2); }

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
