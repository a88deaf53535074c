// Attention of a chunk of new tokens over the paged cache (the prefill counterpart of the decode
// step's paged attention: store_k/v_cache_ragged and flash_attention_ragged of decoder.py:425-437 for
// any number of new rows per request).
//
// Request b brings rows [off[b], off[b + 1]) of q, k_new and v_new; the i-th of them is logical row
// p = start[b] + i of the request. It sees row r when r <= p and (no window, or r > p - window, or
// r < prefix[b]), and
//   out = sum_r e^(s_r - m) v_r / sum_r e^(s_r - m),   s_r = scale q . k_r,   m = max_r s_r.
// Rows below start[b] come from the pool, the new ones from k_new / v_new, which are stored into the
// pool by the same call.
//
// Work. A unit is (query tile, KV head, page): a query tile is 128 (token, query head of the KV head)
// pairs of one request, a page its 128 rows. Pages that no token of the tile sees are left out. The units of
// the call, in the order request, tile, head, page, are dealt to one CTA per SM in equal runs, whatever
// the lengths: a run may begin and end inside a tile's pages. A tile that lies in one run is written
// straight to out; the parts of one that was cut go to the workspace as (m, l, sum) and a second launch
// joins them in the order of the pages. Every CTA finds its run from the lengths on the device.
//
// A CTA: 8 warps load the page's rows into registers (two 32 KB granules in flight), turn them into
// tensor-core operands in a ring of shared memory, and store the new rows; one warp issues tcgen05.mma;
// 8 warps do the softmax, two threads per query row. The query operand and the weights P are read by the
// tensor core from TMEM, so shared memory carries each key and value once:
//   S = Q K^T (TMEM, two buffers) -> softmax warps -> P (in S's place) -> P V (TMEM) -> added to the
//   sums in registers, in fp32 with round-to-nearest, after each page.
//
// fp32: a product of fp32 rows is three products of fp16 halves, hi x hi + hi x lo + lo x hi, where
// x = hi + lo to 2^-22 of x: 8 rows of k, a query row and the 64 columns of a page's v are scaled by a power of two
// that brings their largest element to [2^14, 2^15), and the weights by 2^14, so the halves keep their bits
// over fp16's exponent range. The small products go into the accumulator first: the tensor core's
// additions truncate, and only the last 8 then round at the result's full size. bf16: one product; the
// weights are rounded to bf16, as the tensor core takes both operands in one type.
// Values that are not finite are kept out of the V operand (0 x inf would reach rows that do not see
// them) and added to the rows that do see them.
#include <algorithm>

#include "common.cuh"
#include "kernels.h"
#include "sm100.cuh"

namespace uocr {
namespace {

constexpr int kPageRows = 128;  // rows of a page, and of a unit
constexpr int kDim = 128;
constexpr int kTile = 128;      // (token, head) rows of a query tile
constexpr int kTeamWarps = 8, kLoadWarps = 8;
constexpr int kThreads = 32 * (kTeamWarps + kLoadWarps + 1);
constexpr int kStages = 6;      // ring of granules: 64 rows of k, or 64 columns of v
constexpr int kSlotFloats = kTile * (kDim + 2);  // a part: sums [128 columns][128 rows], m [128], l [128]
constexpr int kInfoInts = 8;    // per CTA: states of its two slots, then the tile's place
constexpr uint32_t kTeamBar = 1, kLoadBar = 2;
constexpr float kLog2e = 1.44269504088896341f;

// TMEM columns
constexpr uint32_t kColS = 0, kColPv = 256, kColQ = 384;

struct Shared {
    uint64_t full[kStages], empty[kStages], s_full[2], p_full[2], pv_full, pv_free, q_full, drain;
    uint32_t tmem;
    volatile int abort;
    int left;                    // this CTA's units
    int b, qt, head, j;          // and where they begin
    float kscale[8][16];         // by unit: 1 / scale of 8 rows of k
    float vscale[8][2];          // by unit: 1 / scale of 64 columns of v
    alignas(16) uint16_t vbad[8][2][8];      // by unit: rows with values that are not finite
    float vmax[2][kLoadWarps];
    float xmax[2][2][kTile], xsum[2][kTile];
};

struct Request {
    int lo, n, start, prefix;
};

UOCR_DEV Request request_at(const ChunkArgs& a, int b) {
    Request r;
    r.lo = min(max(__ldg(a.offsets + b), 0), a.T);
    r.n = max(min(__ldg(a.offsets + b + 1), a.T) - r.lo, 0);
    r.start = min(max(__ldg(a.start + b), 0), a.lut_cols * kPageRows);
    r.prefix = a.prefix ? max(__ldg(a.prefix + b), 0) : 0;
    return r;
}

// A query tile's pages: columns [0, head_pages) and [tail_page, ...) of its lookup row, `count` in all.
struct Tile {
    int first_pos, last_pos;  // logical rows of its first and last token
    int head_pages, tail_page, count;
    UOCR_DEV int page(int j) const { return j < head_pages ? j : j - head_pages + tail_page; }
};

UOCR_DEV Tile tile_at(const ChunkArgs& a, const Request& r, int qt, int g) {
    Tile t;
    const int r0 = qt * kTile;
    t.first_pos = r.start + r0 / g;
    t.last_pos = r.start + min(r.n - 1, (r0 + kTile - 1) / g);
    t.head_pages = t.tail_page = 0;
    if (a.window > 0) {
        t.tail_page = max(0, t.first_pos - a.window + 1) / kPageRows;
        t.head_pages = min((min(r.prefix, t.last_pos + 1) + kPageRows - 1) / kPageRows, t.tail_page);
    }
    t.count = t.head_pages + t.last_pos / kPageRows + 1 - t.tail_page;
    return t;
}

// The walk over a CTA's units, a segment (pages of one tile and head) at a time; every warp walks by
// itself.
struct Walk {
    int b, qt, head, j, n, tiles;  // segment: pages j .. j + n - 1 of the tile's
    int left;                      // units behind this segment
    Request r;
    Tile t;
    UOCR_DEV void enter(const ChunkArgs& a, int g) {
        t = tile_at(a, r, qt, g);
        n = min(t.count - j, left);
        left -= n;
    }
    UOCR_DEV bool begin(const ChunkArgs& a, const Shared& s, int g) {
        left = s.left;
        if (left <= 0) return false;
        b = s.b, qt = s.qt, head = s.head, j = s.j;
        r = request_at(a, b);
        tiles = (r.n * g + kTile - 1) / kTile;
        enter(a, g);
        return true;
    }
    UOCR_DEV bool next(const ChunkArgs& a, int g) {
        if (left <= 0) return false;
        j = 0;
        if (++head == a.kv_heads) {
            head = 0;
            if (++qt >= tiles) {
                qt = 0;
                do {  // left > 0: another request with rows follows
                    ++b;
                    r = request_at(a, b);
                } while (r.n == 0 && b < a.B - 1);
                tiles = (r.n * g + kTile - 1) / kTile;
            }
        }
        enter(a, g);
        return true;
    }
    UOCR_DEV bool whole() const { return j == 0 && n == t.count; }
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

// All threads: this CTA's run of units, into s. scratch: B long longs of shared memory.
__device__ void find_run(const ChunkArgs& a, Shared& s, long long* scratch, int g) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int b = warp; b < a.B; b += kThreads / 32) {
        const Request r = request_at(a, b);
        const int tiles = (r.n * g + kTile - 1) / kTile;
        long long sum = 0;
        for (int qt = lane; qt < tiles; qt += 32) sum += tile_at(a, r, qt, g).count;
#pragma unroll
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) scratch[b] = sum * a.kv_heads;
    }
    __syncthreads();
    if (warp == 0) {
        long long total = 0;
        for (int b = lane; b < a.B; b += 32) total += scratch[b];
#pragma unroll
        for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
        const long long ctas = min((long long)gridDim.x, total);
        long long u0 = 0, u1 = 0;
        if ((long long)blockIdx.x < ctas) u0 = total * blockIdx.x / ctas, u1 = total * (blockIdx.x + 1) / ctas;
        if (lane == 0) s.left = (int)(u1 - u0);
        if (u1 > u0) {
            int b = 0;
            long long before = 0;  // units in front of request b
            for (int b0 = 0; b0 < a.B; b0 += 32) {
                const long long mine = b0 + lane < a.B ? scratch[b0 + lane] : 0;
                const long long upto = before + warp_scan(mine, lane);
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
            const int tiles = (r.n * g + kTile - 1) / kTile;
            for (int q0 = 0; q0 < tiles; q0 += 32) {
                const int count = q0 + lane < tiles ? tile_at(a, r, q0 + lane, g).count : 0;
                const long long upto = before + warp_scan((long long)count * a.kv_heads, lane);
                const uint32_t hit = __ballot_sync(0xffffffffu, upto > u0);
                if (hit) {
                    if (lane == __ffs(hit) - 1) {
                        const long long in = u0 - (upto - (long long)count * a.kv_heads);
                        s.b = b, s.qt = q0 + lane, s.head = (int)(in / count), s.j = (int)(in % count);
                    }
                    break;
                }
                before = __shfl_sync(0xffffffffu, upto, 31);
            }
        }
    }
    __syncthreads();
}

UOCR_DEV bool wait(Shared& s, uint64_t* bar, uint32_t parity) {
    if (mbar_wait_warp(bar, parity, &s.abort, nullptr)) return true;
    s.abort = 1;
    return false;
}

// ---- tensor-core operands ---------------------------------------------------------------------
// D[tmem] (+)= A[tmem] * B[smem], kind::f16, one thread issues.
UOCR_DEV void umma_ts_f16(uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// A value granule: 64 columns contiguous per row (MN-major), 128-byte swizzle, 8-row groups 1024 bytes
// apart; the granule is one column block wide, so the stride between column blocks is never used.
UOCR_DEV uint64_t desc_mn_sw128(uint32_t addr) {
    return (uint64_t)((addr >> 4) & 0x3FFFu) | (uint64_t)(1024 >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 |
           (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// M 128, N 64; fp16 or bf16 operands; B from keys (K-major) or values (MN-major: bit 16)
template <bool kF32>
constexpr uint32_t idesc(bool mn) {
    return (1u << 4) | (kF32 ? 0u : (1u << 7) | (1u << 10)) | (mn ? 1u << 16 : 0u) | (64u >> 3) << 17 | (128u >> 4) << 24;
}

template <int N>
UOCR_DEV void tmem_st(uint32_t addr, const uint32_t* r);
template <>
UOCR_DEV void tmem_st<8>(uint32_t addr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(addr), "r"(r[0]),
                 "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
// tcgen05.wait::ld that marks r[] as written by it: no use of r[] moves in front of it
UOCR_DEV void tmem_wait_ld16(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :
                 : "memory");
}
UOCR_DEV void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

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
// two values as fp16 halves: hi takes the upper 11 bits (exactly), lo the rest (rounded to 11 bits)
UOCR_DEV void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
    const float xh = __uint_as_float(__float_as_uint(x) & 0xFFFFE000u), yh = __uint_as_float(__float_as_uint(y) & 0xFFFFE000u);
    hi = pack_f16(xh, yh);
    lo = pack_f16(__fsub_rn(x, xh), __fsub_rn(y, yh));
}
// 2^(14 - e) and its inverse for the largest magnitude's bits (e its exponent, from -112 up: below that
// the values are smaller than 2^14 after scaling, which costs them bits they do not have)
UOCR_DEV float scale_up(uint32_t bits) { return __uint_as_float((268u - max(bits >> 23, 15u)) << 23); }
UOCR_DEV float scale_down(uint32_t bits) { return __uint_as_float((max(bits >> 23, 15u) - 14u) << 23); }

UOCR_DEV uint4 ldg_stream(const void* p) { return ldg_nc_v4(p); }

// ---- loading warps ----------------------------------------------------------------------------
// The granules of a segment in the order in which the tensor core takes them: K(0), K(1), V(0), K(2),
// V(1), ..., each as two halves (64 rows of k; 64 columns of v).
struct Granules {
    Walk w;
    int jj, half;
    bool v, more;
    uint32_t unit0;  // units in front of the segment
    UOCR_DEV void begin(const ChunkArgs& a, const Shared& s, int g) {
        more = w.begin(a, s, g);
        jj = half = 0, v = false, unit0 = 0;
    }
    UOCR_DEV void next(const ChunkArgs& a, int g) {
        if (half == 0) {
            half = 1;
            return;
        }
        half = 0;
        if (!v && jj >= 1) {
            v = true;
            return;
        }
        ++jj;
        v = jj >= w.n;
        if (jj > w.n) {
            unit0 += w.n;
            more = w.next(a, g);
            jj = 0, v = false;
        }
    }
};

// What a loaded granule needs when it is turned into an operand.
struct Loaded {
    char* store;    // the page's row 0 of this head (this half) in the pool, for the new rows to store
    uint32_t bits;  // first page row to store, rows to store (8 bits each), half, v, unit & 7
    UOCR_DEV void set(uint32_t unit, int half, bool v, int row0, int own) {
        bits = (uint32_t)row0 | (uint32_t)own << 8 | (uint32_t)half << 16 | (uint32_t)v << 17 | (unit & 7) << 18;
    }
    UOCR_DEV int row0() const { return bits & 255; }
    UOCR_DEV int own() const { return bits >> 8 & 255; }
    UOCR_DEV int half() const { return bits >> 16 & 1; }
    UOCR_DEV bool v() const { return bits >> 17 & 1; }
    UOCR_DEV uint32_t unit() const { return bits >> 18 & 7; }
};

// fp32: a thread holds 8 x 16 bytes: 4 dimensions of 8 rows of k, or 4 columns of 8 rows of v.
// bf16: 4 x 16 bytes: 8 dimensions of 4 rows.
template <bool kF32>
struct Lanes {
    static constexpr int kWords = kF32 ? 8 : 4;
    static constexpr int kElt = kF32 ? 4 : 2;
    // page row of word i, and the byte of the row's 128 (k) or 64 (v) elements
    static UOCR_DEV int row(bool v, int half, int i, int wc, int lane) {
        if (kF32) return v ? wc * 16 + 2 * i + (lane >> 4) : half * 64 + wc * 8 + i;
        return v ? wc * 16 + 4 * i + (lane >> 3) : half * 64 + wc * 8 + 2 * i + (lane >> 4);
    }
    static UOCR_DEV int byte(bool v, int lane) {
        if (kF32) return (v ? lane & 15 : lane) * 16;
        return (v ? lane & 7 : lane & 15) * 16;
    }
};

template <bool kF32>
UOCR_DEV void load_granule(const ChunkArgs& a, const Granules& gr, int g, int wc, int lane,
                           uint4 (&x)[Lanes<kF32>::kWords], Loaded& info) {
    using L = Lanes<kF32>;
    const Walk& w = gr.w;
    const int j = gr.v ? gr.jj - 1 : gr.jj, t = w.t.page(w.j + j);
    const size_t row_bytes = (size_t)a.kv_heads * kDim * L::kElt;
    const size_t column = (size_t)w.head * kDim * L::kElt + (gr.v ? gr.half * 64 * L::kElt : 0);
    const uint32_t id = t < a.lut_cols ? __ldg(a.lut + (size_t)w.b * a.lut_cols + t) : 0xFFFFFFFFu;
    char* page = static_cast<char*>(a.pool) +
                 (((size_t)min(id, (uint32_t)(a.pages - 1)) * 2 + (gr.v ? 1 : 0)) * a.layers + a.layer) * (kPageRows * row_bytes) +
                 column;
    const char* fresh = static_cast<const char*>(gr.v ? a.v : a.k) + column;
    const size_t fresh_ld = (size_t)(gr.v ? a.v_ld : a.k_ld) * L::kElt;
    const int r0 = t * kPageRows;
#pragma unroll
    for (int i = 0; i < L::kWords; ++i) {
        const int row = L::row(gr.v, gr.half, i, wc, lane), r = r0 + row;
        const char* p = r >= w.r.start ? fresh + (size_t)(w.r.lo + r - w.r.start) * fresh_ld : page + (size_t)row * row_bytes;
        x[i] = r <= w.t.last_pos ? ldg_stream(p + L::byte(gr.v, lane)) : make_uint4(0, 0, 0, 0);
    }
    // This tile stores the new rows whose first query head lies in it: every new row is of one tile.
    const int i0 = (w.qt * kTile + g - 1) / g, i1 = min(w.r.n, (w.qt * kTile + kTile + g - 1) / g);
    const int s0 = min(max(w.r.start + i0 - r0, 0), kPageRows), s1 = min(w.r.start + i1 - r0, kPageRows);
    info.store = page;
    info.set(gr.unit0 + j, gr.half, gr.v, s0, id < (uint32_t)a.pages ? max(s1 - s0, 0) : 0);
}

template <bool kF32>
UOCR_DEV void convert_granule(const ChunkArgs& a, Shared& s, unsigned char* stage, int wc, int lane,
                              uint4 (&x)[Lanes<kF32>::kWords], const Loaded& info) {
    using L = Lanes<kF32>;
    const size_t row_bytes = (size_t)a.kv_heads * kDim * L::kElt;
    const int half = info.half();
    const bool is_v = info.v();
    if (info.own() > 0) {
#pragma unroll
        for (int i = 0; i < L::kWords; ++i) {
            const int row = L::row(is_v, half, i, wc, lane);
            if ((unsigned)(row - info.row0()) < (unsigned)info.own())
                *reinterpret_cast<uint4*>(info.store + (size_t)row * row_bytes + L::byte(is_v, lane)) = x[i];
        }
    }
    const uint32_t ub = info.unit();
    if constexpr (kF32) {
        uint32_t top = 0;
        auto largest = [&] {
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                m = max(m, max(x[i].x & 0x7FFFFFFFu, x[i].y & 0x7FFFFFFFu));
                m = max(m, max(x[i].z & 0x7FFFFFFFu, x[i].w & 0x7FFFFFFFu));
            }
            return __reduce_max_sync(0xffffffffu, m);
        };
        top = largest();
        uint32_t bad = 0;  // v rows of this warp with values that are not finite
        if (top >= 0x7F800000u) {
            // rare: v loses these values here (the softmax warps add them to the rows that see them);
            // a key keeps them (its scores become NaN), but they set no scale
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                uint32_t* e = &x[i].x;
                bool row_bad = false;
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const bool inf = (e[c] & 0x7F800000u) == 0x7F800000u;
                    row_bad |= inf;
                    if (inf && is_v) e[c] = 0;
                    else if (inf) e[c] = 0x7FFFFFFFu;
                    else m = max(m, e[c] & 0x7FFFFFFFu);
                }
                const uint32_t who = __ballot_sync(0xffffffffu, row_bad);
                if (who & 0x0000FFFFu) bad |= 1u << (2 * i);
                if (who & 0xFFFF0000u) bad |= 2u << (2 * i);
            }
            top = __reduce_max_sync(0xffffffffu, m);
        }
        if (is_v) {
            // one scale for the granule: the rows are summed over
            if (lane == 0) {
                s.vmax[half][wc] = __uint_as_float(top);
                s.vbad[ub][half][wc] = (uint16_t)bad;
            }
            named_bar_sync(kLoadBar, 32 * kLoadWarps);
            top = __reduce_max_sync(0xffffffffu, __float_as_uint(s.vmax[half][lane & 7]));
            if (wc == 0 && lane == 0) s.vscale[ub][half] = scale_down(top);
        } else if (lane == 0) {
            s.kscale[ub][half * 8 + wc] = scale_down(top);
        }
        const float up = scale_up(top);
        const uint32_t base = smem_addr(stage);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float f0 = __uint_as_float(x[i].x) * up, f1 = __uint_as_float(x[i].y) * up;
            const float f2 = __uint_as_float(x[i].z) * up, f3 = __uint_as_float(x[i].w) * up;
            uint2 hi, lo;
            split2(f0, f1, hi.x, lo.x);
            split2(f2, f3, hi.y, lo.y);
            // 8 bytes (4 elements) of a 128-byte operand row, its 16-byte chunks swizzled by the row
            int row = L::row(is_v, half, i, wc, lane);
            const int c8 = lane & 15;  // 8-byte word of the 64-element row
            uint32_t at;
            if (is_v) at = row * 128;
            else row &= 63, at = (lane >> 4) * 8192 + row * 128;
            at += (((c8 >> 1) ^ (row & 7)) << 4) + (c8 & 1) * 8;
            asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(base + at), "r"(hi.x), "r"(hi.y) : "memory");
            asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(base + 16384 + at), "r"(lo.x), "r"(lo.y) : "memory");
        }
    } else {
        if (is_v) {
            uint32_t any = 0;
            auto odd = [](uint32_t w) { return ((w & 0x7F807F80u) + 0x00800080u) & 0x80008000u; };
#pragma unroll
            for (int i = 0; i < 4; ++i) any |= odd(x[i].x) | odd(x[i].y) | odd(x[i].z) | odd(x[i].w);
            uint32_t bad = 0;
            if (__any_sync(0xffffffffu, any != 0)) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t* e = &x[i].x;
                    uint32_t row_bad = 0;
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const uint32_t o = odd(e[c]);
                        row_bad |= o;
                        if (o & 0x00008000u) e[c] &= 0xFFFF0000u;
                        if (o & 0x80000000u) e[c] &= 0x0000FFFFu;
                    }
                    const uint32_t who = __ballot_sync(0xffffffffu, row_bad != 0);
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        if (who >> (8 * q) & 0xFFu) bad |= 1u << (4 * i + q);
                }
            }
            if (lane == 0) s.vbad[ub][half][wc] = (uint16_t)bad;
        }
        const uint32_t base = smem_addr(stage);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            int row = L::row(is_v, half, i, wc, lane);
            uint32_t at;
            if (is_v) at = row * 128;
            else row &= 63, at = ((lane >> 3) & 1) * 8192 + row * 128;
            at += ((lane & 7) ^ (row & 7)) << 4;
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(base + at), "r"(x[i].x), "r"(x[i].y), "r"(x[i].z),
                         "r"(x[i].w)
                         : "memory");
        }
    }
}

template <bool kF32>
__device__ void load_role(const ChunkArgs& a, Shared& s, unsigned char* ring, int g) {
    constexpr int kBytes = kF32 ? 32768 : 16384;
    const int wc = (threadIdx.x >> 5) - kTeamWarps, lane = threadIdx.x & 31;
    Granules gr;
    gr.begin(a, s, g);
    if (!gr.more) return;
    uint4 x[2][Lanes<kF32>::kWords];
    Loaded info[2];
    load_granule<kF32>(a, gr, g, wc, lane, x[0], info[0]);
    bool have = true;
    uint32_t stage = 0, phase = 0;
    auto step = [&](int now, int ahead) {
        gr.next(a, g);
        const bool more = gr.more;
        if (more) load_granule<kF32>(a, gr, g, wc, lane, x[ahead], info[ahead]);
        if (!wait(s, &s.empty[stage], phase ^ 1)) return false;
        convert_granule<kF32>(a, s, ring + stage * kBytes, wc, lane, x[now], info[now]);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.full[stage]);
        if (++stage == kStages) stage = 0, phase ^= 1;
        have = more;
        return true;
    };
    while (have) {
        if (!step(0, 1)) return;
        if (!have) break;
        if (!step(1, 0)) return;
    }
}

// ---- the issuing warp -------------------------------------------------------------------------
template <bool kF32>
__device__ void mma_role(const ChunkArgs& a, Shared& s, unsigned char* ring, int g) {
    constexpr int kBytes = kF32 ? 32768 : 16384;
    const int lane = threadIdx.x & 31;
    const uint32_t tmem = s.tmem, base = smem_addr(ring);
    uint32_t stage = 0, phase = 0, unit0 = 0, seg = 0;
    Walk w;
    // a finished granule: its MMAs issued, its stage given back
    auto granule = [&](auto&& issue) {
        if (!wait(s, &s.full[stage], phase)) return false;
        tc_fence_after();
        if (lane == 0) {
            issue(base + stage * kBytes);
            umma_commit(&s.empty[stage]);
        }
        __syncwarp();
        if (++stage == kStages) stage = 0, phase ^= 1;
        return true;
    };
    auto run = [&] {
        for (bool more = w.begin(a, s, g); more; more = w.next(a, g), ++seg) {
            if (!wait(s, &s.q_full, seg & 1)) return;
            tc_fence_after();
            const int n = w.n;
            for (int jj = 0; jj <= n; ++jj) {
                if (jj < n) {
                    const uint32_t u = unit0 + jj, d = tmem + kColS + (u & 1) * 128;
                    for (int half = 0; half < 2; ++half) {
                        const bool ok = granule([&](uint32_t k) {
                            const uint32_t dh = d + half * 64, q = tmem + kColQ;
#pragma unroll
                            for (int p = kF32 ? 0 : 2; p < 3; ++p) {  // q lo x k hi, q hi x k lo, q hi x k hi
#pragma unroll
                                for (int i = 0; i < 8; ++i)
                                    umma_ts_f16(dh, q + (p == 0 ? 64 : 0) + i * 8,
                                                umma_desc_sw128(k + (p == 1 ? 16384 : 0) + (i >> 2) * 8192 + (i & 3) * 32),
                                                idesc<kF32>(false), p != (kF32 ? 0 : 2) || i != 0);
                            }
                        });
                        if (!ok) return;
                    }
                    if (lane == 0) umma_commit(&s.s_full[u & 1]);
                    __syncwarp();
                }
                if (jj >= 1) {
                    const uint32_t u = unit0 + jj - 1, pa = tmem + kColS + (u & 1) * 128;
                    if (!wait(s, &s.p_full[u & 1], (u >> 1) & 1) || !wait(s, &s.pv_free, (u & 1) ^ 1)) return;
                    tc_fence_after();
                    for (int half = 0; half < 2; ++half) {
                        const bool ok = granule([&](uint32_t v) {
                            const uint32_t dh = tmem + kColPv + half * 64;
#pragma unroll
                            for (int p = kF32 ? 0 : 2; p < 3; ++p) {  // p lo x v hi, p hi x v lo, p hi x v hi
#pragma unroll
                                for (int i = 0; i < 8; ++i)
                                    umma_ts_f16(dh, pa + i * 16 + (p == 0 ? 8 : 0),
                                                desc_mn_sw128(v + (p == 1 ? 16384 : 0) + i * 2048), idesc<kF32>(true),
                                                p != (kF32 ? 0 : 2) || i != 0);
                            }
                        });
                        if (!ok) return;
                    }
                    if (lane == 0) umma_commit(&s.pv_full);
                    __syncwarp();
                }
            }
            unit0 += n;
        }
    };
    run();
    // every MMA of this CTA has finished before its TMEM is freed
    if (lane == 0) umma_commit(&s.drain);
    __syncwarp();
    mbar_wait_warp(&s.drain, 0, nullptr, nullptr);
}

// ---- the softmax warps ------------------------------------------------------------------------
// Thread (row, half): row of the query tile (its TMEM lane), columns and dimensions [64 half, 64 half + 64).
template <bool kF32>
__device__ __noinline__ void add_bad_values(const ChunkArgs& a, const Walk& w, int t, int row, bool seen, int half,
                                            float* out64) {
    // value row `row` of page t: what is not finite of this half's 64 columns, into out64 (else 0)
    const int r = t * kPageRows + row;
    const size_t elt = kF32 ? 4 : 2;
    const uint32_t id = t < a.lut_cols ? __ldg(a.lut + (size_t)w.b * a.lut_cols + t) : 0xFFFFFFFFu;
    const size_t row_elts = (size_t)a.kv_heads * kDim;
    const char* p = r >= w.r.start
                        ? static_cast<const char*>(a.v) + ((size_t)(w.r.lo + r - w.r.start) * a.v_ld + w.head * kDim) * elt
                        : static_cast<const char*>(a.pool) +
                              (((((size_t)min(id, (uint32_t)(a.pages - 1)) * 2 + 1) * a.layers + a.layer) * kPageRows + row) *
                                   row_elts +
                               w.head * kDim) *
                                  elt;
    for (int d = 0; d < 64; ++d) {
        const float v = kF32 ? reinterpret_cast<const float*>(p)[half * 64 + d]
                             : bf16f(reinterpret_cast<const uint16_t*>(p)[half * 64 + d]);
        if (seen && (__float_as_uint(v) & 0x7F800000u) == 0x7F800000u) out64[d] += v;
    }
}

// Which of 32 columns from c0 on a row sees: c <= hi and (c >= lo or c < pre), all relative to the page.
UOCR_DEV uint32_t seen_mask(int c0, int hi, int lo, int pre) {
    auto below = [](int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; };
    return below(hi + 1 - c0) & (~below(lo - c0) | below(pre - c0));
}

template <bool kF32>
__device__ void team_role(const ChunkArgs& a, Shared& s, float* slots, int* info, int g) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int half = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lanes = s.tmem + ((uint32_t)(warp & 3) << 21);  // lane field: bits 16 up, 32 lanes a warp
    const float factor = fabsf(a.scale) * kLog2e;  // the scale's sign is in the query operand
    float qscale = 0.f;
    bool alive = true;

    // the query row of a segment into TMEM; qscale: 1 / its scale, times the softmax's factor
    auto load_query = [&](const Walk& w) {
        const int R = w.qt * kTile + row;
        const bool valid = R < w.r.n * g;
        const char* p = static_cast<const char*>(a.q) +
                        ((size_t)(w.r.lo + (valid ? R / g : 0)) * a.q_ld + (size_t)(w.head * g + (valid ? R % g : 0)) * kDim) *
                            (kF32 ? 4 : 2);
        if constexpr (kF32) {
            const float4* q4 = reinterpret_cast<const float4*>(p);
            uint32_t m = 0;
            if (valid) {
#pragma unroll 8
                for (int i = 0; i < 32; ++i) {
                    const uint4 v = *reinterpret_cast<const uint4*>(q4 + i);
                    const uint32_t e[4] = {v.x & 0x7FFFFFFFu, v.y & 0x7FFFFFFFu, v.z & 0x7FFFFFFFu, v.w & 0x7FFFFFFFu};
#pragma unroll
                    for (int c = 0; c < 4; ++c) m = max(m, e[c] < 0x7F800000u ? e[c] : 0u);
                }
            }
            const float up = a.scale < 0.f ? -scale_up(m) : scale_up(m);
            qscale = scale_down(m) * factor;
#pragma unroll
            for (int c = 0; c < 4; ++c) {  // 16 dimensions at a time
                uint32_t hi[8], lo[8];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float4 v = valid ? q4[half * 16 + c * 4 + i] : make_float4(0.f, 0.f, 0.f, 0.f);
                    split2(v.x * up, v.y * up, hi[2 * i], lo[2 * i]);
                    split2(v.z * up, v.w * up, hi[2 * i + 1], lo[2 * i + 1]);
                }
                tmem_st<8>(lanes + kColQ + half * 32 + c * 8, hi);
                tmem_st<8>(lanes + kColQ + 64 + half * 32 + c * 8, lo);
            }
        } else {
            qscale = factor;
            const uint4* q4 = reinterpret_cast<const uint4*>(p) + half * 8;
            const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                uint32_t x[8];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const uint4 v = valid ? q4[c * 2 + i] : make_uint4(0, 0, 0, 0);
                    x[4 * i] = v.x ^ flip, x[4 * i + 1] = v.y ^ flip, x[4 * i + 2] = v.z ^ flip, x[4 * i + 3] = v.w ^ flip;
                }
                tmem_st<8>(lanes + kColQ + half * 32 + c * 8, x);
            }
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.q_full);
    };

    float acc[64];
    float m = 0.f, l = 0.f, alpha = 1.f;

    // acc = acc * alpha + (P V of unit u), and the values of page t that were kept out of it
    auto add_pv = [&](const Walk& w, uint32_t u, int t, bool live, int pos) {
        if (alive && !wait(s, &s.pv_full, u & 1)) alive = false;
        if (alive && live) {
            tc_fence_after();
            const float f = kF32 ? s.vscale[u & 7][half] : 1.f;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                uint32_t x[16];
                tmem_ld_32x32b_x16(lanes + kColPv + half * 64 + c * 16, x);
                tmem_wait_ld16(x);
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[c * 16 + i] = fmaf(acc[c * 16 + i], alpha, __uint_as_float(x[i]) * f);
            }
            uint32_t bad = 0;
            const uint4* vb = reinterpret_cast<const uint4*>(s.vbad[u & 7][half]);  // 8 x 16 rows
            bad = vb->x | vb->y | vb->z | vb->w;
            if (bad) {
                for (int q = 0; q < 128; ++q) {
                    if (!(s.vbad[u & 7][half][q >> 4] >> (q & 15) & 1)) continue;
                    const int r = t * kPageRows + q;
                    const bool seen = r <= pos && (a.window <= 0 || r > pos - a.window || r < w.r.prefix);
                    float extra[64];
                    for (int d = 0; d < 64; ++d) extra[d] = 0.f;
                    add_bad_values<kF32>(a, w, t, q, seen, half, extra);
#pragma unroll
                    for (int d = 0; d < 64; ++d) acc[d] += extra[d];
                }
            }
            tc_fence_before();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.pv_free);
    };

    Walk w;
    bool more = w.begin(a, s, g);
    int state[2] = {0, 0}, place[4] = {0, 0, 0, 0};
    uint32_t unit0 = 0;
    if (more) load_query(w);
    while (more) {
        const int R = w.qt * kTile + row, rows = w.r.n * g - w.qt * kTile;  // valid rows of the tile
        const bool live = (warp & 3) * 32 < rows;                           // this warp has some
        const int pos = w.r.start + R / g;
        m = -INFINITY, l = 0.f;
        float alpha_next = 1.f;
#pragma unroll
        for (int i = 0; i < 64; ++i) acc[i] = 0.f;
        for (int j = 0; j < w.n; ++j) {
            const uint32_t u = unit0 + j, buf = u & 1;
            const int t = w.t.page(w.j + j), c0 = t * kPageRows;
            if (alive && !wait(s, &s.s_full[buf], (u >> 1) & 1)) alive = false;
            tc_fence_after();
            const uint32_t sa = lanes + kColS + buf * 128 + half * 64;
            // does every row of the tile see the whole page?
            const bool all = c0 + kPageRows - 1 <= w.t.first_pos &&
                             (a.window <= 0 || c0 > w.t.last_pos - a.window || c0 + kPageRows <= w.r.prefix);
            uint32_t mask[2] = {0xffffffffu, 0xffffffffu};
            if (!all) {
                const int lo = a.window > 0 ? pos - a.window + 1 - c0 : -kPageRows;
#pragma unroll
                for (int c = 0; c < 2; ++c) mask[c] = seen_mask(half * 64 + c * 32, pos - c0, lo, w.r.prefix - c0);
            }
            // 1 / (scale of 8 columns' keys) x the query's: read where it is used
            auto f = [&](int i) { return kF32 ? s.kscale[u & 7][half * 8 + i] * qscale : qscale; };
            float top = -INFINITY;
            if (alive && live) {
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t x[16];
                    tmem_ld_32x32b_x16(sa + c * 16, x);
                    tmem_wait_ld16(x);
                    if (!all) {
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            if (!(mask[c >> 1] >> ((c & 1) * 16 + i) & 1)) x[i] = 0xFF800000u;
                    }
#pragma unroll
                    for (int i = 0; i < 16; i += 8) {
                        float t8 = __uint_as_float(x[i]);
#pragma unroll
                        for (int e = 1; e < 8; ++e) t8 = fmaxf(t8, __uint_as_float(x[i + e]));
                        top = fmaxf(top, t8 == -INFINITY ? t8 : t8 * f(c * 2 + i / 8));
                    }
                }
            }
            s.xmax[buf][half][row] = top;
            named_bar_sync(kTeamBar, 32 * kTeamWarps);
            top = fmaxf(top, s.xmax[buf][half ^ 1][row]);
            const float mn = fmaxf(m, top);
            alpha_next = mn == -INFINITY ? 1.f : exp2_fast(m - mn);
            m = mn;
            const float shift = (mn == -INFINITY ? 0.f : mn) - (kF32 ? 14.f : 0.f);
            if (alive && live) {
                float sum = 0.f;
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t x[16];
                    tmem_ld_32x32b_x16(sa + c * 16, x);
                    tmem_wait_ld16(x);
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        float y = fmaf(__uint_as_float(x[i]), f(c * 2 + i / 8), -shift);
                        if (!all && !(mask[c >> 1] >> ((c & 1) * 16 + i) & 1)) y = -INFINITY;
                        x[i] = __float_as_uint(exp2_fast(y));
                    }
#pragma unroll
                    for (int i = 0; i < 16; ++i) sum += __uint_as_float(x[i]);
                    uint32_t hi[8], lo[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float p0 = __uint_as_float(x[2 * i]), p1 = __uint_as_float(x[2 * i + 1]);
                        if constexpr (kF32) split2(p0, p1, hi[i], lo[i]);
                        else hi[i] = pack_bf16(p0, p1);
                    }
                    // in the place of the 16 scores just read
                    tmem_st<8>(sa + c * 16, hi);
                    if constexpr (kF32) tmem_st<8>(sa + c * 16 + 8, lo);
                }
                l = l * alpha_next + sum;
                tmem_wait_st();
                tc_fence_before();
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&s.p_full[buf]);
            if (j > 0) add_pv(w, u - 1, w.t.page(w.j + j - 1), live, pos);
            alpha = alpha_next;
        }
        const Walk done = w;
        const uint32_t last = unit0 + w.n - 1;
        unit0 += w.n;
        more = w.next(a, g);
        if (more) load_query(w);  // every score of the finished segment has been read: its query is free
        add_pv(done, last, done.t.page(done.j + done.n - 1), live, pos);
        s.xsum[half][row] = l;
        named_bar_sync(kTeamBar, 32 * kTeamWarps);
        const float total = s.xsum[0][row] + s.xsum[1][row];
        const bool mine = row < rows;
        if (!alive) {
#pragma unroll
            for (int i = 0; i < 64; ++i) acc[i] = NAN;
        }
        if (done.whole()) {
            if (mine) {
                const float inv = 1.f / total;
                const size_t at = ((size_t)(done.r.lo + R / g) * a.heads + done.head * g + R % g) * kDim + half * 64;
                if constexpr (kF32) {
                    float4* o = reinterpret_cast<float4*>(static_cast<float*>(a.out) + at);
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        o[i] = make_float4(acc[4 * i] * inv, acc[4 * i + 1] * inv, acc[4 * i + 2] * inv, acc[4 * i + 3] * inv);
                } else {
                    uint4* o = reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + at);
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        o[i] = make_uint4(pack_bf16(acc[8 * i] * inv, acc[8 * i + 1] * inv),
                                          pack_bf16(acc[8 * i + 2] * inv, acc[8 * i + 3] * inv),
                                          pack_bf16(acc[8 * i + 4] * inv, acc[8 * i + 5] * inv),
                                          pack_bf16(acc[8 * i + 6] * inv, acc[8 * i + 7] * inv));
                }
            }
        } else {
            const int slot = done.j == 0 ? 1 : 0;
            float* part = slots + ((size_t)blockIdx.x * 2 + slot) * kSlotFloats;
            if (mine) {
#pragma unroll
                for (int i = 0; i < 64; ++i) part[(half * 64 + i) * kTile + row] = acc[i];
                if (half == 0) {
                    part[kDim * kTile + row] = m;
                    part[(kDim + 1) * kTile + row] = total;
                }
            }
            state[slot] = slot == 0 && done.j + done.n == done.t.count ? 2 : 1;
            if (slot == 1) place[0] = done.r.lo, place[1] = done.qt * kTile, place[2] = min(rows, kTile), place[3] = done.head;
        }
    }
    if (threadIdx.x == 0) {
        int* o = info + blockIdx.x * kInfoInts;
        o[0] = state[0], o[1] = state[1];
        for (int i = 0; i < 4; ++i) o[2 + i] = place[i];
    }
}

template <bool kF32>
__global__ void __launch_bounds__(kThreads, 1) chunk_attention_kernel(ChunkArgs a, float* slots, int* info) {
    extern __shared__ unsigned char raw[];
    __shared__ Shared s;
    unsigned char* ring = raw + ((1024 - (smem_addr(raw) & 1023)) & 1023);
    const int warp = threadIdx.x >> 5;
    const int g = a.heads / a.kv_heads;
    if (threadIdx.x == 0) {
        for (int i = 0; i < kStages; ++i) mbar_init(&s.full[i], kLoadWarps), mbar_init(&s.empty[i], 1);
        for (int i = 0; i < 2; ++i) mbar_init(&s.s_full[i], 1), mbar_init(&s.p_full[i], kTeamWarps);
        mbar_init(&s.pv_full, 1), mbar_init(&s.pv_free, kTeamWarps), mbar_init(&s.q_full, kTeamWarps), mbar_init(&s.drain, 1);
        fence_mbar_init();
        s.abort = 0;
    }
    if (warp == kTeamWarps + kLoadWarps) tmem_alloc(&s.tmem, 512);
    tc_fence_before();
    find_run(a, s, reinterpret_cast<long long*>(ring), g);
    tc_fence_after();
    pdl_launch_dependents();
    if (warp < kTeamWarps) team_role<kF32>(a, s, slots, info, g);
    else if (warp < kTeamWarps + kLoadWarps) load_role<kF32>(a, s, ring, g);
    else mma_role<kF32>(a, s, ring, g);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == kTeamWarps + kLoadWarps) tmem_dealloc(s.tmem, 512);
}

// The parts of a tile that was cut: CTA c's slot 1 begins it, slot 0 of the CTAs behind it continues it.
// out = sum_i 2^(m_i - M) sum_i / sum_i 2^(m_i - M) l_i, in the order of the pages. A block joins 16
// columns of one tile.
template <bool kF32>
__global__ void __launch_bounds__(256) chunk_join_kernel(ChunkArgs a, const float* slots, const int* info, int ctas) {
    pdl_wait_prior_grid();
    const int c = blockIdx.x, g = a.heads / a.kv_heads;
    const int* o = info + c * kInfoInts;
    if (o[1] == 0) return;
    const int lo = o[2], r0 = o[3], rows = o[4], head = o[5];
    const int row = threadIdx.x & 127, c0 = blockIdx.y * 16 + (threadIdx.x >> 7) * 8;
    if (row >= rows) return;
    int end = c + 1;  // one behind the last CTA of this tile
    while (end < ctas && info[end * kInfoInts] == 1) ++end;
    end = min(end + 1, ctas);
    float M = -INFINITY;
    for (int d = c; d < end; ++d) M = fmaxf(M, slots[((size_t)d * 2 + (d == c)) * kSlotFloats + kDim * kTile + row]);
    float l = 0.f, x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = 0.f;
    for (int d = c; d < end; ++d) {
        const float* part = slots + ((size_t)d * 2 + (d == c)) * kSlotFloats;
        const float md = part[kDim * kTile + row];
        const float f = md == -INFINITY ? 0.f : exp2_fast(md - M);  // a part in which the row sees nothing
        l = fmaf(part[(kDim + 1) * kTile + row], f, l);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = fmaf(part[(c0 + i) * kTile + row], f, x[i]);
    }
    const float inv = 1.f / l;
    const int R = r0 + row;
    const size_t at = ((size_t)(lo + R / g) * a.heads + head * g + R % g) * kDim + c0;
    if constexpr (kF32) {
        float4* out = reinterpret_cast<float4*>(static_cast<float*>(a.out) + at);
        out[0] = make_float4(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
        out[1] = make_float4(x[4] * inv, x[5] * inv, x[6] * inv, x[7] * inv);
    } else {
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + at) =
            make_uint4(pack_bf16(x[0] * inv, x[1] * inv), pack_bf16(x[2] * inv, x[3] * inv), pack_bf16(x[4] * inv, x[5] * inv),
                       pack_bf16(x[6] * inv, x[7] * inv));
    }
}

template <bool kF32>
cudaError_t launch(const ChunkArgs& a, void* ws, int sms, cudaStream_t st) {
    const size_t smem = (size_t)kStages * (kF32 ? 32768 : 16384) + 1024;
    auto kernel = chunk_attention_kernel<kF32>;
    cudaError_t err = ensure_smem_optin(reinterpret_cast<const void*>(kernel), smem);
    if (err != cudaSuccess) return err;
    int* info = static_cast<int*>(ws);
    float* slots = reinterpret_cast<float*>(static_cast<char*>(ws) + ((size_t)sms * kInfoInts * 4 + 255) / 256 * 256);
    kernel<<<sms, kThreads, smem, st>>>(a, slots, info);
    err = cudaGetLastError();
    if (err != cudaSuccess) return err;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(sms, kDim / 16), cfg.blockDim = dim3(256), cfg.stream = st;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr, cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, chunk_join_kernel<kF32>, a, static_cast<const float*>(slots),
                              static_cast<const int*>(info), sms);
}

}  // namespace

size_t chunk_workspace_bytes(int sms) {
    return ((size_t)sms * kInfoInts * 4 + 255) / 256 * 256 + (size_t)sms * 2 * kSlotFloats * sizeof(float);
}

cudaError_t launch_chunk_attention(const ChunkArgs& a, void* ws, int sms, cudaStream_t st) {
    if (a.B <= 0 || a.T <= 0) return cudaSuccess;
    return a.bf16 ? launch<false>(a, ws, sms, st) : launch<true>(a, ws, sms, st);
}

}  // namespace uocr
