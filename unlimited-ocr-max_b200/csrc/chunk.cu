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
// A CTA: 7 warps load the page's rows into registers (two 32 KB granules in flight), turn them into
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
constexpr int kTeamWarps = 8, kLoadWarps = 7;  // with the issuing warp 16: 128 registers a thread
constexpr int kThreads = 32 * (kTeamWarps + kLoadWarps + 1);
constexpr int kTeamRegs = 112, kLoadRegs = 144;  // of the launch's 16 warps x 128
static_assert(kTeamWarps * kTeamRegs + (kLoadWarps + 1) * kLoadRegs <= 16 * 128, "the split draws on the launch's registers");
// Ring of operands: a page's 128 rows of k or of v, as two blocks of 64 columns [128 rows][128 bytes]; fp32: the
// lo halves behind the hi halves.
template <bool kF32>
constexpr int kStageBytes = kF32 ? 65536 : 32768;
template <bool kF32>
constexpr int kStages = kF32 ? 3 : 6;
constexpr int kMaxStages = 6;
constexpr int kSlotFloats = kTile * (kDim + 2);  // a part: sums [128 columns][128 rows], m [128], l [128]
constexpr int kInfoInts = 8;    // per CTA: states of its two slots, then the tile's place
constexpr uint32_t kTeamBar = 1, kLoadBar = 2;
constexpr float kLog2e = 1.44269504088896341f;

// TMEM columns
constexpr uint32_t kColS = 0, kColPv = 256, kColQ = 384;

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

// A CTA's run: its units, and where they begin.
struct Run {
    int left, b, qt, head, j;
};

// The walk over a CTA's units, a segment (pages of one tile and head) at a time; every warp walks by
// itself, with its walk in shared memory (a register per field would spill).
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
    UOCR_DEV bool begin(const ChunkArgs& a, const Run& s, int g) {
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

struct Shared {
    uint64_t full[kMaxStages], empty[kMaxStages], s_full[2], p_full[2], pv_full, pv_free, q_full, drain;
    uint32_t tmem;
    volatile int abort;
    Run run;
    Walk walk[kThreads / 32], done[kTeamWarps];
    alignas(16) float kscale[8][kPageRows];  // by unit: 1 / scale of each row of k
    float vscale[8];                         // by unit: 1 / scale of v
    alignas(16) uint32_t vbad[8][8];         // by unit: each loading warp's rows of v that are not finite
    float vmax[2][8];
    float xmax[2][2][kTile], xsum[2][kTile];
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
        if (lane == 0) s.run.left = (int)(u1 - u0);
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
                        s.run = Run{s.run.left, b, q0 + lane, (int)(in / count), (int)(in % count)};
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
// D[tmem] (+)= A[tmem] * B[smem], kind::f16, one thread issues. The descriptor's upper word is a constant.
UOCR_DEV void umma_ts_f16(uint32_t d, uint32_t a, uint32_t desc_lo, uint32_t desc_hi, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b64 b, {%2, %3};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t}" ::"r"(d),
        "r"(a), "r"(desc_lo), "r"(desc_hi), "r"(idesc), "r"(accumulate)
        : "memory");
}
UOCR_DEV bool elect_one() {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok));
    return ok != 0;
}
// Shared-memory descriptors, 128-byte swizzle: 8-row groups 1024 bytes apart (the upper word); keys K-major (the
// leading stride is not used), values MN-major, their 64-column blocks 16 KB apart.
constexpr uint32_t kDescHi = (1024 >> 4) | 1u << 14 | 2u << 29;
constexpr uint32_t kDescKeys = 1u << 16, kDescValues = (16384u >> 4) << 16;
UOCR_DEV uint32_t desc_lo(uint32_t addr, uint32_t kind) { return ((addr >> 4) & 0x3FFFu) | kind; }
// M 128, N 128; fp16 or bf16 operands; B from keys (K-major) or values (MN-major: bit 16)
template <bool kF32>
constexpr uint32_t idesc(bool mn) {
    return (1u << 4) | (kF32 ? 0u : (1u << 7) | (1u << 10)) | (mn ? 1u << 16 : 0u) | (128u >> 3) << 17 | (128u >> 4) << 24;
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

// ---- loading warps ----------------------------------------------------------------------------
// Operands in the order in which the tensor core takes them, over a segment: K(0), K(1), V(0), K(2), V(1), ...,
// V(n - 1). A warp takes a run of rows of each, a word (16 bytes of a thread) being one row of fp32 or two of bf16.
template <bool kF32>
struct Rows {
    static constexpr int kElt = kF32 ? 4 : 2;
    static constexpr int kPer = kF32 ? 1 : 2;      // rows of a word
    static constexpr int kWords = kF32 ? 19 : 10;  // words of a thread
    static constexpr int kRun = kWords * kPer;     // rows of a warp (the last one has fewer)
    static_assert(kRun * kLoadWarps >= kPageRows && kRun <= 32, "the warps cover a page");
};

// One operand to load: where this thread's words lie.
struct Op {
    char* pool;          // its first word in the pool's page
    const char* fresh;   // and where it lies among the new rows (rows from `cached` on are read there)
    long long fresh_step;
    int cached, known;   // page rows [0, cached) are in the pool, [cached, known) new, the others not there
    int own0, own1;      // new rows that this tile stores: those whose first query head lies in it
    uint32_t unit;
    bool v;
};

struct Ops {
    Walk& w;
    int jj;
    bool v, more;
    uint32_t unit0;  // units in front of the segment
    uint32_t id;     // the operand's page id, read one operand ahead of its rows
    UOCR_DEV int page() const { return w.t.page(w.j + (v ? jj - 1 : jj)); }
    UOCR_DEV void fetch(const ChunkArgs& a) { id = __ldg(a.lut + (size_t)w.b * a.lut_cols + page()); }
    UOCR_DEV void begin(const ChunkArgs& a, const Shared& s, int g) {
        more = w.begin(a, s.run, g);
        __syncwarp();
        jj = 0, v = false, unit0 = 0;
        if (more) fetch(a);
    }
    UOCR_DEV void next(const ChunkArgs& a, int g) {
        if (!v && jj >= 1) {
            v = true;
        } else {
            ++jj;
            v = jj >= w.n;
            if (jj > w.n) {
                unit0 += w.n;
                __syncwarp();
                more = w.next(a, g);
                __syncwarp();
                jj = 0, v = false;
            }
        }
        if (more) fetch(a);
    }
    template <bool kF32>
    UOCR_DEV Op op(const ChunkArgs& a, int g, int row0, int byte) const {
        using R = Rows<kF32>;
        const size_t row_bytes = (size_t)a.kv_heads * (kDim * R::kElt);
        const int column = w.head * (kDim * R::kElt) + byte, r0 = page() * kPageRows;
        const long long ld = (v ? a.v_ld : a.k_ld) * R::kElt;
        Op o;
        o.pool = static_cast<char*>(a.pool) +
                 ((((size_t)min(id, (uint32_t)(a.pages - 1)) * 2 + v) * a.layers + a.layer) * kPageRows + row0) * row_bytes + column;
        o.cached = w.r.start - r0;
        o.fresh = static_cast<const char*>(v ? a.v : a.k) + (w.r.lo + row0 - o.cached) * ld + column;
        o.fresh_step = ld * R::kPer;
        o.known = min(kPageRows, w.t.last_pos + 1 - r0);
        const bool stored = id < (uint32_t)a.pages;
        o.own0 = w.r.start + (w.qt * kTile + g - 1) / g - r0;
        o.own1 = stored ? w.r.start + min(w.r.n, (w.qt * kTile + kTile + g - 1) / g) - r0 : o.own0;
        o.unit = unit0 + (v ? jj - 1 : jj), o.v = v;
        return o;
    }
};

template <bool kF32>
UOCR_DEV uint4 load_word(const ChunkArgs& a, const Op& o, int row0, int i) {
    using R = Rows<kF32>;
    const int row = row0 + i * R::kPer;
    if (row >= o.known) return make_uint4(0, 0, 0, 0);
    return ldg_nc_v4(row < o.cached ? o.pool + (size_t)i * (a.kv_heads * (kDim * R::kElt * R::kPer))
                                    : o.fresh + i * o.fresh_step);
}

UOCR_DEV bool odd_f32(uint32_t e) { return (e & 0x7F800000u) == 0x7F800000u; }
UOCR_DEV uint32_t odd_bf16(uint32_t e) { return ((e & 0x7F807F80u) + 0x00800080u) & 0x80008000u; }  // per half, its top bit
UOCR_DEV uint32_t top_of(const uint4& x) {
    return max(max(x.x & 0x7FFFFFFFu, x.y & 0x7FFFFFFFu), max(x.z & 0x7FFFFFFFu, x.w & 0x7FFFFFFFu));
}

template <bool kF32>
__device__ void load_role(const ChunkArgs& a, Shared& s, unsigned char* ring, int g) {
    using R = Rows<kF32>;
    const int wc = (threadIdx.x >> 5) - kTeamWarps, lane = threadIdx.x & 31;
    const int row0 = wc * R::kRun + (kF32 ? 0 : lane >> 4), byte = (kF32 ? lane : lane & 15) * 16;
    Ops ops{s.walk[kTeamWarps + wc]};
    ops.begin(a, s, g);
    if (!ops.more) return;
    // an operand's words: as each is turned into its halves, its register takes the next operand's word
    uint4 x[R::kWords];
    Op now = ops.template op<kF32>(a, g, row0, byte);
#pragma unroll
    for (int i = 0; i < R::kWords; ++i) x[i] = load_word<kF32>(a, now, row0, i);
    uint32_t stage = 0, phase = 0;
    for (;;) {
        ops.next(a, g);
        const bool more = ops.more;
        Op ahead = now;
        if (more) ahead = ops.template op<kF32>(a, g, row0, byte);
        else ahead.known = 0;
        if (now.own0 < kPageRows && now.own1 > now.own0) {
#pragma unroll
            for (int i = 0; i < R::kWords; ++i) {
                const int row = row0 + i * R::kPer;
                if (row >= now.own0 && row < min(now.own1, kPageRows))
                    *reinterpret_cast<uint4*>(now.pool + (size_t)i * (a.kv_heads * (kDim * R::kElt * R::kPer))) = x[i];
            }
        }
        const uint32_t ub = now.unit & 7;
        float up = 1.f;
        if (now.v) {
            // values that are not finite leave the operand; fp32: one scale for the page, whose rows are summed over
            uint32_t top = 0, bad = 0;
#pragma unroll
            for (int i = 0; i < R::kWords; ++i)
                top = kF32 ? max(top, top_of(x[i])) : top | odd_bf16(x[i].x) | odd_bf16(x[i].y) | odd_bf16(x[i].z) | odd_bf16(x[i].w);
            if (kF32) top = __reduce_max_sync(0xffffffffu, top);
            if (kF32 ? top >= 0x7F800000u : __any_sync(0xffffffffu, top != 0)) {  // rare
                top = 0;
#pragma unroll
                for (int i = 0; i < R::kWords; ++i) {
                    bool row_bad = false;
                    auto drop = [&](uint32_t& e) {
                        if (kF32) {
                            if (odd_f32(e)) e = 0, row_bad = true;
                        } else {
                            const uint32_t o = odd_bf16(e);
                            if (o & 0x00008000u) e &= 0xFFFF0000u;
                            if (o & 0x80000000u) e &= 0x0000FFFFu;
                            row_bad |= o != 0;
                        }
                    };
                    drop(x[i].x), drop(x[i].y), drop(x[i].z), drop(x[i].w);
                    const uint32_t who = __ballot_sync(0xffffffffu, row_bad);
                    if (kF32) bad |= (who ? 1u : 0u) << i;
                    else bad |= ((who & 0xFFFFu ? 1u : 0u) | (who >> 16 ? 2u : 0u)) << (2 * i);
                    if (kF32) top = max(top, top_of(x[i]));
                }
                if (kF32) top = __reduce_max_sync(0xffffffffu, top);
            }
            if (lane == 0) s.vbad[ub][wc] = bad;
            if constexpr (kF32) {
                if (lane == 0) s.vmax[now.unit & 1][wc] = __uint_as_float(top);
                named_bar_sync(kLoadBar, 32 * kLoadWarps);
                top = __reduce_max_sync(0xffffffffu, __float_as_uint(s.vmax[now.unit & 1][lane % kLoadWarps]));
                if (wc == 0 && lane == 0) s.vscale[ub] = scale_down(top);
                up = scale_up(top);
            }
        }
        if (!wait(s, &s.empty[stage], phase ^ 1)) return;
        const uint32_t base = smem_addr(ring) + stage * kStageBytes<kF32>;
        uint32_t my_top = 0;  // lane i: the largest magnitude of row i of k
#pragma unroll
        for (int i = 0; i < R::kWords; ++i) {
            const int row = row0 + i * R::kPer;
            if constexpr (kF32) {
                if (!now.v) {
                    uint32_t top = __reduce_max_sync(0xffffffffu, top_of(x[i]));
                    if (top >= 0x7F800000u) {  // rare: its scores become NaN; it sets no scale
                        uint32_t m = 0;
                        auto mark = [&](uint32_t& e) {
                            if (odd_f32(e)) e = 0x7FFFFFFFu;
                            else m = max(m, e & 0x7FFFFFFFu);
                        };
                        mark(x[i].x), mark(x[i].y), mark(x[i].z), mark(x[i].w);
                        top = __reduce_max_sync(0xffffffffu, m);
                    }
                    if (lane == i) my_top = top;
                    up = scale_up(top);
                }
                uint2 hi, lo;
                split2(__uint_as_float(x[i].x) * up, __uint_as_float(x[i].y) * up, hi.x, lo.x);
                split2(__uint_as_float(x[i].z) * up, __uint_as_float(x[i].w) * up, hi.y, lo.y);
                x[i] = load_word<kF32>(a, ahead, row0, i);
                // 8 bytes (4 columns) of a block's 128-byte row, whose 16-byte chunks are swizzled by the row
                const uint32_t at = base + (lane >> 4) * 16384 + row * 128 + ((((lane & 15) >> 1) ^ (row & 7)) << 4) + (lane & 1) * 8;
                if (row < kPageRows) {
                    asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(at), "r"(hi.x), "r"(hi.y) : "memory");
                    asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(at + 32768), "r"(lo.x), "r"(lo.y) : "memory");
                }
            } else {
                const uint32_t at = base + ((lane >> 3) & 1) * 16384 + row * 128 + (((lane & 7) ^ (row & 7)) << 4);
                if (row < kPageRows)
                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(x[i].x), "r"(x[i].y), "r"(x[i].z),
                                 "r"(x[i].w)
                                 : "memory");
                x[i] = load_word<kF32>(a, ahead, row0, i);
            }
        }
        if (kF32 && !now.v && lane < R::kRun && wc * R::kRun + lane < kPageRows)
            s.kscale[ub][wc * R::kRun + lane] = scale_down(my_top);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.full[stage]);
        if (++stage == kStages<kF32>) stage = 0, phase ^= 1;
        if (!more) return;
        now = ahead;
    }
}

// ---- the issuing warp -------------------------------------------------------------------------
template <bool kF32>
__device__ void mma_role(const ChunkArgs& a, Shared& s, unsigned char* ring, int g) {
    const uint32_t tmem = s.tmem, base = smem_addr(ring);
    uint32_t stage = 0, phase = 0, unit0 = 0, seg = 0;
    Walk& w = s.walk[kTeamWarps + kLoadWarps];
    // one operand: its MMAs issued (D = sum over the products of A's halves and the operand's, 16 of the summed
    // dimension at a time), its stage given back, the result announced
    auto product = [&](uint32_t d, uint32_t ta, uint32_t a_step, uint32_t a_lo, uint32_t kind, uint32_t b_step2, uint32_t b_step8,
                       uint32_t id, uint64_t* done) {
        if (!wait(s, &s.full[stage], phase)) return false;
        tc_fence_after();
        if (elect_one()) {
            const uint32_t b = desc_lo(base + stage * kStageBytes<kF32>, kind);
#pragma unroll
            for (int p = kF32 ? 0 : 2; p < 3; ++p) {  // lo x hi, hi x lo, hi x hi
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    umma_ts_f16(d, ta + i * a_step + (p == 0 ? a_lo : 0),
                                b + (i & 3) * b_step2 + (i >> 2) * b_step8 + (p == 1 ? 32768 >> 4 : 0), kDescHi, id,
                                p != (kF32 ? 0 : 2) || i != 0);
            }
            umma_commit(&s.empty[stage]);
            umma_commit(done);
        }
        __syncwarp();
        if (++stage == kStages<kF32>) stage = 0, phase ^= 1;
        return true;
    };
    auto run = [&] {
        auto next = [&](bool first) {
            __syncwarp();
            const bool more = first ? w.begin(a, s.run, g) : w.next(a, g);
            __syncwarp();
            return more;
        };
        for (bool more = next(true); more; more = next(false), ++seg) {
            if (!wait(s, &s.q_full, seg & 1)) return;
            tc_fence_after();
            const int n = w.n;
            for (int jj = 0; jj <= n; ++jj) {
                if (jj < n) {  // S = Q K^T: 16 dimensions of K are 32 bytes of a row, 64 a block
                    const uint32_t u = unit0 + jj;
                    if (!product(tmem + kColS + (u & 1) * 128, tmem + kColQ, 8, 64, kDescKeys, 32 >> 4, 16384 >> 4,
                                 idesc<kF32>(false), &s.s_full[u & 1]))
                        return;
                }
                if (jj >= 1) {  // P V: 16 rows of V are 2048 bytes of both its blocks
                    const uint32_t u = unit0 + jj - 1;
                    if (!wait(s, &s.p_full[u & 1], (u >> 1) & 1) || !wait(s, &s.pv_free, (u & 1) ^ 1)) return;
                    if (!product(tmem + kColPv, tmem + kColS + (u & 1) * 128, 16, 8, kDescValues, 2048 >> 4, 8192 >> 4,
                                 idesc<kF32>(true), &s.pv_full))
                        return;
                }
            }
            unit0 += n;
        }
    };
    run();
    // every MMA of this CTA has finished before its TMEM is freed
    if (elect_one()) umma_commit(&s.drain);
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
    const uint32_t id = __ldg(a.lut + (size_t)w.b * a.lut_cols + t);
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
            const float f = kF32 ? s.vscale[u & 7] : 1.f;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                uint32_t x[16];
                tmem_ld_32x32b_x16(lanes + kColPv + half * 64 + c * 16, x);
                tmem_wait_ld16(x);
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[c * 16 + i] = fmaf(acc[c * 16 + i], alpha, __uint_as_float(x[i]) * f);
            }
            const uint4* vb = reinterpret_cast<const uint4*>(s.vbad[u & 7]);
            if (vb[0].x | vb[0].y | vb[0].z | vb[0].w | vb[1].x | vb[1].y | vb[1].z) {
                for (int q = 0; q < kPageRows; ++q) {
                    if (!(s.vbad[u & 7][q / Rows<kF32>::kRun] >> (q % Rows<kF32>::kRun) & 1)) continue;
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

    Walk& w = s.walk[warp];
    Walk& done = s.done[warp];
    bool more = w.begin(a, s.run, g);
    __syncwarp();
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
            // 1 / scale of a column's keys
            const float* ks = &s.kscale[u & 7][half * 64];
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
                    for (int i = 0; i < 16; i += 4) {
                        const float4 k4 = kF32 ? *reinterpret_cast<const float4*>(ks + c * 16 + i) : make_float4(1.f, 1.f, 1.f, 1.f);
                        top = fmaxf(fmaxf(top, __uint_as_float(x[i]) * k4.x), __uint_as_float(x[i + 1]) * k4.y);
                        top = fmaxf(fmaxf(top, __uint_as_float(x[i + 2]) * k4.z), __uint_as_float(x[i + 3]) * k4.w);
                    }
                }
            }
            top *= qscale;  // -inf * 0 (nothing seen, a query of zeros): NaN, which is no maximum
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
                    for (int i = 0; i < 16; i += 4) {
                        const float4 k4 = kF32 ? *reinterpret_cast<const float4*>(ks + c * 16 + i) : make_float4(1.f, 1.f, 1.f, 1.f);
                        const float kk[4] = {k4.x, k4.y, k4.z, k4.w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            float y = __uint_as_float(x[i + e]);
                            y = fmaf(kF32 ? y * kk[e] : y, qscale, -shift);
                            if (!all && !(mask[c >> 1] >> ((c & 1) * 16 + i + e) & 1)) y = -INFINITY;
                            x[i + e] = __float_as_uint(exp2_fast(y));
                        }
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
        const uint32_t last = unit0 + w.n - 1;
        unit0 += w.n;
        done = w;
        __syncwarp();
        more = w.next(a, g);
        __syncwarp();
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
        for (int i = 0; i < kMaxStages; ++i) mbar_init(&s.full[i], kLoadWarps), mbar_init(&s.empty[i], 1);
        for (int i = 0; i < 2; ++i) mbar_init(&s.s_full[i], 1), mbar_init(&s.p_full[i], kTeamWarps);
        mbar_init(&s.pv_full, 1), mbar_init(&s.pv_free, kTeamWarps), mbar_init(&s.q_full, kTeamWarps), mbar_init(&s.drain, 1);
        fence_mbar_init();
        s.abort = 0;
        for (int i = 0; i < 8; ++i) s.vbad[i][7] = 0;
    }
    if (warp == kTeamWarps + kLoadWarps) tmem_alloc(&s.tmem, 512);
    tc_fence_before();
    find_run(a, s, reinterpret_cast<long long*>(ring), g);
    tc_fence_after();
    pdl_launch_dependents();
    if (warp < kTeamWarps) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kTeamRegs));
        team_role<kF32>(a, s, slots, info, g);
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kLoadRegs));
        if (warp < kTeamWarps + kLoadWarps) load_role<kF32>(a, s, ring, g);
        else mma_role<kF32>(a, s, ring, g);
    }
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
    const size_t smem = (size_t)kStages<kF32> * kStageBytes<kF32> + 1024;
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
