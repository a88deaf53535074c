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
// straight to out; the parts of one that was cut go to the workspace as (m, l, sum) and a last launch
// joins them in the order of the pages. Every CTA finds its run from the lengths on the device.
//
// Three launches, each begun while the one in front of it ends:
// 1. chunk_operands_kernel turns every visible page's k and v and every query tile into the tensor core's operands, in
//    the workspace, and stores the new rows in the pool. Each row is converted once, however many query tiles read
//    it (8192 fp32 tokens of 10 heads: 1.05 ms in a first version, 1.72 with every tile's CTA converting them for itself;
//    0.46 ms now).
// 2. chunk_attention_kernel: one warp copies operands into a ring in shared memory (bulk copies), one issues
//    tcgen05.mma, 8 warps do the softmax, two threads per query row. The query operand and the weights P are read by
//    the tensor core from TMEM, so shared memory carries each key and value once:
//      S = Q K^T (TMEM, two buffers) -> softmax warps -> P (in S's place) -> P V (TMEM) -> added to the
//      sums in registers, in fp32 with round-to-nearest, after each page (bf16: after 16).
// 3. chunk_join_kernel.
//
// fp32: a product of fp32 rows is three products of fp16 halves, hi x hi + hi x lo + lo x hi, where
// x = hi + lo to 2^-22 of x: a query row, and a row of k or v (all of a page's rows where they are of like size), are
// scaled by a power of two that brings their largest element to [2^14, 2^15), and a row's weights on a page to at most
// 2^14, so the halves keep their bits over fp16's exponent range. The small products go into the accumulator
// first: the tensor core's additions truncate, and only the last 8 then round at the result's full size. bf16: one
// product; the weights are rounded to bf16, as the tensor core takes both operands in one type (0.0022 of the result off
// against 64 bits, of which rounding the result itself is 0.0017; halves of the weights would cost a second product).
// Values that are not finite are kept out of the V operand (0 x inf would reach rows that do not see
// them) and added to the rows that do see them; elements of fp32 keys that are not finite are kept out of the K operand, and
// make the rows' scores by themselves. A hidden row has the weight 0, and its size takes no part either: where a page's rows of
// values are not within 2^10 of one another, each has a scale of its own, which goes into its weight (8192 tokens with
// such pages throughout: 541 us against 459).
//
// Measured (B200). fp32, 8192 tokens of 10 heads: operands 64 us (HBM, 5.2 TB/s), attention 380 us (1.38 PFLOP/s of fp16
// products, 0.82 of a cuBLAS bf16 burst; a page takes 3900 cycles, of which the tensor core works 3.1 k: the rest is the softmax
// warps' exponentials, rounding and waits), joining 5 us; long loops of calls run into the power limit
// (530 us a call). bf16, requests of 2048 and 767 tokens over 6000 and 2249
// rows, 32 heads over 8: operands 27 us, attention 337 us (3000 cycles a page, the tensor core 1024: the
// softmax warps bound it, 1024 for the exponentials alone). Taken and dropped: four threads a row (spills; 4700 cycles),
// k and v of a page converted by CTAs of their own (no faster), exponentials and rounding alternated (no change).
#include "chunk.cuh"

namespace uocr {
namespace {

constexpr int kTile = 128;      // (token, head) rows of a query tile
constexpr int kLead = 3;        // what a tile costs beside its pages (2 to 4 measure alike)
constexpr int kTeamWarps = 8;   // softmax; then a warpgroup: the issuing warp, the copying warp and two idle ones
constexpr int kThreads = 32 * (kTeamWarps + 4);
constexpr int kLaunchRegs = 168, kTeamRegs = 216, kOtherRegs = 72;  // a thread
static_assert(kTeamWarps * kTeamRegs + 4 * kOtherRegs <= (kTeamWarps + 4) * kLaunchRegs, "a split of the launch's registers");
// An operand: a page's 128 rows of k or of v of one head, as two blocks of 64 columns [128 rows][128 bytes]; fp32:
// the lo halves behind the hi halves.
template <bool kF32>
constexpr int kOperandBytes = kF32 ? 65536 : 32768;
template <bool kF32>
constexpr int kStages = kF32 ? 3 : 6;  // of operands in shared memory
constexpr int kMaxStages = 6;
constexpr uint32_t kTeamBar = 1, kPairBar = 2;  // all softmax warps; the two warps of 32 rows (kPairBar + 0..3)

// TMEM columns
constexpr uint32_t kColS = 0, kColPv = 256, kColQ = 384;

// Beside a page's operands: 1 / scale of each row of k, and of all of them where they share one (else 0); the binary
// logarithms of 1 / scale of each row of v and of all of them (kUnlike: they do not share one); are there rows of v or k that
// are not finite (kBad), and which. bf16 has values_are and bad only, and there: are there finite values of 2^65 or more (kLarge)?
constexpr uint32_t kUnlike = 1, kLarge = 2, kBad = 4;
struct alignas(16) PageMeta {
    float keys[kPageRows], values_log2[kPageRows];
    float all_keys, all_values_log2;
    uint32_t values_are, keys_are;
    uint32_t bad[4], bad_keys[4];
};

// The operands of a pass, made by the first launch. Keys and values: page p of request b and head h (of the pass)
// at index (b * lut_cols + p) * pass_heads + h, k, then v. Queries: tile t of request b at index
// (query_base(b) + t) * pass_heads + h, 16 bytes of row r at (group * 128 + r) * 16 bytes as TMEM takes them (fp32: hi
// halves in groups 0 to 15, lo halves in 16 to 31; bf16: 16 groups), and each row's 1 / scale times the
// softmax's factor.
struct Images {
    unsigned char* operands;
    PageMeta* meta;
    unsigned char* queries;
    float* qscale;
};
template <bool kF32>
constexpr int kQueryBytes = kTile * kDim * (kF32 ? 4 : 2);
// Tiles of the requests in front of b fit below: floor(x + y) + 1 >= floor(x) + ceil(y).
UOCR_DEV int query_base(const Request& r, int b, int g) { return r.lo * g / kTile + b; }

struct Shared {
    PageMeta meta[8];  // by unit
    uint64_t full[kMaxStages], empty[kMaxStages], s_full[2], p_full[2], pv_full[2], pv_free, q_full, drain;
    uint32_t tmem;
    volatile int abort;
    Run run;
    Walk walk[kThreads / 32], now[kTeamWarps];
    float xmax[2][2][kTile], xsum[2][kTile], xref[2][kTile];
};

// Has the phase of `parity` completed? (No suspension, unlike try_wait.)
UOCR_DEV bool mbar_test(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok)
                 : "r"(smem_addr(bar)), "r"(parity)
                 : "memory");
    return ok != 0;
}
// A whole warp's bounded wait.
UOCR_DEV bool wait(Shared& s, uint64_t* bar, uint32_t parity) {
    if (__all_sync(0xffffffffu, mbar_test(bar, parity))) return true;
    if (mbar_wait_warp(bar, parity, &s.abort, nullptr)) return true;
    s.abort = 1;
    return false;
}

// ---- tensor-core operands ---------------------------------------------------------------------
// D[tmem] (+)= A[tmem] * B[smem], kind::f16, where `me` (one lane of a converged warp: the operands stay in uniform
// registers, from which the tensor core takes them). The descriptor's upper word is a constant.
UOCR_DEV void umma_ts_f16(uint32_t me, uint32_t d, uint32_t a, uint32_t desc_lo, uint32_t desc_hi, uint32_t idesc,
                          uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t.reg .b64 b;\n\tsetp.ne.b32 e, %6, 0;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b64 b, {%2, %3};\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t}" ::"r"(d),
        "r"(a), "r"(desc_lo), "r"(desc_hi), "r"(idesc), "r"(accumulate), "r"(me)
        : "memory");
}
UOCR_DEV void umma_commit_if(uint32_t me, uint64_t* bar) {
    asm volatile(
        "{\n\t.reg .pred e;\n\tsetp.ne.b32 e, %1, 0;\n\t"
        "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_addr(bar)),
        "r"(me)
        : "memory");
}
UOCR_DEV uint32_t elect_one() {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok));
    return ok;
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
// 64 columns into x, complete on return (the waits mark x as written by them: no use moves in front of them).
UOCR_DEV void tmem_ld64(uint32_t addr, uint32_t (&x)[64]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]), "=r"(x[4]), "=r"(x[5]), "=r"(x[6]), "=r"(x[7]), "=r"(x[8]), "=r"(x[9]), "=r"(x[10]), "=r"(x[11]), "=r"(x[12]), "=r"(x[13]), "=r"(x[14]), "=r"(x[15]), "=r"(x[16]), "=r"(x[17]), "=r"(x[18]), "=r"(x[19]), "=r"(x[20]), "=r"(x[21]), "=r"(x[22]), "=r"(x[23]), "=r"(x[24]), "=r"(x[25]), "=r"(x[26]), "=r"(x[27]), "=r"(x[28]), "=r"(x[29]), "=r"(x[30]), "=r"(x[31])
                 : "r"(addr + 0));
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : "=r"(x[32]), "=r"(x[33]), "=r"(x[34]), "=r"(x[35]), "=r"(x[36]), "=r"(x[37]), "=r"(x[38]), "=r"(x[39]), "=r"(x[40]), "=r"(x[41]), "=r"(x[42]), "=r"(x[43]), "=r"(x[44]), "=r"(x[45]), "=r"(x[46]), "=r"(x[47]), "=r"(x[48]), "=r"(x[49]), "=r"(x[50]), "=r"(x[51]), "=r"(x[52]), "=r"(x[53]), "=r"(x[54]), "=r"(x[55]), "=r"(x[56]), "=r"(x[57]), "=r"(x[58]), "=r"(x[59]), "=r"(x[60]), "=r"(x[61]), "=r"(x[62]), "=r"(x[63])
                 : "r"(addr + 32));
    asm volatile("tcgen05.wait::ld.sync.aligned;" : "+r"(x[0]), "+r"(x[1]), "+r"(x[2]), "+r"(x[3]), "+r"(x[4]), "+r"(x[5]), "+r"(x[6]), "+r"(x[7]), "+r"(x[8]), "+r"(x[9]), "+r"(x[10]), "+r"(x[11]), "+r"(x[12]), "+r"(x[13]), "+r"(x[14]), "+r"(x[15]) : : "memory");
    asm volatile("tcgen05.wait::ld.sync.aligned;" : "+r"(x[16]), "+r"(x[17]), "+r"(x[18]), "+r"(x[19]), "+r"(x[20]), "+r"(x[21]), "+r"(x[22]), "+r"(x[23]), "+r"(x[24]), "+r"(x[25]), "+r"(x[26]), "+r"(x[27]), "+r"(x[28]), "+r"(x[29]), "+r"(x[30]), "+r"(x[31]) : : "memory");
    asm volatile("tcgen05.wait::ld.sync.aligned;" : "+r"(x[32]), "+r"(x[33]), "+r"(x[34]), "+r"(x[35]), "+r"(x[36]), "+r"(x[37]), "+r"(x[38]), "+r"(x[39]), "+r"(x[40]), "+r"(x[41]), "+r"(x[42]), "+r"(x[43]), "+r"(x[44]), "+r"(x[45]), "+r"(x[46]), "+r"(x[47]) : : "memory");
    asm volatile("tcgen05.wait::ld.sync.aligned;" : "+r"(x[48]), "+r"(x[49]), "+r"(x[50]), "+r"(x[51]), "+r"(x[52]), "+r"(x[53]), "+r"(x[54]), "+r"(x[55]), "+r"(x[56]), "+r"(x[57]), "+r"(x[58]), "+r"(x[59]), "+r"(x[60]), "+r"(x[61]), "+r"(x[62]), "+r"(x[63]) : : "memory");
}
UOCR_DEV void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// two values as fp16 halves: hi takes the upper 11 bits (exactly), lo the rest (rounded to 11 bits)
UOCR_DEV void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
    const uint32_t xh = __float_as_uint(x) & 0xFFFFE000u, yh = __float_as_uint(y) & 0xFFFFE000u;
    uint32_t xl, yl;
    unpair(add2(pair(x, y), pair(xh ^ 0x80000000u, yh ^ 0x80000000u)), xl, yl);
    hi = pack_f16(__uint_as_float(xh), __uint_as_float(yh));
    lo = pack_f16(__uint_as_float(xl), __uint_as_float(yl));
}
// 2^(14 - e) and its inverse for the largest magnitude's bits (e its exponent, from -112 up: below that
// the values are smaller than 2^14 after scaling, which costs them bits they do not have)
UOCR_DEV float scale_up(uint32_t bits) { return __uint_as_float((268u - max(bits >> 23, 15u)) << 23); }
UOCR_DEV float scale_down(uint32_t bits) { return __uint_as_float((max(bits >> 23, 15u) - 14u) << 23); }
UOCR_DEV float scale_down_log2(uint32_t bits) { return (float)((int)max(bits >> 23, 15u) - 141); }

// ---- the first launch: rows into operands ------------------------------------------------------
UOCR_DEV bool odd_f32(uint32_t e) { return (e & 0x7F800000u) == 0x7F800000u; }
UOCR_DEV uint32_t large_bf16(uint32_t e) { return e & e << 1 & 0x40004000u; }  // per half: 2^65 or more, odd ones among them
UOCR_DEV uint32_t odd_bf16(uint32_t e) { return ((e & 0x7F807F80u) + 0x00800080u) & 0x80008000u; }  // per half, its top bit
UOCR_DEV uint32_t top_of(const uint4& x) {
    return max(max(x.x & 0x7FFFFFFFu, x.y & 0x7FFFFFFFu), max(x.z & 0x7FFFFFFFu, x.w & 0x7FFFFFFFu));
}

// A query tile of head `head` (of the pass): 128 rows of q. A warp takes 16 rows.
template <bool kF32>
UOCR_DEV void query_operand(const ChunkArgs& a, const Images& im, int f, int head) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = a.heads / a.kv_heads;
    int b = 0;
    for (int hi = a.B - 1; b < hi;) {  // the last request whose tiles begin at f or below
        const int mid = (b + hi + 1) / 2;
        if (query_base(request_at(a, mid), mid, g) <= f) b = mid; else hi = mid - 1;
    }
    const Request r = request_at(a, b);
    const int qt = f - query_base(r, b, g), rows = r.n * g - qt * kTile;
    if (qt < 0 || rows <= 0) return;
    const size_t index = (size_t)f * a.pass_heads + head;
    unsigned char* out = im.queries + index * kQueryBytes<kF32>;
    const float factor = fabsf(a.scale) * kLog2e;  // the scale's sign goes into the operand
    constexpr int kElt = kF32 ? 4 : 2, kPer = kF32 ? 1 : 2, kWords = 16 / kPer;
    uint4 x[kWords];
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
        const int row = warp * 16 + i * kPer + (kF32 ? 0 : lane >> 4), R = qt * kTile + row;
        x[i] = make_uint4(0, 0, 0, 0);
        if (row < rows)
            x[i] = ldg_nc_v4(static_cast<const char*>(a.q) +
                             ((r.lo + token_of(a, R)) * a.q_ld + (size_t)((a.head0 + head) * g + R - token_of(a, R) * g) * kDim) * kElt +
                             (kF32 ? lane : lane & 15) * 16);
    }
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
        const int row = warp * 16 + i * kPer + (kF32 ? 0 : lane >> 4);
        if constexpr (kF32) {
            auto finite = [](uint32_t e) { return (e & 0x7FFFFFFFu) < 0x7F800000u ? e & 0x7FFFFFFFu : 0u; };
            const uint32_t top = __reduce_max_sync(0xffffffffu, max(max(finite(x[i].x), finite(x[i].y)), max(finite(x[i].z), finite(x[i].w))));
            const float up = a.scale < 0.f ? -scale_up(top) : scale_up(top);
            uint2 hi, lo;
            split2(__uint_as_float(x[i].x) * up, __uint_as_float(x[i].y) * up, hi.x, lo.x);
            split2(__uint_as_float(x[i].z) * up, __uint_as_float(x[i].w) * up, hi.y, lo.y);
            unsigned char* at = out + ((lane >> 1) * kTile + row) * 16 + (lane & 1) * 8;
            *reinterpret_cast<uint2*>(at) = hi;
            *reinterpret_cast<uint2*>(at + 16 * kTile * 16) = lo;
            // never 0: a hidden score is -inf times this
            if (lane == 0) im.qscale[index * kTile + row] = fmaxf(scale_down(top) * factor, 1e-37f);
        } else {
            const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u;
            *reinterpret_cast<uint4*>(out + ((lane & 15) * kTile + row) * 16) =
                make_uint4(x[i].x ^ flip, x[i].y ^ flip, x[i].z ^ flip, x[i].w ^ flip);
            if ((lane & 15) == 0) im.qscale[index * kTile + row] = fmaxf(factor, 1e-37f);
        }
    }
}

// A CTA per page (of a request's table) and head, then per query tile and head. Pages: their rows of k and v become
// operands, and their new rows are stored in the pool. A warp takes 16 rows; a word (16 bytes of a thread) is one
// row of fp32 or two of bf16; 16 words of each thread are in flight, 128 KB an SM. Bound: HBM: 64 pages of 10 heads of fp32
// (84 MB read, 84 MB written) in 33 us after its launch, 5.1 TB/s; no call reads less, and the writes mostly stay in L2.
template <bool kF32>
__global__ void __launch_bounds__(256, 2) chunk_operands_kernel(ChunkArgs a, Images im) {
    pdl_launch_dependents();
    constexpr int kElt = kF32 ? 4 : 2, kPer = kF32 ? 1 : 2, kWords = 16 / kPer;
    __shared__ uint32_t tops[8], bads[8];
    if (blockIdx.x >= (unsigned)(a.B * a.lut_cols)) {
        query_operand<kF32>(a, im, blockIdx.x - a.B * a.lut_cols, blockIdx.y);
        return;
    }
    const int b = blockIdx.x / a.lut_cols, page = blockIdx.x % a.lut_cols, head = a.head0 + blockIdx.y;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = a.heads / a.kv_heads;
    const Request r = request_at(a, b);
    if (r.n == 0) return;
    const Tile first = tile_at(a, r, 0, kTile);
    const int last = r.start + r.n - 1, r0 = page * kPageRows;
    if (r0 > last || (page < first.tail_page && r0 >= r.prefix)) return;  // no token of the request sees it
    const uint32_t id = __ldg(a.lut + (size_t)b * a.lut_cols + page);
    const size_t row_bytes = (size_t)a.kv_heads * (kDim * kElt);
    const size_t index = ((size_t)b * a.lut_cols + page) * a.pass_heads + blockIdx.y;
    const int row0 = warp * 16 + (kF32 ? 0 : lane >> 4), byte = (kF32 ? lane : lane & 15) * 16;
    const int cached = r.start - r0, known = min(kPageRows, last + 1 - r0);
    PageMeta& meta = im.meta[index];
    for (int v = 0; v < 2; ++v) {  // rows pass L2 by (read and stored once), where the operands should stay: 8 x 512 fp32 79.4 -> 78.3 us
        char* pool = static_cast<char*>(a.pool) +
                     ((((size_t)min(id, (uint32_t)(a.pages - 1)) * 2 + v) * a.layers + a.layer) * kPageRows) * row_bytes +
                     (size_t)head * (kDim * kElt) + byte;
        const long long ld = (v ? a.v_ld : a.k_ld) * kElt;
        const char* fresh = static_cast<const char*>(v ? a.v : a.k) + (r.lo - cached) * ld + head * (kDim * kElt) + byte;
        uint4 x[kWords];
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            const int row = row0 + i * kPer;
            x[i] = make_uint4(0, 0, 0, 0);
            if (row < known) x[i] = __ldcs(reinterpret_cast<const uint4*>(row < cached ? pool + row * row_bytes : fresh + row * ld));
        }
        if (known > cached && id < (uint32_t)a.pages) {
#pragma unroll
            for (int i = 0; i < kWords; ++i) {
                const int row = row0 + i * kPer;
                if (row >= cached && row < known) __stcs(reinterpret_cast<uint4*>(pool + row * row_bytes), x[i]);
            }
        }
        auto any_bad = [&] {
            uint32_t any = 0;
            for (int i = 0; i < 8; ++i) any |= bads[i];
            return any ? kBad : 0u;
        };
        uint32_t my_top = 0;  // fp32: lane i has the largest magnitude of row i
        if constexpr (kF32) {
            uint32_t bad = 0;
#pragma unroll
            for (int i = 0; i < kWords; ++i) {
                uint32_t top = __reduce_max_sync(0xffffffffu, top_of(x[i]));
                if (top >= 0x7F800000u) {  // rare. Elements that are not finite leave the operand and set no scale
                    uint32_t m = 0;
                    auto mark = [&](uint32_t& e) {
                        if (odd_f32(e)) e = 0;
                        else m = max(m, e & 0x7FFFFFFFu);
                    };
                    mark(x[i].x), mark(x[i].y), mark(x[i].z), mark(x[i].w);
                    top = __reduce_max_sync(0xffffffffu, m);
                    bad |= 1u << i;
                }
                if (lane == i) my_top = top;
            }
            uint32_t page_top = __reduce_max_sync(0xffffffffu, my_top);
            __syncthreads();  // tops may still be read
            if (lane == 0) tops[warp] = page_top, bads[warp] = bad;
            __syncthreads();
            page_top = __reduce_max_sync(0xffffffffu, tops[lane & 7]);
            // A row within 2^10 of the page's largest can take the page's scale (its halves still hold 2^-29 of it). A key
            // that is not has its own. Values are summed over the rows: one scale for all of them, or each its
            // own, for the largest may be one that a token does not see.
            const bool near = my_top == 0 || (my_top >> 23) + 10 >= page_top >> 23;
            const bool all = __syncthreads_and(near || lane >= 16);
            if (v ? all : near) my_top = page_top;
            if (lane < 16) (v ? meta.values_log2 : meta.keys)[warp * 16 + lane] = v ? scale_down_log2(my_top) : scale_down(my_top);
            if (threadIdx.x == 0) {
                if (v) {
                    meta.all_values_log2 = all ? scale_down_log2(page_top) : 0.f;
                    meta.values_are = (all ? 0 : kUnlike) | any_bad();
                } else {
                    meta.all_keys = all ? scale_down(page_top) : 0.f;
                    meta.keys_are = any_bad();
                }
            }
        } else if (v) {
            // values that are not finite leave the operand
            uint32_t large = 0, bad = 0;
            auto look = [&] {
                large = 0;
#pragma unroll
                for (int i = 0; i < kWords; ++i) large |= large_bf16(x[i].x) | large_bf16(x[i].y) | large_bf16(x[i].z) | large_bf16(x[i].w);
            };
            look();
            if (__any_sync(0xffffffffu, large != 0)) {  // rare
#pragma unroll
                for (int i = 0; i < kWords; ++i) {
                    bool row_bad = false;
                    auto drop = [&](uint32_t& e) {
                        const uint32_t o = odd_bf16(e);
                        if (o & 0x00008000u) e &= 0xFFFF0000u;
                        if (o & 0x80000000u) e &= 0x0000FFFFu;
                        row_bad |= o != 0;
                    };
                    drop(x[i].x), drop(x[i].y), drop(x[i].z), drop(x[i].w);
                    const uint32_t who = __ballot_sync(0xffffffffu, row_bad);
                    bad |= ((who & 0xFFFFu ? 1u : 0u) | (who >> 16 ? 2u : 0u)) << (2 * i);
                }
                look();
            }
            if (lane == 0) bads[warp] = bad;
            large = __syncthreads_or(large != 0);
            if (threadIdx.x == 0) meta.values_are = (large ? kLarge : 0) | any_bad();
        }
        if ((kF32 || v) && threadIdx.x < 4) (v ? meta.bad : meta.bad_keys)[threadIdx.x] = bads[2 * threadIdx.x] | bads[2 * threadIdx.x + 1] << 16;
        unsigned char* out = im.operands + (index * 2 + v) * kOperandBytes<kF32>;
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            const int row = row0 + i * kPer;
            if constexpr (kF32) {
                const float up = scale_up(__shfl_sync(0xffffffffu, my_top, i));
                uint2 hi, lo;
                split2(__uint_as_float(x[i].x) * up, __uint_as_float(x[i].y) * up, hi.x, lo.x);
                split2(__uint_as_float(x[i].z) * up, __uint_as_float(x[i].w) * up, hi.y, lo.y);
                // 8 bytes (4 columns) of a block's 128-byte row, whose 16-byte chunks are swizzled by the row
                unsigned char* at = out + (lane >> 4) * 16384 + row * 128 + ((((lane & 15) >> 1) ^ (row & 7)) << 4) + (lane & 1) * 8;
                *reinterpret_cast<uint2*>(at) = hi;
                *reinterpret_cast<uint2*>(at + 32768) = lo;
            } else {
                *reinterpret_cast<uint4*>(out + ((lane >> 3) & 1) * 16384 + row * 128 + (((lane & 7) ^ (row & 7)) << 4)) = x[i];
            }
        }
    }
}

// ---- the copying warp ---------------------------------------------------------------------------
// Operands in the order in which the tensor core takes them, over a segment: K(0), K(1), V(0), K(2), V(1), ...,
// V(n - 1). One thread.
template <bool kF32>
__device__ void copy_role(const ChunkArgs& a, Shared& s, unsigned char* ring, const Images& im, int g) {
    Walk& w = s.walk[kTeamWarps + 1];
    uint32_t stage = 0, phase = 0, unit0 = 0, issued = 0;
    auto copy = [&](bool v, int j) {
        const size_t index = ((size_t)w.b * a.lut_cols + w.t.page(w.j + j)) * a.pass_heads + w.head;
        const uint32_t u = (unit0 + j) & 7;
        const PageMeta& meta = im.meta[index];
        if (!mbar_wait(&s.empty[stage], phase ^ 1, nullptr)) return false;
        constexpr uint32_t kSkip = kF32 ? 0 : offsetof(PageMeta, all_keys), kMetaBytes = sizeof(PageMeta) - kSkip;
        mbar_arrive_expect_tx(&s.full[stage], kOperandBytes<kF32> + (v ? 0 : kMetaBytes));
        bulk_g2s(ring + stage * kOperandBytes<kF32>, im.operands + (index * 2 + v) * kOperandBytes<kF32>, kOperandBytes<kF32>,
                 &s.full[stage]);
        if (!v)
            bulk_g2s(reinterpret_cast<char*>(&s.meta[u]) + kSkip, reinterpret_cast<const char*>(&meta) + kSkip, kMetaBytes,
                     &s.full[stage]);
        ++issued;
        if (++stage == kStages<kF32>) stage = 0, phase ^= 1;
        return true;
    };
    auto run = [&] {
        w = s.run.first;
        for (bool more = s.run.some; more; more = w.next(a, g, kTile, kLead)) {
            const int n = w.n;
            for (int jj = 0; jj <= n; ++jj) {
                if (jj < n && !copy(false, jj)) return false;
                if (jj >= 1 && !copy(true, jj - 1)) return false;
            }
            unit0 += n;
        }
        return true;
    };
    if (!run()) s.abort = 1;  // a wait gave up
    // The copies in flight land before this CTA's memory is given back (the issuing warp has seen them all, unless it gave up)
    for (uint32_t k = 0; k < kStages<kF32> && k < issued; ++k) {
        if (stage == 0) stage = kStages<kF32>, phase ^= 1;
        mbar_wait(&s.full[--stage], phase, nullptr);
    }
}

// Pages whose products are added in TMEM.
template <bool kF32>
constexpr int kSumPages = kF32 ? 1 : 16;

// ---- the issuing warp -------------------------------------------------------------------------
// One warp, converged, one lane of which issues. A page's P V and the scores of the page after the next are issued as one
// run of MMAs, in whose middle the tensor core waits for nothing: the scores go where the weights lay, and MMAs run
// in the order in which they are issued. Meanwhile the softmax warps have the page between them.
template <bool kF32>
__device__ void mma_role(const ChunkArgs& a, Shared& s, unsigned char* ring, int g) {
    const uint32_t base = smem_addr(ring), me = elect_one();
    Walk& w = s.walk[kTeamWarps];
    uint32_t stage = 0, phase = 0, unit0 = 0, seg = 0, sums = 0;  // sums: begun so far in TMEM
    auto look = [&](uint64_t* bar, uint32_t parity) { return mbar_test(bar, parity); };
    // the operand `ahead` of the next one
    auto full = [&](uint32_t ahead) {
        const bool wraps = stage + ahead >= kStages<kF32>;
        return look(&s.full[wraps ? stage + ahead - kStages<kF32> : stage + ahead], phase ^ (wraps ? 1 : 0));
    };
    auto bounded = [&](auto&& all) {  // looks at all the barriers at once, until all are passed
        if (__all_sync(0xffffffffu, all())) return true;
        const uint64_t t0 = global_timer_ns();
        while (!__all_sync(0xffffffffu, all())) {
            if (__any_sync(0xffffffffu, s.abort || global_timer_ns() - t0 > kWaitBudgetNs)) {
                s.abort = 1;
                return false;
            }
        }
        return true;
    };
    // the MMAs of the next operand: D = sum over the products of A's halves and the operand's, 16 of the summed dimension
    // at a time; its stage given back, the result announced
    auto product = [&](uint32_t d, uint32_t ta, uint32_t a_step, uint32_t a_lo, uint32_t kind, uint32_t b_step2, uint32_t b_step8,
                       uint32_t id, uint32_t accumulate, uint64_t* done) __attribute__((always_inline)) {
        const uint32_t b = desc_lo(base + stage * kOperandBytes<kF32>, kind);
#pragma unroll
        for (int p = kF32 ? 0 : 2; p < 3; ++p) {  // lo x hi, hi x lo, hi x hi
#pragma unroll
            for (int i = 0; i < 8; ++i)
                umma_ts_f16(me, d, ta + i * a_step + (p == 0 ? a_lo : 0),
                            b + (i & 3) * b_step2 + (i >> 2) * b_step8 + (p == 1 ? 32768 >> 4 : 0), kDescHi, id,
                            p != (kF32 ? 0 : 2) || i != 0 ? 1u : accumulate);
        }
        umma_commit_if(me, &s.empty[stage]);
        umma_commit_if(me, done);
        if (++stage == kStages<kF32>) stage = 0, phase ^= 1;
    };
    auto run = [&] {
        auto next = [&](bool first) {
            return __any_sync(0xffffffffu, first ? warp_first(w, s.run) : warp_next(w, a, g, kTile, kLead));
        };
        for (bool more = next(true); more; more = next(false), ++seg) {
            const int n = __reduce_max_sync(0xffffffffu, w.n);
            if (!bounded([&] { return look(&s.q_full, seg & 1); })) return;
            for (int j = -2; j < n; ++j) {  // P V of page j, scores of page j + 2
                const uint32_t u = unit0 + j, buf = u & 1;
                const bool values = j >= 0, scores = j + 2 < n;
                const bool fresh = values && j % kSumPages<kF32> == 0;  // a new sum, once the last one has been taken
                const uint32_t taken = fresh ? sums++ : 0;
                // 16 dimensions of K are 32 bytes of a row, 64 a block; 16 rows of V are 2048 bytes of both its blocks
                if (!bounded([&] {
                        return (!values || look(&s.p_full[buf], (u >> 1) & 1)) && (!(values || scores) || full(0)) &&
                               (!(values && scores) || full(1)) && (taken == 0 || look(&s.pv_free, (taken - 1) & 1));
                    }))
                    return;
                tc_fence_after();
                if (values)
                    product(kColPv, kColS + buf * 128, 16, 8, kDescValues, 2048 >> 4, 8192 >> 4, idesc<kF32>(true), !fresh,
                            &s.pv_full[buf]);
                if (scores)
                    product(kColS + buf * 128, kColQ, 8, 64, kDescKeys, 32 >> 4, 16384 >> 4, idesc<kF32>(false), 0, &s.s_full[buf]);
            }
            unit0 += n;
        }
    };
    if (s.tmem == 0) run();
    else s.abort = 1;  // never: all 512 columns are ours
    // the MMAs have finished before the CTA's TMEM is freed
    umma_commit_if(me, &s.drain);
    mbar_wait_warp(&s.drain, 0, nullptr, nullptr);
}

// ---- the softmax warps ------------------------------------------------------------------------
// Two threads per row of the query tile (its TMEM lane): columns and dimensions [64 half, 64 half + 64) each. A row's
// sums are of 2^(score - m) and of that times values; m is at most 7 below the row's maximum so far, and where a page
// exceeds that the row's warps raise m and scale what they have. bf16: the weights in the operand are 2^(score - m), and the
// tensor core adds the products of 16 pages in TMEM, which then come into the threads' registers. fp32: of one page, for
// its own additions truncate (the threads' round to nearest: 8.6e-7 off at 8192 rows, 1.2e-6 with two pages to a sum and
// no faster); the weights' fp16 halves resolve 2^-25, so they are 2^(score - the page's maximum + 14), 2^-39 of the page's
// largest, and the page's sum takes 2^(its maximum - m - 14): weights of 2^-60 beside values of 2^70 count in full.
// m is `room` above the maximum. From a page on on which a row sees large values it is so by the logarithm of the tile's rows and
// the headroom, so that the sums stay below the values, up to the type's largest ones. Up to there it is 28 below in fp32, where the
// scale of a page's sum is 2^-28 of its values (so values down to the type's smallest normal ones keep their bits). Large:
// in bf16 the page has some of 2^65 or more; in fp32 the largest product of a weight and a value of the page reaches 2^50 or so, the
// weight 1 being the largest so far (a page's sum is below 2^86 until then, 2^22 of them in range). The row's own products: what it
// does not see does not decide.
constexpr float kHeadroom = 7.f, kLift = 14.f, kLarge32 = 64.f;
template <bool kF32>
constexpr float kRoom = kF32 ? -28.f : 0.f;
// Row `row` of the keys (v 0) or values (1) of page t (this head's 128 columns).
template <bool kF32>
UOCR_DEV const char* cache_row(const ChunkArgs& a, const Walk& w, int t, int row, int v) {
    constexpr int kElt = kF32 ? 4 : 2;
    const int r = t * kPageRows + row, column = (a.head0 + w.head) * kDim;
    if (r >= w.r.start) return static_cast<const char*>(v ? a.v : a.k) + ((size_t)(w.r.lo + r - w.r.start) * (v ? a.v_ld : a.k_ld) + column) * kElt;
    const uint32_t id = min(__ldg(a.lut + (size_t)w.b * a.lut_cols + t), (uint32_t)(a.pages - 1));
    return static_cast<const char*>(a.pool) +
           (((((size_t)id * 2 + v) * a.layers + a.layer) * kPageRows + row) * ((size_t)a.kv_heads * kDim) + column) * kElt;
}

// Which of 32 columns from c0 on a row sees: c <= hi and (c >= lo or c < pre), all relative to the page.
UOCR_DEV uint32_t seen_mask(int c0, int hi, int lo, int pre) {
    auto below = [](int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; };
    return below(hi + 1 - c0) & (~below(lo - c0) | below(pre - c0));
}

template <bool kF32>
__device__ void team_role(const ChunkArgs& a, Shared& s, const Images& im, const ChunkParts& parts, int g) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int half = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;  // TMEM address: lane from bit 16 up, 32 lanes a warp; columns from 0
    float qscale = 0.f;
    bool alive = true;
    const uint32_t tid = threadIdx.x;
    const uint32_t pair_bar = kPairBar + (warp & 3);

    // A segment's queries into TMEM (half 0 of the threads the hi halves, half 1 the lo ones; bf16: half the dimensions
    // each), once all have read the last one's scores.
    auto load_query = [&](const Walk& w) __attribute__((always_inline)) {
        const size_t index = (size_t)(query_base(w.r, w.b, g) + w.qt) * a.pass_heads + w.head;
        const uint4* p = reinterpret_cast<const uint4*>(im.queries + index * kQueryBytes<kF32>) + half * (kF32 ? 16 : 8) * kTile + row;
        uint32_t x[kF32 ? 64 : 32];
#pragma unroll
        for (int i = 0; i < (kF32 ? 16 : 8); ++i) {
            const uint4 v = ldg_nc_v4(p + i * kTile);
            x[4 * i] = v.x, x[4 * i + 1] = v.y, x[4 * i + 2] = v.z, x[4 * i + 3] = v.w;
        }
        qscale = __ldg(im.qscale + index * kTile + row);
        named_bar_sync(kTeamBar, 32 * kTeamWarps);
#pragma unroll
        for (int i = 0; i < (kF32 ? 8 : 4); ++i) tmem_st<8>(lanes + kColQ + half * (kF32 ? 64 : 32) + i * 8, x + 8 * i);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.q_full);
    };

    uint64_t acc[32];  // 64 sums, in pairs
    float m = -INFINITY, l = 0.f;

    // acc = (acc + the sum in TMEM, unit u its last page's, times its values' scale) * keep; ends = false: the sum stays
    // in TMEM, and it and acc become keep times as large.
    auto take_sum = [&](uint32_t u, float scale, float keep, bool ends, bool live) __attribute__((always_inline)) {
        if (alive && !wait(s, &s.pv_full[u & 1], (u >> 1) & 1)) alive = false;
        tc_fence_after();
        if (alive && live) {
            const uint64_t k2 = pair(keep, keep), f2 = ends ? pair(scale * keep, scale * keep) : 0;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                uint32_t x[32];
                tmem_ld_32x32b_x32(lanes + kColPv + half * 64 + c * 32, x);
                tmem_wait_ld_tie(x);
                if (ends) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) acc[c * 16 + i] = fma2(pair(x[2 * i], x[2 * i + 1]), f2, mul2(acc[c * 16 + i], k2));
                } else {
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        acc[c * 16 + i] = mul2(acc[c * 16 + i], k2);
                        unpair(mul2(pair(x[2 * i], x[2 * i + 1]), k2), x[2 * i], x[2 * i + 1]);
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) tmem_st<8>(lanes + kColPv + half * 64 + c * 32 + i * 8, x + 8 * i);
                }
            }
            if (!ends) tmem_wait_st();
            tc_fence_before();
        }
        __syncwarp();
        if (ends && lane == 0) mbar_arrive(&s.pv_free);
    };

    // fp32: the scores of this half's keys of page t that have elements that are not finite, kept out of the operand: those
    // elements alone make the score, an infinity or NaN, whatever it is scaled by later. In the place of the tensor core's scores.
    auto fix_scores = [&](const Walk& w, uint32_t u, int t, int R, uint32_t sa) {
        const bool valid = R < w.r.n * g;
        const float* q = static_cast<const float*>(a.q) + (valid ? (size_t)(w.r.lo + token_of(a, R)) * a.q_ld : 0) +
                         (size_t)((a.head0 + w.head) * g + (valid ? R - token_of(a, R) * g : 0)) * kDim;
#pragma unroll 1
        for (int c = 0; c < 64; ++c) {
            const int key = half * 64 + c;
            if (!(s.meta[u & 7].bad_keys[key >> 5] >> (key & 31) & 1)) continue;
            const float* k = reinterpret_cast<const float*>(cache_row<true>(a, w, t, key, 0));
            float sum = 0.f;
#pragma unroll 1
            for (int d = 0; valid && d < kDim; ++d)
                if (odd_f32(__float_as_uint(k[d]))) sum = fmaf(q[d], k[d], sum);
            __syncwarp();
            asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};" ::"r"(sa + c), "r"(__float_as_uint(sum * a.scale)) : "memory");
        }
        tmem_wait_st();
    };

    // The values of page t that are not finite and were kept out of its operand
    auto add_bad = [&](const Walk& w, uint32_t u, int t, int pos) __attribute__((always_inline)) {
        for (int q = 0; q < kPageRows; ++q) {
            if (!(s.meta[u & 7].bad[q >> 5] >> (q & 31) & 1)) continue;
            const int r = t * kPageRows + q;
            const bool seen = r <= pos && (a.window <= 0 || r > pos - a.window || r < w.r.prefix);
            if (!seen) continue;
            const char* p = cache_row<kF32>(a, w, t, q, 1) + half * (kF32 ? 256 : 128);
            auto odd = [](float v) { return odd_f32(__float_as_uint(v)) ? v : 0.f; };
#pragma unroll
            for (int d = 0; d < 32; ++d) {
                float v0, v1;
                if constexpr (kF32) {
                    const float2 v = reinterpret_cast<const float2*>(p)[d];
                    v0 = v.x, v1 = v.y;
                } else {
                    const uint32_t v = reinterpret_cast<const uint32_t*>(p)[d];
                    v0 = bf16lo(v), v1 = bf16hi(v);
                }
                acc[d] = add2(acc[d], pair(odd(v0), odd(v1)));
            }
        }
    };

    Walk& w = s.walk[warp];
    Walk& now = s.now[warp];  // the segment at work
    bool more = warp_first(w, s.run);
    int state[2] = {0, 0}, place[4] = {0, 0, 0, 0};
    uint32_t unit0 = 0;
    if (more) load_query(w);
    while (more) {
        __syncwarp();
        if (lane == 0) now = w;
        __syncwarp();
        const int R = now.qt * kTile + row, rows = now.r.n * g - now.qt * kTile;  // valid rows of the tile
        const bool live = (warp & 3) * 32 < rows;                                 // this warp has some
        const int pos = now.r.start + token_of(a, R);
        m = -INFINITY, l = 0.f;
#pragma unroll
        for (int i = 0; i < 64; ++i) acc[i] = 0;
        more = warp_next(w, a, g, kTile, kLead);  // w is one ahead from here on
        const int n = now.n, first_pos = now.t.first_pos, last_pos = now.t.last_pos, prefix = now.r.prefix;
        const int head_pages = now.t.head_pages - now.j, tail_page = now.t.tail_page - head_pages;  // page of the segment's j
        float sum_scale = 1.f;  // of the sum in TMEM
        float room = kRoom<kF32>;
        for (int j = 0;; ++j) {
            if (j == n) {  // the next segment's queries, while the last products run
                if (more) load_query(w);
                break;
            }
            const uint32_t u = unit0 + j, sa = lanes + kColS + (u & 1) * 128 + half * 64;
            const int c0 = (j < head_pages ? now.j + j : j + tail_page) * kPageRows;
            if (alive && !wait(s, &s.s_full[u & 1], (u >> 1) & 1)) alive = false;
            tc_fence_after();
            const bool run = alive && live;
            // does every row of the tile see the whole page?
            const bool all = c0 + kPageRows - 1 <= first_pos &&
                             (a.window <= 0 || c0 > last_pos - a.window || c0 + kPageRows <= prefix);
            // keys of one scale: it goes into the factor; else 1 / scale of each one's key (a branch, rarely taken)
            const PageMeta& pm = s.meta[u & 7];
            const float4 page = kF32 ? *reinterpret_cast<const float4*>(&pm.all_keys) : make_float4(1.f, 0.f, 0.f, 0.f);
            const uint32_t values_are = kF32 ? __float_as_uint(page.z) : pm.values_are;
            const float all_keys = page.x;
            float factor = kF32 && all_keys != 0.f ? fmaxf(qscale * all_keys, 1e-37f) : qscale;
            uint32_t x[64];
            float top = -INFINITY;
            if (run) {
                if (kF32 && __float_as_uint(page.w)) fix_scores(now, u, c0 / kPageRows, R, sa);
                tmem_ld64(sa, x);
                if (kF32 && all_keys == 0.f) {
                    asm volatile("");
#pragma unroll
                    for (int i = 0; i < 64; i += 4) {
                        const float4 k4 = *reinterpret_cast<const float4*>(pm.keys + half * 64 + i);
                        unpair(mul2(pair(x[i], x[i + 1]), pair(k4.x, k4.y)), x[i], x[i + 1]);
                        unpair(mul2(pair(x[i + 2], x[i + 3]), pair(k4.z, k4.w)), x[i + 2], x[i + 3]);
                    }
                }
                if (!all) {
                    asm volatile("");  // a branch, not 64 selects on every page
                    const int lo = a.window > 0 ? pos - a.window + 1 - c0 : -kPageRows;
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const uint32_t mask = seen_mask(half * 64 + c * 32, pos - c0, lo, prefix - c0);
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (!(mask >> i & 1)) x[c * 32 + i] = 0xFF800000u;
                    }
                }
                float top2 = -INFINITY;
#pragma unroll
                for (int i = 0; i < 64; i += 4) {
                    top = fmaxf(fmaxf(top, __uint_as_float(x[i])), __uint_as_float(x[i + 1]));
                    top2 = fmaxf(fmaxf(top2, __uint_as_float(x[i + 2])), __uint_as_float(x[i + 3]));
                }
                top = fmaxf(top, top2) * factor;
            }
            // NaN: a warp that has given up; its partner then does too, so that both go the same way below
            s.xmax[u & 1][half][row] = alive ? fmaxf(top, -INFINITY) : NAN;
            named_bar_sync(pair_bar, 64);
            const float other = s.xmax[u & 1][half ^ 1][row];
            alive = alive && other == other;
            const float page_max = fmaxf(top, other);
            // The operand's weights are 2^(score - ref), in fp32 times 2^14; products with the values' operand count 2^ref_log2 more.
            float ref = page_max, ref_log2 = page.y, unlike_sum = 0.f;
            const bool unlike = kF32 && alive && (values_are & kUnlike);
            if (unlike) {
                // A scale for each row of v: its weight takes 1 / scale, and the operand's weights are relative to the largest
                // of these products, of the rows that this one sees. l takes the weights alone.
                float most = -INFINITY;
                if (run) {
                    const float shift = kLift - (page_max == -INFINITY ? 0.f : page_max);
#pragma unroll
                    for (int i = 0; i < 64; ++i) {
                        const float score = __uint_as_float(x[i]) * factor;
                        unlike_sum += exp2_fast(score + shift);
                        const float w = score + pm.values_log2[half * 64 + i];
                        most = fmaxf(most, w);
                        x[i] = __float_as_uint(w);
                    }
                }
                s.xref[half][row] = most;
                named_bar_sync(pair_bar, 64);
                ref = fmaxf(most, s.xref[half ^ 1][row]);
                ref_log2 = 0.f;
                factor = 1.f;
            }
            float mn = fmaxf(m, page_max + room), keep = 1.f;
            if (room == kRoom<kF32> && (kF32 ? ref + ref_log2 > mn + kLarge32 : (values_are & kLarge) && page_max != -INFINITY)) {
                asm volatile("");  // a branch, rarely taken
                room = kHeadroom + 7.f + (32 - __clz(now.t.count - 1));
                mn += room - kRoom<kF32>;
            }
            const bool raised = __any_sync(0xffffffffu, mn > m + kHeadroom);  // the same in both warps of the rows
            if (raised) {
                keep = mn == -INFINITY ? 1.f : exp2_fast(m - mn);
                l *= keep;
                m = mn;
            }
            // a weight of 1 in the operand counts `unit` in l, and a product `sum_scale` in the sums
            if (!kF32) ref = m;
            const float unit = !kF32 ? 1.f : page_max == -INFINITY ? 0.f : exp2_fast(page_max - m - kLift);
            const float old_scale = sum_scale;
            if (kF32) sum_scale = ref == -INFINITY ? 0.f : exp2_fast(ref - m + (ref_log2 - kLift));
            const bool fresh = j % kSumPages<kF32> == 0;  // a new sum in TMEM
            if (run) {
                const float base = (kF32 ? kLift : 0.f) - (ref == -INFINITY ? 0.f : ref);
                const uint64_t q2 = pair(factor, factor), s2 = pair(base, base);
                uint64_t sum2[2] = {0, 0};
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    uint32_t p0, p1;
                    unpair(fma2(pair(x[2 * i], x[2 * i + 1]), q2, s2), p0, p1);
                    x[2 * i] = __float_as_uint(exp2_fast(__uint_as_float(p0)));
                    x[2 * i + 1] = __float_as_uint(exp2_fast(__uint_as_float(p1)));
                }
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t hi[8], lo[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const uint32_t e0 = x[c * 16 + 2 * i], e1 = x[c * 16 + 2 * i + 1];
                        sum2[i & 1] = add2(sum2[i & 1], pair(e0, e1));
                        if constexpr (kF32) split2(__uint_as_float(e0), __uint_as_float(e1), hi[i], lo[i]);
                        else hi[i] = pack_bf16(__uint_as_float(e0), __uint_as_float(e1));
                    }
                    // in the place of the 16 scores
                    tmem_st<8>(sa + c * 16, hi);
                    if constexpr (kF32) tmem_st<8>(sa + c * 16 + 8, lo);
                }
                uint32_t u0, u1;
                unpair(add2(sum2[0], sum2[1]), u0, u1);
                l += (unlike ? unlike_sum : __uint_as_float(u0) + __uint_as_float(u1)) * unit;
                tmem_wait_st();
                tc_fence_before();
            }
            // the sum that ends here: its last product has run meanwhile
            if (j > 0 && (fresh || raised)) take_sum(u - 1, old_scale, keep, fresh, live);
            __syncwarp();
            if (lane == 0) mbar_arrive(&s.p_full[u & 1]);
            if (values_are & kBad) add_bad(now, u, c0 / kPageRows, pos);
        }
        if (a.expire >> warp & 1) s.abort = 1, alive = false;
        take_sum(unit0 + n - 1, sum_scale, 1.f, true, live);
        unit0 += n;
        // to out, or column by column to the workspace
        // A warp that gave up set s.abort in front of the arrivals that let others go on, so that whoever worked on what it left sees it
        // here. NaN in one half's l makes the row NaN in both, here or by way of the parts' l.
        s.xsum[half][row] = alive && !s.abort ? l : NAN;
        named_bar_sync(pair_bar, 64);
        const float total = s.xsum[0][row] + s.xsum[1][row];
        const bool whole = now.whole();
        const float f = whole ? 1.f / total : 1.f;
        const uint64_t f2 = pair(f, f);
        const int slot = now.j == 0 ? 1 : 0;
        float* part = parts.slots + ((size_t)blockIdx.x * 2 + slot) * slot_floats(kTile);
        if (whole && row < rows) {
            const size_t at = ((size_t)(now.r.lo + pos - now.r.start) * a.heads + (a.head0 + now.head) * g + R - (pos - now.r.start) * g) * kDim + half * 64;
            auto two = [&](int i) {
                uint32_t y0, y1;
                unpair(mul2(acc[i], f2), y0, y1);
                return pack_bf16(__uint_as_float(y0), __uint_as_float(y1));
            };
#pragma unroll
            for (int i = 0; i < (kF32 ? 16 : 8); ++i) {
                uint4 v;
                if constexpr (kF32) {
                    unpair(mul2(acc[2 * i], f2), v.x, v.y);
                    unpair(mul2(acc[2 * i + 1], f2), v.z, v.w);
                    reinterpret_cast<uint4*>(static_cast<float*>(a.out) + at)[i] = v;
                } else {
                    v = make_uint4(two(4 * i), two(4 * i + 1), two(4 * i + 2), two(4 * i + 3));
                    reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + at)[i] = v;
                }
            }
        } else if (!whole && row < rows) {
            float* o = part + half * 64 * kTile + row;
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                uint32_t y0, y1;
                unpair(mul2(acc[i], f2), y0, y1);
                o[2 * i * kTile] = __uint_as_float(y0), o[(2 * i + 1) * kTile] = __uint_as_float(y1);
            }
        }
        named_bar_sync(pair_bar, 64);  // xsum is free again
        if (!whole) {
            if (half == 0 && row < rows) {
                part[kDim * kTile + row] = m;
                part[(kDim + 1) * kTile + row] = total;
            }
            state[slot] = slot == 0 && now.j + now.n == now.t.count ? 2 : 1;
            if (slot == 1)
                place[0] = now.r.lo, place[1] = now.qt * kTile, place[2] = min(rows, kTile), place[3] = a.head0 + now.head;
        }
    }
    if (tid == 0) {
        int* o = parts.info + blockIdx.x * kInfoInts;
        o[0] = state[0], o[1] = state[1];
        for (int i = 0; i < 4; ++i) o[2 + i] = place[i];
    }
}

template <bool kF32>
__global__ void __launch_bounds__(kThreads, 1) chunk_attention_kernel(const __grid_constant__ ChunkArgs a, const __grid_constant__ Images im, const __grid_constant__ ChunkParts parts) {
    extern __shared__ unsigned char raw[];
    __shared__ Shared s;
    unsigned char* ring = raw + ((1024 - (smem_addr(raw) & 1023)) & 1023);
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
    const int g = a.heads / a.kv_heads;
    if (threadIdx.x == 0) {
        for (int i = 0; i < kMaxStages; ++i) mbar_init(&s.full[i], 1), mbar_init(&s.empty[i], 1);
        for (int i = 0; i < 2; ++i) mbar_init(&s.s_full[i], 1), mbar_init(&s.p_full[i], kTeamWarps), mbar_init(&s.pv_full[i], 1);
        mbar_init(&s.pv_free, kTeamWarps), mbar_init(&s.q_full, kTeamWarps), mbar_init(&s.drain, 1);
        fence_mbar_init();
        s.abort = 0;
    }
    if (warp == kTeamWarps) tmem_alloc(&s.tmem, 512);
    tc_fence_before();
    find_run(a, s.run, reinterpret_cast<uint32_t*>(ring), g, kTile, kLead);
    tc_fence_after();
    pdl_launch_dependents();
    if (warp < kTeamWarps) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kTeamRegs));
        pdl_wait_prior_grid();
        team_role<kF32>(a, s, im, parts, g);
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
        if (warp == kTeamWarps) {
            mma_role<kF32>(a, s, ring, g);
        } else if (threadIdx.x == 32 * (kTeamWarps + 1)) {
            fence_proxy_async_smem();  // the ring was find_run's scratch
            pdl_wait_prior_grid();
            fence_proxy_async_global();  // the operands were stored through the generic proxy
            copy_role<kF32>(a, s, ring, im, g);
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == kTeamWarps) tmem_dealloc(s.tmem, 512);
}

// The parts of a tile that was cut: CTA c's slot 1 begins it, slot 0 of the CTAs behind it continues it.
// out = sum_i 2^(m_i - M) sum_i / sum_i 2^(m_i - M) l_i, in the order of the pages. A block joins as
// many groups of 8 columns of a tile as it has threads for. Bound: the latency of three dependent reads (states, m and l,
// sums), 4 to 6 us of which the launch hides half; a tile of 8192 tokens is cut at most once or twice.
template <bool kF32>
__global__ void __launch_bounds__(256) chunk_join_kernel(ChunkArgs a, ChunkParts p) {
    pdl_wait_prior_grid();
    const float* slots = p.slots;
    const int* info = p.info;
    const int ctas = p.ctas, tile = p.tile;
    const size_t slot = slot_floats(tile);
    const int c = blockIdx.x, g = a.heads / a.kv_heads;
    const int4 head4 = *reinterpret_cast<const int4*>(info + c * kInfoInts);      // states, lo, first row
    const int2 tail2 = *reinterpret_cast<const int2*>(info + c * kInfoInts + 4);  // rows, head
    if (head4.y == 0) return;
    // one behind the last CTA of this tile: the states of 32 CTAs at a time
    int end = c + 1;
    for (;; end += 32) {
        const int d = end + (threadIdx.x & 31);
        const uint32_t last = __ballot_sync(0xffffffffu, d >= ctas || info[d * kInfoInts] != 1);
        if (last) {
            end = min(end + __ffs(last), ctas);
            break;
        }
    }
    const int lo = head4.z, r0 = head4.w, rows = tail2.x, head = tail2.y;
    // threads by row, then by 8 columns: few rows take few threads' time
    const int group = blockIdx.y * (256 / tile) + threadIdx.x / tile, row = threadIdx.x % tile, c0 = group * 8;
    if (row >= rows || group >= kDim / 8) return;
    // a running maximum, the next part on its way
    float M = -INFINITY, l = 0.f, x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = 0.f;
#pragma unroll 4
    for (int d = c; d < end; ++d) {
        const float* part = slots + ((size_t)d * 2 + (d == c)) * slot;
        const float md = part[kDim * tile + row], ld = part[(kDim + 1) * tile + row];
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = part[(c0 + i) * tile + row];
        const float mn = fmaxf(M, md), base = mn == -INFINITY ? 0.f : mn;  // -inf: parts in which the row sees nothing
        const float keep = exp2_fast(M - base), f = exp2_fast(md - base);
        M = mn;
        l = fmaf(ld, f, l * keep);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = fmaf(y[i], f, x[i] * keep);
    }
    const float inv = 1.f / l;
    const int R = r0 + row;
    const size_t at = ((size_t)(lo + token_of(a, R)) * a.heads + head * g + R - token_of(a, R) * g) * kDim + c0;
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

template <typename... P, typename... A>
cudaError_t launch_dependent(void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t st, A... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid, cfg.blockDim = dim3(threads), cfg.dynamicSmemBytes = smem, cfg.stream = st;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr, cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, P(args)...);
}

// Query tiles of the call, at most (query_base).
int query_tiles(const ChunkArgs& a) { return (int)((long long)a.T * (a.heads / a.kv_heads) / kTile) + a.B; }

template <bool kF32>
cudaError_t launch(const ChunkArgs& a, const Images& im, const ChunkParts& parts, cudaStream_t st) {
    const size_t smem = (size_t)kStages<kF32> * kOperandBytes<kF32> + 1024;
    auto kernel = chunk_attention_kernel<kF32>;
    cudaError_t err = ensure_smem_optin(reinterpret_cast<const void*>(kernel), smem);
    if (err != cudaSuccess) return err;
    chunk_operands_kernel<kF32><<<dim3(a.B * a.lut_cols + query_tiles(a), a.pass_heads), 256, 0, st>>>(a, im);
    err = cudaGetLastError();
    if (err != cudaSuccess) return err;
    err = launch_dependent(kernel, dim3(parts.ctas), kThreads, smem, st, a, im, parts);
    if (err != cudaSuccess) return err;
    return launch_chunk_join(a, parts, st);
}

// Operands and what lies beside them, of one page or query tile and one head.
size_t page_bytes(const ChunkArgs& a) { return 2 * (size_t)(a.bf16 ? kOperandBytes<false> : kOperandBytes<true>) + sizeof(PageMeta); }
size_t query_bytes(const ChunkArgs& a) { return (a.bf16 ? kQueryBytes<false> : kQueryBytes<true>) + kTile * sizeof(float); }
// The operands of one KV head.
size_t head_bytes(const ChunkArgs& a) {
    return (size_t)a.B * a.lut_cols * page_bytes(a) + (size_t)query_tiles(a) * query_bytes(a);
}

// The KV heads of one pass: their operands stay within 1 GiB (one head at least); a call with more takes several.
constexpr size_t kPassBytes = size_t(1) << 30;
int heads_of_pass(const ChunkArgs& a) {
    return (int)std::max<size_t>(1, std::min<size_t>(a.kv_heads, kPassBytes / head_bytes(a)));
}

size_t parts_bytes(int sms, int tile) {
    return ((size_t)sms * kInfoInts * 4 + 255) / 256 * 256 + ((size_t)sms * 2 * tile * (kDim + 2) * 4 + 255) / 256 * 256;
}

}  // namespace

cudaError_t launch_chunk_join(const ChunkArgs& a, const ChunkParts& p, cudaStream_t st) {
    const int groups = 256 / p.tile;  // of 8 columns, a block
    const dim3 grid(p.ctas, (kDim / 8 + groups - 1) / groups);
    return launch_dependent(a.bf16 ? chunk_join_kernel<false> : chunk_join_kernel<true>, grid, 256, 0, st, a, p);
}

// Rows of a query tile: 1 to 8 where a request has few (token, head) rows of a KV head on average (chunk_rows.cu: bound by
// the cache's bytes), else 128 (tensor cores). One form for the whole call, by T (rows in no request among them) and B
// (empty requests among them), as the lengths are on the device: 63 single tokens over 639 rows and a chunk of 512 over
// 7700 take 1149 us in one call, 82 + 105 in two; 7 single tokens over 8000 rows beside that chunk 401, 109 + 105 in two.
// Measured at 8 requests of 8000 rows, 10 heads: fp32, 16 rows 274 us against 353; bf16 (16 heads), 8 rows 217 us against
// 287; beyond the rule, a little earlier: fp32, 24 rows 464 us against 359; bf16, 9 rows 469 against 292. The tile's rows
// cost time too (fp32, 2 to 8 rows: 107 to 145 us): a whole average is taken for every request's number of rows, with
// another one they differ and twice the average less one is provided for, since a second tile reads the cache again.
static int tile_rows(const ChunkArgs& a) {
    const long long rows = (long long)a.T * (a.heads / a.kv_heads);
    if (rows > (a.bf16 ? 8ll : 16ll) * a.B) return kTile;
    const long long wanted = rows % a.B ? 2 * rows - a.B : rows;
    for (int t : {1, 2, 3, 4, 6})
        if (wanted <= (long long)t * a.B) return t;
    return 8;
}

size_t chunk_workspace_bytes(const ChunkArgs& a, int sms) {
    if (tile_rows(a) < kTile) return parts_bytes(sms, tile_rows(a));
    return parts_bytes(sms, kTile) + head_bytes(a) * heads_of_pass(a);
}

cudaError_t launch_chunk_attention(const ChunkArgs& args, void* ws, int sms, cudaStream_t st) {
    ChunkArgs a = args;
    const int g = a.heads / a.kv_heads;
    a.expire = g_chunk_expire;
    a.group_shift = 32;
    while (g >> (a.group_shift - 31)) ++a.group_shift;
    a.group_mul = ((1ull << a.group_shift) + g - 1) / g;
    if (a.B <= 0 || a.T <= 0) return cudaSuccess;
    char* w = static_cast<char*>(ws);
    ChunkParts parts{reinterpret_cast<float*>(w + ((size_t)sms * kInfoInts * 4 + 255) / 256 * 256), reinterpret_cast<int*>(w), sms,
                     tile_rows(a)};
    if (parts.tile < kTile) {
        a.head0 = 0, a.pass_heads = a.kv_heads;
        return launch_chunk_rows(a, parts, st);
    }
    const int heads = heads_of_pass(a);
    const size_t pages = (size_t)a.B * a.lut_cols * heads, tiles = (size_t)query_tiles(a) * heads;
    Images im;
    im.operands = reinterpret_cast<unsigned char*>(w + parts_bytes(sms, kTile));
    im.queries = im.operands + pages * (page_bytes(a) - sizeof(PageMeta));
    im.meta = reinterpret_cast<PageMeta*>(im.queries + tiles * (query_bytes(a) - kTile * sizeof(float)));
    im.qscale = reinterpret_cast<float*>(im.meta + pages);
    for (a.head0 = 0; a.head0 < a.kv_heads; a.head0 += heads) {
        a.pass_heads = std::min(heads, a.kv_heads - a.head0);
        const cudaError_t err = a.bf16 ? launch<false>(a, im, parts, st) : launch<true>(a, im, parts, st);
        if (err != cudaSuccess) return err;
    }
    return cudaSuccess;
}

}  // namespace uocr
