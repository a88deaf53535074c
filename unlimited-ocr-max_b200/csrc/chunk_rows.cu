// The chunk attention of few query rows per request and KV head (a decode step, drafted tokens, a decode step of
// shared heads): each cached row is used a handful of times, so the call is bound by reading the cache (HBM), and the
// products run on the fp32 units straight from the loaded rows -- turning the rows into tensor-core operands would
// take longer than they are needed.
//
// A query tile is NQ (token, head) rows, in shared memory; a unit (tile, KV head, page) is shared by 8 warps, 16 rows
// of the page each, and each warp keeps a softmax of its own over its rows: no barrier between the pages. A row of k
// lies in 8 lanes; the dot products of 4 rows are reduced together, so that a lane ends with one row's scores. A row of
// v lies in all 32 lanes, 4 columns each. While a page's scores are computed its values are on their way, and the next
// page's keys while the values are summed: 64 KB of k and 64 KB of v a SM (fp32). The warps' results are joined
// when a tile's run of pages ends, the runs' results by the joining launch.
//
// The weights of a row are held by two lanes and read back by all: (p, p) as one 8-byte word feeds a packed fp32 product
// without a move. bf16 rows are widened where they are used, exactly; nothing is rounded before the result.
//
// Measured (B200, fp32, 10 heads): 8 requests over 8000 rows, 656 MB: 1 row each 105 us (6.2 TB/s), 4 rows 110, 8 rows
// 145 (the fp32 units bound it: every element takes part in 8 products). 1 to 5 drafted tokens over contexts of 997 to
// 8000 rows, 368 MB: 74 us, 5.0 TB/s (the request of 5 has two tiles of 3 and is read twice). Short calls are bound by
// latency: one request of 640 rows 11.0 us with the joining launch, 8 requests of 77 to 639 rows (29 MB) 14.5; 256
// requests of 100 rows (265 MB) 74 us, 3.6 TB/s: tiles of one page, 4 us each for the chain table, keys, scores, values,
// join (the next tile found a tile ahead: 71 us, but 11.5 for the one request, and not kept). Smaller units would
// shorten it for one short request only, and cost the long ones their streams.
#include <type_traits>

#include "chunk.cuh"

namespace uocr {
namespace {

constexpr int kWarps = 8, kThreads = 32 * kWarps;
constexpr int kLead = 1;  // what a tile costs beside its pages

template <int NQ>
struct Shared {
    Run run;
    Walk walk[kWarps];
    float4 q[2][NQ][kDim / 4];           // this segment's queries and the next one's, times scale log2(e)
    float2 p[kWarps][16][NQ];            // a warp's weights, twice each; -0 for a row that is not seen
    alignas(16) float sum[kWarps][NQ][kDim];
    float m[kWarps][NQ], l[kWarps][NQ];
};

UOCR_DEV float warp_max(float v) {
    float r;
    asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}

// The words of a warp's 16 rows of a page. k: word (i, c) is row 4 i + lane / 8, 16 bytes lane % 8 + 8 c; v: word r is
// row r, 4 columns of this lane.
template <bool kF32>
struct Words {
    static constexpr int kElt = kF32 ? 4 : 2, kChunks = kF32 ? 4 : 2;
    uint4 k[4][kChunks];
    uint2 v[16][kF32 ? 2 : 1];
};

// Where a unit's rows lie.
struct Place {
    const char *k_pool, *v_pool, *k_new, *v_new;  // page row 0 of this head
    int cached, known;                            // page rows [0, cached) in the pool, [cached, known) new
    int own0, own1;                               // new rows that this tile stores
    int c0;                                       // the page's first logical row
};

template <bool kF32>
UOCR_DEV Place place_of(const ChunkArgs& a, const Walk& w, int j, uint32_t id, int g, int tile) {
    constexpr int kElt = kF32 ? 4 : 2;
    Place p;
    p.c0 = w.t.page(w.j + j) * kPageRows;
    const size_t row_bytes = (size_t)a.kv_heads * (kDim * kElt), plane = (size_t)a.layers * kPageRows * row_bytes;
    const int column = w.head * (kDim * kElt);
    const char* pool = static_cast<const char*>(a.pool) +
                       ((size_t)min(id, (uint32_t)(a.pages - 1)) * 2 * a.layers + a.layer) * (kPageRows * row_bytes) + column;
    p.k_pool = pool, p.v_pool = pool + plane;
    p.cached = w.r.start - p.c0, p.known = min(kPageRows, w.t.last_pos + 1 - p.c0);
    p.k_new = static_cast<const char*>(a.k) + (w.r.lo - p.cached) * (a.k_ld * kElt) + column;
    p.v_new = static_cast<const char*>(a.v) + (w.r.lo - p.cached) * (a.v_ld * kElt) + column;
    // new rows whose first query head lies in this tile
    p.own0 = p.cached + token_of(a, w.qt * tile + g - 1);
    p.own1 = id < (uint32_t)a.pages ? p.cached + min(w.r.n, token_of(a, w.qt * tile + tile + g - 1)) : p.own0;
    return p;
}

template <bool kF32>
UOCR_DEV void load_keys(const ChunkArgs& a, const Place& p, int row0, int lane, Words<kF32>& x) {
    using W = Words<kF32>;
    const int first = row0 + (lane >> 3);
    const size_t row_bytes = (size_t)a.kv_heads * (kDim * W::kElt);
    const char* s = p.k_pool + first * row_bytes + (lane & 7) * 16;
    if (p.cached >= kPageRows) {  // the whole page is cached: addresses by addition
#pragma unroll
        for (int i = 0; i < 4; ++i, s += 4 * row_bytes)
#pragma unroll
            for (int c = 0; c < W::kChunks; ++c) x.k[i][c] = ldg_nc_v4(s + c * 128);
        return;
    }
    const long long ld = a.k_ld * W::kElt;
    const char* f = p.k_new + first * ld + (lane & 7) * 16;
#pragma unroll
    for (int i = 0; i < 4; ++i, s += 4 * row_bytes, f += 4 * ld) {
        const int row = first + 4 * i;
        const char* from = row < p.cached ? s : f;
#pragma unroll
        for (int c = 0; c < W::kChunks; ++c) x.k[i][c] = row < p.known ? ldg_nc_v4(from + c * 128) : make_uint4(0, 0, 0, 0);
    }
}
template <bool kF32>
UOCR_DEV void load_values(const ChunkArgs& a, const Place& p, int row0, int lane, Words<kF32>& x) {
    using W = Words<kF32>;
    auto load = [&](int r, const char* from) {
        if constexpr (kF32) {
            const uint4 v = ldg_nc_v4(from);
            x.v[r][0] = make_uint2(v.x, v.y), x.v[r][1] = make_uint2(v.z, v.w);
        } else {
            x.v[r][0] = ldg_nc_v2(from);
        }
    };
    const size_t row_bytes = (size_t)a.kv_heads * (kDim * W::kElt);
    const char* s = p.v_pool + row0 * row_bytes + lane * (kF32 ? 16 : 8);
    if (p.cached >= kPageRows) {
#pragma unroll
        for (int r = 0; r < 16; ++r, s += row_bytes) load(r, s);
        return;
    }
    const long long ld = a.v_ld * W::kElt;
    const char* f = p.v_new + row0 * ld + lane * (kF32 ? 16 : 8);
#pragma unroll
    for (int r = 0; r < 16; ++r, s += row_bytes, f += ld) {
        x.v[r][0] = x.v[r][kF32 ? 1 : 0] = make_uint2(0, 0);
        if (row0 + r < p.known) load(r, row0 + r < p.cached ? s : f);
    }
}

// The new rows of k (those of v are stored once they have arrived).
template <bool kF32>
UOCR_DEV void store_new_keys(const ChunkArgs& a, const Place& p, int row0, int lane, const Words<kF32>& x) {
    using W = Words<kF32>;
    const size_t row_bytes = (size_t)a.kv_heads * (kDim * W::kElt);
    auto mine = [&](int row) { return row >= p.own0 && row < p.own1 && row < kPageRows && row >= 0; };
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = row0 + 4 * i + (lane >> 3);
        if (!mine(row)) continue;
#pragma unroll
        for (int c = 0; c < W::kChunks; ++c)
            *reinterpret_cast<uint4*>(const_cast<char*>(p.k_pool) + row * row_bytes + (lane & 7) * 16 + c * 128) = x.k[i][c];
    }
}

template <bool kF32, int NQ>
__global__ void __launch_bounds__(kThreads, 1) chunk_rows_kernel(const __grid_constant__ ChunkArgs a, const __grid_constant__ ChunkParts parts) {
    using W = Words<kF32>;
    extern __shared__ char raw[];
    Shared<NQ>& s = *reinterpret_cast<Shared<NQ>*>(raw);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tid = threadIdx.x;
    const int g = a.heads / a.kv_heads, row0 = warp * 16;
    find_run(a, s.run, reinterpret_cast<uint32_t*>(raw + sizeof(Shared<NQ>)), g, NQ, kLead);
    pdl_launch_dependents();
    Walk& w = s.walk[warp];
    bool more = warp_first(w, s.run);
    int state[2] = {0, 0}, where[4] = {0, 0, 0, 0};
    const float factor = a.scale * kLog2e;
    // a segment's queries: thread (row, 4 columns)
    auto load_query = [&](int buf) {
        for (int e = tid; e < NQ * (kDim / 4); e += kThreads) {
            const int R = w.qt * NQ + e / (kDim / 4);
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            if (R < w.r.n * g) {
                const size_t at = (w.r.lo + token_of(a, R)) * a.q_ld + (size_t)(w.head * g + R - token_of(a, R) * g) * kDim + (e % (kDim / 4)) * 4;
                if constexpr (kF32) {
                    v = *reinterpret_cast<const float4*>(static_cast<const float*>(a.q) + at);
                } else {
                    const uint2 u = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(a.q) + at);
                    v = make_float4(bf16lo(u.x), bf16hi(u.x), bf16lo(u.y), bf16hi(u.y));
                }
            }
            s.q[buf][e / (kDim / 4)][e % (kDim / 4)] = make_float4(v.x * factor, v.y * factor, v.z * factor, v.w * factor);
        }
    };
    auto page_id = [&](int j) { return __ldg(a.lut + (size_t)w.b * a.lut_cols + w.t.page(w.j + j)); };
    W x;
    Place pl;
    if (more) {
        pl = place_of<kF32>(a, w, 0, page_id(0), g, NQ);
        load_keys<kF32>(a, pl, row0, lane, x);
        load_query(0);
    }
    __syncthreads();
    for (int buf = 0; more; buf ^= 1) {
        float m[NQ], l[NQ];
        uint64_t acc[NQ][2];  // 4 columns, in pairs
#pragma unroll
        for (int j = 0; j < NQ; ++j) m[j] = -INFINITY, l[j] = 0.f, acc[j][0] = acc[j][1] = 0;
        const int n = w.n, qt = w.qt, head = w.head, lo = w.r.lo, start = w.r.start, prefix = w.r.prefix;
        const int rows = min(NQ, w.r.n * g - qt * NQ);
        const bool whole = w.whole(), begins = w.j == 0, ends = w.j + w.n == w.t.count;
        const int first_pos = w.t.first_pos, last_pos = w.t.last_pos;
        // weights are 1 / (a power of two not below the rows of the tile's pages) at most: sums stay below the values
        const float most = __uint_as_float((127 - 7 - (32 - __clz(w.t.count - 1))) << 23);
        for (int u = 0; u < n; ++u) {
            uint32_t id = 0;
            if (u + 1 < n) id = page_id(u + 1);
            load_values<kF32>(a, pl, row0, lane, x);
            const int c0 = pl.c0;
            const bool stores = pl.own1 > pl.own0;
            if (stores) store_new_keys<kF32>(a, pl, row0, lane, x);
            // scores: this lane ends with row `mine` of the warp's 16 (two lanes each)
            const int mine = 4 * ((lane >> 1) & 3) + (lane >> 3);
            float sc[NQ];
#pragma unroll
            for (int j = 0; j < NQ; ++j) {
                uint64_t d2[4] = {0, 0, 0, 0};  // sums over even and odd dimensions
#pragma unroll
                for (int c = 0; c < W::kChunks; ++c) {
                    if constexpr (kF32) {
                        const float4 q = s.q[buf][j][(lane & 7) + 8 * c];
                        const uint64_t q0 = pair(q.x, q.y), q1 = pair(q.z, q.w);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const uint4& k = x.k[i][c];
                            d2[i] = fma2(q1, pair(k.z, k.w), fma2(q0, pair(k.x, k.y), d2[i]));
                        }
                    } else {
                        const float4 qa = s.q[buf][j][2 * ((lane & 7) + 8 * c)], qb = s.q[buf][j][2 * ((lane & 7) + 8 * c) + 1];
                        const uint64_t q0 = pair(qa.x, qa.y), q1 = pair(qa.z, qa.w), q2 = pair(qb.x, qb.y), q3 = pair(qb.z, qb.w);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const uint4& k = x.k[i][c];
                            auto two = [](uint32_t w) { return pair(w << 16, w & 0xFFFF0000u); };
                            d2[i] = fma2(q1, two(k.y), fma2(q0, two(k.x), d2[i]));
                            d2[i] = fma2(q3, two(k.w), fma2(q2, two(k.z), d2[i]));
                        }
                    }
                }
                float d[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t e, o;
                    unpair(d2[i], e, o);
                    d[i] = __uint_as_float(e) + __uint_as_float(o);
                }
                // 4 sums over 8 lanes: lanes with bit 2 take sums 2 and 3, with bit 1 the second of their two
                const bool up2 = lane & 4, up1 = lane & 2;
                float e0 = up2 ? d[2] : d[0], e1 = up2 ? d[3] : d[1];
                e0 += __shfl_xor_sync(0xffffffffu, up2 ? d[0] : d[2], 4);
                e1 += __shfl_xor_sync(0xffffffffu, up2 ? d[1] : d[3], 4);
                float f = up1 ? e1 : e0;
                f += __shfl_xor_sync(0xffffffffu, up1 ? e0 : e1, 2);
                sc[j] = f + __shfl_xor_sync(0xffffffffu, f, 1);
            }
            // the next page's keys (the next segment's where this one ends)
            Place next = pl;
            if (u + 1 < n) {
                next = place_of<kF32>(a, w, u + 1, id, g, NQ);
                load_keys<kF32>(a, next, row0, lane, x);
            }
            // does every row of the tile see the whole page?
            const bool all = c0 + kPageRows - 1 <= first_pos &&
                             (a.window <= 0 || c0 > last_pos - a.window || c0 + kPageRows <= prefix);
#pragma unroll
            for (int j = 0; j < NQ; ++j) {
                bool seen = true;
                if (!all) {
                    const int pos = start + token_of(a, qt * NQ + j), r = c0 + row0 + mine;
                    seen = r <= pos && (a.window <= 0 || r > pos - a.window || r < prefix);
                    if (!seen) sc[j] = -INFINITY;
                }
                const float mn = fmaxf(m[j], warp_max(sc[j]));
                const float p = exp2_fast(sc[j] - (mn == -INFINITY ? 0.f : mn)) * most;
                const float alpha = mn == -INFINITY ? 1.f : exp2_fast(m[j] - mn);
                m[j] = mn;
                l[j] = l[j] * alpha + p;
                const uint64_t a2 = pair(alpha, alpha);
                acc[j][0] = mul2(acc[j][0], a2), acc[j][1] = mul2(acc[j][1], a2);
                if (!(lane & 1)) s.p[warp][mine][j] = seen ? make_float2(p, p) : make_float2(-0.f, -0.f);
            }
            __syncwarp();
            if (stores) {  // the new rows of v
                const size_t row_bytes = (size_t)a.kv_heads * (kDim * W::kElt);
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int row = row0 + r;
                    if (row < pl.own0 || row >= pl.own1) continue;
                    char* o = const_cast<char*>(pl.v_pool) + row * row_bytes + lane * (kF32 ? 16 : 8);
                    if constexpr (kF32) *reinterpret_cast<uint4*>(o) = make_uint4(x.v[r][0].x, x.v[r][0].y, x.v[r][1].x, x.v[r][1].y);
                    else *reinterpret_cast<uint2*>(o) = x.v[r][0];
                }
            }
            auto add_rows = [&](auto masked) __attribute__((always_inline)) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    uint64_t v0, v1;
                    if constexpr (kF32) v0 = pair(x.v[r][0].x, x.v[r][0].y), v1 = pair(x.v[r][1].x, x.v[r][1].y);
                    else v0 = pair(x.v[r][0].x << 16, x.v[r][0].x & 0xFFFF0000u), v1 = pair(x.v[r][0].y << 16, x.v[r][0].y & 0xFFFF0000u);
#pragma unroll
                    for (int j = 0; j < NQ; ++j) {
                        const float2 p = s.p[warp][r][j];
                        if (decltype(masked)::value && __float_as_int(p.x) < 0) continue;  // not seen: whatever the row holds stays out
                        const uint64_t p2 = pair(p.x, p.y);
                        acc[j][0] = fma2(p2, v0, acc[j][0]), acc[j][1] = fma2(p2, v1, acc[j][1]);
                    }
                }
            };
            if (all) add_rows(std::false_type{});
            else add_rows(std::true_type{});
            __syncwarp();
            pl = next;
        }
        // the next segment's first keys and queries are on their way while this one is joined
        more = warp_next(w, a, g, NQ, kLead);
        if (more) {
            pl = place_of<kF32>(a, w, 0, page_id(0), g, NQ);
            load_keys<kF32>(a, pl, row0, lane, x);
        }
#pragma unroll
        for (int j = 0; j < NQ; ++j) {
            float t = lane & 1 ? 0.f : l[j];  // two lanes hold each row
#pragma unroll
            for (int o = 16; o; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
            if (lane == 0) s.m[warp][j] = m[j], s.l[warp][j] = t;
            *reinterpret_cast<ulonglong2*>(&s.sum[warp][j][4 * lane]) = make_ulonglong2(acc[j][0], acc[j][1]);
        }
        if (more) load_query(buf ^ 1);
        __syncthreads();
        const int slot = begins ? 1 : 0;
        float* part = parts.slots + ((size_t)blockIdx.x * 2 + slot) * slot_floats(NQ);
        for (int e = tid; e < rows * (kDim / 2); e += kThreads) {  // (row, 2 columns)
            const int j = e / (kDim / 2), d = (e % (kDim / 2)) * 2;
            float M = -INFINITY, L = 0.f;
#pragma unroll
            for (int k = 0; k < kWarps; ++k) M = fmaxf(M, s.m[k][j]);
            float2 o = make_float2(0.f, 0.f);
#pragma unroll
            for (int k = 0; k < kWarps; ++k) {
                const float mk = s.m[k][j], f = mk == -INFINITY ? 0.f : exp2_fast(mk - M);
                L = fmaf(s.l[k][j], f, L);
                // a warp that has seen nothing has sums of 0; scores that are all NaN leave a sum of NaN
                const float2 v = *reinterpret_cast<const float2*>(&s.sum[k][j][d]);
                o.x = fmaf(v.x, f, o.x), o.y = fmaf(v.y, f, o.y);
            }
            if (whole) {
                const float inv = 1.f / L;
                const int R = qt * NQ + j;
                const size_t at = ((size_t)(lo + token_of(a, R)) * a.heads + head * g + R - token_of(a, R) * g) * kDim + d;
                if constexpr (kF32) *reinterpret_cast<float2*>(static_cast<float*>(a.out) + at) = make_float2(o.x * inv, o.y * inv);
                else *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.out) + at) = pack_bf16(o.x * inv, o.y * inv);
            } else {
                part[d * NQ + j] = o.x, part[(d + 1) * NQ + j] = o.y;
                if (d == 0) part[kDim * NQ + j] = M, part[(kDim + 1) * NQ + j] = L;
            }
        }
        if (!whole) {
            state[slot] = slot == 0 && ends ? 2 : 1;
            if (slot == 1) where[0] = lo, where[1] = qt * NQ, where[2] = rows, where[3] = head;
        }
        __syncthreads();
    }
    if (tid == 0) {
        int* o = parts.info + blockIdx.x * kInfoInts;
        o[0] = state[0], o[1] = state[1];
        for (int i = 0; i < 4; ++i) o[2 + i] = where[i];
    }
}

template <bool kF32, int NQ>
cudaError_t launch(const ChunkArgs& a, const ChunkParts& parts, cudaStream_t st) {
    const size_t smem = sizeof(Shared<NQ>) + (size_t)a.B * sizeof(uint32_t);
    auto kernel = chunk_rows_kernel<kF32, NQ>;
    cudaError_t err = ensure_smem_optin(reinterpret_cast<const void*>(kernel), sizeof(Shared<NQ>) + kChunkMaxRequests * sizeof(uint32_t));
    if (err != cudaSuccess) return err;
    kernel<<<parts.ctas, kThreads, smem, st>>>(a, parts);
    err = cudaGetLastError();
    return err != cudaSuccess ? err : launch_chunk_join(a, parts, st);
}

}  // namespace

cudaError_t launch_chunk_rows(const ChunkArgs& a, const ChunkParts& parts, cudaStream_t st) {
    switch (parts.tile) {
        case 1: return a.bf16 ? launch<false, 1>(a, parts, st) : launch<true, 1>(a, parts, st);
        case 2: return a.bf16 ? launch<false, 2>(a, parts, st) : launch<true, 2>(a, parts, st);
        case 3: return a.bf16 ? launch<false, 3>(a, parts, st) : launch<true, 3>(a, parts, st);
        case 4: return a.bf16 ? launch<false, 4>(a, parts, st) : launch<true, 4>(a, parts, st);
        case 6: return a.bf16 ? launch<false, 6>(a, parts, st) : launch<true, 6>(a, parts, st);
        default: return a.bf16 ? launch<false, 8>(a, parts, st) : launch<true, 8>(a, parts, st);
    }
}

}  // namespace uocr
