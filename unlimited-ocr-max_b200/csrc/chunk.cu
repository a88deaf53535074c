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
#include <algorithm>

#include "common.cuh"
#include "kernels.h"

namespace uocr {
namespace {

constexpr int kPageRows = 128;
constexpr int kDim = 128;

UOCR_DEV float4 load4(const float* p) { return *reinterpret_cast<const float4*>(p); }
UOCR_DEV float4 load4(const uint16_t* p) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    return make_float4(bf16lo(v.x), bf16hi(v.x), bf16lo(v.y), bf16hi(v.y));
}
UOCR_DEV void store4(float* p, float4 v) { *reinterpret_cast<float4*>(p) = v; }
UOCR_DEV void store4(uint16_t* p, float4 v) {
    *reinterpret_cast<uint2*>(p) = make_uint2((uint32_t)f32_to_bf16_rne(v.x) | (uint32_t)f32_to_bf16_rne(v.y) << 16,
                                              (uint32_t)f32_to_bf16_rne(v.z) | (uint32_t)f32_to_bf16_rne(v.w) << 16);
}

// Request b's new rows [lo, hi), clamped into the call's T rows.
UOCR_DEV void request_rows(const ChunkArgs& a, int b, int& lo, int& hi) {
    lo = min(max(a.offsets[b], 0), a.T);
    hi = min(max(a.offsets[b + 1], lo), a.T);
}

// The request whose rows hold row t, or -1 (a row in front of the first or behind the last request).
UOCR_DEV int request_of(const ChunkArgs& a, int t) {
    int lo = 0, hi = a.B;
    while (lo < hi) {  // the last b with offsets[b] <= t
        const int mid = (lo + hi) / 2;
        if (a.offsets[mid + 1] <= t) lo = mid + 1; else hi = mid;
    }
    return lo < a.B && a.offsets[lo] <= t ? lo : -1;
}

template <typename E>
UOCR_DEV E* pool_row(const ChunkArgs& a, int b, int kv, int row, int head, uint32_t page) {
    return static_cast<E*>(a.pool) + ((((size_t)page * 2 + kv) * a.layers + a.layer) * kPageRows + row % kPageRows) *
                                         ((size_t)a.kv_heads * kDim) +
           (size_t)head * kDim;
}

// The simplest form: a warp per (new row, head), lane l holding dimensions 4l .. 4l + 3, one visible
// row at a time with a running maximum. Bound by the shuffles of the dot products.
template <typename E>
__global__ void __launch_bounds__(256) chunk_rows_kernel(ChunkArgs a) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long unit = (long long)blockIdx.x * 8 + warp;
    const int t = (int)(unit / a.heads), h = (int)(unit % a.heads);
    if (t >= a.T) return;
    const int b = request_of(a, t);
    if (b < 0) return;
    int lo, hi;
    request_rows(a, b, lo, hi);
    if (t < lo || t >= hi) return;
    const int cap = a.lut_cols * kPageRows;
    const int start = min(max(a.start[b], 0), cap), p = start + (t - lo);
    const int g = a.heads / a.kv_heads, hk = h / g;
    const uint32_t* lut = a.lut + (size_t)b * a.lut_cols;
    const E* kn = static_cast<const E*>(a.k);
    const E* vn = static_cast<const E*>(a.v);
    if (h % g == 0 && p < cap && lut[p / kPageRows] < (uint32_t)a.pages) {
        store4(pool_row<E>(a, b, 0, p, hk, lut[p / kPageRows]) + 4 * lane, load4(kn + (size_t)t * a.k_ld + hk * kDim + 4 * lane));
        store4(pool_row<E>(a, b, 1, p, hk, lut[p / kPageRows]) + 4 * lane, load4(vn + (size_t)t * a.v_ld + hk * kDim + 4 * lane));
    }
    const float4 q = load4(static_cast<const E*>(a.q) + (size_t)t * a.q_ld + h * kDim + 4 * lane);
    const int first = a.prefix ? a.prefix[b] : 0;
    const int low = a.window > 0 ? max(0, p - a.window + 1) : 0;
    float m = -INFINITY, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int r = low > 0 && first <= 0 ? low : 0; r <= p; ++r) {
        if (r < low && r >= first) {
            r = low - 1;
            continue;
        }
        float4 k, v;
        if (r >= start) {
            k = load4(kn + (size_t)(lo + r - start) * a.k_ld + hk * kDim + 4 * lane);
            v = load4(vn + (size_t)(lo + r - start) * a.v_ld + hk * kDim + 4 * lane);
        } else {
            const uint32_t page = min(lut[r / kPageRows], (uint32_t)(a.pages - 1));
            k = load4(pool_row<E>(a, b, 0, r, hk, page) + 4 * lane);
            v = load4(pool_row<E>(a, b, 1, r, hk, page) + 4 * lane);
        }
        float s = warp_sum_butterfly(q.x * k.x + q.y * k.y + q.z * k.z + q.w * k.w) * a.scale;
        const float mn = fmaxf(m, s), keep = expf(m - mn), w = expf(s - mn);
        l = l * keep + w;
        o.x = o.x * keep + w * v.x, o.y = o.y * keep + w * v.y;
        o.z = o.z * keep + w * v.z, o.w = o.w * keep + w * v.w;
        m = mn;
    }
    const float inv = 1.f / l;
    store4(static_cast<E*>(a.out) + ((size_t)t * a.heads + h) * kDim + 4 * lane,
           make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
}

}  // namespace

size_t chunk_workspace_bytes(int sms) { return 0; }

cudaError_t launch_chunk_attention(const ChunkArgs& a, void* ws, int sms, cudaStream_t st) {
    if (a.B <= 0 || a.T <= 0) return cudaSuccess;
    const int grid = (int)(((long long)a.T * a.heads + 7) / 8);
    if (a.bf16) chunk_rows_kernel<uint16_t><<<grid, 256, 0, st>>>(a);
    else chunk_rows_kernel<float><<<grid, 256, 0, st>>>(a);
    return cudaGetLastError();
}

}  // namespace uocr
