// Moving the page pool's contents: whole pages (uocr_copy_pages: a fork's last page, copy-on-write, a
// defragmented pool) and single rows (uocr_compact_rows: evicted rows dropped). The pool is
// [pages][2 (k, v) x layers = planes][128 rows][row_bytes]; neither operator looks at the elements.
// No counterpart in the reference, whose cache (kv_cache.py:1-40) neither forks nor evicts.
#include <algorithm>

#include "common.cuh"
#include "kernels.h"

namespace uocr {
namespace {

constexpr int kPageRows = 128;
constexpr int kCopyThreads = 256;
constexpr int kCopyUnroll = 4;  // 16-byte words of a thread in flight: 16 KB per CTA

// A plane's first rows[i] rows are contiguous, so entry i is `planes` copies of rows[i] * row_bytes
// bytes. One CTA per 16 KB of a plane; CTAs behind the entry's rows leave at once. Bound: HBM (each
// byte read and written once).
__global__ void __launch_bounds__(kCopyThreads) copy_pages_kernel(char* __restrict__ pool, int pages, int planes,
                                                                  int row_bytes, const int32_t* __restrict__ src,
                                                                  const int32_t* __restrict__ dst,
                                                                  const int32_t* __restrict__ rows) {
    const int i = blockIdx.z;
    const int from = src[i], to = dst[i];
    if ((unsigned)from >= (unsigned)pages || (unsigned)to >= (unsigned)pages || from == to) return;
    const int n = rows ? min(max(rows[i], 0), kPageRows) : kPageRows;
    const int words = n * (row_bytes / 16);
    const int w0 = blockIdx.x * (kCopyThreads * kCopyUnroll) + threadIdx.x;
    const size_t plane_bytes = (size_t)kPageRows * row_bytes;
    const uint4* a = reinterpret_cast<const uint4*>(pool + ((size_t)from * planes + blockIdx.y) * plane_bytes);
    uint4* b = reinterpret_cast<uint4*>(pool + ((size_t)to * planes + blockIdx.y) * plane_bytes);
    uint4 v[kCopyUnroll];
#pragma unroll
    for (int j = 0; j < kCopyUnroll; ++j)
        if (w0 + j * kCopyThreads < words) v[j] = __ldcs(a + w0 + j * kCopyThreads);
#pragma unroll
    for (int j = 0; j < kCopyUnroll; ++j)
        if (w0 + j * kCopyThreads < words) __stcs(b + w0 + j * kCopyThreads, v[j]);
}

struct CompactArgs {
    char* pool;
    const int32_t *src_lut, *dst_lut, *keep, *keep_len;
    int pages, planes, row_bytes, src_cols, dst_cols, max_keep;
};

// New row i of request b is its old row keep[b][i], in every plane. One CTA per request and plane
// walks the request's rows upwards in groups: a group is read, then (after a barrier) written. The
// kept rows ascend, so keep[i] >= i, and a group's writes (rows below its end) touch no source of a
// later group (keep[i'] >= i' >= the group's end): the compaction may be in place.
__global__ void __launch_bounds__(256) compact_rows_kernel(CompactArgs a) {
    const int b = blockIdx.y, plane = blockIdx.x;
    const int n = min(min(max(a.keep_len[b], 0), a.max_keep), a.dst_cols * kPageRows);
    const int words = a.row_bytes / 16;
    const int32_t* keep = a.keep + (size_t)b * a.max_keep;
    for (int i = 0; i < n; ++i) {
        const int k = keep[i];
        if (k < 0 || k >= a.src_cols * kPageRows) continue;  // the same for every thread
        const int from = a.src_lut[(size_t)b * a.src_cols + k / kPageRows];
        const int to = a.dst_lut[(size_t)b * a.dst_cols + i / kPageRows];
        if ((unsigned)from >= (unsigned)a.pages || (unsigned)to >= (unsigned)a.pages) continue;
        const size_t fo = (((size_t)from * a.planes + plane) * kPageRows + k % kPageRows) * a.row_bytes;
        const size_t to_ = (((size_t)to * a.planes + plane) * kPageRows + i % kPageRows) * a.row_bytes;
        if (fo == to_) continue;
        for (int w = threadIdx.x; w < words; w += blockDim.x)  // a thread reads and writes its own words only
            reinterpret_cast<uint4*>(a.pool + to_)[w] = reinterpret_cast<const uint4*>(a.pool + fo)[w];
    }
}

}  // namespace

cudaError_t launch_copy_pages(void* pool, int pages, int layers, int row_bytes, const int32_t* src, const int32_t* dst,
                              const int32_t* rows, int n, cudaStream_t st) {
    if (n <= 0) return cudaSuccess;
    const int words = kPageRows * (row_bytes / 16), per = kCopyThreads * kCopyUnroll;
    for (int i0 = 0; i0 < n; i0 += 65535) {  // the grid's z extent
        const dim3 grid((words + per - 1) / per, 2 * layers, std::min(n - i0, 65535));
        copy_pages_kernel<<<grid, kCopyThreads, 0, st>>>(static_cast<char*>(pool), pages, 2 * layers, row_bytes, src + i0,
                                                         dst + i0, rows ? rows + i0 : nullptr);
    }
    return cudaGetLastError();
}

cudaError_t launch_compact_rows(void* pool, int pages, int layers, int row_bytes, const int32_t* src_lut, int src_cols,
                                const int32_t* dst_lut, int dst_cols, const int32_t* keep, int max_keep,
                                const int32_t* keep_len, int B, cudaStream_t st) {
    if (B <= 0 || max_keep <= 0) return cudaSuccess;
    CompactArgs a{static_cast<char*>(pool), src_lut, dst_lut, keep, keep_len, pages, 2 * layers, row_bytes, src_cols,
                  dst_cols, max_keep};
    compact_rows_kernel<<<dim3(2 * layers, B), 256, 0, st>>>(a);
    return cudaGetLastError();
}

}  // namespace uocr
