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
// byte read and written once): 64 pages of 15.7 MB in 298 us, 6.8 TB/s; 8 tails of 7 to
// 123 rows, 131 MB, in 20.2 us, 6.5 TB/s.
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
    int lanes;   // words (16 bytes) of a row that a CTA moves: a power of two, at most 64
    int slices;  // CTAs across a row
};

constexpr int kMoveThreads = 256;
constexpr int kMoveUnroll = 8;  // words of a thread in flight: 32 KB per CTA
constexpr int kScanUnroll = 4;

// New row i of request b is its old row keep[b][i], in every plane. The kept rows ascend, so keep[i] >= i; rows up to
// the first that changes place stay. A CTA moves `lanes` words of a plane's rows, in groups: a group is read, then
// (after a barrier) written. Its writes (rows below the group's end) touch no source of a later group
// (keep[i'] >= i' >= that end), so walking upwards compacts in place; with a slice and plane to itself the
// CTA needs no order against others. Where no row to move lies below the rows written (keep[first] >= n), or the
// tables share no page, the groups are independent and the rows are dealt to `splits` CTAs. Bound: HBM (each moved
// row read and written once): 609 MB in 99.7 us, 6.1 TB/s; few rows by three dependent reads (kept rows, tables, rows).
__global__ void __launch_bounds__(kMoveThreads) compact_rows_kernel(CompactArgs a, int splits) {
    __shared__ long long from[2][kMoveThreads * kMoveUnroll / 16], to[2][kMoveThreads * kMoveUnroll / 16];
    __shared__ int first_shared;
    const int b = blockIdx.z, plane = blockIdx.y, slice = blockIdx.x % a.slices, split = blockIdx.x / a.slices;
    const int tid = threadIdx.x;
    const int n = min(min(max(a.keep_len[b], 0), a.max_keep), a.dst_cols * kPageRows);
    const int32_t* keep = a.keep + (size_t)b * a.max_keep;
    const int32_t* src = a.src_lut + (size_t)b * a.src_cols;
    const int32_t* dst = a.dst_lut + (size_t)b * a.dst_cols;
    // the first row that changes place
    if (tid == 0) first_shared = n;
    __syncthreads();
    for (int i0 = 0; i0 < n; i0 += kMoveThreads * kScanUnroll) {
        int k[kScanUnroll];  // in flight together: a load at a time costs 1 us for every 256 rows that stay
#pragma unroll
        for (int u = 0; u < kScanUnroll; ++u) {
            const int i = i0 + u * kMoveThreads + tid;
            k[u] = i < n ? keep[i] : 0;
        }
        int at = n;
#pragma unroll
        for (int u = kScanUnroll - 1; u >= 0; --u) {
            const int i = i0 + u * kMoveThreads + tid;
            if (i < n && (k[u] != i || i >= a.src_cols * kPageRows || src[i / kPageRows] != dst[i / kPageRows])) at = i;
        }
        at = __reduce_min_sync(0xffffffffu, at);
        if ((tid & 31) == 0 && at < n) atomicMin(&first_shared, at);
        if (__syncthreads_or(at < n)) break;
    }
    const int first = first_shared;
    if (first >= n) return;
    int begin = first, end = n;
    bool ordered = false;
    if (keep[first] < n) {  // a row to move may be one that is written: do the tables share a page?
        const int used = (n + kPageRows - 1) / kPageRows;
        bool shared = src == dst;
        for (int c = tid; !shared && c < a.src_cols; c += kMoveThreads) {
            const int page = src[c];
            for (int k = first / kPageRows; k < used; ++k) shared |= dst[k] == page;
        }
        ordered = __syncthreads_or(shared);
    }
    const int per = kMoveThreads / a.lanes, group = per * kMoveUnroll;  // rows at a time, rows of a group
    if (ordered) {
        if (split) return;
    } else {
        const int groups = (n - first + group - 1) / group, share = (groups + splits - 1) / splits * group;
        begin = first + split * share, end = min(n, begin + share);
        if (begin >= end) return;
    }
    const int word = slice * a.lanes + tid % a.lanes, row = tid / a.lanes;
    const bool live = word < a.row_bytes / 16;
    char* base = a.pool + (size_t)plane * kPageRows * a.row_bytes + (size_t)word * 16;
    // where the rows of the group at i0 lie (-1: not moved)
    auto locate = [&](int i0, int buf) {
        for (int r = tid; r < group; r += kMoveThreads) {
            const int i = i0 + r, k = i < end ? keep[i] : -1;
            long long f = -1, t = -1;
            if (k >= 0 && k < a.src_cols * kPageRows) {
                const int p = src[k / kPageRows], q = dst[i / kPageRows];
                if ((unsigned)p < (unsigned)a.pages && (unsigned)q < (unsigned)a.pages) {
                    f = ((long long)p * a.planes * kPageRows + k % kPageRows) * a.row_bytes;
                    t = ((long long)q * a.planes * kPageRows + i % kPageRows) * a.row_bytes;
                    if (f == t) f = -1;
                }
            }
            from[buf][r] = f, to[buf][r] = t;
        }
    };
    locate(begin, 0);
    __syncthreads();
    int buf = 0;
    for (int i0 = begin; i0 < end; i0 += group, buf ^= 1) {
        uint4 v[kMoveUnroll];
#pragma unroll
        for (int u = 0; u < kMoveUnroll; ++u) {
            const long long f = from[buf][u * per + row];
            if (live && f >= 0) v[u] = *reinterpret_cast<const uint4*>(base + f);
        }
        if (i0 + group < end) locate(i0 + group, buf ^ 1);
        __syncthreads();  // the group has been read, and the next one's rows are located
#pragma unroll
        for (int u = 0; u < kMoveUnroll; ++u) {
            const int r = u * per + row;
            if (live && from[buf][r] >= 0) *reinterpret_cast<uint4*>(base + to[buf][r]) = v[u];
        }
        __syncthreads();  // from and to of this group are free again
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
                  dst_cols, max_keep, 0, 0};
    const int words = row_bytes / 16;
    a.lanes = 16;
    while (a.lanes < 64 && a.lanes < words) a.lanes *= 2;
    a.slices = (words + a.lanes - 1) / a.lanes;
    // About 8 CTAs per SM, none with less than a group: 128 of 640 rows moved, 12 layers of 10 heads, 10.4 us (16 per SM 13.4,
    // 4 per SM 8.4); 8 requests of 2320 rows, 4 layers of 8 heads in bf16, 99.7 us (99.7, 103).
    const int group = kMoveThreads / a.lanes * kMoveUnroll;
    const long long others = (long long)a.slices * a.planes * B, wanted = (148 * 8 + others - 1) / others;
    const int splits = (int)std::max<long long>(1, std::min<long long>(wanted, (max_keep + group - 1) / group));
    compact_rows_kernel<<<dim3(a.slices * splits, a.planes, B), kMoveThreads, 0, st>>>(a, splits);
    return cudaGetLastError();
}

}  // namespace uocr
