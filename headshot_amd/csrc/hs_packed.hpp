// What the kernels over packed and paged sequences share: the sequence that a
// row or a tile belongs to, page lookups, and the host's checks.
#pragma once

#include "hs_common.hpp"

namespace hs {

// Sequence s of packed rows as [begin, end), held to the n rows given whatever
// the offsets hold.
struct RowRange {
    int begin, end;
};
__device__ __forceinline__ RowRange row_range(const int* __restrict__ offsets, int s, int n) {
    const int b = min(max(offsets[s], 0), n);
    return {b, min(max(offsets[s + 1], b), n)};
}

// The sequence that row `row` of the packed rows lies in, or -1: the last one
// that begins at or before the row, if it reaches past it.
__device__ __forceinline__ int sequence_of(const int* __restrict__ offsets, int b, int row) {
    int lo = 0, hi = b;
    while (lo < hi) {  // the first sequence that begins behind the row
        const int mid = (lo + hi) >> 1;
        if (offsets[mid] <= row)
            lo = mid + 1;
        else
            hi = mid;
    }
    return lo > 0 && row < offsets[lo] ? lo - 1 : -1;
}

// Keys of sequence s that its row of the page table has room for.
__device__ __forceinline__ int64_t held_length(const int* __restrict__ lens, int s, int max_pages, int page_shift) {
    const int64_t room = static_cast<int64_t>(max_pages) << page_shift;
    const int64_t len = lens[s];
    return len < 0 ? 0 : len < room ? len : room;
}

// Log2 of a power of two, -1 for anything else.
inline int exact_log2(int32_t v) { return v > 0 && (v & (v - 1)) == 0 ? __builtin_ctz(static_cast<unsigned>(v)) : -1; }

// Rows of `width` elements, `stride` apart, as a byte range's length.
inline int64_t row_bytes(int64_t n, int64_t stride, int64_t width, hs_dtype dt) {
    return n > 0 ? ((n - 1) * stride + width) * dtype_size(dt) : 0;
}

// Shape rules that every entry point over head-vector rows shares.
inline hs_status check_heads(const char* op, hs_dtype dt, int32_t h, int32_t h_kv, int32_t d) {
    if (!valid_dtype(dt)) return fail(HS_EINVAL, "%s: unknown dtype", op);
    if (h < 0 || h_kv <= 0 || h % h_kv != 0)
        return fail(HS_EINVAL, "%s: %d query heads over %d key heads", op, h, h_kv);
    if (h > 4096) return fail(HS_EINVAL, "%s: more than 4096 heads", op);
    if (d != 64 && d != 128) return fail(HS_EUNSUPPORTED, "%s: unsupported head_dim %d", op, d);
    return HS_OK;
}

// Rows of n tokens: a stride that holds a row and keeps every row on a 16-byte
// boundary.
inline hs_status check_rows(const char* op, const char* what, const void* p, int64_t n, int64_t stride, int64_t width,
                            hs_dtype dt) {
    if (n == 0 || width == 0) return HS_OK;
    if (!p) return fail(HS_EINVAL, "%s: null %s", op, what);
    if (stride < width) return fail(HS_EINVAL, "%s: %s rows overlap", op, what);
    if (too_large(n, stride)) return fail(HS_EINVAL, "%s: %s too large", op, what);
    if (!aligned16(p) || stride * dtype_size(dt) % 16 != 0)
        return fail(HS_EUNSUPPORTED, "%s: %s rows must be 16-byte aligned", op, what);
    return HS_OK;
}

}  // namespace hs
