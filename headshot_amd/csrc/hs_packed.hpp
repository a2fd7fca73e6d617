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

__device__ __forceinline__ int lane_value(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }

// Sum of v over this lane and the ones before it (DPP: shifts within rows of
// 16, then the rows' sums).
template <int CTRL, int ROW_MASK = 0xF>
__device__ __forceinline__ int dpp_zero(int v) {
    return __builtin_amdgcn_update_dpp(0, v, CTRL, ROW_MASK, 0xF, false);
}
__device__ __forceinline__ int wave_prefix_sum(int v) {
    v += dpp_zero<0x111>(v);  // row_shr 1, 2, 4, 8
    v += dpp_zero<0x112>(v);
    v += dpp_zero<0x114>(v);
    v += dpp_zero<0x118>(v);
    v += dpp_zero<kRowBcast15, 0xA>(v);
    v += dpp_zero<kRowBcast31, 0xC>(v);
    return v;
}

// Which sequence the tile-th tile of bm rows belongs to, all sequences' tiles
// counted one after the other, its rows, and the tile's number within it; false
// past the last. The lengths are device data, so a launch has as many workgroups as
// there can be tiles and each finds its own (64 sequences a step).
__device__ __forceinline__ bool find_tile(const int* __restrict__ offsets, int b, int n, int bm, int tile, int& s,
                                          RowRange& rows, int& local) {
    const int lane = lane_id();
    int before = 0;
    for (int base = 0; base < b; base += 64) {
        int count = 0;
        RowRange r = {};
        if (base + lane < b) {
            r = row_range(offsets, base + lane, n);
            count = static_cast<int>((static_cast<int64_t>(r.end - r.begin) + bm - 1) / bm);
        }
        const int sum = wave_prefix_sum(count);
        const uint64_t hit = __ballot(before + sum > tile);
        if (hit) {
            const int l = __builtin_ctzll(hit);
            s = base + l;
            rows = {lane_value(r.begin, l), lane_value(r.end, l)};
            local = tile - before - (lane_value(sum, l) - lane_value(count, l));
            return true;
        }
        before += lane_value(sum, 63);
    }
    return false;
}

// Keys of sequence s that its row of the page table has room for.
// (max_pages * page is below 2^30.)
__device__ __forceinline__ int held_length(const int* __restrict__ lens, int s, int max_pages, int page_shift) {
    return min(max(lens[s], 0), max_pages << page_shift);
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
    if (stride >= (1 << 22)) return fail(HS_EINVAL, "%s: %s rows of 2^22 elements or more apart", op, what);
    if (too_large(n, stride)) return fail(HS_EINVAL, "%s: %s too large", op, what);
    if (!aligned16(p) || stride * dtype_size(dt) % 16 != 0)
        return fail(HS_EUNSUPPORTED, "%s: %s rows must be 16-byte aligned", op, what);
    return HS_OK;
}

}  // namespace hs
