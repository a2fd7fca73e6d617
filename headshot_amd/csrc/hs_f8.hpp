// A cache held in 8 bits: e4m3 codes (sign, 4 bits of exponent, 3 of mantissa;
// no infinities, one NaN a sign) and, for each page and head, one scale 2^(c -
// 127) of which c is kept (E8M0). A code times a scale has 4 significant bits, so
// bf16 holds it as it is, whatever the scale, and f16 from 2^-14 to its largest; below,
// f16 rounds it to a multiple of 2^-24, as it would have rounded the row.
#pragma once

#include "hs_paged.hpp"

namespace hs {
namespace {

constexpr int kScaleBias = 127;
constexpr int kScaleLeast = kScaleBias - 117;  // 448 2^-117: codes from 2^-126
constexpr int kScaleMost = kScaleBias + 120;

// The largest magnitude that a cache of T's rows holds, 15/8 2^15 and 15/8 2^127:
// what would round to the next code is no T. (f16's own largest, 65504, is as far
// from it as any value may be from its code, 2^-4.)
template <typename T>
constexpr float kHeldMost = sizeof(T) == 2 ? 61440.0f : 3.1901471898837979e38f;

__device__ __forceinline__ float scale_value(uint32_t c) { return u2f(c << 23); }

// Kept form of the least scale 2^e with most <= 448 2^e = 7/8 2^(e + 9), most
// finite: its exponent less 8, or less 9 up to 7/8 of the next power of two.
__device__ __forceinline__ int scale_for(float most) {
    const uint32_t b = f2u(most);
    const int e = static_cast<int>(b >> 23) - 8 + ((b & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    return max(e, kScaleLeast);
}

// 8 codes to 8 halves of T, times a scale.
__device__ __forceinline__ u32x4 f16_of_codes(uint32_t lo, uint32_t hi, float scale) {
    u32x4 r;
    r[0] = h22u(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, scale, false));
    r[1] = h22u(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, scale, true));
    r[2] = h22u(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, scale, false));
    r[3] = h22u(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, scale, true));
    return r;
}
__device__ __forceinline__ u32x4 bf16_of_codes(uint32_t lo, uint32_t hi, float scale) {
    u32x4 r;
    r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false));
    r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true));
    r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false));
    r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true));
    return r;
}

// As a cache of T's rows takes them to the matrix cores.
template <typename T>
__device__ __forceinline__ u32x4 values_of(uint32_t lo, uint32_t hi, float scale) {
    return sizeof(T) == 2 ? f16_of_codes(lo, hi, scale) : bf16_of_codes(lo, hi, scale);
}

// A scalar address that stays one beside a lane's offset: the compiler keeps their sum,
// two registers of every lane's, where it can.
__device__ __forceinline__ const uint8_t* scalar_address(const uint8_t* p) {
    auto global = (const __attribute__((address_space(1))) uint8_t*)p;
    asm("" : "+s"(global));
    return (const uint8_t*)global;
}

// One code, as values_of has it.
template <typename T>
__device__ __forceinline__ float value_of(uint32_t code, float scale) {
    const u32x4 x = values_of<T>(code, 0, scale);
    return sizeof(T) == 2 ? static_cast<float>(u2h2(x[0]).x) : u2f(x[0] << 16);
}

// Infinities and NaN among 8 values turned into zeros; whether there were any.
template <typename T>
__device__ __forceinline__ bool zero_odd(u32x4& x) {
    constexpr uint32_t kExp = sizeof(T) == 2 ? 0x7C00u : 0x7F80u;
    bool any = false;
#pragma unroll
    for (int w = 0; w < 4; w++) {
        const uint32_t keep = ((x[w] & kExp) == kExp ? 0u : 0xFFFFu) | ((x[w] & kExp << 16) == kExp << 16 ? 0u : 0xFFFF0000u);
        any |= keep != 0xFFFFFFFFu;
        x[w] &= keep;
    }
    return any;
}

// The least scale, as kept, with which a code passes f16 (448 2^8) or bf16 (448
// 2^120), which makes it infinite.
template <typename T>
constexpr uint32_t kScaleWide = kScaleBias + (sizeof(T) == 2 ? 8 : 120);

// Whether there can be infinite ones among the values of keys [begin, end). All lanes
// of the wave call it.
template <typename T, typename A>
__device__ __forceinline__ bool any_infinite(const A& a, const int* pages, int kv, int begin, int end) {
    bool any = false;
    for (int i = (begin >> a.page_shift) + lane_id(); begin < end && i <= (end - 1) >> a.page_shift; i += 64) {
        const int p = pages[i];
        if (p >= 0 && p < a.n_pages) any |= a.v_scale[static_cast<int64_t>(p) * a.h_kv + kv] >= kScaleWide<T>;
    }
    return __any(any);
}

// A sum that is no number is put aside as a NaN that nothing else makes, which the
// first infinity or NaN among its values replaces; the others add up. What is left of
// those is what the sum was.
constexpr uint32_t kAside = 0x7FC0DE00u;
__device__ __forceinline__ float put_aside(float x) { return fabsf(x) < INFINITY ? x : u2f(kAside | (x != x ? 0u : x > 0.0f ? 1u : 2u)); }
__device__ __forceinline__ float with_odd(float sum, float v) {
    return fabsf(v) < INFINITY ? sum : (f2u(sum) & ~3u) == kAside ? v : sum + v;
}
__device__ __forceinline__ float taken_back(float x) {
    const uint32_t was = f2u(x) & 3u;
    return (f2u(x) & ~3u) != kAside ? x : was == 0 ? u2f(0x7FC00000u) : was == 1 ? INFINITY : -INFINITY;
}

// 4 values to 4 codes, rounded to nearest even. (In range: a finite value past
// 448 would become NaN.)
__device__ __forceinline__ uint32_t codes_of(float a, float b, float c, float d) {
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, lo, true));
}

// 4 codes times 2^-down, rounded again.
__device__ __forceinline__ uint32_t codes_down(uint32_t w, int down) {
    const float f = u2f(static_cast<uint32_t>(127 - min(down, 126)) << 23);
    const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
    return codes_of(lo.x * f, lo.y * f, hi.x * f, hi.y * f);
}

// 8 f32 values in parts whose sum they are, 8 leading bits each (cut, not rounded:
// what is left is exact, and a value near f32's largest stays one).
__device__ __forceinline__ void cut3(const float (&x)[8], u32x4 (&part)[3]) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        uint32_t a = f2u(x[2 * i]), b = f2u(x[2 * i + 1]);
#pragma unroll
        for (int p = 0; p < 3; p++) {
            part[p][i] = __builtin_amdgcn_perm(b, a, 0x07060302u);
            if (p < 2) {
                a = f2u(u2f(a) - u2f(a & 0xFFFF0000u));
                b = f2u(u2f(b) - u2f(b & 0xFFFF0000u));
            }
        }
    }
}

// The host's checks of such a cache.
[[maybe_unused]] hs_status check_cache_f8(const char* op, const void* k_cache, const void* v_cache, const void* k_scale,
                                          const void* v_scale, const void* page_table, const void* lens, int32_t page,
                                          int32_t n_pages, int32_t max_pages, int32_t h_kv, int32_t d) {
    if (hs_status rc = check_cache(op, k_cache, v_cache, page_table, lens, page, n_pages, max_pages, h_kv, d)) return rc;
    if (n_pages > 0 && (!k_scale || !v_scale)) return fail(HS_EINVAL, "%s: null scales", op);
    return HS_OK;
}

// A call that attends over such a cache, n rows of q.
struct AttendCall {
    const void* q;
    int64_t q_stride;
    const void *k_cache, *v_cache, *k_scale, *v_scale, *page_table, *lens;
    void *out, *workspace;
    int64_t workspace_bytes, n;
    int32_t h, h_kv, d, page, n_pages, max_pages;
    float scale;
};

[[maybe_unused]] hs_status check_attend_f8(const char* op, hs_dtype dt, const AttendCall& c, int64_t need) {
    const int64_t width = static_cast<int64_t>(c.h) * c.d;
    if (hs_status rc = check_rows(op, "q", c.q, c.n, c.q_stride, width, dt)) return rc;
    if (!c.out) return fail(HS_EINVAL, "%s: null out", op);
    if (hs_status rc = check_cache_f8(op, c.k_cache, c.v_cache, c.k_scale, c.v_scale, c.page_table, c.lens, c.page, c.n_pages, c.max_pages, c.h_kv, c.d))
        return rc;
    if (!aligned16(c.out) || !aligned16(c.workspace)) return fail(HS_EUNSUPPORTED, "%s: out and workspace must be 16-byte aligned", op);
    if (need > 0 && (!c.workspace || c.workspace_bytes < need))
        return fail(HS_EINVAL, "%s: workspace of %lld bytes, %lld needed", op, static_cast<long long>(c.workspace_bytes), static_cast<long long>(need));
    const int64_t scales = static_cast<int64_t>(c.n_pages) * c.h_kv, codes = scales * c.page * c.d, bytes = c.n * width * dtype_size(dt);
    const ByteRange in[5] = {{c.q, row_bytes(c.n, c.q_stride, width, dt)}, {c.k_cache, codes}, {c.v_cache, codes}, {c.k_scale, scales}, {c.v_scale, scales}};
    for (const ByteRange& r : in) {
        if (overlaps(c.out, bytes, r.p, r.bytes)) return fail(HS_EINVAL, "%s: out overlaps another buffer", op);
        if (overlaps(c.workspace, need, r.p, r.bytes)) return fail(HS_EINVAL, "%s: workspace overlaps an input", op);
    }
    if (overlaps(c.out, bytes, c.workspace, need)) return fail(HS_EINVAL, "%s: out overlaps another buffer", op);
    if (!std::isfinite(c.scale)) return fail(HS_EINVAL, "%s: scale must be finite", op);
    return HS_OK;
}

}  // namespace
}  // namespace hs
