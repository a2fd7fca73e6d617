// A wave's attention of up to 32 rows over keys of a cache held in 8 bits, kStep keys
// at a time on its own: what single tokens (hs_paged_f8.hip) and tiles of few rows
// (hs_prompts_f8.hip) do between finding their keys and joining their waves.
#pragma once

#include "hs_f8.hpp"

namespace hs {
namespace {

template <typename T, int D, int R>
struct Steps8 {
    static constexpr bool kHalf = sizeof(T) == 2;
    static constexpr int kStep = D == 64 && R == 1 ? 64 : 32;  // keys per wave and step
    static constexpr int kKeys = kPagedWaves * kStep;  // of the workgroup and step
    static constexpr int kParts = kHalf ? 1 : 3;    // of a query value
    static constexpr int kSums = kHalf ? 2 : 3;     // of a weight
    static constexpr int kTiles = kStep / 16;
    static constexpr int KL = D / 64;               // loads of a lane per row of K
    static constexpr int kRowLanes = D / 16;        // lanes per row of V
    static constexpr int kVRows = 64 / kRowLanes;   // rows per load of a wave
    static constexpr int kVLoads = kStep / kVRows;
    static constexpr int kPitch = D + 16;           // (hs_paged.hip)
    static constexpr int kOPitch = D + 4;
};

template <typename T>
__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
    if constexpr (sizeof(T) == 2)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(as_h8(a), as_h8(b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// What attend_steps says of its sums.
constexpr int kLeftOut = 1;  // infinities or NaN went in as zeros
constexpr int kOdd = 2;      // some are no numbers

// Infinities and NaN among the values: a channel's are its sum, in the rows that see
// any. A channel of which all rows see them has a sum that is no number already, but
// maybe another one, since an infinity times a weight of 0, or the parts of one, is
// NaN; so where there are infinities, too, they are added by themselves over all keys,
// else over the steps that left them out. `sums`: the wave's in LDS, rows of kOPitch,
// each lane with its own. (In registers this takes some from the keys' loop: 8 f32
// tokens each of 32 sequences, 32 heads of 128 over 8, 83 us for 76.)
template <typename T, int D, int R, bool MASKED, typename A>
__device__ __forceinline__ void odd_values(const A& a, const int* pages, int kv, int begin, int end, const int (&seen)[R], int least,
                                           int what, float* sums) {
    using P = Steps8<T, D, R>;
    if (__builtin_expect(what == 0, 1)) return;
    const bool all = what & kOdd && any_infinite<T>(a, pages, kv, begin, end);
    if (!all && !(what & kLeftOut)) return;
    const int lane = lane_id(), n = lane & 15, g = lane >> 4;
    float* mine = sums + n * P::kOPitch + 4 * g;
    const auto each = [&](auto f) {
#pragma unroll 1
        for (int x = 0; x < R * D / 4; x++) {
            float* p = mine + x / (D / 4) * 16 * P::kOPitch + x % (D / 4) / 4 * 16 + x % 4;
            *p = f(*p);
        }
    };
    if (all) each(put_aside);
#pragma unroll 1
    for (int key0 = begin + wave_in_block() * P::kStep; key0 < end; key0 += P::kKeys) {
        if (!all && key0 + P::kStep <= least) continue;
#pragma unroll 1
        for (int key = key0; key < min(key0 + P::kStep, end); key++) {
            const Tile16 tile = tile_of(a, pages[key >> a.page_shift], kv, key);
            if (!tile.there) continue;
            const uint8_t* p = static_cast<const uint8_t*>(a.v) + tile.row * D + 4 * g;
            const float scale = scale_value(a.v_scale[tile.row >> a.page_shift]);
            uint32_t w[D / 16];
#pragma unroll
            for (int i = 0; i < D / 16; i++) w[i] = *reinterpret_cast<const uint32_t*>(p + 16 * i);
#pragma unroll
            for (int i = 0; i < D / 16; i++) {
                u32x4 x = values_of<T>(w[i], 0, scale);
                if (!zero_odd<T>(x)) continue;
#pragma unroll 1
                for (int j = 0; j < 4; j++) {
                    const float v = value_of<T>(w[i] >> 8 * j & 0xFFu, scale);
#pragma unroll
                    for (int r = 0; r < R; r++) {
                        float* at = mine + r * 16 * P::kOPitch + 16 * i + j;
                        if (!MASKED || key < seen[r]) *at = with_odd(*at, v);
                    }
                }
            }
        }
    }
    if (all) each(taken_back);
}

// The wave's steps of keys [begin, end): R sets of 16 rows, lane (n, g) with row n
// of each, whose query lies at qr; its sums of channels 16 i + 4 g + .., its largest
// score (log2) and its sum of weights. `vs` is the wave's slice of LDS. MASKED: a row
// sees keys below `seen`, all of them those below `least`, else all see all; in a step
// that some row does not see whole, infinities and NaN go into the sums as zeros, and
// to the rows that see them afterwards (odd_values, which what is returned is for).
// WHOLE: pages of at least 16 keys, so that 16 keys from a multiple of 16 lie in
// one page; else a lane looks one key's up, a step ahead, and rows take it from there
// (by each row, when its codes are asked for: 42 us for 33 of 32 sequences of up to 4000
// keys, 32 heads of 128 over 8, pages of 8).
//
// A lane's 16-byte load of a row of K is 16 dims, two operands of 8: dims 64 i +
// 16 g + 8 e, which the queries follow.
template <typename T, int D, int R, bool WHOLE, bool MASKED, typename A>
__device__ __forceinline__ int attend_steps(const A& a, const int* pages, int kv, int begin, int end, const T* const (&qr)[R],
                                             const int (&seen)[R], int least, uint16_t* vs, f32x4 (&o)[R][D / 16],
                                             float (&m)[R], float (&l)[R]) {
    using P = Steps8<T, D, R>;
    constexpr int kStep = P::kStep, KL = P::KL, kTiles = P::kTiles, DB = D / 16;
    // registers short of what the loop holds (8 tokens each of 32 sequences of up to 4000
    // keys, 32 heads of 128 over 8: 67 us, and 76 without)
    constexpr bool kTight = WHOLE && R == 2 && D == 128 && !P::kHalf;
    const int lane = lane_id(), n = lane & 15, g = lane >> 4;
    bool odd = false;

    // Q^T as the B operand, column n a row; a negative scale is taken as one of -q
    const float c = fmaxf(fabsf(a.scale) * 1.4426950408889634f, 1.4e-45f);
    u32x4 qa[R][2 * KL][P::kParts];
#pragma unroll
    for (int r = 0; r < R; r++)
#pragma unroll
        for (int i = 0; i < 2 * KL; i++) {
            const T* p = qr[r] + 64 * (i / 2) + 16 * g + 8 * (i % 2);
            if constexpr (P::kHalf) {
                qa[r][i][0] = ld16(p);
                if (a.scale < 0.0f) qa[r][i][0] ^= 0x80008000u;
            } else {
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; e++) x[e] = a.scale < 0.0f ? -p[e] : p[e];
                cut3(x, qa[r][i]);
            }
        }

    const uint8_t* kb = static_cast<const uint8_t*>(a.k);
    const uint8_t* vb = static_cast<const uint8_t*>(a.v);
    auto scale_of = [&](const uint8_t* scales, const Tile16& tile) {
        return tile.there ? scales[tile.row >> a.page_shift] : static_cast<uint8_t>(kScaleBias);
    };
    u32x4 kr[kTiles * KL], vr[P::kVLoads];
    // WHOLE: of the step's 16-key tiles, their pages, and the keys up to which
    // those loaded are there; else the lane's key's page, and by row of the lane
    int page[WHOLE ? kTiles : 1], k_end[kTiles], v_end[kTiles];
    uint32_t ks[kTiles], vx[WHOLE ? kTiles : P::kVLoads];  // scales as kept
    uint32_t k_ok = 0, v_ok = 0;
    const int v_row = lane / P::kRowLanes, v_col = lane % P::kRowLanes * 16;
    const uint32_t k_lane = n * D + 16 * g, v_lane = v_row * D + v_col;
    auto find_pages = [&](int key0) {
#pragma unroll
        for (int i = 0; i < (WHOLE ? kTiles : 1); i++)
            page[i] = pages[min(key0 + (WHOLE ? 16 * i : lane % kStep), end - 1) >> a.page_shift];
    };
    auto load_k = [&](int key0) {
        k_ok = 0;
#pragma unroll
        for (int i = 0; i < kTiles; i++) {
            const int key = key0 + 16 * i + (WHOLE ? 0 : n);
            const Tile16 tile = tile_of(a, WHOLE ? page[i] : __shfl(page[0], 16 * i + n, 64), kv, key);
            const uint8_t* p = kb + tile.row * D;
            if constexpr (kTight) p = scalar_address(p);
            p += WHOLE ? k_lane : 16 * g;
#pragma unroll
            for (int x = 0; x < KL; x++) kr[i * KL + x] = ld16_nt(p + 64 * x);
            ks[i] = scale_of(a.k_scale, tile);
            k_end[i] = tile.there ? end : 0;
            if (!WHOLE && tile.there && key < end) k_ok |= 1u << i;
        }
    };
    // of the half-step h, from key key0 + 32 h on
    constexpr int kHalfLoads = P::kVLoads / (kStep / 32);
    auto load_v = [&](int key0, int h) {
        if constexpr (WHOLE) {
            constexpr int kPer = P::kVLoads / kTiles;
#pragma unroll
            for (int i = 2 * h; i < 2 * h + 2; i++) {
                const Tile16 tile = tile_of(a, page[i], kv, key0 + 16 * i);
                const uint8_t* p = vb + tile.row * D;
                if constexpr (kTight) p = scalar_address(p);
#pragma unroll
                for (int x = 0; x < kPer; x++) vr[i * kPer + x] = ld16_nt(p + v_lane + P::kVRows * x * D);
                vx[i] = scale_of(a.v_scale, tile);
                v_end[i] = tile.there ? end : 0;
            }
        } else {
            v_ok &= ~(((1u << kHalfLoads) - 1) << h * kHalfLoads);
#pragma unroll
            for (int i = h * kHalfLoads; i < (h + 1) * kHalfLoads; i++) {
                const int key = key0 + P::kVRows * i + v_row;
                const Tile16 tile = tile_of(a, __shfl(page[0], P::kVRows * i + v_row, 64), kv, key);
                if (tile.there && key < end) v_ok |= 1u << i;
                vr[i] = ld16_nt(vb + tile.row * D + v_col);
                vx[i] = scale_of(a.v_scale, tile);
            }
        }
    };

#pragma unroll
    for (int r = 0; r < R; r++) {
#pragma unroll
        for (int i = 0; i < DB; i++) o[r][i] = f32x4{};
        m[r] = kNone, l[r] = 0.0f;  // l: this lane's keys only
    }
    const int start = begin + wave_in_block() * kStep;
    if (start < end) {
        find_pages(start);
        load_k(start);
#pragma unroll
        for (int h = 0; h < kStep / 32; h++) load_v(start, h);
        find_pages(start + P::kKeys);
    }
#pragma unroll 1
    for (int key0 = start; key0 < end; key0 += P::kKeys) {
        const bool more = key0 + P::kKeys < end;
        // S^T: register j of lane (n, g) is key 16 i + 4 g + j, row n
        f32x4 sc[R][kTiles];
#pragma unroll
        for (int i = 0; i < kTiles; i++) {
            const float scale = scale_value(ks[i]);
            f32x4 acc[R][2] = {};
#pragma unroll
            for (int x = 0; x < 2 * KL; x++) {
                const u32x4& codes = kr[i * KL + x / 2];
                const u32x4 k = values_of<T>(codes[2 * (x % 2)], codes[2 * (x % 2) + 1], scale);
#pragma unroll
                for (int r = 0; r < R; r++)
#pragma unroll
                    for (int p = P::kParts - 1; p >= 0; p--) acc[r][x % 2] = mfma16<T>(k, qa[r][x][p], acc[r][x % 2]);
            }
#pragma unroll
            for (int r = 0; r < R; r++) sc[r][i] = acc[r][0] + acc[r][1];
        }
        // scores of keys that are not there; the lane's are rows 4 g + j, which
        // lanes 4 g + j have looked up
        bool some = false;
#pragma unroll
        for (int i = 0; i < kTiles; i++) {
            if constexpr (WHOLE) {
                if (key0 + 16 * i + 16 > k_end[i]) {
                    const int left = k_end[i] - key0 - 16 * i - 4 * g;
#pragma unroll
                    for (int r = 0; r < R; r++)
#pragma unroll
                        for (int j = 0; j < 4; j++)
                            if (j >= left) sc[r][i][j] = -INFINITY;
                }
                some |= key0 + 16 * i < k_end[i];
            } else {
                const uint64_t there = __ballot(k_ok >> i & 1);
#pragma unroll
                for (int r = 0; r < R; r++)
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        if (!(there >> (4 * g + j) & 1)) sc[r][i][j] = -INFINITY;
                some |= there != 0;
            }
        }
        const bool masked = MASKED && key0 + kStep > least;  // some row does not see all of the step's keys
        if (masked) {
#pragma unroll
            for (int r = 0; r < R; r++)
#pragma unroll
                for (int i = 0; i < kTiles; i++)
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        if (key0 + 16 * i + 4 * g + j >= seen[r]) sc[r][i][j] = -INFINITY;
        }
        if (more) load_k(key0 + P::kKeys);

        // rounded before the maximum is taken off: that one then weighs 1
#pragma unroll
        for (int r = 0; r < R; r++) {
            float mx = -INFINITY;
#pragma unroll
            for (int i = 0; i < kTiles; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    sc[r][i][j] = as_f32(sc[r][i][j] * c);
                    mx = fmaxf(mx, sc[r][i][j]);
                }
            mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
            mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
            const float next = fmaxf(fmaxf(m[r], mx), some ? kFloor : kNone);
            const float corr = __builtin_amdgcn_exp2f(m[r] - next);
            m[r] = next;
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < kTiles; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    sc[r][i][j] = __builtin_amdgcn_exp2f(sc[r][i][j] - m[r]);
                    if constexpr (P::kHalf) sc[r][i][j] *= kHalfUnit;
                    sum += sc[r][i][j];
                }
            l[r] = fmaf(l[r], corr, sum);
#pragma unroll
            for (int i = 0; i < DB; i++) o[r][i] *= corr;
        }
        // O^T += V^T P^T, 32 keys at a time
#pragma unroll
        for (int h = 0; h < kStep / 32; h++) {
            // rows that are not there count as zeros: their weight is 0, and 0
            // times what they hold may not be
            bool gaps = !WHOLE && __any((v_ok >> h * kHalfLoads & ((1u << kHalfLoads) - 1)) != (1u << kHalfLoads) - 1);
#pragma unroll
            for (int i = 2 * h; i < 2 * h + 2; i++) gaps |= WHOLE && key0 + 16 * i + 16 > v_end[i];
            if (gaps) {
#pragma unroll
                for (int i = h * kHalfLoads; i < (h + 1) * kHalfLoads; i++)
                    if (WHOLE ? key0 + P::kVRows * i + v_row >= v_end[P::kVRows * i / 16] : !(v_ok >> i & 1)) vr[i] = u32x4{};
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
            for (int i = h * kHalfLoads; i < (h + 1) * kHalfLoads; i++) {
                const float scale = scale_value(vx[WHOLE ? P::kVRows * i / 16 : i]);
                uint16_t* p = vs + (P::kVRows * (i - h * kHalfLoads) + v_row) * P::kPitch + v_col;
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    u32x4 v = values_of<T>(vr[i][2 * x], vr[i][2 * x + 1], scale);
                    if (masked) odd |= zero_odd<T>(v);
                    st16(p + 8 * x, v);
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            if (more) load_v(key0 + P::kKeys, h);
            u32x4 p[R][P::kSums];
#pragma unroll
            for (int r = 0; r < R; r++) {
                if constexpr (P::kHalf) {
#pragma unroll
                    for (int i = 0; i < 2; i++)
#pragma unroll
                        for (int j = 0; j < 4; j += 2) {
                            const float x = sc[r][2 * h + i][j], y = sc[r][2 * h + i][j + 1];
                            f16x2 w, rest;
                            w.x = static_cast<f16>(x), w.y = static_cast<f16>(y);
                            rest.x = static_cast<f16>(x - static_cast<float>(w.x));
                            rest.y = static_cast<f16>(y - static_cast<float>(w.y));
                            p[r][0][2 * i + j / 2] = h22u(w), p[r][1][2 * i + j / 2] = h22u(rest);
                        }
                } else {
                    float x[8];
#pragma unroll
                    for (int e = 0; e < 8; e++) x[e] = sc[r][2 * h + e / 4][e % 4];
                    cut3(x, p[r]);
                }
            }
            const uint16_t* va = vs + (4 * g + n / 4) * P::kPitch + 4 * (n % 4);
#pragma unroll
            for (int i = 0; i < DB; i++) {
                const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(va + 16 * i)));
                const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(va + 16 * P::kPitch + 16 * i)));
                u32x4 w;
                w[0] = lo[0], w[1] = lo[1], w[2] = hi[0], w[3] = hi[1];
#pragma unroll
                for (int r = 0; r < R; r++)
#pragma unroll
                    for (int x = P::kSums - 1; x >= 0; x--) o[r][i] = mfma16<T>(w, p[r][x], o[r][i]);
            }
        }
        if (more) find_pages(key0 + 2 * P::kKeys);
    }
#pragma unroll
    for (int r = 0; r < R; r++) {
        l[r] += __shfl_xor(l[r], 16, 64);
        l[r] += __shfl_xor(l[r], 32, 64);
    }
    bool wild = false;
#pragma unroll
    for (int r = 0; r < R; r++)
#pragma unroll
        for (int i = 0; i < DB; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) wild |= !(fabsf(o[r][i][j]) < INFINITY);
    return (MASKED && __any(odd) ? kLeftOut : 0) | (__any(wild) ? kOdd : 0);
}

}  // namespace
}  // namespace hs
