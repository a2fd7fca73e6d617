// A paged key-value cache for gfx950: appending new tokens (with QK-norm and
// the position rotation) and the attention of one new token per sequence.
#include <type_traits>

#include "hs_paged.hpp"

namespace hs {
namespace {

template <typename T, int D, bool NORM, bool ROPE>
__global__ __launch_bounds__(256) void kv_append_kernel(AppendArgs<T> a) {
    append_rows<T, D, NORM, ROPE>(a, static_cast<int>(blockIdx.x) * 4 + wave_in_block());
}

template <typename T, int D>
void launch_append(hipStream_t st, const AppendArgs<T>& a) {
    const int64_t units = static_cast<int64_t>(a.n) * a.parts;
    const dim3 grid(static_cast<uint32_t>(ceil_div(units, 4)));
    const bool norm = a.qn_w || a.kn_w, rope = a.sin_tab != nullptr;
    if (norm && rope)
        kv_append_kernel<T, D, true, true><<<grid, dim3(256), 0, st>>>(a);
    else if (norm)
        kv_append_kernel<T, D, true, false><<<grid, dim3(256), 0, st>>>(a);
    else if (rope)
        kv_append_kernel<T, D, false, true><<<grid, dim3(256), 0, st>>>(a);
    else
        kv_append_kernel<T, D, false, false><<<grid, dim3(256), 0, st>>>(a);
}

// ---------------------------------------------------------------------------
// attention_paged
//
// Bandwidth: every key and value is read once, by the workgroup of its
// (sequence, key head, range of keys), for all query heads of that key head (up
// to 16 a pass) at once. A wave takes kStep keys at a time on its own: scores
// transposed on the matrix cores, S^T = K Q^T with the query heads as columns,
// so that lanes n, n + 16, .. share query head n; K straight from memory as the
// A operand; V through the wave's own slice of LDS, from which V^T takes P^T as
// the scores' registers hold it. Loads run a step ahead. The four waves' (O, m,
// l) join in LDS, the ranges of a sequence in a second launch.
//
// 64 sequences of up to 8192 keys, 32 heads of 128 over 8, f16: 179 us, 5.8
// TB/s; one token over 130531 keys of 16 heads of 64 91 us, 5.9 TB/s. 19
// sequences of up to 3001 keys, 28 heads of 64 over 4, 13 us.
//
// Ranges: a sequence's keys are cut into pieces of `chunk` units of 4 kStep
// keys, the same for all sequences of the call. A piece costs some 5 us before
// its first product (lengths, pages, keys: one load behind the other) and a
// unit 1 us, so pieces are as many as the chip holds at once while that leaves
// them up to four units, and then four times as many, which evens their ends
// out. Lengths are device data: each workgroup computes chunk and finds its
// piece from all of them (64 a step).

template <typename T, int D>
struct Paged {
    static constexpr bool kHalf = sizeof(T) == 2;
    static constexpr int kStep = kHalf ? 32 : 16;  // keys per wave and step
    static constexpr int kUnit = kPagedWaves * kStep;
    static constexpr int V = Vec<T>::N;
    static constexpr int kRowLanes = D / V;               // 16-byte pieces of a row
    static constexpr int kVRows = 64 / kRowLanes;         // rows per load of a wave
    static constexpr int kVLoads = kStep / kVRows;
    static constexpr int kKLoads = kStep / 16 * (D * static_cast<int>(sizeof(T)) / 64);
    // LDS pitch of V's rows in elements. f16: the transposing read takes 8 rows
    // of 32 bytes at a time, which start 32 bytes apart modulo the 64 banks;
    // f32: 4 rows of 64 bytes, 4 rows apart.
    static constexpr int kPitch = kHalf ? D + 16 : D + 4;
    static constexpr int kOPitch = D + 4;
    static constexpr int kPerCu = D == 64 ? 4 : 3;  // workgroups, by their registers
    struct Smem {
        union {
            T v[kPagedWaves][kStep * kPitch];
            float o[kPagedWaves][kGroup * kOPitch];
        };
        float m[kPagedWaves][kGroup], l[kPagedWaves][kGroup];
    };
};

// WHOLE: pages of at least 16 keys, so that 16 keys from a multiple of 16 lie in
// one page; else each row looks its own up.
template <typename T, int D, bool WHOLE>
__global__ __launch_bounds__(64 * kPagedWaves, D == 64 ? 4 : 3) void attention_paged_kernel(PagedArgs a) {
    using P = Paged<T, D>;
    constexpr int V = P::V, kStep = P::kStep;
    __shared__ __align__(16) typename P::Smem sm;
    const int lane = lane_id(), wave = wave_in_block();
    const int n = lane & 15, g = lane >> 4;

    Piece t;
    if (!find_piece(a, P::kUnit, t)) return;  // workgroup-uniform, before any barrier
    const int s = t.s, begin = t.begin, end = t.end, count = t.count, kv = t.kv, pass = t.pass;
    const int live_heads = min(a.width, a.group - pass * a.width);
    const int head0 = kv * a.group + pass * a.width;

    // Q^T as the B operand, column n the query head (a copy of the last beyond
    // them); a negative scale is taken as one of -q
    const float c = fmaxf(fabsf(a.scale) * 1.4426950408889634f, 1.4e-45f);
    const T* qr = static_cast<const T*>(a.q) + s * a.q_stride + (head0 + min(n, live_heads - 1)) * D;
    constexpr int KS = D * static_cast<int>(sizeof(T)) / 64;  // 16-byte pieces of a row per lane group
    u32x4 qa[KS];
#pragma unroll
    for (int i = 0; i < KS; i++) {
        qa[i] = ld16(qr + (4 * i + g) * V);
        if (a.scale < 0.0f) qa[i] ^= P::kHalf ? 0x80008000u : 0x80000000u;
    }

    const int* pages = a.page_table + static_cast<int64_t>(s) * a.max_pages;
    const T* kb = static_cast<const T*>(a.k);
    const T* vb = static_cast<const T*>(a.v);
    auto page_of = [&](int key) { return pages[min(key, end - 1) >> a.page_shift]; };
    u32x4 kr[P::kKLoads], vr[P::kVLoads];
    constexpr int kTiles = kStep / 16;
    // WHOLE: of the step's 16-key tiles, their pages, and the keys up to which
    // those loaded are there; else by row of the lane
    int page[kTiles], k_end[kTiles], v_end[kTiles];
    uint32_t k_ok = 0, v_ok = 0;
    const uint32_t k_lane = n * D + g * V, v_lane = lane / P::kRowLanes * D + lane % P::kRowLanes * V;
    auto find_pages = [&](int key0) {
#pragma unroll
        for (int i = 0; i < kTiles; i++) page[i] = page_of(key0 + 16 * i);
    };
    auto load_k = [&](int key0) {
        k_ok = 0;
#pragma unroll
        for (int i = 0; i < kTiles; i++) {
            const int key = key0 + 16 * i + (WHOLE ? 0 : n);
            const Tile16 tile = tile_of(a, WHOLE ? page[i] : page_of(key), kv, key);
            const T* p = kb + tile.row * D + (WHOLE ? k_lane : g * V);
#pragma unroll
            for (int x = 0; x < KS; x++) kr[i * KS + x] = ld16_nt(p + 4 * x * V);
            k_end[i] = tile.there ? end : 0;
            if (!WHOLE && tile.there && key < end) k_ok |= 1u << i;
        }
    };
    auto load_v = [&](int key0) {
        v_ok = 0;
        if constexpr (WHOLE) {
#pragma unroll
            for (int i = 0; i < kTiles; i++) {
                const Tile16 tile = tile_of(a, page[i], kv, key0 + 16 * i);
                const T* p = vb + tile.row * D;
#pragma unroll
                for (int x = 0; x < P::kVLoads / kTiles; x++)
                    vr[i * (P::kVLoads / kTiles) + x] = ld16_nt(p + v_lane + P::kVRows * x * D);
                v_end[i] = tile.there ? end : 0;
            }
        } else {
#pragma unroll
            for (int i = 0; i < P::kVLoads; i++) {
                const int key = key0 + P::kVRows * i + lane / P::kRowLanes;
                const Tile16 tile = tile_of(a, page_of(key), kv, key);
                if (tile.there && key < end) v_ok |= 1u << i;
                vr[i] = ld16_nt(vb + tile.row * D + lane % P::kRowLanes * V);
            }
        }
    };

    constexpr int DB = D / 16;
    f32x4 o[DB];
#pragma unroll
    for (int i = 0; i < DB; i++) o[i] = f32x4{};
    float m = kNone, l = 0.0f;  // l: this lane's keys only
    T* vs = sm.v[wave];
    const int start = begin + wave * kStep;
    if (start < end) {
        if (WHOLE) find_pages(start);
        load_v(start);
        load_k(start);
        if (WHOLE) find_pages(start + P::kUnit);
    }
    for (int key0 = start; key0 < end; key0 += P::kUnit) {
        const bool more = key0 + P::kUnit < end;
        // rows that are not there count as zeros: their weight is 0, and 0
        // times what they hold may not be
        bool gaps = !WHOLE && __any(v_ok != (1u << P::kVLoads) - 1);
#pragma unroll
        for (int i = 0; i < kTiles; i++) gaps |= WHOLE && key0 + 16 * i + 16 > v_end[i];
        if (gaps) {
#pragma unroll
            for (int i = 0; i < P::kVLoads; i++) {
                const int row = P::kVRows * i + lane / P::kRowLanes;
                if (WHOLE ? key0 + row >= v_end[P::kVRows * i / 16] : !(v_ok >> i & 1)) vr[i] = u32x4{};
            }
        }
        bool odd = false;  // f16: an infinity or NaN among the values
        if constexpr (P::kHalf) {
            u16x2 most = {0, 0};
#pragma unroll
            for (int i = 0; i < P::kVLoads; i++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, vr[i][e] & 0x7FFF7FFFu));
            odd = __any(most.x >= 0x7C00 || most.y >= 0x7C00);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int i = 0; i < P::kVLoads; i++)
            st16(vs + (P::kVRows * i + lane / P::kRowLanes) * P::kPitch + lane % P::kRowLanes * V, vr[i]);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (more) load_v(key0 + P::kUnit);

        // S^T: register j of lane (n, g) is key 16 i + 4 g + j, query head n
        f32x4 sc[kStep / 16];
#pragma unroll
        for (int i = 0; i < kStep / 16; i++) {
            f32x4 acc[2] = {f32x4{}, f32x4{}};
#pragma unroll
            for (int x = 0; x < KS; x++) {
                if constexpr (P::kHalf) {
                    acc[0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_h8(kr[i * KS + x]), as_h8(qa[x]), acc[0], 0, 0, 0);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        acc[e % 2] = __builtin_amdgcn_mfma_f32_16x16x4f32(u2f(kr[i * KS + x][e]), u2f(qa[x][e]), acc[e % 2], 0, 0, 0);
                }
            }
            sc[i] = acc[0] + acc[1];
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
                    for (int j = 0; j < 4; j++)
                        if (j >= left) sc[i][j] = -INFINITY;
                }
                some |= key0 + 16 * i < k_end[i];
            } else {
                const uint64_t there = __ballot(k_ok >> i & 1);
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (!(there >> (4 * g + j) & 1)) sc[i][j] = -INFINITY;
                some |= there != 0;
            }
        }
        if (more) {
            load_k(key0 + P::kUnit);
            if (WHOLE) find_pages(key0 + 2 * P::kUnit);
        }

        // rounded before the maximum is taken off: that one then weighs 1
        float mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < kStep / 16; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                sc[i][j] = as_f32(sc[i][j] * c);
                mx = fmaxf(mx, sc[i][j]);
            }
        mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        const float next = fmaxf(fmaxf(m, mx), some ? kFloor : kNone);
        const float corr = __builtin_amdgcn_exp2f(m - next);
        m = next;
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < kStep / 16; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                sc[i][j] = __builtin_amdgcn_exp2f(sc[i][j] - m);
                if constexpr (P::kHalf) sc[i][j] *= kHalfUnit;
                sum += sc[i][j];
            }
        l = fmaf(l, corr, sum);
#pragma unroll
        for (int i = 0; i < DB; i++) o[i] *= corr;
        // O^T += V^T P^T
        if constexpr (P::kHalf) {
            u32x4 p, rest;
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int j = 0; j < 4; j += 2) {
                    f16x2 w, r;
                    w.x = static_cast<f16>(sc[i][j]), w.y = static_cast<f16>(sc[i][j + 1]);
                    r.x = static_cast<f16>(sc[i][j] - static_cast<float>(w.x));
                    r.y = static_cast<f16>(sc[i][j + 1] - static_cast<float>(w.y));
                    p[2 * i + j / 2] = h22u(w), rest[2 * i + j / 2] = h22u(r);
                }
            const T* va = vs + (4 * g + n / 4) * P::kPitch + 4 * (n % 4);
            auto read_v = [&](int i) {
                const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(va + 16 * i)));
                const u32x2 hi =
                    __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(va + 16 * P::kPitch + 16 * i)));
                u32x4 w;
                w[0] = lo[0], w[1] = lo[1], w[2] = hi[0], w[3] = hi[1];
                return as_h8(w);
            };
#pragma unroll
            for (int i = 0; i < DB; i++) {
                const h8 w = read_v(i);
                o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w, as_h8(p), o[i], 0, 0, 0);
                if (!odd) o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w, as_h8(rest), o[i], 0, 0, 0);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int i = 0; i < DB; i++)
                    o[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(vs[(4 * g + j) * P::kPitch + 16 * i + n], sc[0][j], o[i], 0, 0, 0);
        }
    }
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);

    join_waves<T, D, false>(a, sm, s, count, head0, live_heads, o, m, l, [](float*) {});
}

// f32, a key head of one query head (no sharing): the matrix instructions would
// take 2048 cycles for 16 keys of 128 dims, fifteen sixteenths of them for
// columns that are not there, and the vector ones take some 500. Lanes r, r +
// 16, .. hold key row r between them (K) and sum its product by halves and
// quarters; V's rows lie a few to a load, each lane summing its four channels.
// 16 heads of 128, us here and on the matrix instructions: 8 sequences of 400
// keys 15.7, 17.2, of 800 24.5, 28.8, one of 8000 27.6, 30.8 (4.8 TB/s). With
// two query heads to a key head the matrix instructions take 17.3 for 800.
// (16 waves to a workgroup, so that 1024 keys need no second launch, are slower:
// a CU draws some 50 GB/s, and the longest sequence waits for its one.)
template <int D>
struct PagedSingle {
    static constexpr int W = kPagedWaves;
    static constexpr int kUnit = 16 * W;
    static constexpr int kPerCu = 4;
    struct Smem {
        float q[D];  // (registers hold K and V)
        float o[W][D];
        float m[W], l[W];
    };
};

template <int D, bool WHOLE>
__global__ __launch_bounds__(64 * kPagedWaves, 4) void paged_single_kernel(PagedArgs a) {
    using P = PagedSingle<D>;
    constexpr int W = P::W;
    constexpr int KS = D / 16, kRowLanes = D / 4, kVRows = 64 / kRowLanes, kVLoads = 16 / kVRows;
    __shared__ __align__(16) typename P::Smem sm;
    Piece t;
    if (!find_piece(a, P::kUnit, t)) return;  // workgroup-uniform, before any barrier
    const int lane = lane_id(), wave = wave_in_block();
    const int n = lane & 15, g = lane >> 4;
    const float c = a.scale * 1.4426950408889634f;
    if (threadIdx.x < D) sm.q[threadIdx.x] = static_cast<const float*>(a.q)[t.s * a.q_stride + t.kv * D + threadIdx.x];
    const int* pages = a.page_table + static_cast<int64_t>(t.s) * a.max_pages;
    const float* kb = static_cast<const float*>(a.k);
    const float* vb = static_cast<const float*>(a.v);
    auto page_of = [&](int key) { return pages[min(key, t.end - 1) >> a.page_shift]; };
    u32x4 kr[KS], vr[kVLoads];
    bool k_ok = false;
    uint32_t v_ok = 0;  // by load
    int v_end = 0;      // WHOLE: the keys below it are there
    int page = 0;       // WHOLE: of the step's 16 keys
    const uint32_t v_lane = lane / kRowLanes * D + lane % kRowLanes * 4;
    auto load_k = [&](int key0) {
        if constexpr (WHOLE) {
            const Tile16 tile = tile_of(a, page, t.kv, key0);
            k_ok = tile.there && key0 + n < t.end;
            const float* p = kb + tile.row * D;
#pragma unroll
            for (int i = 0; i < KS; i++) kr[i] = ld16_nt(p + (n * D + 4 * g) + 16 * i);
        } else {
            const Tile16 tile = tile_of(a, page_of(key0 + n), t.kv, key0 + n);
            k_ok = tile.there && key0 + n < t.end;
            const float* p = kb + tile.row * D + 4 * g;
#pragma unroll
            for (int i = 0; i < KS; i++) kr[i] = ld16_nt(p + 16 * i);
        }
    };
    auto load_v = [&](int key0) {
        if constexpr (WHOLE) {
            const Tile16 tile = tile_of(a, page, t.kv, key0);
            const float* p = vb + tile.row * D;
#pragma unroll
            for (int i = 0; i < kVLoads; i++) vr[i] = ld16_nt(p + v_lane + kVRows * i * D);
            v_end = tile.there ? t.end : 0;
        } else {
            v_ok = 0;
#pragma unroll
            for (int i = 0; i < kVLoads; i++) {
                const int key = key0 + kVRows * i + lane / kRowLanes;
                const Tile16 tile = tile_of(a, page_of(key), t.kv, key);
                if (tile.there && key < t.end) v_ok |= 1u << i;
                vr[i] = ld16_nt(vb + tile.row * D + lane % kRowLanes * 4);
            }
        }
    };
    float o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    float m = kNone, l = 0.0f;  // l: the lane's key row only
    const int start = t.begin + 16 * wave;
    if (start < t.end) {
        if (WHOLE) page = page_of(start);
        load_k(start);
        load_v(start);
        if (WHOLE) page = page_of(start + P::kUnit);
    }
    __syncthreads();
#pragma unroll 1
    for (int key0 = start; key0 < t.end; key0 += P::kUnit) {
        const bool more = key0 + P::kUnit < t.end;
        float dot[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < KS; i++) {
            const float4 q = ld_f32x4(&sm.q[16 * i + 4 * g]);
            dot[0] = fmaf(u2f(kr[i][0]), q.x, dot[0]);
            dot[1] = fmaf(u2f(kr[i][1]), q.y, dot[1]);
            dot[2] = fmaf(u2f(kr[i][2]), q.z, dot[2]);
            dot[3] = fmaf(u2f(kr[i][3]), q.w, dot[3]);
        }
        float s = (dot[0] + dot[1]) + (dot[2] + dot[3]);
        s += __shfl_xor(s, 16, 64);
        s += __shfl_xor(s, 32, 64);
        // rounded before the maximum is taken off: that one then weighs 1
        s = k_ok ? as_f32(s * c) : -INFINITY;
        const bool some = __any(k_ok);
        if (more) load_k(key0 + P::kUnit);
        float mx = s;
        mx = fmaxf(mx, dpp<kQuadXor1>(mx));
        mx = fmaxf(mx, dpp<kQuadXor2>(mx));
        mx = fmaxf(mx, dpp<kRowHalfMirror>(mx));
        mx = fmaxf(mx, dpp<kRowMirror>(mx));
        const float next = fmaxf(fmaxf(m, mx), some ? kFloor : kNone);
        const float corr = __builtin_amdgcn_exp2f(m - next);
        m = next;
        const float p = __builtin_amdgcn_exp2f(s - m);
        l = fmaf(l, corr, p);
#pragma unroll
        for (int e = 0; e < 4; e++) o[e] *= corr;
        // a row that is not there weighs 0, and 0 times what it holds may not be 0
        if (WHOLE ? key0 + 16 > v_end : __any(v_ok != (1u << kVLoads) - 1)) {
#pragma unroll
            for (int i = 0; i < kVLoads; i++)
                if (WHOLE ? key0 + kVRows * i + lane / kRowLanes >= v_end : !(v_ok >> i & 1)) vr[i] = u32x4{};
        }
#pragma unroll
        for (int i = 0; i < kVLoads; i++) {
            const float w = __shfl(p, kVRows * i + lane / kRowLanes, 64);
#pragma unroll
            for (int e = 0; e < 4; e++) o[e] = fmaf(w, u2f(vr[i][e]), o[e]);
        }
        if (more) {
            load_v(key0 + P::kUnit);
            if (WHOLE) page = page_of(key0 + 2 * P::kUnit);
        }
    }
    l = sum16(l);
#pragma unroll
    for (int e = 0; e < 4; e++) {
        if constexpr (D == 64) o[e] += __shfl_xor(o[e], 16, 64);
        o[e] += __shfl_xor(o[e], 32, 64);
    }
    if (lane < kRowLanes) *reinterpret_cast<f32x4*>(&sm.o[wave][4 * lane]) = f32x4{o[0], o[1], o[2], o[3]};
    if (lane == 0) sm.m[wave] = m, sm.l[wave] = l;
    __syncthreads();
    if (threadIdx.x >= D / 4) return;
    float top = sm.m[0];
#pragma unroll
    for (int w = 1; w < W; w++) top = fmaxf(top, sm.m[w]);
    f32x4 sum = {};
    float weight = 0.0f;
#pragma unroll
    for (int w = 0; w < W; w++) {
        const float f = __builtin_amdgcn_exp2f(sm.m[w] - top);
        sum += *reinterpret_cast<const f32x4*>(&sm.o[w][4 * threadIdx.x]) * f;
        weight = fmaf(sm.l[w], f, weight);
    }
    const int d0 = 4 * threadIdx.x;
    if (t.count == 1) {
        f32x4 x;
#pragma unroll
        for (int e = 0; e < 4; e++) x[e] = top == kNone ? 0.0f : sum[e] / weight;
        *reinterpret_cast<f32x4*>(static_cast<float*>(a.out) + (static_cast<int64_t>(t.s) * a.h + t.kv) * D + d0) = x;
    } else {
        const int64_t row = blockIdx.x;
        *reinterpret_cast<f32x4*>(a.ws_o + row * D + d0) = sum;
        if (d0 == 0) a.ws_ml[2 * row] = top, a.ws_ml[2 * row + 1] = weight;
    }
}

template <typename T, int D>
hs_status launch_paged(const char* op, hipStream_t st, const PagedArgs& a) {
    if constexpr (sizeof(T) == 4) {
        if (a.h == a.h_kv) {
            using P = PagedSingle<D>;
            return launch_pieces<T, D, false>(op, st, a, paged_single_kernel<D, true>, paged_single_kernel<D, false>, P::kUnit, P::kPerCu);
        }
    }
    using P = Paged<T, D>;
    return launch_pieces<T, D, false>(op, st, a, attention_paged_kernel<T, D, true>, attention_paged_kernel<T, D, false>, P::kUnit, P::kPerCu);
}

}  // namespace
}  // namespace hs

extern "C" hs_status hs_kv_append(hs_stream_t stream, hs_dtype dt, const void* q, int64_t q_stride, const void* k,
                                  int64_t k_stride, const void* v, int64_t v_stride, const float* qn_w,
                                  const float* qn_b, const float* kn_w, const float* kn_b, const float* sin_tab,
                                  const float* cos_tab, int32_t table_rows, const void* positions,
                                  const void* offsets, const void* page_table, const void* lens, void* q_out,
                                  void* k_out, void* k_cache, void* v_cache, int64_t n, int32_t b, int32_t h,
                                  int32_t h_kv, int32_t d, int32_t page, int32_t n_pages, int32_t max_pages,
                                  float eps) {
    using namespace hs;
    const char* op = "kv_append";
    AppendCall c{q, k, v, q_stride, k_stride, v_stride, qn_w, qn_b, kn_w, kn_b, sin_tab, cos_tab, table_rows, positions,
                 offsets, page_table, lens, q_out, k_out, n, b, h, h_kv, d, page, n_pages, max_pages, eps};
    bool done = false;
    if (hs_status rc = check_append(op, dt, c, done)) return rc;
    if (done) return HS_OK;
    if (hs_status rc = check_cache(op, k_cache, v_cache, page_table, lens, page, n_pages, max_pages, h_kv, d)) return rc;
    const int64_t cache = static_cast<int64_t>(n_pages) * page * h_kv * d * dtype_size(dt);
    const ByteRange outs[4] = {c.q_rows(dt), c.k_rows(dt), {k_cache, cache}, {v_cache, cache}};
    if (hs_status rc = check_append_overlaps(op, dt, c, outs, 4)) return rc;
    const int64_t heads = static_cast<int64_t>(c.h) + 2 * h_kv;
    // waves per token: as many heads each as two loads hold
    const int parts = static_cast<int>(ceil_div(heads, dt == HS_F16 ? 1024 / d : 512 / d));
    if (n * parts >= (int64_t{1} << 26)) return fail(HS_EINVAL, "%s: too many tokens", op);
    const auto run = [&](auto zero) {
        using T = decltype(zero);
        AppendArgs<T> a;
        c.fill(a);
        a.k_cache = static_cast<T*>(k_cache), a.v_cache = static_cast<T*>(v_cache);
        a.parts = parts, a.heads = static_cast<int>(heads);
        if (d == 64)
            launch_append<T, 64>(static_cast<hipStream_t>(stream), a);
        else
            launch_append<T, 128>(static_cast<hipStream_t>(stream), a);
    };
    if (dt == HS_F16)
        run(f16{});
    else
        run(float{});
    return check_launch(op);
}

extern "C" int64_t hs_attention_paged_workspace(int32_t b, int32_t h, int32_t h_kv, int32_t d) {
    if (b <= 0 || h <= 0 || h > 4096 || h_kv <= 0 || h % h_kv != 0 || (d != 64 && d != 128)) return 0;
    using namespace hs;
    if (static_cast<int64_t>(b) * h >= (int64_t{1} << 23)) return 0;
    return PagedPlan(b, h, h_kv, kMostPerCu).rows * (d + 2) * 4 + static_cast<int64_t>(b) * 8;
}

extern "C" hs_status hs_attention_paged(hs_stream_t stream, hs_dtype dt, const void* q, int64_t q_stride,
                                        const void* k_cache, const void* v_cache, const void* page_table,
                                        const void* lens, void* out, void* workspace, int64_t workspace_bytes,
                                        int32_t b, int32_t h, int32_t h_kv, int32_t d, int32_t page,
                                        int32_t n_pages, int32_t max_pages, float scale) {
    using namespace hs;
    const char* op = "attention_paged";
    if (hs_status rc = check_heads(op, dt, h, h_kv, d)) return rc;
    if (b < 0) return fail(HS_EINVAL, "%s: negative count", op);
    if (b == 0 || h == 0) return HS_OK;
    if (static_cast<int64_t>(b) * h >= (int64_t{1} << 23)) return fail(HS_EINVAL, "%s: b * Hq must be below 2^23", op);
    const int64_t width = static_cast<int64_t>(h) * d;
    if (hs_status rc = check_rows(op, "q", q, b, q_stride, width, dt)) return rc;
    if (!out) return fail(HS_EINVAL, "%s: null out", op);
    if (hs_status rc = check_cache(op, k_cache, v_cache, page_table, lens, page, n_pages, max_pages, h_kv, d)) return rc;
    if (!aligned16(out) || !aligned16(workspace)) return fail(HS_EUNSUPPORTED, "%s: out and workspace must be 16-byte aligned", op);
    const int64_t need = hs_attention_paged_workspace(b, h, h_kv, d);
    if (need > 0 && (!workspace || workspace_bytes < need))
        return fail(HS_EINVAL, "%s: workspace of %lld bytes, %lld needed", op, static_cast<long long>(workspace_bytes), static_cast<long long>(need));
    const int64_t e = dtype_size(dt), cache = static_cast<int64_t>(n_pages) * page * h_kv * d * e;
    const int64_t in_bytes = row_bytes(b, q_stride, width, dt), out_bytes = b * width * e;
    if (overlaps(out, out_bytes, q, in_bytes) || overlaps(out, out_bytes, k_cache, cache) || overlaps(out, out_bytes, v_cache, cache) ||
        overlaps(out, out_bytes, workspace, need))
        return fail(HS_EINVAL, "%s: out overlaps another buffer", op);
    if (overlaps(workspace, need, q, in_bytes) || overlaps(workspace, need, k_cache, cache) || overlaps(workspace, need, v_cache, cache))
        return fail(HS_EINVAL, "%s: workspace overlaps an input", op);
    if (!std::isfinite(scale)) return fail(HS_EINVAL, "%s: scale must be finite", op);
    PagedArgs a;
    a.q = q, a.k = k_cache, a.v = v_cache, a.out = out, a.q_stride = q_stride;
    a.ws_o = static_cast<float*>(workspace);
    a.page_table = static_cast<const int*>(page_table), a.lens = static_cast<const int*>(lens);
    a.b = b, a.h = h, a.h_kv = h_kv, a.page_shift = exact_log2(page), a.n_pages = n_pages;
    a.max_pages = n_pages > 0 ? max_pages : 0;  // no page to read: no sequence has keys
    a.scale = scale;
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (dt == HS_F16) return d == 64 ? launch_paged<f16, 64>(op, st, a) : launch_paged<f16, 128>(op, st, a);
    return d == 64 ? launch_paged<float, 64>(op, st, a) : launch_paged<float, 128>(op, st, a);
}
