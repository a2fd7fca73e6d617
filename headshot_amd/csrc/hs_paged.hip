// A paged key-value cache for gfx950: appending new tokens (with QK-norm and
// the position rotation) and the attention of one new token per sequence.
#include <cmath>
#include <type_traits>

#include "hs_packed.hpp"

namespace hs {
namespace {

// ---------------------------------------------------------------------------
// kv_append
//
// Bandwidth: one pass over the rows. A wave takes one token and up to two loads
// of its heads, q | k | v one after the other, so there are many waves with a
// few loads each (6 a token: 16381 tokens of 48 heads of 128 f16, rotated, 76
// us, 5.8 TB/s; 82 with one wave a token). A head vector is spread over G lanes.
// Two chunks each, [c, c + V) and [D/2 + c, .. + V) with V elements per 16-byte
// load, put a rotation's pair into one lane and make a norm one G-lane sum of
// both. f16 vectors of 64 are a 128-byte line, which two such loads would touch
// by halves: there a lane takes one chunk, the upper half's in reverse, so that a
// pair sits in mirror lanes, and two heads instead (10992 tokens of 48 heads,
// QK-norm: 32 us, 5.0 TB/s; 42 by halves). A step's few tokens take 3-5 us, a
// chain of four loads.

template <int G>
__device__ __forceinline__ float lanes_sum(float v) {
    v += dpp<kQuadXor1>(v);
    v += dpp<kQuadXor2>(v);
    if constexpr (G >= 8) v += dpp<kRowHalfMirror>(v);
    if constexpr (G >= 16) v += dpp<kRowMirror>(v);
    return v;
}

template <typename T>
struct AppendArgs {
    const T *q, *k, *v;
    int64_t q_stride, k_stride, v_stride;
    const float *qn_w, *qn_b, *kn_w, *kn_b, *sin_tab, *cos_tab;
    const int *positions, *offsets, *page_table, *lens;
    T *q_out, *k_out, *k_cache, *v_cache;
    int n, b, h, h_kv, table_rows, page_shift, n_pages, max_pages, parts;
    float eps;
};

template <typename T, int D, bool NORM, bool ROPE>
__global__ __launch_bounds__(256) void kv_append_kernel(AppendArgs<T> a) {
    constexpr bool kLine = sizeof(T) == 2 && D == 64;  // one chunk per lane and head
    constexpr int V = Vec<T>::N, G = kLine ? D / V : D / (2 * V), HPW = 64 / G * (kLine ? 2 : 1);
    const int unit = static_cast<int>(blockIdx.x) * 4 + wave_in_block();
    const int token = unit / a.parts;
    if (token >= a.n) return;  // wave-uniform; no barriers
    int s = token, pos;
    if (a.offsets) {
        s = sequence_of(a.offsets, a.b, token);
        if (s < 0) return;
        pos = a.lens[s] - (a.offsets[s + 1] - token);
    } else {
        pos = a.lens[s] - 1;
    }
    // the token's place: row `slot` of each head's page, or none
    const int entry = pos >> a.page_shift;
    int page = -1;
    if (pos >= 0 && entry < a.max_pages) page = a.page_table[static_cast<int64_t>(s) * a.max_pages + entry];
    const bool placed = page >= 0 && page < a.n_pages;
    const int64_t slot = pos & ((1 << a.page_shift) - 1);

    const int lane = lane_id(), piece = lane % G;
    const int c = kLine && piece >= G / 2 ? D / 2 + (G - 1 - piece) * V : piece * V;
    const int c2 = kLine ? c : D / 2 + c;  // the second chunk's channels
    float cl[V], ch[V], sl[V], sh[V];
    bool rot = false;
    if constexpr (ROPE) {
        const int row = a.positions ? a.positions[token] : pos;
        rot = row >= 0 && row < a.table_rows;
        if (rot) {
            const float* cr = a.cos_tab + static_cast<int64_t>(row) * D;
            const float* sr = a.sin_tab + static_cast<int64_t>(row) * D;
            const float sign = kLine && piece < G / 2 ? -1.0f : 1.0f;
#pragma unroll
            for (int e = 0; e < V; e++) cl[e] = cr[c + e], sl[e] = sign * sr[c + e];
            if constexpr (!kLine) {
#pragma unroll
                for (int e = 0; e < V; e++) ch[e] = cr[c2 + e], sh[e] = sr[c2 + e];
            }
        }
    }
    const int part = unit - token * a.parts;
    const int heads = a.h + 2 * a.h_kv;
    const auto source = [&](int j) {
        return j < a.h            ? a.q + static_cast<int64_t>(token) * a.q_stride + j * D
               : j < a.h + a.h_kv ? a.k + static_cast<int64_t>(token) * a.k_stride + (j - a.h) * D
                                  : a.v + static_cast<int64_t>(token) * a.v_stride + (j - a.h - a.h_kv) * D;
    };
    // head j's chunk of channels ch0 to where it goes
    const auto put = [&](int j, int ch0, u32x4 x) {
        if (j < a.h) {
            st_stream(a.q_out + (static_cast<int64_t>(token) * a.h + j) * D + ch0, x);
            return;
        }
        const bool is_v = j >= a.h + a.h_kv;
        const int head = is_v ? j - a.h - a.h_kv : j - a.h;
        if (placed)
            st_stream((is_v ? a.v_cache : a.k_cache) + ((((static_cast<int64_t>(page) * a.h_kv + head) << a.page_shift) + slot) * D + ch0), x);
        if (!is_v && a.k_out) st_stream(a.k_out + (static_cast<int64_t>(token) * a.h_kv + head) * D + ch0, x);
    };
    const auto normalise = [&](float (&x)[V], const float* w, const float* b, int ch0, float mean, float inv) {
#pragma unroll
        for (int e = 0; e < V; e++) x[e] = fmaf((x[e] - mean) * inv, w[ch0 + e], b[ch0 + e]);
    };
    for (int j0 = part * HPW; j0 < heads; j0 += a.parts * HPW) {
        if constexpr (kLine) {
            const int j[2] = {j0 + lane / G, j0 + 64 / G + lane / G};
            u32x4 raw[2];
#pragma unroll
            for (int u = 0; u < 2; u++)
                if (j[u] < heads) raw[u] = ld_stream(source(j[u]) + c);
#pragma unroll
            for (int u = 0; u < 2; u++) {
                if (j[u] >= heads) continue;
                if ((NORM || rot) && j[u] < a.h + a.h_kv) {
                    float x[V];
                    unpack(raw[u], x, T{});
                    const float* w = j[u] < a.h ? a.qn_w : a.kn_w;
                    if (NORM && w) {
                        float sum = 0.0f, sq = 0.0f;
#pragma unroll
                        for (int e = 0; e < V; e++) sum += x[e];
                        const float mean = lanes_sum<G>(sum) * (1.0f / D);
#pragma unroll
                        for (int e = 0; e < V; e++) sq = fmaf(x[e] - mean, x[e] - mean, sq);
                        normalise(x, w, j[u] < a.h ? a.qn_b : a.kn_b, c, mean, rsqrtf(lanes_sum<G>(sq) * (1.0f / D) + a.eps));
                    }
                    if (rot) {
#pragma unroll
                        for (int e = 0; e < V; e++) x[e] = fmaf(x[e], cl[e], dpp<kRowHalfMirror>(x[e]) * sl[e]);
                    }
                    raw[u] = pack(x, T{});
                }
                put(j[u], c, raw[u]);
            }
        } else {
            const int j = j0 + lane / G;
            if (j >= heads) continue;
            const T* src = source(j);
            u32x4 lo = ld_stream(src + c), hi = ld_stream(src + c2);
            if ((NORM || rot) && j < a.h + a.h_kv) {
                float x[V], y[V];
                unpack(lo, x, T{});
                unpack(hi, y, T{});
                const float* w = j < a.h ? a.qn_w : a.kn_w;
                if (NORM && w) {
                    float sum = 0.0f, sq = 0.0f;
#pragma unroll
                    for (int e = 0; e < V; e++) sum += x[e] + y[e];
                    const float mean = lanes_sum<G>(sum) * (1.0f / D);
#pragma unroll
                    for (int e = 0; e < V; e++) sq = fmaf(x[e] - mean, x[e] - mean, fmaf(y[e] - mean, y[e] - mean, sq));
                    const float inv = rsqrtf(lanes_sum<G>(sq) * (1.0f / D) + a.eps);
                    const float* b = j < a.h ? a.qn_b : a.kn_b;
                    normalise(x, w, b, c, mean, inv);
                    normalise(y, w, b, c2, mean, inv);
                }
                if (rot) {
#pragma unroll
                    for (int e = 0; e < V; e++) {
                        const float u = x[e], v = y[e];
                        x[e] = fmaf(u, cl[e], -(v * sl[e]));
                        y[e] = fmaf(v, ch[e], u * sh[e]);
                    }
                }
                lo = pack(x, T{});
                hi = pack(y, T{});
            }
            put(j, c, lo);
            put(j, c2, hi);
        }
    }
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

typedef f16 h8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

__device__ __forceinline__ h8 as_h8(u32x4 v) { return __builtin_bit_cast(h8, v); }

constexpr int kGroup = 16;  // query heads per pass
constexpr int kRounds = 4;  // rounds of workgroups that a long call makes
constexpr int kMostPerCu = 4;  // workgroups of any of the kernels
constexpr int kPagedWaves = 4;
constexpr float kNone = -3.0e38f;   // a running maximum that has seen no key
constexpr float kFloor = -2.9e38f;  // the least of one that has
// f16: a weight goes to the product with V as two f16 values, its 11 leading bits
// and the next 11, which makes the product as good as one of f32 weights (errors
// against 64 bits 2.5e-4 with the leading bits alone, 2.0e-4 so, which is the
// result's rounding) for 1-2% of the time. The largest weight of a step is this
// unit, so that the others, f16 being subnormal below 2^-14, are 2^-40 of it off at
// most (of a unit of 1, 45% at a score 17 nats below). The second part times an
// infinity is NaN or the other infinity: a step that has one among its values
// leaves the second parts out.
constexpr float kHalfUnit = 32768.0f;

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

struct PagedArgs {
    const void *q, *k, *v;
    void* out;
    float *ws_o, *ws_ml;  // per (piece, query head): D sums; maximum and weight sum
    int* ws_cut;          // per sequence: its first piece, its pieces
    const int *page_table, *lens;
    int64_t q_stride;
    int b, h, h_kv, page_shift, n_pages, max_pages;
    float per_round;  // 1 / ranges that the chip holds at once
    int group, passes, width;  // query heads per key head, passes over them, heads per pass
    float scale;
};

// Units of keys per piece. The total is summed in f32, whose error (2^-24 a
// step) per_round covers, so that there are never more pieces than the launch
// has workgroups for.
__device__ __forceinline__ int units_per_piece(const PagedArgs& a, int unit) {
    float total = 0.0f;
    for (int base = 0; base < a.b; base += 64) {
        const int s = base + lane_id();
        total += s < a.b ? static_cast<float>((held_length(a.lens, s, a.max_pages, a.page_shift) + unit - 1) / unit) : 0.0f;
    }
    const float per = wave_sum(total) * a.per_round;
    return static_cast<int>(fminf(fmaxf(fmaxf(ceilf(per * (1.0f / kRounds)), fminf(ceilf(per), 4.0f)), 1.0f), 16777216.0f));
}
__device__ __forceinline__ int pieces_of(const PagedArgs& a, int s, int unit, int chunk) {
    const uint32_t units = static_cast<uint32_t>((held_length(a.lens, s, a.max_pages, a.page_shift) + unit - 1) / unit);
    return units <= static_cast<uint32_t>(chunk) ? 1 : static_cast<int>((units + chunk - 1) / static_cast<uint32_t>(chunk));
}

// A workgroup's piece: keys [begin, end) of sequence s, the local-th of its
// count pieces, key head kv, pass `pass` over its query heads.
struct Piece {
    int s, begin, end, count, kv, pass;
};
__device__ __forceinline__ bool find_piece(const PagedArgs& a, int unit, Piece& t) {
    const int lane = lane_id();
    const int heads = a.h_kv * a.passes;
    const int piece = static_cast<int>(blockIdx.x) / heads;
    const int rest = static_cast<int>(blockIdx.x) - piece * heads;
    t.kv = rest / a.passes, t.pass = rest - t.kv * a.passes;
    const int chunk = units_per_piece(a, unit);
    int local = 0, before = 0;
    t.s = -1;
    for (int base = 0; base < a.b; base += 64) {
        const int c = base + lane < a.b ? pieces_of(a, base + lane, unit, chunk) : 0;
        const int sum = wave_prefix_sum(c);
        const uint64_t hit = __ballot(before + sum > piece);
        if (hit) {
            const int l = __builtin_ctzll(hit);
            t.s = base + l;
            t.count = lane_value(c, l);
            local = piece - before - (lane_value(sum, l) - t.count);
            break;
        }
        before += lane_value(sum, 63);
    }
    if (t.s < 0) return false;
    const int len = held_length(a.lens, t.s, a.max_pages, a.page_shift);
    const int64_t first = static_cast<int64_t>(local) * chunk * unit, last = first + static_cast<int64_t>(chunk) * unit;
    t.begin = static_cast<int>(first < len ? first : len), t.end = static_cast<int>(last < len ? last : len);
    if (local == 0 && rest == 0 && threadIdx.x == 0) a.ws_cut[2 * t.s] = piece, a.ws_cut[2 * t.s + 1] = t.count;
    return true;
}

// Where key `key`'s row lies in the pool (in rows), page 0's where its page is
// none of the pool's.
struct Tile16 {
    int64_t row;
    bool there;
};
__device__ __forceinline__ Tile16 tile_of(const PagedArgs& a, int page, int kv, int key) {
    const bool there = page >= 0 && page < a.n_pages;
    return {((static_cast<int64_t>(there ? page : 0) * a.h_kv + kv) << a.page_shift) + (key & ((1 << a.page_shift) - 1)), there};
}

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

    // join the waves
    __syncthreads();
    if (n < live_heads) {
#pragma unroll
        for (int i = 0; i < DB; i++) *reinterpret_cast<f32x4*>(&sm.o[wave][n * P::kOPitch + 16 * i + 4 * g]) = o[i];
        if (g == 0) sm.m[wave][n] = m, sm.l[wave][n] = l;
    }
    __syncthreads();
    for (int x = threadIdx.x; x < live_heads * (D / 4); x += 64 * kPagedWaves) {
        const int head = x / (D / 4), d0 = x % (D / 4) * 4;
        float top = sm.m[0][head];
#pragma unroll
        for (int w = 1; w < kPagedWaves; w++) top = fmaxf(top, sm.m[w][head]);
        f32x4 sum = {};
        float weight = 0.0f;
#pragma unroll
        for (int w = 0; w < kPagedWaves; w++) {
            const float f = __builtin_amdgcn_exp2f(sm.m[w][head] - top);
            sum += *reinterpret_cast<const f32x4*>(&sm.o[w][head * P::kOPitch + d0]) * f;
            weight = fmaf(sm.l[w][head], f, weight);
        }
        if (count == 1) {
            T* orow = static_cast<T*>(a.out) + (static_cast<int64_t>(s) * a.h + head0 + head) * D + d0;
#pragma unroll
            for (int e = 0; e < 4; e++) orow[e] = static_cast<T>(top == kNone ? 0.0f : sum[e] / weight);
        } else {
            const int64_t row = static_cast<int64_t>(blockIdx.x) * a.width + head;
            *reinterpret_cast<f32x4*>(a.ws_o + row * D + d0) = sum;
            if (d0 == 0) a.ws_ml[2 * row] = top, a.ws_ml[2 * row + 1] = weight;
        }
    }
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

// The pieces of one (sequence, query head) joined, THREADS / (D / 4) at a time.
template <typename T, int D, int THREADS>
__global__ __launch_bounds__(THREADS) void paged_join_kernel(PagedArgs a) {
    constexpr int kLanes = D / 4, kRows = THREADS / kLanes;
    __shared__ __align__(16) f32x4 part[kRows][kLanes];
    __shared__ float tops[kRows], weights[kRows];
    const int s = static_cast<int>(blockIdx.x) / a.h, head = static_cast<int>(blockIdx.x) - s * a.h;
    const int64_t before = a.ws_cut[2 * s];
    const int count = a.ws_cut[2 * s + 1];
    if (count == 1) return;  // workgroup-uniform: written by its only piece
    const int kv = head / a.group, in_group = head - kv * a.group;
    const int pass = in_group / a.width, x = in_group - pass * a.width;
    const auto row_of = [&](int i) { return (((before + i) * a.h_kv + kv) * a.passes + pass) * a.width + x; };
    const int row = threadIdx.x / kLanes, col = threadIdx.x % kLanes;
    float top = kNone, weight = 0.0f;
    f32x4 sum = {};
    for (int i = row; i < count; i += kRows) {
        const int64_t r = row_of(i);
        const float m = a.ws_ml[2 * r], l = a.ws_ml[2 * r + 1];
        const f32x4 v = *reinterpret_cast<const f32x4*>(a.ws_o + r * D + 4 * col);
        const float next = fmaxf(top, m);
        const float old = __builtin_amdgcn_exp2f(top - next), f = __builtin_amdgcn_exp2f(m - next);
        sum = sum * old + v * f;
        weight = fmaf(weight, old, l * f);
        top = next;
    }
    part[row][col] = sum;
    if (col == 0) tops[row] = top, weights[row] = weight;
    __syncthreads();
    if (row != 0) return;
    const int rows = min(kRows, count);
    for (int i = 0; i < rows; i++) top = fmaxf(top, tops[i]);
    sum = f32x4{}, weight = 0.0f;
    for (int i = 0; i < rows; i++) {
        const float f = __builtin_amdgcn_exp2f(tops[i] - top);
        sum += part[i][col] * f;
        weight = fmaf(weights[i], f, weight);
    }
    T* orow = static_cast<T*>(a.out) + (static_cast<int64_t>(s) * a.h + head) * D + 4 * col;
#pragma unroll
    for (int e = 0; e < 4; e++) orow[e] = static_cast<T>(top == kNone ? 0.0f : sum[e] / weight);
}

// How the query heads of a key head are taken, and how many pieces there are
// at most.
struct PagedPlan {
    int group, passes, width;
    int64_t heads, ranges, items, rows;
    PagedPlan(int b, int h, int h_kv, int per_cu) {
        group = h / h_kv;
        passes = static_cast<int>(ceil_div(group, kGroup));
        width = static_cast<int>(ceil_div(group, passes));
        heads = static_cast<int64_t>(h_kv) * passes;
        ranges = ceil_div(per_cu * num_cus(), heads);
        items = (ranges * kRounds + b) * heads;  // each sequence's last piece may be short
        rows = items * width;
    }
};

template <typename T, int D, typename K>
hs_status launch_pieces(const char* op, hipStream_t st, PagedArgs a, K whole, K rows, int unit, int per_cu) {
    const PagedPlan plan(a.b, a.h, a.h_kv, per_cu);
    a.ws_ml = a.ws_o + plan.rows * D;
    a.ws_cut = reinterpret_cast<int*>(a.ws_ml + 2 * plan.rows);
    a.group = plan.group, a.passes = plan.passes, a.width = plan.width;
    // (rounded up by twice the error of the kernels' sum over the lengths)
    a.per_round = static_cast<float>((1.0 + (a.b / 64 + 64) * 0x1p-23) / static_cast<double>(plan.ranges));
    // no more pieces than a table's width of keys has, either
    const int64_t most = ceil_div(static_cast<int64_t>(a.max_pages) << a.page_shift, int64_t{unit});
    const int64_t items = a.b * plan.heads * (most > 1 ? most : 1);
    const dim3 grid(static_cast<uint32_t>(items < plan.items ? items : plan.items));
    (a.page_shift >= 4 ? whole : rows)<<<grid, dim3(64 * kPagedWaves), 0, st>>>(a);
    if (hs_status rc = check_launch(op)) return rc;
    if (most <= 1) return HS_OK;  // no sequence has two pieces
    const int64_t joined = static_cast<int64_t>(a.b) * a.h;
    const dim3 joins(static_cast<uint32_t>(joined));
    // few rows may have a thousand pieces each
    if (joined <= 64)
        paged_join_kernel<T, D, 1024><<<joins, dim3(1024), 0, st>>>(a);
    else
        paged_join_kernel<T, D, 256><<<joins, dim3(256), 0, st>>>(a);
    return check_launch(op);
}

template <typename T, int D>
hs_status launch_paged(const char* op, hipStream_t st, const PagedArgs& a) {
    if constexpr (sizeof(T) == 4) {
        if (a.h == a.h_kv) {
            using P = PagedSingle<D>;
            return launch_pieces<T, D>(op, st, a, paged_single_kernel<D, true>, paged_single_kernel<D, false>, P::kUnit, P::kPerCu);
        }
    }
    using P = Paged<T, D>;
    return launch_pieces<T, D>(op, st, a, attention_paged_kernel<T, D, true>, attention_paged_kernel<T, D, false>, P::kUnit, P::kPerCu);
}

hs_status check_cache(const char* op, const void* k_cache, const void* v_cache, const void* page_table,
                      const void* lens, int32_t page, int32_t n_pages, int32_t max_pages, int32_t h_kv, int32_t d) {
    if (page <= 0 || n_pages < 0 || max_pages < 0) return fail(HS_EINVAL, "%s: page %d, n_pages %d, max_pages %d", op, page, n_pages, max_pages);
    if (exact_log2(page) < 0) return fail(HS_EUNSUPPORTED, "%s: page %d is no power of two", op, page);
    if (static_cast<int64_t>(max_pages) * page >= (int64_t{1} << 30)) return fail(HS_EINVAL, "%s: max_pages * page must be below 2^30", op);
    if (too_large(static_cast<int64_t>(n_pages) * page, static_cast<int64_t>(h_kv) * d))
        return fail(HS_EINVAL, "%s: cache too large", op);
    if (!lens || (max_pages > 0 && !page_table) || (n_pages > 0 && (!k_cache || !v_cache)))
        return fail(HS_EINVAL, "%s: null cache, page_table or lens", op);
    if (!aligned16(k_cache) || !aligned16(v_cache)) return fail(HS_EUNSUPPORTED, "%s: caches must be 16-byte aligned", op);
    return HS_OK;
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
    if (hs_status rc = check_heads(op, dt, q ? h : 0, h_kv, d)) return rc;
    if (n < 0 || b < 0 || table_rows < 0) return fail(HS_EINVAL, "%s: negative count", op);
    if (!offsets && n != b) return fail(HS_EINVAL, "%s: without offsets, one token per sequence (n %lld, b %d)", op, static_cast<long long>(n), b);
    if ((!qn_w) != (!qn_b) || (!kn_w) != (!kn_b)) return fail(HS_EINVAL, "%s: norm weight and bias go together", op);
    if ((!sin_tab) != (!cos_tab)) return fail(HS_EINVAL, "%s: sin and cos tables go together", op);
    if (positions && !sin_tab) return fail(HS_EINVAL, "%s: positions without tables", op);
    if ((qn_w || kn_w) && !(eps > 0.0f)) return fail(HS_EINVAL, "%s: eps must be positive", op);
    if (!q) h = 0;
    const int64_t heads = static_cast<int64_t>(h) + 2 * h_kv;
    if (n >= (int64_t{1} << 30) / heads) return fail(HS_EINVAL, "%s: n * (Hq + 2 Hkv) must be below 2^30", op);
    if (too_large(table_rows, d)) return fail(HS_EINVAL, "%s: tables too large", op);
    if (n == 0 || b == 0) return HS_OK;
    if (hs_status rc = check_rows(op, "q", q, h ? n : 0, q_stride, static_cast<int64_t>(h) * d, dt)) return rc;
    if (hs_status rc = check_rows(op, "k", k, n, k_stride, static_cast<int64_t>(h_kv) * d, dt)) return rc;
    if (hs_status rc = check_rows(op, "v", v, n, v_stride, static_cast<int64_t>(h_kv) * d, dt)) return rc;
    if (h && !q_out) return fail(HS_EINVAL, "%s: null q_out", op);
    if (hs_status rc = check_cache(op, k_cache, v_cache, page_table, lens, page, n_pages, max_pages, h_kv, d)) return rc;
    if (!aligned16(q_out) || !aligned16(k_out)) return fail(HS_EUNSUPPORTED, "%s: outputs must be 16-byte aligned", op);
    const int64_t e = dtype_size(dt), cache = static_cast<int64_t>(n_pages) * page * h_kv * d * e;
    struct Range {
        const void* p;
        int64_t bytes;
    };
    const Range outs[4] = {{h ? q_out : nullptr, n * h * d * e}, {k_out, k_out ? n * h_kv * d * e : 0}, {k_cache, cache}, {v_cache, cache}};
    const Range ins[3] = {{q, h ? row_bytes(n, q_stride, static_cast<int64_t>(h) * d, dt) : 0},
                          {k, row_bytes(n, k_stride, static_cast<int64_t>(h_kv) * d, dt)},
                          {v, row_bytes(n, v_stride, static_cast<int64_t>(h_kv) * d, dt)}};
    for (int i = 0; i < 4; i++) {
        for (const Range& r : ins)
            if (overlaps(outs[i].p, outs[i].bytes, r.p, r.bytes)) return fail(HS_EINVAL, "%s: an output overlaps an input", op);
        for (int j = 0; j < i; j++)
            if (overlaps(outs[i].p, outs[i].bytes, outs[j].p, outs[j].bytes)) return fail(HS_EINVAL, "%s: outputs overlap", op);
    }
    // waves per token: as many heads each as two loads hold
    const int parts = static_cast<int>(ceil_div(heads, dt == HS_F16 ? 1024 / d : 512 / d));
    if (n * parts >= (int64_t{1} << 26)) return fail(HS_EINVAL, "%s: too many tokens", op);
    const auto run = [&](auto zero) {
        using T = decltype(zero);
        AppendArgs<T> a;
        a.q = static_cast<const T*>(q), a.k = static_cast<const T*>(k), a.v = static_cast<const T*>(v);
        a.q_stride = q_stride, a.k_stride = k_stride, a.v_stride = v_stride;
        a.qn_w = qn_w, a.qn_b = qn_b, a.kn_w = kn_w, a.kn_b = kn_b, a.sin_tab = sin_tab, a.cos_tab = cos_tab;
        a.positions = static_cast<const int*>(positions), a.offsets = static_cast<const int*>(offsets);
        a.page_table = static_cast<const int*>(page_table), a.lens = static_cast<const int*>(lens);
        a.q_out = static_cast<T*>(q_out), a.k_out = static_cast<T*>(k_out);
        a.k_cache = static_cast<T*>(k_cache), a.v_cache = static_cast<T*>(v_cache);
        a.n = static_cast<int>(n), a.b = b, a.h = h, a.h_kv = h_kv, a.table_rows = table_rows;
        a.page_shift = exact_log2(page), a.n_pages = n_pages, a.max_pages = max_pages, a.eps = eps;
        a.parts = parts;
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
