// What the caches of full and of 8 bits share: a token's rows on their way to the
// cache, the cut of a call's keys into pieces and their join, and the host's
// checks. (Everything is a translation unit's own: kernels are instantiated where
// they are launched.)
#pragma once

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

// V floats by 16-byte loads.
template <int V>
__device__ __forceinline__ void ld_values(const float* p, float (&f)[V]) {
#pragma unroll
    for (int i = 0; i < V / 4; i++) {
        const float4 x = ld_f32x4(p + 4 * i);
        f[4 * i] = x.x, f[4 * i + 1] = x.y, f[4 * i + 2] = x.z, f[4 * i + 3] = x.w;
    }
}

template <typename T>
struct AppendArgs {
    const T *q, *k, *v;
    int64_t q_stride, k_stride, v_stride;
    const float *qn_w, *qn_b, *kn_w, *kn_b, *sin_tab, *cos_tab;
    const int *positions, *offsets, *page_table, *lens;
    T *q_out, *k_out, *k_cache, *v_cache;
    int n, b, h, h_kv, table_rows, page_shift, n_pages, max_pages, parts;
    int heads;  // taken of the row's: all, or the first ones (a cache of 8 bits takes its own)
    float eps;
};

template <typename T, int D, bool NORM, bool ROPE>
__device__ __forceinline__ void append_rows(const AppendArgs<T>& a, int unit) {
    constexpr bool kLine = sizeof(T) == 2 && D == 64;  // one chunk per lane and head
    constexpr int V = Vec<T>::N, G = kLine ? D / V : D / (2 * V), HPW = 64 / G * (kLine ? 2 : 1);
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
            ld_values(cr + c, cl), ld_values(sr + c, sl);
#pragma unroll
            for (int e = 0; e < V; e++) sl[e] *= sign;
            if constexpr (!kLine) ld_values(cr + c2, ch), ld_values(sr + c2, sh);
        }
    }
    const int part = unit - token * a.parts;
    const int heads = a.heads;
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

// ---------------------------------------------------------------------------
// attention of single tokens

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
// infinity is NaN or the other infinity: over full caches a step that has one among
// its values leaves the second parts out; over 8 bits see odd_values.
constexpr float kHalfUnit = 32768.0f;

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
template <typename A>
__device__ __forceinline__ Tile16 tile_of(const A& a, int page, int kv, int key) {
    const bool there = page >= 0 && page < a.n_pages;
    return {((static_cast<int64_t>(there ? page : 0) * a.h_kv + kv) << a.page_shift) + (key & ((1 << a.page_shift) - 1)), there};
}

// Sums times a factor; `keep`: an infinite one stays where the factor is 0.
template <typename K>
__device__ __forceinline__ f32x4 times(f32x4 x, float f, K keep) {
    f32x4 y = x * f;
    if constexpr (decltype(keep)::value) {
#pragma unroll
        for (int e = 0; e < 4; e++) y[e] = y[e] != y[e] ? x[e] : y[e];
    }
    return y;
}
// Sums that f(keep) joins. KEEP: where one is NaN, it is done again with what is
// infinite kept (kept at once, one token over 130531 keys takes 55 us for 53).
template <bool KEEP = true, typename F>
__device__ __forceinline__ f32x4 joined(F f) {
    f32x4 x = f(std::false_type{});
    if constexpr (KEEP) {
        if (x[0] != x[0] || x[1] != x[1] || x[2] != x[2] || x[3] != x[3]) {
            const f32x4 y = f(std::true_type{});
#pragma unroll
            for (int e = 0; e < 4; e++) x[e] = x[e] != x[e] ? y[e] : x[e];
        }
    }
    return x;
}

// A workgroup's waves' sums of up to kGroup query heads joined in LDS: the result,
// or the piece's in the workspace. Lane (n, g) holds channels 16 i + 4 g + .. of
// head n; l is a head's whole sum of the wave. KEEP: as there. `mend`: what the wave
// does to its sums in LDS.
template <typename T, int D, bool KEEP, typename S, typename F>
__device__ __forceinline__ void join_waves(const PagedArgs& a, S& sm, int s, int count, int head0, int live_heads,
                                           const f32x4 (&o)[D / 16], float m, float l, F mend) {
    constexpr int kOPitch = D + 4;
    const int lane = lane_id(), wave = wave_in_block(), n = lane & 15, g = lane >> 4;
    __syncthreads();
    if (n < live_heads) {
#pragma unroll
        for (int i = 0; i < D / 16; i++) *reinterpret_cast<f32x4*>(&sm.o[wave][n * kOPitch + 16 * i + 4 * g]) = o[i];
        if (g == 0) sm.m[wave][n] = m, sm.l[wave][n] = l;
    }
    mend(sm.o[wave]);
    __syncthreads();
    for (int x = threadIdx.x; x < live_heads * (D / 4); x += 64 * kPagedWaves) {
        const int head = x / (D / 4), d0 = x % (D / 4) * 4;
        float top = sm.m[0][head];
#pragma unroll
        for (int w = 1; w < kPagedWaves; w++) top = fmaxf(top, sm.m[w][head]);
        float weight = 0.0f;
        const f32x4 sum = joined<KEEP>([&](auto keep) {
            f32x4 all = {};
            weight = 0.0f;
#pragma unroll
            for (int w = 0; w < kPagedWaves; w++) {
                const float f = __builtin_amdgcn_exp2f(sm.m[w][head] - top);
                all += times(*reinterpret_cast<const f32x4*>(&sm.o[w][head * kOPitch + d0]), f, keep);
                weight = fmaf(sm.l[w][head], f, weight);
            }
            return all;
        });
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

// The pieces of one (sequence, query head) joined, THREADS / (D / 4) at a time.
template <typename T, int D, int THREADS, bool KEEP>
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
    float top, weight;
    part[row][col] = joined<KEEP>([&](auto keep) {
        f32x4 sum = {};
        top = kNone, weight = 0.0f;
        for (int i = row; i < count; i += kRows) {
            const int64_t r = row_of(i);
            const float m = a.ws_ml[2 * r], l = a.ws_ml[2 * r + 1];
            const f32x4 v = *reinterpret_cast<const f32x4*>(a.ws_o + r * D + 4 * col);
            const float next = fmaxf(top, m);
            const float old = __builtin_amdgcn_exp2f(top - next), f = __builtin_amdgcn_exp2f(m - next);
            sum = times(sum, old, keep) + times(v, f, keep);
            weight = fmaf(weight, old, l * f);
            top = next;
        }
        return sum;
    });
    if (col == 0) tops[row] = top, weights[row] = weight;
    __syncthreads();
    if (row != 0) return;
    const int rows = min(kRows, count);
    for (int i = 0; i < rows; i++) top = fmaxf(top, tops[i]);
    const f32x4 sum = joined<KEEP>([&](auto keep) {
        f32x4 all = {};
        weight = 0.0f;
        for (int i = 0; i < rows; i++) {
            const float f = __builtin_amdgcn_exp2f(tops[i] - top);
            all += times(part[i][col], f, keep);
            weight = fmaf(weights[i], f, weight);
        }
        return all;
    });
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

// The pieces' kernel (of whole 16 keys in a page, or by rows) and their join.
template <typename T, int D, bool KEEP, typename A, typename K>
hs_status launch_pieces(const char* op, hipStream_t st, A a, K whole, K rows, int unit, int per_cu) {
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
        paged_join_kernel<T, D, 1024, KEEP><<<joins, dim3(1024), 0, st>>>(a);
    else
        paged_join_kernel<T, D, 256, KEEP><<<joins, dim3(256), 0, st>>>(a);
    return check_launch(op);
}

[[maybe_unused]] hs_status check_cache(const char* op, const void* k_cache, const void* v_cache, const void* page_table,
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

struct ByteRange {
    const void* p;
    int64_t bytes;
};

// A call that appends, and what its checks leave of it (h is 0 without q).
struct AppendCall {
    const void *q, *k, *v;
    int64_t q_stride, k_stride, v_stride;
    const float *qn_w, *qn_b, *kn_w, *kn_b, *sin_tab, *cos_tab;
    int32_t table_rows;
    const void *positions, *offsets, *page_table, *lens;
    void *q_out, *k_out;
    int64_t n;
    int32_t b, h, h_kv, d, page, n_pages, max_pages;
    float eps;

    int64_t q_width() const { return static_cast<int64_t>(h) * d; }
    int64_t kv_width() const { return static_cast<int64_t>(h_kv) * d; }
    ByteRange q_rows(hs_dtype dt) const { return {h ? q_out : nullptr, n * q_width() * dtype_size(dt)}; }
    ByteRange k_rows(hs_dtype dt) const { return {k_out, k_out ? n * kv_width() * dtype_size(dt) : 0}; }
    template <typename T>
    void fill(AppendArgs<T>& a) const {
        a.q = static_cast<const T*>(q), a.k = static_cast<const T*>(k), a.v = static_cast<const T*>(v);
        a.q_stride = q_stride, a.k_stride = k_stride, a.v_stride = v_stride;
        a.qn_w = qn_w, a.qn_b = qn_b, a.kn_w = kn_w, a.kn_b = kn_b, a.sin_tab = sin_tab, a.cos_tab = cos_tab;
        a.positions = static_cast<const int*>(positions), a.offsets = static_cast<const int*>(offsets);
        a.page_table = static_cast<const int*>(page_table), a.lens = static_cast<const int*>(lens);
        a.q_out = static_cast<T*>(q_out), a.k_out = static_cast<T*>(k_out);
        a.n = static_cast<int>(n), a.b = b, a.h = h, a.h_kv = h_kv, a.table_rows = table_rows;
        a.page_shift = exact_log2(page), a.n_pages = n_pages, a.max_pages = max_pages, a.eps = eps;
    }
};

// Everything but the cache; done: nothing to append.
[[maybe_unused]] hs_status check_append(const char* op, hs_dtype dt, AppendCall& c, bool& done) {
    if (hs_status rc = check_heads(op, dt, c.q ? c.h : 0, c.h_kv, c.d)) return rc;
    if (c.n < 0 || c.b < 0 || c.table_rows < 0) return fail(HS_EINVAL, "%s: negative count", op);
    if (!c.offsets && c.n != c.b)
        return fail(HS_EINVAL, "%s: without offsets, one token per sequence (n %lld, b %d)", op, static_cast<long long>(c.n), c.b);
    if ((!c.qn_w) != (!c.qn_b) || (!c.kn_w) != (!c.kn_b)) return fail(HS_EINVAL, "%s: norm weight and bias go together", op);
    if ((!c.sin_tab) != (!c.cos_tab)) return fail(HS_EINVAL, "%s: sin and cos tables go together", op);
    if (c.positions && !c.sin_tab) return fail(HS_EINVAL, "%s: positions without tables", op);
    if ((c.qn_w || c.kn_w) && !(c.eps > 0.0f)) return fail(HS_EINVAL, "%s: eps must be positive", op);
    if (!c.q) c.h = 0;
    const int64_t heads = static_cast<int64_t>(c.h) + 2 * c.h_kv;
    if (c.n >= (int64_t{1} << 30) / heads) return fail(HS_EINVAL, "%s: n * (Hq + 2 Hkv) must be below 2^30", op);
    if (too_large(c.table_rows, c.d)) return fail(HS_EINVAL, "%s: tables too large", op);
    if ((done = c.n == 0 || c.b == 0)) return HS_OK;
    if (hs_status rc = check_rows(op, "q", c.q, c.h ? c.n : 0, c.q_stride, c.q_width(), dt)) return rc;
    if (hs_status rc = check_rows(op, "k", c.k, c.n, c.k_stride, c.kv_width(), dt)) return rc;
    if (hs_status rc = check_rows(op, "v", c.v, c.n, c.v_stride, c.kv_width(), dt)) return rc;
    if (c.h && !c.q_out) return fail(HS_EINVAL, "%s: null q_out", op);
    return HS_OK;
}

[[maybe_unused]] hs_status check_append_overlaps(const char* op, hs_dtype dt, const AppendCall& c, const ByteRange* outs, int count) {
    if (!aligned16(c.q_out) || !aligned16(c.k_out)) return fail(HS_EUNSUPPORTED, "%s: outputs must be 16-byte aligned", op);
    const ByteRange ins[3] = {{c.q, c.h ? row_bytes(c.n, c.q_stride, c.q_width(), dt) : 0},
                              {c.k, row_bytes(c.n, c.k_stride, c.kv_width(), dt)},
                              {c.v, row_bytes(c.n, c.v_stride, c.kv_width(), dt)}};
    for (int i = 0; i < count; i++) {
        for (const ByteRange& r : ins)
            if (overlaps(outs[i].p, outs[i].bytes, r.p, r.bytes)) return fail(HS_EINVAL, "%s: an output overlaps an input", op);
        for (int j = 0; j < i; j++)
            if (overlaps(outs[i].p, outs[i].bytes, outs[j].p, outs[j].bytes)) return fail(HS_EINVAL, "%s: outputs overlap", op);
    }
    return HS_OK;
}

}  // namespace
}  // namespace hs
