// A paged key-value cache held in 8 bits for gfx950: appending new tokens and the
// attention of one new token per sequence.
#include <algorithm>
#include <type_traits>

#include "hs_steps_f8.hpp"

namespace hs {
namespace {

// ---------------------------------------------------------------------------
// kv_append
//
// A page's new keys of one head take a scale together, so a unit of work is one
// page of a sequence, and its rows are read, normalised and rotated into registers,
// their largest magnitude gives the scale, and the codes follow. A page that the
// call goes on with keeps the larger scale of the two; where that is the new one, the
// older codes are brought to it, which is exact but for those that become subnormal.
//
// A page's rows are held by one wave where it has at most 2048 / D, else by two or
// four; pages of more than four times that are read twice. A wave goes through several
// heads' keys, or values, with the next head's rows under way, so that the place and
// the rotation of its rows are looked up once.
//
// Prompts make two launches, of the queries' rows as kv_append's and of the pages,
// which want different registers (102 us in one for 75); a step is one. Bandwidth:
// 16381 tokens, 32 heads of 128 over 8, rotated, f16, 75 us, 5.0 TB/s, of which the
// pages are 28 (21 without the rotation); 10992 tokens, 16 heads of 64, QK-norm, 36
// us, 3.2 TB/s: pages of 64 by two waves (40 us by four, half of them idle). 8 and 32
// waves a CU for 16: 78 and 76 us.
template <typename T>
struct Append8Args {
    AppendArgs<T> rows;  // q, and k where its rows are asked for
    const int *offsets, *page_table, *lens;
    uint8_t *k_cache, *v_cache, *k_scale, *v_scale;
    int n_pages, row_blocks;
    int split;  // waves (W of them: workgroups) that share a page's heads
};

__device__ __forceinline__ float wave_max(float v) {
    v = fmaxf(v, dpp<kQuadXor1>(v));
    v = fmaxf(v, dpp<kQuadXor2>(v));
    v = fmaxf(v, dpp<kRowHalfMirror>(v));
    v = fmaxf(v, dpp<kRowMirror>(v));
    v = fmaxf(v, __shfl_xor(v, 16, 64));
    return fmaxf(v, __shfl_xor(v, 32, 64));
}

// A unit's place: tokens [token, token + rows) of the call become rows [first,
// first + rows) of page `page`.
struct PageUnit {
    int token, rows, first, page, pos;
};
template <typename T>
__device__ __forceinline__ bool find_unit(const Append8Args<T>& a, int index, PageUnit& t) {
    const AppendArgs<T>& r = a.rows;
    const int shift = r.page_shift, limit = r.max_pages << shift;
    int s, entry, begin, end, m_end;  // keys [begin, end) of the sequence; its tokens end at row m_end
    if (!a.offsets) {
        s = index;
        if (s >= r.b) return false;
        const int len = a.lens[s];
        begin = len - 1, end = len, m_end = s + 1;
        if (begin < 0 || begin >= limit) return false;
        entry = begin >> shift;
    } else {
        const int lane = lane_id();
        int before = 0;
        s = -1;
        for (int base = 0; base < r.b; base += 64) {
            int count = 0, b0 = 0, e0 = 0, z0 = 0;
            if (base + lane < r.b) {
                const RowRange q = row_range(a.offsets, base + lane, r.n);
                // Token of key p: p + z0. The sequence's last one is key len - 1, also where
                // its rows end past the ones given, which are then the first of them.
                if (q.end > q.begin) {
                    z0 = a.offsets[base + lane + 1] - max(a.lens[base + lane], 0);
                    b0 = max(q.begin - z0, 0), e0 = min(q.end - z0, limit);
                    if (e0 > b0) count = ((e0 - 1) >> shift) - (b0 >> shift) + 1;
                }
            }
            const int sum = wave_prefix_sum(count);
            const uint64_t hit = __ballot(before + sum > index);
            if (hit) {
                const int l = __builtin_ctzll(hit);
                s = base + l;
                begin = lane_value(b0, l), end = lane_value(e0, l), m_end = lane_value(z0, l);
                entry = (begin >> shift) + index - before - (lane_value(sum, l) - lane_value(count, l));
                break;
            }
            before += lane_value(sum, 63);
        }
        if (s < 0) return false;
        m_end += end;  // as if the sequence ended at `end`
    }
    t.page = a.page_table[static_cast<int64_t>(s) * r.max_pages + entry];
    if (t.page < 0 || t.page >= a.n_pages) return false;
    const int lo = max(begin, entry << shift), hi = min(end, (entry + 1) << shift);
    t.pos = lo, t.first = lo & ((1 << shift) - 1), t.rows = hi - lo;
    t.token = m_end - (end - lo);
    return true;
}

template <typename T, int D, bool NORM, bool ROPE, int W>
__device__ __forceinline__ void append_page(const Append8Args<T>& a, int index) {
    const AppendArgs<T>& r = a.rows;
    constexpr int V = Vec<T>::N, G = D / (2 * V), kRows = 64 / G;  // rows per load
    constexpr int kHeld = 2048 / D, P = kHeld / kRows;             // rows and loads that a wave holds
    __shared__ float tops[2][W];
    const int lane = lane_id(), wave = W == 1 ? 0 : wave_in_block();
    const int unit = index / (2 * a.split), which = index - unit * 2 * a.split;
    const bool is_v = which >= a.split;
    PageUnit t;
    if (!find_unit(a, unit, t)) return;  // the same for all waves of a unit
    const int64_t stride = is_v ? r.v_stride : r.k_stride;
    const T* rows = (is_v ? r.v : r.k) + t.token * stride;
    const int64_t block0 = static_cast<int64_t>(t.page) * r.h_kv;
    uint8_t* scales = (is_v ? a.v_scale : a.k_scale) + block0;
    const int piece = lane % G, c = piece * V, c2 = D / 2 + c;
    const bool norm = NORM && !is_v && r.kn_w, rope = ROPE && !is_v;
    const int rounds = W == 1 ? 1 : (t.rows + kHeld * W - 1) / (kHeld * W);
    const auto row_of = [&](int round, int i) { return (round * W + wave) * kHeld + i * kRows + lane / G; };

    // a row's place in the tables, or none; kept for the rows of the only round
    float cl[P][V], ch[P][V], sl[P][V], sh[P][V];
    bool turns[P];
    const auto find_turn = [&](int row, int i) {
        turns[i] = false;
        if (!rope || row >= t.rows) return;
        const int at = r.positions ? r.positions[t.token + row] : t.pos + row;
        turns[i] = at >= 0 && at < r.table_rows;
        if (!turns[i]) return;
        const float* cr = r.cos_tab + static_cast<int64_t>(at) * D;
        const float* sr = r.sin_tab + static_cast<int64_t>(at) * D;
        ld_values(cr + c, cl[i]), ld_values(cr + c2, ch[i]), ld_values(sr + c, sl[i]), ld_values(sr + c2, sh[i]);
    };
    u32x4 lo[P], hi[P];
    const auto load = [&](int round, int head) {
#pragma unroll
        for (int i = 0; i < P; i++) {
            const int row = row_of(round, i);
            lo[i] = hi[i] = u32x4{};
            if (row >= t.rows) continue;
            const T* p = rows + row * stride + head * D;
            lo[i] = ld_stream(p + c), hi[i] = ld_stream(p + c2);
        }
    };
    // load i's two chunks as the cache is to take them
    const auto turned = [&](int i, float (&x)[V], float (&y)[V]) {
        unpack(lo[i], x, T{});
        unpack(hi[i], y, T{});
        if (norm) {
            float sum = 0.0f, sq = 0.0f;
#pragma unroll
            for (int e = 0; e < V; e++) sum += x[e] + y[e];
            const float mean = lanes_sum<G>(sum) * (1.0f / D);
#pragma unroll
            for (int e = 0; e < V; e++) sq = fmaf(x[e] - mean, x[e] - mean, fmaf(y[e] - mean, y[e] - mean, sq));
            const float inv = rsqrtf(lanes_sum<G>(sq) * (1.0f / D) + r.eps);
            float wl[V], wh[V], bl[V], bh[V];
            ld_values(r.kn_w + c, wl), ld_values(r.kn_w + c2, wh), ld_values(r.kn_b + c, bl), ld_values(r.kn_b + c2, bh);
#pragma unroll
            for (int e = 0; e < V; e++) {
                x[e] = fmaf((x[e] - mean) * inv, wl[e], bl[e]);
                y[e] = fmaf((y[e] - mean) * inv, wh[e], bh[e]);
            }
        }
        if (rope && turns[i]) {
#pragma unroll
            for (int e = 0; e < V; e++) {
                const float u = x[e], v = y[e];
                x[e] = fmaf(u, cl[i][e], -(v * sl[i][e]));
                y[e] = fmaf(v, ch[i][e], u * sh[i][e]);
            }
        }
    };
    const auto held = [&](float x) { return fabsf(x) < INFINITY ? fminf(fmaxf(x, -kHeldMost<T>), kHeldMost<T>) : x; };

    const int head0 = is_v ? which - a.split : which;
    load(rounds - 1, head0);
    if (rounds == 1) {
#pragma unroll
        for (int i = 0; i < P; i++) find_turn(row_of(0, i), i);
    }
    int turn = 0;
    for (int head = head0; head < r.h_kv; head += a.split, turn ^= 1) {
        uint8_t* codes = (is_v ? a.v_cache : a.k_cache) + ((block0 + head) << r.page_shift) * D;
        const int old = t.first > 0 ? min(static_cast<int>(scales[head]), kScaleMost) : 0;
        float x[P][V], y[P][V], most = 0.0f;
        for (int round = rounds - 1; round >= 0; round--) {
            if (round < rounds - 1) load(round, head);
#pragma unroll
            for (int i = 0; i < P; i++) {
                if (rounds > 1) find_turn(row_of(round, i), i);
                turned(i, x[i], y[i]);
                if (row_of(round, i) >= t.rows) continue;
#pragma unroll
                for (int e = 0; e < V; e++) {
                    const float m = fabsf(x[i][e]), n = fabsf(y[i][e]);
                    most = fmaxf(most, fmaxf(m < INFINITY ? m : 0.0f, n < INFINITY ? n : 0.0f));
                }
            }
        }
        if (rounds == 1 && head + a.split < r.h_kv) load(0, head + a.split);
        most = wave_max(most);
        if constexpr (W > 1) {
            if (lane == 0) tops[turn][wave] = most;
            __syncthreads();  // (every wave has read the old scale, too)
#pragma unroll
            for (int w = 0; w < W; w++) most = fmaxf(most, tops[turn][w]);
        }
        const int next = max(old, scale_for(fminf(most, kHeldMost<T>)));
        const float inv = scale_value(2 * kScaleBias - next);
        for (int round = 0; round < rounds; round++) {
            if (round > 0) load(round, head);
#pragma unroll
            for (int i = 0; i < P; i++) {
                const int row = row_of(round, i);
                if (round > 0) {
                    find_turn(row, i);
                    turned(i, x[i], y[i]);
                }
                if (row >= t.rows) continue;
                uint8_t* p = codes + static_cast<int64_t>(t.first + row) * D;
#pragma unroll
                for (int half = 0; half < 2; half++) {
                    const float(&z)[V] = half ? y[i] : x[i];
                    uint32_t w[V / 4];
#pragma unroll
                    for (int e = 0; e < V / 4; e++)
                        w[e] = codes_of(held(z[4 * e]) * inv, held(z[4 * e + 1]) * inv, held(z[4 * e + 2]) * inv, held(z[4 * e + 3]) * inv);
                    uint32_t* at = reinterpret_cast<uint32_t*>(p + (half ? c2 : c));
                    if constexpr (V == 8)
                        *reinterpret_cast<u32x2*>(at) = u32x2{w[0], w[1]};
                    else
                        *at = w[0];
                }
            }
        }
        if (next > old && t.first > 0) {
            for (int64_t i = (wave * 64 + lane) * 16; i < static_cast<int64_t>(t.first) * D; i += W * 1024) {
                u32x4 w = ld16(codes + i);
#pragma unroll
                for (int e = 0; e < 4; e++) w[e] = codes_down(w[e], next - old);
                st16(codes + i, w);
            }
        }
        if (wave == 0 && lane == 0) scales[head] = static_cast<uint8_t>(next);
        if (rounds > 1 && head + a.split < r.h_kv) load(rounds - 1, head + a.split);
    }
}

// A call's rows, then its pages.
template <typename T, int D, bool NORM, bool ROPE>
__global__ __launch_bounds__(256) void kv_append_f8_kernel(Append8Args<T> a) {
    const int block = blockIdx.x;
    if (block < a.row_blocks)
        append_rows<T, D, NORM, ROPE>(a.rows, block * 4 + wave_in_block());
    else
        append_page<T, D, NORM, ROPE, 1>(a, (block - a.row_blocks) * 4 + wave_in_block());
}
template <typename T, int D, bool NORM, bool ROPE>
__global__ __launch_bounds__(256) void append_rows_kernel(Append8Args<T> a) {
    append_rows<T, D, NORM, ROPE>(a.rows, static_cast<int>(blockIdx.x) * 4 + wave_in_block());
}
template <typename T, int D, bool NORM, bool ROPE, int W>
__global__ __launch_bounds__(W == 2 ? 128 : 256) void append_pages_kernel(Append8Args<T> a) {
    append_page<T, D, NORM, ROPE, W>(a, W == 1 ? static_cast<int>(blockIdx.x) * 4 + wave_in_block() : static_cast<int>(blockIdx.x));
}

template <typename T, int D, bool NORM, bool ROPE>
hs_status launch_append_f8(const char* op, hipStream_t st, Append8Args<T> a, int64_t row_blocks, int64_t pages) {
    const int h_kv = a.rows.h_kv, page = 1 << a.rows.page_shift;
    a.row_blocks = static_cast<int>(row_blocks);
    if (!a.offsets) {
        a.split = h_kv;
        const int64_t blocks = row_blocks + ceil_div(pages * 2 * h_kv, 4);
        kv_append_f8_kernel<T, D, NORM, ROPE><<<dim3(static_cast<uint32_t>(blocks)), dim3(256), 0, st>>>(a);
        return check_launch(op);
    }
    const int waves = page <= 2048 / D ? 1 : page <= 4096 / D ? 2 : 4;
    // a page's heads by so many waves that the chip has 16 waves a CU
    a.split = static_cast<int>(std::clamp<int64_t>(ceil_div(int64_t{16} * num_cus(), 2 * pages * waves), 1, h_kv));
    const int64_t units = pages * 2 * a.split;
    const auto go = [&](auto kernel, int64_t blocks, int threads) { kernel<<<dim3(static_cast<uint32_t>(blocks)), dim3(threads), 0, st>>>(a); };
    if (waves == 1)
        go(append_pages_kernel<T, D, NORM, ROPE, 1>, ceil_div(units, 4), 256);
    else if (waves == 2)
        go(append_pages_kernel<T, D, NORM, ROPE, 2>, units, 128);
    else
        go(append_pages_kernel<T, D, NORM, ROPE, 4>, units, 256);
    if (hs_status rc = check_launch(op)) return rc;
    if (row_blocks) append_rows_kernel<T, D, NORM, ROPE><<<dim3(static_cast<uint32_t>(row_blocks)), dim3(256), 0, st>>>(a);
    return check_launch(op);
}

// ---------------------------------------------------------------------------
// attention_paged
//
// Single tokens: as attention_paged (hs_paged.hip), of half its bytes or a
// quarter. A wave takes kStep keys at a time on its own; codes become f16 (f16
// caches) or bf16 (f32) values with their page's scale on the way (hs_f8.hpp): K's in
// the registers that the load filled, as the A operand of S^T = K Q^T, V's on
// their way to the wave's slice of LDS, from which V^T takes P^T. What the codes
// leave to round is the query and the weights: in f16 weights go as two f16 values
// of 11 bits each (the queries are f16), in f32 both go as three bf16 ones, which
// hold all 24 bits.
//
// 64 sequences of up to 8192 keys, 32 heads of 128 over 8, f16: 103 us, 5.0 TB/s, of
// which the join is 5 (the same loads with nothing computed: 98); one token over
// 130531 keys of 16 heads of 64 53 us, 5.0 TB/s (48); eight f32 sequences of up to
// 800, 16 heads of 128, 13 us; 32 sequences of up to 4000, 16 heads of 64, 33 (f32 35),
// over pages of 8 keys 35 (38). At head dim 64 a wave's step is 64 keys: 30 us, and 34
// with steps of 32; at 128 it is 32, as steps of 64 spill. Pieces are made of 256 keys:
// 29 us, and 33 made of 128 (20 sequences of up to 3001, 16 heads of 128).
template <typename T, int D>
struct Paged8 : Steps8<T, D, 1> {
    using S = Steps8<T, D, 1>;
    static constexpr int kUnit = 256;               // keys of which pieces are made
    // workgroups of a CU, by their registers (with one more, spilled: the f32 figures
    // above 74 and 106 us)
    static constexpr int per_cu(bool whole) { return D == 64 ? (S::kHalf && whole ? 4 : 3) : S::kHalf || whole ? 3 : 2; }
    struct Smem {
        union {
            uint16_t v[kPagedWaves][32 * S::kPitch];  // half of a step's keys at a time
            float o[kPagedWaves][kGroup * S::kOPitch];
        };
        float m[kPagedWaves][kGroup], l[kPagedWaves][kGroup];
    };
};

struct Paged8Args : PagedArgs {
    const uint8_t *k_scale, *v_scale;
};

template <typename T, int D, bool WHOLE>
__global__ __launch_bounds__(64 * kPagedWaves, (Paged8<T, D>::per_cu(WHOLE))) void attention_paged_f8_kernel(Paged8Args a) {
    using P = Paged8<T, D>;
    __shared__ __align__(16) typename P::Smem sm;

    Piece t;
    if (!find_piece(a, P::kUnit, t)) return;  // workgroup-uniform, before any barrier
    const int s = t.s, begin = t.begin, end = t.end, count = t.count, kv = t.kv, pass = t.pass;
    const int live_heads = min(a.width, a.group - pass * a.width);
    const int head0 = kv * a.group + pass * a.width;

    // (a copy of the last query head beyond them)
    const T* q[1] = {static_cast<const T*>(a.q) + s * a.q_stride + (head0 + min(lane_id() & 15, live_heads - 1)) * D};
    f32x4 o[1][D / 16];
    float m[1], l[1];
    const int* pages = a.page_table + static_cast<int64_t>(s) * a.max_pages;
    const int odd = attend_steps<T, D, 1, WHOLE, false>(a, pages, kv, begin, end, q, {0}, 0, sm.v[wave_in_block()], o, m, l);
    join_waves<T, D, true>(a, sm, s, count, head0, live_heads, o[0], m[0], l[0],
                           [&](float* sums) { odd_values<T, D, 1, false>(a, pages, kv, begin, end, {0}, 0, odd, sums); });
}

template <typename T, int D>
hs_status launch_paged_f8(const char* op, hipStream_t st, const Paged8Args& a) {
    using P = Paged8<T, D>;
    return launch_pieces<T, D, true>(op, st, a, attention_paged_f8_kernel<T, D, true>, attention_paged_f8_kernel<T, D, false>, P::kUnit, P::per_cu(a.page_shift >= 4));
}

}  // namespace
}  // namespace hs

extern "C" hs_status hs_kv_append_f8(hs_stream_t stream, hs_dtype dt, const void* q, int64_t q_stride, const void* k,
                                     int64_t k_stride, const void* v, int64_t v_stride, const float* qn_w,
                                     const float* qn_b, const float* kn_w, const float* kn_b, const float* sin_tab,
                                     const float* cos_tab, int32_t table_rows, const void* positions,
                                     const void* offsets, const void* page_table, const void* lens, void* q_out,
                                     void* k_out, void* k_cache, void* v_cache, void* k_scale, void* v_scale,
                                     int64_t n, int32_t b, int32_t h, int32_t h_kv, int32_t d, int32_t page,
                                     int32_t n_pages, int32_t max_pages, float eps) {
    using namespace hs;
    const char* op = "kv_append_f8";
    AppendCall c{q, k, v, q_stride, k_stride, v_stride, qn_w, qn_b, kn_w, kn_b, sin_tab, cos_tab, table_rows, positions,
                 offsets, page_table, lens, q_out, k_out, n, b, h, h_kv, d, page, n_pages, max_pages, eps};
    bool done = false;
    if (hs_status rc = check_append(op, dt, c, done)) return rc;
    if (done) return HS_OK;
    if (hs_status rc = check_cache_f8(op, k_cache, v_cache, k_scale, v_scale, page_table, lens, page, n_pages, max_pages, h_kv, d)) return rc;
    const int64_t cache = static_cast<int64_t>(n_pages) * page * h_kv * d, scales = static_cast<int64_t>(n_pages) * h_kv;
    const ByteRange outs[6] = {c.q_rows(dt), c.k_rows(dt), {k_cache, cache}, {v_cache, cache}, {k_scale, scales}, {v_scale, scales}};
    if (hs_status rc = check_append_overlaps(op, dt, c, outs, 6)) return rc;
    // rows of q, and of k where they are asked for: waves as kv_append's
    const int64_t heads = static_cast<int64_t>(c.h) + (k_out ? h_kv : 0);
    const int parts = static_cast<int>(ceil_div(heads, dt == HS_F16 ? 1024 / d : 512 / d));
    const int64_t row_blocks = ceil_div(n * parts, 4);
    // pages that the tokens can lie in, at most
    const int64_t pages = offsets ? n / page + 2 * std::min<int64_t>(b, n) : b;
    if (row_blocks + ceil_div(pages * 2 * h_kv, page <= 2048 / d || !offsets ? 4 : 1) >= (int64_t{1} << 23)) return fail(HS_EINVAL, "%s: too many tokens", op);
    const auto run = [&](auto zero) {
        using T = decltype(zero);
        Append8Args<T> a;
        c.fill(a.rows);
        a.rows.parts = parts, a.rows.heads = static_cast<int>(heads);
        a.rows.k_cache = a.rows.v_cache = nullptr, a.rows.n_pages = 0;  // rows only
        a.offsets = static_cast<const int*>(offsets), a.page_table = static_cast<const int*>(page_table);
        a.lens = static_cast<const int*>(lens);
        a.k_cache = static_cast<uint8_t*>(k_cache), a.v_cache = static_cast<uint8_t*>(v_cache);
        a.k_scale = static_cast<uint8_t*>(k_scale), a.v_scale = static_cast<uint8_t*>(v_scale);
        a.n_pages = n_pages;
        const auto st = static_cast<hipStream_t>(stream);
        const bool norm = qn_w || kn_w, rope = sin_tab;
        const auto go = [&](auto dim) {
            constexpr int D = decltype(dim)::value;
            if (norm) return rope ? launch_append_f8<T, D, true, true>(op, st, a, row_blocks, pages) : launch_append_f8<T, D, true, false>(op, st, a, row_blocks, pages);
            return rope ? launch_append_f8<T, D, false, true>(op, st, a, row_blocks, pages) : launch_append_f8<T, D, false, false>(op, st, a, row_blocks, pages);
        };
        return d == 64 ? go(std::integral_constant<int, 64>{}) : go(std::integral_constant<int, 128>{});
    };
    return dt == HS_F16 ? run(f16{}) : run(float{});
}

extern "C" int64_t hs_attention_paged_f8_workspace(int32_t b, int32_t h, int32_t h_kv, int32_t d) {
    return hs_attention_paged_workspace(b, h, h_kv, d);  // pieces are cut alike
}

extern "C" hs_status hs_attention_paged_f8(hs_stream_t stream, hs_dtype dt, const void* q, int64_t q_stride,
                                           const void* k_cache, const void* v_cache, const void* k_scale,
                                           const void* v_scale, const void* page_table, const void* lens, void* out,
                                           void* workspace, int64_t workspace_bytes, int32_t b, int32_t h,
                                           int32_t h_kv, int32_t d, int32_t page, int32_t n_pages, int32_t max_pages,
                                           float scale) {
    using namespace hs;
    const char* op = "attention_paged_f8";
    if (hs_status rc = check_heads(op, dt, h, h_kv, d)) return rc;
    if (b < 0) return fail(HS_EINVAL, "%s: negative count", op);
    if (b == 0 || h == 0) return HS_OK;
    if (static_cast<int64_t>(b) * h >= (int64_t{1} << 23)) return fail(HS_EINVAL, "%s: b * Hq must be below 2^23", op);
    const int64_t need = hs_attention_paged_f8_workspace(b, h, h_kv, d);
    if (hs_status rc = check_attend_f8(op, dt, {q, q_stride, k_cache, v_cache, k_scale, v_scale, page_table, lens, out, workspace,
                                                workspace_bytes, b, h, h_kv, d, page, n_pages, max_pages, scale}, need))
        return rc;
    Paged8Args p;
    p.q = q, p.k = k_cache, p.v = v_cache, p.out = out, p.q_stride = q_stride;
    p.ws_o = static_cast<float*>(workspace);
    p.page_table = static_cast<const int*>(page_table), p.lens = static_cast<const int*>(lens);
    p.k_scale = static_cast<const uint8_t*>(k_scale), p.v_scale = static_cast<const uint8_t*>(v_scale);
    p.b = b, p.h = h, p.h_kv = h_kv, p.page_shift = exact_log2(page), p.n_pages = n_pages;
    p.max_pages = n_pages > 0 ? max_pages : 0;  // no page to read: no sequence has keys
    p.scale = scale;
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (dt == HS_F16) return d == 64 ? launch_paged_f8<f16, 64>(op, st, p) : launch_paged_f8<f16, 128>(op, st, p);
    return d == 64 ? launch_paged_f8<float, 64>(op, st, p) : launch_paged_f8<float, 128>(op, st, p);
}
