// Attention of several new tokens per sequence over a paged cache held in 8 bits,
// for gfx950: O_i = sum_j w_ij v_j / sum_j w_ij, w_ij = exp(scale q_i k_j - m_i) over
// the keys j of its sequence that query i sees, in one pass over the keys with a
// running m_i.
//
// A workgroup takes a tile of one sequence and key head: kRows rows, a row being a
// token and one of the query heads that share the key head, tokens first. So few
// tokens of shared heads fill a tile, and a key is read and turned from its code
// once for all heads that see it. Keys go through LDS 64 at a time, double
// buffered: codes of the next ones lie in registers while these compute, and become
// f16 (f16 caches) or bf16 (f32) values with their page's scale on the way into LDS
// (hs_f8.hpp). Scores are transposed, S^T = K Q^T: lanes n and n + 32 hold row n's, so
// its statistics are the lane's own, and V^T takes P^T from the registers that the
// scores were in.
//
// Lengths are device data: the launch has a workgroup for every item that there
// can be, and each finds its own. Where tiles are few the keys are cut into pieces,
// of which an item is one, and a second launch joins them.
//
// Bounds: f16, matrix and vector issue, which overlap in part (at head dim 64 the
// exponentials alone take as many cycles as the products): 8192 tokens over
// themselves, 32 heads of 128 over 8, 1.18 ms, 930 TFLOP/s, causal 0.62 ms, 885; 16
// heads of 64 0.34 ms, 800 (a plain product of 8192^3 reaches 1090 to 1246). f32, three
// products for one of f16, of bf16 values: 4096 tokens, 32 heads of 128 over 8, 657
// us, 418 TFLOP/s, 16 heads of 64 202 us, 340 (the f32 matrix instructions' plain
// product reaches 154). (Codes asked for two tiles ahead gain 2% at head dim 128 and
// spill in f32: 4096 tokens of 32 heads 742 us.) Sequences of few tokens: few_rows.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "hs_steps_f8.hpp"

namespace hs {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kXcds = 8;
constexpr int kBN = 64;  // keys per tile

__device__ __forceinline__ uint32_t pk_f16(float a, float b) {
    f16x2 h;
    h.x = static_cast<f16>(a), h.y = static_cast<f16>(b);
    return h22u(h);
}
// v of this lane and of lane ^ 32, in the same order in both.
__device__ __forceinline__ f32x2 both_halves(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(f2u(v), f2u(v), false, false);
    return f32x2{u2f(static_cast<uint32_t>(r[0])), u2f(static_cast<uint32_t>(r[1]))};
}
__device__ __forceinline__ float halves_max(float v) {
    const f32x2 r = both_halves(v);
    return fmaxf(r.x, r.y);
}
__device__ __forceinline__ float halves_sum(float v) {
    const f32x2 r = both_halves(v);
    return r.x + r.y;
}

struct PromptArgs {
    const void* q;
    const uint8_t *k, *v, *k_scale, *v_scale;
    void* out;
    int64_t q_stride;
    const int *page_table, *lens, *offsets;
    int n, b, h, h_kv, group, page_shift, n_pages, max_pages, causal;
    float scale;
    // keys cut into pieces
    int4* cut;            // per tile: its first item, its pieces, its first row of all, its rows; behind them the tiles' number
    float *ws_o, *ws_ml;  // per (item, key head, row of the tile): D sums; maximum and weight sum
    int tiles;            // of a key head at most
    int places;           // workgroups of a key head that the chip holds at once; 0: whole keys
    bool one_round;       // fewer tiles than those
    int items, blocks;    // items of a key head that the launch has, blocks of 32 rows of each
};

// One sequence: its queries' rows, the first one's key number and the keys it holds.
// (Its last query is its last key, also where its rows end past the ones given.)
struct PromptSeq {
    int q0, nq, key0, nk;
};
__device__ __forceinline__ PromptSeq sequence_at(const PromptArgs& a, int s) {
    const RowRange r = row_range(a.offsets, s, a.n);
    const int nq = r.end - r.begin;
    return {r.begin, nq, nq > 0 ? max(a.lens[s], 0) - (a.offsets[s + 1] - r.begin) : 0, held_length(a.lens, s, a.max_pages, a.page_shift)};
}
// Keys that the sequence's query i sees.
__device__ __forceinline__ int keys_seen(const PromptSeq& t, int i, int causal) {
    if (causal == 0) return t.nk;
    const int at = t.key0 + i;
    if (at < 0) return 0;
    const int64_t end = causal == 1 ? static_cast<int64_t>(at) + 1 : (static_cast<int64_t>(at / causal) + 1) * causal;
    return end < t.nk ? static_cast<int>(end) : t.nk;
}

// An item: piece `piece` of the pieces of a tile. `fair` units of 64 keys are what each
// of the key head's places on the chip gets of all tiles' work (half of a causal
// mask's own keys count). Where tiles are fewer than places, one sequence's tiles are cut
// into as many whole fair parts as they have, so that the call is one round, and those
// of several into pieces of up to `most` units: a fair part, larger by what rounding
// up to whole pieces adds, half a piece a tile as a rule, and then by what it adds
// (whole fair parts of each are up to two long: 8 tokens each of 32 sequences of up to
// 4000 keys, 32 heads of 128 over 8, 84 us for 64). Else only tiles that would outlast
// the others are cut, into pieces of 3/4 of a fair part. A
// sequence's pieces are of one size, `chunk`. Every workgroup computes this from all
// lengths, 64 a step. The total is at least half of the exact one, so a call's items
// do not pass 8/3 of the places and its tiles; what else offsets that do not ascend
// may come to is left out.
constexpr int kLeastUnits = 8;  // (4: one token each of 32 sequences, 28 heads of 64 over 4, 21.5 us for 19.6; 12: 21.7)
constexpr float kLonger = 16.0f;  // units that a tile's writing and joining of pieces cost, and more

struct PromptItem {
    int s, tiles, local;  // sequence, its tiles, the one
    int piece, pieces, chunk, item;  // item: piece 0's
    int tile;                        // of the call's
};
__device__ __forceinline__ int tiles_of(const PromptArgs& a, int nq, int rows) {
    return static_cast<int>((static_cast<int64_t>(nq) * a.group + rows - 1) / rows);
}
__device__ __forceinline__ int wave_most(int v) {
    v = max(v, dpp_zero<kQuadXor1>(v));
    v = max(v, dpp_zero<kQuadXor2>(v));
    v = max(v, dpp_zero<kRowHalfMirror>(v));
    v = max(v, dpp_zero<kRowMirror>(v));
    return max(max(lane_value(v, 0), lane_value(v, 16)), max(lane_value(v, 32), lane_value(v, 48)));
}
__device__ __forceinline__ bool find_item(const PromptArgs& a, int rows, int index, PromptItem& t) {
    const int lane = lane_id();
    // of the sequence base + lane: its tiles, and its keys in units
    const auto sizes = [&](int base) {
        if (base + lane >= a.b) return int2{0, 0};
        const PromptSeq s = sequence_at(a, base + lane);
        return int2{tiles_of(a, s.nq, rows), (s.nk + kBN - 1) / kBN};
    };
    const int2 first = sizes(0);  // read once: few calls have more than 64
    float fair = 16777216.0f, most = fair;
    if (a.places > 0) {
        float total = 0.0f, tiles = 0.0f;
        for (int base = 0; base < a.b; base += 64) {
            const int2 x = base ? sizes(base) : first;
            int masked = 0;
            if (a.causal && base + lane < a.b) {
                const PromptSeq s = sequence_at(a, base + lane);
                masked = max(min(s.nq, s.nk) - a.causal, 0);
            }
            total += static_cast<float>(x.x) * (static_cast<float>(x.y) - static_cast<float>(masked) * (0.5f / kBN));
            tiles += static_cast<float>(x.x);
        }
        const float places = static_cast<float>(a.places);
        fair = fmaxf(wave_sum(total) / places, static_cast<float>(kLeastUnits));
        most = fair;
        if (a.one_round && a.b > 1) {
            most = fair * places / (places - 0.5f * fminf(wave_sum(tiles), places));
            float items = 0.0f;
            for (int base = 0; base < a.b; base += 64) {
                const int2 x = base ? sizes(base) : first;
                items += static_cast<float>(x.x) * ceilf(static_cast<float>(x.y) / most);
            }
            most *= fmaxf(wave_sum(items) / places, 1.0f);
        }
    }
    int tiles_before = 0, items_before = 0;
    for (int base = 0; base < a.b; base += 64) {
        const int2 x = base ? sizes(base) : first;
        const int tiles = x.x, units = x.y;
        int pieces = 1;
        if (a.one_round)
            pieces = max(static_cast<int>(a.b > 1 ? ceilf(static_cast<float>(units) / most) : static_cast<float>(units) / fair), 1);
        else if (static_cast<float>(units) > fair + kLonger)
            pieces = static_cast<int>(ceilf(static_cast<float>(units) / (0.75f * fair)));
        const int chunk = max((units + pieces - 1) / pieces, 1);
        // in several rounds the sequences of long pieces first, by quarters of the
        // longest, so that a call does not end on them (309 us for 360 of five prompts;
        // in one round it is 3 us of finding work)
        const bool ordered = a.b > 1 && !a.one_round;
        int tile_sum = 0, item_sum = 0, tile_end = 0, item_end = 0;
        const int longest = ordered ? wave_most(chunk) : chunk;
        const int quarter = ordered ? min((longest - chunk) * 4 / longest, 3) : 0;
        for (int k = 0; k < (ordered ? 4 : 1); k++) {
            const int tile_add = wave_prefix_sum(quarter == k ? tiles : 0);
            const int item_add = wave_prefix_sum(quarter == k ? tiles * pieces : 0);
            if (quarter == k) tile_sum = tile_end + tile_add, item_sum = item_end + item_add;
            tile_end += lane_value(tile_add, 63), item_end += lane_value(item_add, 63);
        }
        const uint64_t hit = __ballot(items_before + item_sum > index && items_before + item_sum - tiles * pieces <= index);
        if (hit) {
            const int l = __builtin_ctzll(hit);
            t.s = base + l;
            t.tiles = lane_value(tiles, l), t.pieces = lane_value(pieces, l), t.chunk = lane_value(chunk, l);
            const int before = items_before + lane_value(item_sum, l) - t.tiles * t.pieces;
            // all tiles' first pieces, then their second ones, ..: sizes fall slowly
            // with the number. (Workgroups go to an XCD's four engines in turn and wait
            // for theirs: with a tile's long and short pieces beside each other two
            // engines had all the long ones, 2048 tokens over 4096 took 188 us for 179.)
            const int rest = index - before;
            t.piece = rest / t.tiles;
            t.local = rest - t.piece * t.tiles;
            t.item = before + t.local * t.pieces;
            t.tile = tiles_before + lane_value(tile_sum, l) - t.tiles + t.local;
            return t.item + t.pieces <= a.items;
        }
        tiles_before += tile_end, items_before += item_end;
    }
    return false;
}
// Pieces of a tile whose last query sees `most` keys: the ones that see any.
__device__ __forceinline__ int pieces_seen(int most, int chunk) {
    return max(static_cast<int>((most + static_cast<int64_t>(kBN) * chunk - 1) / (static_cast<int64_t>(kBN) * chunk)), 1);
}

// What a workgroup works on.
struct PromptTile {
    PromptSeq seq;
    int s, kv;
    int first, rows;              // its rows of the sequence's: from `first` on, and how many the sequence has
    int begin, end, count, item;  // keys of the piece, of how many the tile has, its place
};
// Workgroup b runs on XCD b % 8: where the key heads divide by it, an XCD takes h_kv
// / 8 of them in a row, so that a head's tiles read their keys through one L2. A
// sequence's last queries see the most keys and go first.
__device__ __forceinline__ bool prompt_tile(const PromptArgs& a, int rows, PromptTile& t) {
    const int b = blockIdx.x;
    int index;
    if (a.h_kv % kXcds == 0) {
        const int slot = b / kXcds, heads = a.h_kv / kXcds;
        index = slot / heads;
        t.kv = b % kXcds * heads + slot % heads;
    } else {
        index = b / a.h_kv;
        t.kv = b % a.h_kv;
    }
    PromptItem c;
    if (a.places > 0 && b == 0) {
        int tiles = 0;
        for (int base = 0; base < a.b && tiles < a.tiles; base += 64) {
            const int s = base + lane_id();
            tiles += lane_value(wave_prefix_sum(s < a.b ? tiles_of(a, sequence_at(a, s).nq, rows) : 0), 63);
        }
        if (threadIdx.x == 0) a.cut[a.tiles] = {min(tiles, a.tiles), 0, 0, 0};
    }
    if (!find_item(a, rows, index, c)) return false;
    t.s = c.s, t.seq = sequence_at(a, c.s);
    t.rows = t.seq.nq * a.group;
    t.first = (c.tiles - 1 - c.local) * rows;
    const int most = keys_seen(t.seq, (min(t.first + rows, t.rows) - 1) / a.group, a.causal);
    t.count = pieces_seen(most, c.chunk), t.item = c.item + c.piece;
    if (a.places > 0 && c.piece == 0 && t.kv == 0 && threadIdx.x == 0 && c.tile < a.tiles)
        a.cut[c.tile] = {c.item, t.count, t.seq.q0 * a.group + t.first, min(t.rows - t.first, rows)};
    if (c.piece >= t.count) return false;
    const int64_t begin = static_cast<int64_t>(c.piece) * c.chunk * kBN;
    t.begin = static_cast<int>(begin);
    t.end = c.piece + 1 < t.count ? static_cast<int>(begin + static_cast<int64_t>(c.chunk) * kBN) : most;
    return true;
}

// A reference before any score: finite, so that a masked score weighs nothing.
constexpr float kStart = -3.0e38f;

// Whether there are any of the keys [begin, end). (Asked of a row whose weights come to
// 0: of one that sees no key the result is 0, of one whose scores are all -infinity
// NaN. A piece's row of the latter kind has a maximum above kStart.)
__device__ __forceinline__ bool any_keys(const PromptArgs& a, const int* pages, int begin, int end) {
    for (int i = begin >> a.page_shift; begin < end && i <= (end - 1) >> a.page_shift; i++)
        if (pages[i] >= 0 && pages[i] < a.n_pages) return true;
    return false;
}
// A result of sums over their weight, which are none's where `none`.
__device__ __forceinline__ float over_weight(float sum, float weight, bool none) {
    return weight != 0.0f ? sum / weight : none ? 0.0f : u2f(0x7FC00000u);
}

// A piece's 32 rows of a wave in the workspace: D sums each as the lanes hold them,
// registers 4 i .. + 4 of all lanes after one another, so that a store is 1 KiB in a
// row (by rows, it is 32 bytes of each).
__device__ __forceinline__ int64_t partial_block(const PromptArgs& a, int item, int kv, int wave) {
    return (static_cast<int64_t>(item) * a.h_kv + kv) * a.blocks + wave;
}
__device__ __forceinline__ int64_t row_out(const PromptArgs& a, const PromptSeq& s, int kv, int row) {
    const int token = row / a.group;
    return static_cast<int64_t>(s.q0 + token) * a.h + kv * a.group + (row - token * a.group);
}

// The reference of a row's weights is set this far (log2) below its largest score,
// so that its largest weight is 2^12: f16 weights keep 11 bits down to 2^-26 of the
// largest. It moves when one would pass f16.
//
// A weight is one f16 value here, and two in few_rows and attention_paged, whose time is
// the keys' bytes. Two would bring the results' distance from 64 bits from 2.8e-4 to the
// 2.07e-4 that their own rounding makes (1374 tokens over 30228, 16 heads of 64), for
// half as many products again: 378 us for 260, five prompts of 32 heads of 128 over 8
// 396 for 311, 8192 tokens over themselves 870 for 640 and, 16 heads of 64, 600 for 342.
constexpr float kWeightBits = 12.0f;
constexpr float kPastF16 = 65520.0f;  // the least that f16 rounds to infinity
// Tiles for which a wave looks for the scores' maximum ahead of the weights once
// references have moved.
constexpr int kWary = 8;
// A maximum (log2) beyond which its rounding, 2^-24 of it, shows in a weight.
constexpr float kFar = 65536.0f;

template <typename T, int D, int W>
struct Prompt8 {
    static constexpr bool kHalf = sizeof(T) == 2;
    static constexpr int kThr = 64 * W, kRows = 32 * W;
    static constexpr int kParts = kHalf ? 1 : 3;   // of a query value and of a weight
    static constexpr int KS = D / 16, DB = D / 32;
    static constexpr int kLoad = kBN * D / kThr < 16 ? kBN * D / kThr : 16;  // codes of a load
    static constexpr int kPieces = D / kLoad;      // loads of a row
    static constexpr int kRowStep = kThr / kPieces, kWaveRows = 64 / kPieces;
    static constexpr int kPer = kBN / kRowStep;    // loads of a thread
    // 16-bit values per row: K's 16 rows at one column, and the transposing read's 4
    // rows of 64 bytes, touch every bank once
    static constexpr int kKPitch = D + 8, kVPitch = D + 32;
    // waves of a SIMD, by the registers and LDS; workgroups of a CU
    static constexpr int kPerCu = D == 64 ? (kHalf ? (W == 8 ? 4 : 3) : 3) : 2;
    static constexpr int kGroups = kPerCu * 4 / W;
    struct Smem {
        uint16_t k[2][kBN * kKPitch];
        uint16_t v[2][kBN * kVPitch];
        uint8_t there[2][kBN];
        int gap[2];  // the tile of each buffer if some of its keys are not there
        int odd;     // a tile whose values not every row sees holds infinities or NaN, left out
    };
};

template <typename T>
__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
    if constexpr (sizeof(T) == 2)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(as_h8(a), as_h8(b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// A sequence of up to 16 R rows: its waves take the keys in turn, each all rows, as
// single tokens' do, and join in LDS. A tile's scheme has one wave of four compute and
// one tile of keys under way; this one is bound by memory: 2 tokens each of 32 sequences
// of up to 4000 keys, 16 heads of 64, 38 us, 3.3 TB/s (65), 32 heads of 128 over 8, 43
// (62; f32 45, 90), 8 tokens each, R = 2, 50 (65); with a prompt of 512 tokens beside 31
// single ones 46 (77). 128 tokens, 28 heads of 64 over 4, 26: finding the work, the first
// codes and the join are 13 of them. (A long prompt's last few rows stay a tile, beside
// its others: 168 us, 179 as these; f32 at head dim 128 by rows spills with R = 2, 142 us
// for 95.)
template <typename T, int D>
struct FewRows {
    using S = Steps8<T, D, 2>;
    union {
        uint16_t v[kPagedWaves][32 * S::kPitch];
        float o[kPagedWaves][32 * S::kOPitch];
    };
    float m[kPagedWaves][32], l[kPagedWaves][32];
};
template <typename T, int D, int R, bool WHOLE>
__device__ __forceinline__ void few_rows(const PromptArgs& a, const PromptTile& t, FewRows<T, D>& sm) {
    using S = Steps8<T, D, R>;
    constexpr int DB = D / 16;
    const int lane = lane_id(), wave = wave_in_block(), n = lane & 15, g = lane >> 4;
    const int* pages = a.page_table + static_cast<int64_t>(t.s) * a.max_pages;
    const T* q[R];
    int seen[R];
#pragma unroll
    for (int i = 0; i < R; i++) {
        const int r = min(t.first + 16 * i + n, t.rows - 1), token = r / a.group;
        q[i] = static_cast<const T*>(a.q) + (t.seq.q0 + token) * a.q_stride + (t.kv * a.group + (r - token * a.group)) * D;
        seen[i] = keys_seen(t.seq, token, a.causal);
    }
    const int least = keys_seen(t.seq, t.first / a.group, a.causal);
    f32x4 o[R][DB];
    float m[R], l[R];
    const int odd = attend_steps<T, D, R, WHOLE, true>(a, pages, t.kv, t.begin, t.end, q, seen, least, sm.v[wave], o, m, l);
    const int live = min(t.rows - t.first, 16 * R);
    __syncthreads();
#pragma unroll
    for (int r = 0; r < R; r++) {
        const int row = 16 * r + n;
#pragma unroll
        for (int i = 0; i < DB; i++) *reinterpret_cast<f32x4*>(&sm.o[wave][row * S::kOPitch + 16 * i + 4 * g]) = o[r][i];
        if (g == 0) sm.m[wave][row] = m[r], sm.l[wave][row] = l[r];
    }
    odd_values<T, D, R, true>(a, pages, t.kv, t.begin, t.end, seen, least, odd, sm.o[wave]);
    __syncthreads();
    const int64_t block = partial_block(a, t.item, t.kv, 0);
    for (int x = threadIdx.x; x < 8 * D; x += 64 * kPagedWaves) {
        // pieces as the other tiles' (partial_block), else rows of channels
        const bool piece = t.count > 1;
        const int row = piece ? x % 32 : x / (D / 4), d0 = piece ? x / 64 * 8 + x / 32 % 2 * 4 : x % (D / 4) * 4;
        if (row >= live) continue;
        float top = sm.m[0][row];
#pragma unroll
        for (int w = 1; w < kPagedWaves; w++) top = fmaxf(top, sm.m[w][row]);
        float weight = 0.0f;
#pragma unroll
        for (int w = 0; w < kPagedWaves; w++) weight = fmaf(sm.l[w][row], __builtin_amdgcn_exp2f(sm.m[w][row] - top), weight);
        const f32x4 sum = joined([&](auto keep) {
            f32x4 s = {};
#pragma unroll
            for (int w = 0; w < kPagedWaves; w++)
                s += times(*reinterpret_cast<const f32x4*>(&sm.o[w][row * S::kOPitch + d0]), __builtin_amdgcn_exp2f(sm.m[w][row] - top), keep);
            return s;
        });
        if (weight == 0.0f) {
            const bool sees = any_keys(a, pages, t.begin, min(keys_seen(t.seq, (t.first + row) / a.group, a.causal), t.end));
            top = sees ? kFloor : kStart;
        }
        if (piece) {
            st16(a.ws_o + block * 32 * D + x * 4, __builtin_bit_cast(u32x4, sum));
            const int64_t at = block * 32 + row;
            if (d0 == 0) a.ws_ml[2 * at] = top, a.ws_ml[2 * at + 1] = weight;
        } else {
            T* orow = static_cast<T*>(a.out) + row_out(a, t.seq, t.kv, t.first + row) * D + d0;
            float y[4];
#pragma unroll
            for (int e = 0; e < 4; e++) y[e] = over_weight(sum[e], weight, top == kStart);
            if constexpr (sizeof(T) == 2)
                *reinterpret_cast<u32x2*>(orow) = u32x2{pk_f16(y[0], y[1]), pk_f16(y[2], y[3])};
            else
                *reinterpret_cast<f32x4*>(orow) = f32x4{y[0], y[1], y[2], y[3]};
        }
    }
}

// WHOLE: pages of at least 16 keys, so that a wave's load, 8 or 16 rows, lies in one
// page, is 1 KiB or half of that in a row, and has a scalar address (8192 tokens, 32
// heads of 128 over 8: 1210 us, 1240 by rows of the lanes).
template <typename T, int D, int W, bool WHOLE>
__global__ __launch_bounds__(64 * W, (Prompt8<T, D, W>::kPerCu)) void prompts_f8_kernel(PromptArgs a) {
    using F = Prompt8<T, D, W>;
    constexpr int KS = F::KS, DB = F::DB, kPer = F::kPer;
    __shared__ __align__(16) union {
        typename F::Smem tile;
        FewRows<T, D> few;
    } lds;
    auto& sm = lds.tile;
    PromptTile t;
    if (!prompt_tile(a, F::kRows, t)) return;  // workgroup-uniform, before any barrier
    if constexpr (W == kPagedWaves) {
        if (t.rows <= 16) return few_rows<T, D, 1, WHOLE>(a, t, lds.few);
        if ((WHOLE || F::kHalf || D == 64) && t.rows <= 32) return few_rows<T, D, 2, WHOLE>(a, t, lds.few);
    }
    const int tid = threadIdx.x, lane = lane_id(), wave = wave_in_block();
    const int n = lane & 31, hh = lane >> 5;

    // The keys seen grow with the token: the tile's last live row has the most
    const int row = t.first + 32 * wave + n;
    const bool live = t.first + 32 * wave < t.rows;  // wave-uniform
    const auto seen_by = [&](int r) { return keys_seen(t.seq, min(r, t.rows - 1) / a.group, a.causal); };
    const int seen = seen_by(row);
    const int wave_least = seen_by(t.first + 32 * wave);
    const int wave_most = live ? seen_by(t.first + 32 * wave + 31) : 0;
    const int tile_least = seen_by(t.first);
    const int tile0 = t.begin / kBN, ntiles = (t.end + kBN - 1) / kBN;

    // Q^T as the B operand: lane (n, hh) holds dims 16 ks + 8 hh .. + 8. A
    // negative scale is taken as one of -q.
    const float c = fmaxf(fabsf(a.scale) * 1.4426950408889634f, 1.4e-45f);
    u32x4 qa[KS][F::kParts];
    {
        const int r = min(row, t.rows - 1), token = r / a.group;
        const T* qr = static_cast<const T*>(a.q) + (t.seq.q0 + token) * a.q_stride + (t.kv * a.group + (r - token * a.group)) * D + 8 * hh;
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            if constexpr (F::kHalf) {
                u32x4 x = ld16(qr + 16 * ks);
                qa[ks][0] = a.scale < 0.0f ? x ^ 0x80008000u : x;
            } else {
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; e++) x[e] = a.scale < 0.0f ? -qr[16 * ks + e] : qr[16 * ks + e];
                cut3(x, qa[ks]);
            }
        }
        // arrived before the loop, whose prefetches it would wait for otherwise
#pragma unroll
        for (int ks = 0; ks < KS; ks++) asm volatile("" ::"v"(qa[ks][0]));
    }

    f32x16 o[DB];
#pragma unroll
    for (int i = 0; i < DB; i++) o[i] = f32x16{};
    float m = kStart, l = 0.0f;
    int wary = 0;  // tiles to go

    // Staging: load i of the thread is row row0 + kRowStep i of the tile, kLoad
    // codes at `piece`. Pages are looked up a tile ahead of the codes.
    constexpr int kWords = F::kLoad / 4;
    typedef uint32_t codes_t __attribute__((ext_vector_type(kWords)));
    const int row0 = tid / F::kPieces, piece = tid % F::kPieces;
    const int* pages = a.page_table + static_cast<int64_t>(t.s) * a.max_pages;
    int page[kPer];
    codes_t pk[kPer], pv[kPer];
    uint32_t pks[kPer], pvs[kPer];
    uint32_t ok = 0;  // by load: a key of the piece that there is (WHOLE: its page is)
    auto find_pages = [&](int key0) {
#pragma unroll
        for (int i = 0; i < kPer; i++) {
            const int r = WHOLE ? wave * F::kWaveRows : row0;
            page[i] = pages[min(key0 + r + i * F::kRowStep, t.end - 1) >> a.page_shift];
        }
    };
    auto load = [&](int key0) {
        ok = 0;
#pragma unroll
        for (int i = 0; i < kPer; i++) {
            const int key = key0 + (WHOLE ? wave * F::kWaveRows : row0) + i * F::kRowStep;
            const bool there = page[i] >= 0 && page[i] < a.n_pages && (WHOLE || key < t.end);
            const int64_t block = static_cast<int64_t>(there ? page[i] : 0) * a.h_kv + t.kv;
            const int64_t at = ((block << a.page_shift) + (WHOLE || there ? key & ((1 << a.page_shift) - 1) : 0)) * D;
            const uint32_t lane_at = WHOLE ? lane * F::kLoad : piece * F::kLoad;
            const uint8_t *kp = a.k + at, *vp = a.v + at;
            // (without, 8192 tokens, 16 heads of 64, take 361 us for 342; the others lose 1% by it)
            if constexpr (W == 8 && D == 64) kp = scalar_address(kp), vp = scalar_address(vp);
            pk[i] = *reinterpret_cast<const codes_t*>(kp + lane_at);
            pv[i] = *reinterpret_cast<const codes_t*>(vp + lane_at);
            pks[i] = a.k_scale[block], pvs[i] = a.v_scale[block];
            ok |= there ? 1u << i : 0u;
        }
    };
    auto store = [&](int buf, int j) {
        const bool masked = j * kBN + kBN > tile_least;  // some row does not see all of these values
        const bool last = j * kBN + kBN > t.end;
        bool odd = false;
#pragma unroll
        for (int i = 0; i < kPer; i++) {
            const int r = row0 + i * F::kRowStep;
            float vs = scale_value(pvs[i]);
            const float ks = scale_value(pks[i]);
            if (WHOLE ? last || !(ok >> i & 1) : true) {
                const bool there = (ok >> i & 1) && j * kBN + r < t.end;
                if (piece == 0) sm.there[buf][r] = there;
                if (!there) {
                    if (j * kBN + r < t.end) sm.gap[buf] = j;
                    pv[i] = codes_t{}, vs = 1.0f;
                }
            } else if (piece == 0) {
                sm.there[buf][r] = 1;
            }
#pragma unroll
            for (int half = 0; half < F::kLoad / 8; half++) {
                uint16_t* kp = &sm.k[buf][r * F::kKPitch + piece * F::kLoad + 8 * half];
                uint16_t* vp = &sm.v[buf][r * F::kVPitch + piece * F::kLoad + 8 * half];
                st16(kp, values_of<T>(pk[i][2 * half], pk[i][2 * half + 1], ks));
                u32x4 x = values_of<T>(pv[i][2 * half], pv[i][2 * half + 1], vs);
                if (masked) odd |= zero_odd<T>(x);
                st16(vp, x);
            }
        }
        if (odd) sm.odd = 1;
    };
    if (tid == 0) sm.odd = 0, sm.gap[0] = sm.gap[1] = -1;
    __syncthreads();
    if (tile0 < ntiles) {
        find_pages(tile0 * kBN);
        load(tile0 * kBN);
        if (tile0 + 1 < ntiles) find_pages((tile0 + 1) * kBN);
        store(tile0 & 1, tile0);
    }
    __syncthreads();
#pragma unroll 1
    for (int j = tile0; j < ntiles; j++) {
        const int cur = j & 1, key0 = j * kBN;
        if (j + 1 < ntiles) {
            load(key0 + kBN);
            if (j + 2 < ntiles) find_pages(key0 + 2 * kBN);
        }
        if (key0 < wave_most) {
            // S^T: s[i] holds keys 32 i .. + 32 of the tile, register r of lane
            // (n, hh) key 8 (r / 4) + 4 hh + r % 4, row n
            const bool gap = sm.gap[cur] == j;
            f32x16 s[2];
            const f32x16 z = {};
            const uint16_t* ka = sm.k[cur] + n * F::kKPitch + 8 * hh;
#pragma unroll
            for (int ks = 0; ks < KS; ks++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const u32x4 k = ld16(ka + 32 * i * F::kKPitch + 16 * ks);
#pragma unroll
                    for (int p = F::kParts - 1; p >= 0; p--)
                        s[i] = mfma32<T>(k, qa[ks][p], ks || p + 1 < F::kParts ? s[i] : z);
                }
            if (key0 + kBN > wave_least) {
#pragma unroll
                for (int i = 0; i < 2; i++)
#pragma unroll
                    for (int r = 0; r < 16; r++)
                        if (key0 + 32 * i + 8 * (r / 4) + 4 * hh + r % 4 >= seen) s[i][r] = -INFINITY;
            }
            if (gap) {
#pragma unroll
                for (int i = 0; i < 2; i++)
#pragma unroll
                    for (int r = 0; r < 16; r++)
                        if (!sm.there[cur][32 * i + 8 * (r / 4) + 4 * hh + r % 4]) s[i][r] = -INFINITY;
            }
            // O^T += V^T P^T. The transposing read gives lane i of 16 channel i of 4
            // keys: two reads make the 8 keys, in the scores' order.
            const uint16_t* va = sm.v[cur] + (4 * hh + (n & 15) / 4) * F::kVPitch + (n & 16) + 4 * (n & 3);
            auto read_v = [&](int g, int db) {
                const uint16_t* r0 = va + 16 * g * F::kVPitch + 32 * db;
                const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)r0));
                const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(r0 + 8 * F::kVPitch)));
                u32x4 w;
                w[0] = lo[0], w[1] = lo[1], w[2] = hi[0], w[3] = hi[1];
                return w;
            };
            if constexpr (F::kHalf) {
                u32x4 p[2][2];
                // The tile's weights against a reference, rounded to f16, and the
                // sum of the rounded ones over the lane's keys, in f32 like the
                // product's.
                auto weights = [&](float mul, float ref) {
                    const f16x2 one = {static_cast<f16>(1.0f), static_cast<f16>(1.0f)};
                    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int i = 0; i < 2; i++)
#pragma unroll
                        for (int r = 0; r < 16; r += 2) {
                            const uint32_t w = pk_f16(__builtin_amdgcn_exp2f(fmaf(s[i][r], mul, -ref)),
                                                      __builtin_amdgcn_exp2f(fmaf(s[i][r + 1], mul, -ref)));
                            p[i][r / 8][r % 8 / 2] = w;
                            sum[r / 2 % 4] = __builtin_amdgcn_fdot2(u2h2(w), one, sum[r / 2 % 4], false);
                        }
                    return (sum[0] + sum[1]) + (sum[2] + sum[3]);
                };
                // Past the first tile the weights are taken against the reference
                // as it is; only a row of which one does not fit f16, so that its
                // sum is infinite, moves its own. Where the wave's references have
                // moved lately, the scores' maximum says so ahead of the weights.
                bool own = j == tile0 || fabsf(m) > kFar, move = wary > 0 || __any(own);
                if (!move) {
                    const float sum = weights(c, m);
                    own = !(halves_sum(sum) < INFINITY);
                    move = __any(own);
                    if (!move) l += sum;
                }
                if (move) {
                    float mx = s[0][0];
#pragma unroll
                    for (int i = 0; i < 2; i++)
#pragma unroll
                        for (int r = 0; r < 16; r++) mx = fmaxf(mx, s[i][r]);
                    mx = halves_max(mx);
                    // (a row that has seen no key takes its reference from the first)
                    own |= m == kStart || __builtin_amdgcn_exp2f(fmaf(mx, c, -m)) >= kPastF16;
                    // (a maximum of 2^26 and more may round 8 further down, too far)
                    const float top = mx * c, low = top - kWeightBits;
                    const float next = own ? fmaxf(m, top - low > kWeightBits + 2.0f ? top : low) : m;
                    float corr = 1.0f;
                    wary--;
                    if (__any(next != m)) {
                        corr = __builtin_amdgcn_exp2f(m - next);
                        wary = kWary;
#pragma unroll
                        for (int i = 0; i < DB; i++) o[i] *= corr;
                    }
                    // The multiply-add leaves the rounding of s c in the exponent:
                    // where that is not small, the product is rounded first, as
                    // the reference's was.
                    const bool far = __any(fabsf(next) > kFar);
                    if (far) {
#pragma unroll
                        for (int i = 0; i < 2; i++)
#pragma unroll
                            for (int r = 0; r < 16; r++) s[i][r] = as_f32(s[i][r] * c) - next;
                    }
                    l = fmaf(l, corr, weights(far ? 1.0f : c, far ? 0.0f : next));
                    m = next;
                }
#pragma unroll
                for (int g = 0; g < 4; g++)
#pragma unroll
                    for (int db = 0; db < DB; db++) o[db] = mfma32<T>(read_v(g, db), p[g / 2][g % 2], o[db]);
            } else {
                // rounded before the maximum is taken off: that one then weighs 1
                float mx = -INFINITY;
#pragma unroll
                for (int i = 0; i < 2; i++)
#pragma unroll
                    for (int r = 0; r < 16; r++) {
                        s[i][r] = as_f32(s[i][r] * c);
                        mx = fmaxf(mx, s[i][r]);
                    }
                const float next = fmaxf(m, halves_max(mx));
                const float corr = __builtin_amdgcn_exp2f(m - next);
                m = next;
                float sum = 0.0f;
#pragma unroll
                for (int i = 0; i < DB; i++) o[i] *= corr;
#pragma unroll
                for (int g = 0; g < 4; g++) {
                    float x[8];
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        x[e] = __builtin_amdgcn_exp2f(s[g / 2][8 * (g % 2) + e] - m);
                        sum += x[e];
                    }
                    u32x4 p[3];
                    cut3(x, p);
#pragma unroll
                    for (int db = 0; db < DB; db++) {
                        const u32x4 v = read_v(g, db);
#pragma unroll
                        for (int i = 2; i >= 0; i--) o[db] = mfma32<T>(v, p[i], o[db]);
                    }
                }
                l = fmaf(l, corr, sum);
            }
        }
        if (j + 1 < ntiles) store(cur ^ 1, j + 1);
        __syncthreads();
    }
    // Infinities and NaN among the values (odd_values)
    bool all = false;
#pragma unroll
    for (int db = 0; db < DB; db++)
#pragma unroll
        for (int x = 0; x < 16; x++) all |= !(fabsf(o[db][x]) < INFINITY);
    all = __any(all) && any_infinite<T>(a, pages, t.kv, t.begin, t.end);
    if (row >= t.rows) return;
    if (__builtin_expect(tile0 < ntiles && (all || sm.odd), 0)) {
        const auto each = [&](auto f) {
#pragma unroll
            for (int db = 0; db < DB; db++)
#pragma unroll
                for (int x = 0; x < 16; x++) o[db][x] = f(o[db][x]);
        };
        if (all) each(put_aside);
        for (int key = all ? t.begin : max(tile_least / kBN * kBN, t.begin); key < min(seen, t.end); key++) {
            const int p = pages[key >> a.page_shift];
            if (p < 0 || p >= a.n_pages) continue;
            const int64_t block = static_cast<int64_t>(p) * a.h_kv + t.kv;
            const uint8_t* r = a.v + ((block << a.page_shift) + (key & ((1 << a.page_shift) - 1))) * D + 4 * hh;
            const float scale = scale_value(a.v_scale[block]);
#pragma unroll
            for (int db = 0; db < DB; db++)
#pragma unroll
                for (int x = 0; x < 16; x++) o[db][x] = with_odd(o[db][x], value_of<T>(r[32 * db + 8 * (x / 4) + x % 4], scale));
        }
        if (all) each(taken_back);
    }
    const float lsum = halves_sum(l);
    if (lsum == 0.0f) m = any_keys(a, pages, t.begin, min(seen, t.end)) ? kFloor : kStart;
    if (t.count > 1) {
        const int64_t block = partial_block(a, t.item, t.kv, wave);
        float* p = a.ws_o + block * 32 * D + lane * 4;
#pragma unroll
        for (int db = 0; db < DB; db++)
#pragma unroll
            for (int r4 = 0; r4 < 4; r4++) {
                u32x4 w;
#pragma unroll
                for (int e = 0; e < 4; e++) w[e] = f2u(o[db][4 * r4 + e]);
                st16_nt(p + (4 * db + r4) * 256, w);
            }
        const int64_t at = block * 32 + n;
        if (hh == 0) a.ws_ml[2 * at] = m, a.ws_ml[2 * at + 1] = lsum;
        return;
    }
    const float inv = 1.0f / lsum, empty = over_weight(0.0f, 0.0f, m == kStart);
    T* orow = static_cast<T*>(a.out) + row_out(a, t.seq, t.kv, row) * D + 4 * hh;
#pragma unroll
    for (int db = 0; db < DB; db++)
#pragma unroll
        for (int r4 = 0; r4 < 4; r4++) {
            float x[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if constexpr (F::kHalf)
                    x[e] = lsum == 0.0f ? empty : o[db][4 * r4 + e] * inv;
                else
                    x[e] = lsum == 0.0f ? empty : o[db][4 * r4 + e] / lsum;
            }
            if constexpr (F::kHalf)
                *reinterpret_cast<u32x2*>(orow + 32 * db + 8 * r4) = u32x2{pk_f16(x[0], x[1]), pk_f16(x[2], x[3])};
            else
                *reinterpret_cast<f32x4*>(orow + 32 * db + 8 * r4) = f32x4{x[0], x[1], x[2], x[3]};
        }
}

// The pieces of one tile's rows joined, four channels of a row to a thread, as the
// workspace has them; `share` workgroups to a tile. SPREAD: few tiles, a wave takes
// every fourth piece of 64 threads' channels.
struct Joined {
    f32x4 sum;
    float top, weight;
    template <typename K>
    __device__ __forceinline__ void add(f32x4 v, float m, float l, K keep) {
        const float next = fmaxf(top, m);
        const float old = __builtin_amdgcn_exp2f(top - next), f = __builtin_amdgcn_exp2f(m - next);
        sum = times(sum, old, keep) + times(v, f, keep);
        weight = fmaf(weight, old, l * f);
        top = next;
    }
};
template <typename T, int D, bool SPREAD>
__global__ __launch_bounds__(256) void prompts_join_kernel(PromptArgs a, int share) {
    constexpr int kParts = D / 32 * (SPREAD ? 4 : 1);  // of a block of 32 rows
    __shared__ Joined others[3][SPREAD ? 64 : 1];
    const int tile_head = static_cast<int>(blockIdx.x) / share;
    const int tile = tile_head / a.h_kv, kv = tile_head - tile * a.h_kv;
    const int4 c = a.cut[tile];
    const int item = c.x, count = c.y, rows = c.w;
    if (tile >= a.cut[a.tiles].x || count <= 1) return;  // written by its only piece
    // (what offsets that do not ascend leave of a cut)
    if (item < 0 || item + count > a.items || rows > 32 * a.blocks || c.z < 0 || c.z + rows > a.n * a.group) return;
    const int lane = threadIdx.x % 64, wave = wave_in_block();
    const int64_t step = static_cast<int64_t>(a.h_kv) * a.blocks;
    for (int x = static_cast<int>(blockIdx.x) - tile_head * share; x < (rows + 31) / 32 * kParts; x += share) {
        const int block = x / kParts, part = x - block * kParts, row = 32 * block + lane % 32;
        const int at = SPREAD ? part : 4 * part + wave;  // 32 rows of 8 channels
        const int64_t from = partial_block(a, item, kv, block);
        const float* o = a.ws_o + from * 32 * D + (at * 64 + lane) * 4;
        const float* ml = a.ws_ml + (from * 32 + lane % 32) * 2;
        constexpr int kAhead = 4, kStep = SPREAD ? 4 : 1;  // pieces whose loads are under way at once
        Joined j;
        // (streamed past the caches where there is much of it: 311 us for 317 of the
        // prompts; few tokens' 28 for 27)
        const auto add = [&](auto stream, auto keep) {
            j = {f32x4{}, kStart, 0.0f};
            for (int i0 = SPREAD ? wave : 0; i0 < count; i0 += kAhead * kStep) {
                f32x2 stat[kAhead];
                u32x4 v[kAhead];
#pragma unroll
                for (int i = 0; i < kAhead; i++) {
                    if (i0 + i * kStep >= count) break;  // wave-uniform
                    const int64_t piece = (i0 + i * kStep) * step;
                    stat[i] = *reinterpret_cast<const f32x2*>(ml + piece * 64);
                    v[i] = decltype(stream)::value ? ld16_nt(o + piece * 32 * D) : ld16(o + piece * 32 * D);
                }
#pragma unroll
                for (int i = 0; i < kAhead; i++)
                    if (i0 + i * kStep < count) j.add(__builtin_bit_cast(f32x4, v[i]), stat[i].x, stat[i].y, keep);
            }
        };
        j.sum = joined([&](auto keep) {
            if (rows > 32 && !decltype(keep)::value)
                add(std::true_type{}, keep);
            else
                add(std::false_type{}, keep);
            return j.sum;
        });
        if constexpr (SPREAD) {
            __syncthreads();  // the last round's have been read
            if (wave > 0) others[wave - 1][lane] = j;
            __syncthreads();
            if (wave > 0) continue;
            const Joined own = j;
            j.sum = joined([&](auto keep) {
                j = own;
#pragma unroll
                for (int w = 0; w < 3; w++) j.add(others[w][lane].sum, others[w][lane].top, others[w][lane].weight, keep);
                return j.sum;
            });
        }
        if (row >= rows) continue;
        const int all = c.z + row, token = all / a.group;
        const int64_t to = static_cast<int64_t>(token) * a.h + kv * a.group + (all - token * a.group);
        T* orow = static_cast<T*>(a.out) + to * D + 8 * at + 4 * (lane / 32);
        float y[4];
#pragma unroll
        for (int e = 0; e < 4; e++) y[e] = over_weight(j.sum[e], j.weight, j.top == kStart);
        if constexpr (sizeof(T) == 2)
            *reinterpret_cast<u32x2*>(orow) = u32x2{pk_f16(y[0], y[1]), pk_f16(y[2], y[3])};
        else
            *reinterpret_cast<f32x4*>(orow) = f32x4{y[0], y[1], y[2], y[3]};
    }
}

// How a call is cut into tiles, and whether its keys are. Eight waves (256 rows)
// stage and turn a key once for twice the rows, which pays in f16 where the tiles are
// two to a CU and sequences long (us with 128 and 256 rows: 8192 tokens, 32 heads of
// 128 over 8, 1209, 1180, 16 heads of 64 402, 343; eight of 1374, 16 heads of 64, 107,
// 125; f32, 4096 tokens of 16 heads of 64, 206, 216).
struct PromptPlan {
    int64_t tiles;          // of a key head, as many as sequences of these rows can have
    int64_t places, items;  // of a key head: on the chip at once (0: whole keys), and in the call at most
    bool one_round;         // fewer tiles than places
    int64_t blocks;  // of 32 rows of a tile
    int rows;
    PromptPlan(hs_dtype dt, int64_t n, int64_t b, int64_t h, int64_t h_kv, int d, int64_t keys, bool whole) {
        const int64_t group = h / h_kv;
        rows = whole && dt == HS_F16 && n * group / 256 * h_kv >= 2 * num_cus() && n >= 512 * b ? 256 : 128;
        const int64_t slots = num_cus() * per_cu(dt, d, rows);
        tiles = n * group / rows + (b < n ? b : n);
        items = tiles, blocks = 0;
        places = slots / h_kv;
        one_round = tiles < places;
        // (a workspace for every item that there can be: fewer than seven times the places
        // of all key heads, 243 MB on 256 CUs. Where key heads fill the chip by themselves,
        // it would be that of each of them, and nothing is gained)
        if (keys <= kLeastUnits * kBN || places < 2 || tiles >= 4 * places) places = 0;
        if (!places) return;
        items = 3 * places + tiles;
        blocks = ceil_div(std::min<int64_t>(n * group, rows), 32);
    }
    static int per_cu(hs_dtype dt, int d, int rows) {
        const bool half = dt == HS_F16;
        if (rows == 256) return d == 64 ? Prompt8<f16, 64, 8>::kGroups : Prompt8<f16, 128, 8>::kGroups;
        return d == 64 ? (half ? Prompt8<f16, 64, 4>::kGroups : Prompt8<float, 64, 4>::kGroups)
                       : (half ? Prompt8<f16, 128, 4>::kGroups : Prompt8<float, 128, 4>::kGroups);
    }
    int64_t workspace(int64_t h_kv, int d) const { return places ? (tiles + 1) * 16 + items * h_kv * blocks * 32 * (d + 2) * 4 : 0; }
};

}  // namespace
}  // namespace hs

extern "C" int64_t hs_attention_prompts_f8_workspace(hs_dtype dt, int64_t n, int32_t b, int32_t h, int32_t h_kv,
                                                     int32_t d, int32_t page, int32_t max_pages, int32_t causal) {
    using namespace hs;
    if (n <= 0 || b <= 0 || h <= 0 || causal < 0 || n >= (int64_t{1} << 30) / h || exact_log2(page) < 0 || max_pages < 0) return 0;
    if (static_cast<int64_t>(max_pages) * page >= (int64_t{1} << 30)) return 0;
    if (check_heads("attention_prompts_f8_workspace", dt, h, h_kv, d)) return 0;
    return PromptPlan(dt, n, b, h, h_kv, d, static_cast<int64_t>(max_pages) * page, page >= 16).workspace(h_kv, d);
}

extern "C" hs_status hs_attention_prompts_f8(hs_stream_t stream, hs_dtype dt, const void* q, int64_t q_stride,
                                             const void* k_cache, const void* v_cache, const void* k_scale,
                                             const void* v_scale, const void* page_table, const void* lens,
                                             const void* offsets, void* out, void* workspace, int64_t workspace_bytes,
                                             int64_t n, int32_t b, int32_t h, int32_t h_kv, int32_t d, int32_t page,
                                             int32_t n_pages, int32_t max_pages, int32_t causal, float scale) {
    using namespace hs;
    const char* op = "attention_prompts_f8";
    if (hs_status rc = check_heads(op, dt, h, h_kv, d)) return rc;
    if (n < 0 || b < 0) return fail(HS_EINVAL, "%s: negative count", op);
    if (causal < 0) return fail(HS_EINVAL, "%s: causal %d", op, causal);
    if (n == 0 || b == 0 || h == 0) return HS_OK;
    if (n >= (int64_t{1} << 30) / h) return fail(HS_EINVAL, "%s: n * Hq must be below 2^30", op);
    if (!offsets) return fail(HS_EINVAL, "%s: null offsets", op);
    const int64_t need = hs_attention_prompts_f8_workspace(dt, n, b, h, h_kv, d, page, max_pages, causal);
    if (hs_status rc = check_attend_f8(op, dt, {q, q_stride, k_cache, v_cache, k_scale, v_scale, page_table, lens, out, workspace,
                                                workspace_bytes, n, h, h_kv, d, page, n_pages, max_pages, scale}, need))
        return rc;
    PromptArgs a;
    a.q = q, a.q_stride = q_stride, a.out = out;
    a.k = static_cast<const uint8_t*>(k_cache), a.v = static_cast<const uint8_t*>(v_cache);
    a.k_scale = static_cast<const uint8_t*>(k_scale), a.v_scale = static_cast<const uint8_t*>(v_scale);
    a.page_table = static_cast<const int*>(page_table), a.lens = static_cast<const int*>(lens);
    a.offsets = static_cast<const int*>(offsets);
    a.n = static_cast<int>(n), a.b = b, a.h = h, a.h_kv = h_kv, a.group = h / h_kv, a.page_shift = exact_log2(page);
    a.n_pages = n_pages, a.max_pages = n_pages > 0 ? max_pages : 0;  // no page to read: no sequence has keys
    a.causal = causal, a.scale = scale;
    const PromptPlan plan(dt, n, b, h, h_kv, d, static_cast<int64_t>(max_pages) * page, page >= 16);
    const int threads = 2 * plan.rows;
    const int64_t groups = plan.items * h_kv;
    if (groups >= (int64_t{1} << 31) / threads) return fail(HS_EINVAL, "%s: too many sequences and heads", op);
    a.cut = static_cast<int4*>(workspace), a.tiles = static_cast<int>(plan.tiles);
    a.ws_o = static_cast<float*>(workspace) + (plan.tiles + 1) * 4;
    a.ws_ml = a.ws_o + (plan.places ? plan.items * h_kv * plan.blocks * 32 * d : 0);
    a.places = static_cast<int>(plan.places), a.one_round = plan.one_round;
    a.items = static_cast<int>(plan.items), a.blocks = static_cast<int>(plan.blocks);
    hipStream_t st = static_cast<hipStream_t>(stream);
    const auto go = [&](auto kernel, auto join, auto spread) {
        kernel<<<dim3(static_cast<uint32_t>(groups)), dim3(threads), 0, st>>>(a);
        if (hs_status rc = check_launch(op)) return rc;
        if (!plan.places) return HS_OK;
        const int64_t heads = plan.tiles * h_kv, whole = plan.blocks * (d / 32);
        // (a tile's blocks to several workgroups: the join of five prompts 14.6 us for 15.9)
        const bool few = heads * whole < 4 * num_cus();
        const int64_t share = few ? 4 * whole : std::max<int64_t>(std::min(whole, 16 * num_cus() / heads), 1);
        (few ? spread : join)<<<dim3(static_cast<uint32_t>(heads * share)), dim3(256), 0, st>>>(a, static_cast<int>(share));
        return check_launch(op);
    };
    const bool whole = page >= 16, wide = plan.rows == 256;
    const auto pick = [&](auto zero) {
        using T = decltype(zero);
        if (d == 64)
            return go(wide ? prompts_f8_kernel<f16, 64, 8, true> : whole ? prompts_f8_kernel<T, 64, 4, true> : prompts_f8_kernel<T, 64, 4, false>,
                      prompts_join_kernel<T, 64, false>, prompts_join_kernel<T, 64, true>);
        return go(wide ? prompts_f8_kernel<f16, 128, 8, true> : whole ? prompts_f8_kernel<T, 128, 4, true> : prompts_f8_kernel<T, 128, 4, false>,
                  prompts_join_kernel<T, 128, false>, prompts_join_kernel<T, 128, true>);
    };
    return dt == HS_F16 ? pick(f16{}) : pick(float{});
}
