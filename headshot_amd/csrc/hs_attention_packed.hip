// Attention of packed sequences for gfx950: whole prompts of different lengths
// in one call, causal by token or by group of tokens, query heads sharing key
// heads: O_i = sum_j w_ij v_j / sum_j w_ij, w_ij = exp(scale q_i k_j - m_i) over
// the keys j that query i sees, in one pass over the keys with a running m_i.
//
// A workgroup takes a tile of one sequence's queries and one head, and finds
// both on the device: lengths are device data, and the launch has a workgroup
// for every tile that there can be. Keys past the tile's last query's are not
// read, a wave whose queries see none of a tile sits it out, and only tiles that
// some query sees in part are masked. Few queries over many keys are split over
// the keys, too (PackedPlan).
//
// Bounds: matrix and vector issue, and the ends of calls of one to two rounds of
// workgroups. f16: by frames, 10992 tokens of 16 heads of 64, 210-218 us (745-773
// TFLOP/s; CUs busy 84% of it, their matrix cores 44% of that); prompts of 12926
// tokens, 32 heads of 128 over 8, 524-560 us (865-925 TFLOP/s; 92%, 44%); a plain
// product of 8192^3 reaches 1246. f32, head dim 64: 4122 tokens by frames 215-229
// us (135-144 TFLOP/s; some 360 us on the f32 matrix instructions, whose plain
// product reaches 154). Short calls are a chain of loads, find a tile, read it,
// multiply, of 6 us and more: eight f32 sequences of up to 200 tokens, 16 heads
// of 128, 20 us.
#include <cmath>

#include "hs_packed.hpp"

namespace hs {
namespace {

typedef f16 h8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

constexpr int kXcds = 8;
constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kBM = 32 * kWaves;  // queries per workgroup
constexpr int kBN = 64;           // keys per tile

__device__ __forceinline__ h8 as_h8(u32x4 v) { return __builtin_bit_cast(h8, v); }
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

struct PackedArgs {
    const void *q, *k, *v;
    void* out;
    int64_t q_stride, k_stride, v_stride;
    const int *q_off, *k_off;  // k_off null: the queries'
    int n_q, n_k, b, h, h_kv, causal;
    int share;  // log2 of the query heads that a workgroup takes
    float scale;
    // split keys only
    float *ws_o, *ws_ml;  // per (item, head, row of the tile): D sums; maximum and weight sum
    float per_piece;      // 1 / pieces wanted of a head
    int items, pitch;     // items of a head that the launch has, rows of each
};

// What a workgroup works on: a tile of one sequence's queries, one head.
struct PackedTile {
    int q0, nq;       // first query of the sequence's rows, its queries
    int k0, nk;       // the keys likewise
    int first, head;  // first query of the tile, within the sequence, and head
    // split keys: those of this piece, of how many the tile has, and its place
    int begin, end, count, item;
};

// Keys that query i of a sequence sees.
__device__ __forceinline__ int keys_seen(int i, int nq, int nk, int causal) {
    if (causal == 0) return nk;
    const int at = i + nk - nq;
    if (at < 0) return 0;
    if (causal == 1) return at + 1;
    const int64_t end = (static_cast<int64_t>(at / causal) + 1) * causal;
    return end < nk ? static_cast<int>(end) : nk;
}

// Split keys: where the tiles of a call are few, its keys are cut into pieces of
// `chunk` units of 64, and an item is a piece of a tile; a second launch joins
// them. chunk makes them as many as wanted and, lengths being device data, every
// workgroup computes it from all of them (64 a step). A piece has kLeastUnits
// units at least: it costs some 5 us before its first product and a unit 0.7 us.
// (16 queries over 131072 keys, 32 heads of 128 over 8, f16: 118 us, 4.6 TB/s;
// whole, 2.8 ms. 1374 tokens, 16 heads of 64, over 30000 keys: 264 us, 440.)
constexpr int kLeastUnits = 4;

struct PackedCut {
    RowRange q, k;
    int tiles;  // of the sequence
    int local;  // the tile among them
    int piece, pieces, chunk;
    int item;   // piece 0's
};
__device__ __forceinline__ int units_of(const RowRange& k) { return (k.end - k.begin + kBN - 1) / kBN; }

// The tile numbered `index` of a call (BY_TILE) or the item. chunk is at least
// half the total of tiles times units over the pieces wanted (the f32 sum's error
// is covered by per_piece), so a sequence's items pass neither twice those and
// its tiles nor 31 bits whatever the offsets hold.
template <bool BY_TILE>
__device__ __forceinline__ bool find_cut(const PackedArgs& a, int bm, int index, PackedCut& t) {
    const int lane = lane_id();
    const auto ranges = [&](int s, RowRange& q, RowRange& k) {
        q = row_range(a.q_off, s, a.n_q);
        k = a.k_off ? row_range(a.k_off, s, a.n_k) : q;
    };
    float total = 0.0f;
    for (int base = 0; base < a.b; base += 64) {
        RowRange q = {}, k = {};
        if (base + lane < a.b) ranges(base + lane, q, k);
        const int masked = a.causal ? min(q.end - q.begin, k.end - k.begin) : 0;  // up to half of the keys, on average
        total += static_cast<float>((q.end - q.begin + bm - 1) / bm) *
                 (static_cast<float>(units_of(k)) - static_cast<float>(masked) * (0.5f / kBN));
    }
    t.chunk = static_cast<int>(fminf(fmaxf(ceilf(wave_sum(total) * a.per_piece), static_cast<float>(kLeastUnits)), 16777216.0f));
    int tiles_before = 0, items_before = 0;
    for (int base = 0; base < a.b; base += 64) {
        RowRange q = {}, k = {};
        if (base + lane < a.b) ranges(base + lane, q, k);
        const int tiles = (q.end - q.begin + bm - 1) / bm;
        const int pieces = max((units_of(k) + t.chunk - 1) / t.chunk, 1);
        const int tile_sum = wave_prefix_sum(tiles), item_sum = wave_prefix_sum(tiles * pieces);
        const uint64_t hit = __ballot((BY_TILE ? tiles_before + tile_sum : items_before + item_sum) > index);
        if (hit) {
            const int l = __builtin_ctzll(hit);
            t.q = {lane_value(q.begin, l), lane_value(q.end, l)};
            t.k = {lane_value(k.begin, l), lane_value(k.end, l)};
            t.tiles = lane_value(tiles, l), t.pieces = lane_value(pieces, l);
            const int before = items_before + lane_value(item_sum, l) - t.tiles * t.pieces;
            t.local = BY_TILE ? index - tiles_before - (lane_value(tile_sum, l) - t.tiles) : (index - before) / t.pieces;
            t.item = before + t.local * t.pieces;
            // in another order from tile to tile: the last pieces, which an early
            // tile's queries do not see, are not one XCD's
            t.piece = BY_TILE ? 0 : (index - t.item + t.local) % t.pieces;
            return t.item + t.pieces <= a.items;  // more than that: offsets that do not ascend
        }
        tiles_before += lane_value(tile_sum, 63), items_before += lane_value(item_sum, 63);
    }
    return false;
}
// Pieces of a tile whose last query sees `most` keys: the ones that see any.
__device__ __forceinline__ int pieces_seen(int most, int chunk) {
    return max((most + kBN * chunk - 1) / (kBN * chunk), 1);
}

// Workgroup b's tile. A sequence's last queries see the most keys and go first,
// tile by tile over the heads, so that the first workgroups, two and more to a
// CU, are not all a head's longest. Workgroup b runs on XCD b % 8: where the
// heads divide by it, an XCD takes h / 8 heads in a row, so that the heads of a
// key head, and a head's tiles, read their keys through one L2.
template <bool SPLIT>
__device__ __forceinline__ bool packed_tile(const PackedArgs& a, int bm, PackedTile& t) {
    const int b = blockIdx.x;
    const int all = a.h >> a.share;
    int tile;
    if (all % kXcds == 0) {
        const int slot = b / kXcds, heads = all / kXcds;
        tile = slot / heads;
        t.head = b % kXcds * heads + slot % heads;
    } else {
        tile = b / all;
        t.head = b % all;
    }
    t.head <<= a.share;
    if constexpr (SPLIT) {
        PackedCut c;
        if (!find_cut<false>(a, bm, tile, c)) return false;
        t.q0 = c.q.begin, t.nq = c.q.end - c.q.begin, t.k0 = c.k.begin, t.nk = c.k.end - c.k.begin;
        t.first = (c.tiles - 1 - c.local) * bm;
        const int most = keys_seen(min(t.first + bm, t.nq) - 1, t.nq, t.nk, a.causal);
        t.count = pieces_seen(most, c.chunk), t.item = c.item + c.piece;
        if (c.piece >= t.count) return false;
        t.begin = c.piece * c.chunk * kBN;
        t.end = c.piece + 1 < t.count ? t.begin + c.chunk * kBN : most;
        return true;
    }
    int s, local;
    RowRange q;
    if (!find_tile(a.q_off, a.b, a.n_q, bm, tile, s, q, local)) return false;
    const RowRange k = a.k_off ? row_range(a.k_off, s, a.n_k) : q;
    t.q0 = q.begin, t.nq = q.end - q.begin, t.k0 = k.begin, t.nk = k.end - k.begin;
    t.first = ((t.nq + bm - 1) / bm - 1 - local) * bm;
    t.begin = 0, t.end = keys_seen(min(t.first + bm, t.nq) - 1, t.nq, t.nk, a.causal), t.count = 1;
    return true;
}

// Row `row` of the tile's place in the workspace.
__device__ __forceinline__ int64_t partial_row(const PackedArgs& a, const PackedTile& t, int row) {
    return (static_cast<int64_t>(t.item) * a.h + t.head) * a.pitch + row;
}
// A piece's sums of a query, in the layout of the 32 x 32 products.
template <int DB>
__device__ __forceinline__ void put_partial(const PackedArgs& a, const PackedTile& t, int row, int hh, const f32x16 (&o)[DB],
                                            float m, float l, float factor) {
    const int64_t at = partial_row(a, t, row);
    float* p = a.ws_o + at * 32 * DB + 4 * hh;
#pragma unroll
    for (int db = 0; db < DB; db++)
#pragma unroll
        for (int r4 = 0; r4 < 4; r4++) {
            u32x4 w;
#pragma unroll
            for (int e = 0; e < 4; e++) w[e] = f2u(o[db][4 * r4 + e] * factor);
            st16(p + 32 * db + 8 * r4, w);
        }
    if (hh == 0) a.ws_ml[2 * at] = m, a.ws_ml[2 * at + 1] = l * factor;
}

// An infinity or NaN among a tile's values, where some queries see them and
// others do not, must not meet the others' weights, which are 0: such values go
// into LDS as zeros, and a workgroup that has met any adds them here to the sums
// of the queries that do see them. A weight is positive, so what they make of a
// sum is what they sum to. First: the first key that some query of the workgroup
// does not see, seen: the end of the query's own; o as the kernels hold it, channel 32 db + 8 (r / 4) + 4 hh + r %
// 4 in register r.
template <typename T, int DB>
__device__ __forceinline__ void add_odd(f32x16 (&o)[DB], const PackedArgs& a, const PackedTile& t, int kv, int tile,
                                        int first, int seen, int hh) {
    for (int key = max(first / tile * tile, t.begin); key < min(seen, t.end); key++) {
        const T* row = static_cast<const T*>(a.v) + (t.k0 + key) * a.v_stride + kv * 32 * DB + 4 * hh;
#pragma unroll
        for (int db = 0; db < DB; db++)
#pragma unroll
            for (int r = 0; r < 16; r++) {
                const float x = static_cast<float>(row[32 * db + 8 * (r / 4) + r % 4]);
                if ((f2u(x) & 0x7F800000u) == 0x7F800000u) o[db][r] += x;
            }
    }
}

// ---------------------------------------------------------------------------
// f16
//
// Flash attention on v_mfma_f32_32x32x16_f16, scores transposed: a wave takes
// 32 queries, and S^T = K Q^T puts one query in a lane's column (lanes n and n
// + 32 share its keys), so its softmax statistics are the lane's own. Keys go
// through LDS 64 at a time, double-buffered, the next tile's rows in registers
// while the current one computes; V^T comes through the transposing LDS read
// and takes P^T from the registers that the scores were in.
//
// LDS rows are padded so that 16 rows' reads of K at one column, and the
// transposing read's 4 rows of 64 bytes, touch every bank once; every read is
// then one register and a constant. (Unpadded rows with permuted pieces let a
// third more waves of four-wave workgroups in, but the addresses cost more
// registers than there are.)
//
// Eight waves share the keys and their staging (two workgroups per CU at head
// dim 64, one at 128), four where the grid is small. SUB tiles lie between two
// barriers: with one workgroup on a CU the waves drift apart in between, one's
// softmax beside another's products (prompts of 32 heads of 128: 528 us with two
// tiles, 551 with one; at head dim 64 two tiles leave one workgroup: 224 for
// 213).
template <int D, int W, int SUB>
struct FlashF16 {
    static constexpr int kKeys = SUB * kBN;       // keys between barriers
    static constexpr int kThr = 64 * W;
    static constexpr int kQueries = 32 * W;
    static constexpr int KS = D / 16;             // 16-dim slices of a score
    static constexpr int DB = D / 32;             // 32-channel blocks of an output
    static constexpr int kPieces = D / 8;         // 16-byte pieces of a row
    static constexpr int kPer = kKeys * kPieces / kThr;
    static constexpr int kRowStep = kThr / kPieces;          // rows per load of the workgroup
    static constexpr int kKPitch = D + 8, kVPitch = D + 32;  // halves
    struct Smem {
        f16 k[2][kKeys * kKPitch];
        f16 v[2][kKeys * kVPitch];
        int odd;  // a tile whose values not every query sees holds an infinity or NaN
    };
};

// A query's reference is set this far (log2) below its largest score, so that its
// largest weight is 2^12: weights keep f16's 11 bits down to 2^-26 of the largest,
// and below, where f16 is subnormal, are at most 2^-37 of it off. (With a largest
// weight of 1 a key 17 nats above the others, of value 0, left them up to 45%
// off.) A weight may then grow 16 times past the largest before it passes f16 and
// the reference moves, which scores that spread wide do more often (16 heads of
// 64, 10992 tokens by frames, scores of standard deviation 1 and 3 nats: 213 and
// 227 us, 207 and 209 with 1; with 2^13 2% more at 1, with 2^14 12%).
constexpr float kWeightBits = 12.0f;
constexpr float kPastF16 = 65520.0f;  // the least that f16 rounds to infinity
// Tiles for which a wave looks for the scores' maximum ahead of the weights once
// references have moved: weights that do not fit are computed twice, which is
// some 190 instructions against 20 (3 nats: 227 us, 249 without; 4 and 16 tiles
// within 1%). A query's result is the same either way.
constexpr int kWary = 8;
// A reference before any score. It is finite, so that a masked score
// weighs exp2(-inf - kFloor) = 0 against it.
constexpr float kFloor = -3.0e38f;
// A maximum (log2) beyond which its rounding, 2^-24 of it, shows in a weight.
constexpr float kFar = 65536.0f;

template <int D, int W, int SUB, bool SPLIT>
__global__ __launch_bounds__(64 * W, D == 64 ? (W == 8 ? 4 : 3) : 2) void packed_f16_kernel(PackedArgs a) {
    using F = FlashF16<D, W, SUB>;
    constexpr int KS = F::KS, DB = F::DB, kPer = F::kPer;
    __shared__ __align__(16) typename F::Smem sm;
    PackedTile t;
    const int share = W == 4 ? a.share : 0, rows = F::kQueries >> share;
    if (!packed_tile<SPLIT>(a, rows, t)) return;  // workgroup-uniform, before any barrier
    const int tid = threadIdx.x, lane = lane_id(), wave = wave_in_block();
    const int n = lane & 31, hh = lane >> 5;
    const int kv = t.head / (a.h / a.h_kv);
    const int block = 32 * (wave & ((W >> share) - 1));  // the wave's queries
    t.head += wave * 32 / rows;

    // The keys seen grow with the query: the tile's last live query has the most
    const int qi = t.first + block + n;
    const bool live = t.first + block < t.nq;  // wave-uniform
    const int seen = keys_seen(min(qi, t.nq - 1), t.nq, t.nk, a.causal);
    const int wave_least = keys_seen(min(t.first + block, t.nq - 1), t.nq, t.nk, a.causal);
    const int wave_most = live ? keys_seen(min(t.first + block + 31, t.nq - 1), t.nq, t.nk, a.causal) : 0;
    const int tile_least = keys_seen(t.first, t.nq, t.nk, a.causal);
    const int tile0 = SPLIT ? t.begin / F::kKeys : 0, ntiles = (t.end + F::kKeys - 1) / F::kKeys;

    // Q^T as the B operand: lane (n, hh) holds dims 16 ks + 8 hh .. + 8. A
    // negative scale is taken as one of -q.
    const float c = fmaxf(fabsf(a.scale) * 1.4426950408889634f, 1.4e-45f);
    const uint32_t flip = a.scale < 0.0f ? 0x80008000u : 0u;
    h8 qa[KS];
    {
        const f16* qr = static_cast<const f16*>(a.q) + (t.q0 + min(qi, t.nq - 1)) * a.q_stride + t.head * D + 8 * hh;
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            u32x4 x = ld16(qr + 16 * ks);
            x ^= flip;
            qa[ks] = as_h8(x);
        }
        // arrived before the loop, whose prefetches it would wait for otherwise
#pragma unroll
        for (int ks = 0; ks < KS; ks++) asm volatile("" ::"v"(qa[ks]));
    }

    f32x16 o[DB];
#pragma unroll
    for (int i = 0; i < DB; i++) o[i] = f32x16{};
    float m = kFloor, l = 0.0f;
    int wary = 0;  // tiles to go

    // Staging: load i of the thread is row row0 + kRowStep i, piece `piece`. The
    // tile's address is the scalar part of the load's, the thread's the other.
    const int row0 = tid / F::kPieces, piece = tid % F::kPieces;
    const uint32_t k_off = (row0 * static_cast<uint32_t>(a.k_stride) + piece * 8) * 2;
    const uint32_t v_off = (row0 * static_cast<uint32_t>(a.v_stride) + piece * 8) * 2;
    const char* kb = reinterpret_cast<const char*>(static_cast<const f16*>(a.k) + t.k0 * a.k_stride + kv * D);
    const char* vb = reinterpret_cast<const char*>(static_cast<const f16*>(a.v) + t.k0 * a.v_stride + kv * D);
    u32x4 pk[kPer], pv[kPer];
    auto load = [&](int key0) {
        const char* kt = kb + static_cast<int64_t>(key0) * a.k_stride * 2;
        const char* vt = vb + static_cast<int64_t>(key0) * a.v_stride * 2;
        if (key0 + F::kKeys <= t.nk) {
#pragma unroll
            for (int i = 0; i < kPer; i++) {
                pk[i] = ld16(kt + static_cast<int64_t>(i * F::kRowStep) * a.k_stride * 2 + k_off);
                pv[i] = ld16(vt + static_cast<int64_t>(i * F::kRowStep) * a.v_stride * 2 + v_off);
            }
        } else {
#pragma unroll
            for (int i = 0; i < kPer; i++) {
                const uint32_t row = min(row0 + i * F::kRowStep, t.nk - 1 - key0);  // past the end: masked
                pk[i] = ld16(kt + (row * static_cast<uint32_t>(a.k_stride) + piece * 8) * 2);
                pv[i] = ld16(vt + (row * static_cast<uint32_t>(a.v_stride) + piece * 8) * 2);
            }
        }
    };
    const int k_at = row0 * F::kKPitch + piece * 8, v_at = row0 * F::kVPitch + piece * 8;
    auto store = [&](int buf, int key0) {
        if (key0 + F::kKeys > tile_least) {  // some query does not see all of these values
            bool odd = false;
#pragma unroll
            for (int i = 0; i < kPer; i++)
#pragma unroll
                for (int w = 0; w < 4; w++) {
                    const uint32_t x = pv[i][w];
                    const uint32_t keep = ((x & 0x7C00u) == 0x7C00u ? 0u : 0xFFFFu) | ((x & 0x7C000000u) == 0x7C000000u ? 0u : 0xFFFF0000u);
                    odd |= keep != 0xFFFFFFFFu;
                    pv[i][w] = x & keep;
                }
            if (odd) sm.odd = 1;
        }
#pragma unroll
        for (int i = 0; i < kPer; i++) {
            st16(&sm.k[buf][k_at + i * F::kRowStep * F::kKPitch], pk[i]);
            st16(&sm.v[buf][v_at + i * F::kRowStep * F::kVPitch], pv[i]);
        }
    };
    if (tid == 0) sm.odd = 0;
    __syncthreads();
    if (tile0 < ntiles) {
        load(tile0 * F::kKeys);
        store(tile0 & 1, tile0 * F::kKeys);
    }
    __syncthreads();
    for (int j = tile0; j < ntiles; j++) {
        const int cur = j & 1;
        if (j + 1 < ntiles) load((j + 1) * F::kKeys);
#pragma unroll
        for (int sub = 0; sub < SUB; sub++) {
            const int key0 = j * F::kKeys + sub * kBN;
            if (key0 >= wave_most) continue;
            // S^T: s[kb] holds keys 32 kb .. + 32 of the tile, register r of
            // lane (n, hh) key 8 (r / 4) + 4 hh + r % 4, query n
            f32x16 s[2];
            const f32x16 z = {};
            const f16* ka = sm.k[cur] + (sub * kBN + n) * F::kKPitch + 8 * hh;
#pragma unroll
            for (int ks = 0; ks < KS; ks++)
#pragma unroll
                for (int i = 0; i < 2; i++)
                    s[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(as_h8(ld16(ka + 32 * i * F::kKPitch + 16 * ks)), qa[ks],
                                                                  ks ? s[i] : z, 0, 0, 0);
            if (key0 + kBN > wave_least) {
#pragma unroll
                for (int i = 0; i < 2; i++)
#pragma unroll
                    for (int r = 0; r < 16; r++)
                        if (key0 + 32 * i + 8 * (r / 4) + 4 * hh + r % 4 >= seen) s[i][r] = -INFINITY;
            }
            u32x4 p[2][2];
            // The tile's weights against a reference, rounded to f16 (see
            // kWeightBits), and the sum of the rounded ones over the lane's
            // keys, in f32 like the product's.
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
            // as it is; only a query of which one does not fit f16, so that its
            // sum is infinite, moves its own. Where the wave's references have
            // moved lately, the scores' maximum says so ahead of the weights.
            bool own = key0 == (SPLIT ? t.begin : 0) || fabsf(m) > kFar, move = wary > 0 || __any(own);
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
                own |= __builtin_amdgcn_exp2f(fmaf(mx, c, -m)) >= kPastF16;
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
            // O^T += V^T P^T. The transposing read gives lane i of 16 channel
            // i of 4 keys: two reads make the 8 keys, in the scores' order.
            const int vrow = 4 * hh + (n & 15) / 4;
            const f16* va = sm.v[cur] + (sub * kBN + vrow) * F::kVPitch + (n & 16) + 4 * (n & 3);
            auto read_v = [&](int g, int db) {
                const f16* r0 = va + 16 * g * F::kVPitch + 32 * db;
                const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)r0));
                const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(r0 + 8 * F::kVPitch)));
                u32x4 w;
                w[0] = lo[0], w[1] = lo[1], w[2] = hi[0], w[3] = hi[1];
                return w;
            };
#pragma unroll
            for (int g = 0; g < 4; g++)
#pragma unroll
                for (int db = 0; db < DB; db++)
                    o[db] = __builtin_amdgcn_mfma_f32_32x32x16_f16(as_h8(read_v(g, db)), as_h8(p[g / 2][g % 2]), o[db], 0, 0, 0);
        }
        if (j + 1 < ntiles) store(cur ^ 1, (j + 1) * F::kKeys);
        __syncthreads();
    }
    if (qi >= t.nq) return;
    if (tile0 < ntiles && sm.odd) add_odd<f16, DB>(o, a, t, kv, F::kKeys, tile_least, seen, hh);
    if (SPLIT && t.count > 1) {
        put_partial<DB>(a, t, block + n, hh, o, m, halves_sum(l), 1.0f);
        return;
    }
    const float inv = 1.0f / halves_sum(l);
    f16* orow = static_cast<f16*>(a.out) + (static_cast<int64_t>(t.q0 + qi) * a.h + t.head) * D + 4 * hh;
#pragma unroll
    for (int db = 0; db < DB; db++)
#pragma unroll
        for (int r4 = 0; r4 < 4; r4++) {
            float x[4];
#pragma unroll
            for (int e = 0; e < 4; e++) x[e] = seen > 0 ? o[db][4 * r4 + e] * inv : 0.0f;
            u32x2 w;
            w[0] = pk_f16(x[0], x[1]), w[1] = pk_f16(x[2], x[3]);
            *reinterpret_cast<u32x2*>(orow + 32 * db + 8 * r4) = w;
        }
}

// ---------------------------------------------------------------------------
// f32
//
// The same transposed scheme on v_mfma_f32_32x32x2_f32: register j of a
// 4-element piece is a product's two dims (8 g + j and 8 g + 4 + j, by lane
// half), and score register r, the key 8 (r / 4) + 4 hh + r % 4, multiplies that
// key's row of V as it lies. One tile in LDS, the next in registers.
template <int D>
struct FlashF32 {
    static constexpr int DB = D / 32;
    static constexpr int kRowChunks = D / 4;
    static constexpr int kPer = kBN * kRowChunks / kThreads;
    // floats per row: 16-byte reads of 16 rows 4 banks apart in K; in V the two
    // halves read rows 4 apart, half the banks each
    static constexpr int kKPitch = D + 4, kVPitch = D + 8;
    struct Smem {
        float k[kBN * kKPitch];
        float v[kBN * kVPitch];
        int odd;
    };
};

__device__ __forceinline__ bool odd_f32(uint32_t bits) { return (bits & 0x7F800000u) == 0x7F800000u; }

// The tile's queries, those of lanes with `mine` stored; every wave of the
// workgroup calls it (barriers inside).
template <int D, bool SPLIT>
__device__ __forceinline__ void packed_f32_tile(const PackedArgs& a, const PackedTile& t, typename FlashF32<D>::Smem& sm, bool mine) {
    using F = FlashF32<D>;
    constexpr int DB = F::DB, kPer = F::kPer;
    const int tid = threadIdx.x, lane = lane_id(), wave = wave_in_block();
    const int n = lane & 31, hh = lane >> 5;
    const int kv = t.head / (a.h / a.h_kv);
    const float* kb = static_cast<const float*>(a.k) + t.k0 * a.k_stride + kv * D;
    const float* vb = static_cast<const float*>(a.v) + t.k0 * a.v_stride + kv * D;

    const int qi = t.first + 32 * wave + n;
    const bool live = t.first + 32 * wave < t.nq;
    const int seen = keys_seen(min(qi, t.nq - 1), t.nq, t.nk, a.causal);
    const int wave_least = keys_seen(min(t.first + 32 * wave, t.nq - 1), t.nq, t.nk, a.causal);
    const int wave_most = live ? keys_seen(min(t.first + 32 * wave + 31, t.nq - 1), t.nq, t.nk, a.causal) : 0;
    const int tile_least = keys_seen(t.first, t.nq, t.nk, a.causal);
    const int begin = SPLIT ? t.begin : 0;

    const float c = fmaxf(fabsf(a.scale) * 1.4426950408889634f, 1.4e-45f);
    const uint32_t flip = a.scale < 0.0f ? 0x80000000u : 0u;
    u32x4 qv[D / 8];
    {
        const float* qr = static_cast<const float*>(a.q) + (t.q0 + min(qi, t.nq - 1)) * a.q_stride + t.head * D + 4 * hh;
#pragma unroll
        for (int i = 0; i < D / 8; i++) qv[i] = ld16(qr + 8 * i) ^ flip;
    }
    f32x16 o[DB];
#pragma unroll
    for (int i = 0; i < DB; i++) o[i] = f32x16{};
    float m = kFloor, l = 0.0f;

    u32x4 pk[kPer], pv[kPer];
    const int row0 = tid / F::kRowChunks, col0 = tid % F::kRowChunks * 4;
    constexpr int kRowStep = kThreads / F::kRowChunks;
    auto load = [&](int key0) {
#pragma unroll
        for (int i = 0; i < kPer; i++) {
            const int64_t row = min(key0 + row0 + kRowStep * i, t.nk - 1);  // past the end: masked
            pk[i] = ld16(kb + row * a.k_stride + col0);
            pv[i] = ld16(vb + row * a.v_stride + col0);
        }
    };
    __syncthreads();
    if (tid == 0) sm.odd = 0;
    if (begin < t.end) load(begin);
#pragma unroll 1
    for (int key0 = begin; key0 < t.end; key0 += kBN) {
        __syncthreads();  // the previous tile has been read
        if (key0 + kBN > tile_least) {  // some query does not see all of these values
            bool odd = false;
#pragma unroll
            for (int i = 0; i < kPer; i++)
#pragma unroll
                for (int w = 0; w < 4; w++)
                    if (odd_f32(pv[i][w])) odd = true, pv[i][w] = 0;
            if (odd) sm.odd = 1;
        }
#pragma unroll
        for (int i = 0; i < kPer; i++) {
            st16(&sm.k[(row0 + kRowStep * i) * F::kKPitch + col0], pk[i]);
            st16(&sm.v[(row0 + kRowStep * i) * F::kVPitch + col0], pv[i]);
        }
        __syncthreads();
        if (key0 + kBN < t.end) load(key0 + kBN);
        if (key0 >= wave_most) continue;

        f32x16 s[2] = {f32x16{}, f32x16{}};
        const float* ka = sm.k + n * F::kKPitch + 4 * hh;
#pragma unroll
        for (int g = 0; g < D / 8; g++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const u32x4 x = ld16(ka + 32 * i * F::kKPitch + 8 * g);
#pragma unroll
                for (int e = 0; e < 4; e++)
                    s[i] = __builtin_amdgcn_mfma_f32_32x32x2f32(u2f(x[e]), u2f(qv[g][e]), s[i], 0, 0, 0);
            }
        if (key0 + kBN > wave_least) {
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int r = 0; r < 16; r++)
                    if (key0 + 32 * i + 8 * (r / 4) + 4 * hh + r % 4 >= seen) s[i][r] = -INFINITY;
        }
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
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int r = 0; r < 16; r++) {
                s[i][r] = __builtin_amdgcn_exp2f(s[i][r] - m);
                sum += s[i][r];
            }
        l = fmaf(l, corr, sum);
#pragma unroll
        for (int i = 0; i < DB; i++) o[i] *= corr;
        const float* va = sm.v + 4 * hh * F::kVPitch + n;
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int r = 0; r < 16; r++)
#pragma unroll
                    for (int db = 0; db < DB; db++)
                        o[db] = __builtin_amdgcn_mfma_f32_32x32x2f32(va[(32 * i + 8 * (r / 4) + r % 4) * F::kVPitch + 32 * db], s[i][r],
                                                                     o[db], 0, 0, 0);
    }
    __syncthreads();
    if (qi >= t.nq || !mine) return;
    if (sm.odd) add_odd<float, DB>(o, a, t, kv, kBN, tile_least, seen, hh);
    if (SPLIT && t.count > 1) {
        put_partial<DB>(a, t, 32 * wave + n, hh, o, m, halves_sum(l), 1.0f);
        return;
    }
    const float lsum = halves_sum(l);
    float* orow = static_cast<float*>(a.out) + (static_cast<int64_t>(t.q0 + qi) * a.h + t.head) * D + 4 * hh;
#pragma unroll
    for (int db = 0; db < DB; db++)
#pragma unroll
        for (int r4 = 0; r4 < 4; r4++) {
            u32x4 w;
#pragma unroll
            for (int e = 0; e < 4; e++) w[e] = f2u(seen > 0 ? o[db][4 * r4 + e] / lsum : 0.0f);
            st16(orow + 32 * db + 8 * r4, w);
        }
}

template <int D, bool SPLIT>
__global__ __launch_bounds__(kThreads, 2) void packed_f32_kernel(PackedArgs a) {
    __shared__ __align__(16) typename FlashF32<D>::Smem sm;
    PackedTile t;
    if (!packed_tile<SPLIT>(a, kBM, t)) return;  // workgroup-uniform, before any barrier
    packed_f32_tile<D, SPLIT>(a, t, sm, true);
}

// f32, head dim 64, on the bf16 matrix instructions, sixteen times the f32
// ones' rate: each value is three bf16 (split3) and a product six of theirs
// with f32 accumulators, to 2^-24 of it as one f32 rounding. Queries are split
// once, K and V as their tiles are staged, the weights where the f16 kernel
// rounds them. The small products are summed ahead of the large one in the
// scores and in accumulators of their own in the output, so that they add no
// rounding of full size; a weight carries a factor 2^23, so that it keeps its 24
// bits down to 2^-126 of the largest. One tile in LDS (two workgroups per CU:
// one stages while the other multiplies), the next in registers.
//
// A query above 2^50 in magnitude, and every query of a tile that stages such a
// key or value, an infinity or NaN, or a nonzero value below 2^-100 (where
// bf16's last part ends), is computed again on the f32 instructions.
typedef bf16x8 b8;
constexpr int kSD = 64, kSKPitch = kSD + 8, kSVPitch = kSD + 32;
constexpr uint32_t kSplitMaxBits = 0x58800000u;  // 2^50
constexpr float kSplitScale = 0x1p23f;
// The reference moves where a lane's row sum over a tile passes this, to a
// maximum this far (log2) above it.
constexpr float kRowSumMax = 32768.0f;
constexpr float kLazyMax = 8.0f;

struct SplitSmem {
    uint16_t k[3][kBN * kSKPitch];
    uint16_t v[3][kBN * kSVPitch];
};

__device__ __forceinline__ b8 as_b8(u32x4 v) { return __builtin_bit_cast(b8, v); }

// 8 floats as h, m and l pieces.
__device__ __forceinline__ void split_piece(const u32x4 (&f)[2], u32x4 (&part)[3]) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        uint32_t h, m, l;
        split3(u2f(f[i / 2][2 * (i % 2)]), u2f(f[i / 2][2 * (i % 2) + 1]), h, m, l);
        part[0][i] = h, part[1][i] = m, part[2][i] = l;
    }
}
__device__ __forceinline__ uint32_t largest(uint32_t most, const u32x4 (&f)[2]) {
#pragma unroll
    for (int i = 0; i < 8; i++) most = max(most, f[i / 4][i % 4] & 0x7FFFFFFFu);
    return most;
}

template <bool SPLIT>
__global__ __launch_bounds__(kThreads, 2) void packed_split_kernel(PackedArgs a) {
    union Smem {
        SplitSmem split;
        FlashF32<kSD>::Smem f32;
    };
    __shared__ __align__(16) Smem smem;
    __shared__ int again;  // bit 0: every query of the tile, bit 1: some
    SplitSmem& sm = smem.split;
    PackedTile t;
    if (!packed_tile<SPLIT>(a, kBM, t)) return;  // workgroup-uniform, before any barrier
    const int tid = threadIdx.x, lane = lane_id(), wave = wave_in_block();
    const int n = lane & 31, hh = lane >> 5;
    const int kv = t.head / (a.h / a.h_kv);
    const float* kb = static_cast<const float*>(a.k) + t.k0 * a.k_stride + kv * kSD;
    const float* vb = static_cast<const float*>(a.v) + t.k0 * a.v_stride + kv * kSD;
    const int qi = t.first + 32 * wave + n;
    const bool live = t.first + 32 * wave < t.nq;
    const int seen = keys_seen(min(qi, t.nq - 1), t.nq, t.nk, a.causal);
    const int wave_least = keys_seen(min(t.first + 32 * wave, t.nq - 1), t.nq, t.nk, a.causal);
    const int wave_most = live ? keys_seen(min(t.first + 32 * wave + 31, t.nq - 1), t.nq, t.nk, a.causal) : 0;
    const int begin = SPLIT ? t.begin : 0;
    const float c = a.scale * 1.4426950408889634f;  // goes into the queries
    if (tid == 0) again = 0;
    __syncthreads();

    // staging: piece i of the thread is row 32 i + tid / 8, dims 8 (tid % 8) .. + 8
    const int prow = tid / 8, pd = 8 * (tid % 8);
    u32x4 kr[2][2], vr[2][2];
    auto load = [&](int key0) {
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int64_t row = min(key0 + 32 * i + prow, t.nk - 1);  // past the end: masked
#pragma unroll
            for (int e = 0; e < 2; e++) {
                kr[i][e] = ld16(kb + row * a.k_stride + pd + 4 * e);
                vr[i][e] = ld16(vb + row * a.v_stride + pd + 4 * e);
            }
        }
    };
    uint32_t big = 0;  // of K and V
    SplitSmall small;  // of V
    auto stage = [&]() {
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int row = 32 * i + prow;
            u32x4 part[3];
            split_piece(kr[i], part);
#pragma unroll
            for (int p = 0; p < 3; p++) st16(&sm.k[p][row * kSKPitch + pd], part[p]);
            split_piece(vr[i], part);
#pragma unroll
            for (int p = 0; p < 3; p++) st16(&sm.v[p][row * kSVPitch + pd], part[p]);
            big = largest(largest(big, kr[i]), vr[i]);
#pragma unroll
            for (int e = 0; e < 4; e++) small.note(u2f(vr[i][e / 2][2 * (e % 2)]), u2f(vr[i][e / 2][2 * (e % 2) + 1]));
        }
    };
    if (begin < t.end) load(begin);

    u32x4 qp[3][4];
    bool bad_q;
    {
        const float* qr = static_cast<const float*>(a.q) + (t.q0 + min(qi, t.nq - 1)) * a.q_stride + t.head * kSD + 8 * hh;
        uint32_t qbig = 0;
#pragma unroll
        for (int ks = 0; ks < 4; ks++) {
            u32x4 f[2] = {ld16(qr + 16 * ks), ld16(qr + 16 * ks + 4)};
#pragma unroll
            for (int e = 0; e < 8; e++) f[e / 4][e % 4] = f2u(u2f(f[e / 4][e % 4]) * c);
            u32x4 part[3];
            split_piece(f, part);
            qp[0][ks] = part[0], qp[1][ks] = part[1], qp[2][ks] = part[2];
            qbig = largest(qbig, f);
        }
        const auto both = __builtin_amdgcn_permlane32_swap(qbig, qbig, false, false);
        bad_q = max(static_cast<uint32_t>(both[0]), static_cast<uint32_t>(both[1])) > kSplitMaxBits;
    }

    f32x16 o[2] = {f32x16{}, f32x16{}}, ol[2] = {f32x16{}, f32x16{}};
    float m = kFloor, l = 0.0f;
#pragma unroll 1
    for (int key0 = begin; key0 < t.end; key0 += kBN) {
        __syncthreads();  // the previous tile has been read
        stage();
        __syncthreads();
        const bool more = key0 + kBN < t.end;
        if (key0 >= wave_most) {
            if (more) load(key0 + kBN);
            continue;
        }
        f32x16 s[2];
        const f32x16 z = {};
        const int koff = n * kSKPitch + 8 * hh;
        auto read_k = [&](u32x4(&dst)[2], int part, int ks) {
#pragma unroll
            for (int i = 0; i < 2; i++) dst[i] = ld16(sm.k[part] + koff + 32 * i * kSKPitch + 16 * ks);
        };
        auto score = [&](const u32x4(&kk)[2], const u32x4& qq, bool first) {
#pragma unroll
            for (int i = 0; i < 2; i++)
                s[i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_b8(kk[i]), as_b8(qq), first ? z : s[i], 0, 0, 0);
        };
        // the small products slice by slice (h read a slice ahead, m and l
        // under the products before theirs), then h h
        u32x4 kh[2][2], km[2], kl[2];
        read_k(kh[0], 0, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);  // LDS reads
#pragma unroll
        for (int ks = 0; ks < 4; ks++) {
            read_k(km, 1, ks);
            read_k(kl, 2, ks);
            read_k(kh[(ks + 1) & 1], 0, (ks + 1) & 3);
            score(kh[ks & 1], qp[1][ks], ks == 0);
            score(kh[ks & 1], qp[2][ks], false);
            score(km, qp[1][ks], false);
            score(km, qp[0][ks], false);
            score(kl, qp[0][ks], false);
            __builtin_amdgcn_sched_group_barrier(0x100, 6, 0);
            __builtin_amdgcn_sched_group_barrier(0x008, 10, 0);  // MFMAs
        }
#pragma unroll
        for (int ks = 0; ks < 4; ks++) {
            if (ks < 3) read_k(kh[(ks + 1) & 1], 0, ks + 1);
            score(kh[ks & 1], qp[0][ks], false);
            if (ks < 3) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
            __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
        }
        if (key0 + kBN > wave_least) {
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int r = 0; r < 16; r++)
                    if (key0 + 32 * i + 8 * (r / 4) + 4 * hh + r % 4 >= seen) s[i][r] = -INFINITY;
        }
        // the next rows once the scores' operands have left the registers (at
        // the top of the tile they spilled: 286 us for 220)
        if (more) load(key0 + kBN);
        u32x4 wp[3][2][2];
        auto weights = [&](float ref) {
            float ps[2] = {0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int w = 0; w < 8; w++) {
                    float p[2];
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        p[e] = kSplitScale * __builtin_amdgcn_exp2f(s[i][2 * w + e] - ref);
                        ps[e] += p[e];
                    }
                    uint32_t h, md, lo;
                    split3(p[0], p[1], h, md, lo);
                    wp[0][i][w / 4][w % 4] = h, wp[1][i][w / 4][w % 4] = md, wp[2][i][w / 4][w % 4] = lo;
                }
            return ps[0] + ps[1];
        };
        // the reference moves on the first tile and where a weight might pass
        // 2^15 times the largest at it, for the query's own sums only
        bool own = key0 == begin, move = own;
        if (!move) {
            const float ps = weights(m);
            own = !(halves_max(ps) <= kRowSumMax * kSplitScale);
            move = __any(own);
            if (!move) l += ps;
        }
        if (move) {
            float mx = s[0][0];
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int r = 0; r < 16; r++) mx = fmaxf(mx, s[i][r]);
            const float cand = fmaxf(m, halves_max(mx));
            const float next = own && cand > m + kLazyMax ? cand : m;
            const float corr = __builtin_amdgcn_exp2f(m - next);
            l = fmaf(l, corr, weights(next));
            m = next;
#pragma unroll
            for (int i = 0; i < 2; i++) o[i] *= corr, ol[i] *= corr;
        }
        const int l16 = n & 15;
        const int voff = (4 * hh + l16 / 4) * kSVPitch + (n & 16) + 4 * (l16 % 4);
        auto read_v = [&](u32x4(&dst)[2], int part, int g) {
#pragma unroll
            for (int db = 0; db < 2; db++) {
                const uint16_t* r0 = sm.v[part] + voff + 16 * g * kSVPitch + 32 * db;
                const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)r0));
                const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(r0 + 8 * kSVPitch)));
                dst[db][0] = lo[0], dst[db][1] = lo[1], dst[db][2] = hi[0], dst[db][3] = hi[1];
            }
        };
        auto add = [&](f32x16(&acc)[2], const u32x4(&vv)[2], const u32x4& w) {
#pragma unroll
            for (int db = 0; db < 2; db++)
                acc[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_b8(vv[db]), as_b8(w), acc[db], 0, 0, 0);
        };
        u32x4 vh[2][2], vm[2], vl[2];
        read_v(vh[0], 0, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
        for (int g = 0; g < 4; g++) {
            read_v(vm, 1, g);
            read_v(vl, 2, g);
            if (g < 3) read_v(vh[(g + 1) & 1], 0, g + 1);
            const u32x4 wh = wp[0][g / 2][g % 2], wm = wp[1][g / 2][g % 2], wl = wp[2][g / 2][g % 2];
            add(o, vh[g & 1], wh);
            add(ol, vh[g & 1], wm);
            add(ol, vh[g & 1], wl);
            add(ol, vm, wm);
            add(ol, vm, wh);
            add(ol, vl, wh);
            if (g < 3)
                __builtin_amdgcn_sched_group_barrier(0x100, 12, 0);
            else
                __builtin_amdgcn_sched_group_barrier(0x100, 8, 0);
            __builtin_amdgcn_sched_group_barrier(0x008, 12, 0);
        }
    }
    const bool bad_kv = big > kSplitMaxBits || small.seen();
    if (bad_kv || bad_q) atomicOr(&again, (bad_kv ? 1 : 0) | (bad_q ? 2 : 0));
    __syncthreads();
    const int redo = again;
    const bool mine = (redo & 1) != 0 || bad_q;
    if (SPLIT && t.count > 1) {
        if (qi < t.nq && !mine) {
#pragma unroll
            for (int db = 0; db < 2; db++) o[db] += ol[db];
            put_partial<2>(a, t, 32 * wave + n, hh, o, m, halves_sum(l), 1.0f / kSplitScale);
        }
    } else if (qi < t.nq && !mine) {
        const float lsum = halves_sum(l);
        float* orow = static_cast<float*>(a.out) + (static_cast<int64_t>(t.q0 + qi) * a.h + t.head) * kSD + 4 * hh;
#pragma unroll
        for (int db = 0; db < 2; db++)
#pragma unroll
            for (int r4 = 0; r4 < 4; r4++) {
                u32x4 w;
#pragma unroll
                for (int e = 0; e < 4; e++) w[e] = f2u(seen > 0 ? (o[db][4 * r4 + e] + ol[db][4 * r4 + e]) / lsum : 0.0f);
                st16(orow + 32 * db + 8 * r4, w);
            }
    }
    if (redo) packed_f32_tile<kSD, SPLIT>(a, t, smem.f32, mine);  // workgroup-uniform
}

// f32, short sequences: a serial chain per query, so it is cut as finely as the
// matrix instructions allow. A workgroup takes 16 queries and its four waves
// share their keys, 16 at a time in turn, on v_mfma_f32_16x16x4_f32: K as the A
// operand straight from memory, V through the wave's own slice of LDS; the four
// (O, m, l) join in LDS.
template <int D>
struct FewF32 {
    static constexpr int kQueries = 16;
    static constexpr int kRowLanes = D / 4, kVRows = 64 / kRowLanes, kVLoads = 16 / kVRows;
    static constexpr int kPitch = D + 4;
    struct Smem {
        union {
            float v[kWaves][16 * kPitch];
            float o[kWaves][kQueries * kPitch];
        };
        float m[kWaves][kQueries], l[kWaves][kQueries];
        int odd;  // as in the kernels above
    };
};

typedef float f32x4 __attribute__((ext_vector_type(4)));

template <int D, bool SPLIT>
__global__ __launch_bounds__(kThreads, D == 64 ? 2 : 3) void packed_few_f32_kernel(PackedArgs a) {
    using F = FewF32<D>;
    constexpr int KS = D / 16, DB = D / 16;
    __shared__ __align__(16) typename F::Smem sm;
    PackedTile t;
    if (!packed_tile<SPLIT>(a, F::kQueries, t)) return;  // workgroup-uniform, before any barrier
    const int lane = lane_id(), wave = wave_in_block();
    const int n = lane & 15, g = lane >> 4;
    const int kv = t.head / (a.h / a.h_kv);
    const float* kb = static_cast<const float*>(a.k) + t.k0 * a.k_stride + kv * D;
    const float* vb = static_cast<const float*>(a.v) + t.k0 * a.v_stride + kv * D;
    const int qi = t.first + n;
    const int seen = keys_seen(min(qi, t.nq - 1), t.nq, t.nk, a.causal);
    const int least = keys_seen(t.first, t.nq, t.nk, a.causal);
    const int begin = (SPLIT ? t.begin : 0) + 16 * wave;

    const float c = fmaxf(fabsf(a.scale) * 1.4426950408889634f, 1.4e-45f);
    const uint32_t flip = a.scale < 0.0f ? 0x80000000u : 0u;
    const float* qr = static_cast<const float*>(a.q) + (t.q0 + min(qi, t.nq - 1)) * a.q_stride + t.head * D + 4 * g;
    u32x4 qv[KS];
#pragma unroll
    for (int i = 0; i < KS; i++) qv[i] = ld16(qr + 16 * i) ^ flip;
    f32x4 o[DB];
#pragma unroll
    for (int i = 0; i < DB; i++) o[i] = f32x4{};
    float m = kFloor, l = 0.0f;  // l: this lane's keys only
    if (threadIdx.x == 0) sm.odd = 0;
    __syncthreads();
    float* vs = sm.v[wave];
    u32x4 kr[KS], vr[F::kVLoads];
    auto load_v = [&](int key0) {
#pragma unroll
        for (int i = 0; i < F::kVLoads; i++) {
            const int64_t row = min(key0 + F::kVRows * i + lane / F::kRowLanes, t.nk - 1);
            vr[i] = ld16(vb + row * a.v_stride + lane % F::kRowLanes * 4);
        }
    };
    auto load_k = [&](int key0) {
        const float* kp = kb + static_cast<int64_t>(min(key0 + n, t.nk - 1)) * a.k_stride + 4 * g;
#pragma unroll
        for (int i = 0; i < KS; i++) kr[i] = ld16(kp + 16 * i);
    };
    constexpr int kTurn = 16 * kWaves;
    if (begin < t.end) load_v(begin), load_k(begin);
#pragma unroll 1
    for (int key0 = begin; key0 < t.end; key0 += kTurn) {
        const bool partial = key0 + 16 > least;  // some query does not see all of these keys
        if (partial) {
#pragma unroll
            for (int i = 0; i < F::kVLoads; i++)
#pragma unroll
                for (int w = 0; w < 4; w++)
                    if (odd_f32(vr[i][w])) sm.odd = 1, vr[i][w] = 0;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int i = 0; i < F::kVLoads; i++) {
            st16(vs + (F::kVRows * i + lane / F::kRowLanes) * F::kPitch + lane % F::kRowLanes * 4, vr[i]);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (key0 + kTurn < t.end) load_v(key0 + kTurn);
        f32x4 acc[4] = {f32x4{}, f32x4{}, f32x4{}, f32x4{}};
#pragma unroll
        for (int i = 0; i < KS; i++)
#pragma unroll
            for (int e = 0; e < 4; e++)
                acc[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(u2f(kr[i][e]), u2f(qv[i][e]), acc[e], 0, 0, 0);
        f32x4 s = (acc[0] + acc[1]) + (acc[2] + acc[3]);
        // rounded before the maximum is taken off: that one then weighs 1
#pragma unroll
        for (int j = 0; j < 4; j++) s[j] = as_f32(s[j] * c);
        if (key0 + kTurn < t.end) load_k(key0 + kTurn);
        if (partial)
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (key0 + 4 * g + j >= seen) s[j] = -INFINITY;
        float mx = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
        mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        const float next = fmaxf(m, mx);
        const float corr = __builtin_amdgcn_exp2f(m - next);
        m = next;
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            s[j] = __builtin_amdgcn_exp2f(s[j] - m);
            sum += s[j];
        }
        l = fmaf(l, corr, sum);
#pragma unroll
        for (int i = 0; i < DB; i++) o[i] *= corr;
        const float* va = vs + 4 * g * F::kPitch + n;
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int i = 0; i < DB; i++)
                    o[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(va[j * F::kPitch + 16 * i], s[j], o[i], 0, 0, 0);
    }
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < DB; i++) *reinterpret_cast<f32x4*>(&sm.o[wave][n * F::kPitch + 16 * i + 4 * g]) = o[i];
    if (g == 0) sm.m[wave][n] = m, sm.l[wave][n] = l;
    __syncthreads();
    for (int x = threadIdx.x; x < F::kQueries * (D / 4); x += kThreads) {
        const int q = x / (D / 4), d0 = x % (D / 4) * 4;
        if (t.first + q >= t.nq) break;
        const int keys = keys_seen(t.first + q, t.nq, t.nk, a.causal);
        float top = sm.m[0][q];
#pragma unroll
        for (int w = 1; w < kWaves; w++) top = fmaxf(top, sm.m[w][q]);
        f32x4 sum = {};
        float weight = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; w++) {
            const float f = __builtin_amdgcn_exp2f(sm.m[w][q] - top);
            sum += *reinterpret_cast<const f32x4*>(&sm.o[w][q * F::kPitch + d0]) * f;
            weight = fmaf(sm.l[w][q], f, weight);
        }
        if (sm.odd)
            for (int key = max(least / 16 * 16, t.begin); key < min(keys, t.end); key++) {
                const u32x4 v = ld16(vb + key * a.v_stride + d0);
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (odd_f32(v[e])) sum[e] += u2f(v[e]);
            }
        if (SPLIT && t.count > 1) {
            const int64_t at = partial_row(a, t, q);
            *reinterpret_cast<f32x4*>(a.ws_o + at * D + d0) = sum;
            if (d0 == 0) a.ws_ml[2 * at] = top, a.ws_ml[2 * at + 1] = weight;
            continue;
        }
        float* orow = static_cast<float*>(a.out) + (static_cast<int64_t>(t.q0 + t.first + q) * a.h + t.head) * D + d0;
        u32x4 w;
#pragma unroll
        for (int e = 0; e < 4; e++) w[e] = f2u(keys > 0 ? sum[e] / weight : 0.0f);
        st16(orow, w);
    }
}

// Sums of two pieces joined. An infinity of values stays one where the other
// piece's maximum leaves it a weight of 0.
__device__ __forceinline__ void join_sums(f32x4& sum, float& weight, float& top, f32x4 v, float l, float m) {
    const float next = fmaxf(top, m);
    const float old = __builtin_amdgcn_exp2f(top - next), f = __builtin_amdgcn_exp2f(m - next);
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const float x = sum[e] * old, y = v[e] * f;
        sum[e] = (x != x ? sum[e] : x) + (y != y ? v[e] : y);
    }
    weight = fmaf(weight, old, l * f);
    top = next;
}

// The pieces of a tile's queries joined: a workgroup takes one (query, head), its
// threads the pieces (SHARE), or kRows of them, each its pieces in turn.
template <typename T, int D, bool SHARE>
__global__ __launch_bounds__(kThreads) void packed_join_kernel(PackedArgs a, int bm) {
    constexpr int kLanes = D / 4, kRows = kThreads / kLanes;
    __shared__ __align__(16) f32x4 part[kRows][kLanes];
    __shared__ float tops[kRows], weights[kRows];
    const int group = threadIdx.x / kLanes, col = threadIdx.x % kLanes;
    const int per_tile = SHARE ? a.pitch : (a.pitch + kRows - 1) / kRows;
    const int tile_head = static_cast<int>(blockIdx.x) / per_tile;
    const int tile = tile_head / a.h, head = tile_head - tile * a.h;
    PackedCut c;
    if (!find_cut<true>(a, bm, tile, c)) return;  // workgroup-uniform, as what follows
    const int nq = c.q.end - c.q.begin, nk = c.k.end - c.k.begin;
    const int first = (c.tiles - 1 - c.local) * bm, rows = min(bm, nq - first);
    const int count = pieces_seen(keys_seen(first + rows - 1, nq, nk, a.causal), c.chunk);
    if (count == 1) return;  // written by its only piece
    const int row0 = static_cast<int>(blockIdx.x) - tile_head * per_tile;
    const int row = SHARE ? row0 : row0 * kRows + group;
    float top = kFloor, weight = 0.0f;
    f32x4 sum = {};
    if (row < rows) {
        PackedTile t;
        t.head = head;
        for (int i = SHARE ? group : 0; i < count; i += SHARE ? kRows : 1) {
            t.item = c.item + i;
            const int64_t at = partial_row(a, t, row);
            const float m = a.ws_ml[2 * at], l = a.ws_ml[2 * at + 1];
            const f32x4 v = *reinterpret_cast<const f32x4*>(a.ws_o + at * D + 4 * col);
            join_sums(sum, weight, top, v, l, m);
        }
    }
    if constexpr (SHARE) {
        part[group][col] = sum;
        if (col == 0) tops[group] = top, weights[group] = weight;
        __syncthreads();
        if (group != 0) return;
        for (int i = 1; i < min(kRows, count); i++) join_sums(sum, weight, top, part[i][col], weights[i], tops[i]);
    }
    if (row >= rows) return;
    const bool sees = keys_seen(first + row, nq, nk, a.causal) > 0;
    T* orow = static_cast<T*>(a.out) + (static_cast<int64_t>(c.q.begin + first + row) * a.h + head) * D + 4 * col;
#pragma unroll
    for (int e = 0; e < 4; e++) orow[e] = static_cast<T>(sees ? sum[e] / weight : 0.0f);
}

// How a call is cut into tiles and whether its keys are split.
struct PackedPlan {
    enum Kernel { kWide, kFour, kTile, kFew } kernel;
    int bm, share;          // queries of a tile; log2 of the heads that a workgroup takes
    int64_t tiles;          // of a head, as many as sequences of these rows can have
    int64_t pieces, items;  // of a head: wanted, and what they can come to; 0: whole keys
    int64_t pitch;
    PackedPlan(hs_dtype dt, int64_t n_q, int64_t n_k, int64_t b, int64_t h, int64_t h_kv, int d, int causal) {
        const int64_t cus = num_cus(), group = h / h_kv;
        const bool half = dt == HS_F16;
        // Enough keys for a second launch to pay (us split and whole, f16, one
        // causal sequence: 4 heads of 128 over 2, 2000 tokens 27, 49, 1200 22, 33;
        // 8 heads of 64, 2000 tokens 27, 35; 4 of 64, 1500 27, 28)
        const bool long_keys = n_k >= (d == 64 ? 1536 : 1024) && n_k >= 256 * b;
        // f16, few queries a sequence: two or four query heads of a key head share
        // a workgroup and its keys, which leaves no wave idle (32 heads of 128
        // over 8, split: 16 queries over 131072 keys 118 us, 221 by head; four
        // times 64 over 30000 205, 285)
        share = 0;
        if (half && n_q <= 64 * b && group % 2 == 0) share = n_q <= 32 * b && group % 4 == 0 ? 2 : 1;
        const int64_t all = h >> share;
        const auto cut = [&](Kernel k, int rows) { kernel = k, bm = rows, tiles = n_q / rows + (b < n_q ? b : n_q); };
        // (All figures are of one sequence or of equal ones, and the rules see the
        // average: a long sequence among many short ones may run as they do.)
        // f16: tiles of 256 queries for long sequences that make enough of them,
        // 128 else: more reuse against more masked keys and longer tails (us with
        // 128 and 256; 16 heads of 64: one sequence of 12000 tokens 694, 630, of
        // 6000 182, 195, eight of 1374, causal, 58, 66; 32 heads of 128 over 8:
        // 12000 2486, 2236, 4122 362, 345, 2748 160, 171, twenty of 300 68, 81).
        // f32: tiles of 32 queries a wave where they fill the chip's SIMDs and
        // themselves, else 16 by four waves, which at head dim 128, on the same
        // instructions, are but a third behind (us with 16 and with tiles; 16
        // heads of 64: one sequence of 1000 tokens 49, 65, eight of 200 27, 24, a
        // hundred of 50 41, 46; 32 heads of 128, causal: one of 1283 168, 199, of
        // 2000 381, 356, twenty of 300 255, 286); tiles, too, that split many keys
        // (one head of 7000 causal tokens: of 64 117, 63, of 128 288, 142; 16 of
        // 128, 1100 over 5000 551, 471; but 4 of 128, 2000 causal tokens 75, 85).
        if (half) {
            (n_q / 256 + b) * h >= 2 * cus && n_q >= 2048 * b ? cut(kWide, 256) : cut(kFour, 128 >> share);
        } else {
            const int64_t blocks = (n_q / 32 + b) * h;
            const bool tiled = d == 64 ? (blocks >= 4 * cus || long_keys) && n_q >= 128 * b
                                       : (blocks >= 7 * cus && n_q >= 640 * b) ||
                                             (long_keys && n_q >= 256 * b && (!causal || n_k >= 4096 * b));
            tiled ? cut(kTile, kBM) : cut(kFew, 16);
        }
        pieces = items = pitch = 0;
        // Keys are split where the tiles fill less than half of the chip, or less
        // than all of it under a causal mask, whose last tile would hold the call
        // up: in f32, and in f16 where sequences are long enough for the pieces'
        // traffic (us split and whole; f32, 16 heads of 64, 3000 tokens 162, 195,
        // 8 of 128 over 2, 6000 794, 1011; f16, 5 heads of 64, 7000 and 5000
        // tokens 95, 108, 8 of 128 over 2, 6000 134, 146, but 16 over 4, 3000 86,
        // 76). Into as many pieces as the chip holds at once, or twice that where
        // a tile would have but two or three (1374 tokens over 30000, 16 heads of
        // 64, f32: 1082 us, 1204), and those only of many keys (4 heads of 128
        // over 2, f16, five sequences of 4395 keys 46, 68; 16 of 64, one of 1600,
        // not causal, 38, 29) or in the tiles of f32 (16 of 64, 1600, 85, 101).
        // The causal mask empties up to half of the items, beyond those.
        const int64_t slots = cus * (kernel == kFew || (half && d == 64) ? 3 : 2);
        const bool uneven = causal && (!half || n_k >= 5120 * b);
        const bool coarse = 4 * tiles * all > slots;
        if (kernel == kWide || (uneven ? 1 : 2) * tiles * all > slots || !long_keys) return;
        if (coarse && kernel != kTile && n_k < 4096) return;
        pieces = (coarse && kernel != kFew ? 2 : 1) * slots / all - tiles;
        if (pieces < 1) pieces = 1;
        items = (causal ? 2 : 1) * pieces + tiles;
        pitch = n_q < bm ? n_q : bm;
    }
    int64_t workspace(int64_t h, int d) const { return items * h * pitch * (d + 2) * 4; }
};

}  // namespace
}  // namespace hs

extern "C" int64_t hs_attention_packed_workspace(hs_dtype dt, int64_t n_q, int64_t n_k, int32_t b, int32_t h,
                                                 int32_t h_kv, int32_t d, int32_t causal) {
    using namespace hs;
    if (n_q <= 0 || n_k <= 0 || b <= 0 || h <= 0 || causal < 0 || n_k >= (int64_t{1} << 30) || n_q >= (int64_t{1} << 30) / h) return 0;
    if (check_heads("attention_packed_workspace", dt, h, h_kv, d)) return 0;
    return PackedPlan(dt, n_q, n_k, b, h, h_kv, d, causal).workspace(h, d);
}

extern "C" hs_status hs_attention_packed(hs_stream_t stream, hs_dtype dt, const void* q, int64_t q_stride,
                                         const void* k, int64_t k_stride, const void* v, int64_t v_stride,
                                         const void* q_offsets, const void* k_offsets, void* out, void* workspace,
                                         int64_t workspace_bytes, int64_t n_q, int64_t n_k, int32_t b, int32_t h,
                                         int32_t h_kv, int32_t d, int32_t causal, float scale) {
    using namespace hs;
    const char* op = "attention_packed";
    if (hs_status rc = check_heads(op, dt, h, h_kv, d)) return rc;
    if (n_q < 0 || n_k < 0 || b < 0) return fail(HS_EINVAL, "%s: negative count", op);
    if (causal < 0) return fail(HS_EINVAL, "%s: causal %d", op, causal);
    if (!k_offsets && n_q != n_k) return fail(HS_EINVAL, "%s: without k_offsets, as many keys as queries", op);
    if (n_q == 0 || b == 0 || h == 0) return HS_OK;
    if (n_k >= (int64_t{1} << 30) || n_q >= (int64_t{1} << 30) / h)
        return fail(HS_EINVAL, "%s: n_q * Hq and n_k must be below 2^30", op);
    const int64_t width = static_cast<int64_t>(h) * d, kv_width = static_cast<int64_t>(h_kv) * d;
    if (hs_status rc = check_rows(op, "q", q, n_q, q_stride, width, dt)) return rc;
    if (hs_status rc = check_rows(op, "k", k, n_k, k_stride, kv_width, dt)) return rc;
    if (hs_status rc = check_rows(op, "v", v, n_k, v_stride, kv_width, dt)) return rc;
    if (!out || !q_offsets) return fail(HS_EINVAL, "%s: null out or q_offsets", op);
    if (!aligned16(out) || !aligned16(workspace)) return fail(HS_EUNSUPPORTED, "%s: out and workspace must be 16-byte aligned", op);
    const PackedPlan plan(dt, n_q, n_k, b, h, h_kv, d, causal);
    const int64_t need = plan.workspace(h, d);
    if (need > 0 && (!workspace || workspace_bytes < need))
        return fail(HS_EINVAL, "%s: workspace of %lld bytes, %lld needed", op, static_cast<long long>(workspace_bytes), static_cast<long long>(need));
    const int64_t out_bytes = n_q * width * dtype_size(dt);
    const int64_t q_bytes = row_bytes(n_q, q_stride, width, dt), k_bytes = row_bytes(n_k, k_stride, kv_width, dt);
    const int64_t v_bytes = row_bytes(n_k, v_stride, kv_width, dt);
    if (overlaps(out, out_bytes, q, q_bytes) || overlaps(out, out_bytes, k, k_bytes) || overlaps(out, out_bytes, v, v_bytes))
        return fail(HS_EINVAL, "%s: out overlaps an input", op);
    if (overlaps(workspace, need, q, q_bytes) || overlaps(workspace, need, k, k_bytes) || overlaps(workspace, need, v, v_bytes) ||
        overlaps(workspace, need, out, out_bytes))
        return fail(HS_EINVAL, "%s: workspace overlaps another buffer", op);
    if (!std::isfinite(scale)) return fail(HS_EINVAL, "%s: scale must be finite", op);
    PackedArgs a;
    a.q = q, a.k = k, a.v = v, a.out = out;
    a.q_stride = q_stride, a.k_stride = k_stride, a.v_stride = v_stride;
    a.q_off = static_cast<const int*>(q_offsets);
    a.k_off = static_cast<const int*>(k_offsets);
    a.n_q = static_cast<int>(n_q), a.n_k = static_cast<int>(n_k), a.b = b, a.h = h, a.h_kv = h_kv;
    a.causal = causal, a.scale = scale, a.share = plan.share;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int threads = plan.kernel == PackedPlan::kWide ? 512 : kThreads;
    const int64_t per_head = plan.items ? plan.items : plan.tiles;
    const int64_t groups = per_head * (h >> plan.share);
    if (groups >= (int64_t{1} << 31) / threads) return fail(HS_EINVAL, "%s: too many sequences and heads", op);
    const auto go = [&](auto kernel) {
        kernel<<<dim3(static_cast<uint32_t>(groups)), dim3(threads), 0, st>>>(a);
        return check_launch(op);
    };
    if (plan.kernel == PackedPlan::kWide) return d == 64 ? go(packed_f16_kernel<64, 8, 1, false>) : go(packed_f16_kernel<128, 8, 2, false>);
    if (!plan.items) {
        if (plan.kernel == PackedPlan::kFour) return d == 64 ? go(packed_f16_kernel<64, 4, 1, false>) : go(packed_f16_kernel<128, 4, 1, false>);
        if (plan.kernel == PackedPlan::kTile) return d == 64 ? go(packed_split_kernel<false>) : go(packed_f32_kernel<128, false>);
        return d == 64 ? go(packed_few_f32_kernel<64, false>) : go(packed_few_f32_kernel<128, false>);
    }
    a.ws_o = static_cast<float*>(workspace);
    a.ws_ml = a.ws_o + plan.items * h * plan.pitch * d;
    // (rounded up by twice the error of the kernels' sum over the sequences)
    a.per_piece = static_cast<float>((1.0 + (b / 64 + 64) * 0x1p-23) / static_cast<double>(plan.pieces));
    a.items = static_cast<int>(plan.items), a.pitch = static_cast<int>(plan.pitch);
    hs_status rc;
    if (plan.kernel == PackedPlan::kFour)
        rc = d == 64 ? go(packed_f16_kernel<64, 4, 1, true>) : go(packed_f16_kernel<128, 4, 1, true>);
    else if (plan.kernel == PackedPlan::kTile)
        rc = d == 64 ? go(packed_split_kernel<true>) : go(packed_f32_kernel<128, true>);
    else
        rc = d == 64 ? go(packed_few_f32_kernel<64, true>) : go(packed_few_f32_kernel<128, true>);
    if (rc) return rc;
    // few queries: a workgroup each (7000 of one head of 64: 19 us so, 11 by 16)
    const int64_t together = kThreads / (d / 4);
    const bool share = plan.tiles * h * plan.pitch < together * num_cus();
    const int64_t rows = share ? plan.pitch : ceil_div(plan.pitch, together);
    const auto join = [&](auto kernel) {
        kernel<<<dim3(static_cast<uint32_t>(plan.tiles * h * rows)), dim3(kThreads), 0, st>>>(a, plan.bm);
        return check_launch(op);
    };
    if (dt == HS_F16) {
        if (d == 64) return share ? join(packed_join_kernel<f16, 64, true>) : join(packed_join_kernel<f16, 64, false>);
        return share ? join(packed_join_kernel<f16, 128, true>) : join(packed_join_kernel<f16, 128, false>);
    }
    if (d == 64) return share ? join(packed_join_kernel<float, 64, true>) : join(packed_join_kernel<float, 64, false>);
    return share ? join(packed_join_kernel<float, 128, true>) : join(packed_join_kernel<float, 128, false>);
}
