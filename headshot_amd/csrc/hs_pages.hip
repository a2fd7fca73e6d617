// Pages handed out on the GPU for gfx950: sequences' new lengths become entries of
// the page table, and the positions and places of their new tokens.
//
// Free pages lie in a ring, `count` of them from place `head` on; a call takes from
// its front and gives back behind its end, so that what it reads there and what it
// writes are apart and the two need no order between them. Prefix sums over the
// sequences give each its share: one workgroup makes them, a thread a sequence;
// the entries (a wave a sequence) and the tokens (a thread each) then follow from
// those alone. Latency: a short call is one launch of that workgroup, a long one a
// second launch of many.
#include <climits>

#include "hs_packed.hpp"

namespace hs {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kPlanWaves = kPlanThreads / 64;
constexpr int kLongest = 1 << 30;  // tokens of a sequence

struct PlanArgs {
    const int* counts;
    int *lens, *page_table, *free, *state, *offsets, *positions;
    int64_t* slots;
    int4* plan;  // long calls: per sequence, then {head, count}
    int n, b, page_shift, n_pages, max_pages;
};

// What a sequence has and gets: `old` tokens; entries [have, want) to fill from the
// taken-th page of the ring on (taken < 0: none), or [want, have) to clear, of which
// those below `end` go back as the taken-th and on.
struct Share {
    int old, have, want, taken, end;
};
struct Ring {
    int head, count;
};

__device__ __forceinline__ int entries_of(int tokens, int shift) { return (tokens >> shift) + ((tokens & ((1 << shift) - 1)) != 0); }
__device__ __forceinline__ bool is_page(const PlanArgs& a, int p) { return p >= 0 && p < a.n_pages; }

// The ring's at-th page of the n_pages places from its head.
__device__ __forceinline__ int* ring_at(const PlanArgs& a, const Ring& r, int at) {
    const int i = r.head + at;  // both below n_pages
    return a.free + (i >= a.n_pages ? i - a.n_pages : i);
}
__device__ __forceinline__ int page_taken(const PlanArgs& a, const Ring& r, const Share& s, int entry) {
    const int at = s.taken + entry - s.have;
    return s.taken >= 0 && at < r.count ? *ring_at(a, r, at) : -1;
}

template <typename V>
__device__ __forceinline__ V wave_scan(V v) {
    const int lane = lane_id();
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const V u = __shfl_up(v, d, 64);
        if (lane >= d) v += u;
    }
    return v;
}

// The sequences' shares, `keep` taking each; lens, offsets and the ring's state as
// the call leaves them. All threads of the workgroup call it and get the ring as it
// was.
template <typename K>
__device__ __forceinline__ Ring make_shares(const PlanArgs& a, K keep) {
    __shared__ int64_t sums[kPlanWaves][4];
    const int lane = lane_id(), wave = wave_in_block();
    Ring ring = {a.state[0], a.state[1]};
    ring.count = min(max(ring.count, 0), a.n_pages);
    ring.head = a.n_pages > 0 && ring.head >= 0 ? ring.head % a.n_pages : 0;
    int64_t asked = 0, back = 0, rows = 0, wanted = 0;  // by the sequences before
    for (int base = 0; base < a.b; base += kPlanThreads) {
        const int s = base + static_cast<int>(threadIdx.x);
        Share t = {0, 0, 0, -1, 0};
        int64_t v[4] = {0, 0, 0, 0};  // pages asked for, given back, new tokens, pages wanted
        int after = 0;
        if (s < a.b) {
            const int change = a.counts[s];
            t.old = min(max(a.lens[s], 0), kLongest);
            const int64_t sum = static_cast<int64_t>(t.old) + change;
            after = static_cast<int>(min(max(sum, int64_t{0}), int64_t{kLongest}));
            const int all_have = entries_of(t.old, a.page_shift), all_want = entries_of(after, a.page_shift);
            t.have = min(all_have, a.max_pages), t.want = min(all_want, a.max_pages);
            const int* entries = a.page_table + static_cast<int64_t>(s) * a.max_pages;
            t.end = t.want;
            if (t.want > t.have && (t.have == 0 || is_page(a, entries[t.have - 1]))) v[0] = t.want - t.have;
            if (t.want < t.have) {
                int lo = t.want, hi = t.have;  // the first entry that is no page
                while (lo < hi) {
                    const int mid = (lo + hi) >> 1;
                    if (is_page(a, entries[mid]))
                        lo = mid + 1;
                    else
                        hi = mid;
                }
                t.end = lo, v[1] = lo - t.want;
            }
            v[2] = max(change, 0);
            v[3] = max(all_want - all_have, 0);
        }
        int64_t mine[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            mine[i] = wave_scan(v[i]);
            if (lane == 63) sums[wave][i] = mine[i];
        }
        __syncthreads();
        int64_t before[4] = {asked, back, rows, wanted}, total[4] = {asked, back, rows, wanted};
        for (int w = 0; w < kPlanWaves; w++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if (w < wave) before[i] += sums[w][i];
                total[i] += sums[w][i];
            }
        __syncthreads();  // sums are written again
        if (s < a.b) {
            const int64_t first = v[0] > 0 ? before[0] + mine[0] - v[0] : v[1] > 0 ? before[1] + mine[1] - v[1] : -1;
            t.taken = static_cast<int>(first);
            keep(s, t);
            a.lens[s] = after;
            a.offsets[s + 1] = static_cast<int>(min(before[2] + mine[2], int64_t{INT_MAX}));
        }
        asked = total[0], back = total[1], rows = total[2], wanted = total[3];
    }
    if (threadIdx.x == 0) {
        const int taken = static_cast<int>(min(asked, static_cast<int64_t>(ring.count)));
        const int given = static_cast<int>(min(back, static_cast<int64_t>(a.n_pages - ring.count)));
        a.offsets[0] = 0;
        a.state[0] = a.n_pages > 0 ? (ring.head + taken) % a.n_pages : 0;
        a.state[1] = ring.count - taken + given;
        a.state[2] = static_cast<int>(min(wanted - taken, int64_t{INT_MAX}));
    }
    return ring;
}

// A sequence's entries, by one wave.
__device__ __forceinline__ void fill_entries(const PlanArgs& a, const Ring& r, int s, const Share& t) {
    int* entries = a.page_table + static_cast<int64_t>(s) * a.max_pages;
    for (int e = t.have + lane_id(); e < t.want; e += 64) entries[e] = page_taken(a, r, t, e);
    for (int e = t.want + lane_id(); e < t.have; e += 64) {
        const int at = r.count + t.taken + e - t.want;
        if (e < t.end && at < a.n_pages) *ring_at(a, r, at) = entries[e];
        entries[e] = -1;
    }
}

// Token `row`, the i-th new one of sequence s.
__device__ __forceinline__ void place_token(const PlanArgs& a, const Ring& r, int s, const Share& t, int row, int i) {
    const int64_t pos = static_cast<int64_t>(t.old) + i, entry = pos >> a.page_shift;
    if (a.positions) a.positions[row] = static_cast<int>(min(pos, int64_t{INT_MAX}));
    if (!a.slots) return;
    int page = -1;
    if (entry < a.max_pages)
        page = entry < t.have ? a.page_table[static_cast<int64_t>(s) * a.max_pages + entry] : page_taken(a, r, t, static_cast<int>(entry));
    a.slots[row] = is_page(a, page) ? (static_cast<int64_t>(page) << a.page_shift) + (pos & ((1 << a.page_shift) - 1)) : -1;
}

// Short calls: at most kPlanThreads sequences.
__global__ __launch_bounds__(kPlanThreads) void plan_short_kernel(PlanArgs a) {
    __shared__ Share shares[kPlanThreads];
    const Ring ring = make_shares(a, [&](int s, const Share& t) { shares[s] = t; });
    __syncthreads();  // shares and offsets
    for (int s = wave_in_block(); s < a.b; s += kPlanWaves) fill_entries(a, ring, s, shares[s]);
    const int rows = min(a.offsets[a.b], a.n);
    for (int row = threadIdx.x; row < rows; row += kPlanThreads) {
        const int s = sequence_of(a.offsets, a.b, row);
        if (s >= 0) place_token(a, ring, s, shares[s], row, row - a.offsets[s]);
    }
}

__device__ __forceinline__ int4 packed_share(const Share& t) { return {t.old, t.have, t.want, t.taken}; }

__global__ __launch_bounds__(kPlanThreads) void plan_shares_kernel(PlanArgs a) {
    int* ends = reinterpret_cast<int*>(a.plan + a.b + 1);
    const Ring ring = make_shares(a, [&](int s, const Share& t) { a.plan[s] = packed_share(t), ends[s] = t.end; });
    if (threadIdx.x == 0) a.plan[a.b] = {ring.head, ring.count, 0, 0};
}

__global__ __launch_bounds__(256) void plan_rest_kernel(PlanArgs a, int entry_blocks) {
    const int* ends = reinterpret_cast<const int*>(a.plan + a.b + 1);
    const int4 r = a.plan[a.b];
    const Ring ring = {r.x, r.y};
    const auto share = [&](int s) {
        const int4 p = a.plan[s];
        return Share{p.x, p.y, p.z, p.w, ends[s]};
    };
    const int block = blockIdx.x;
    if (block < entry_blocks) {
        const int s = block * 4 + wave_in_block();
        if (s < a.b) fill_entries(a, ring, s, share(s));
        return;
    }
    const int64_t row = static_cast<int64_t>(block - entry_blocks) * 256 + threadIdx.x;
    if (row >= min(a.offsets[a.b], a.n)) return;
    const int s = sequence_of(a.offsets, a.b, static_cast<int>(row));
    if (s >= 0) place_token(a, ring, s, share(s), static_cast<int>(row), static_cast<int>(row) - a.offsets[s]);
}

// One launch for calls that one workgroup is not long over.
bool is_short(int64_t n, int32_t b, int32_t max_pages) {
    return n <= 4096 && b <= kPlanThreads && static_cast<int64_t>(b) * max_pages <= (1 << 18);
}

bool aligned_to(const void* p, uintptr_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

}  // namespace
}  // namespace hs

extern "C" int64_t hs_plan_pages_workspace(int64_t n, int32_t b, int32_t max_pages) {
    if (n < 0 || b < 0 || max_pages < 0 || hs::is_short(n, b, max_pages)) return 0;
    return (static_cast<int64_t>(b) + 1) * 16 + static_cast<int64_t>(b) * 4;
}

extern "C" hs_status hs_plan_pages(hs_stream_t stream, const void* counts, void* lens, void* page_table, void* free,
                                   void* state, void* offsets, void* positions, void* slots, void* workspace,
                                   int64_t workspace_bytes, int64_t n, int32_t b, int32_t page, int32_t n_pages,
                                   int32_t max_pages) {
    using namespace hs;
    const char* op = "plan_pages";
    if (n < 0 || b < 0 || n_pages < 0 || max_pages < 0) return fail(HS_EINVAL, "%s: negative count", op);
    if (page <= 0) return fail(HS_EINVAL, "%s: page %d", op, page);
    if (exact_log2(page) < 0) return fail(HS_EUNSUPPORTED, "%s: page %d is no power of two", op, page);
    if (static_cast<int64_t>(max_pages) * page >= (int64_t{1} << 30)) return fail(HS_EINVAL, "%s: max_pages * page must be below 2^30", op);
    if (n >= (int64_t{1} << 30) || n_pages >= (1 << 30) || b >= (1 << 30) || static_cast<int64_t>(b) * max_pages >= (int64_t{1} << 31))
        return fail(HS_EINVAL, "%s: n, b, n_pages and b * max_pages / 2 must be below 2^30", op);
    if (!state || !offsets || (b > 0 && (!counts || !lens || (max_pages > 0 && !page_table))) || (n_pages > 0 && !free))
        return fail(HS_EINVAL, "%s: null counts, lens, page_table, free, state or offsets", op);
    const int64_t need = hs_plan_pages_workspace(n, b, max_pages);
    if (need > 0 && (!workspace || workspace_bytes < need))
        return fail(HS_EINVAL, "%s: workspace of %lld bytes, %lld needed", op, static_cast<long long>(workspace_bytes), static_cast<long long>(need));
    for (const void* p : {counts, static_cast<const void*>(lens), static_cast<const void*>(page_table), static_cast<const void*>(free),
                          static_cast<const void*>(state), static_cast<const void*>(offsets), static_cast<const void*>(positions)})
        if (!aligned_to(p, 4)) return fail(HS_EUNSUPPORTED, "%s: arrays must be aligned to their elements", op);
    if (!aligned_to(slots, 8) || !aligned16(workspace)) return fail(HS_EUNSUPPORTED, "%s: arrays must be aligned to their elements", op);
    const struct {
        const void* p;
        int64_t bytes;
    } all[9] = {{counts, b * int64_t{4}},      {lens, b * int64_t{4}},       {page_table, static_cast<int64_t>(b) * max_pages * 4},
                {free, n_pages * int64_t{4}},  {state, 12},                  {offsets, (b + int64_t{1}) * 4},
                {positions, positions ? n * 4 : 0}, {slots, slots ? n * 8 : 0}, {workspace, need}};
    for (int i = 0; i < 9; i++)
        for (int j = 0; j < i; j++)
            if (overlaps(all[i].p, all[i].bytes, all[j].p, all[j].bytes)) return fail(HS_EINVAL, "%s: arrays overlap", op);
    PlanArgs a;
    a.counts = static_cast<const int*>(counts), a.lens = static_cast<int*>(lens), a.page_table = static_cast<int*>(page_table);
    a.free = static_cast<int*>(free), a.state = static_cast<int*>(state), a.offsets = static_cast<int*>(offsets);
    a.positions = static_cast<int*>(positions), a.slots = static_cast<int64_t*>(slots), a.plan = static_cast<int4*>(workspace);
    a.n = static_cast<int>(n), a.b = b, a.page_shift = exact_log2(page), a.n_pages = n_pages, a.max_pages = max_pages;
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (need == 0) {
        plan_short_kernel<<<dim3(1), dim3(kPlanThreads), 0, st>>>(a);
        return check_launch(op);
    }
    plan_shares_kernel<<<dim3(1), dim3(kPlanThreads), 0, st>>>(a);
    if (hs_status rc = check_launch(op)) return rc;
    const int64_t entries = ceil_div(b, 4), tokens = positions || slots ? ceil_div(n, 256) : 0;
    if (entries + tokens > 0) plan_rest_kernel<<<dim3(static_cast<uint32_t>(entries + tokens)), dim3(256), 0, st>>>(a, static_cast<int>(entries));
    return check_launch(op);
}
