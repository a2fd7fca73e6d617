// Pages handed out on the GPU for gfx950: sequences' new lengths become entries of
// the page table, and the positions and places of their new tokens.
//
// Free pages lie in a ring, `count` of them from place `head` on; a call takes from
// its front and gives back behind its end, so that what it reads there and what it
// writes are apart and the two need no order between them. Prefix sums over the
// sequences give each its share: one workgroup makes them, a thread a sequence;
// the entries (a wave a sequence) and the tokens (a thread each) then follow from
// those alone. Latency: a short call is one launch of that workgroup, a long one a
// second launch of many. 256 sequences that move a few tokens each take 5.6 us on
// the device, 64 that admit or drop prompts of up to 8192 tokens 3.0 and 5.3.
#include <climits>

#include "hs_packed.hpp"

namespace hs {
namespace {

constexpr int kPlanThreads = 1024;
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

// Sums over this lane and the ones before it. 64 bits in two parts: 64 times 16 bits
// and 64 times 31 - 16 stay whole.
__device__ __forceinline__ int64_t wave_sums(int64_t v) {
    const int lo = wave_prefix_sum(static_cast<int>(v & 0xFFFF)), hi = wave_prefix_sum(static_cast<int>(v >> 16));
    return (static_cast<int64_t>(hi) << 16) + lo;
}
__device__ __forceinline__ int64_t lane_value64(int64_t v, int lane) {
    const uint32_t lo = lane_value(static_cast<int>(v), lane);
    return (static_cast<int64_t>(lane_value(static_cast<int>(v >> 32), lane)) << 32) | lo;
}

// The sequences' shares, `keep` taking each and its first row; lens, offsets and the
// ring's state as the call leaves them. All threads of the workgroup (W waves) call
// it and get the ring as it was.
template <int W, typename K>
__device__ __forceinline__ Ring make_shares(const PlanArgs& a, K keep) {
    __shared__ int64_t sums[W][4];
    const int lane = lane_id(), wave = wave_in_block();
    Ring ring = {a.state[0], a.state[1]};
    ring.count = min(max(ring.count, 0), a.n_pages);
    ring.head = a.n_pages > 0 && ring.head >= 0 ? ring.head % a.n_pages : 0;
    int64_t before[4] = {0, 0, 0, 0};  // by the sequences before: pages asked for, given back, new tokens, pages wanted
    for (int base = 0; base < a.b; base += 64 * W) {
        const int s = base + static_cast<int>(threadIdx.x);
        Share t = {0, 0, 0, -1, 0};
        int64_t v[4] = {0, 0, 0, 0};
        int after = 0;
        if (s < a.b) {
            const int change = a.counts[s];
            t.old = min(max(a.lens[s], 0), kLongest);
            const int64_t sum = static_cast<int64_t>(t.old) + change;
            after = static_cast<int>(min(max(sum, int64_t{0}), int64_t{kLongest}));
            const int all_have = entries_of(t.old, a.page_shift), all_want = entries_of(after, a.page_shift);
            t.have = min(all_have, a.max_pages), t.want = min(all_want, a.max_pages);
            const int* entries = a.page_table + static_cast<int64_t>(s) * a.max_pages;
            // Entries are pages up to the first that was not there, so the last says
            // whether all are.
            const bool whole = t.have == 0 || is_page(a, entries[t.have - 1]);
            t.end = t.have;
            if (t.want > t.have && whole) v[0] = t.want - t.have;
            if (t.want < t.have) {
                if (!whole) {
                    int lo = t.want, hi = t.have - 1;
                    while (lo < hi) {
                        const int mid = (lo + hi) >> 1;
                        if (is_page(a, entries[mid]))
                            lo = mid + 1;
                        else
                            hi = mid;
                    }
                    t.end = lo;
                }
                v[1] = t.end - t.want;
            }
            v[2] = max(change, 0);
            v[3] = max(all_want - all_have, 0);
        }
        int64_t mine[4];
        mine[0] = wave_prefix_sum(static_cast<int>(v[0])), mine[1] = wave_prefix_sum(static_cast<int>(v[1]));  // below 2^31: the table's entries
        mine[2] = wave_sums(v[2]), mine[3] = wave_sums(v[3]);
        if (lane == 63) {
#pragma unroll
            for (int i = 0; i < 4; i++) sums[wave][i] = mine[i];
        }
        __syncthreads();
        int64_t first[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int64_t total = wave_sums(lane < W ? sums[lane][i] : 0);
            first[i] = before[i] + (wave > 0 ? lane_value64(total, wave - 1) : 0) + mine[i] - v[i];
            before[i] += lane_value64(total, W - 1);
        }
        if (base + 64 * W < a.b) __syncthreads();  // sums are written again
        if (s < a.b) {
            t.taken = static_cast<int>(v[0] > 0 ? first[0] : v[1] > 0 ? first[1] : -1);
            const int row = static_cast<int>(min(first[2], int64_t{INT_MAX})), next = static_cast<int>(min(first[2] + v[2], int64_t{INT_MAX}));
            keep(s, t, next);
            if (s == 0) a.offsets[0] = row;
            a.lens[s] = after;
            a.offsets[s + 1] = next;
        }
    }
    if (threadIdx.x == 0) {
        const int taken = static_cast<int>(min(before[0], static_cast<int64_t>(ring.count)));
        const int given = static_cast<int>(min(before[1], static_cast<int64_t>(a.n_pages - ring.count)));
        if (a.b == 0) a.offsets[0] = 0;
        a.state[0] = a.n_pages > 0 ? (ring.head + taken) % a.n_pages : 0;
        a.state[1] = ring.count - taken + given;
        a.state[2] = static_cast<int>(min(before[3] - taken, int64_t{INT_MAX}));
    }
    return ring;
}

// A sequence's entries, `step` lanes of them at a time, this one the lane-th.
__device__ __forceinline__ void fill_entries(const PlanArgs& a, const Ring& r, int s, const Share& t, int lane, int step) {
    int* entries = a.page_table + static_cast<int64_t>(s) * a.max_pages;
    for (int e = t.have + lane; e < t.want; e += step) entries[e] = page_taken(a, r, t, e);
    for (int e = t.want + lane; e < t.have; e += step) {
        const int64_t at = static_cast<int64_t>(r.count) + t.taken + e - t.want;
        if (e < t.end && at < a.n_pages) *ring_at(a, r, static_cast<int>(at)) = entries[e];
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

// Short calls, of as many sequences as the workgroup has threads. A sequence that
// moves a few pages is its thread's, one of more a wave's.
constexpr int kFewPages = 4;

template <int W>
__global__ __launch_bounds__(64 * W) void plan_short_kernel(PlanArgs a) {
    __shared__ Share shares[64 * W];
    __shared__ int offsets[64 * W + 1];
    const Ring ring = make_shares<W>(a, [&](int s, const Share& t, int next) { shares[s] = t, offsets[s + 1] = next; });
    if (threadIdx.x == 0) offsets[0] = 0;
    __syncthreads();
    const auto moved = [](const Share& t) { return abs(t.want - t.have); };
    const int mine = threadIdx.x;
    const bool many = mine < a.b && moved(shares[mine]) > kFewPages;
    if (mine < a.b && !many) fill_entries(a, ring, mine, shares[mine], 0, 1);
    for (uint64_t left = __ballot(many); left; left &= left - 1) {  // each wave its own threads' sequences
        const int s = wave_in_block() * 64 + __builtin_ctzll(left);
        fill_entries(a, ring, s, shares[s], lane_id(), 64);
    }
    const int rows = min(offsets[a.b], a.n);
    for (int row = threadIdx.x; row < rows; row += 64 * W) {
        int lo = 0, hi = a.b;  // the first sequence that ends behind the row
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (offsets[mid + 1] <= row)
                lo = mid + 1;
            else
                hi = mid;
        }
        place_token(a, ring, lo, shares[lo], row, row - offsets[lo]);
    }
}

__device__ __forceinline__ int4 packed_share(const Share& t) { return {t.old, t.have, t.want, t.taken}; }

__global__ __launch_bounds__(kPlanThreads) void plan_shares_kernel(PlanArgs a) {
    int* ends = reinterpret_cast<int*>(a.plan + a.b + 1);
    const Ring ring = make_shares<kPlanThreads / 64>(a, [&](int s, const Share& t, int) { a.plan[s] = packed_share(t), ends[s] = t.end; });
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
        if (s < a.b) fill_entries(a, ring, s, share(s), lane_id(), 64);
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
        if (b <= 256 && n <= 1024)
            plan_short_kernel<4><<<dim3(1), dim3(256), 0, st>>>(a);
        else
            plan_short_kernel<kPlanThreads / 64><<<dim3(1), dim3(kPlanThreads), 0, st>>>(a);
        return check_launch(op);
    }
    plan_shares_kernel<<<dim3(1), dim3(kPlanThreads), 0, st>>>(a);
    if (hs_status rc = check_launch(op)) return rc;
    const int64_t entries = ceil_div(b, 4), tokens = positions || slots ? ceil_div(n, 256) : 0;
    if (entries + tokens > 0) plan_rest_kernel<<<dim3(static_cast<uint32_t>(entries + tokens)), dim3(256), 0, st>>>(a, static_cast<int>(entries));
    return check_launch(op);
}
