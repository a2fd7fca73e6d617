// A paged key-value cache for gfx950: appending new tokens (with QK-norm and
// the position rotation) and the attention of one new token per sequence.
#include <math.h>

#include "hs_packed.hpp"

namespace hs {
namespace {

// ---------------------------------------------------------------------------
// kv_append
//
// A head vector is spread over G = D / 2V lanes (V elements per 16-byte load),
// each holding the two chunks [c, c + V) and [D/2 + c, .. + V): a rotation's
// pair sits in one lane and a norm is one G-lane sum of both. A wave takes one
// token and walks its heads, q | k | v one after the other, 64 / G at a time,
// so the token's table rows are read into registers once for all of them.

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
    constexpr int V = Vec<T>::N, G = D / (2 * V), HPW = 64 / G;
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

    const int lane = lane_id();
    const int c = (lane % G) * V;
    float cl[V], ch[V], sl[V], sh[V];
    bool rot = false;
    if constexpr (ROPE) {
        const int row = a.positions ? a.positions[token] : pos;
        rot = row >= 0 && row < a.table_rows;
        if (rot) {
            const float* cr = a.cos_tab + static_cast<int64_t>(row) * D + c;
            const float* sr = a.sin_tab + static_cast<int64_t>(row) * D + c;
#pragma unroll
            for (int e = 0; e < V; e++) cl[e] = cr[e], ch[e] = cr[D / 2 + e], sl[e] = sr[e], sh[e] = sr[D / 2 + e];
        }
    }
    const int part = unit - token * a.parts;
    const int heads = a.h + 2 * a.h_kv;
    for (int j = part * HPW + lane / G; j < heads; j += a.parts * HPW) {
        const bool is_q = j < a.h, is_v = j >= a.h + a.h_kv;
        const int head = is_q ? j : is_v ? j - a.h - a.h_kv : j - a.h;
        const T* src = is_q   ? a.q + static_cast<int64_t>(token) * a.q_stride
                       : is_v ? a.v + static_cast<int64_t>(token) * a.v_stride
                              : a.k + static_cast<int64_t>(token) * a.k_stride;
        src += head * D + c;
        u32x4 lo = ld_stream(src), hi = ld_stream(src + D / 2);
        if ((NORM || ROPE) && !is_v) {
            float x[V], y[V];
            unpack(lo, x, T{});
            unpack(hi, y, T{});
            if constexpr (NORM) {
                const float* w = is_q ? a.qn_w : a.kn_w;
                const float* b = is_q ? a.qn_b : a.kn_b;
                if (w) {
                    float sum = 0.0f;
#pragma unroll
                    for (int e = 0; e < V; e++) sum += x[e] + y[e];
                    const float mean = lanes_sum<G>(sum) * (1.0f / D);
                    float sq = 0.0f;
#pragma unroll
                    for (int e = 0; e < V; e++) {
                        x[e] -= mean, y[e] -= mean;
                        sq = fmaf(x[e], x[e], fmaf(y[e], y[e], sq));
                    }
                    const float inv = rsqrtf(lanes_sum<G>(sq) * (1.0f / D) + a.eps);
#pragma unroll
                    for (int e = 0; e < V; e++) {
                        x[e] = fmaf(x[e] * inv, w[c + e], b[c + e]);
                        y[e] = fmaf(y[e] * inv, w[D / 2 + c + e], b[D / 2 + c + e]);
                    }
                }
            }
            if (rot) {
#pragma unroll
                for (int e = 0; e < V; e++) {
                    const float u = x[e], w = y[e];
                    x[e] = fmaf(u, cl[e], -(w * sl[e]));
                    y[e] = fmaf(w, ch[e], u * sh[e]);
                }
            }
            lo = pack(x, T{});
            hi = pack(y, T{});
        }
        if (is_q) {
            T* dst = a.q_out + (static_cast<int64_t>(token) * a.h + head) * D + c;
            st_stream(dst, lo);
            st_stream(dst + D / 2, hi);
            continue;
        }
        if (placed) {
            T* dst = (is_v ? a.v_cache : a.k_cache) +
                     ((((static_cast<int64_t>(page) * a.h_kv + head) << a.page_shift) + slot) * D + c);
            st_stream(dst, lo);
            st_stream(dst + D / 2, hi);
        }
        if (!is_v && a.k_out) {
            T* dst = a.k_out + (static_cast<int64_t>(token) * a.h_kv + head) * D + c;
            st_stream(dst, lo);
            st_stream(dst + D / 2, hi);
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
// attention_paged: one wave per (sequence, query head), its lanes over the head
// dim, key by key.

template <typename T, int D>
__global__ __launch_bounds__(64) void attention_paged_kernel(
    const T* __restrict__ q, int64_t q_stride, const T* __restrict__ k_cache, const T* __restrict__ v_cache,
    const int* __restrict__ page_table, const int* __restrict__ lens, T* __restrict__ out, int h, int h_kv,
    int page_shift, int n_pages, int max_pages, float scale) {
    constexpr int E = D / 64;
    const int s = blockIdx.x / h, head = blockIdx.x % h, kv = head / (h / h_kv);
    const int lane = lane_id();
    const int64_t len = held_length(lens, s, max_pages, page_shift);
    float qv[E], o[E];
#pragma unroll
    for (int e = 0; e < E; e++)
        qv[e] = static_cast<float>(q[s * q_stride + head * D + lane + 64 * e]) * scale, o[e] = 0.0f;
    float m = -INFINITY, l = 0.0f;
    bool any = false;
    for (int64_t key = 0; key < len; key++) {
        const int page = page_table[static_cast<int64_t>(s) * max_pages + (key >> page_shift)];
        if (page < 0 || page >= n_pages) continue;
        any = true;
        const int64_t at = (((static_cast<int64_t>(page) * h_kv + kv) << page_shift) + (key & ((1 << page_shift) - 1))) * D + lane;
        float dot = 0.0f;
#pragma unroll
        for (int e = 0; e < E; e++) dot = fmaf(qv[e], static_cast<float>(k_cache[at + 64 * e]), dot);
        const float score = wave_sum(dot);
        const float m_new = fmaxf(m, score);
        const float ref = m_new == -INFINITY ? 0.0f : m_new;
        const float corr = expf(m - ref), p = expf(score - ref);
        l = l * corr + p;
#pragma unroll
        for (int e = 0; e < E; e++) o[e] = o[e] * corr + p * static_cast<float>(v_cache[at + 64 * e]);
        m = m_new;
    }
#pragma unroll
    for (int e = 0; e < E; e++)
        out[(static_cast<int64_t>(s) * h + head) * D + lane + 64 * e] = static_cast<T>(any ? o[e] / l : 0.0f);
}

hs_status check_cache(const char* op, const void* k_cache, const void* v_cache, const void* page_table,
                      const void* lens, int32_t page, int32_t n_pages, int32_t max_pages, int32_t h_kv, int32_t d) {
    if (page <= 0 || n_pages < 0 || max_pages < 0) return fail(HS_EINVAL, "%s: page %d, n_pages %d, max_pages %d", op, page, n_pages, max_pages);
    if (exact_log2(page) < 0) return fail(HS_EUNSUPPORTED, "%s: page %d is no power of two", op, page);
    if (static_cast<int64_t>(max_pages) * page >= (int64_t{1} << 31)) return fail(HS_EINVAL, "%s: max_pages * page must be below 2^31", op);
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
    if (n >= (int64_t{1} << 31) / heads) return fail(HS_EINVAL, "%s: n * (Hq + 2 Hkv) must be below 2^31", op);
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
        a.parts = 1;
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
    if (b <= 0 || h <= 0 || h_kv <= 0 || h % h_kv != 0 || (d != 64 && d != 128)) return 0;
    return 0;
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
    if (static_cast<int64_t>(b) * h >= (int64_t{1} << 24)) return fail(HS_EINVAL, "%s: b * Hq must be below 2^24", op);
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
    const auto run = [&](auto zero) {
        using T = decltype(zero);
        const dim3 grid(static_cast<uint32_t>(b * h));
        const auto go = [&](auto kernel) {
            kernel<<<grid, dim3(64), 0, static_cast<hipStream_t>(stream)>>>(
                static_cast<const T*>(q), q_stride, static_cast<const T*>(k_cache), static_cast<const T*>(v_cache),
                static_cast<const int*>(page_table), static_cast<const int*>(lens), static_cast<T*>(out), h, h_kv,
                exact_log2(page), n_pages, max_pages, scale);
        };
        if (d == 64)
            go(attention_paged_kernel<T, 64>);
        else
            go(attention_paged_kernel<T, 128>);
    };
    if (dt == HS_F16)
        run(f16{});
    else
        run(float{});
    return check_launch(op);
}
