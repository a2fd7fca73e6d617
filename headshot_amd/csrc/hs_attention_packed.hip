// Attention of packed sequences for gfx950: whole prompts of different lengths
// in one call, causal by token or by group of tokens, query heads sharing key
// heads.
#include <math.h>

#include "hs_packed.hpp"

namespace hs {
namespace {

// One wave per (query row, head), its lanes over the head dim, key by key.
template <typename T, int D>
__global__ __launch_bounds__(64) void attention_packed_kernel(
    const T* __restrict__ q, int64_t q_stride, const T* __restrict__ k, int64_t k_stride, const T* __restrict__ v,
    int64_t v_stride, const int* __restrict__ q_off, const int* __restrict__ k_off, T* __restrict__ out, int n_q,
    int n_k, int b, int h, int h_kv, int causal, float scale) {
    constexpr int E = D / 64;
    const int row = blockIdx.x / h, head = blockIdx.x % h, kv = head / (h / h_kv);
    const int lane = lane_id();
    const int s = sequence_of(q_off, b, row);
    if (s < 0) return;
    const RowRange qr = row_range(q_off, s, n_q), kr = row_range(k_off, s, n_k);
    const int nk = kr.end - kr.begin;
    const int at = row - qr.begin + nk - (qr.end - qr.begin);
    int seen = nk;
    if (causal > 0) seen = at < 0 ? 0 : static_cast<int>(min<int64_t>(nk, (static_cast<int64_t>(at / causal) + 1) * causal));
    float qv[E], o[E];
#pragma unroll
    for (int e = 0; e < E; e++)
        qv[e] = static_cast<float>(q[row * q_stride + head * D + lane + 64 * e]) * scale, o[e] = 0.0f;
    float m = -INFINITY, l = 0.0f;
    for (int key = 0; key < seen; key++) {
        const T* kp = k + (kr.begin + key) * k_stride + kv * D + lane;
        const T* vp = v + (kr.begin + key) * v_stride + kv * D + lane;
        float dot = 0.0f;
#pragma unroll
        for (int e = 0; e < E; e++) dot = fmaf(qv[e], static_cast<float>(kp[64 * e]), dot);
        const float score = wave_sum(dot);
        const float m_new = fmaxf(m, score);
        const float ref = m_new == -INFINITY ? 0.0f : m_new;
        const float corr = expf(m - ref), p = expf(score - ref);
        l = l * corr + p;
#pragma unroll
        for (int e = 0; e < E; e++) o[e] = o[e] * corr + p * static_cast<float>(vp[64 * e]);
        m = m_new;
    }
#pragma unroll
    for (int e = 0; e < E; e++)
        out[(static_cast<int64_t>(row) * h + head) * D + lane + 64 * e] = static_cast<T>(seen > 0 ? o[e] / l : 0.0f);
}

}  // namespace
}  // namespace hs

extern "C" hs_status hs_attention_packed(hs_stream_t stream, hs_dtype dt, const void* q, int64_t q_stride,
                                         const void* k, int64_t k_stride, const void* v, int64_t v_stride,
                                         const void* q_offsets, const void* k_offsets, void* out, int64_t n_q,
                                         int64_t n_k, int32_t b, int32_t h, int32_t h_kv, int32_t d, int32_t causal,
                                         float scale) {
    using namespace hs;
    const char* op = "attention_packed";
    if (hs_status rc = check_heads(op, dt, h, h_kv, d)) return rc;
    if (n_q < 0 || n_k < 0 || b < 0) return fail(HS_EINVAL, "%s: negative count", op);
    if (causal < 0) return fail(HS_EINVAL, "%s: causal %d", op, causal);
    if (!k_offsets && n_q != n_k) return fail(HS_EINVAL, "%s: without k_offsets, as many keys as queries", op);
    if (n_q == 0 || b == 0 || h == 0) return HS_OK;
    if (n_k >= (int64_t{1} << 31) || n_q >= (int64_t{1} << 31) / h)
        return fail(HS_EINVAL, "%s: n_q * Hq and n_k must be below 2^31", op);
    const int64_t width = static_cast<int64_t>(h) * d, kv_width = static_cast<int64_t>(h_kv) * d;
    if (hs_status rc = check_rows(op, "q", q, n_q, q_stride, width, dt)) return rc;
    if (hs_status rc = check_rows(op, "k", k, n_k, k_stride, kv_width, dt)) return rc;
    if (hs_status rc = check_rows(op, "v", v, n_k, v_stride, kv_width, dt)) return rc;
    if (!out || !q_offsets) return fail(HS_EINVAL, "%s: null out or q_offsets", op);
    if (!aligned16(out)) return fail(HS_EUNSUPPORTED, "%s: out must be 16-byte aligned", op);
    const int64_t out_bytes = n_q * width * dtype_size(dt);
    if (overlaps(out, out_bytes, q, row_bytes(n_q, q_stride, width, dt)) ||
        overlaps(out, out_bytes, k, row_bytes(n_k, k_stride, kv_width, dt)) ||
        overlaps(out, out_bytes, v, row_bytes(n_k, v_stride, kv_width, dt)))
        return fail(HS_EINVAL, "%s: out overlaps an input", op);
    const auto run = [&](auto zero) {
        using T = decltype(zero);
        const dim3 grid(static_cast<uint32_t>(n_q * h));
        const auto go = [&](auto kernel) {
            kernel<<<grid, dim3(64), 0, static_cast<hipStream_t>(stream)>>>(
                static_cast<const T*>(q), q_stride, static_cast<const T*>(k), k_stride, static_cast<const T*>(v),
                v_stride, static_cast<const int*>(q_offsets),
                static_cast<const int*>(k_offsets ? k_offsets : q_offsets), static_cast<T*>(out),
                static_cast<int>(n_q), static_cast<int>(n_k), b, h, h_kv, causal, scale);
        };
        if (d == 64)
            go(attention_packed_kernel<T, 64>);
        else
            go(attention_packed_kernel<T, 128>);
    };
    if (dt == HS_F16)
        run(f16{});
    else
        run(float{});
    return check_launch(op);
}
