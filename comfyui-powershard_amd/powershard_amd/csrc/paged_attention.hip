// paged_attention.hip -- attention of one new token per sequence over the paged key-value cache.
//
// The plain kernel: a workgroup per sequence and head, 256 tokens at a time, with the running maximum
// and sum of the softmax.
#include "kv_cache.hpp"

#include <math.h>

namespace psq {
namespace {

constexpr int kThreads = 256;

struct AttnArgs {
    const uint16_t *q;
    int64_t q_batch, q_head;
    const uint8_t *kc, *vc;
    const float *ks, *vs;
    int64_t num_pages;
    const int32_t *table;
    int64_t table_stride, table_cols;
    const int32_t *lengths;
    uint16_t *out;
    float *lse;
    int64_t window;
    int page, Hq, Hkv, D;
    float scale;
};

template <int DT, int CODES>
__device__ __forceinline__ float cache_elem(const uint8_t *pool, int64_t i)
{
    if constexpr (CODES == PSQ_CODES_I8) return (float)(int8_t)pool[i];
    else if constexpr (CODES == PSQ_CODES_E4M3) return e4m3_to_f32(pool[i]);
    else return half_to_f32<DT>(((const uint16_t *)pool)[i]);
}

template <int DT, int CODES>
__global__ void __launch_bounds__(kThreads)
paged_attention_kernel(AttnArgs a)
{
    __shared__ float q[256], p[kThreads], red[2];
    __shared__ int64_t rows[kThreads];
    const int tid = threadIdx.x, h = blockIdx.x, b = blockIdx.y, hk = h / (a.Hq / a.Hkv);
    if (tid < a.D) q[tid] = half_to_f32<DT>(a.q[b * a.q_batch + h * a.q_head + tid]);
    const int64_t cap = a.table_cols * a.page;
    int64_t len = max(a.lengths[b], 0);
    bool bad = len > cap;
    len = min(len, cap);
    int64_t t0 = a.window > 0 ? max((int64_t)0, len - a.window) : 0;
    float m = -INFINITY, l = 0.0f, o = 0.0f;
    for (; t0 < len; t0 += kThreads) {
        const int n = (int)min((int64_t)kThreads, len - t0);
        float s = -INFINITY;
        __syncthreads();
        if (tid < n) {
            const int64_t t = t0 + tid;
            int64_t pg = a.table[b * a.table_stride + t / a.page];
            if (pg < 0 || pg >= a.num_pages) pg = -1;
            rows[tid] = pg < 0 ? -1 : (pg * a.Hkv + hk) * a.page + t % a.page;
            if (pg >= 0) {
                float dot = 0.0f;
                for (int d = 0; d < a.D; d++) dot += q[d] * cache_elem<DT, CODES>(a.kc, rows[tid] * a.D + d);
                s = dot * a.scale * (CODES == PSQ_CODES_NONE ? 1.0f : a.ks[rows[tid]]);
            } else {
                s = NAN;
            }
        }
        p[tid] = s;
        __syncthreads();
        if (tid == 0) {
            float top = m;
            for (int i = 0; i < n; i++) top = __builtin_elementwise_maximum(top, p[i]);
            red[0] = top;
        }
        __syncthreads();
        const float top = red[0], base = top == -INFINITY ? 0.0f : top;
        p[tid] = tid < n ? expf(s - base) : 0.0f;
        __syncthreads();
        const float keep = expf(m - base);
        l *= keep;
        o *= keep;
        m = top;
        for (int i = 0; i < n; i++) {
            l += p[i];
            if (tid < a.D && rows[i] >= 0)
                o += p[i] * (CODES == PSQ_CODES_NONE ? 1.0f : a.vs[rows[i]]) * cache_elem<DT, CODES>(a.vc, rows[i] * a.D + tid);
        }
    }
    float y = len == 0 ? 0.0f : o / l;
    if (bad) y = NAN;
    if (tid < a.D) a.out[((int64_t)b * a.Hq + h) * a.D + tid] = (uint16_t)f32_to_half<DT>(y);
    if (a.lse && tid == 0) a.lse[(int64_t)b * a.Hq + h] = bad ? NAN : m + logf(l);
}

}  // namespace
}  // namespace psq

extern "C" {

int64_t psq_paged_attention_workspace_bytes(int codes, int64_t B, int Hq, int Hkv, int D, int64_t max_len)
{
    (void)codes, (void)B, (void)Hq, (void)Hkv, (void)D, (void)max_len;
    return 0;
}

int psq_paged_attention(int codes, const void *q, int dtype, int64_t q_batch, int64_t q_head, const void *k_cache,
                        const void *v_cache, const float *k_scale, const float *v_scale, int64_t num_pages, int page_size,
                        const int32_t *block_table, int64_t table_stride, int64_t table_cols, const int32_t *lengths, int64_t B,
                        int Hq, int Hkv, int D, float scale, int64_t window, int64_t max_len, void *out, float *lse,
                        void *workspace, int64_t workspace_bytes, void *stream)
{
    using namespace psq;
    const char *name = "paged_attention";
    if (B < 0 || Hq < 0 || table_cols < 0 || window < 0 || max_len < 0 || workspace_bytes < 0)
        return set_error(PSQ_E_ARG, "%s: negative size", name);
    if (dtype != PSQ_BF16 && dtype != PSQ_F16) return set_error(PSQ_E_ARG, "%s: queries must be bf16 or f16 (dtype %d)", name, dtype);
    if (int e = check_kv_cache(name, codes, k_cache, v_cache, k_scale, v_scale, num_pages, page_size, Hkv, D)) return e;
    if (B == 0 || Hq == 0) return PSQ_OK;
    if (!q || !out || !lengths || (table_cols && !block_table)) return set_error(PSQ_E_ARG, "%s: null pointer", name);
    if (Hq % Hkv || Hq > 65535) return set_error(PSQ_E_SHAPE, "%s: %d heads do not share %d kv heads", name, Hq, Hkv);
    if (((uintptr_t)q | (uintptr_t)out) & 15 || (q_batch | q_head) & 7)
        return set_error(PSQ_E_SHAPE, "%s: queries and output must be 16-byte aligned, query strides multiples of 8", name);
    if (((uintptr_t)block_table | (uintptr_t)lengths | (uintptr_t)lse) & 3)
        return set_error(PSQ_E_SHAPE, "%s: misaligned table, lengths or lse", name);
    if (B > 65535 || table_cols > 0x7fffffffLL / page_size)
        return set_error(PSQ_E_SHAPE, "%s: %lld sequences of %lld pages are too many", name, (long long)B,
                         (long long)table_cols);
    (void)workspace, (void)max_len;
    if (int e = require_device()) return e;
    const AttnArgs a{(const uint16_t *)q, q_batch, q_head, (const uint8_t *)k_cache, (const uint8_t *)v_cache, k_scale, v_scale,
                     num_pages, block_table, table_stride, table_cols, lengths, (uint16_t *)out, lse, window, page_size, Hq, Hkv,
                     D, scale};
    hipStream_t st = (hipStream_t)stream;
    const dim3 grid((unsigned)Hq, (unsigned)B);
    auto go = [&](auto dtc) {
        constexpr int DT = decltype(dtc)::value;
        if (codes == PSQ_CODES_I8) paged_attention_kernel<DT, PSQ_CODES_I8><<<grid, kThreads, 0, st>>>(a);
        else if (codes == PSQ_CODES_E4M3) paged_attention_kernel<DT, PSQ_CODES_E4M3><<<grid, kThreads, 0, st>>>(a);
        else paged_attention_kernel<DT, PSQ_CODES_NONE><<<grid, kThreads, 0, st>>>(a);
        return check_launch(name);
    };
    return dtype == PSQ_BF16 ? go(std::integral_constant<int, PSQ_BF16>{}) : go(std::integral_constant<int, PSQ_F16>{});
}

}  // extern "C"
