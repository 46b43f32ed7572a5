// kv_cache.hip -- a paged key-value cache, quantized as it is written, and its read-back.
//
//   write: scale = max|row| / LIM, codes = round(row LIM / max|row|) per token and head (D elements)
//   read:  round_out(code scale)
// Bound by memory: 2 bytes in, 1 out per element written, 1 in and 2 out per element read.  A lane has 16
// elements of a row's key and of its value (16 bytes of codes each; their place in the pool is worked out
// once for both, in 32 bits), a row the D / 16 lanes next to each other, so its maximum is a few
// cross-lane steps and nothing goes through LDS.
#include "kv_cache.hpp"

namespace psq {
namespace {

constexpr int kThreads = 256;

struct KvArgs {
    const uint16_t *k, *v;
    int64_t k_token, k_head, v_token, v_head;
    const int64_t *slots;
    uint8_t *kc, *vc;
    float *ks, *vs;
    int64_t T, nslots;
    int H, D, page;
};

// L lanes per row (the power of two that covers D / 16), rows = (token, head)
template <int DT, int CODES, int L>
__global__ void __launch_bounds__(kThreads)
kv_write_kernel(KvArgs a)
{
    constexpr float LIM = CODES == PSQ_CODES_E4M3 ? 448.0f : 127.0f;
    const uint32_t r = blockIdx.x * (kThreads / L) + threadIdx.x / L, t = r / (uint32_t)a.H, h = r - t * a.H;
    const int e = (threadIdx.x & (L - 1)) * 16;
    if (t >= a.T) return;   // all lanes of a row leave together
    const int64_t s = a.slots[t];
    if (s < 0 || s >= a.nslots) return;
    const int64_t at = pool_row(s, h, a.H, a.page);
    const uint16_t *k = a.k + t * a.k_token + h * a.k_head + e, *v = a.v + t * a.v_token + h * a.v_head + e;
    const bool here = e < a.D;
    if constexpr (CODES == PSQ_CODES_NONE) {
        if (!here) return;
        v4i *kc = (v4i *)((uint16_t *)a.kc + at * a.D + e), *vc = (v4i *)((uint16_t *)a.vc + at * a.D + e);
        const v4i k0 = ((const v4i *)k)[0], k1 = ((const v4i *)k)[1], v0 = ((const v4i *)v)[0], v1 = ((const v4i *)v)[1];
        kc[0] = k0, kc[1] = k1, vc[0] = v0, vc[1] = v1;
    } else {
        float fk[16] = {}, fv[16] = {};
        if (here) {
            load16<DT>(k, fk);
            load16<DT>(v, fv);
        }
        float mk = absmax16(fk), mv = absmax16(fv);
#pragma unroll
        for (int o = 1; o < L; o <<= 1) {
            mk = __builtin_elementwise_maximum(mk, __shfl_xor(mk, o, 64));
            mv = __builtin_elementwise_maximum(mv, __shfl_xor(mv, o, 64));
        }
        const bool zk = mk < zero_below(LIM), zv = mv < zero_below(LIM);
        const v4i qk = codes16<CODES>(fk, zk ? 0.0f : LIM / mk), qv = codes16<CODES>(fv, zv ? 0.0f : LIM / mv);
        if (here) {
            *(v4i *)(a.kc + at * a.D + e) = qk;
            *(v4i *)(a.vc + at * a.D + e) = qv;
        }
        if (e == 0) {
            a.ks[at] = zk ? 1.0f : mk / LIM;
            a.vs[at] = zv ? 1.0f : mv / LIM;
        }
    }
}

// 16 elements of a pool's row as fp32
template <int DT, int CODES>
__device__ __forceinline__ void row16(const uint8_t *pool, const float *scale, int64_t at, int D, int e, float (&f)[16])
{
    if constexpr (CODES == PSQ_CODES_NONE) {
        load16<DT>((const uint16_t *)pool + at * D + e, f);
    } else {
        // read once: kept out of the caches, which then hold the rows written (65489 x 8 x 128 93 -> 83 us;
        // non-temporal stores as well: 125)
        const v4i q = __builtin_nontemporal_load((const v4i *)(pool + at * D + e));
        const float s = scale[at];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t w = (uint32_t)q[i];
            float x[4];
            if constexpr (CODES == PSQ_CODES_I8) {
#pragma unroll
                for (int j = 0; j < 4; j++) x[j] = (float)(int8_t)(w >> (8 * j));
            } else {
                const f32x2_t lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
                x[0] = lo[0], x[1] = lo[1], x[2] = hi[0], x[3] = hi[1];
            }
#pragma unroll
            for (int j = 0; j < 4; j++) f[4 * i + j] = x[j] * s;
        }
    }
}

template <int OUT>
__device__ __forceinline__ void store16(void *out, int64_t o, const float (&f)[16])
{
    if constexpr (OUT == PSQ_F32) {
#pragma unroll
        for (int i = 0; i < 4; i++) ((v4f *)((float *)out + o))[i] = v4f{f[4 * i], f[4 * i + 1], f[4 * i + 2], f[4 * i + 3]};
    } else {
#pragma unroll
        for (int i = 0; i < 2; i++)
            ((v4i *)((uint16_t *)out + o))[i] =
                v4i{(int)pack_half2<OUT>(f[8 * i], f[8 * i + 1]), (int)pack_half2<OUT>(f[8 * i + 2], f[8 * i + 3]),
                    (int)pack_half2<OUT>(f[8 * i + 4], f[8 * i + 5]), (int)pack_half2<OUT>(f[8 * i + 6], f[8 * i + 7])};
    }
}

template <int DT, int CODES, int OUT>
__global__ void __launch_bounds__(kThreads)
kv_read_kernel(KvArgs a, void *k, void *v)
{
    const uint32_t per = (uint32_t)a.D / 16, i = blockIdx.x * kThreads + threadIdx.x;
    const uint32_t r = i / per, t = r / (uint32_t)a.H, h = r - t * a.H;
    const int e = (int)(i - r * per) * 16;
    if (t >= a.T) return;
    const int64_t s = a.slots[t];
    float fk[16] = {}, fv[16] = {};
    if (s >= 0 && s < a.nslots) {
        const int64_t at = pool_row(s, h, a.H, a.page);
        row16<DT, CODES>(a.kc, a.ks, at, a.D, e, fk);
        row16<DT, CODES>(a.vc, a.vs, at, a.D, e, fv);
    }
    store16<OUT>(k, (int64_t)r * a.D + e, fk);
    store16<OUT>(v, (int64_t)r * a.D + e, fv);
}

template <int DT, int CODES>
int launch_write(const KvArgs &a, hipStream_t st)
{
    const int need = a.D / 16, L = need <= 1 ? 1 : need <= 2 ? 2 : need <= 4 ? 4 : need <= 8 ? 8 : 16;
    const unsigned grid = (unsigned)((a.T * a.H * L + kThreads - 1) / kThreads);
    switch (L) {
#define PSQ_CASE(N) case N: kv_write_kernel<DT, CODES, N><<<grid, kThreads, 0, st>>>(a); break;
        PSQ_CASE(1) PSQ_CASE(2) PSQ_CASE(4) PSQ_CASE(8) PSQ_CASE(16)
#undef PSQ_CASE
    }
    return check_launch("kv_write");
}

}  // namespace
}  // namespace psq

extern "C" {

int psq_kv_write(int codes, const void *k, const void *v, int dtype, int64_t k_token, int64_t k_head, int64_t v_token,
                 int64_t v_head, const int64_t *slots, int64_t T, int Hkv, int D, void *k_cache, void *v_cache,
                 float *k_scale, float *v_scale, int64_t num_pages, int page_size, void *stream)
{
    using namespace psq;
    const char *name = "kv_write";
    if (T < 0) return set_error(PSQ_E_ARG, "%s: negative size", name);
    if (dtype != PSQ_BF16 && dtype != PSQ_F16) return set_error(PSQ_E_ARG, "%s: rows must be bf16 or f16 (dtype %d)", name, dtype);
    if (int e = check_kv_cache(name, codes, k_cache, v_cache, k_scale, v_scale, num_pages, page_size, Hkv, D)) return e;
    if (T == 0 || num_pages == 0) return PSQ_OK;
    if (!k || !v || !slots) return set_error(PSQ_E_ARG, "%s: null pointer", name);
    if (((uintptr_t)k | (uintptr_t)v) & 15 || ((uintptr_t)slots & 7) || (k_token | k_head | v_token | v_head) & 7)
        return set_error(PSQ_E_SHAPE, "%s: rows must be 16-byte aligned, their strides multiples of 8", name);
    if (T > 0x0fffffffLL || T * Hkv > 0x0fffffffLL)   // (32-bit thread numbers, 16 a row at most)
        return set_error(PSQ_E_SHAPE, "%s: T=%lld too large", name, (long long)T);
    if (int e = require_device()) return e;
    const KvArgs a{(const uint16_t *)k, (const uint16_t *)v, k_token, k_head, v_token, v_head, slots, (uint8_t *)k_cache,
                   (uint8_t *)v_cache, k_scale, v_scale, T, num_pages * page_size, Hkv, D, page_size};
    hipStream_t st = (hipStream_t)stream;
    if (codes == PSQ_CODES_NONE) return launch_write<PSQ_BF16, PSQ_CODES_NONE>(a, st);
    if (codes == PSQ_CODES_I8)
        return dtype == PSQ_BF16 ? launch_write<PSQ_BF16, PSQ_CODES_I8>(a, st) : launch_write<PSQ_F16, PSQ_CODES_I8>(a, st);
    return dtype == PSQ_BF16 ? launch_write<PSQ_BF16, PSQ_CODES_E4M3>(a, st) : launch_write<PSQ_F16, PSQ_CODES_E4M3>(a, st);
}

int psq_kv_read(int codes, const int64_t *slots, int64_t T, const void *k_cache, const void *v_cache, int cache_dtype,
                const float *k_scale, const float *v_scale, int64_t num_pages, int page_size, int Hkv, int D, void *k, void *v,
                int out_dtype, void *stream)
{
    using namespace psq;
    const char *name = "kv_read";
    if (T < 0) return set_error(PSQ_E_ARG, "%s: negative size", name);
    if (!valid_dtype(out_dtype)) return set_error(PSQ_E_ARG, "%s: bad output dtype %d", name, out_dtype);
    if (int e = check_kv_cache(name, codes, k_cache, v_cache, k_scale, v_scale, num_pages, page_size, Hkv, D)) return e;
    if (codes == PSQ_CODES_NONE && cache_dtype != PSQ_BF16 && cache_dtype != PSQ_F16)
        return set_error(PSQ_E_ARG, "%s: the cache must be bf16 or f16 (dtype %d)", name, cache_dtype);
    if (T == 0) return PSQ_OK;
    if (!k || !v || !slots) return set_error(PSQ_E_ARG, "%s: null pointer", name);
    if (((uintptr_t)k | (uintptr_t)v) & 15 || ((uintptr_t)slots & 7))
        return set_error(PSQ_E_SHAPE, "%s: rows must be 16-byte aligned", name);
    if (T > 0x0fffffffLL || T * Hkv > 0x0fffffffLL)   // (32-bit thread numbers, 16 a row at most)
        return set_error(PSQ_E_SHAPE, "%s: T=%lld too large", name, (long long)T);
    if (int e = require_device()) return e;
    const KvArgs a{nullptr, nullptr, 0, 0, 0, 0, slots, (uint8_t *)k_cache, (uint8_t *)v_cache, (float *)k_scale,
                   (float *)v_scale, T, num_pages * page_size, Hkv, D, page_size};
    hipStream_t st = (hipStream_t)stream;
    const unsigned grid = (unsigned)((T * Hkv * (D / 16) + kThreads - 1) / kThreads);
    auto out = [&](auto dtc, auto cc) {
        constexpr int DT = decltype(dtc)::value, C = decltype(cc)::value;
        if (out_dtype == PSQ_BF16) kv_read_kernel<DT, C, PSQ_BF16><<<grid, kThreads, 0, st>>>(a, k, v);
        else if (out_dtype == PSQ_F16) kv_read_kernel<DT, C, PSQ_F16><<<grid, kThreads, 0, st>>>(a, k, v);
        else kv_read_kernel<DT, C, PSQ_F32><<<grid, kThreads, 0, st>>>(a, k, v);
        return check_launch(name);
    };
    using BF = std::integral_constant<int, PSQ_BF16>;
    using HF = std::integral_constant<int, PSQ_F16>;
    if (codes == PSQ_CODES_I8) return out(BF{}, std::integral_constant<int, PSQ_CODES_I8>{});
    if (codes == PSQ_CODES_E4M3) return out(BF{}, std::integral_constant<int, PSQ_CODES_E4M3>{});
    if (cache_dtype == PSQ_BF16) return out(BF{}, std::integral_constant<int, PSQ_CODES_NONE>{});
    return out(HF{}, std::integral_constant<int, PSQ_CODES_NONE>{});
}

}  // extern "C"
