// kv_cache.hip -- a paged key-value cache, quantized as it is written, and its read-back.
//
//   write: scale = max|row| / LIM, codes = round(row LIM / max|row|) per token and head (D elements)
//   read:  round_out(code scale)
// A row belongs to the lanes that hold 8 of its elements each (16-byte loads of the 16-bit side), so its
// maximum is a few cross-lane steps and nothing goes through LDS.  Keys and values go in one launch.
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

// 8 fp32 values of a 16-byte load
template <int DT>
__device__ __forceinline__ void to_f32x8(const v4i &raw, float (&f)[8])
{
#pragma unroll
    for (int i = 0; i < 4; i++) {
        f[2 * i] = half_to_f32<DT>((uint32_t)raw[i]);
        f[2 * i + 1] = half_to_f32<DT>((uint32_t)raw[i] >> 16);
    }
}

// row of the pools that slot s of head h occupies
__device__ __forceinline__ int64_t pool_row(int64_t s, int h, int H, int page)
{
    const int64_t p = s / page;
    return (p * H + h) * page + (s - p * page);
}

// L lanes per row (the power of two that covers D / 8), rows = (token, head)
template <int DT, int CODES, int L>
__global__ void __launch_bounds__(kThreads)
kv_write_kernel(KvArgs a)
{
    constexpr float LIM = CODES == PSQ_CODES_E4M3 ? 448.0f : 127.0f;
    const int64_t r = ((int64_t)blockIdx.x * kThreads + threadIdx.x) / L;
    const int e = (threadIdx.x & (L - 1)) * 8;
    const bool value = blockIdx.y != 0;
    const int64_t t = r / a.H;
    const int h = (int)(r - t * a.H);
    if (t >= a.T) return;   // all lanes of a row leave together
    const int64_t s = a.slots[t];
    if (s < 0 || s >= a.nslots) return;
    const int64_t at = pool_row(s, h, a.H, a.page);
    const uint16_t *src = (value ? a.v + t * a.v_token + h * a.v_head : a.k + t * a.k_token + h * a.k_head) + e;
    v4i raw = {0, 0, 0, 0};
    if (e < a.D) raw = *(const v4i *)src;
    uint8_t *pool = value ? a.vc : a.kc;
    if constexpr (CODES == PSQ_CODES_NONE) {
        if (e < a.D) *(v4i *)((uint16_t *)pool + at * a.D + e) = raw;
    } else {
        float f[8];
        to_f32x8<DT>(raw, f);
        float m = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; j++) m = __builtin_elementwise_maximum(m, __builtin_fabsf(f[j]));
#pragma unroll
        for (int o = 1; o < L; o <<= 1) m = __builtin_elementwise_maximum(m, __shfl_xor(m, o, 64));
        const bool zero = m < kKvTiny;
        const float mul = zero ? 0.0f : LIM / m;
        if (e == 0) (value ? a.vs : a.ks)[at] = zero ? 1.0f : m / LIM;
#pragma unroll
        for (int j = 0; j < 8; j++) f[j] *= mul;
        v2i q;
        if constexpr (CODES == PSQ_CODES_I8)
            q = v2i{(int)i8_codes4(f[0], f[1], f[2], f[3], kRoundMagic), (int)i8_codes4(f[4], f[5], f[6], f[7], kRoundMagic)};
        else
            q = v2i{(int)e4m3_codes4(f[0], f[1], f[2], f[3]), (int)e4m3_codes4(f[4], f[5], f[6], f[7])};
        if (e < a.D) *(v2i *)(pool + at * a.D + e) = q;
    }
}

template <int DT, int CODES, int OUT>
__global__ void __launch_bounds__(kThreads)
kv_read_kernel(KvArgs a, void *k, void *v)
{
    const int per = a.D / 8;
    const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    const int64_t r = i / per;
    const int e = (int)(i - r * per) * 8;
    const bool value = blockIdx.y != 0;
    const int64_t t = r / a.H;
    const int h = (int)(r - t * a.H);
    if (t >= a.T) return;
    const int64_t s = a.slots[t];
    float f[8] = {};
    if (s >= 0 && s < a.nslots) {
        const int64_t at = pool_row(s, h, a.H, a.page);
        const uint8_t *pool = value ? a.vc : a.kc;
        if constexpr (CODES == PSQ_CODES_NONE) {
            to_f32x8<DT>(*(const v4i *)((const uint16_t *)pool + at * a.D + e), f);
        } else {
            const v2i q = *(const v2i *)(pool + at * a.D + e);
            const float scale = (value ? a.vs : a.ks)[at];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const uint32_t c = (uint32_t)q[j >> 2] >> (8 * (j & 3)) & 0xffu;
                f[j] = (CODES == PSQ_CODES_I8 ? (float)(int8_t)c : e4m3_to_f32(c)) * scale;
            }
        }
    }
    const int64_t o = r * a.D + e;
    void *out = value ? v : k;
    if constexpr (OUT == PSQ_F32) {
        ((v4f *)((float *)out + o))[0] = v4f{f[0], f[1], f[2], f[3]};
        ((v4f *)((float *)out + o))[1] = v4f{f[4], f[5], f[6], f[7]};
    } else {
        *(v4i *)((uint16_t *)out + o) = v4i{(int)pack_half2<OUT>(f[0], f[1]), (int)pack_half2<OUT>(f[2], f[3]),
                                           (int)pack_half2<OUT>(f[4], f[5]), (int)pack_half2<OUT>(f[6], f[7])};
    }
}

template <int DT, int CODES>
int launch_write(const KvArgs &a, hipStream_t st)
{
    const int need = a.D / 8;
    const int L = need <= 2 ? 2 : need <= 4 ? 4 : need <= 8 ? 8 : need <= 16 ? 16 : 32;
    const dim3 grid((unsigned)((a.T * a.H * L + kThreads - 1) / kThreads), 2);
    switch (L) {
#define PSQ_CASE(N) case N: kv_write_kernel<DT, CODES, N><<<grid, kThreads, 0, st>>>(a); break;
        PSQ_CASE(2) PSQ_CASE(4) PSQ_CASE(8) PSQ_CASE(16) PSQ_CASE(32)
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
    if (T * Hkv > 0x3fffffffLL || T > 0x3fffffffLL)
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
    if (T * Hkv > 0x3fffffffLL || T > 0x3fffffffLL)
        return set_error(PSQ_E_SHAPE, "%s: T=%lld too large", name, (long long)T);
    if (int e = require_device()) return e;
    const KvArgs a{nullptr, nullptr, 0, 0, 0, 0, slots, (uint8_t *)k_cache, (uint8_t *)v_cache, (float *)k_scale,
                   (float *)v_scale, T, num_pages * page_size, Hkv, D, page_size};
    hipStream_t st = (hipStream_t)stream;
    const dim3 grid((unsigned)((T * Hkv * (D / 8) + kThreads - 1) / kThreads), 2);
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
