// kv_cache.hpp -- what the paged cache's kernels share: its shape, rows of 16 elements, codes.
#pragma once

#include "quantize.hpp"

namespace psq {

// 16 elements of DT (16-byte aligned) as fp32
template <int DT>
__device__ __forceinline__ void load16(const uint16_t *p, float (&f)[16])
{
    const v4i raw[2] = {((const v4i *)p)[0], ((const v4i *)p)[1]};
    to_f32<DT>(raw, f);
}

// row of the pools that slot s of head h occupies
__device__ __forceinline__ int64_t pool_row(int64_t s, uint32_t h, int heads, int page)
{
    const int64_t p = s >> 32 ? s / page : (int64_t)((uint32_t)s / (uint32_t)page);
    return (p * heads + h) * page + (s - p * page);
}

// 16 codes of f at mul
template <int CODES>
__device__ __forceinline__ v4i codes16(const float (&f)[16], float mul)
{
    v4i q;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float u0 = f[4 * i] * mul, u1 = f[4 * i + 1] * mul, u2 = f[4 * i + 2] * mul, u3 = f[4 * i + 3] * mul;
        if constexpr (CODES == PSQ_CODES_I8) q[i] = (int)i8_codes4(u0, u1, u2, u3, kRoundMagic);
        else q[i] = (int)e4m3_codes4(u0, u1, u2, u3);
    }
    return q;
}

// Two fp32 values whose low 16 bits are zero as a packed bf16 pair.
__device__ __forceinline__ uint32_t pack_exact_bf16(float lo, float hi)
{
    return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
}

template <int B>
__device__ __forceinline__ float i8_byte_f32(uint32_t w)
{
    float f;
    if constexpr (B == 0)
        asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_0" : "=v"(f) : "v"(w));
    else if constexpr (B == 1)
        asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_1" : "=v"(f) : "v"(w));
    else if constexpr (B == 2)
        asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_2" : "=v"(f) : "v"(w));
    else
        asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_3" : "=v"(f) : "v"(w));
    return f;
}

// Bytes 2 H and 2 H + 1 of w, codes, as a packed pair of DT.
template <int DT, int CODES, int H>
__device__ __forceinline__ uint32_t code_pair(uint32_t w)
{
    if constexpr (CODES == PSQ_CODES_E4M3) {
        if constexpr (DT == PSQ_BF16)
            return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w, 1.0f, H != 0));
        else
            return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.0f, H != 0));
    } else if constexpr (DT == PSQ_BF16) {
        return pack_exact_bf16(i8_byte_f32<2 * H>(w), i8_byte_f32<2 * H + 1>(w));
    } else {
        // the biased byte under the f16 exponent of 1024 is 1152 + q (integers to 2048 are exact)
        const uint32_t h = __builtin_amdgcn_perm(0x64646464u, w ^ 0x80808080u, H ? 0x04030402u : 0x04010400u);
        const f16x2_t q = __builtin_bit_cast(f16x2_t, h) - f16x2_t{(_Float16)1152.0f, (_Float16)1152.0f};
        return __builtin_bit_cast(uint32_t, q);
    }
}

// host checks of the pools: sizes, alignment, scales present exactly with codes
inline int check_kv_cache(const char *name, int codes, const void *k_cache, const void *v_cache, const float *k_scale,
                          const float *v_scale, int64_t num_pages, int page_size, int Hkv, int D)
{
    if (codes < PSQ_CODES_NONE || codes > PSQ_CODES_E4M3) return set_error(PSQ_E_ARG, "%s: bad codes %d", name, codes);
    if (num_pages < 0 || page_size <= 0 || Hkv <= 0 || D <= 0) return set_error(PSQ_E_ARG, "%s: bad cache size", name);
    if (num_pages && (!k_cache || !v_cache || (codes != PSQ_CODES_NONE && (!k_scale || !v_scale))))
        return set_error(PSQ_E_ARG, "%s: null pool", name);
    if (D % 16 || D > 256) return set_error(PSQ_E_SHAPE, "%s: head dim %d must be a multiple of 16 in 16..256", name, D);
    if (page_size % 16 || page_size > 65536)
        return set_error(PSQ_E_SHAPE, "%s: page size %d must be a multiple of 16 up to 65536", name, page_size);
    if (Hkv > 65535 || num_pages > 0x7fffffffLL || (int64_t)Hkv * page_size * D > 0x3fffffffLL ||
        num_pages * Hkv * (page_size / 16) > 0x7fffffffLL)
        return set_error(PSQ_E_SHAPE, "%s: a page of %d heads x %d x %d, or %lld pages, is too large", name, Hkv, page_size, D,
                         (long long)num_pages);
    if (((uintptr_t)k_cache | (uintptr_t)v_cache) & 15 || ((uintptr_t)k_scale | (uintptr_t)v_scale) & 15)
        return set_error(PSQ_E_SHAPE, "%s: pools must be 16-byte aligned", name);
    return PSQ_OK;
}

}  // namespace psq
