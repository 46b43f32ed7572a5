// kv_cache.hpp -- what the paged cache's kernels share: its shape.
#pragma once

#include "quantize.hpp"

namespace psq {

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
