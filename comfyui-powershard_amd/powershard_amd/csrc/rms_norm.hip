// rms_norm.hip -- RMS norm of x + residual whose rows leave as the int8 / e4m3 operand of the W8A8 and
// fp8 GEMMs (or in 16 bits), ConvRot rotation included.
//
//   h = round16(x + residual), u = 2^-k T(h w), y = u r, r = 1 / sqrt(mean(h^2) + eps)
//   codes = round(y LIM / max|y|), scale = max|y| / LIM
// r > 0 is one number for the row: it cancels out of the codes (y LIM / max|y| = u LIM / max|u|) and
// enters the scale alone, so the row is read once, its sum of squares and its maximum are reduced side
// by side behind one barrier, and the normalized row is never formed.  Codes and rotation are those of
// quantize_rows.hip (same thread layout: a thread owns chunks of 16 consecutive elements, a workgroup
// one row).
#include "quantize.hpp"

namespace psq {
namespace {

constexpr int kChunk = 16;
constexpr int kMaxThreads = 1024;
constexpr int kMaxK = kChunk * kMaxThreads * 2;

// 16 elements as fp32.  ONCE: read once, non-temporally (quantize_rows.hip says what that leaves in the caches).
template <int DT, bool ONCE = false>
__device__ __forceinline__ void load16(const void *p, float (&v)[16])
{
    if constexpr (DT == PSQ_F32) {
        const v4f *f = (const v4f *)p;
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) v[4 * i + j] = f[i][j];
    } else {
        v4i raw[2];
        raw[0] = ONCE ? __builtin_nontemporal_load((const v4i *)p) : ((const v4i *)p)[0];
        raw[1] = ONCE ? __builtin_nontemporal_load((const v4i *)p + 1) : ((const v4i *)p)[1];
        to_f32<DT>(raw, v);
    }
}

template <int DT>
__device__ __forceinline__ void pack16(const float (&v)[16], v4i (&o)[2])
{
#pragma unroll
    for (int i = 0; i < 4; i++) {
        o[0][i] = (int)pack_half2<DT>(v[2 * i], v[2 * i + 1]);
        o[1][i] = (int)pack_half2<DT>(v[8 + 2 * i], v[8 + 2 * i + 1]);
    }
}

struct NormArgs {
    const uint16_t *x, *res;
    const uint8_t *w;
    uint16_t *sum;
    const float *static_scale;
    uint8_t *out;
    float *scale;
    int64_t ldx, ldr, lds, ldo;
    int K, wdt;
    float eps, inv_k;
};

template <int DT, int CODES, int ROTK, int P>
__global__ void __launch_bounds__(kMaxThreads)
add_rms_norm_kernel(NormArgs a)
{
    __shared__ float wave_sum[kMaxThreads / 64];
    __shared__ uint32_t wave_amax[kMaxThreads / 64];
    const int t = threadIdx.x, T = blockDim.x, lc = lane_chunk<ROTK>(t);
    const int64_t row = blockIdx.x;
    constexpr float LIM = CODES == PSQ_CODES_E4M3 ? 448.0f : 127.0f;
    const float post = ROTK ? __builtin_ldexpf(1.0f, -ROTK) : 1.0f;
    float v[P][16];
    float ss = 0.0f, m = 0.0f;
#pragma unroll
    for (int c = 0; c < P; c++) {
        const int e = (c * T + lc) * kChunk;
        float w[16];
        if (e < a.K) {
            load16<DT, true>(a.x + row * a.ldx + e, v[c]);
            if (a.res) {
                float r[16];
                load16<DT, true>(a.res + row * a.ldr + e, r);
#pragma unroll
                for (int j = 0; j < 16; j++) v[c][j] += r[j];
                v4i h[2];
                pack16<DT>(v[c], h);
                ((v4i *)(a.sum + row * a.lds + e))[0] = h[0];
                ((v4i *)(a.sum + row * a.lds + e))[1] = h[1];
                to_f32<DT>(h, v[c]);
            }
            if (a.wdt == PSQ_F32) load16<PSQ_F32>(a.w + 4 * (int64_t)e, w);
            else if (a.wdt == PSQ_F16) load16<PSQ_F16>(a.w + 2 * (int64_t)e, w);
            else load16<PSQ_BF16>(a.w + 2 * (int64_t)e, w);
        } else {
#pragma unroll
            for (int j = 0; j < 16; j++) v[c][j] = w[j] = 0.0f;
        }
#pragma unroll
        for (int j = 0; j < 16; j++) {
            ss = __builtin_fmaf(v[c][j], v[c][j], ss);
            v[c][j] *= w[j];
        }
        rotate16<ROTK>(v[c]);
        m = __builtin_elementwise_maximum(m, absmax16(v[c]));
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) ss += __shfl_xor(ss, o, 64);
    const uint32_t bits = wave_max_bits(__float_as_uint(m));
    if ((t & 63) == 0) {
        wave_sum[t >> 6] = ss;
        wave_amax[t >> 6] = bits;
    }
    __syncthreads();
    float total = 0.0f;
    uint32_t top = 0;
    for (int i = 0; i < T >> 6; i++) {
        total += wave_sum[i];
        top = max(top, wave_amax[i]);
    }
    const float amax = __uint_as_float(top);
    const float r = 1.0f / __builtin_sqrtf(__builtin_fmaf(total, a.inv_k, a.eps));
    const bool zero = amax < zero_below(LIM);
    const float mul = CODES == PSQ_CODES_NONE ? r * post
                      : a.static_scale        ? (r * post) / *a.static_scale
                      : zero                  ? 0.0f
                                              : LIM / amax;
    if (CODES != PSQ_CODES_NONE && t == 0)
        a.scale[row] = a.static_scale ? *a.static_scale : zero ? 1.0f : (amax * (r * post)) / LIM;
#pragma unroll
    for (int c = 0; c < P; c++) {
        if ((c * T + lc) * kChunk >= a.K) continue;
        const int64_t o = row * a.ldo + (int64_t)(c * T + (lc ^ rev_lanes<ROTK>())) * kChunk;
#pragma unroll
        for (int j = 0; j < 16; j++) v[c][j] *= mul;
        if constexpr (CODES == PSQ_CODES_NONE) {
            v4i y[2];
            pack16<DT>(v[c], y);
            ((v4i *)((uint16_t *)a.out + o))[0] = y[0];
            ((v4i *)((uint16_t *)a.out + o))[1] = y[1];
        } else {
            uint32_t q[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float *u = &v[c][4 * i];
                if constexpr (CODES == PSQ_CODES_I8) q[i] = i8_codes4(u[0], u[1], u[2], u[3], kRoundMagic);
                else q[i] = e4m3_codes4(u[0], u[1], u[2], u[3]);
            }
            *(v4i *)(a.out + o) = v4i{(int)q[0], (int)q[1], (int)q[2], (int)q[3]};
        }
    }
}

template <int DT, int CODES, int P>
int launch(const NormArgs &a, int64_t M, int rotk, int threads, hipStream_t st)
{
    const dim3 grid((unsigned)M), block(threads);
    switch (rotk) {
#define PSQ_CASE(RK) case RK: add_rms_norm_kernel<DT, CODES, RK, P><<<grid, block, 0, st>>>(a); break;
        PSQ_CASE(0) PSQ_CASE(1) PSQ_CASE(2) PSQ_CASE(3) PSQ_CASE(4) PSQ_CASE(5)
#undef PSQ_CASE
    default:
        return set_error(PSQ_E_SHAPE, "rotation group 4^%d unsupported", rotk);
    }
    return check_launch("add_rms_norm");
}

template <int DT, int CODES>
int launch_codes(const NormArgs &a, int64_t M, int rotk, hipStream_t st)
{
    const int chunks = a.K / kChunk, P = chunks <= kMaxThreads ? 1 : 2;
    const int threads = ((chunks + P - 1) / P + 63) / 64 * 64;
    return P == 1 ? launch<DT, CODES, 1>(a, M, rotk, threads, st) : launch<DT, CODES, 2>(a, M, rotk, threads, st);
}

}  // namespace
}  // namespace psq

extern "C" int psq_add_rms_norm(int codes, const void *x, int x_dtype, int64_t ldx, const void *residual, int64_t ldr,
                                const void *weight, int weight_dtype, float eps, void *sum, int64_t lds, int rot_group,
                                const float *static_scale, void *out, int64_t ldo, float *scale, int64_t M, int64_t K,
                                void *stream)
{
    using namespace psq;
    const char *name = "add_rms_norm";
    if (codes < PSQ_CODES_NONE || codes > PSQ_CODES_E4M3) return set_error(PSQ_E_ARG, "%s: bad codes %d", name, codes);
    if (M < 0 || K < 0) return set_error(PSQ_E_ARG, "%s: negative size", name);
    if (x_dtype != PSQ_BF16 && x_dtype != PSQ_F16)
        return set_error(PSQ_E_ARG, "%s: rows must be bf16 or f16 (dtype %d)", name, x_dtype);
    if (!valid_dtype(weight_dtype)) return set_error(PSQ_E_ARG, "%s: bad weight dtype %d", name, weight_dtype);
    if (!(eps >= 0.0f)) return set_error(PSQ_E_ARG, "%s: eps must be 0 or more", name);
    if (M == 0) return PSQ_OK;
    if (!x || !weight || !out || (codes != PSQ_CODES_NONE && !scale) || !residual != !sum)
        return set_error(PSQ_E_ARG, "%s: null pointer (a residual comes with a sum)", name);
    if (codes == PSQ_CODES_NONE && static_scale) return set_error(PSQ_E_ARG, "%s: 16-bit rows take no static scale", name);
    if (K == 0 || K % kChunk || K > kMaxK)
        return set_error(PSQ_E_SHAPE, "%s: K=%lld must be a positive multiple of 16 and <= %d", name, (long long)K, kMaxK);
    const int64_t step = codes == PSQ_CODES_NONE ? 8 : 16;
    if (ldx < K || ldx % 8 || ldo < K || ldo % step || (residual && (ldr < K || ldr % 8 || lds < K || lds % 8)))
        return set_error(PSQ_E_SHAPE, "%s: row strides must cover K and be multiples of 8 (codes: 16)", name);
    if (((uintptr_t)x | (uintptr_t)residual | (uintptr_t)sum | (uintptr_t)weight | (uintptr_t)out) & 15)
        return set_error(PSQ_E_SHAPE, "%s: rows and weight must be 16-byte aligned", name);
    if (M > 0x7fffffffLL) return set_error(PSQ_E_SHAPE, "%s: M=%lld too large", name, (long long)M);
    int rotk = 0;
    if (int e = rot_log4(rot_group, K, rotk)) return e;
    if (int e = require_device()) return e;
    const NormArgs a{(const uint16_t *)x, (const uint16_t *)residual, (const uint8_t *)weight, (uint16_t *)sum, static_scale,
                     (uint8_t *)out, scale, ldx, ldr, lds, ldo, (int)K, weight_dtype, eps, 1.0f / (float)K};
    hipStream_t st = (hipStream_t)stream;
    auto go = [&](auto dtc) {
        constexpr int DT = decltype(dtc)::value;
        if (codes == PSQ_CODES_I8) return launch_codes<DT, PSQ_CODES_I8>(a, M, rotk, st);
        if (codes == PSQ_CODES_E4M3) return launch_codes<DT, PSQ_CODES_E4M3>(a, M, rotk, st);
        return launch_codes<DT, PSQ_CODES_NONE>(a, M, rotk, st);
    };
    return x_dtype == PSQ_BF16 ? go(std::integral_constant<int, PSQ_BF16>{}) : go(std::integral_constant<int, PSQ_F16>{});
}
