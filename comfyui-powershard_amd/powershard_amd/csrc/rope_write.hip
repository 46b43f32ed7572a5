// rope_write.hip -- new tokens' queries and keys turned to their positions, keys and values appended to the
// paged key-value cache, quantized on the way.
//
//   t = position[axis(i)] f_i;  a' = a cos t - b sin t,  b' = b cos t + a sin t  for pair i = (a, b)
//   q: rounded to its type; k, v: codes and scales as in kv_cache.hip, k's from the turned values in fp32
// Bound by memory: queries 2 bytes in and 2 out per element, keys and values 2 in and 1 or 2 out.
// 8191 tokens, 40 heads on 8 of 128, e4m3, with the read-back: 60.8 us, 4.4 TB/s (a large copy: 4.75); 4095 tokens, 64 heads on 16
// of 64, three axes, f16, likewise: 30.2 us, 4.45 TB/s; one token: 12 us for both calls, the host's part (kernels 3.6 + 2.5).
// A lane has 16 elements of a row: its 8 pairs, where it turns (the two pieces of 8 elements that are half
// the rotary dims apart, or 16 neighbours where pairs are neighbours), else 16 neighbours.  A row is the
// D / 16 lanes next to each other.  The angles of a workgroup's tokens are worked out once, into LDS, and all heads'
// rows read them there.
// Angles are products in 64 bits, in turns, of which the whole turns are dropped before anything is rounded to
// 32: a sine of angle t is off by at most 2^-22, of the fp32 steps, and 3 |t| 2^-53, of the products in 64 bits (which
// passes the first from |t| = 2^30 on; at 2^31 both together were 4.2e-7, at 2^24 and below 1.6e-7).
#include "kv_cache.hpp"

#include <algorithm>

namespace psq {
namespace {

constexpr int kThreads = 256;
constexpr int kTokens = 4;   // of a workgroup, at most

struct RopeArgs {
    const uint16_t *q, *k, *v;
    int64_t q_token, q_head, k_token, k_head, v_token, v_head;
    const void *positions;
    int64_t axis_stride;
    const int32_t *axis;
    const double *freq;
    const int64_t *slots;
    uint16_t *out;
    uint8_t *kc, *vc;
    float *ks, *vs;
    int64_t T, nslots;
    int wide, axes, rotary;    // wide: positions of 64 bits
    int Hq, H, D, page;
    int tokens;                // of a workgroup
};

// (cos, sin) of r turns, |r| <= 1/2: quarters taken off, then the two power series on |angle| <= pi / 4, whose
// first terms left out are below 2^-28 and 2^-33.
__device__ __forceinline__ f32x2_t cos_sin_turns(float r)
{
    const float n = __builtin_rintf(4.0f * r);
    const float x = __builtin_fmaf(n, -0.25f, r) * 6.283185307179586f, y = x * x;
    const float s = x * __builtin_fmaf(y, __builtin_fmaf(y, __builtin_fmaf(y, __builtin_fmaf(y, 1.0f / 362880, -1.0f / 5040), 1.0f / 120), -1.0f / 6), 1.0f);
    const float c = __builtin_fmaf(y, __builtin_fmaf(y, __builtin_fmaf(y, __builtin_fmaf(y, __builtin_fmaf(y, -1.0f / 3628800, 1.0f / 40320), -1.0f / 720), 1.0f / 24), -0.5f), 1.0f);
    const int quarter = (int)n & 3;
    const float a = quarter & 1 ? s : c, b = quarter & 1 ? c : s;
    return f32x2_t{quarter == 1 || quarter == 2 ? -a : a, quarter & 2 ? -b : b};
}

// L lanes per row (the power of two that covers D / 16); PAIRED: pairs are neighbours
template <int DT, int CODES, int L, bool PAIRED>
__global__ void __launch_bounds__(kThreads)
rope_write_kernel(RopeArgs a)
{
    constexpr float LIM = CODES == PSQ_CODES_E4M3 ? 448.0f : 127.0f;
    constexpr int kRows = kThreads / L;
    __shared__ f32x2_t turn[kTokens * 128];
    const int tid = threadIdx.x, lane = tid & (L - 1), e = lane * 16, half = a.rotary / 2;
    const int64_t t0 = (int64_t)blockIdx.x * a.tokens;
    const int n = (int)min((int64_t)a.tokens, a.T - t0), per = a.Hq + 2 * a.H, rows = n * per;
    const bool here = e < a.D, turns = e < a.rotary;
    // where the lane's elements are: 8 at e0, 8 at e1
    const int e0 = turns && !PAIRED ? e / 2 : e, e1 = turns && !PAIRED ? half + e / 2 : e + 8;

    for (int i = tid; i < n * half; i += kThreads) {
        const int t = i / half, p = i - t * half;
        const int64_t at = t0 + t + (a.axis ? (int64_t)min(max(a.axis[p], 0), a.axes - 1) * a.axis_stride : 0);
        const double pos = a.wide ? (double)((const int64_t *)a.positions)[at] : (double)((const int32_t *)a.positions)[at];
        const double x = pos * a.freq[p] * 0.15915494309189535;
        turn[t * 128 + p] = cos_sin_turns((float)(x - __builtin_rint(x)));
    }
    __syncthreads();

    for (int r0 = blockIdx.y * kRows; r0 < rows; r0 += gridDim.y * kRows) {
        const int r = r0 + tid / L;
        if (r >= rows) break;   // (the lanes of a row leave together)
        const int t = (uint32_t)r / (uint32_t)per, h = r - t * per;
        const bool is_q = h < a.Hq, is_k = !is_q && h < a.Hq + a.H;
        const int64_t tok = t0 + t;
        const uint16_t *src = is_q ? a.q + tok * a.q_token + h * a.q_head
                              : is_k ? a.k + tok * a.k_token + (h - a.Hq) * a.k_head
                                     : a.v + tok * a.v_token + (h - a.Hq - a.H) * a.v_head;
        int64_t at = 0;
        if (!is_q) {
            const int64_t s = a.slots[tok];
            if (s < 0 || s >= a.nslots) continue;
            at = pool_row(s, is_k ? h - a.Hq : h - a.Hq - a.H, a.H, a.page);
        }
        const bool move = (is_q || is_k) && turns;
        const int p0 = is_q || is_k ? e0 : e, p1 = is_q || is_k ? e1 : e + 8;
        float f[16] = {};
        if (here) {
            const v4i raw[2] = {*(const v4i *)(src + p0), *(const v4i *)(src + p1)};
            to_f32<DT>(raw, f);
            if (move) {
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const f32x2_t cs = turn[t * 128 + e / 2 + i];
                    float &x = f[PAIRED ? 2 * i : i], &y = f[PAIRED ? 2 * i + 1 : i + 8];
                    const float u = x * cs[0] - y * cs[1], w = y * cs[0] + x * cs[1];
                    x = u, y = w;
                }
            }
        }
        if (CODES == PSQ_CODES_NONE || is_q) {
            uint16_t *dst = is_q ? a.out + (tok * a.Hq + h) * (int64_t)a.D : (uint16_t *)(is_k ? a.kc : a.vc) + at * a.D;
            if (here) {
                *(v4i *)(dst + p0) = v4i{(int)pack_half2<DT>(f[0], f[1]), (int)pack_half2<DT>(f[2], f[3]), (int)pack_half2<DT>(f[4], f[5]), (int)pack_half2<DT>(f[6], f[7])};
                *(v4i *)(dst + p1) = v4i{(int)pack_half2<DT>(f[8], f[9]), (int)pack_half2<DT>(f[10], f[11]), (int)pack_half2<DT>(f[12], f[13]), (int)pack_half2<DT>(f[14], f[15])};
            }
        } else {
            float m = absmax16(f);
#pragma unroll
            for (int o = 1; o < L; o <<= 1) m = __builtin_elementwise_maximum(m, __shfl_xor(m, o, 64));
            const bool zero = m < zero_below(LIM);
            const v4i c = codes16<CODES>(f, zero ? 0.0f : LIM / m);
            uint8_t *dst = (is_k ? a.kc : a.vc) + at * a.D;
            if (here) {
                *(v2i *)(dst + p0) = v2i{c[0], c[1]};
                *(v2i *)(dst + p1) = v2i{c[2], c[3]};
            }
            if (lane == 0) (is_k ? a.ks : a.vs)[at] = zero ? 1.0f : m / LIM;
        }
    }
}

template <int DT, int CODES, int L>
void launch(const RopeArgs &a, bool paired, hipStream_t st)
{
    const int64_t blocks = (a.T + a.tokens - 1) / a.tokens, rows = (int64_t)a.tokens * (a.Hq + 2 * a.H);
    const int64_t passes = (rows * L + kThreads - 1) / kThreads;
    const dim3 grid((unsigned)blocks, (unsigned)std::min<int64_t>(passes, std::max<int64_t>(1, 1024 / blocks)));
    if (paired) rope_write_kernel<DT, CODES, L, true><<<grid, kThreads, 0, st>>>(a);
    else rope_write_kernel<DT, CODES, L, false><<<grid, kThreads, 0, st>>>(a);
}

template <int DT, int CODES>
int launch_dim(const RopeArgs &a, bool paired, hipStream_t st)
{
    const int need = a.D / 16;
    if (need <= 1) launch<DT, CODES, 1>(a, paired, st);
    else if (need <= 2) launch<DT, CODES, 2>(a, paired, st);
    else if (need <= 4) launch<DT, CODES, 4>(a, paired, st);
    else if (need <= 8) launch<DT, CODES, 8>(a, paired, st);
    else launch<DT, CODES, 16>(a, paired, st);
    return check_launch("rope_kv_write");
}

}  // namespace
}  // namespace psq

extern "C" int psq_rope_kv_write(int codes, const void *q, const void *k, const void *v, int dtype, int64_t q_token, int64_t q_head,
                                 int64_t k_token, int64_t k_head, int64_t v_token, int64_t v_head, const void *positions,
                                 int positions_bits, int axes, int64_t axis_stride, const int32_t *pair_axis, const double *inv_freq,
                                 int rotary, int interleaved, const int64_t *slots, int64_t T, int Hq, int Hkv, int D, void *k_cache,
                                 void *v_cache, float *k_scale, float *v_scale, int64_t num_pages, int page_size, void *q_out, void *stream)
{
    using namespace psq;
    const char *name = "rope_kv_write";
    if (T < 0 || Hq < 0) return set_error(PSQ_E_ARG, "%s: negative size", name);
    if (dtype != PSQ_BF16 && dtype != PSQ_F16) return set_error(PSQ_E_ARG, "%s: rows must be bf16 or f16 (dtype %d)", name, dtype);
    if (positions_bits != 32 && positions_bits != 64) return set_error(PSQ_E_ARG, "%s: positions have 32 or 64 bits", name);
    if (int e = check_kv_cache(name, codes, k_cache, v_cache, k_scale, v_scale, num_pages, page_size, Hkv, D)) return e;
    if (rotary <= 0 || rotary % 16 || rotary > D)
        return set_error(PSQ_E_SHAPE, "%s: %d rotary dims must be a multiple of 16, at most %d", name, rotary, D);
    if (axes < 1 || (axes > 1 && !pair_axis)) return set_error(PSQ_E_ARG, "%s: %d axes need the axis of each pair", name, axes);
    if (T == 0) return PSQ_OK;
    if (!k || !v || !slots || !positions || !inv_freq || (Hq && (!q || !q_out))) return set_error(PSQ_E_ARG, "%s: null pointer", name);
    if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)q_out) & 15 || (q_token | q_head | k_token | k_head | v_token | v_head) & 7)
        return set_error(PSQ_E_SHAPE, "%s: rows must be 16-byte aligned, their strides multiples of 8", name);
    if (((uintptr_t)slots | (uintptr_t)inv_freq) & 7 || (uintptr_t)pair_axis & 3 || (uintptr_t)positions & (positions_bits / 8 - 1))
        return set_error(PSQ_E_SHAPE, "%s: misaligned slots, positions, axes or frequencies", name);
    if (Hq > 65535 || T > 0x7fffffffLL) return set_error(PSQ_E_SHAPE, "%s: T=%lld or %d heads too large", name, (long long)T, Hq);
    if (int e = require_device()) return e;
    RopeArgs a{(const uint16_t *)q, (const uint16_t *)k, (const uint16_t *)v, q_token, q_head, k_token, k_head, v_token, v_head,
               positions, axis_stride, pair_axis, inv_freq, slots, (uint16_t *)q_out, (uint8_t *)k_cache, (uint8_t *)v_cache, k_scale,
               v_scale, T, num_pages * page_size, positions_bits == 64, axes, rotary, Hq, Hkv, D, page_size, 1};
    // a workgroup has several tokens' angles where the workgroups fill the chip all the same
    if (T >= 1024 * kTokens) a.tokens = kTokens;
    hipStream_t st = (hipStream_t)stream;
    auto go = [&](auto dtc) {
        constexpr int DT = decltype(dtc)::value;
        if (codes == PSQ_CODES_I8) return launch_dim<DT, PSQ_CODES_I8>(a, interleaved != 0, st);
        if (codes == PSQ_CODES_E4M3) return launch_dim<DT, PSQ_CODES_E4M3>(a, interleaved != 0, st);
        return launch_dim<DT, PSQ_CODES_NONE>(a, interleaved != 0, st);
    };
    return dtype == PSQ_BF16 ? go(std::integral_constant<int, PSQ_BF16>{}) : go(std::integral_constant<int, PSQ_F16>{});
}
