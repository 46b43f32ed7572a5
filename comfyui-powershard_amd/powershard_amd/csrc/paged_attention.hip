// paged_attention.hip -- attention of one new token per sequence over the paged key-value cache.
//
//   s_t = scale (q . k_t) ks_t,  p = softmax(s),  out = sum_t p_t vs_t v_t
//
// Bound by the cache's bytes: each key and value is read once for the G = Hq / Hkv heads that share it.
// A workgroup of 4 waves takes a run of tokens of one sequence and kv head, for up to 16 of its heads
// (more heads to a kv head: more workgroups, which find the cache's lines in the last-level cache; waves of
// one workgroup side by side on the same tokens measured slower, 16 x 8192, 64 heads on one 32 | 42 us (28 now),
// their runs being shorter and their parts longer); its waves take steps of 32 tokens in turn, and each keeps a running maximum, sum and output of its own
// (no barrier inside the run).  Everything goes from memory to registers in the layout that the matrix
// instructions read (16x16x32, fp32 accumulation), with no LDS and no cross-lane move of keys, values or
// probabilities.  Lane l, m = l & 15, g = l >> 4:
//   S^T = K Q^T: K rows are tokens (lane row m), the contraction index 8 g + j stands for the dims that
//     the lane has loaded, 16 bytes at 16 g of each 64-byte run of the row (Q is laid out to match);
//     the result holds head m in the lane, tokens 4 g + i of each of the two tiles of 16;
//   O^T = V^T P^T: those 8 probabilities are, as they are, the lane's part of P^T if contraction index
//     8 g + j stands for token 4 g + j of tile 0 (j < 4) and 4 g + j - 4 of tile 1 (j >= 4).  For V^T the
//     lane loads, of each of these 8 tokens, the dims m DV .. m DV + DV - 1 (whole rows per 16 lanes) and
//     transposes 8 tokens x DV dims in its registers by byte permutes; row m of product dt is dim
//     m DV + dt.
// int8 and e4m3 codes are exact in bf16 (and f16), so they enter the products as they are; key scales
// multiply the fp32 scores, value scales the fp32 probabilities.  A probability enters its product as a
// pair of 16-bit numbers, p = hi + lo, two instructions each: 16 bits of it or more take part, and the
// matrix units stay far below what the loads leave them.  bf16 pairs hold them over fp32's range.  f16 pairs end
// at 2^-24, so with f16 values p, and the sums over it, are held 2^15 times as large (p <= 1): 16 bits of it down to
// 2^-30, and no more than 2^-40 lost below.
//
// Work is dealt in rounds of 128 tokens (a step of each wave).  The rounds of all units (sequence, kv
// head, head tile), in their order, are cut into equal runs, one per workgroup, as many workgroups as the
// chip holds at once: ragged lengths cost no balance, the host needs no lengths, and a unit is cut only
// where a run ends.  A workgroup writes its parts of cut units (two at most) to the workspace and counts
// itself when its run is done; the last one of a unit, or a second kernel (see plan()), adds the parts up
// in their order, so results do not depend on timing.  With the second kernel the workspace carries parts
// from one launch to the next: another call's kernels between them (a second host thread on the stream) would
// write over them, so such a call's workspace is its own (psq_paged_attention_own_workspace).
#include "kv_cache.hpp"

#include <algorithm>
#include <math.h>

namespace psq {
namespace {

typedef float v2f __attribute__((ext_vector_type(2)));

constexpr int kWaves = 4, kThreads = 64 * kWaves;
constexpr int kStep = 32;                       // tokens of a wave's step
constexpr int kTile = 16;                       // heads of a workgroup; tokens of a group (one page holds it)
constexpr int kGrain = kStep * kWaves;          // tokens of a workgroup's round
constexpr int64_t kCounterBytes = 64 * 1024;    // arrival counters of the GEMMs at the workspace's head
constexpr int SC1 = 16;                         // cache-policy bit sc1 of the buffer intrinsics
constexpr float kF16Unit = 0x1p15f;             // of probabilities with f16 values
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// A cut unit that a run has part of: its sequence, index in it, first run and number of parts.
struct Cut { int b, unit, first, parts; };

// workgroups that a CU holds at once (4 waves; 512, 256 and 168 registers a lane)
constexpr int groups_per_cu(int D, bool codes) { return D > 128 ? (codes ? 2 : 1) : 3; }

struct AttnArgs {
    const uint16_t *q;
    int64_t q_batch, q_head;
    const uint8_t *kc, *vc;
    const float *ks, *vs;
    const int32_t *table;
    int64_t table_stride;
    const int32_t *lengths;
    uint16_t *out;
    float *lse;
    uint32_t *count;       // one per run: of the unit that it begins
    Cut *cut;              // one per unit, where parts are joined apart
    float *part;           // two per run
    int part_floats;       // of one part
    int num_pages, cap;    // cap: tokens that a table row has room for
    int B, page, Hq, Hkv, D, G, tiles, window;
    int alone;             // units stay whole, a workgroup each
    int apart;             // parts are joined by a kernel of their own
    float scale;           // times log2(e)
    float per_unit;        // 1 / the unit that probabilities are held in
    int sinks;
};

template <int DT>
__device__ __forceinline__ v4f mfma(const v4i &a, const v4i &b, const v4f &c)
{
    if constexpr (DT == PSQ_BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}

// over the four lane groups g
__device__ __forceinline__ float group_max(float x)
{
    const uint32_t u = __float_as_uint(x);
    const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const float y = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(y), __float_as_uint(y), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

__device__ __forceinline__ float group_sum(float x)
{
    const uint32_t u = __float_as_uint(x);
    const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const float y = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(y), __float_as_uint(y), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// a value that all lanes hold, in scalar registers
__device__ __forceinline__ uint64_t uniform(uint64_t x)
{
    return (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(x >> 32)) << 32 |
           (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)x);
}

__device__ __forceinline__ void lower_priority(int to)
{
    if (to == 2) __builtin_amdgcn_s_setprio(2);
    else if (to == 1) __builtin_amdgcn_s_setprio(1);
    else __builtin_amdgcn_s_setprio(0);
}

// x / y, by the short division where x allows it
__device__ __forceinline__ uint64_t divide(uint64_t x, uint32_t y)
{
    return uniform(x >> 32 ? x / y : (uint64_t)((uint32_t)x / y));
}

// Sums of parts, kept at the maximum M: first brought to a new one, then a part (at maximum m) added.
__device__ __forceinline__ float scale_to(float from, float to)
{
    return __builtin_amdgcn_exp2f(from - (to == -INFINITY ? 0.0f : to));
}

__device__ __forceinline__ void join_move(float &M, float &L, v4f &acc, float to)
{
    const float e = scale_to(M, to);
    L *= e;
#pragma unroll
    for (int c = 0; c < 4; c++) acc[c] *= e;
    M = to;
}

__device__ __forceinline__ void join_add(float M, float &L, v4f &acc, float m, float l, const v4f &y)
{
    const float e = scale_to(m, M);
    L += l * e;
#pragma unroll
    for (int c = 0; c < 4; c++) acc[c] += y[c] * e;
}

// Four dims of a head's output from the sums at maximum M (in units of log2), and its lse.  none: no
// token, zeros (tokens whose scores are all -inf: 0 / 0, as softmax).
template <int DT>
__device__ __forceinline__ void finish(const AttnArgs &a, int64_t head, int D, int d4, const v4f &acc, float M, float L, bool none)
{
    const float r = none ? 0.0f : 1.0f / L;
    *(v2i *)(a.out + head * D + 4 * d4) = v2i{(int)pack_half2<DT>(acc[0] * r, acc[1] * r), (int)pack_half2<DT>(acc[2] * r, acc[3] * r)};
    if (a.lse && d4 == 0) a.lse[head] = none ? -INFINITY : M * kLn2 + logf(L * a.per_unit);
}

// Adds up the parts of heads h0 .. h0 + n - 1 of a cut unit: part 0 is its first run's second, the others the
// first ones of the runs after it.  A thread has one quad of dims (of every 256 / quads-th part, where
// these are few), U parts' loads in flight.  h0 is one of the unit's heads.  smem: 6 KB.
template <int DT, int U>
__device__ __forceinline__ void join_parts(const AttnArgs &a, const Cut &cut, int h0, int n, float *smem)
{
    const int tid = threadIdx.x;
    const int hk = cut.unit / a.tiles, ht = cut.unit - hk * a.tiles, heads = min(a.G - ht * kTile, kTile);
    const int64_t row0 = cut.b * (int64_t)a.Hq + hk * a.G + ht * kTile;
    const int quads = a.D / 4, first = h0 * quads, items = min(heads - h0, n) * quads, sharers = max(kThreads / items, 1);
    const int share = sharers > 1 ? tid / items : 0;
    const __amdgpu_buffer_rsrc_t rs = raw_rsrc(a.part + (int64_t)(2 * cut.first) * a.part_floats);
    const int pitch = a.part_floats * 4, ml_at = heads * a.D * 4;
    v4f *red = (v4f *)smem;
    v2f *red_ml = (v2f *)(smem + 4 * kThreads);
    __syncthreads();   // LDS is free
    for (int i = tid - share * items; i < items && share < sharers; i += kThreads) {
        const int q = first + i, h = q / quads;
        float M = -INFINITY, L = 0.0f;
        v4f acc = {0, 0, 0, 0};
        for (int s0 = share; s0 < cut.parts; s0 += U * sharers) {
            v4i y[U];
            v2i ml[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int s = s0 + u * sharers, at = (s == 0 ? 1 : 2 * s) * pitch;
                y[u] = v4i{0, 0, 0, 0}, ml[u] = v2i{(int)0xff800000, 0};   // no part: maximum -inf, sum 0
                if (s < cut.parts) {
                    y[u] = __builtin_amdgcn_raw_buffer_load_b128(rs, at + q * 16, 0, SC1);
                    ml[u] = __builtin_amdgcn_raw_buffer_load_b64(rs, at + ml_at + 8 * h, 0, SC1);
                }
            }
            float top = M;
#pragma unroll
            for (int u = 0; u < U; u++) top = fmaxf(top, __int_as_float(ml[u][0]));
            join_move(M, L, acc, top);
#pragma unroll
            for (int u = 0; u < U; u++)
                join_add(M, L, acc, __int_as_float(ml[u][0]), __int_as_float(ml[u][1]), __builtin_bit_cast(v4f, y[u]));
        }
        if (sharers == 1) {
            finish<DT>(a, row0 + h, a.D, q - h * quads, acc, M, L, false);
        } else {
            red[tid] = acc;
            red_ml[tid] = v2f{M, L};
        }
    }
    if (sharers == 1) return;
    __syncthreads();
    if (tid < items) {
        const int q = first + tid, h = q / quads;
        float M = -INFINITY, L = 0.0f;
        v4f acc = {0, 0, 0, 0};
        for (int k = 0; k < sharers; k++) M = fmaxf(M, red_ml[k * items + tid][0]);
        for (int k = 0; k < sharers; k++) join_add(M, L, acc, red_ml[k * items + tid][0], red_ml[k * items + tid][1], red[k * items + tid]);
        finish<DT>(a, row0 + h, a.D, q - h * quads, acc, M, L, false);
    }
}

// A step's registers.  DD: head dims they are laid out for; PART: D < DD, the rest of a row is not there.
template <int CODES, int DD, bool PART>
struct Step {
    static constexpr int ES = CODES == PSQ_CODES_NONE ? 2 : 1;
    static constexpr int KL = DD * ES / 64;       // 16-byte loads of a key row per lane group
    static constexpr int DV = DD / 16, VW = DV * ES / 4;
    v4i k[2][KL];
    uint32_t v[8][VW];
    v4f ks[2], vs[2];

    // groups ga, gb: rows 16 ga .. and 16 gb .. of the pools
    __device__ __forceinline__ void load_keys(const AttnArgs &a, uint32_t ga, uint32_t gb, int m, int g)
    {
        const int row = (PART ? a.D : DD) * ES;
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const int64_t grp = t ? gb : ga;
            const uint8_t *kp = a.kc + grp * (kTile * row);
#pragma unroll
            for (int c = 0; c < KL; c++) {
                const int at = 64 * c + 16 * g;
                if (PART) k[t][c] = v4i{0, 0, 0, 0};
                if (!PART || at < row) k[t][c] = *(const v4i *)(kp + (uint32_t)(m * row + at));
            }
            if constexpr (ES == 1) ks[t] = *(const v4f *)(a.ks + grp * kTile + 4 * g);
        }
    }

    __device__ __forceinline__ void load_values(const AttnArgs &a, uint32_t ga, uint32_t gb, int m, int g)
    {
        const int row = (PART ? a.D : DD) * ES;
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const int64_t grp = t ? gb : ga;
            const uint8_t *vp = a.vc + grp * (kTile * row);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                uint32_t *w = v[4 * t + i];
                const uint8_t *src = vp + (uint32_t)((4 * g + i) * row + m * (DV * ES));
                if (PART)
#pragma unroll
                    for (int c = 0; c < VW; c++) w[c] = 0;
                if (!PART || m * DV < a.D) {
                    if constexpr (VW == 1) w[0] = *(const uint32_t *)src;
                    else if constexpr (VW == 2) { const v2i x = *(const v2i *)src; w[0] = x[0], w[1] = x[1]; }
                    else {
#pragma unroll
                        for (int c = 0; c < VW; c += 4) {
                            const v4i x = *(const v4i *)(src + 4 * c);
                            w[c] = x[0], w[c + 1] = x[1], w[c + 2] = x[2], w[c + 3] = x[3];
                        }
                    }
                }
            }
            if constexpr (ES == 1) vs[t] = *(const v4f *)(a.vs + grp * kTile + 4 * g);
        }
    }
};

// SINKS: a window's sinks (a kernel of its own: 61 x 4096 int8 without a window 55.5 us with one for both, 54.7 so)
template <int DT, int CODES, int DD, bool PART, bool SINKS>
__global__ void __launch_bounds__(kThreads, groups_per_cu(DD, CODES != PSQ_CODES_NONE))
paged_attention_kernel(AttnArgs a)
{
    using S = Step<CODES, DD, PART>;
    constexpr int ES = S::ES, DV = S::DV, VW = S::VW, NC = DD / 32;
    constexpr int PVT = CODES == PSQ_CODES_NONE ? DT : PSQ_BF16;   // of the second product
    extern __shared__ __attribute__((aligned(16))) float smem[];
    __shared__ float wave_m[kWaves][kTile], wave_l[kWaves][kTile];
    __shared__ uint32_t wave_rounds[kWaves], start_r;
    __shared__ int start_b, joins[2];

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int m = lane & 15, g = lane >> 4;
    const int D = PART ? a.D : DD, per_page = a.page / kTile, units = a.Hkv * a.tiles;   // (units of a sequence)

    // ---- the workgroup's run of rounds
    // With sinks tokens are counted without those between them and the window (whole groups: skip of them, from
    // sink_end on); len and lo, the end of what the window hides, are such counts.
    const int sink_end = (a.sinks + kTile - 1) & ~(kTile - 1);
    auto span = [&](int b, int &len, int &lo, int &skip, bool &past) {   // tokens of sequence b; its rounds
        len = max(a.lengths[b], 0);
        past = len > a.cap;
        len = min(len, a.cap);
        lo = a.window ? max(len - a.window, 0) : 0;
        skip = SINKS ? max((lo & ~(kTile - 1)) - sink_end, 0) : 0;
        len -= skip, lo -= skip;
        return past ? 1 : max((len - (SINKS ? 0 : lo & ~(kTile - 1)) + kGrain - 1) / kGrain, 1);
    };
    int len, lo, skip, rounds;
    bool past;
    // Each wave scans the lengths for itself where it holds them (64 sequences), else the workgroup does.
    const bool narrow = a.B <= 64;
    const int each = a.alone ? 0 : narrow ? 1 : (a.B + kThreads - 1) / kThreads;   // sequences of a thread
    const int mine_at = narrow ? lane : tid * each;
    uint32_t own = 0;
    for (int i = 0; i < each; i++)
        if (mine_at + i < a.B) own += span(mine_at + i, len, lo, skip, past);
    uint32_t before = own;                                  // rounds up to and with this thread's
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t y = __shfl_up(before, o, 64);
        before += lane >= o ? y : 0;
    }
    uint32_t total = (uint32_t)__builtin_amdgcn_readlane((int)before, 63);
    if (!narrow) {
        if (lane == 63) wave_rounds[wave] = before;
        __syncthreads();
        total = 0;
#pragma unroll
        for (int i = 0; i < kWaves; i++) {
            before += i < wave ? wave_rounds[i] : 0;
            total += wave_rounds[i];
        }
    }
    before -= own;
    const uint64_t all = uniform((uint64_t)total * units);
    const uint32_t w = blockIdx.x;
    const uint32_t runs = a.alone ? gridDim.x : (uint32_t)max(min((uint64_t)gridDim.x, all), (uint64_t)1);
    auto first_of = [&](uint32_t w) { return all >> 32 ? uniform(w * all / runs) : divide(w * all, runs); };
    uint64_t x = 0, end;
    int b, unit, r = 0;
    if (a.alone) {
        b = w / (uint32_t)units, unit = w - b * units;
        end = rounds = span(b, len, lo, skip, past);
    } else {
        if (w >= runs) return;
        x = first_of(w), end = first_of(w + 1);
        const uint32_t y = (uint32_t)divide(x, units);      // the thread whose sequences hold the run's start
        const bool here = y >= before && y < before + own;
        uint32_t at;
        if (narrow) {
            b = __builtin_ctzll(__ballot(here));
            at = (uint32_t)__builtin_amdgcn_readlane((int)before, b);
        } else {
            if (here) {
                int i = mine_at;
                for (;; i++) {
                    const int n = span(i, len, lo, skip, past);
                    if (y < before + n) break;
                    before += n;
                }
                start_b = i;
                start_r = before;
            }
            __syncthreads();
            b = __builtin_amdgcn_readfirstlane(start_b);
            at = (uint32_t)__builtin_amdgcn_readfirstlane(start_r);
        }
        rounds = span(b, len, lo, skip, past);
        const uint64_t in = x - (uint64_t)at * units;
        unit = (int)divide(in, rounds), r = (int)(in - (uint64_t)unit * rounds);
    }
    Cut cut[2] = {};       // what the run has part of: a unit that it goes on with, and one that it leaves

    // ---- the segment of the run at hand: n rounds of one unit, tokens c0 .. hi - 1 (so counted)
    int n, hk, ht, heads, c0, hi, steps;
    int64_t head0;
    v4i qf[NC];
    S st;
    uint32_t grp;          // the pool groups of 32 steps, one per lane: lane 2 s + t has tile t of step s
    bool wild;             // a page outside the pool
    auto groups = [&](int s0) {
        const int t = c0 + kStep * wave + (s0 + (lane >> 1)) * kGrain + kTile * (lane & 1);
        bool out = false;
        grp = 0;
        if (t < hi) {
            const uint32_t i = (uint32_t)(!SINKS || t < sink_end ? t : t + skip) / kTile, col = i / (uint32_t)per_page;
            const int pg = a.table[b * a.table_stride + col];
            out = pg < 0 || pg >= a.num_pages;
            grp = out ? 0 : ((uint32_t)pg * a.Hkv + hk) * per_page + (i - col * per_page);
        }
        wild = __any(out);
    };
    auto load_keys = [&](int s) {
        const int i = 2 * (s & 31);
        st.load_keys(a, __builtin_amdgcn_readlane(grp, i), __builtin_amdgcn_readlane(grp, i + 1), m, g);
    };
    auto load_values = [&](int s) {
        const int i = 2 * (s & 31);
        st.load_values(a, __builtin_amdgcn_readlane(grp, i), __builtin_amdgcn_readlane(grp, i + 1), m, g);
    };
    auto begin = [&]() {   // the first step's loads (no page, no load: the caller looks at wild)
        wild = false;
        if (steps) groups(0);
        if (steps && !wild) {
            load_keys(0);
            load_values(0);
        }
    };
    auto open = [&]() {
        n = (int)min(end - x, (uint64_t)(rounds - r));
        hk = unit / a.tiles, ht = unit - hk * a.tiles, heads = min(a.G - ht * kTile, kTile);
        head0 = b * (int64_t)a.Hq + hk * a.G + ht * kTile;
        c0 = (SINKS ? 0 : lo & ~(kTile - 1)) + r * kGrain, hi = past ? c0 : min(c0 + n * kGrain, len);
        steps = c0 + kStep * wave < hi ? (hi - c0 - kStep * wave + kGrain - 1) / kGrain : 0;
        const uint16_t *q = a.q + b * a.q_batch + (int64_t)(hk * a.G + ht * kTile + m) * a.q_head;
#pragma unroll
        for (int c = 0; c < NC; c++) {
            const int d = ES == 2 ? 32 * c + 8 * g : 64 * (c >> 1) + 16 * g + 8 * (c & 1);
            qf[c] = v4i{0, 0, 0, 0};
            if (m < heads && (!PART || d < D)) qf[c] = *(const v4i *)(q + d);
        }
        begin();
    };
    open();
    // Waves of the workgroups that came to a CU first go ahead of the others' (finishing a third earlier at
    // equal runs): each steps its priority down by quarters of its run, and they finish together (128 x 8192
    // bf16 390 -> 387.5 us, 61 x 4096 int8 66 -> 64).
    const uint64_t from = x;
    const uint32_t quarter = (uint32_t)((end - x + 3) / 4);
    uint32_t mark = quarter;
    int priority = 3;
    __builtin_amdgcn_s_setprio(3);

    for (;;) {
    v4f o[DV];
    constexpr int LD = DD + 4;
    auto place = [&]() {   // o to the wave's rows of the LDS
        if (m < heads) {
            float *row = smem + (wave * heads + m) * LD;
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int dt = 0; dt < DV; dt += 4)
                    *(v4f *)(row + (4 * g + i) * DV + dt) = v4f{o[dt][i], o[dt + 1][i], o[dt + 2][i], o[dt + 3][i]};
        }
    };
    float run_m, run_l;
    bool pair = true;      // probabilities as hi + lo
    // The step's keys and values are in flight or here.  The next step's loads go into the same registers
    // as soon as these are read: its keys before the softmax, its values after the second product.
    auto compute = [&](int s, bool more) {
        const int t0 = c0 + kStep * wave + s * kGrain;
        v4f sc[2];
#pragma unroll
        for (int t = 0; t < 2; t++) {
            v4f x = {0, 0, 0, 0};
#pragma unroll
            for (int c = 0; c < NC; c++) {
                v4i kf;
                if constexpr (ES == 2) {
                    kf = st.k[t][c];
                } else {
                    const uint32_t w0 = (uint32_t)st.k[t][c >> 1][2 * (c & 1)], w1 = (uint32_t)st.k[t][c >> 1][2 * (c & 1) + 1];
                    kf = v4i{(int)code_pair<DT, CODES, 0>(w0), (int)code_pair<DT, CODES, 1>(w0),
                             (int)code_pair<DT, CODES, 0>(w1), (int)code_pair<DT, CODES, 1>(w1)};
                }
                x = mfma<DT>(kf, qf[c], x);
            }
#pragma unroll
            for (int i = 0; i < 4; i++) sc[t][i] = x[i] * a.scale * (ES == 1 ? st.ks[t][i] : 1.0f);
        }
        if (more) load_keys(s + 1);
        if (t0 < lo || t0 + kStep > hi) {
            // tokens outside: score -inf, and nothing of what their places hold (NaN, Inf) reaches the sums
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int tok = t0 + kTile * t + 4 * g + i;
                    if ((tok < lo && (!SINKS || tok >= a.sinks)) || tok >= hi) {
                        sc[t][i] = -INFINITY;
                        if constexpr (ES == 1) st.vs[t][i] = 0.0f;
                        if constexpr (CODES != PSQ_CODES_I8) {
#pragma unroll
                            for (int c = 0; c < VW; c++) st.v[4 * t + i][c] = 0;
                        }
                    }
                }
        }
        float top = fmaxf(fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[0][2], sc[0][3])),
                          fmaxf(fmaxf(sc[1][0], sc[1][1]), fmaxf(sc[1][2], sc[1][3])));
        top = group_max(top);
        if (__any(top > run_m)) {
            const float next = fmaxf(run_m, top);
            const float keep = next == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(run_m - next);
            run_m = next;
            run_l *= keep;
#pragma unroll
            for (int dt = 0; dt < DV; dt++)
#pragma unroll
                for (int i = 0; i < 4; i++) o[dt][i] *= keep;
        }
        const float ref = run_m == -INFINITY ? 0.0f : run_m;
        float p[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            p[j] = __builtin_amdgcn_exp2f(sc[j >> 2][j & 3] - ref);
            if constexpr (PVT == PSQ_F16) p[j] *= kF16Unit;
            run_l += p[j];
            if constexpr (ES == 1) p[j] *= st.vs[j >> 2][j & 3];
        }
        v4i ph, pl;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const uint32_t h = pack_half2<PVT>(p[2 * j], p[2 * j + 1]);
            ph[j] = (int)h;
            pl[j] = (int)pack_half2<PVT>(p[2 * j] - half_to_f32<PVT>(h), p[2 * j + 1] - half_to_f32<PVT>(h >> 16));
        }
        if (!pair)
#pragma unroll
            for (int j = 0; j < 4; j++) ph[j] = pl[j] = (int)pack_half2<PVT>(0.5f * p[2 * j], 0.5f * p[2 * j + 1]);
#pragma unroll
        for (int dt = 0; dt < DV; dt++) {
            v4i vf;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if constexpr (ES == 2) {
                    vf[j] = (int)__builtin_amdgcn_perm(st.v[2 * j + 1][dt >> 1], st.v[2 * j][dt >> 1],
                                                       dt & 1 ? 0x07060302u : 0x05040100u);
                } else {
                    const uint32_t w = __builtin_amdgcn_perm(st.v[2 * j + 1][dt >> 2], st.v[2 * j][dt >> 2],
                                                             dt & 2 ? 0x07030602u : 0x05010400u);
                    vf[j] = (int)(dt & 1 ? code_pair<PSQ_BF16, CODES, 1>(w) : code_pair<PSQ_BF16, CODES, 0>(w));
                }
            }
            o[dt] = mfma<PVT>(vf, ph, o[dt]);
            o[dt] = mfma<PVT>(vf, pl, o[dt]);
        }
    };

    for (;;) {
#pragma unroll
        for (int dt = 0; dt < DV; dt++) o[dt] = v4f{0, 0, 0, 0};
        run_m = -INFINITY, run_l = 0.0f;
        const uint32_t done = (uint32_t)(x - from);
        for (int s = 0; s < steps && !wild; s++) {
            bool more = s + 1 < steps;
            if (more && ((s + 1) & 31) == 0) {
                groups(s + 1);
                more = !wild;
            }
            if (done + s >= mark) {
                mark += quarter;
                lower_priority(--priority);
            }
            compute(s, more);
            if (more) load_values(s + 1);
        }
        // An infinite value meets lo = 0 or lo < 0 in the second product: NaN where the sum is infinite.
        // Once more, then, with p as the sum of two equal halves (the precision of one 16-bit number), for the
        // sums that were NaN; the others wait in the wave's part of the LDS, which is free until its sums go there.
        float any = 0.0f;
#pragma unroll
        for (int dt = 0; dt < DV; dt++)
#pragma unroll
            for (int i = 0; i < 4; i++) any = __builtin_fmaf(o[dt][i], 0.0f, any);
        if (!pair || wild || !__any(any != any)) break;
        pair = false;
        place();
        begin();
    }
    if (wild || past) run_m = 0.0f, run_l = NAN;

    // ---- the waves' sums into one: each wave's output at its own maximum, in LDS
    run_l = group_sum(run_l);
    if (g == 0) {
        wave_m[wave][m] = run_m;
        wave_l[wave][m] = run_l;
    }
    if (!pair) {
        float *row = smem + (wave * heads + m) * LD + 4 * g * DV;
        if (m < heads)
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int dt = 0; dt < DV; dt++) {
                    const float first = row[i * DV + dt];
                    o[dt][i] = first == first ? first : o[dt][i];
                }
    }
    place();
    // the run's next segment: its first loads travel while this one's sums are put together
    const bool whole = n == rounds, none = len == 0 && !past;
    const int quads = D / 4, these = heads;
    const int64_t row0 = head0;
    const int slot = r == 0;
    if (!whole) {
        auto owner = [&](uint64_t y) { return (int)(all >> 32 ? uniform(((y + 1) * runs - 1) / all) : divide((y + 1) * runs - 1, (uint32_t)all)); };
        const int first = slot ? (int)w : owner(x - r);
        cut[slot] = Cut{b, unit, first, owner(x - r + rounds - 1) - first + 1};
    }
    if (a.apart && slot && tid == 0) a.cut[b * units + unit] = whole ? Cut{} : cut[1];   // (its first run says so)
    x += n;
    const bool last = x >= end;
    if (!last) {
        r = 0;
        if (++unit == units) {
            unit = 0;
            rounds = span(++b, len, lo, skip, past);
        }
        open();
    }
    stage_barrier();       // (a barrier that leaves loads in flight)
    const __amdgpu_buffer_rsrc_t part = raw_rsrc(a.part + (int64_t)(2 * w + slot) * a.part_floats);
    for (int i = tid; i < these * quads; i += kThreads) {
        const int h = i / quads, d4 = i - h * quads;
        const float M = fmaxf(fmaxf(wave_m[0][h], wave_m[1][h]), fmaxf(wave_m[2][h], wave_m[3][h]));
        v4f acc = {0, 0, 0, 0};
        float L = 0.0f;
#pragma unroll
        for (int v = 0; v < kWaves; v++) join_add(M, L, acc, wave_m[v][h], wave_l[v][h], *(const v4f *)(smem + (v * these + h) * LD + 4 * d4));
        if (whole) {
            finish<DT>(a, row0 + h, D, d4, acc, M, L, none);
        } else {
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(v4i, acc), part, i * 16, 0, SC1);
            if (d4 == 0)
                __builtin_amdgcn_raw_buffer_store_b64(v2i{__float_as_int(M), __float_as_int(L)}, part, (these * D + 2 * h) * 4, 0, SC1);
        }
    }
    if (last) break;
    stage_barrier();       // LDS is free again
    }
    if (a.apart || cut[0].parts + cut[1].parts == 0) return;

    // ---- the run's parts are written (around the XCDs' own L2s, sc1: the count needs only the wait for the
    // stores); the workgroup that counts last adds a unit up
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (tid < 2) {
        const int first = tid ? cut[1].first : cut[0].first, parts = tid ? cut[1].parts : cut[0].parts;
        if (parts) {
            const bool join = atomicAdd(a.count + first, 1u) == (uint32_t)parts - 1;
            // every other part has been counted: zero again for the next launch
            if (join) __hip_atomic_store(a.count + first, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            joins[tid] = join;
        } else {
            joins[tid] = 0;
        }
    }
    __syncthreads();
#pragma clang loop unroll(disable)
    for (int i = 0; i < 2; i++)
        if (__builtin_amdgcn_readfirstlane(joins[i])) join_parts<DT, DD == 64 ? 8 : 16>(a, i ? cut[1] : cut[0], 0, kTile, smem);
}

// The join as a kernel of its own: a workgroup per unit and head of it.
template <int DT>
__global__ void __launch_bounds__(kThreads)
join_parts_kernel(AttnArgs a)
{
    __shared__ __attribute__((aligned(16))) float smem[6 * kThreads];
    const Cut cut = a.cut[blockIdx.x];
    const int heads = a.G - cut.unit % a.tiles * kTile;   // the last tile of a kv head may have fewer than the grid
    if (cut.parts && (int)blockIdx.y < heads) join_parts<DT, 8>(a, cut, blockIdx.y, 1, smem);
}

// ------------------------------------------------------------------ the launch
// As many workgroups as the chip holds, no more than the rounds can fill.  A unit's parts are joined by its
// last workgroup where one round of loads per thread holds them (few parts, or few dims to a part), else by
// a kernel of their own, which spreads the unit's heads over the chip; two workgroups per CU then fill the
// memory system with fewer parts than three.  us a call, joined inside | apart (the second launch is
// 3.5 us of the host's time, which bounds the small calls): 1 x 2000 tokens, 40 heads on 8, int8 14.0 | 18.7;
// 1 x 4000, 16 on 16 13.8 | 18.2; 61 x 4096, 40 on 8 63.5 | 65.9; 128 x 8192, 64 on 8, bf16 377 | 386;
// 4 x 16000, 40 on 8 30.1 | 26.0; 1 x 131071, 40 on 8, fp8 66.6 | 57.9 (3 per CU 58.9); 1 x 30000, 8 on 1
// 35 | 18; 8 x 6000, 16 on 1, 256 dims 33 | 19.  At the limit of one round, 8 heads of 128 dims, int8, 4000
// tokens: 12 parts a unit 20.1 | 20.2, 16 18.7 | 19.0, 24 16.8 | 15.7.
// Where a part has more quads of dims than a workgroup threads, these take turns, and the limit is 4 parts a
// unit: 16 heads of 256 dims, int8, 4000 tokens, 3 parts 89.2 | 85.5, 4 63.9 | 63.2, 5 64.7 | 57.4, 8 40.7 | 37.2,
// 12 39.1 | 29.7 (1500 tokens, 4 32.1 | 31.8, 5 39.9 | 32.6); 5 heads of 256 dims 4 59.1 | 58.4, 5 54.2 | 51.0; 16 heads
// of 128 dims 4 48.9 | 53.4, 5 45.5 | 46.8, 8 29.1 | 31.6, 12 22.8 | 21.2 (1500 tokens, 4 24.2 | 29.1, 5 27.8 | 26.3).
struct Plan {
    int tiles, part_floats;
    bool apart;
    int64_t groups, cuts_at, parts_at, bytes;
};

Plan plan(int codes, int64_t B, int Hq, int Hkv, int D, int64_t max_len)
{
    Plan p{};
    const int G = Hq / Hkv;
    p.tiles = (G + kTile - 1) / kTile;
    const int heads = std::min(G, kTile);
    const int64_t units = B * Hkv * p.tiles;
    const int64_t rounds = std::max<int64_t>((max_len + kGrain - 1) / kGrain, 1) * units;
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess) dev = 0;
    const int cus = cu_count(dev);
    const int most = groups_per_cu(D, codes != PSQ_CODES_NONE);
    p.groups = std::min<int64_t>(cus * most, rounds);
    const int items = heads * D / 4, loads = (D <= 64 ? 8 : 16) * std::max(kThreads / items, 1);   // of join_parts
    p.apart = p.groups > units * (items > kThreads ? 4 : loads);
    if (p.apart) p.groups = std::min<int64_t>(cus * std::min(most, 2), rounds);
    p.part_floats = (heads * (D + 2) + 31) / 32 * 32;   // whole lines
    p.cuts_at = kCounterBytes;
    p.parts_at = p.cuts_at + (p.apart ? units * (int64_t)sizeof(Cut) + 255 : 0) / 256 * 256;
    // units of one round cannot be cut
    p.bytes = max_len <= kGrain ? 0 : p.parts_at + 2 * p.groups * p.part_floats * 4;
    return p;
}

template <int DT, int CODES, int DD, bool PART, bool SINKS = false>
int launch(const AttnArgs &a, int64_t groups, hipStream_t st)
{
    if constexpr (!SINKS)
        if (a.sinks) return launch<DT, CODES, DD, PART, true>(a, groups, st);
    // the waves' outputs, then (joining) 256 quads with their maxima and sums
    const int lds = std::max(kWaves * std::min(a.G, kTile) * (DD + 4), 6 * kThreads) * 4;
    auto *kernel = paged_attention_kernel<DT, CODES, DD, PART, SINKS>;
    if (lds > 48 * 1024) {
        static bool raised[64] = {};
        int dev = 0;
        if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return set_error(PSQ_E_DEVICE, "no current HIP device");
        if (!raised[dev]) {
            if (hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, 80 * 1024) != hipSuccess)
                return set_error(PSQ_E_DEVICE, "paged_attention: cannot raise the LDS size");
            raised[dev] = true;
        }
    }
    kernel<<<(unsigned)groups, kThreads, lds, st>>>(a);
    if (a.apart) join_parts_kernel<DT><<<dim3((unsigned)(a.B * a.Hkv * a.tiles), std::min(a.G, kTile)), kThreads, 0, st>>>(a);
    return check_launch("paged_attention");
}

template <int DT, int CODES>
int launch_dim(const AttnArgs &a, int64_t groups, hipStream_t st)
{
    if (a.D == 64) return launch<DT, CODES, 64, false>(a, groups, st);
    if (a.D == 128) return launch<DT, CODES, 128, false>(a, groups, st);
    if (a.D == 256) return launch<DT, CODES, 256, false>(a, groups, st);
    if (a.D < 64) return launch<DT, CODES, 64, true>(a, groups, st);
    if (a.D < 128) return launch<DT, CODES, 128, true>(a, groups, st);
    return launch<DT, CODES, 256, true>(a, groups, st);
}

}  // namespace
}  // namespace psq

extern "C" {

int64_t psq_paged_attention_workspace_bytes(int codes, int64_t B, int Hq, int Hkv, int D, int64_t max_len)
{
    if (B <= 0 || Hq <= 0 || Hkv <= 0 || D <= 0 || max_len <= 0 || Hq % Hkv || B > 65535) return 0;
    return psq::plan(codes, B, Hq, Hkv, D, std::min<int64_t>(max_len, 0x7fffffffLL)).bytes;
}

int psq_paged_attention_own_workspace(int codes, int64_t B, int Hq, int Hkv, int D, int64_t max_len)
{
    if (psq_paged_attention_workspace_bytes(codes, B, Hq, Hkv, D, max_len) <= 0) return 0;
    return psq::plan(codes, B, Hq, Hkv, D, std::min<int64_t>(max_len, 0x7fffffffLL)).apart;
}

int psq_paged_attention_sinks(int codes, const void *q, int dtype, int64_t q_batch, int64_t q_head, const void *k_cache,
                              const void *v_cache, const float *k_scale, const float *v_scale, int64_t num_pages, int page_size,
                              const int32_t *block_table, int64_t table_stride, int64_t table_cols, const int32_t *lengths, int64_t B,
                              int Hq, int Hkv, int D, float scale, int64_t window, int64_t sinks, int64_t max_len, void *out,
                              float *lse, void *workspace, int64_t workspace_bytes, void *stream)
{
    using namespace psq;
    const char *name = "paged_attention";
    if (B < 0 || Hq < 0 || table_cols < 0 || window < 0 || sinks < 0 || max_len < 0 || workspace_bytes < 0)
        return set_error(PSQ_E_ARG, "%s: negative size", name);
    if (sinks && !window) return set_error(PSQ_E_ARG, "%s: sinks are of a window", name);
    if (dtype != PSQ_BF16 && dtype != PSQ_F16) return set_error(PSQ_E_ARG, "%s: queries must be bf16 or f16 (dtype %d)", name, dtype);
    if (int e = check_kv_cache(name, codes, k_cache, v_cache, k_scale, v_scale, num_pages, page_size, Hkv, D)) return e;
    if (B == 0 || Hq == 0) return PSQ_OK;
    if (!q || !out || !lengths || (table_cols && !block_table)) return set_error(PSQ_E_ARG, "%s: null pointer", name);
    if (Hq % Hkv || Hq > 65535) return set_error(PSQ_E_SHAPE, "%s: %d heads do not share %d kv heads", name, Hq, Hkv);
    if (((uintptr_t)q | (uintptr_t)out) & 15 || (q_batch | q_head) & 7)
        return set_error(PSQ_E_SHAPE, "%s: queries and output must be 16-byte aligned, query strides multiples of 8", name);
    if (((uintptr_t)block_table | (uintptr_t)lengths | (uintptr_t)lse) & 3)
        return set_error(PSQ_E_SHAPE, "%s: misaligned table, lengths or lse", name);
    if (B > 65535 || table_cols > 0x3fffffffLL / page_size || B * (table_cols * page_size / kGrain + 1) > 0x7fffffffLL)
        return set_error(PSQ_E_SHAPE, "%s: %lld sequences of %lld pages are too many", name, (long long)B, (long long)table_cols);
    if ((uintptr_t)workspace & 255) return set_error(PSQ_E_SHAPE, "%s: the workspace must be 256-byte aligned", name);
    const int64_t cap = table_cols * page_size;
    const Plan p = plan(codes, B, Hq, Hkv, D, std::min(max_len, cap));
    const bool alone = !p.bytes || !workspace || workspace_bytes < p.bytes;
    const int64_t groups = alone ? B * Hkv * p.tiles : p.groups;
    if (groups > 0x7fffffffLL) return set_error(PSQ_E_SHAPE, "%s: %lld workgroups are too many", name, (long long)groups);
    if (int e = require_device()) return e;
    const AttnArgs a{(const uint16_t *)q, q_batch, q_head, (const uint8_t *)k_cache, (const uint8_t *)v_cache, k_scale, v_scale,
                     block_table, table_stride, lengths, (uint16_t *)out, lse,
                     (uint32_t *)workspace, (Cut *)((uint8_t *)workspace + p.cuts_at), (float *)((uint8_t *)workspace + p.parts_at),
                     p.part_floats, (int)num_pages, (int)cap, (int)B, page_size, Hq, Hkv, D, Hq / Hkv, p.tiles,
                     (int)std::min<int64_t>(window, cap), alone, !alone && p.apart, scale * kLog2e,
                     codes == PSQ_CODES_NONE && dtype == PSQ_F16 ? 1.0f / kF16Unit : 1.0f, (int)std::min<int64_t>(sinks, cap)};
    hipStream_t st = (hipStream_t)stream;
    auto go = [&](auto dtc) {
        constexpr int DT = decltype(dtc)::value;
        if (codes == PSQ_CODES_I8) return launch_dim<DT, PSQ_CODES_I8>(a, groups, st);
        if (codes == PSQ_CODES_E4M3) return launch_dim<DT, PSQ_CODES_E4M3>(a, groups, st);
        return launch_dim<DT, PSQ_CODES_NONE>(a, groups, st);
    };
    return dtype == PSQ_BF16 ? go(std::integral_constant<int, PSQ_BF16>{}) : go(std::integral_constant<int, PSQ_F16>{});
}

int psq_paged_attention(int codes, const void *q, int dtype, int64_t q_batch, int64_t q_head, const void *k_cache,
                        const void *v_cache, const float *k_scale, const float *v_scale, int64_t num_pages, int page_size,
                        const int32_t *block_table, int64_t table_stride, int64_t table_cols, const int32_t *lengths, int64_t B,
                        int Hq, int Hkv, int D, float scale, int64_t window, int64_t max_len, void *out, float *lse,
                        void *workspace, int64_t workspace_bytes, void *stream)
{
    return psq_paged_attention_sinks(codes, q, dtype, q_batch, q_head, k_cache, v_cache, k_scale, v_scale, num_pages, page_size, block_table,
                                     table_stride, table_cols, lengths, B, Hq, Hkv, D, scale, window, 0, max_len, out, lse, workspace,
                                     workspace_bytes, stream);
}

}  // extern "C"
