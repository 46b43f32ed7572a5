// block_attention.hpp -- attention of many rows per sequence over the paged key-value cache: the kernel of
// psq_paged_prompt_attention and psq_paged_tree_attention (block_attention.hip has the entry points).
//
//   s = scale (q . k_t) ks_t over the tokens t that the row sees,  p = softmax(s),  out = sum_t p_t vs_t v_t
//
// Rows are (token, head of a kv head's group): a tile of 128 rows of one sequence and kv head meets tiles of 64
// keys, which a workgroup of 4 waves brings to LDS once for all of them, as 16-bit elements (codes are converted
// on the way; they are exact in 16 bits).  A wave has 32 rows, one per lane in both halves (32x32x16 matrix
// instructions, fp32 accumulation).  Lane l, n = l & 31, h = l >> 5:
//   S^T = K Q^T: the lane holds row n's scores of keys 8 (i >> 2) + 4 h + (i & 3), i < 16, of each 32 keys;
//   O^T = V^T P^T: those probabilities are, as they are, the lane's part of P^T if contraction index 8 h + j of
//     keys 16 u .. stands for key 16 u + 8 (j >> 2) + 4 h + (j & 3); the transposed LDS reads deliver V^T to match.
// So softmax statistics take one exchange between the halves, and probabilities move between no lanes.
//
// Statistics are fp32.  The maximum that scores are taken off is raised only when a row's has grown by 2^8 since
// (a raise multiplies the row's whole output); probabilities are at most 2^8 then, held 2^7 times as large in f16.
// A probability enters the second product as one 16-bit number (off by half a step, as the output is), with f16
// rows on codes, whose values are bf16, as the sum of two.
//
// Many tiles of rows: a workgroup each, those with most keys first.  Few: the key tiles of all units (sequence, kv
// head, tile of rows), in their order, are cut into equal runs, one per workgroup, as many as the chip holds: the
// host needs no lengths.  A workgroup leaves its parts of cut units (two at most) in the workspace, and a second
// kernel adds them up in their order.
//
// Tiles that all rows of a wave see whole take no masks.  In the others a masked score is -inf whatever its key
// holds.  A masked value would still poison a row if it were infinite or NaN (0 * inf): sums that come out NaN are
// worked out once more, carefully, with the values that are not finite taken out of the product and counted for
// the rows that do see them.
#pragma once

#include "kv_cache.hpp"

#include <algorithm>
#include <math.h>

namespace psq {
namespace block {

constexpr int kWaves = 4, kThreads = 64 * kWaves;
constexpr int kRows = 32 * kWaves;      // of a workgroup's tile
constexpr int kKeys = 64;               // of a key tile
constexpr int kGroup = 16;              // tokens of a group (one page holds it)
constexpr int kLook = 64 / (kKeys / kGroup);   // key tiles whose pages are looked up at once
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kGrowth = 8.0f;         // log2 of what a row's maximum may grow before it is raised
constexpr int kF16Unit = 7;             // log2 of the unit of f16 probabilities

struct Args {
    const uint16_t *q;
    int64_t q_token, q_head;
    const uint8_t *kc, *vc;
    const float *ks, *vs;
    const int32_t *table;
    int64_t table_stride;
    const int32_t *lengths, *starts, *parents, *drafts;
    uint16_t *out;
    float *lse;
    float *part;           // two per run: of the unit that it goes on with, of the one that it leaves
    int runs;              // 0: units stay whole
    int least;             // key tiles of a run, at least
    int num_pages, cols, B, T, N, page, Hq, Hkv, D, G;   // T: tokens of q; N: drafts per sequence (0: prompts)
    int window, sinks;
    int flip;              // of the queries' sign bits (0x8000: negative scale)
    int mute;              // queries count as zero (scale 0)
    float scale;           // |scale| log2(e)
};

typedef short v4s __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4s *lds_v4s;

template <int DT>
__device__ __forceinline__ v16f mfma(const v4i &a, const v4i &b, const v16f &c)
{
    if constexpr (DT == PSQ_BF16)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}

// 16 bytes per lane from descriptor base + off into LDS at dst + 16 lane.  The compiler would wait for a load that
// it knows of before the next transposed LDS read, whatever place that reads; the tile loop has its own waits.
__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t rs, lds_ptr dst, uint32_t off)
{
    const uint32_t to = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)dst);
    uint32_t m0;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %3, 0 offen lds\n\ts_mov_b32 m0, %0"
                 : "=&s"(m0) : "s"(to), "v"(off), "s"(rs) : "memory");
}

// Order of N steps of READS LDS reads and MFMAS matrix instructions each: the reads of DEPTH steps go ahead.
template <int N, int READS, int DEPTH, int MFMAS = 1>
__device__ __forceinline__ void ahead()
{
    __builtin_amdgcn_sched_group_barrier(0x100, READS * DEPTH, 0);
    static_for<N - DEPTH>([](auto) {
        __builtin_amdgcn_sched_group_barrier(0x8, MFMAS, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
    });
    __builtin_amdgcn_sched_group_barrier(0x8, MFMAS * DEPTH, 0);
}

// over the two halves of the wave
__device__ __forceinline__ float half_max(float x)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __builtin_elementwise_maximum(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float half_sum(float x)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// A sequence's tokens: its rows of q (n tokens from `first`), its length, and for trees the tokens in front of the
// drafts and the drafts that there are.  b = B: the rows behind the last sequence, which see nothing.
struct Seq { int first, n, len, text, drafts; };

__device__ __forceinline__ Seq sequence(const Args &a, int b)
{
    Seq s{};
    if (a.N) {
        s.first = b * a.N, s.n = a.N, s.len = max(a.lengths[b], 0);
        s.drafts = min(a.drafts ? min(max(a.drafts[b], 0), a.N) : a.N, s.len);
        s.text = s.len - s.drafts;
    } else {
        s.first = min(max(a.starts[b], 0), a.T);
        s.n = b == a.B ? a.T - s.first : min(max(a.starts[b + 1], s.first), a.T) - s.first;
        s.len = b == a.B ? 0 : max(a.lengths[b], 0);
        s.text = s.len;
    }
    return s;
}

__device__ __forceinline__ int row_tiles(const Args &a, const Seq &s) { return (s.n * a.G + kRows - 1) / kRows; }

// The key tiles that rows r0 .. r1 of a sequence need, in a list: those of the sinks, then lo .. hi - 1.
struct Keys {
    int sinks, lo, hi;
    __device__ __forceinline__ int count() const { return sinks + hi - lo; }
    __device__ __forceinline__ int tile(int i) const { return i < sinks ? i : i - sinks + lo; }
};

__device__ __forceinline__ Keys keys_of(const Args &a, const Seq &s, int r0, int r1)
{
    // positions of the first and the last row's token
    const int p0 = a.N ? s.text : s.len - s.n + r0 / a.G, p1 = a.N ? s.len - 1 : s.len - s.n + r1 / a.G;
    Keys k;
    k.hi = max(min(p1 + 1, s.len) + kKeys - 1, 0) / kKeys;
    k.lo = a.window ? min(max(p0 - a.window + 1, 0) / kKeys, k.hi) : 0;
    k.sinks = min((a.sinks + kKeys - 1) / kKeys, k.lo);
    return k;
}

// sum of weight(i), i < count, over all lanes
template <class F>
__device__ __forceinline__ uint32_t sum_of(int count, F weight)
{
    uint32_t x = 0;
    for (int i = threadIdx.x & 63; i < count; i += 64) x += weight(i);
#pragma unroll
    for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o, 64);
    return (uint32_t)__builtin_amdgcn_readfirstlane((int)x);
}

// the i whose weight holds place `value` of the weights laid end to end, and what is in front of it
template <class F>
__device__ __forceinline__ int find(int count, uint32_t value, uint32_t &before, F weight)
{
    const int lane = threadIdx.x & 63;
    before = 0;
    for (int c = 0;; c += 64) {
        const uint32_t own = c + lane < count ? weight(c + lane) : 0;
        uint32_t to = own;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t y = __shfl_up(to, o, 64);
            to += lane >= o ? y : 0;
        }
        const uint64_t in = __ballot(value - before < to);   // (weights in front are counted off)
        if (in || c + 64 >= count) {
            const int at = in ? __builtin_ctzll(in) : 63;
            before += (uint32_t)__builtin_amdgcn_readlane((int)(to - own), at);
            return c + at;
        }
        before += (uint32_t)__builtin_amdgcn_readlane((int)to, 63);
    }
}

// 16 bytes of codes as 16 elements of DT
template <int DT, int CODES>
__device__ __forceinline__ void widen(const v4i &c, v4i (&w)[2])
{
#pragma unroll
    for (int i = 0; i < 4; i++) {
        w[i >> 1][2 * (i & 1)] = (int)code_pair<DT, CODES, 0>((uint32_t)c[i]);
        w[i >> 1][2 * (i & 1) + 1] = (int)code_pair<DT, CODES, 1>((uint32_t)c[i]);
    }
}

// DD: head dims that tiles are laid out for; PART: D < DD, the rest of a row is not there.
template <int DD>
struct Layout {
    static constexpr int PITCH = 2 * DD, TILE = kKeys * PITCH;      // bytes of a row, a tile
    static constexpr int BUFFER = 2 * TILE + 2 * kKeys * 4;         // keys, values, their scales
    // 16-byte chunk c of row r is stored at chunk c ^ kx(r) (keys), c ^ vx(r) (values): the lanes that the
    // LDS serves together then hit all banks
    static __device__ __forceinline__ int kx(int r) { return DD == 64 ? (r >> 1) & 7 : r & 15; }
    static __device__ __forceinline__ int vx(int r) { return DD == 64 ? (r >> 1 & 1) << 2 : (r & 3) << 2; }
};

// A part: sums of 4 dims of a row, [dims / 4][rows], then the rows' maxima (log2) and sums of weights (-1: sees nothing).
template <int DD>
constexpr int part_floats() { return kRows * (DD + 2); }

// Runs: the key tiles of all units laid end to end, a sequence's units (kv head, tile of rows) with as many each.
struct Runs {
    uint32_t all, runs;
    __device__ __forceinline__ uint32_t first(uint32_t w) const { return (uint32_t)uniform64((uint64_t)w * all / runs); }
    __device__ __forceinline__ uint32_t owner(uint32_t x) const { return (uint32_t)uniform64((((uint64_t)x + 1) * runs - 1) / all); }
    static __device__ __forceinline__ uint64_t uniform64(uint64_t x)
    {
        return (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)x);
    }
};

__device__ __forceinline__ int key_tiles(const Args &a, const Seq &s) { return max(keys_of(a, s, 0, s.n * a.G - 1).count(), 1); }

__device__ __forceinline__ uint32_t weight_of(const Args &a, int b)
{
    const Seq s = sequence(a, b);
    return s.n ? (uint32_t)row_tiles(a, s) * a.Hkv * key_tiles(a, s) : 0;
}

__device__ __forceinline__ Runs runs_of(const Args &a, int count)
{
    Runs r;
    r.all = sum_of(count, [&](int b) { return weight_of(a, b); });
    r.runs = min((uint32_t)a.runs, max(r.all / (uint32_t)a.least, 1u));
    return r;
}

template <int DT, int CODES, int DD, bool PART>
__global__ void __launch_bounds__(kThreads, DD > 128 ? 1 : 2)
block_attention_kernel(Args a)
{
    using L = Layout<DD>;
    constexpr int ES = CODES == PSQ_CODES_NONE ? 2 : 1;
    constexpr int PVT = CODES == PSQ_CODES_NONE ? DT : PSQ_BF16;   // of the second product
    constexpr bool PAIR = CODES != PSQ_CODES_NONE && DT == PSQ_F16;
    constexpr int NC = DD / 16, ND = DD / 32;
    constexpr int CH = DD / 8;                        // 16-byte chunks of a row of 16-bit elements
    extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 31, h = lane >> 5;
    const int D = PART ? a.D : DD, per_page = a.page / kGroup;

    // ---- the workgroup's units
    const int count = a.N ? a.B : a.B + 1;
    int b, r0, first = 0, tiles = 0;       // key tiles first .. of the unit's list are the workgroup's
    uint32_t hk, x = 0, end = 0;
    Runs runs{};
    if (!a.runs) {
        auto tiles_of = [&](int b) { return (uint32_t)row_tiles(a, sequence(a, b)); };
        const uint32_t all = sum_of(count, tiles_of), units = all * a.Hkv;
        if (blockIdx.x >= units) return;
        // Workgroups of an XCD share a kv head's keys and values in its L2; the rows that see most go first.
        const uint32_t rank = (uint32_t)xcd_rank(blockIdx.x, units);
        hk = rank / all;
        uint32_t before;
        const uint32_t place = all - 1 - (rank - hk * all);
        b = __builtin_amdgcn_readfirstlane(find(count, place, before, tiles_of));
        r0 = (int)(place - before) * kRows;
    } else {
        runs = runs_of(a, count);
        const uint32_t w = (uint32_t)xcd_rank(blockIdx.x, a.runs);
        if (w >= runs.runs) return;
        x = runs.first(w), end = runs.first(w + 1);
    }

    do {
    bool whole = true;
    if (a.runs) {
        uint32_t before;
        b = __builtin_amdgcn_readfirstlane(find(count, x, before, [&](int b) { return weight_of(a, b); }));
        const Seq s = sequence(a, b);
        const uint32_t each = (uint32_t)key_tiles(a, s), per = (uint32_t)row_tiles(a, s), unit = (x - before) / each;
        hk = unit / per, r0 = (int)(unit - hk * per) * kRows;
        first = (int)(x - before - unit * each);
        tiles = (int)min(each - first, end - x);
        whole = tiles == (int)each;
        x += tiles;
    }
    const Seq s = sequence(a, b);
    const int rows = min(s.n * a.G - r0, kRows);
    const Keys keys = a.runs ? keys_of(a, s, 0, s.n * a.G - 1) : keys_of(a, s, r0, r0 + rows - 1);
    const Keys own = keys_of(a, s, r0, r0 + rows - 1);
    const int last = min(first + (a.runs ? tiles : keys.count()), keys.count());
    // the next tile of the list from i on that these rows need
    auto next_of = [&](int i) {
        const int t = i < last ? keys.tile(i) : own.hi;
        if (t >= own.hi) return last;
        return t >= own.lo || t * kKeys < a.sinks ? i : min(i + own.lo - t, last);
    };

    // ---- the lane's row
    const int wrow = r0 + 32 * wave, row = wrow + n, mine = min(max(rows - 32 * wave, 0), 32);
    const bool valid = n < mine;
    const int token = valid ? row / a.G : 0, head = (int)hk * a.G + (valid ? row - token * a.G : 0);
    int pos = -1;                       // -1: sees nothing
    uint64_t way = 0;                   // drafts that the row sees
    if (a.N) {
        // lane i: draft i, its way to the text by steps of doubled length
        const int p = lane < s.drafts ? a.parents[b * a.N + lane] : -1;
        int up = p >= 0 && p < lane ? p : -1;
        uint64_t path = 1ull << lane;
#pragma unroll
        for (int o = 0; o < 6; o++) {
            const int from = up < 0 ? lane : up;
            const uint32_t lo = __shfl((uint32_t)path, from, 64), hi = __shfl((uint32_t)(path >> 32), from, 64);
            const int next = __shfl(up, from, 64);
            if (up >= 0) path |= (uint64_t)hi << 32 | lo, up = next;
        }
        const int depth = __popcll(path) - 1, at = token < 64 ? token : 0;
        if (a.window) {
            // the drafts on the way that are in the window or among the sinks: those of the nearest depths
            uint64_t near = 0;
            for (int i = 0; i < 64; i++) {
                const int d = __builtin_amdgcn_readlane(depth, i);
                if ((path >> i & 1) && (d > depth - a.window || s.text + d < a.sinks)) near |= 1ull << i;
            }
            path = near;
        }
        way = (uint64_t)__shfl((uint32_t)(path >> 32), at, 64) << 32 | __shfl((uint32_t)path, at, 64);
        const int d = __shfl(depth, at, 64);
        if (valid && token < s.drafts) pos = s.text + d;
        else way = 0;
    } else if (valid) {
        pos = s.len - s.n + token;
    }
    const int low = a.window ? pos - a.window + 1 : 0;
    // of the wave: keys up to full_hi, from full_lo or among the sinks, are seen by all rows; keys past any_hi, or before
    // any_lo and past the sinks, by none
    const int w0 = a.N ? s.text : s.len - s.n + wrow / a.G, w1 = a.N ? s.len - 1 : s.len - s.n + (wrow + max(mine, 1) - 1) / a.G;
    const int full_hi = a.N ? s.text - 1 : w0, full_lo = a.window ? w1 - a.window + 1 : 0, any_hi = w1, any_lo = a.window ? w0 - a.window + 1 : 0;

    v4i qf[NC];
    {
        const uint16_t *q = a.q + (int64_t)(s.first + token) * a.q_token + head * a.q_head;
        const uint32_t flip = (uint32_t)a.flip << 16 | (uint32_t)a.flip;
#pragma unroll
        for (int c = 0; c < NC; c++) {
            const int d = 16 * c + 8 * h;
            qf[c] = v4i{0, 0, 0, 0};
            if (valid && !a.mute && (!PART || d < D)) qf[c] = *(const v4i *)(q + d) ^ (int)flip;
        }
    }

    // ---- bringing key tiles to LDS: wave w has group w of a tile's four
    const int row_bytes = D * ES;
    uint32_t grp;          // lane 4 i + g: pool group of tile base + i's group g
    uint64_t there, wild;  // tokens that are there; whose page is not
    int base = 0;
    auto look = [&](int i) {
        base = i;
        const int j = i + (lane >> 2), t = j < last ? keys.tile(j) * kKeys + kGroup * (lane & 3) : s.len;
        bool in = t < s.len, out = false;
        grp = 0;
        if (in) {
            const uint32_t g = (uint32_t)t / kGroup, col = g / (uint32_t)per_page;
            const int pg = col < (uint32_t)a.cols ? a.table[b * a.table_stride + col] : -1;
            out = pg < 0 || pg >= a.num_pages;
            grp = out ? 0 : ((uint32_t)pg * a.Hkv + hk) * per_page + (g - col * per_page);
        }
        there = __ballot(in && !out);
        wild = __ballot(out);
    };
    constexpr int CP = DD / 16 * kGroup / 64;     // 16-byte pieces of codes that a lane has of its wave's group
    v4i kreg[ES == 1 ? CP : 1], vreg[ES == 1 ? CP : 1];
    float sreg = 0.0f;
    uint32_t koff[ES == 2 ? kGroup * L::PITCH / 1024 : 1], voff[ES == 2 ? kGroup * L::PITCH / 1024 : 1];
    if constexpr (ES == 2) {
#pragma unroll
        for (int i = 0; i < kGroup * L::PITCH / 1024; i++) {
            const int at = i * 64 + lane, r = at / CH, c = at % CH, ck = c ^ L::kx(r), cv = c ^ L::vx(r);
            koff[i] = (uint32_t)(r * row_bytes + (PART && ck * 8 >= D ? 0 : ck * 16));
            voff[i] = (uint32_t)(r * row_bytes + (PART && cv * 8 >= D ? 0 : cv * 16));
        }
    }
    auto stage = [&](int i, uint8_t *buf) {       // tile i's loads (codes: into registers)
        const int bit = 4 * (i - base) + wave;
        const bool here = there >> bit & 1;
        const int64_t g = (uint32_t)__builtin_amdgcn_readlane((int)grp, bit);
        if constexpr (ES == 2) {
            if (!here) return;
            const __amdgpu_buffer_rsrc_t rk = raw_rsrc(a.kc + g * (kGroup * row_bytes)), rv = raw_rsrc(a.vc + g * (kGroup * row_bytes));
            uint8_t *k = buf + wave * kGroup * L::PITCH, *v = k + L::TILE;
#pragma unroll
            for (int j = 0; j < kGroup * L::PITCH / 1024; j++) {
                dma16(rk, (lds_ptr)(k + 1024 * j), koff[j]);
                dma16(rv, (lds_ptr)(v + 1024 * j), voff[j]);
            }
        } else {
            // places behind the sequence hold zeros
            const int left = here ? s.len - (keys.tile(i) * kKeys + kGroup * wave) : 0;
            const uint8_t *k = a.kc + g * (kGroup * row_bytes), *v = a.vc + g * (kGroup * row_bytes);
#pragma unroll
            for (int j = 0; j < CP; j++) {
                const int at = 64 * j + lane, r = at / (DD / 16), c = at % (DD / 16);
                kreg[j] = vreg[j] = v4i{0, 0, 0, 0};
                if (r < left && (!PART || c * 16 < D)) {
                    kreg[j] = *(const v4i *)(k + r * row_bytes + c * 16);
                    vreg[j] = *(const v4i *)(v + r * row_bytes + c * 16);
                }
            }
            sreg = 0.0f;
            if (lane < 32 && n % kGroup < left) sreg = (lane < kGroup ? a.ks : a.vs)[g * kGroup + n % kGroup];
        }
    };
    // values of 16 bits where no tokens are (behind the sequence, on pages that are not there): zeros, by the wave that
    // brings the others of the group
    auto clear = [&](int t0, uint32_t astray, uint8_t *buf) {
        const int left = astray >> wave & 1 ? 0 : s.len - t0 - kGroup * wave;
        uint8_t *v = buf + L::TILE + wave * kGroup * L::PITCH;
        for (int at = lane; at < kGroup * CH; at += 64)
            if (at / CH >= left) *(v4i *)(v + at * 16) = v4i{0, 0, 0, 0};
    };
    auto deliver = [&](uint8_t *buf) {            // codes from registers to LDS
        if constexpr (ES == 1) {
            uint8_t *k = buf + wave * kGroup * L::PITCH, *v = k + L::TILE;
#pragma unroll
            for (int j = 0; j < CP; j++) {
                const int at = 64 * j + lane, r = at / (DD / 16), c = 2 * (at % (DD / 16));
                v4i w[2];
                widen<DT, CODES>(kreg[j], w);
                *(v4i *)(k + r * L::PITCH + (c ^ L::kx(r)) * 16) = w[0];
                *(v4i *)(k + r * L::PITCH + ((c + 1) ^ L::kx(r)) * 16) = w[1];
                widen<PVT, CODES>(vreg[j], w);
                *(v4i *)(v + r * L::PITCH + (c ^ L::vx(r)) * 16) = w[0];
                *(v4i *)(v + r * L::PITCH + ((c + 1) ^ L::vx(r)) * 16) = w[1];
            }
            float *sc = (float *)(buf + 2 * L::TILE);
            if (lane < 32) sc[(lane < kGroup ? 0 : kKeys) + wave * kGroup + n % kGroup] = sreg;
        }
    };

    // ---- a key tile of the wave's rows
    v16f o[ND];
    float run_m, run_l;    // the maximum that scores are taken off (in their own units); the lane's part of the sum
    const uint32_t klane = n * L::PITCH + ((h ^ L::kx(n)) << 4);
    const uint32_t vlane = (4 * h + (n & 15) / 4) * L::PITCH + ((((n >> 4) << 1 | (n & 3) >> 1) ^ L::vx((n & 15) / 4)) << 4) + (n & 1) * 8;
    auto compute = [&](auto carefulc, int tile0, bool edge, uint32_t astray, const uint8_t *buf) {
        constexpr bool CAREFUL = decltype(carefulc)::value;
        v16f sc[2];
#pragma unroll
        for (int t = 0; t < 2; t++) {
#pragma unroll
            for (int i = 0; i < 16; i++) sc[t][i] = 0.0f;
#pragma unroll
            for (int c = 0; c < NC; c++)
                if (!PART || 16 * c < D) sc[t] = mfma<DT>(*(const v4i *)(buf + 32 * t * L::PITCH + (klane ^ (c << 5))), qf[c], sc[t]);
        }
        if constexpr (!PART) ahead<2 * NC, 1, 4>();
        const float *scales = (const float *)(buf + 2 * L::TILE);
        if constexpr (ES == 1) {
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    const v4f x = *(const v4f *)(scales + 32 * t + 2 * i + 4 * h);
#pragma unroll
                    for (int j = 0; j < 4; j++) sc[t][i + j] *= x[j];
                }
        }
        uint32_t seen = 0;
        int t0 = tile0;
        if (CAREFUL || edge) {
            asm volatile("" : "+v"(t0));   // (a branch, not selects that all tiles pay for)
            // key 32 t + 8 (i >> 2) + (i & 3) of the lane's against these
            const int at = t0 + 4 * h, to = min(pos, s.text - 1) - at, from = low - at, sinks = a.sinks - at, text = s.text - at;
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const int k = 32 * t + 8 * (i >> 2) + (i & 3);
                    bool see = (k <= to) & ((k >= from) | (k < sinks));
                    if (a.N) {
                        const uint32_t draft = (uint32_t)(k - text);
                        see |= (draft < 64) & ((uint32_t)(way >> (draft & 63)) & 1);
                    }
                    if (astray >> (2 * t + (i >> 3)) & 1) sc[t][i] = NAN;    // its page is not there
                    if (!see) sc[t][i] = -INFINITY;
                    if (CAREFUL) seen |= (uint32_t)see << (16 * t + i);
                }
        }
        // (NaN wins; it raises nothing, and the row's sum will be NaN)
        float top = __builtin_elementwise_maximum(sc[0][0], sc[1][0]);
#pragma unroll
        for (int i = 1; i < 16; i++) top = __builtin_elementwise_maximum(top, __builtin_elementwise_maximum(sc[0][i], sc[1][i]));
        top = half_max(top);
        // (a maximum that comes first, or is raised from -inf, is any growth)
        const bool raise = top * a.scale > run_m * a.scale + kGrowth;
        if (__any(raise)) {
            const float next = raise ? top : run_m;    // (each row by itself: its result does not depend on the others')
            float keep = next == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((run_m - next) * a.scale);
            if (CAREFUL) keep = fmaxf(keep, 0x1p-126f);   // (an infinite sum stays one)
            run_m = next;
            run_l *= keep;
#pragma unroll
            for (int d = 0; d < ND; d++)
#pragma unroll
                for (int i = 0; i < 16; i++) o[d][i] *= keep;
        }
        const float ref = (PVT == PSQ_F16 ? kF16Unit : 0) - (run_m == -INFINITY ? 0.0f : run_m * a.scale);
        v4i ph[4], pl[PAIR ? 4 : 1];
#pragma unroll
        for (int t = 0; t < 2; t++) {
#pragma unroll
            for (int i = 0; i < 16; i++) {
                sc[t][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][i], a.scale, ref));
                run_l += sc[t][i];
            }
            if constexpr (ES == 1) {
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    const v4f x = *(const v4f *)(scales + kKeys + 32 * t + 2 * i + 4 * h);
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        sc[t][i + j] *= x[j];
                        if (CAREFUL && !(seen >> (16 * t + i + j) & 1)) sc[t][i + j] = 0.0f;   // (its scale may be infinite)
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int d = 0; d < 4; d++) {
                    const float x = sc[t][8 * u + 2 * d], y = sc[t][8 * u + 2 * d + 1];
                    const uint32_t p = pack_half2<PVT>(x, y);
                    ph[2 * t + u][d] = (int)p;
                    if constexpr (PAIR) pl[2 * t + u][d] = (int)pack_half2<PVT>(x - half_to_f32<PVT>(p), y - half_to_f32<PVT>(p >> 16));
                }
        }
        const uint8_t *vb = buf + L::TILE;
#pragma unroll
        for (int u = 0; u < 4; u++) {
#pragma unroll
            for (int d = 0; d < ND; d++) {
                if (PART && 32 * d >= D) break;
                const uint8_t *src = vb + 16 * u * L::PITCH + (vlane ^ (d << 6));
                const v4s x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)src);
                const v4s y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)(src + 8 * L::PITCH));
                const v2i xi = __builtin_bit_cast(v2i, x), yi = __builtin_bit_cast(v2i, y);
                v4i vf{xi[0], xi[1], yi[0], yi[1]};
                if constexpr (CAREFUL) {
                    constexpr uint32_t EXP = PVT == PSQ_BF16 ? 0x7f80 : 0x7c00, ONE = PVT == PSQ_BF16 ? 0x3f80 : 0x3c00;
                    v4i up, down, look;     // ones where a value is +inf, is -inf (NaN: both); where a key is seen
                    bool any = false;
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        uint32_t c = 0, pu = 0, pd = 0, ps = 0;
#pragma unroll
                        for (int k = 0; k < 2; k++) {
                            const uint32_t w = (uint32_t)vf[e] >> (16 * k) & 0xffff;
                            const bool odd = (w & EXP) == EXP, nan = odd & ((w & (EXP ^ 0x7fff)) != 0);
                            any |= odd;
                            c |= (odd ? 0 : w) << (16 * k);
                            pu |= (odd & (nan | !(w & 0x8000)) ? ONE : 0) << (16 * k);
                            pd |= (odd & (nan | ((w & 0x8000) != 0)) ? ONE : 0) << (16 * k);
                            ps |= (seen >> (8 * u + 2 * e + k) & 1 ? ONE : 0) << (16 * k);
                        }
                        vf[e] = (int)c, up[e] = (int)pu, down[e] = (int)pd, look[e] = (int)ps;
                    }
                    if (__any(any)) {
                        v16f zero = {};
                        const v16f more = mfma<PVT>(up, look, zero), less = mfma<PVT>(down, look, zero);
#pragma unroll
                        for (int i = 0; i < 16; i++) {
                            if (more[i] > 0.0f) o[d][i] += INFINITY;
                            if (less[i] > 0.0f) o[d][i] -= INFINITY;
                        }
                    }
                }
                o[d] = mfma<PVT>(vf, ph[u], o[d]);
                if constexpr (PAIR) o[d] = mfma<PVT>(vf, pl[u], o[d]);
            }
        }
        if constexpr (!PART && !CAREFUL) ahead<4 * ND, 2, 4, PAIR ? 2 : 1>();
    };

    // All of the workgroup's key tiles of the unit.
    auto pass = [&](auto carefulc) {
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
            for (int i = 0; i < 16; i++) o[d][i] = 0.0f;
        run_m = -INFINITY, run_l = 0.0f;
        uint32_t here = 0, next = L::BUFFER;   // offsets of the buffers
        uint32_t astray = 0;
        __syncthreads();                       // LDS is free
        int i = next_of(first);
        if (i < last) {
            look(i);
            stage(i, smem);
            astray = (uint32_t)wild & 15;
            deliver(smem);
        }
        while (i < last) {
            const int j = next_of(i + 1), t0 = keys.tile(i) * kKeys, t1 = t0 + kKeys - 1;
            wait_vmcnt<0>();
            if (ES == 2 && (t1 >= s.len || astray)) clear(t0, astray, smem + here);
            stage_barrier();                   // the tile is here, and the one before it is done with
            uint32_t gone = 0;
            if (j < last) {
                if (j - base >= kLook) look(j);
                stage(j, smem + next);
                gone = (uint32_t)(wild >> (4 * (j - base))) & 15;
            }
            if (mine > 0 && t0 <= any_hi && (t1 >= any_lo || t0 < a.sinks))
                compute(carefulc, t0, !(t1 <= full_hi && (t0 >= full_lo || t1 < a.sinks) && !astray), astray, smem + here);
            if (j < last) deliver(smem + next);
            astray = gone, i = j;
            std::swap(here, next);
        }
    };
    pass(std::false_type{});
    float any = 0.0f;
#pragma unroll
    for (int d = 0; d < ND; d++)
        if (!PART || 32 * d < D)
#pragma unroll
            for (int i = 0; i < 16; i++) any = __builtin_fmaf(o[d][i], 0.0f, any);
    if (__syncthreads_or(any != any)) pass(std::true_type{});

    // ---- the rows' outputs, or the part of them
    run_l = half_sum(run_l);
    const float top = run_m * a.scale - (PVT == PSQ_F16 ? kF16Unit : 0);     // (in log2, the weights' unit taken off)
    const int64_t at = (int64_t)(s.first + token) * a.Hq + head;
    if (valid && whole) {
        const float r = pos < 0 ? 0.0f : 1.0f / run_l;    // (sees nothing: zeros)
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const int dim = 32 * d + 2 * i + 4 * h;
                if (!PART || dim < D)
                    *(v2i *)(a.out + at * D + dim) = v2i{(int)pack_half2<DT>(o[d][i] * r, o[d][i + 1] * r), (int)pack_half2<DT>(o[d][i + 2] * r, o[d][i + 3] * r)};
            }
        if (a.lse && h == 0) a.lse[at] = pos < 0 ? -INFINITY : top * kLn2 + logf(run_l);
    } else if (valid) {
        float *part = a.part + (2 * (int64_t)xcd_rank(blockIdx.x, a.runs) + (first == 0)) * part_floats<DD>();
        const int r = 32 * wave + n;
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
            for (int i = 0; i < 16; i += 4)
                ((v4f *)part)[(8 * d + i / 2 + h) * kRows + r] = v4f{o[d][i], o[d][i + 1], o[d][i + 2], o[d][i + 3]};
        if (h == 0) part[kRows * DD + r] = top, part[kRows * (DD + 1) + r] = pos < 0 ? -1.0f : run_l;
    }
    } while (x < end);
}

// Adds up the parts of a cut unit: a workgroup has 1024 / DD of its rows, a thread one row's 4 dims.
template <int DT, int DD>
__global__ void __launch_bounds__(kThreads)
join_kernel(Args a)
{
    constexpr int kJoin = 1024 / DD, U = 8;
    const int count = a.N ? a.B : a.B + 1;
    auto units_of = [&](int b) { return (uint32_t)row_tiles(a, sequence(a, b)) * a.Hkv; };
    if (blockIdx.x >= sum_of(count, units_of)) return;
    uint32_t before;
    const int b = __builtin_amdgcn_readfirstlane(find(count, blockIdx.x, before, units_of));
    const Seq s = sequence(a, b);
    const uint32_t unit = blockIdx.x - before, each = (uint32_t)key_tiles(a, s), per = (uint32_t)row_tiles(a, s), hk = unit / per;
    const int r0 = (int)(unit - hk * per) * kRows, r = (int)blockIdx.y * kJoin + (threadIdx.x & (kJoin - 1)), quad = threadIdx.x / kJoin;
    const Runs runs = runs_of(a, count);
    const uint32_t x = sum_of(b, [&](int b) { return weight_of(a, b); }) + unit * each;
    const uint32_t w0 = runs.owner(x), parts = runs.owner(x + each - 1) - w0 + 1;
    if (parts == 1 || r0 + r >= s.n * a.G || 4 * quad >= a.D) return;
    float M = -INFINITY, L = 0.0f;
    v4f acc = {0, 0, 0, 0};
    bool none = false;
    for (uint32_t p0 = 0; p0 < parts; p0 += U) {
        v4f y[U];
        float m[U], l[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const uint32_t p = p0 + u;
            y[u] = v4f{0, 0, 0, 0}, m[u] = -INFINITY, l[u] = 0.0f;
            if (p < parts) {
                const float *part = a.part + (2 * (int64_t)(w0 + p) + (p == 0)) * part_floats<DD>();
                y[u] = ((const v4f *)part)[quad * kRows + r];
                m[u] = part[kRows * DD + r], l[u] = part[kRows * (DD + 1) + r];
            }
        }
        float to = M;
#pragma unroll
        for (int u = 0; u < U; u++) to = fmaxf(to, m[u]);
        // (2^-126 and not less: an infinite sum stays one)
        auto scale_to = [&](float from) { return fmaxf(__builtin_amdgcn_exp2f(from - (to == -INFINITY ? 0.0f : to)), 0x1p-126f); };
        const float e = scale_to(M);
        L *= e, M = to;
#pragma unroll
        for (int c = 0; c < 4; c++) acc[c] *= e;
#pragma unroll
        for (int u = 0; u < U; u++) {
            const float f = scale_to(m[u]);
            none |= l[u] < 0.0f;
            L += l[u] * f;
#pragma unroll
            for (int c = 0; c < 4; c++) acc[c] += y[u][c] * f;
        }
    }
    const int row = r0 + r, token = row / a.G;
    const int64_t at = (int64_t)(s.first + token) * a.Hq + (int)hk * a.G + (row - token * a.G);
    const float i = none ? 0.0f : 1.0f / L;
    *(v2i *)(a.out + at * a.D + 4 * quad) = v2i{(int)pack_half2<DT>(acc[0] * i, acc[1] * i), (int)pack_half2<DT>(acc[2] * i, acc[3] * i)};
    if (a.lse && quad == 0) a.lse[at] = none ? -INFINITY : M * kLn2 + logf(L);
}

template <int DT, int CODES, int DD, bool PART>
int launch(const Args &a, unsigned groups, hipStream_t st)
{
    auto *kernel = block_attention_kernel<DT, CODES, DD, PART>;
    const int lds = 2 * Layout<DD>::BUFFER;
    static bool raised[64] = {};
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return set_error(PSQ_E_DEVICE, "no current HIP device");
    if (!raised[dev]) {
        if (hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess)
            return set_error(PSQ_E_DEVICE, "block attention: cannot raise the LDS size");
        raised[dev] = true;
    }
    kernel<<<a.runs ? a.runs : groups, kThreads, lds, st>>>(a);
    if (a.runs) join_kernel<DT, DD><<<dim3(groups, kRows / (1024 / DD)), kThreads, 0, st>>>(a);
    return check_launch("block attention");
}

template <int DT, int CODES>
int launch_dim(const Args &a, unsigned groups, hipStream_t st)
{
    if (a.D == 64) return launch<DT, CODES, 64, false>(a, groups, st);
    if (a.D == 128) return launch<DT, CODES, 128, false>(a, groups, st);
    if (a.D == 256) return launch<DT, CODES, 256, false>(a, groups, st);
    if (a.D < 64) return launch<DT, CODES, 64, true>(a, groups, st);
    if (a.D < 128) return launch<DT, CODES, 128, true>(a, groups, st);
    return launch<DT, CODES, 256, true>(a, groups, st);
}

// by element type of the queries and kind of cache, each compiled in a file of its own
int launch_bf16(const Args &a, unsigned groups, hipStream_t st);
int launch_f16(const Args &a, unsigned groups, hipStream_t st);
int launch_bf16_i8(const Args &a, unsigned groups, hipStream_t st);
int launch_f16_i8(const Args &a, unsigned groups, hipStream_t st);
int launch_bf16_fp8(const Args &a, unsigned groups, hipStream_t st);
int launch_f16_fp8(const Args &a, unsigned groups, hipStream_t st);

}  // namespace block
}  // namespace psq
