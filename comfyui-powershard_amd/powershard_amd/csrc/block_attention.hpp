// block_attention.hpp -- attention of many rows per sequence over the paged key-value cache: the kernel of
// psq_paged_prompt_attention and psq_paged_tree_attention (block_attention.hip has the entry points).
//
//   s = scale (q . k_t) ks_t over the tokens t that the row sees,  p = softmax(s),  out = sum_t p_t vs_t v_t
//
// Rows are (token, head of a kv head's group): a tile of 32 W rows of one sequence and kv head meets tiles of 64
// keys, which the workgroup of W waves brings to LDS once for all of them, as 16-bit elements.  W is 4; 8 for codes of
// at most 128 dims, which are loaded as they are and widened there (they are exact in 16 bits).  A wave has 32 rows, one
// per lane in both halves (32x32x16 matrix instructions, fp32 accumulation).  Lane l, n = l & 31, h = l >> 5:
//   S^T = K Q^T: the lane holds row n's scores of keys 8 (i >> 2) + 4 h + (i & 3), i < 16, of each 32 keys;
//   O^T = V^T P^T: those probabilities are, as they are, the lane's part of P^T if contraction index 8 h + j of
//     keys 16 u .. stands for key 16 u + 8 (j >> 2) + 4 h + (j & 3); the transposed LDS reads deliver V^T to match.
// So softmax statistics take one exchange between the halves, and probabilities move between no lanes.
//
// Statistics are fp32.  The maximum that scores are taken off is raised only when a row's has grown by 2^8 since
// (a raise multiplies the row's whole output); probabilities are at most 2^8 then, held 2^7 times as large in f16.
// A probability enters the second product as one 16-bit number, off by half a step as the output is (bf16 2^-8, f16 2^-11; on
// codes times its value's scale, in bf16): an output is off by 1.1 to 1.4 times its rounding alone (relative root
// mean square against 64 bits: bf16 0.0017 -> 0.0018 to 0.0023, f16 0.00021 -> 0.00027).  A second number for the rest
// makes 48 products of 32 and some 100 more vector instructions a tile (us, one | two: 8191 tokens bf16 760 | 996, the f16
// window 548 | 697, 512 on 64977 bf16 on int8 916 | 1164, trees of 24 on int8 289 | 322, of 64 on e4m3 361 | 435).  f16 rows on
// codes, whose values are bf16, have it: one bf16 number would be off by 8 times their output's half step.  So has the
// one-token kernel, which waits for memory, for all types.
//
// Many tiles of rows: a workgroup each, those with most keys first.  Few: the key tiles of all units (sequence, kv
// head, tile of rows), in their order, are cut into equal runs, one per workgroup, as many as the chip holds: the
// host needs no lengths.  A workgroup leaves its parts of cut units (two at most) in the workspace, and a second
// kernel adds them up in their order.  plan() chooses, and has times of both.
//
// Tiles come by loads that go to LDS past the registers, some tiles ahead, in rings; the loop waits for them by count.
// The scores of the next tile are worked out while the weights of this one are: matrix and vector instructions
// alternate in one stream, with one barrier a tile.  Bound by the two kinds in turn, not by memory: of a SIMD's cycles the matrix
// unit is busy for 49% and the vector unit for 49% (8191 tokens, bf16; dims of 64, f16 26% and 63%; f16 on int8 40% and
// 56%), so what one wave does in the other's shadow is little, although two share a SIMD.  Per 32 rows x 64 keys x
// 128 dims, 16 bits, beside 32 products of 32 cycles: 155 vector instructions, 32 of them exponentials (188 with what comes
// in front of the loop and behind it), and 107 scalar ones.  Measured: 8191 tokens, 40 heads on 8 of 128, bf16, causal: 690
// to 750 us on several cards, 915 to 1000 TFLOP/s (a library product of 16384^3: 1567); 512 tokens on 64977, f16 on int8:
// 1128 us, 608; 7 prompts with a window of 1024, f16, dims of 64: 519 us, 510; trees of 24 on 61 sequences of up to 4096,
// int8: 288 us; a tree of 16 on 4000: 28.
// The loop has no registers to spare (256 a lane, 512 for dims above 128).  A tile step reloads from scratch, and waits with that
// for all loads before: nothing on 16 bits up to dims of 64, and for bf16 rows on codes above that up to 128; 1 to 3 words
// for the other types up to 128; above, 1 to 8 on 16 bits and 14 to 20 on codes.
// Tried without gain: half the barriers, deeper rings, loads by one wave, wave priorities, chains of products interleaved.
//
// Tiles that all rows of a wave see whole take no masks.  In the others a masked score is -inf whatever its key
// holds.  A masked value would still poison a row if it were infinite or NaN (0 * inf): sums that come out NaN are
// worked out once more, carefully, with the values that are not finite taken out of the product and counted for
// the rows that do see them.
#pragma once

#include "kv_cache.hpp"

#include <algorithm>
#include <math.h>

#define PSQ_INLINE __attribute__((always_inline))   // lambdas over register arrays: a call would put these in memory

namespace psq {
namespace block {

constexpr int kThreads = 256;           // of the joining kernel
constexpr int kKeys = 64;               // of a key tile
constexpr int kGroup = 16;              // tokens of a group (one page holds it)
constexpr int kLook = 64 / (kKeys / kGroup);   // key tiles whose pages are looked up at once
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kGrowth = 8.0f;         // log2 of what a row's maximum may grow before it is raised
constexpr int kF16Unit = 7;             // log2 of the unit of f16 probabilities
constexpr uint32_t kPast = 0x40000000;  // an offset past every group of a pool

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
    int rows;              // of a workgroup's tile, 32 a wave
    int least;             // key tiles of a run, at least
    int num_pages, cols, B, T, N, page, Hq, Hkv, D, G;   // T: tokens of q; N: drafts per sequence (0: prompts)
    int window, sinks;
    int flip;              // of the queries' sign bits (0x8000: negative scale)
    int mute;              // queries count as zero (scale 0)
    float scale;           // |scale| log2(e)
};

typedef short v4s __attribute__((ext_vector_type(4)));
// T at an LDS address
template <class T>
__device__ __forceinline__ __attribute__((address_space(3))) T *at_lds(uint32_t at)
{
    return (__attribute__((address_space(3))) T *)(uintptr_t)at;
}

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
__device__ __forceinline__ void dma16(const v4i &rs, uint32_t dst, uint32_t off)
{
    const uint32_t to = (uint32_t)__builtin_amdgcn_readfirstlane((int)dst);
    uint32_t m0;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %3, 0 offen lds\n\ts_mov_b32 m0, %0"
                 : "=&s"(m0) : "s"(to), "v"(off), "s"(rs) : "memory");
}

// 4 bytes per lane
__device__ __forceinline__ void dma4(const v4i &rs, uint32_t dst, uint32_t off)
{
    const uint32_t to = (uint32_t)__builtin_amdgcn_readfirstlane((int)dst);
    uint32_t m0;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tbuffer_load_dword %2, %3, 0 offen lds\n\ts_mov_b32 m0, %0"
                 : "=&s"(m0) : "s"(to), "v"(off), "s"(rs) : "memory");
}

// x, in a way that what follows from it is worked out here again and not kept in registers, which are short.
template <class T>
__device__ __forceinline__ T again(T x)
{
    asm volatile("" : "+v"(x));
    return x;
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
    // (of a length far past the table no row sees less than one token there: a shorter one that does the same bounds
    // the work, and sums of positions)
    auto length = [&](int n) { return min(max(a.lengths[b], 0), a.cols * a.page + n + kKeys); };
    if (a.N) {
        s.first = b * a.N, s.n = a.N, s.len = length(a.N);
        s.drafts = min(a.drafts ? min(max(a.drafts[b], 0), a.N) : a.N, s.len);
        s.text = s.len - s.drafts;
    } else {
        s.first = min(max(a.starts[b], 0), a.T);
        s.n = b == a.B ? a.T - s.first : min(max(a.starts[b + 1], s.first), a.T) - s.first;
        s.len = b == a.B ? 0 : length(s.n);
        s.text = s.len;
    }
    return s;
}

__device__ __forceinline__ int row_tiles(const Args &a, const Seq &s) { return (s.n * a.G + a.rows - 1) / a.rows; }

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

// DD: head dims that tiles are laid out for; W: waves of a workgroup; ES: bytes of a cached element.
// Keys and values have rings of RK and RV buffers.  While a tile's weights meet its values, the next one's keys are read, and
// loaded are the keys of the tile DK behind it and the values of that DV behind it.  A barrier comes every STEPS tiles
// (two where the LDS holds eight buffers for two workgroups).
// Codes (RAW) are loaded as they are, tiles up to RR behind, each by the wave that widens it later; wide heads' go
// through registers.
template <int DD, int W, int ES>
struct Layout {
    static constexpr bool RAW = ES == 1 && DD <= 128;
    static constexpr int PITCH = 2 * DD, TILE = kKeys * PITCH;          // bytes of a row, a tile
    static constexpr int BUFFER = TILE + (ES == 2 ? 0 : PITCH > 256 ? PITCH : 256);   // and its scales; whole rows
    static constexpr int STEPS = ES == 2 && DD == 64 ? 2 : 1;
    static constexpr int DK = STEPS + 1, DV = STEPS == 2 ? 2 : DD == 256 || ES == 1 ? 1 : 2;
    static constexpr int RK = STEPS == 2 ? 4 : 2, RV = STEPS == 2 ? 4 : DV + 1;
    static constexpr int RW = kKeys / W;                                // rows of a tile that a wave brings
    static constexpr int RR = RAW ? 5 : 0, RAW_TILE = kKeys * (2 * DD + 8);   // keys, values, their scales
    static constexpr int RAW_AT = (RK + RV) * BUFFER, BYTES = RAW_AT + RR * RAW_TILE;
    static constexpr int AHEAD = RAW ? RR : DK;                         // tiles that are known ahead
    // 16-byte chunk c of row r is stored at chunk c ^ kx(r) (keys), c ^ vx(r) (values): the lanes that the
    // LDS serves together then hit all banks
    static __device__ __forceinline__ int kx(int r) { return DD == 64 ? (r >> 1) & 7 : r & 15; }
    static __device__ __forceinline__ int vx(int r) { return DD == 64 ? (r >> 1 & 1) << 2 : (r & 3) << 2; }
};

// A part: sums of 4 dims of a row, [dims / 4][rows], then the rows' maxima (log2) and sums of weights (-1: sees nothing).
constexpr int64_t part_floats(int rows, int DD) { return rows * (DD + 2); }

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

__device__ __forceinline__ Runs runs_of(const Args &a, uint32_t all)
{
    Runs r;
    r.all = all;
    r.runs = min((uint32_t)a.runs, max(r.all / (uint32_t)a.least, 1u));
    return r;
}

// weight(lane), the first 64 sequences'; where a batch has no more, its scans load nothing further
template <class F>
__device__ __forceinline__ uint32_t first_weights(int count, F weight)
{
    const int lane = threadIdx.x & 63;
    return lane < count ? weight(lane) : 0;
}

// A part of a unit, or all of it: the key tiles first .. first + tiles - 1 of the sequence's list (runs), or the rows' own
// list, for rows r0 .. of sequence b and kv head hk.  lds: the tiles' address in LDS.  True: some sum is NaN, and if not CAREFUL that may be for what masks
// hide.
template <int DT, int CODES, int DD, bool PART, int W, bool CAREFUL>
__device__ __forceinline__ bool block_unit(const Args &a, uint32_t lds, int b, uint32_t hk, int r0, int first, int tiles, bool whole)
{
    constexpr int ES = CODES == PSQ_CODES_NONE ? 2 : 1;
    using L = Layout<DD, W, ES>;
    constexpr int PVT = CODES == PSQ_CODES_NONE ? DT : PSQ_BF16;   // of the second product
    constexpr bool PAIR = CODES != PSQ_CODES_NONE && DT == PSQ_F16;
    constexpr int NC = DD / 16, ND = DD / 32;
    constexpr int CH = DD / 8;                        // 16-byte chunks of a row of 16-bit elements

    // (the careful form works everything out for itself: what both share would stay in registers all along)
    const int tid = CAREFUL ? again(threadIdx.x) : threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 31, h = lane >> 5;
    const int D = PART ? a.D : DD, per_page = a.page / kGroup;

    const Seq s = sequence(a, b);
    const int rows = min(s.n * a.G - r0, a.rows);
    const Keys keys = a.runs ? keys_of(a, s, 0, s.n * a.G - 1) : keys_of(a, s, r0, r0 + rows - 1);
    const Keys own = keys_of(a, s, r0, r0 + rows - 1);
    const int last = min(first + (a.runs ? tiles : keys.count()), keys.count());
    // the next tile of the list from i on that these rows need
    auto next_of = [&](int i) PSQ_INLINE {
        const int t = keys.tile(i);
        const int to = t >= own.hi ? last : t >= own.lo || t * kKeys < a.sinks ? i : i + own.lo - t;
        return min(to, last);
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
    // of the wave: keys up to full_hi, from full_lo or among the sinks, are seen by all rows
    const int w0 = a.N ? s.text : s.len - s.n + wrow / a.G, w1 = a.N ? s.len - 1 : s.len - s.n + (wrow + max(mine, 1) - 1) / a.G;
    const int full_hi = a.N ? s.text - 1 : w0, full_lo = a.window ? w1 - a.window + 1 : 0;

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

    // ---- bringing key tiles to LDS
    const int row_bytes = D * ES;
    uint32_t grp;          // lane 4 i + g: pool group of tile base + i's group g
    uint64_t there, wild;  // tokens that are there; whose page is not
    int base = 0;
    auto look = [&](int i) PSQ_INLINE {
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
    // A tile on its way: its number (-1: none), which of its groups have no page; the wave's rows of it: their group and how
    // many hold tokens.
    struct Tile { int number, astray, group, left; };
    const int first_row = wave * L::RW;               // in a tile
    int at_tile;           // the newest tile's place in the list
    auto tile_at = [&](int i) PSQ_INLINE {
        at_tile = i;
        if (i - base >= kLook) look(i);
        const int bit = 4 * (i - base) + first_row / kGroup, number = keys.tile(i);
        const int left = min(max(s.len - (number * kKeys + first_row), 0), L::RW);
        return Tile{i < last ? number : -1, (int)(wild >> (4 * (i - base))) & 15, __builtin_amdgcn_readlane((int)grp, bit),
                    there >> bit & 1 ? left : 0};   // (past the last tile nothing is there)
    };
    auto row_of = [&](const Tile &t) PSQ_INLINE { return (int64_t)(uint32_t)t.group * kGroup + first_row % kGroup; };
    // 16-bit elements go to LDS by themselves: descriptors of rows, past whose tokens loads give zeros, ...
    constexpr int NL = ES == 2 ? L::RW * L::PITCH / 1024 : 0;
    auto descriptor = [&](const uint8_t *pool, const Tile &t) PSQ_INLINE {
        const uint64_t from = (uint64_t)(pool + row_of(t) * row_bytes);
        return v4i{__builtin_amdgcn_readfirstlane((int)from), __builtin_amdgcn_readfirstlane((int)(from >> 32) & 0xffff),
                   __builtin_amdgcn_readfirstlane(t.left * row_bytes), 0x00020000};
    };
    // ... and load j: row lane / CH + 64 j / CH of the wave's, the chunk whose place is lane % CH (dims that are not there:
    // past every end).  Its offset for j = 0, without the row's, in bytes; x: the placement's exclusive or.
    const uint32_t row_off = (uint32_t)(lane / CH * row_bytes);
    const uint32_t key_off = (uint32_t)(lane % CH ^ L::kx(lane / CH) ^ L::kx(first_row)) * 16, value_off = (uint32_t)(lane % CH ^ L::vx(lane / CH) ^ L::vx(first_row)) * 16;
    auto bring = [&](const v4i &rs, uint32_t buffer, int j, uint32_t off, int x) PSQ_INLINE {
        const uint32_t at = off ^ (x * 16), from = at + row_off + j * (64 / CH) * row_bytes;
        dma16(rs, lds + buffer + first_row * L::PITCH + 1024 * j, PART && (int)at >= 2 * D ? kPast : from);
    };
    auto bring_keys = [&](const v4i &rs, uint32_t buffer, int j) PSQ_INLINE { bring(rs, buffer, j, key_off, L::kx(j * (64 / CH))); };
    auto bring_values = [&](const v4i &rs, uint32_t buffer, int j) PSQ_INLINE { bring(rs, buffer, j, value_off, L::vx(j * (64 / CH))); };
    // Codes go through registers: loaded (zeros where no tokens are), then widened into LDS.
    constexpr int CP = ES == 1 ? (DD / 16 * L::RW + 63) / 64 : 1;     // 16-byte pieces of a lane
    struct Codes { v4i piece[CP]; float scale; };
    auto fetch = [&](Codes &c, const uint8_t *pool, const float *scales, const Tile &t) PSQ_INLINE {
        const uint8_t *src = pool + row_of(t) * row_bytes;
#pragma unroll
        for (int j = 0; j < CP; j++) {
            const int at = 64 * j + lane, r = at / (DD / 16), p = at % (DD / 16);
            c.piece[j] = v4i{0, 0, 0, 0};
            if (r < t.left && (!PART || p * 16 < D)) c.piece[j] = *(const v4i *)(src + r * row_bytes + p * 16);
        }
        c.scale = 0.0f;
        if (lane < t.left) c.scale = scales[row_of(t) + lane];
    };
    auto deliver = [&](auto typec, const Codes &codes, uint32_t buffer, auto place) PSQ_INLINE {
        const uint32_t to = lds + buffer + first_row * L::PITCH;
#pragma unroll
        for (int j = 0; j < CP; j++) {
            const int at = 64 * j + lane, r = at / (DD / 16), c = 2 * (at % (DD / 16)), x = place(r) ^ place(first_row);
            v4i w[2];
            widen<decltype(typec)::value, CODES>(codes.piece[j], w);
            if (64 * CP * 16 == L::RW * DD || r < L::RW) {
                *at_lds<v4i>(to + r * L::PITCH + (c ^ x) * 16) = w[0];
                *at_lds<v4i>(to + r * L::PITCH + ((c + 1) ^ x) * 16) = w[1];
            }
        }
        if (lane < L::RW) *at_lds<float>(lds + buffer + L::TILE + 4 * (first_row + lane)) = codes.scale;
    };
    auto deliver_keys = [&](const Codes &c, uint32_t buffer) PSQ_INLINE { deliver(std::integral_constant<int, DT>{}, c, buffer, [](int r) { return L::kx(r); }); };
    auto deliver_values = [&](const Codes &c, uint32_t buffer) PSQ_INLINE { deliver(std::integral_constant<int, PVT>{}, c, buffer, [](int r) { return L::vx(r); }); };
    // or as they are: the wave's rows of a tile's keys and values, and their scales, to a raw buffer ...
    constexpr int PIECES = L::RW * DD / 16;           // lanes that have 16 bytes of them
    auto load_raw = [&](const Tile &t, uint32_t raw) PSQ_INLINE {
        const int64_t row = row_of(t);
        auto rows = [&](const void *pool, int bytes) PSQ_INLINE {
            const uint64_t from = (uint64_t)pool + row * bytes;
            return v4i{__builtin_amdgcn_readfirstlane((int)from), __builtin_amdgcn_readfirstlane((int)(from >> 32) & 0xffff),
                       __builtin_amdgcn_readfirstlane(t.left * bytes), 0x00020000};
        };
        const int p = lane % (DD / 16);
        const uint32_t off = PART && p * 16 >= D ? kPast : (uint32_t)(lane / (DD / 16) * row_bytes + p * 16);
        const uint32_t at = lds + raw + first_row * DD, sc = lds + raw + kKeys * 2 * DD + first_row * 4;
        const v4i rk = rows(a.kc, row_bytes), rv = rows(a.vc, row_bytes), sk = rows(a.ks, 4), sv = rows(a.vs, 4);
        if (PIECES >= 64 || lane < PIECES) {
            dma16(rk, at, off);
            dma16(rv, at + kKeys * DD, off);
        }
        if (lane < L::RW) {
            dma4(sk, sc, (uint32_t)lane * 4);
            dma4(sv, sc + kKeys * 4, (uint32_t)lane * 4);
        }
    };
    // ... and, once they are there, widened into the tile's place
    auto raw_piece = [&](uint32_t raw, int values) PSQ_INLINE {
        Codes c;
        c.piece[0] = *at_lds<const v4i>(lds + raw + values * kKeys * DD + first_row * DD + lane % PIECES * 16);
        c.scale = *at_lds<const float>(lds + raw + kKeys * 2 * DD + values * kKeys * 4 + 4 * (first_row + lane % L::RW));
        return c;
    };
    // a tile at once
    auto take_keys = [&](const Tile &t, uint32_t buffer) PSQ_INLINE {
        if constexpr (ES == 2) {
            const v4i rs = descriptor(a.kc, t);
#pragma unroll
            for (int j = 0; j < NL; j++) bring_keys(rs, buffer, j);
        } else {
            Codes c;
            fetch(c, a.kc, a.ks, t);
            deliver_keys(c, buffer);
        }
    };
    auto take_values = [&](const Tile &t, uint32_t buffer) PSQ_INLINE {
        if constexpr (ES == 2) {
            const v4i rs = descriptor(a.vc, t);
#pragma unroll
            for (int j = 0; j < NL; j++) bring_values(rs, buffer, j);
        } else {
            Codes c;
            fetch(c, a.vc, a.vs, t);
            deliver_values(c, buffer);
        }
    };

    // ---- a key tile of the wave's rows
    v16f o[ND];
    float run_m, run_l;    // the maximum that scores are taken off (in their own units); the lane's part of the sum
    uint32_t seen;         // (carefully) scores that count
    bool raise;            // of the tile's maximum over run_m
    float top;             // of the tile: the lane's, then the row's
    // LDS addresses of the lane's reads in the first buffers.  Chunks are picked by exclusive or of a row's low bits, which
    // the buffers' offsets leave alone.
    const uint32_t klane = lds + n * L::PITCH + ((h ^ L::kx(n)) << 4);
    const uint32_t vlane = lds + (4 * h + (n & 15) / 4) * L::PITCH + ((((n >> 4) << 1 | (n & 3) >> 1) ^ L::vx((n & 15) / 4)) << 4) + (n & 1) * 8;
    auto key = [&](uint32_t at, int t, int c) PSQ_INLINE { return *at_lds<const v4i>((at ^ (c << 5)) + 32 * t * L::PITCH); };
    auto value = [&](uint32_t at, int u, int d) PSQ_INLINE {
        const uint32_t src = (at ^ (d << 6)) + 16 * u * L::PITCH;
        const v2i x = __builtin_bit_cast(v2i, __builtin_amdgcn_ds_read_tr16_b64_v4i16(at_lds<v4s>(src)));
        const v2i y = __builtin_bit_cast(v2i, __builtin_amdgcn_ds_read_tr16_b64_v4i16(at_lds<v4s>(src + 8 * L::PITCH)));
        return v4i{x[0], x[1], y[0], y[1]};
    };
    // scores of a tile from its products: scales, masks, their maximum (turn has done the first, and the last where there are
    // no masks)
    auto scale_keys = [&](v16f (&sc)[2], int q, const v4f &x) PSQ_INLINE {
#pragma unroll
        for (int j = 0; j < 4; j++) sc[q / 4][4 * (q & 3) + j] *= x[j];
    };
    auto scale_of = [&](uint32_t buffer, int q) PSQ_INLINE { return *at_lds<const v4f>(lds + buffer + L::TILE + 4 * (32 * (q / 4) + 8 * (q & 3) + 4 * h)); };
    auto lane_top = [&](const v16f (&sc)[2]) PSQ_INLINE {
        top = __builtin_elementwise_maximum(sc[0][0], sc[1][0]);
#pragma unroll
        for (int i = 1; i < 16; i++) top = __builtin_elementwise_maximum(top, __builtin_elementwise_maximum(sc[0][i], sc[1][i]));
    };
    auto row_top = [&]() PSQ_INLINE {
        // (NaN wins; it raises nothing, and the row's sum will be NaN)
        top = half_max(top);
        // (a maximum that comes first, or is raised from -inf, is any growth)
        raise = top * a.scale > run_m * a.scale + kGrowth;
    };
    auto scores = [&](v16f (&sc)[2], int tile0, bool edge, uint32_t astray) PSQ_INLINE {
        if (CAREFUL) seen = 0;
        if (CAREFUL || edge) {
            int t0 = tile0;
            asm volatile("" : "+v"(t0));   // (a branch, not selects that all tiles pay for)
            if (astray)                    // pages that are not there: NaN
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int i = 0; i < 16; i++)
                        if (astray >> (2 * t + (i >> 3)) & 1) sc[t][i] = NAN;
            // Bits c of a word: key 32 t + c of the lane's half, c = 8 (i >> 2) + (i & 3).  below(x): those with c < x.
            auto below = [](int x) { return x <= 0 ? 0u : x >= 32 ? ~0u : (1u << x) - 1; };
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const int at = t0 + 32 * t + 4 * h, text = s.text - at;
                uint32_t see = below(min(pos + 1, s.text) - at) & (~below(low - at) | below(a.sinks - at));
                if (a.N) see |= text >= 0 ? (text < 32 ? (uint32_t)way << text : 0) : text > -64 ? (uint32_t)(way >> -text) : 0;
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const int on = (int)(see << (31 - (8 * (i >> 2) + (i & 3)))) >> 31;
                    sc[t][i] = __int_as_float((__float_as_int(sc[t][i]) & on) | (~on & (int)0xff800000));
                }
                if (CAREFUL) seen |= ((see & 15) | (see >> 4 & 0xf0) | (see >> 8 & 0xf00) | (see >> 12 & 0xf000)) << (16 * t);
            }
            lane_top(sc);
            row_top();
        }
    };
    auto grow = [&]() PSQ_INLINE {
        if (!__any(raise)) return;
        const float to = raise ? top : run_m;    // (each row by itself: its result does not depend on the others')
        float keep = to == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((run_m - to) * a.scale);
        if (CAREFUL) keep = fmaxf(keep, 0x1p-126f);   // (an infinite sum stays one)
        run_m = to;
        run_l *= keep;
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
            for (int i = 0; i < 16; i++) o[d][i] *= keep;
    };
    // Scores in sc, the tile's values in vb, the next tile's keys in kb: its products into sc, the tile's weights and
    // values into o.
    auto turn = [&](const v16f (&sc)[2], v16f (&next)[2], uint32_t kb, uint32_t vb, auto aside) PSQ_INLINE {
        const uint32_t kat = again(klane + kb), vat = again(vlane + vb);
        const float ref = (PVT == PSQ_F16 ? kF16Unit : 0) - (run_m == -INFINITY ? 0.0f : run_m * a.scale);
        v4i ph[4], pl[PAIR ? 4 : 1];
        v4f vs, ks;        // scales at hand
        // two scores to weights: pair q of the tile's 16
        auto weigh = [&](auto qc) PSQ_INLINE {
            constexpr int Q = decltype(qc)::value, T = Q / 8, I = 2 * (Q & 7);
            float x = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[T][I], a.scale, ref)), y = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[T][I + 1], a.scale, ref));
            run_l += x;
            run_l += y;
            if constexpr (ES == 1) {
                if constexpr (Q % 2 == 0) {
                    vs = scale_of(vb, Q / 2);
                }
                x *= vs[I & 2], y *= vs[(I & 2) + 1];
                if (CAREFUL && !(seen >> (16 * T + I) & 1)) x = 0.0f;        // (its scale may be infinite)
                if (CAREFUL && !(seen >> (16 * T + I + 1) & 1)) y = 0.0f;
            }
            const uint32_t p = pack_half2<PVT>(x, y);
            ph[Q / 4][Q & 3] = (int)p;
            if constexpr (PAIR) {
                const float hx = half_to_f32<PVT>(p), hy = half_to_f32<PVT>(p >> 16);
                x -= hx, y -= hy;
                if (CAREFUL && fabsf(hx) == INFINITY) x = 0.0f;              // (nothing is left of an infinite one)
                if (CAREFUL && fabsf(hy) == INFINITY) y = 0.0f;
                pl[Q / 4][Q & 3] = (int)pack_half2<PVT>(x, y);
            }
        };
        // A slot is a matrix instruction, the LDS read of the one AHEAD slots later, and what vector work it covers:
        // vector and matrix units work at the same time only where the instructions of both take turns (two
        // waves of a SIMD fall into step).  First the next tile's scores, then the values with the weights, of which
        // those of a step of 16 keys are ready when it begins; beside these the maximum of the next tile's.
        constexpr int AHEAD = ES == 1 ? 2 : 4, QK = 2 * NC, ALL = QK + 4 * ND, COVER = QK + 3 * ND;
        if constexpr (CAREFUL) {
            static_for<16>([&](auto q) PSQ_INLINE {
                weigh(q);
                __builtin_amdgcn_sched_barrier(0);   // (here and below: it is not to need more registers than the other)
            });
#pragma unroll
            for (int u = 0; u < 4; u++)
#pragma unroll
                for (int d = 0; d < ND; d++) {
                    constexpr uint32_t EXP = PVT == PSQ_BF16 ? 0x7f80 : 0x7c00, ONE = PVT == PSQ_BF16 ? 0x3f80 : 0x3c00;
                    v4i vf = value(vat, u, d), up, down, is;     // ones where a value is +inf, is -inf (NaN: both); where a key is seen
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
                        vf[e] = (int)c, up[e] = (int)pu, down[e] = (int)pd, is[e] = (int)ps;
                    }
                    if (__any(any)) {
                        v16f zero = {};
                        const v16f more = mfma<PVT>(up, is, zero), less = mfma<PVT>(down, is, zero);
#pragma unroll
                        for (int i = 0; i < 16; i++) {
                            if (more[i] > 0.0f) o[d][i] += INFINITY;
                            if (less[i] > 0.0f) o[d][i] -= INFINITY;
                        }
                    }
                    o[d] = mfma<PVT>(vf, ph[u], o[d]);
                    if constexpr (PAIR) o[d] = mfma<PVT>(vf, pl[u], o[d]);
                    __builtin_amdgcn_sched_barrier(0);
                }
#pragma unroll
            for (int t = 0; t < 2; t++) {
                next[t] = v16f{};
#pragma unroll
                for (int c = 0; c < NC; c++) {
                    next[t] = mfma<DT>(key(kat, t, c), qf[c], next[t]);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            if constexpr (ES == 1)
#pragma unroll
                for (int q = 0; q < 8; q++) scale_keys(next, q, scale_of(kb, q));
            lane_top(next);
            row_top();
            static_for<ALL>([&](auto i) PSQ_INLINE { aside(i); });
        } else {
            v4i f[AHEAD];
            auto read = [&](auto ic) PSQ_INLINE {
                constexpr int I = decltype(ic)::value;
                if constexpr (I < QK) f[I % AHEAD] = key(kat, I / NC, I % NC);
                else if constexpr (I < ALL) f[I % AHEAD] = value(vat, (I - QK) / ND, (I - QK) % ND);
            };
            static_for<AHEAD>([&](auto i) PSQ_INLINE { read(i); });
            static_for<ALL>([&](auto ic) PSQ_INLINE {
                constexpr int I = decltype(ic)::value;
                __builtin_amdgcn_sched_barrier(0);
                if constexpr (I < QK) {
                    if constexpr (I % NC == 0) next[I / NC] = mfma<DT>(f[I % AHEAD], qf[0], v16f{});
                    else next[I / NC] = mfma<DT>(f[I % AHEAD], qf[I % NC], next[I / NC]);
                } else {
                    constexpr int U = (I - QK) / ND, V = (I - QK) % ND;
                    o[V] = mfma<PVT>(f[I % AHEAD], ph[U], o[V]);
                    if constexpr (PAIR) o[V] = mfma<PVT>(f[I % AHEAD], pl[U], o[V]);
                }
                read(std::integral_constant<int, I + AHEAD>{});
                aside(ic);
                // some of the next scores, four at a time: scaled, and their maximum, the row's in the end
                if constexpr (I >= QK) {
                    constexpr int TOP = 4 * ND - 3, P = (I - QK) * 32 / TOP / 4 * 4, E = (I - QK + 1) * 32 / TOP / 4 * 4;
                    static_for<32>([&](auto kc) PSQ_INLINE {
                        constexpr int K = decltype(kc)::value;
                        if constexpr (K >= P && K < E && I - QK < TOP) {
                            if constexpr (ES == 1) {
                                if constexpr (K % 4 == 0) ks = scale_of(kb, K / 4);
                                next[K / 16][K % 16] *= ks[K & 3];
                            }
                            if constexpr (K == 1) top = __builtin_elementwise_maximum(next[0][0], next[0][1]);
                            else if constexpr (K % 2) top = __builtin_elementwise_maximum(top, __builtin_elementwise_maximum(next[K / 16][K % 16 - 1], next[K / 16][K % 16]));
                        }
                    });
                    if constexpr (I - QK == TOP) row_top();
                }
                // pairs q of COVER slots' share
                constexpr int A = I * 16 / COVER, B = (I + 1) * 16 / COVER;
                static_for<16>([&](auto q) PSQ_INLINE {
                    if constexpr (I < COVER && decltype(q)::value >= A && decltype(q)::value < B) weigh(q);
                });
            });
            asm volatile("" : "+v"(run_l));    // (its sums belong to the slots)
            __builtin_amdgcn_sched_barrier(0);
        }
    };

    // All of the workgroup's key tiles of the unit.
    auto pass = [&]() PSQ_INLINE {
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
            for (int i = 0; i < 16; i++) o[d][i] = 0.0f;
        run_m = -INFINITY, run_l = 0.0f;
        __syncthreads();                       // LDS is free
        int i = next_of(first);
        if (i >= last) return;
        // whether a tile's masks hide some of it from some row of the wave
        auto edge = [&](const Tile &t) {
            const int tile0 = t.number * kKeys, tile1 = tile0 + kKeys - 1;
            return !(tile1 <= full_hi && (tile0 >= full_lo || tile1 < a.sinks) && !t.astray);
        };
        constexpr int DK = L::DK, DV = L::DV;
        constexpr uint32_t VALUES = L::RK * L::BUFFER, VALUES_END = L::RAW_AT;
        Tile q[L::AHEAD + 1];                        // the tile at hand and those behind it
        look(i);
#pragma unroll
        for (int d = 0; d < L::AHEAD; d++) {
            q[d] = tile_at(d ? next_of(at_tile + 1) : i);
            if constexpr (L::RAW) {
                load_raw(q[d], L::RAW_AT + d * L::RAW_TILE);
            } else {
                take_keys(q[d], d * L::BUFFER);
                if (d < DV) take_values(q[d], VALUES + d * L::BUFFER);
            }
        }
        wait_vmcnt<0>();
        asm volatile("" ::: "memory");
        if constexpr (L::RAW) {
            deliver_keys(raw_piece(L::RAW_AT, 0), 0);
            deliver_keys(raw_piece(L::RAW_AT + L::RAW_TILE, 0), L::BUFFER);
            deliver_values(raw_piece(L::RAW_AT, 1), VALUES);
        }
        stage_barrier();
        uint32_t raw = L::RAW_AT;              // the raw buffer of the tile at hand, whose codes are done with
        // buffers: of the keys read (the next tile's) and loaded, the values read and loaded
        uint32_t kr = L::BUFFER, kl = DK % L::RK * L::BUFFER, vr = VALUES, vl = VALUES + DV * L::BUFFER;
        auto advance = [](uint32_t &at, uint32_t from, uint32_t end) PSQ_INLINE {
            at += L::BUFFER;
            if (at == end) at = from;
        };
        // q[0]'s scores are in sc, its values and q[1]'s keys here once the loads up to them are; q[0]'s keys are done with.
        // False: q[0] was the last (the products of what lies in place of the next one's keys are not used).
        auto step = [&](auto workc, auto meetc, v16f (&sc)[2], v16f (&to)[2]) PSQ_INLINE {
            constexpr bool WORK = decltype(workc)::value;
            if constexpr (decltype(meetc)::value) {
                if constexpr (!L::RAW) wait_vmcnt<0>();     // (raw tiles are waited for where they are widened)
                stage_barrier();
            }
            q[L::AHEAD] = tile_at(next_of(at_tile + 1));
            if constexpr (L::RAW) {
                auto behind = [&](int tiles) PSQ_INLINE {
                    const uint32_t at = raw + tiles * L::RAW_TILE;
                    return at >= (uint32_t)L::BYTES ? at - L::RR * L::RAW_TILE : at;
                };
                // the wave's own loads of the tile two behind, and those before, are here when as many are on their way as came after
                Codes ck, cv;
                auto convert = [&](auto ic) PSQ_INLINE {
                    constexpr int I = decltype(ic)::value;
                    if constexpr (I == 1) load_raw(q[L::RR], raw);
                    if constexpr (I == 3) {
                        wait_vmcnt<(L::RR - 2) * 4>();
                        asm volatile("" ::: "memory");
                        cv = raw_piece(behind(1), 1);
                    }
                    if constexpr (I == 6) deliver_values(cv, vl);
                    if constexpr (I == 8) ck = raw_piece(behind(2), 0);
                    if constexpr (I == 11) deliver_keys(ck, kl);
                };
                if constexpr (WORK) {
                    grow();
                    turn(sc, to, kr, vr, convert);
                } else {
                    static_for<12>([&](auto ic) PSQ_INLINE { convert(ic); });
                }
                raw = behind(1);
            } else if constexpr (ES == 2) {
                const v4i rv = descriptor(a.vc, q[DV]), rk = descriptor(a.kc, q[DK]);
                auto load = [&](auto ic) PSQ_INLINE {      // one in two slots
                    constexpr int I = decltype(ic)::value;
                    if constexpr (I % 2 == 1 && I / 2 < NL) bring_values(rv, vl, I / 2);
                    else if constexpr (I % 2 == 1 && I / 2 < 2 * NL) bring_keys(rk, kl, I / 2 - NL);
                };
                if constexpr (WORK) {
                    grow();
                    turn(sc, to, kr, vr, load);
                } else {
                    static_for<4 * NL>([&](auto ic) PSQ_INLINE { load(ic); });
                }
            } else {
                Codes ck, cv;
                fetch(cv, a.vc, a.vs, q[DV]);
                fetch(ck, a.kc, a.ks, q[DK]);
                if constexpr (WORK) {
                    grow();
                    turn(sc, to, kr, vr, [](auto) {});
                }
                deliver_values(cv, vl);
                deliver_keys(ck, kl);
            }
            if (q[1].number < 0) return false;
            if constexpr (WORK) scores(to, q[1].number * kKeys, edge(q[1]), (uint32_t)q[1].astray);
#pragma unroll
            for (int d = 0; d < L::AHEAD; d++) q[d] = q[d + 1];
            advance(kr, 0, VALUES), advance(kl, 0, VALUES), advance(vr, VALUES, VALUES_END), advance(vl, VALUES, VALUES_END);
            return true;
        };
        v16f sa[2] = {}, sb[2] = {};
        using Meet = std::true_type;
        using Other = std::bool_constant<L::STEPS == 1>;
        if (mine == 0) {                       // (waves without rows bring their groups)
            while (step(std::false_type{}, Meet{}, sa, sb) && step(std::false_type{}, Other{}, sa, sb)) {}
            return;
        }
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int c = 0; c < NC; c++) sa[t] = mfma<DT>(key(klane, t, c), qf[c], sa[t]);
        if constexpr (ES == 1)
#pragma unroll
            for (int q = 0; q < 8; q++) scale_keys(sa, q, scale_of(0, q));
        lane_top(sa);
        row_top();
        scores(sa, q[0].number * kKeys, edge(q[0]), (uint32_t)q[0].astray);
        using Work = std::true_type;
        while (step(Work{}, Meet{}, sa, sb) && step(Work{}, Other{}, sb, sa)) {}
    };
    pass();
    wait_vmcnt<0>();       // (loads into the LDS end before it may be another's)
    float any = 0.0f;
#pragma unroll
    for (int d = 0; d < ND; d++)
        if (!PART || 32 * d < D)
#pragma unroll
            for (int i = 0; i < 16; i++) any = __builtin_fmaf(o[d][i], 0.0f, any);

    // ---- the rows' outputs, or the part of them
    run_l = half_sum(run_l);
    const float level = run_m * a.scale - (PVT == PSQ_F16 ? kF16Unit : 0);     // (in log2, the weights' unit taken off)
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
        if (a.lse && h == 0) a.lse[at] = pos < 0 ? -INFINITY : level * kLn2 + logf(run_l);
    } else if (valid) {
        float *part = a.part + (2 * (int64_t)xcd_rank(blockIdx.x, a.runs) + (first == 0)) * part_floats(a.rows, DD);
        const int r = 32 * wave + n;
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
            for (int i = 0; i < 16; i += 4)
                ((v4f *)part)[(8 * d + i / 2 + h) * a.rows + r] = v4f{o[d][i], o[d][i + 1], o[d][i + 2], o[d][i + 3]};
        if (h == 0) part[a.rows * DD + r] = level, part[a.rows * (DD + 1) + r] = pos < 0 ? -1.0f : run_l;
    }
    return any != any;
}

template <int DT, int CODES, int DD, bool PART, int W>
__global__ void __launch_bounds__(64 * W, DD > 128 ? 1 : 2)
block_attention_kernel(Args a)
{
    extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
    const uint32_t lds = (uint32_t)(uintptr_t)(lds_ptr)smem;

    // ---- the workgroup's units
    const int count = a.N ? a.B : a.B + 1;
    int b, r0, first = 0, tiles = 0;       // key tiles first .. of the unit's list are the workgroup's
    uint32_t hk, x = 0, end = 0, kept = 0;
    auto weight = [&](int b) { return weight_of(a, b); };
    if (!a.runs) {
        auto tiles_of = [&](int b) { return (uint32_t)row_tiles(a, sequence(a, b)); };
        const uint32_t kept = first_weights(count, tiles_of);
        auto kept_of = [&](int b) { return b < 64 ? kept : tiles_of(b); };
        const uint32_t all = sum_of(count, kept_of), units = all * a.Hkv;
        if (blockIdx.x >= units) return;
        // Workgroups of an XCD share a kv head's keys and values in its L2; the rows that see most go first.
        const uint32_t rank = (uint32_t)xcd_rank(blockIdx.x, units);
        hk = rank / all;
        uint32_t before;
        const uint32_t place = all - 1 - (rank - hk * all);
        b = __builtin_amdgcn_readfirstlane(find(count, place, before, kept_of));
        if (b >= count) return;            // (only of starts that a caller may not give, as below)
        r0 = (int)(place - before) * a.rows;
    } else {
        kept = first_weights(count, weight);
        const Runs runs = runs_of(a, sum_of(count, [&](int b) { return b < 64 ? kept : weight(b); }));
        const uint32_t w = (uint32_t)xcd_rank(blockIdx.x, a.runs);
        if (w >= runs.runs) return;
        x = runs.first(w), end = runs.first(w + 1);
    }

    do {
    bool whole = true;
    if (a.runs) {
        uint32_t before;
        b = __builtin_amdgcn_readfirstlane(find(count, x, before, [&](int b) { return b < 64 ? kept : weight(b); }));
        if (b >= count) return;            // (this and the next too)
        const Seq s = sequence(a, b);
        const uint32_t each = (uint32_t)key_tiles(a, s), per = (uint32_t)row_tiles(a, s), unit = (x - before) / each;
        hk = unit / per;
        if (hk >= (uint32_t)a.Hkv) return;
        r0 = (int)(unit - hk * per) * a.rows;
        first = (int)(x - before - unit * each);
        tiles = (int)min(each - first, end - x);
        whole = tiles == (int)each;
        x += tiles;
    }
    const bool odd = block_unit<DT, CODES, DD, PART, W, false>(a, lds, b, hk, r0, first, tiles, whole);
    // (whether any wave's is; the LDS has no room beside the tiles)
    const bool some = __any(odd);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) *at_lds<int>(lds + 4 * (threadIdx.x / 64)) = some;
    __syncthreads();
    int odds = 0;
#pragma unroll
    for (int w = 0; w < W; w++) odds |= *at_lds<int>(lds + 4 * w);
    if (__builtin_amdgcn_readfirstlane(odds)) {
        auto *args = (const __attribute__((address_space(4))) uint32_t *)__builtin_amdgcn_kernarg_segment_ptr();
        asm volatile("" : "+s"(args));
        uint32_t words[sizeof(Args) / 4];
#pragma unroll
        for (int i = 0; i < (int)(sizeof(Args) / 4); i++) words[i] = args[i];
        block_unit<DT, CODES, DD, PART, W, true>(__builtin_bit_cast(Args, words), lds, b, hk, r0, first, tiles, whole);
    }
    if (x < end) kept = first_weights(count, weight);   // (not kept in a register through the unit)
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
    uint32_t before;
    int b;
    if (a.N) {                             // (as many units each, and a grid with no more)
        const uint32_t units = (uint32_t)((a.N * a.G + a.rows - 1) / a.rows) * a.Hkv;
        b = blockIdx.x / units, before = b * units;
    } else {
        if (blockIdx.x >= sum_of(count, units_of)) return;
        b = __builtin_amdgcn_readfirstlane(find(count, blockIdx.x, before, units_of));
    }
    const Seq s = sequence(a, b);
    const uint32_t unit = blockIdx.x - before, each = (uint32_t)key_tiles(a, s), per = (uint32_t)row_tiles(a, s), hk = unit / per;
    const int r0 = (int)(unit - hk * per) * a.rows, r = (int)blockIdx.y * kJoin + (threadIdx.x & (kJoin - 1)), quad = threadIdx.x / kJoin;
    uint32_t front = 0;                    // key tiles of the sequences in front
    const Runs runs = runs_of(a, sum_of(count, [&](int i) {
        const uint32_t w = weight_of(a, i);
        front += i < b ? w : 0;
        return w;
    }));
#pragma unroll
    for (int o = 32; o; o >>= 1) front += __shfl_xor(front, o, 64);
    const uint32_t x = (uint32_t)__builtin_amdgcn_readfirstlane((int)front) + unit * each;
    const uint32_t w0 = runs.owner(x), parts = runs.owner(x + each - 1) - w0 + 1;
    if (parts == 1 || w0 + parts > (uint32_t)a.runs || r0 + r >= s.n * a.G || 4 * quad >= a.D) return;
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
                const float *part = a.part + (2 * (int64_t)(w0 + p) + (p == 0)) * part_floats(a.rows, DD);
                y[u] = ((const v4f *)part)[quad * a.rows + r];
                m[u] = part[a.rows * DD + r], l[u] = part[a.rows * (DD + 1) + r];
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

template <int DT, int CODES, int DD, bool PART, int W>
int launch(const Args &a, unsigned groups, hipStream_t st)
{
    auto *kernel = block_attention_kernel<DT, CODES, DD, PART, W>;
    constexpr int lds = Layout<DD, W, CODES == PSQ_CODES_NONE ? 2 : 1>::BYTES;
    static_assert(lds <= 160 * 1024 / (W == 4 && DD <= 128 ? 2 : 1), "tiles fit the LDS");
    static bool raised[64] = {};
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return set_error(PSQ_E_DEVICE, "no current HIP device");
    if (!raised[dev]) {
        if (hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess)
            return set_error(PSQ_E_DEVICE, "block attention: cannot raise the LDS size");
        raised[dev] = true;
    }
    kernel<<<a.runs ? a.runs : groups, 64 * W, lds, st>>>(a);
    const int rows = a.N ? min(a.N * a.G, a.rows) : a.rows, join = 1024 / DD;
    if (a.runs) join_kernel<DT, DD><<<dim3(groups, (rows + join - 1) / join), kThreads, 0, st>>>(a);
    return check_launch("block attention");
}

template <int DT, int CODES>
int launch_dim(const Args &a, unsigned groups, hipStream_t st)
{
    constexpr int W = CODES == PSQ_CODES_NONE ? 4 : 8;   // (as a.rows)
    if (a.D == 64) return launch<DT, CODES, 64, false, W>(a, groups, st);
    if (a.D == 128) return launch<DT, CODES, 128, false, W>(a, groups, st);
    if (a.D == 256) return launch<DT, CODES, 256, false, 4>(a, groups, st);
    if (a.D < 64) return launch<DT, CODES, 64, true, W>(a, groups, st);
    if (a.D < 128) return launch<DT, CODES, 128, true, W>(a, groups, st);
    return launch<DT, CODES, 256, true, 4>(a, groups, st);
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
