// block_attention.hip -- the entry points of the attention of prompts and of trees of drafts over the paged
// cache (the kernel is in block_attention.hpp): checks of arguments, and the launch.
#include "block_attention.hpp"
#include "block_plan.hpp"

namespace psq {
namespace block {
namespace {

// Fills in and checks everything but the rows' own arguments; a.T, a.N and a.B are set.
int check(const char *name, Args &a, int codes, const void *q, int dtype, int64_t q_token, int64_t q_head, const void *k_cache,
          const void *v_cache, const float *k_scale, const float *v_scale, int64_t num_pages, int page_size, const int32_t *block_table,
          int64_t table_stride, int64_t table_cols, const int32_t *lengths, int64_t B, int64_t T, int Hq, int Hkv, int D, float scale,
          int64_t window, int64_t sinks, int64_t max_len, void *out, float *lse, const void *workspace, int64_t workspace_bytes)
{
    if (B < 0 || T < 0 || Hq < 0 || table_cols < 0 || window < 0 || sinks < 0 || max_len < 0 || workspace_bytes < 0)
        return set_error(PSQ_E_ARG, "%s: negative size", name);
    if (dtype != PSQ_BF16 && dtype != PSQ_F16) return set_error(PSQ_E_ARG, "%s: queries must be bf16 or f16 (dtype %d)", name, dtype);
    if (sinks && !window) return set_error(PSQ_E_ARG, "%s: sinks are of a window", name);
    if (int e = check_kv_cache(name, codes, k_cache, v_cache, k_scale, v_scale, num_pages, page_size, Hkv, D)) return e;
    if (T == 0 || Hq == 0) return PSQ_OK;
    if (!q || !out || (B && !lengths) || (B && table_cols && !block_table)) return set_error(PSQ_E_ARG, "%s: null pointer", name);
    if (Hq % Hkv || Hq > 65535) return set_error(PSQ_E_SHAPE, "%s: %d heads do not share %d kv heads", name, Hq, Hkv);
    if (((uintptr_t)q | (uintptr_t)out) & 15 || (q_token | q_head) & 7)
        return set_error(PSQ_E_SHAPE, "%s: queries and output must be 16-byte aligned, query strides multiples of 8", name);
    if (((uintptr_t)block_table | (uintptr_t)lengths | (uintptr_t)lse) & 3)
        return set_error(PSQ_E_SHAPE, "%s: misaligned table, lengths or lse", name);
    if (B > 65535 || table_cols > 0x3fffffffLL / page_size)
        return set_error(PSQ_E_SHAPE, "%s: %lld sequences of %lld pages are too many", name, (long long)B, (long long)table_cols);
    // (a rows' number, and that of a workgroup, in 31 bits)
    if (T > 0x3fffffffLL / Hq) return set_error(PSQ_E_SHAPE, "%s: %lld tokens of %d heads are too many", name, (long long)T, Hq);
    // (a length past the table counts as the table's and the rows', and a tile or two: in 31 bits)
    if (table_cols * page_size + T > 0x7fffff00LL)
        return set_error(PSQ_E_SHAPE, "%s: %lld tokens on a table of %lld are too many", name, (long long)T, (long long)(table_cols * page_size));
    if ((uintptr_t)workspace & 255) return set_error(PSQ_E_SHAPE, "%s: the workspace must be 256-byte aligned", name);
    a.q = (const uint16_t *)q, a.q_token = q_token, a.q_head = q_head;
    a.kc = (const uint8_t *)k_cache, a.vc = (const uint8_t *)v_cache, a.ks = k_scale, a.vs = v_scale;
    a.table = block_table, a.table_stride = table_stride, a.lengths = lengths;
    a.out = (uint16_t *)out, a.lse = lse;
    a.num_pages = (int)num_pages, a.cols = (int)table_cols, a.B = (int)B, a.T = (int)T, a.page = page_size;
    a.Hq = Hq, a.Hkv = Hkv, a.D = D, a.G = Hq / Hkv;
    const int64_t far = 0x3fffffff;    // past any length
    a.window = (int)std::min(window, far), a.sinks = (int)std::min(sinks, far);
    a.flip = scale < 0 ? 0x8000 : 0, a.mute = scale == 0;
    a.scale = a.mute ? 1.0f : fabsf(scale) * kLog2e;
    return 1;
}

// Rows of a workgroup's tile; units (sequence, kv head, tile of rows) that there are at most, and the runs that their key
// tiles are cut into (0: they stay whole).
struct Plan { int rows; int64_t units, runs, bytes; };

constexpr int kLeast = 2;    // key tiles of a run (twice as many: a tree of 24 on 8 x 1000, int8, 39 us with either, 8: 46)

Plan plan(int codes, int64_t T, int64_t B, int N, int Hq, int Hkv, int D, int64_t window, int64_t sinks, int64_t max_len)
{
    Plan p{};
    // Sequences that have rows: of fewer rows than sequences some have none.  Rows of one and a kv head, on average and rounded
    // up: with rows there is a unit.
    const int64_t G = Hq / Hkv, some = std::max<int64_t>(N ? B : std::min(B, T), 1), each = (N ? N : (T + some - 1) / some) * G;
    // Codes are widened once per tile of keys, for twice as many rows (512 tokens on 64977, int8: 1257 us with 128, 1133 with
    // 256).  16 bits, 40 heads on 8, bf16, 128 | 256 rows, us: 1024 tokens 41 | 47, 8192 684 | 698; of dims of 64, 16 heads:
    // 1024 23 | 37, 8192 202 | 187 (256 never in front by more than 10%, so these have one form).
    p.rows = D <= 128 && codes != PSQ_CODES_NONE ? 256 : 128;
    p.units = Hkv * (N ? B * ((N * G + p.rows - 1) / p.rows) : T * G / p.rows + B + 1);
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess) dev = 0;
    const int64_t cus = cu_count(dev), slots = cus * (D > 128 || p.rows == 256 ? 1 : 2);
    // Key tiles of a unit, at most, on average and at least, and of a sequence's list, which runs are cut from: a causal
    // unit ends at its own last row, and a run's share counts tiles that its rows do not see.
    const double tokens = (double)each / G, most_len = (double)max_len, rows_tokens = std::max((double)p.rows / G, 1.0);
    const double list = window ? std::min(most_len, (double)window + sinks + tokens) / kKeys + 1 : most_len / kKeys;
    const double most = window ? std::min(most_len, (double)window + sinks + rows_tokens) / kKeys + 1 : list;
    const double cut = window || N ? 0 : std::min(tokens, most_len) / kKeys;
    // Times in tile steps.  kBegin: to begin a unit (its queries, pages and first tiles), and as much again to write parts
    // and join them.  Whole units: their share of a slot, the last round not full; no less than the longest.  Alone on a
    // CU a workgroup takes 0.6 of the time that each of two takes.
    // us, whole | runs (40 heads on 8, dims of 128, bf16): 512 tokens 29 | 57, 2048 82 | 143, 4096 231 | 364, 512 on 8192
    // 223 | 131, trees of 16 on 300 17 | 27, 32 of them on 1000 43 | 53; int8: 2048 on 16384 1214 | 885, 8 x 256 on 4096
    // 360 | 290, 128 on 1024 58 | 41, trees of 64 on 60000 2370 | 183.
    constexpr double kBegin = 5;
    const double units = (double)some * ((each + p.rows - 1) / p.rows) * Hkv, share = units / slots;
    double whole = kBegin + most;
    if (share > 1) whole = std::max(whole, share * (kBegin + most - cut / 2) + (std::ceil(share) - share) * (kBegin + most - cut));
    else if (slots > cus && units <= cus) whole *= 0.6;
    if (whole <= kBegin * (2 + share) + share * list || p.units * (list + 2) > 2147483647.0) return p;
    // A run that goes on with a second unit begins anew.  Where units of that length cut into equal parts make no longer runs
    // than that costs, there are as many runs as parts, and with equal lengths each is of one unit (40 heads on 8, bf16: a
    // tree of 16 on 4000 43.7 -> 27.5 us, of 16 on 1000 30 -> 20, 256 tokens on 3000 64 -> 49, 512 on 8192 131 -> 122).
    const double parts = std::floor(std::min(1 / share, list / kLeast));
    p.runs = parts >= 1 && list / parts <= share * list + kBegin ? (int64_t)(units * parts) : slots;
    const int DD = D <= 64 ? 64 : D <= 128 ? 128 : 256;
    p.bytes = 2 * p.runs * part_floats(p.rows, DD) * 4;
    return p;
}

int run(int codes, int dtype, Args &a, const Plan &p, void *workspace, int64_t workspace_bytes, hipStream_t st)
{
    if (int e = require_device()) return e;
    const unsigned g = (unsigned)p.units;
    a.rows = p.rows;
    if (p.runs && workspace && workspace_bytes >= p.bytes && sums_fit(p.units, (int64_t)a.cols * a.page, a.N ? a.N : a.T, a.window, a.sinks, kKeys))
        a.runs = (int)p.runs, a.least = kLeast, a.part = (float *)workspace;
    if (codes == PSQ_CODES_I8) return dtype == PSQ_BF16 ? launch_bf16_i8(a, g, st) : launch_f16_i8(a, g, st);
    if (codes == PSQ_CODES_E4M3) return dtype == PSQ_BF16 ? launch_bf16_fp8(a, g, st) : launch_f16_fp8(a, g, st);
    return dtype == PSQ_BF16 ? launch_bf16(a, g, st) : launch_f16(a, g, st);
}

}  // namespace
}  // namespace block
}  // namespace psq

extern "C" {

int64_t psq_paged_block_workspace_bytes(int codes, int64_t T, int64_t B, int N, int Hq, int Hkv, int D, int64_t window, int64_t sinks, int64_t max_len)
{
    if (T <= 0 || B <= 0 || N < 0 || N > 64 || Hq <= 0 || Hkv <= 0 || D <= 0 || D > 256 || window < 0 || sinks < 0 || max_len <= 0 || Hq % Hkv ||
        B > 65535 || T > 0x3fffffffLL / Hq)
        return 0;
    return psq::block::plan(codes, T, B, N, Hq, Hkv, D, window, sinks, std::min<int64_t>(max_len, 0x3fffffffLL)).bytes;
}

int psq_paged_prompt_attention(int codes, const void *q, int dtype, int64_t q_token, int64_t q_head, const void *k_cache,
                               const void *v_cache, const float *k_scale, const float *v_scale, int64_t num_pages, int page_size,
                               const int32_t *block_table, int64_t table_stride, int64_t table_cols, const int32_t *starts,
                               const int32_t *lengths, int64_t B, int64_t T, int Hq, int Hkv, int D, float scale, int64_t window,
                               int64_t sinks, int64_t max_len, void *out, float *lse, void *workspace, int64_t workspace_bytes, void *stream)
{
    using namespace psq;
    using namespace psq::block;
    const char *name = "paged_prompt_attention";
    Args a{};
    const int e = check(name, a, codes, q, dtype, q_token, q_head, k_cache, v_cache, k_scale, v_scale, num_pages, page_size, block_table,
                        table_stride, table_cols, lengths, B, T, Hq, Hkv, D, scale, window, sinks, max_len, out, lse, workspace, workspace_bytes);
    if (e <= 0) return e;
    if (!starts) return set_error(PSQ_E_ARG, "%s: null pointer", name);
    if ((uintptr_t)starts & 3) return set_error(PSQ_E_SHAPE, "%s: misaligned starts", name);
    a.starts = starts;
    return run(codes, dtype, a, plan(codes, T, B, 0, Hq, Hkv, D, window, sinks, std::min(max_len, table_cols * page_size)), workspace, workspace_bytes, (hipStream_t)stream);
}

int psq_paged_tree_attention(int codes, const void *q, int dtype, int64_t q_token, int64_t q_head, const void *k_cache,
                             const void *v_cache, const float *k_scale, const float *v_scale, int64_t num_pages, int page_size,
                             const int32_t *block_table, int64_t table_stride, int64_t table_cols, const int32_t *lengths,
                             const int32_t *parents, const int32_t *drafts, int64_t B, int N, int Hq, int Hkv, int D, float scale,
                             int64_t window, int64_t sinks, int64_t max_len, void *out, float *lse, void *workspace, int64_t workspace_bytes,
                             void *stream)
{
    using namespace psq;
    using namespace psq::block;
    const char *name = "paged_tree_attention";
    if (N < 0) return set_error(PSQ_E_ARG, "%s: negative size", name);
    if (N > 64) return set_error(PSQ_E_SHAPE, "%s: %d drafts, at most 64", name, N);
    Args a{};
    const int e = check(name, a, codes, q, dtype, q_token, q_head, k_cache, v_cache, k_scale, v_scale, num_pages, page_size, block_table,
                        table_stride, table_cols, lengths, B, B < 0 ? -1 : B * N, Hq, Hkv, D, scale, window, sinks, max_len, out, lse, workspace,
                        workspace_bytes);
    if (e <= 0) return e;
    if (!parents) return set_error(PSQ_E_ARG, "%s: null pointer", name);
    if (((uintptr_t)parents | (uintptr_t)drafts) & 3) return set_error(PSQ_E_SHAPE, "%s: misaligned parents or drafts", name);
    a.N = N, a.parents = parents, a.drafts = drafts;
    return run(codes, dtype, a, plan(codes, 0, B, N, Hq, Hkv, D, window, sinks, std::min(max_len, table_cols * page_size)), workspace, workspace_bytes, (hipStream_t)stream);
}

}  // extern "C"
