// block_plan.hpp -- what the host works out of a call of block attention that needs no device (block_attention.hpp).
#pragma once

#include <algorithm>
#include <cstdint>

namespace psq {
namespace block {

// Whether the key tiles of all units, as the device adds them up in 32 bits to cut them into runs, stay below 2^32.  The
// lengths that it finds are not bounded by max_len but by the table: one past it counts as the table's tokens, the rows
// n and a tile.  A window leaves its own tokens, the sinks' and the rows', and a tile more at each of their four ends.
inline bool sums_fit(int64_t units, int64_t table_tokens, int64_t n, int64_t window, int64_t sinks, int keys)
{
    int64_t tokens = table_tokens + n + 2 * keys;
    if (window) tokens = std::min(tokens, window + sinks + n + 4 * keys);
    return units <= 0xffffffffLL / (tokens / keys + 1);
}

}  // namespace block
}  // namespace psq
