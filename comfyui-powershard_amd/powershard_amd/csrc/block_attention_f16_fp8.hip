// block_attention_f16_fp8.hip -- the kernels of block_attention.hpp for f16 rows on e4m3 caches.
#include "block_attention.hpp"

int psq::block::launch_f16_fp8(const Args &a, unsigned groups, hipStream_t st) { return launch_dim<PSQ_F16, PSQ_CODES_E4M3>(a, groups, st); }
