// block_attention_bf16_fp8.hip -- the kernels of block_attention.hpp for bf16 rows on e4m3 caches.
#include "block_attention.hpp"

int psq::block::launch_bf16_fp8(const Args &a, unsigned groups, hipStream_t st) { return launch_dim<PSQ_BF16, PSQ_CODES_E4M3>(a, groups, st); }
