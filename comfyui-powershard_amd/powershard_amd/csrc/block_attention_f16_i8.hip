// block_attention_f16_i8.hip -- the kernels of block_attention.hpp for f16 rows on int8 caches.
#include "block_attention.hpp"

int psq::block::launch_f16_i8(const Args &a, unsigned groups, hipStream_t st) { return launch_dim<PSQ_F16, PSQ_CODES_I8>(a, groups, st); }
