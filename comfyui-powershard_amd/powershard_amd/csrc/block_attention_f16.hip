// block_attention_f16.hip -- the kernels of block_attention.hpp for f16 rows on 16-bit caches.
#include "block_attention.hpp"

int psq::block::launch_f16(const Args &a, unsigned groups, hipStream_t st) { return launch_dim<PSQ_F16, PSQ_CODES_NONE>(a, groups, st); }
