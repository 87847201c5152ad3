// Attention over a paged cache of bf16 (kv_attend.h), and the join of its splits
#include "kv_attend.h"
KV_ATTEND_DIMS(bf16, bf16_t, bf16_t)
extern "C" __global__ void __launch_bounds__(256) sox_kv_merge_bf16(sox_kv_attend_args p) { attend_merge<bf16_t>(p); }
