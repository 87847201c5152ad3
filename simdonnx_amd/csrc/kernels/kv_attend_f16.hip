// Attention over a paged cache of f16 (kv_attend.h), and the join of its splits
#include "kv_attend.h"
KV_ATTEND_DIMS(f16, half_t, half_t)
extern "C" __global__ void __launch_bounds__(256) sox_kv_merge_f16(sox_kv_attend_args p) { attend_merge<half_t>(p); }
