// Attention over a paged cache of f32 (kv_attend.h), and the join of its splits
#include "kv_attend.h"
KV_ATTEND_DIMS(f32, float, float)
extern "C" __global__ void __launch_bounds__(256) sox_kv_merge_f32(sox_kv_attend_args p) { attend_merge<float>(p); }
