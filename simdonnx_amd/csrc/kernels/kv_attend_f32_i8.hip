// Attention over a paged cache in 8 bits, queries and outputs in f32 (kv_attend.h)
#include "kv_attend.h"
KV_ATTEND_DIMS(f32_i8, float, int8_t)
