// Attention over a paged cache in 8 bits, queries and outputs in f16 (kv_attend.h)
#include "kv_attend.h"
KV_ATTEND_DIMS(f16_i8, half_t, int8_t)
