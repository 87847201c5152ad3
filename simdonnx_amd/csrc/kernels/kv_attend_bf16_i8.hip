// Attention over a paged cache in 8 bits, queries and outputs in bf16 (kv_attend.h)
#include "kv_attend.h"
KV_ATTEND_DIMS(bf16_i8, bf16_t, int8_t)
