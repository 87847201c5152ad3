// The 8-bit product ring (qgemm_ring.h) with bf16 outputs.
#include "qgemm_ring.h"

SOX_QGEMM_TILES(bf16, bf16_t)
