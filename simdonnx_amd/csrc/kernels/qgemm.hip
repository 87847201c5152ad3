// The 8-bit product ring (qgemm_ring.h) with fp16 outputs.
#include "qgemm_ring.h"

SOX_QGEMM_TILES(f16, half_t)
