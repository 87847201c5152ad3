// The 8-bit product ring (qgemm_ring.h) with fp32 outputs.
#include "qgemm_ring.h"

SOX_QGEMM_TILES(f32, float)
