// The 8-bit product ring (qgemm_ring.h) with fp16 outputs.
#include "qgemm_ring.h"

SOX_QGEMM(f16, half_t, 256x256_w8k128s2, 256, 256, 128, 128, 64, 2, 8, 2, 4, Q_CHUNKS)
SOX_QGEMM_TILES(f16, half_t)
