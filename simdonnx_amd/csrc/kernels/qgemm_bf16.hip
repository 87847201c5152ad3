// The 8-bit product ring (qgemm_ring.h) with bf16 outputs.
#include "qgemm_ring.h"

SOX_QGEMM(bf16, bf16_t, 256x256_w8k128s2, 256, 256, 128, 128, 64, 2, 8, 2, 4, Q_CHUNKS)
SOX_QGEMM_TILES(bf16, bf16_t)
