// Tilings of the 8-bit product ring (qgemm_ring.h): BMxBN tile, wNW waves, kBK bytes of K per slice, sSTAGES.
#include "qgemm_ring.h"

SOX_QGEMM(256x256_w8k64s3, 256, 256, 64, 128, 64, 3, 8, 2, 4)
SOX_QGEMM(128x128_w4k64s2, 128, 128, 64, 64, 64, 2, 4, 2, 4)
SOX_QGEMM(64x64_w4k64s2, 64, 64, 64, 32, 32, 2, 4, 2, 4)
