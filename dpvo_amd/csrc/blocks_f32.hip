// blocks_f32.hip -- the matrix products of the gated blocks (blocks_gemm.h) on float operands
#define BLK_T float
#define BLK_ENTRY gemm_f32
#include "blocks_gemm.h"
