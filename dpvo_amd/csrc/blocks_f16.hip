// blocks_f16.hip -- the matrix products of the gated blocks (blocks_gemm.h) on _Float16 operands
#define BLK_T _Float16
#define BLK_ENTRY gemm_f16
#include "blocks_gemm.h"
