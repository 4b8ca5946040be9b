// blocks_bf16.hip -- the matrix products of the gated blocks (blocks_gemm.h) on __bf16 operands
#define BLK_T __bf16
#define BLK_ENTRY gemm_bf16
#include "blocks_gemm.h"
