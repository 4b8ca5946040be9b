// blocks_norm_bf16.hip -- the residual-norm kernels (blocks_norm.h) with __bf16 branches and __bf16 or f32 residual streams
#include "blocks_norm.h"
namespace blk {
int norm_bf16(const NormArgs& a, int sh, bool back, int64_t blocks, hipStream_t s) {
  return a.p.x_dtype == DPVO_F32 ? norm_pick<float, __bf16>(a, sh, back, blocks, s) : norm_pick<__bf16, __bf16>(a, sh, back, blocks, s);
}
}  // namespace blk
