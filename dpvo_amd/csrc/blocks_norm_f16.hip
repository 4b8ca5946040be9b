// blocks_norm_f16.hip -- the residual-norm kernels (blocks_norm.h) with _Float16 branches and _Float16 or f32 residual streams
#include "blocks_norm.h"
namespace blk {
int norm_f16(const NormArgs& a, int sh, bool back, int64_t blocks, hipStream_t s) {
  return a.p.x_dtype == DPVO_F32 ? norm_pick<float, _Float16>(a, sh, back, blocks, s) : norm_pick<_Float16, _Float16>(a, sh, back, blocks, s);
}
}  // namespace blk
