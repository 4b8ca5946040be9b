// blocks_norm_f32.hip -- the residual-norm kernels (blocks_norm.h) in f32
#include "blocks_norm.h"
namespace blk {
int norm_f32(const NormArgs& a, int sh, bool back, int64_t blocks, hipStream_t s) { return norm_pick<float, float>(a, sh, back, blocks, s); }
}  // namespace blk
