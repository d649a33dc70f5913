// kv_attention_mxfp4.hip -- the matrix kernels of decode attention over a cache of mxfp4 vectors.
#include "kv_attention_tiles.h"

namespace mcop {

int attention_tiles_mxfp4(int shape, bool lines, mcop_dtype dtype, const AttArgs& a, dim3 grid,
                          hipStream_t st) {
  return attention_tiles_for<KV_MXFP4>(shape, lines, dtype, a, grid, st);
}

}  // namespace mcop
