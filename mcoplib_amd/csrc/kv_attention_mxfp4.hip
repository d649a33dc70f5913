// kv_attention_mxfp4.hip -- the matrix kernels of decode attention over a cache of mxfp4 vectors.
#include "kv_attention_tiles.h"

namespace mcop {

int attention_tiles_mxfp4(int shape, mcop_dtype dtype, const AttArgs& a, dim3 grid, size_t lds,
                         hipStream_t st) {
  return attention_tiles_for<KV_MXFP4>(shape, dtype, a, grid, lds, st);
}

}  // namespace mcop
