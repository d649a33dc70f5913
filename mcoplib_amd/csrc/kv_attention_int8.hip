// kv_attention_int8.hip -- the matrix kernels of decode attention over a cache of int8 vectors.
#include "kv_attention_tiles.h"

namespace mcop {

int attention_tiles_int8(int shape, bool lines, mcop_dtype dtype, const AttArgs& a, dim3 grid,
                         hipStream_t st) {
  return attention_tiles_for<KV_INT8>(shape, lines, dtype, a, grid, st);
}

}  // namespace mcop
