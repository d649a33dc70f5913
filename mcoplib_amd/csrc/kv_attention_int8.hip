// kv_attention_int8.hip -- the matrix kernels of decode attention over a cache of int8 vectors.
#include "kv_attention_tiles.h"

namespace mcop {

int attention_tiles_int8(int shape, mcop_dtype dtype, const AttArgs& a, dim3 grid, size_t lds,
                         hipStream_t st) {
  return attention_tiles_for<KV_INT8>(shape, dtype, a, grid, lds, st);
}

}  // namespace mcop
