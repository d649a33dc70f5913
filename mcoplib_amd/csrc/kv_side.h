// kv_side.h -- one side (keys or values) of the quantized paged cache, as its kernels take it, and the
// checks of it that the cache's entry points share.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/mcop_norm.h"
#include "mxfp4.h"

namespace mcop {

constexpr int kKvMostDim = 1024;

enum KvFormat { KV_INT8 = 0, KV_FP8 = 1, KV_MXFP4 = 2 };

// One side (keys or values) of a launch.  Strides of the cache are in bytes for codes, in elements for
// scales; those of the plain tensor in elements.
struct KvSide {
  void* plain;
  uint8_t* codes;
  void* scales;
  int64_t p_token, p_head;
  int64_t c_page, c_token, c_head;
  int64_t s_page, s_token, s_head;
  int dim, lanes;
  Divisor by_passes;  // waves that a token's heads take
};

// The checks that the entry points share of one side, and its form for the kernels.  `heads` is the
// larger of the plain tensor's and the cache's.
inline int side_of(const char* name, const char* what, const mcop_kv_side& in, int fmt,
                   int64_t pages, int64_t page_size, int64_t heads, int64_t tokens, KvSide* out) {
  if (in.head_size <= 0 || in.head_size > kKvMostDim) {
    return set_error(MCOP_E_INVALID, "%s: %s head_size %lld is not in 1..%d", name, what,
                     (long long)in.head_size, kKvMostDim);
  }
  if (fmt == KV_MXFP4 && in.head_size % kMxBlock != 0) {
    return set_error(MCOP_E_INVALID, "%s: %s head_size %lld is not a multiple of the block of 32",
                     name, what, (long long)in.head_size);
  }
  if (!in.plain || (pages > 0 && (!in.codes || !in.scales))) {
    return set_error(MCOP_E_INVALID, "%s: null pointer", name);
  }
  // element offsets of the last vector, which the kernels form in 64 bits
  const int64_t n[8] = {pages, page_size, heads, pages, page_size, heads, tokens, heads};
  const int64_t s[8] = {in.code_page_stride, in.code_token_stride, in.code_head_stride,
                        in.scale_page_stride, in.scale_token_stride, in.scale_head_stride,
                        in.token_stride, in.head_stride};
  for (int d = 0; d < 8; ++d) {
    if (s[d] < 0 || (n[d] > 0 && s[d] > INT64_MAX / 64 / n[d])) {
      return set_error(MCOP_E_INVALID, "%s: bad %s stride %lld", name, what, (long long)s[d]);
    }
  }
  int lanes = 4;
  while (lanes < 64 && lanes * 8 < in.head_size) lanes *= 2;
  *out = KvSide{in.plain, static_cast<uint8_t*>(in.codes), in.scales, in.token_stride,
                in.head_stride, in.code_page_stride, in.code_token_stride, in.code_head_stride,
                in.scale_page_stride, in.scale_token_stride, in.scale_head_stride,
                (int)in.head_size, lanes, Divisor((uint32_t)((heads * lanes + 63) / 64))};
  return MCOP_OK;
}

inline int format_of(mcop_dtype t) {
  return t == MCOP_I8 ? KV_INT8 : t == MCOP_FP8_E4M3FN ? KV_FP8 : t == MCOP_MXFP4 ? KV_MXFP4 : -1;
}

}  // namespace mcop
