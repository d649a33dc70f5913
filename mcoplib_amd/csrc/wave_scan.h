// wave_scan.h -- inclusive sums over a wave's 64 lanes by register moves: within rows of 16, then across them.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mcop {

struct ScanAdd {
  __device__ __forceinline__ uint32_t operator()(uint32_t a, uint32_t b) const { return a + b; }
};
// Sums that stop at 2^31 - 1 (of values up to that).
struct ScanAddUpTo31 {
  __device__ __forceinline__ uint32_t operator()(uint32_t a, uint32_t b) const {
    return min(a + b, 0x7fffffffu);
  }
};

template <class Op = ScanAdd>
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
  const Op op;
  v = op(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xf, 0xf, false));  // row_shr:1
  v = op(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xf, 0xf, false));
  v = op(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xf, 0xf, false));
  v = op(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xf, 0xf, false));
  v = op(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, false));  // row_bcast:15
  v = op(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, false));  // row_bcast:31
  return v;
}
__device__ __forceinline__ uint32_t wave_total(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_readlane((int)wave_scan(v), 63);
}

}  // namespace mcop
