// mxfp4.h -- blocks of 32 values as 4-bit codes with one power-of-two scale (the OCP microscaling
// format MXFP4), and the index arithmetic that the element-wise kernels share.
//
// A block's scale is an exponent byte e (E8M0): 2^(e - 127), or NaN for e = 255.  A code (E2M1) is a
// sign and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6; element 2i of a row is the low half of byte i.  For a
// block whose largest magnitude is A:
//   e = max(floor(log2 A) - 2 + 127, 0)     so that A * 2^(127 - e) lies in [4, 8)
//   code = e2m1(x * 2^(127 - e))            to nearest, ties to even, at most 6 in magnitude
// floor(log2 A) + 127 is A's exponent field as a binary32 value, and 0 where that is subnormal or
// zero: e is then 0 too.  A block with a NaN or an infinity has no such scale: e = 255, codes 0, and
// all of it reads back as NaN.  Scaling by a power of two is exact, so the only rounding is the code's.
// The hardware's conversion (v_cvt_scalef32_pk_fp4_*) takes the scale as the exponent field of a
// binary32 operand, 0 standing for 2^-127; it gives this rounding for every 16-bit input and every
// scale byte below 255 (tests/test_gpu_mxfp4.py).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "rowkern.h"

namespace mcop {

constexpr int kMxBlock = 32;
constexpr uint32_t kInfBits = 0x7f800000u;

// The larger of two packed pairs of 16-bit magnitudes.
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a),
                                                                __builtin_bit_cast(u16x2, b)));
}

// Binary32 bits of the largest magnitude of eight values; NaN's bits where one is NaN (magnitudes
// order as their bits do, with NaN above infinity).
template <class E>
__device__ __forceinline__ uint32_t absmax8(const Pack<typename E::S, 8>& p) {
  if constexpr (sizeof(typename E::S) == 2) {
    const Pack<uint32_t, 4> w = __builtin_bit_cast(Pack<uint32_t, 4>, p);
    uint32_t m = w.v[0] & 0x7fff7fffu;
#pragma unroll
    for (int k = 1; k < 4; ++k) m = max_u16x2(m, w.v[k] & 0x7fff7fffu);
    const uint32_t lo = m & 0xffffu, hi = m >> 16;
    return __builtin_bit_cast(uint32_t, E::to_f((uint16_t)(lo > hi ? lo : hi)));
  } else {
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t b = __builtin_bit_cast(uint32_t, p.v[e]) & 0x7fffffffu;
      m = b > m ? b : m;
    }
    return m;
  }
}
template <int N>
__device__ __forceinline__ uint32_t absmax_bits(const float* f) {
  uint32_t m = 0;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const uint32_t b = __builtin_bit_cast(uint32_t, f[e]) & 0x7fffffffu;
    m = b > m ? b : m;
  }
  return m;
}

// The largest over aligned runs of `lanes` lanes (a power of two of at most 64).
__device__ __forceinline__ uint32_t lanes_max(uint32_t v, int lanes) {
  const AbsMaxOp op;
  if (lanes >= 2) v = op(v, dpp_mov<kDppXor1>(v));
  if (lanes >= 4) v = op(v, dpp_mov<kDppXor2>(v));
  if (lanes >= 8) v = op(v, dpp_mov<kDppHalfMirror>(v));
  if (lanes >= 16) v = op(v, dpp_mov<kDppMirror>(v));
  if (lanes >= 32) v = op(v, (uint32_t)__shfl_xor((int)v, 16, 64));
  if (lanes >= 64) v = op(v, (uint32_t)__shfl_xor((int)v, 32, 64));
  return v;
}

// A block's scale byte from the bits of its largest magnitude, the conversion's operand for it, and
// the value it stands for.
__device__ __forceinline__ uint32_t mx_scale(uint32_t most) {
  const uint32_t field = most >> 23;
  return most >= kInfBits ? 255u : (field > 2 ? field - 2 : 0u);
}
__device__ __forceinline__ float mx_operand(uint32_t e) {
  return __builtin_bit_cast(float, e << 23);
}
__device__ __forceinline__ float mx_value(uint32_t e) {
  return __builtin_bit_cast(float, e == 255 ? 0x7fc00000u : (e == 0 ? 0x00400000u : e << 23));
}

// Eight codes (a dword) of values in the block whose scale byte is e.
template <class E>
__device__ __forceinline__ uint32_t mx_codes8(const Pack<typename E::S, 8>& p, uint32_t e) {
  const float s = mx_operand(e);
  uint32_t r = 0;
  if constexpr (std::is_same_v<E, BF16>) {
    const Pack<bf16x2, 4> w = __builtin_bit_cast(Pack<bf16x2, 4>, p);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, w.v[0], s, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, w.v[1], s, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, w.v[2], s, 2);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, w.v[3], s, 3);
  } else if constexpr (std::is_same_v<E, F16>) {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    const Pack<f16x2, 4> w = __builtin_bit_cast(Pack<f16x2, 4>, p);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, w.v[0], s, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, w.v[1], s, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, w.v[2], s, 2);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, w.v[3], s, 3);
  } else {
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, p.v[0], p.v[1], s, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, p.v[2], p.v[3], s, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, p.v[4], p.v[5], s, 2);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, p.v[6], p.v[7], s, 3);
  }
  return e == 255 ? 0u : r;
}
// The same of N = 4 or 8 binary32 values (four codes are two bytes).
template <int N>
__device__ __forceinline__ uint32_t mx_codes(const float* f, uint32_t e) {
  const float s = mx_operand(e);
  uint32_t r = 0;
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, f[0], f[1], s, 0);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, f[2], f[3], s, 1);
  if constexpr (N == 8) {
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, f[4], f[5], s, 2);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, f[6], f[7], s, 3);
  }
  return e == 255 ? 0u : r;
}

// The values of eight codes, in binary32: exact, infinite past its range.
__device__ __forceinline__ void mx_widen8(float* f, uint32_t codes, uint32_t e) {
  const float s = mx_value(e);
  typedef float f2 __attribute__((ext_vector_type(2)));
  const f2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.0f, 0);
  const f2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.0f, 1);
  const f2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.0f, 2);
  const f2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.0f, 3);
  f[0] = a[0] * s, f[1] = a[1] * s, f[2] = b[0] * s, f[3] = b[1] * s;
  f[4] = c[0] * s, f[5] = c[1] * s, f[6] = d[0] * s, f[7] = d[1] * s;
}

// Eight values as one 16-byte access, streamed, or (fp32) two, each half of every 32 bytes and therefore
// not: streamed, the halves went to memory apart (65536 tokens of 8 x 128 read to fp32 257 us, 171
// so).  LOOSE: at any element alignment.
template <class T, bool LOOSE, bool NT = (sizeof(T) < 4)>
__device__ __forceinline__ Pack<T, 8> load8(const T* p) {
  constexpr int N = 16 / (int)sizeof(T) < 8 ? 16 / (int)sizeof(T) : 8, K = 8 / N;
  constexpr int F = LOOSE ? FORM_RAGGED : FORM_ROWS;
  Pack<T, 8> r;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const Pack<T, N> v = NT ? ldf_nt<F, T, N>(p + k * N) : ldf<F, T, N>(p + k * N);
#pragma unroll
    for (int e = 0; e < N; ++e) r.v[k * N + e] = v.v[e];
  }
  return r;
}
template <class T, bool LOOSE>
__device__ __forceinline__ void store8(T* p, const Pack<T, 8>& v) {
  constexpr int N = 16 / (int)sizeof(T) < 8 ? 16 / (int)sizeof(T) : 8, K = 8 / N;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    Pack<T, N> o;
#pragma unroll
    for (int e = 0; e < N; ++e) o.v[e] = v.v[k * N + e];
    if constexpr (K == 1) stf_nt<(LOOSE ? FORM_RAGGED : FORM_ROWS), T, N>(p + k * N, o);
    else __builtin_memcpy(p + k * N, &o, sizeof(o));
  }
}

// n / d for 0 <= n < 2^31 and a divisor d in [1, 2^31) fixed for the launch (Granlund and Montgomery,
// PLDI 1994): with s = ceil(log2 d) and m = floor(2^32 (2^s - d) / d) + 1 it is
// (hi(n * m) + n) >> s; the sum stays below 2^32 as hi(n * m) <= n.
struct Divisor {
  uint32_t d, mul, shift;
  Divisor() = default;
  explicit Divisor(uint32_t div) : d(div), mul(0), shift(0) {
    while (shift < 31 && (1u << shift) < d) ++shift;
    mul = (uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << shift) - d)) / d + 1);
  }
  __device__ __forceinline__ uint32_t quotient(uint32_t n) const {
    return (__umulhi(n, mul) + n) >> shift;
  }
};

}  // namespace mcop
