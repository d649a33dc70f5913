// mxfp4_mm.hip -- product of two operands of 4-bit blocks (mxfp4.h) on the matrix units:
//   out[m, n] = b(sum_k A[m, k] B[n, k] (+ bias[n])), summed in fp32.
//
// A scaled matrix instruction takes one block of each operand a lane -- 16 bytes of codes and a byte of
// a scale register -- and multiplies by both scales as it sums, so codes go from memory to the
// matrix unit as they are.  Which K a lane's block has is free as long as both operands agree: in
// 16x16x128 instructions the lane of group g = lane / 16 takes blocks 4g..4g+3 of every 16 (512
// values), one in each of four instructions, so that its scales are one dword whose bytes the
// instructions pick in turn.  The weights are the first operand: a lane then holds four consecutive n
// of one m.
#include <hip/hip_runtime.h>

#include "../../include/mcop_norm.h"
#include "mxfp4.h"

namespace mcop {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kFp4 = 4;  // operand format of the matrix instructions

__device__ __forceinline__ i32x8 fp4_operand(i32x4 v) {
  return __builtin_shufflevector(v, v, 0, 1, 2, 3, -1, -1, -1, -1);
}

// Scale bytes b..b+3 of a row of `blocks`, zero past its end (where the codes are zero as well).
template <bool DWORDS>
__device__ __forceinline__ uint32_t scales4(const uint8_t* row, int b, int blocks) {
  if constexpr (DWORDS) {
    return b < blocks ? *reinterpret_cast<const uint32_t*>(row + b) : 0u;
  } else {
    uint32_t v = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (b + e < blocks) v |= (uint32_t)row[b + e] << (8 * e);
    }
    return v;
  }
}

// Few rows: a workgroup makes 16 x 16 of the output, its four waves every fourth chunk of 512 along
// K, straight from memory; the partial sums meet in LDS in the waves' order.
template <class E, bool DWORDS>
__global__ void __launch_bounds__(256)
k_mxfp4_mm_rows(typename E::S* __restrict__ out, const uint8_t* __restrict__ a,
                const uint8_t* __restrict__ as, const uint8_t* __restrict__ b,
                const uint8_t* __restrict__ bs, const typename E::S* __restrict__ bias, int M, int N,
                int blocks) {
  __shared__ f32x4 part[3][64];
  const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
  const int r = lane & 15, g = lane >> 4;
  const int n0 = (int)blockIdx.x * 16, m0 = (int)blockIdx.y * 16;
  const int64_t n = min(n0 + r, N - 1), m = min(m0 + r, M - 1);
  const uint8_t* bp = b + n * blocks * 16;
  const uint8_t* ap = a + m * blocks * 16;
  const uint8_t* bsp = bs + n * blocks;
  const uint8_t* asp = as + m * blocks;
  f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int k = wave * 16; k < blocks; k += 64) {
    const int at = k + 4 * g;
    const uint32_t sb = scales4<DWORDS>(bsp, at, blocks), sa = scales4<DWORDS>(asp, at, blocks);
    i32x4 vb[4], va[4];
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      vb[s] = i32x4{0, 0, 0, 0}, va[s] = i32x4{0, 0, 0, 0};
      if (at + s < blocks) {
        vb[s] = *reinterpret_cast<const i32x4*>(bp + (int64_t)(at + s) * 16);
        va[s] = *reinterpret_cast<const i32x4*>(ap + (int64_t)(at + s) * 16);
      }
    }
#define MCOP_MM(S)                                                                              \
  sum = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fp4_operand(vb[S]), fp4_operand(va[S]), \
                                                         sum, kFp4, kFp4, S, (int)sb, S, (int)sa)
    MCOP_MM(0);
    MCOP_MM(1);
    MCOP_MM(2);
    MCOP_MM(3);
#undef MCOP_MM
  }
  if (wave > 0) part[wave - 1][lane] = sum;
  __syncthreads();
  if (wave > 0) return;
#pragma unroll
  for (int w = 0; w < 3; ++w) sum += part[w][lane];
  if (m0 + r >= M) return;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = n0 + 4 * g + i;
    if (c < N) {
      float v = sum[i];
      if (bias != nullptr) v += E::to_f(bias[c]);
      out[(int64_t)(m0 + r) * N + c] = E::from_f(v);
    }
  }
}

template <class E>
static int product(void* out, const uint8_t* a, const uint8_t* as, const uint8_t* b,
                   const uint8_t* bs, const void* bias, int M, int N, int blocks, hipStream_t st) {
  using S = typename E::S;
  auto* o = static_cast<S*>(out);
  const auto* bi = static_cast<const S*>(bias);
  const dim3 grid((unsigned)((N + 15) / 16), (unsigned)((M + 15) / 16)), block(256);
  if (blocks % 4 == 0 && aligned(4, as, bs)) {
    hipLaunchKernelGGL((k_mxfp4_mm_rows<E, true>), grid, block, 0, st, o, a, as, b, bs, bi, M, N,
                       blocks);
  } else {
    hipLaunchKernelGGL((k_mxfp4_mm_rows<E, false>), grid, block, 0, st, o, a, as, b, bs, bi, M, N,
                       blocks);
  }
  return check_launch("mxfp4_scaled_mm");
}

}  // namespace mcop

extern "C" int mcop_mxfp4_scaled_mm(void* out, mcop_dtype out_dtype, const uint8_t* a,
                                    const uint8_t* a_scales, const uint8_t* b,
                                    const uint8_t* b_scales, const void* bias, int64_t M,
                                    int64_t N, int64_t K, void* stream) {
  using namespace mcop;
  const char* name = "mxfp4_scaled_mm";
  if (M < 0 || N < 0 || K <= 0 || K > INT32_MAX) {
    return set_error(MCOP_E_INVALID, "%s: bad shape M=%lld N=%lld K=%lld", name, (long long)M,
                     (long long)N, (long long)K);
  }
  if (K % kMxBlock != 0) {
    return set_error(MCOP_E_INVALID, "%s: K %lld is not a multiple of the block of 32", name,
                     (long long)K);
  }
  if (M == 0 || N == 0) return MCOP_OK;
  // the grid: at most 2^31 - 1 workgroups along N, 65535 along M
  if (N > ((int64_t)1 << 30) || M > (int64_t)65535 * 16) {
    return set_error(MCOP_E_UNSUPPORTED, "%s: M %lld or N %lld is more than one launch takes "
                     "(%d and 2^30)", name, (long long)M, (long long)N, 65535 * 16);
  }
  if (!out || !a || !a_scales || !b || !b_scales) {
    return set_error(MCOP_E_INVALID, "%s: null pointer", name);
  }
  if (!aligned(16, a, b)) {
    return set_error(MCOP_E_INVALID, "%s: codes must be aligned to 16 bytes", name);
  }
  auto st = static_cast<hipStream_t>(stream);
  const int m = (int)M, n = (int)N, blocks = (int)(K / kMxBlock);
  switch (out_dtype) {
    case MCOP_BF16: return product<BF16>(out, a, a_scales, b, b_scales, bias, m, n, blocks, st);
    case MCOP_F16: return product<F16>(out, a, a_scales, b, b_scales, bias, m, n, blocks, st);
    case MCOP_F32: return product<F32>(out, a, a_scales, b, b_scales, bias, m, n, blocks, st);
    default:
      return set_error(MCOP_E_INVALID, "%s: out dtype %d is not bf16/fp16/fp32", name,
                       (int)out_dtype);
  }
}
