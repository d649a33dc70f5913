// mxfp4_quant.hip -- rows as 4-bit codes with a scale for each 32 values (mxfp4.h), and back.
//
// Both are bound by HBM: 2 + 17/32 bytes an element of a 16-bit tensor.  A lane takes eight
// consecutive values (16 bytes of a 16-bit type, a dword of codes), so that a wave's instruction reads
// 1 KiB in a row, and a block is four lanes, whose largest magnitude is two register moves away.
#include <hip/hip_runtime.h>

#include "../../include/mcop_norm.h"
#include "launch_trace.h"
#include "mxfp4.h"

namespace mcop {

constexpr int kQuantLanes = 256;
constexpr int kQuantUnits = 4;  // of eight values, a lane

// `units` of eight values in all, `row.d` a row.
template <class E, bool LOOSE>
__global__ void __launch_bounds__(kQuantLanes)
k_mxfp4_quant(uint32_t* __restrict__ out, uint8_t* __restrict__ scales,
              const typename E::S* __restrict__ x, int64_t stride, uint32_t units, Divisor row) {
  using S = typename E::S;
  const uint32_t u0 = blockIdx.x * (uint32_t)(kQuantLanes * kQuantUnits) + threadIdx.x;
  Pack<S, 8> v[kQuantUnits];
#pragma unroll
  for (int k = 0; k < kQuantUnits; ++k) {
    uint32_t u = u0 + k * kQuantLanes;
    u = u < units ? u : units - 1;
    const uint32_t r = row.quotient(u);
    v[k] = load8<S, LOOSE>(x + r * stride + (int64_t)(u - r * row.d) * 8);
  }
#pragma unroll
  for (int k = 0; k < kQuantUnits; ++k) {
    const uint32_t u = u0 + k * kQuantLanes;
    // rows are whole blocks, so a block's four lanes are all inside or all past the end
    const uint32_t e = mx_scale(lanes_max(absmax8<E>(v[k]), 4));
    if (u >= units) continue;
    out[u] = mx_codes8<E>(v[k], e);
    if ((u & 3) == 0) scales[u >> 2] = (uint8_t)e;
  }
}

template <class E, bool LOOSE>
__global__ void __launch_bounds__(kQuantLanes)
k_mxfp4_dequant(typename E::S* __restrict__ out, const uint32_t* __restrict__ codes,
                const uint8_t* __restrict__ scales, uint32_t units) {
  using S = typename E::S;
  const uint32_t u0 = blockIdx.x * (uint32_t)(kQuantLanes * kQuantUnits) + threadIdx.x;
  uint32_t c[kQuantUnits], e[kQuantUnits];
#pragma unroll
  for (int k = 0; k < kQuantUnits; ++k) {
    uint32_t u = u0 + k * kQuantLanes;
    u = u < units ? u : units - 1;
    c[k] = __builtin_nontemporal_load(codes + u);
    e[k] = scales[u >> 2];
  }
#pragma unroll
  for (int k = 0; k < kQuantUnits; ++k) {
    const uint32_t u = u0 + k * kQuantLanes;
    if (u >= units) continue;
    float f[8];
    mx_widen8(f, c[k], e[k]);
    Pack<S, 8> o;
#pragma unroll
    for (int i = 0; i < 8; ++i) o.v[i] = E::from_f(f[i]);
    store8<S, LOOSE>(out + (int64_t)u * 8, o);
  }
}

// Rows of one launch: its units stay below 2^31.
static int64_t rows_a_launch(int64_t hidden) { return ((int64_t)1 << 30) / (hidden / 8); }
static unsigned quant_blocks(int64_t units) {
  return (unsigned)((units + kQuantLanes * kQuantUnits - 1) / (kQuantLanes * kQuantUnits));
}

static void trace_rows(const char* name, int64_t rows, int64_t hidden, bool whole, unsigned blocks) {
  trace_launch(name, "rows=%lld hidden=%lld: %d units of 8 values a lane, %s, wgs=%u",
               (long long)rows, (long long)hidden, kQuantUnits,
               whole ? "aligned to 16 bytes" : "any alignment", blocks);
}

template <class E>
static int quant(uint8_t* out, uint8_t* scales, const void* input, int64_t rows, int64_t hidden,
                 int64_t stride, hipStream_t st) {
  using S = typename E::S;
  const bool whole = aligned(16, input) && (stride * (int64_t)sizeof(S)) % 16 == 0;
  const int64_t most = rows_a_launch(hidden);
  for (int64_t r = 0; r < rows; r += most) {
    const int64_t n = rows - r < most ? rows - r : most, units = n * (hidden / 8);
    auto* o = reinterpret_cast<uint32_t*>(out + r * (hidden / 2));
    uint8_t* s = scales + r * (hidden / kMxBlock);
    const S* x = static_cast<const S*>(input) + r * stride;
    const Divisor row((uint32_t)(hidden / 8));
    const dim3 grid(quant_blocks(units)), block(kQuantLanes);
    trace_rows("mxfp4_quant", n, hidden, whole, grid.x);
    if (whole) {
      hipLaunchKernelGGL((k_mxfp4_quant<E, false>), grid, block, 0, st, o, s, x, stride,
                         (uint32_t)units, row);
    } else {
      hipLaunchKernelGGL((k_mxfp4_quant<E, true>), grid, block, 0, st, o, s, x, stride,
                         (uint32_t)units, row);
    }
    if (int rc = check_launch("mxfp4_quant")) return rc;
  }
  return MCOP_OK;
}

template <class E>
static int dequant(void* out, const uint8_t* codes, const uint8_t* scales, int64_t rows,
                   int64_t hidden, hipStream_t st) {
  using S = typename E::S;
  const int64_t most = rows_a_launch(hidden);
  for (int64_t r = 0; r < rows; r += most) {
    const int64_t n = rows - r < most ? rows - r : most, units = n * (hidden / 8);
    S* o = static_cast<S*>(out) + r * hidden;
    const auto* c = reinterpret_cast<const uint32_t*>(codes + r * (hidden / 2));
    const uint8_t* s = scales + r * (hidden / kMxBlock);
    const dim3 grid(quant_blocks(units)), block(kQuantLanes);
    trace_rows("mxfp4_dequant", n, hidden, aligned(16, out), grid.x);
    if (aligned(16, out)) {
      hipLaunchKernelGGL((k_mxfp4_dequant<E, false>), grid, block, 0, st, o, c, s,
                         (uint32_t)units);
    } else {
      hipLaunchKernelGGL((k_mxfp4_dequant<E, true>), grid, block, 0, st, o, c, s,
                         (uint32_t)units);
    }
    if (int rc = check_launch("mxfp4_dequant")) return rc;
  }
  return MCOP_OK;
}

// The shape checks that both share; MCOP_OK with *empty set where there is nothing to do.
static int check_rows(const char* name, int64_t rows, int64_t hidden, const void* a, const void* b,
                      const void* c, bool* empty) {
  *empty = false;
  if (rows < 0 || hidden <= 0 || hidden > INT32_MAX) {
    return set_error(MCOP_E_INVALID, "%s: bad shape num_tokens=%lld hidden_size=%lld", name,
                     (long long)rows, (long long)hidden);
  }
  if (hidden % kMxBlock != 0) {
    return set_error(MCOP_E_INVALID, "%s: hidden_size %lld is not a multiple of the block of 32",
                     name, (long long)hidden);
  }
  if (rows > INT64_MAX / 8 / hidden) {
    return set_error(MCOP_E_INVALID, "%s: bad shape num_tokens=%lld hidden_size=%lld", name,
                     (long long)rows, (long long)hidden);
  }
  if (rows == 0) {
    *empty = true;
    return MCOP_OK;
  }
  if (!a || !b || !c) return set_error(MCOP_E_INVALID, "%s: null pointer", name);
  return MCOP_OK;
}

}  // namespace mcop

extern "C" int mcop_mxfp4_quant(uint8_t* out, uint8_t* scales, const void* input,
                                int64_t num_tokens, int64_t hidden_size,
                                int64_t input_row_stride, mcop_dtype in_dtype, void* stream) {
  using namespace mcop;
  const char* name = "mxfp4_quant";
  bool empty;
  if (int rc = check_rows(name, num_tokens, hidden_size, out, scales, input, &empty)) return rc;
  if (empty) return MCOP_OK;
  if (num_tokens > 1 && (input_row_stride < 0 ||
                         input_row_stride > INT64_MAX / 8 / num_tokens)) {
    return set_error(MCOP_E_INVALID, "%s: bad input_row_stride %lld", name,
                     (long long)input_row_stride);
  }
  if (!aligned(4, out)) {
    return set_error(MCOP_E_INVALID, "%s: out must be aligned to 4 bytes", name);
  }
  auto st = static_cast<hipStream_t>(stream);
  switch (in_dtype) {
    case MCOP_BF16:
      return quant<BF16>(out, scales, input, num_tokens, hidden_size, input_row_stride, st);
    case MCOP_F16:
      return quant<F16>(out, scales, input, num_tokens, hidden_size, input_row_stride, st);
    case MCOP_F32:
      return quant<F32>(out, scales, input, num_tokens, hidden_size, input_row_stride, st);
    default:
      return set_error(MCOP_E_INVALID, "%s: input dtype %d is not bf16/fp16/fp32", name,
                       (int)in_dtype);
  }
}

extern "C" int mcop_mxfp4_dequant(void* out, mcop_dtype out_dtype, const uint8_t* codes,
                                  const uint8_t* scales, int64_t num_tokens, int64_t hidden_size,
                                  void* stream) {
  using namespace mcop;
  const char* name = "mxfp4_dequant";
  bool empty;
  if (int rc = check_rows(name, num_tokens, hidden_size, out, codes, scales, &empty)) return rc;
  if (empty) return MCOP_OK;
  if (!aligned(4, codes)) {
    return set_error(MCOP_E_INVALID, "%s: codes must be aligned to 4 bytes", name);
  }
  auto st = static_cast<hipStream_t>(stream);
  switch (out_dtype) {
    case MCOP_BF16: return dequant<BF16>(out, codes, scales, num_tokens, hidden_size, st);
    case MCOP_F16: return dequant<F16>(out, codes, scales, num_tokens, hidden_size, st);
    case MCOP_F32: return dequant<F32>(out, codes, scales, num_tokens, hidden_size, st);
    default:
      return set_error(MCOP_E_INVALID, "%s: out dtype %d is not bf16/fp16/fp32", name,
                       (int)out_dtype);
  }
}
