// rms_norm_mxfp4.hip -- (residual add +) RMSNorm + 4-bit codes with a scale for each 32 values
// (mxfp4.h), one pass over HBM.
//
// Semantics (per row, a = x [+ r] in fp32, b() = round to the input dtype):
//   after_res <- b(a)
//   rho = 1/sqrt(sum(a^2)/H + eps)     the sum in fp64, every other step rounded to fp32
//   y = b(b(a * rho) * w)
//   scales, codes <- the blocks of 32 of y
// the arithmetic of the per-token and per-group norm-quant kernels up to y, so that y's bits are the
// norm's, and the codes those of mxfp4_quant on it.
//
// The lane mapping is the row kernels' (rowkern.h): vector j = v * tpr + lane.  A block is 32 / VEC
// consecutive lanes of one wave (four of a 16-bit type, eight of fp32).
#include <hip/hip_runtime.h>

#include "../../include/mcop_norm.h"
#include "mxfp4.h"

namespace mcop {

// Scale byte and codes of one vector of y, stored: VEC codes are VEC / 2 bytes.
template <int VEC>
__device__ __forceinline__ void store_block(uint8_t* out, uint8_t* scales, int64_t at,
                                            const float* y, uint32_t e) {
  const uint32_t q = mx_codes<VEC>(y, e);
  if constexpr (VEC == 8) *reinterpret_cast<uint32_t*>(out + at / 2) = q;
  else *reinterpret_cast<uint16_t*>(out + at / 2) = (uint16_t)q;
  if (at % kMxBlock == 0) scales[at / kMxBlock] = (uint8_t)e;
}

// LOOSE: tensors at any element alignment (rows are whole vectors all the same: hidden is a multiple
// of 32).
template <class E, int NV, bool RES, bool LOOSE>
__global__ void __launch_bounds__(max_tpr(E::VEC, NV))
k_rms_norm_mxfp4(uint8_t* __restrict__ out, uint8_t* __restrict__ scales,
                 const typename E::S* x, const typename E::S* __restrict__ w,
                 const typename E::S* res, typename E::S* after, int64_t rows, int hidden, int tpr,
                 float eps) {
  using S = typename E::S;
  constexpr int VEC = E::VEC, F = LOOSE ? FORM_RAGGED : FORM_ROWS;
  __shared__ double red_sum[16];
  const RowPos p = row_pos(rows, tpr);
  const int nvec = hidden / VEC;
  const int64_t base = p.row * (int64_t)hidden, lbase = p.lrow * (int64_t)hidden;
  Pack<S, VEC> xv[NV], rv[NV], wv[NV];
  auto lj_of = [&](int v) { return (int64_t)load_index(vec_index(v, tpr, p.lt), nvec) * VEC; };
#pragma unroll
  for (int v = 0; v < NV; ++v) wv[v] = ldf<F, S, VEC>(w + lj_of(v));
  shared_loads_first();
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    xv[v] = ldf_nt<F, S, VEC>(x + lbase + lj_of(v));
    if constexpr (RES) rv[v] = ldf_nt<F, S, VEC>(res + lbase + lj_of(v));
  }
  float a[NV][VEC];
  double ss = 0.0;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int j = vec_index(v, tpr, p.lt);
    double vs = 0.0;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      float t = E::to_f(xv[v].v[e]);
      if constexpr (RES) t += E::to_f(rv[v].v[e]);
      a[v][e] = t;
      vs = __builtin_fma((double)t, (double)t, vs);
    }
    ss += j < nvec ? vs : 0.0;
    if constexpr (RES) {
      if (p.live && j < nvec) {
        Pack<S, VEC> o;
#pragma unroll
        for (int e = 0; e < VEC; ++e) o.v[e] = E::from_f(a[v][e]);
        stf_nt<F, S, VEC>(after + base + (int64_t)j * VEC, o);
      }
    }
  }
  ss = row_reduce<false, (NV < 8)>(ss, red_sum, tpr, SumOp());
  const float rho = row_inv_rms(ss, hidden, eps);
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int j = vec_index(v, tpr, p.lt);
    norm_weigh<E, VEC, true>(a[v], rho, wv[v]);
    // blocks are whole, so their lanes are all inside the row or all past its end
    const uint32_t e = mx_scale(lanes_max(absmax_bits<VEC>(a[v]), kMxBlock / VEC));
    if (p.live && j < nvec) store_block<VEC>(out, scales, base + (int64_t)j * VEC, a[v], e);
  }
}

// Rows too wide for the registers: one 1024-lane workgroup a row, which reads it twice (the second
// time from the caches for all but the widest), storing after_res in the second pass, by the lane that
// reads it.
template <class E, bool RES, bool LOOSE>
__global__ void __launch_bounds__(kWideLanes)
k_rms_norm_mxfp4_wide(uint8_t* __restrict__ out, uint8_t* __restrict__ scales,
                      const typename E::S* x, const typename E::S* __restrict__ w,
                      const typename E::S* res, typename E::S* after, int hidden, float eps) {
  using S = typename E::S;
  constexpr int VEC = E::VEC, F = LOOSE ? FORM_RAGGED : FORM_ROWS;
  __shared__ double red_sum[16];
  const int nvec = hidden / VEC;
  const int64_t base = (int64_t)blockIdx.x * hidden;
  auto a_of = [&](int j, float* a) {
    widen<E, VEC>(a, ldf<F, S, VEC>(x + base + (int64_t)j * VEC));
    if constexpr (RES) {
      float r[VEC];
      widen<E, VEC>(r, ldf<F, S, VEC>(res + base + (int64_t)j * VEC));
#pragma unroll
      for (int e = 0; e < VEC; ++e) a[e] += r[e];
    }
  };
  double ss = 0.0;
#pragma unroll 4
  for (int j = threadIdx.x; j < nvec; j += kWideLanes) {
    float a[VEC];
    a_of(j, a);
#pragma unroll
    for (int e = 0; e < VEC; ++e) ss = __builtin_fma((double)a[e], (double)a[e], ss);
  }
  ss = row_reduce(ss, red_sum, kWideLanes, SumOp());
  const float rho = row_inv_rms(ss, hidden, eps);
  // nvec is a multiple of a block's lanes, so the lanes of a block leave the loop together
  for (int j = threadIdx.x; j < nvec; j += kWideLanes) {
    float a[VEC];
    a_of(j, a);
    const int64_t at = base + (int64_t)j * VEC;
    if constexpr (RES) {
      Pack<S, VEC> o;
#pragma unroll
      for (int e = 0; e < VEC; ++e) o.v[e] = E::from_f(a[e]);
      stf_nt<F, S, VEC>(after + at, o);
    }
    norm_weigh<E, VEC, true>(a, rho, ldf<F, S, VEC>(w + (int64_t)j * VEC));
    const uint32_t e = mx_scale(lanes_max(absmax_bits<VEC>(a), kMxBlock / VEC));
    store_block<VEC>(out, scales, at, a, e);
  }
}

struct NmArgs {
  uint8_t* out;
  uint8_t* scales;
  const void* x;
  const void* w;
  const void* res;
  void* after;
  int64_t rows;
  int hidden;
  float eps;
};

template <class E, bool RES, bool LOOSE>
static const void* norm_kernel_of(int nv) {
  switch (nv) {
    case 1: return reinterpret_cast<const void*>(&k_rms_norm_mxfp4<E, 1, RES, LOOSE>);
    case 2: return reinterpret_cast<const void*>(&k_rms_norm_mxfp4<E, 2, RES, LOOSE>);
    case 4: return reinterpret_cast<const void*>(&k_rms_norm_mxfp4<E, 4, RES, LOOSE>);
    case 8: return reinterpret_cast<const void*>(&k_rms_norm_mxfp4<E, 8, RES, LOOSE>);
    default: return nullptr;
  }
}

template <class E, bool RES, bool LOOSE>
static int norm_quant(const NmArgs& a, hipStream_t st) {
  using S = typename E::S;
  const char* name = "rms_norm_mxfp4_quant";
  const S* x = static_cast<const S*>(a.x);
  const S* w = static_cast<const S*>(a.w);
  const S* r = static_cast<const S*>(a.res);
  S* after = static_cast<S*>(a.after);
  const KernelOfNv kernels = &norm_kernel_of<E, RES, LOOSE>;
  if (!row_fits(a.hidden, E::VEC, kernels, 64)) {
    if (!wide_rows_ok(name, a.rows)) return MCOP_E_UNSUPPORTED;
    hipLaunchKernelGGL((k_rms_norm_mxfp4_wide<E, RES, LOOSE>), dim3((unsigned)a.rows),
                       dim3(kWideLanes), 0, st, a.out, a.scales, x, w, r, after, a.hidden, a.eps);
    return check_launch(name);
  }
  Geometry g;
  // whole waves a row: a block's lanes must lie inside one row
  if (!choose_geometry(name, a.rows, a.hidden, E::VEC, kernels, &g, 64)) return MCOP_E_UNSUPPORTED;
  const dim3 grid((unsigned)g.blocks), block((unsigned)(g.tpr * g.rpb));
#define MCOP_LAUNCH(NVV)                                                                       \
  hipLaunchKernelGGL((k_rms_norm_mxfp4<E, NVV, RES, LOOSE>), grid, block, 0, st, a.out, a.scales, \
                     x, w, r, after, a.rows, a.hidden, g.tpr, a.eps)
  switch (g.nv) {
    case 1: MCOP_LAUNCH(1); break;
    case 2: MCOP_LAUNCH(2); break;
    case 4: MCOP_LAUNCH(4); break;
    default: MCOP_LAUNCH(8); break;
  }
#undef MCOP_LAUNCH
  return check_launch(name);
}

template <class E>
static int norm_quant(const NmArgs& a, hipStream_t st) {
  const bool whole = aligned(16, a.x, a.w, a.res, a.after);
  if (a.res != nullptr) return whole ? norm_quant<E, true, false>(a, st)
                                     : norm_quant<E, true, true>(a, st);
  return whole ? norm_quant<E, false, false>(a, st) : norm_quant<E, false, true>(a, st);
}

}  // namespace mcop

extern "C" int mcop_rms_norm_mxfp4_quant(uint8_t* out, uint8_t* scales, const void* input,
                                         const void* weight, const void* residual,
                                         void* after_res, int64_t num_tokens,
                                         int64_t hidden_size, mcop_dtype in_dtype, float epsilon,
                                         void* stream) {
  using namespace mcop;
  const char* name = "rms_norm_mxfp4_quant";
  if (num_tokens < 0 || hidden_size <= 0 || hidden_size > INT32_MAX) {
    return set_error(MCOP_E_INVALID, "%s: bad shape num_tokens=%lld hidden_size=%lld", name,
                     (long long)num_tokens, (long long)hidden_size);
  }
  if (hidden_size % kMxBlock != 0) {
    return set_error(MCOP_E_INVALID, "%s: hidden_size %lld is not a multiple of the block of 32",
                     name, (long long)hidden_size);
  }
  if (num_tokens == 0) return MCOP_OK;
  if (!out || !scales || !input || !weight) {
    return set_error(MCOP_E_INVALID, "%s: null pointer", name);
  }
  if ((residual == nullptr) != (after_res == nullptr)) {
    return set_error(MCOP_E_INVALID, "%s: residual and after_res go together", name);
  }
  if (!aligned(4, out)) {
    return set_error(MCOP_E_INVALID, "%s: out must be aligned to 4 bytes", name);
  }
  const NmArgs a{out, scales, input, weight, residual, after_res, num_tokens, (int)hidden_size,
                 epsilon};
  auto st = static_cast<hipStream_t>(stream);
  switch (in_dtype) {
    case MCOP_BF16: return norm_quant<BF16>(a, st);
    case MCOP_F16: return norm_quant<F16>(a, st);
    case MCOP_F32: return norm_quant<F32>(a, st);
    default:
      return set_error(MCOP_E_INVALID, "%s: input dtype %d is not bf16/fp16/fp32", name,
                       (int)in_dtype);
  }
}
