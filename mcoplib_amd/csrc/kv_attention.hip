// kv_attention.hip -- attention of one new token a sequence over the quantized paged cache: the kernel of
// vector arithmetic, the join of split sequences, and the C entry points (kv_attention.h has the mathematics
// and the split).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../../include/mcop_norm.h"
#include "kv_attention_tiles.h"
#include "launch_trace.h"

namespace mcop {

constexpr int kAttRows = 4;  // query heads of a workgroup of the kernel below

// One code's value without its scale (element d of a vector).
template <int FMT>
__device__ __forceinline__ float code_value(const uint8_t* v, int d) {
  if constexpr (FMT == KV_INT8) {
    return (float)(int8_t)v[d];
  } else if constexpr (FMT == KV_FP8) {
    return __builtin_amdgcn_cvt_pk_f32_fp8((int)v[d], false)[0];
  } else {
    return __builtin_amdgcn_cvt_scalef32_pk_f32_fp4((uint32_t)v[d >> 1] >> ((d & 1) * 4), 1.0f, 0)[0];
  }
}

// Joins the waves' parts of `rows` query heads from LDS (m, l [kAttWaves][kAttRows], e [kAttWaves], o
// [kAttWaves][kAttRows][value.dim]) and writes the outputs of query heads head0.. (or, of a split sequence,
// its part).
template <class E>
__device__ __forceinline__ void att_write(const AttArgs& a, const AttChunk& c, int head0, int rows,
                                          const float* m, const float* l, const int* e,
                                          const float* o) {
  int unit = e[0];
#pragma unroll
  for (int w = 1; w < kAttWaves; ++w) unit = max(unit, e[w]);
  for (int r = 0; r < rows; ++r) {
    float top = -__builtin_inff();
#pragma unroll
    for (int w = 0; w < kAttWaves; ++w) top = __builtin_fmaxf(top, m[w * kAttRows + r]);
    float f[kAttWaves], sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kAttWaves; ++w) {
      f[w] = att_weight(m[w * kAttRows + r], top);
      sum += l[w * kAttRows + r] * f[w];
      f[w] *= att_power(e[w] - unit);
    }
    if (c.missing) sum = __builtin_nanf("");
    const int head = head0 + r;
    for (int d = (int)threadIdx.x; d < a.value.dim; d += kAttWaves * 64) {
      float v = 0.0f;
#pragma unroll
      for (int w = 0; w < kAttWaves; ++w) v += o[(w * kAttRows + r) * a.value.dim + d] * f[w];
      if (c.part >= 0) {
        a.parts[((int64_t)c.part * a.query_heads + head) * a.value.dim + d] = v;
      } else {
        static_cast<typename E::S*>(a.value.plain)[c.sequence * a.value.p_token +
                                                   head * a.value.p_head + d] =
            E::from_f(att_value(v, sum, unit));
      }
    }
    if (threadIdx.x == 0) {
      if (c.part >= 0) {
        float* s = a.sums + ((int64_t)c.part * a.query_heads + head) * 4;
        s[0] = top, s[1] = sum, s[2] = (float)unit;
      } else if (a.lse != nullptr) {
        a.lse[(int64_t)c.sequence * a.query_heads + head] = att_lse(top, sum);
      }
    }
  }
}

// The page of position p, or -1.
__device__ __forceinline__ int att_page(const AttArgs& a, int sequence, uint32_t p, uint32_t* off) {
  const uint32_t column = a.by_page.quotient(p);
  *off = p - column * (uint32_t)a.page_size;
  if (column >= (uint32_t)a.columns) return -1;
  const int g = a.table[sequence * a.table_stride + column];
  return g < 0 || g >= a.pages ? -1 : g;
}

// Vector arithmetic: a wave walks every fourth position, its lanes the elements, and every query head's
// product is a sum over the wave.  For head sizes that the matrix kernels are not built for.
template <class E, int FMT, int N>
__global__ void __launch_bounds__(kAttWaves * 64)
k_kv_attention_rows(AttArgs a) {
  extern __shared__ float lds[];  // m, l [waves][rows], e [waves], o [waves][rows][value.dim]
  const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
  uint32_t share;
  int head, block;
  att_place(a, blockIdx.x >> 3, &share, &head, &block);
  const int head0 = head * a.group + block * kAttRows;
  const int rows = min(kAttRows, a.group - block * kAttRows);
  AttWalk walk(a, share, head == 0 && block == 0 && wave == 0);
  AttChunk c;
  while (walk.next(&c)) {
    float q[kAttRows][N], o[kAttRows][N], m[kAttRows], l[kAttRows];
#pragma unroll
    for (int r = 0; r < kAttRows; ++r) {
      const typename E::S* src = static_cast<const typename E::S*>(a.key.plain) +
                                 c.sequence * a.key.p_token + (head0 + min(r, rows - 1)) * a.key.p_head;
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const int d = lane + n * 64;
        q[r][n] = d < a.key.dim ? E::to_f(src[d]) : 0.0f;
        o[r][n] = 0.0f;
      }
      m[r] = -__builtin_inff(), l[r] = 0.0f;
    }
    const int from = max(c.first, c.tile * kAttTile), to = min(c.end, (c.tile + c.tiles) * kAttTile);
    bool missing = false;
    int unit = FMT == KV_MXFP4 ? 0 : kAttNoUnit;
    for (int p = from + wave; p < to; p += kAttWaves) {
      uint32_t off;
      const int page = att_page(a, c.sequence, (uint32_t)p, &off);
      if (page < 0) {
        missing = true;
        continue;
      }
      const uint8_t* k = a.key.codes + page * a.key.c_page + off * a.key.c_token + head * a.key.c_head;
      const uint8_t* v =
          a.value.codes + page * a.value.c_page + off * a.value.c_token + head * a.value.c_head;
      const int64_t ks = page * a.key.s_page + off * a.key.s_token + head * a.key.s_head;
      const int64_t vs = page * a.value.s_page + off * a.value.s_token + head * a.value.s_head;
      float kf[N], vf[N];
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const int d = lane + n * 64;
        kf[n] = vf[n] = 0.0f;
        if (d < a.key.dim) {
          kf[n] = code_value<FMT>(k, d);
          if constexpr (FMT == KV_MXFP4) {
            kf[n] *= mx_value(static_cast<const uint8_t*>(a.key.scales)[ks + (d >> 5)]);
          }
        }
        if (d < a.value.dim) {
          vf[n] = code_value<FMT>(v, d);
          if constexpr (FMT == KV_MXFP4) {
            vf[n] *= mx_value(static_cast<const uint8_t*>(a.value.scales)[vs + (d >> 5)]);
          }
        }
      }
      float k_scale = a.scale, v_scale = 1.0f;
      if constexpr (FMT != KV_MXFP4) {
        k_scale *= static_cast<const float*>(a.key.scales)[ks];
        v_scale = static_cast<const float*>(a.value.scales)[vs];
        const int e = att_unit(v_scale);
        if (e > unit) {
          const float down = att_power(unit - e);
#pragma unroll
          for (int r = 0; r < kAttRows; ++r) {
#pragma unroll
            for (int n = 0; n < N; ++n) o[r][n] *= down;
          }
          unit = e;
        }
        v_scale = __builtin_ldexpf(v_scale, -unit);
      }
#pragma unroll
      for (int r = 0; r < kAttRows; ++r) {
        float s = 0.0f;
#pragma unroll
        for (int n = 0; n < N; ++n) s = __builtin_fmaf(q[r][n], kf[n], s);
#pragma unroll
        for (int x = 1; x < 64; x *= 2) s += __shfl_xor(s, x, 64);
        s *= k_scale;
        const float top = __builtin_fmaxf(m[r], s);
        const float keep = att_weight(m[r], top), w = att_weight(s, top);
        m[r] = top;
        l[r] = l[r] * keep + w;
#pragma unroll
        for (int n = 0; n < N; ++n) o[r][n] = o[r][n] * keep + (w * v_scale) * vf[n];
      }
    }
    float *ms = lds, *ls = ms + kAttWaves * kAttRows;
    int* es = reinterpret_cast<int*>(ls + kAttWaves * kAttRows);
    float* os = reinterpret_cast<float*>(es + kAttWaves);
    if (lane == 0) es[wave] = unit;
#pragma unroll
    for (int r = 0; r < kAttRows; ++r) {
      if (lane == 0) {
        ms[wave * kAttRows + r] = m[r];
        ls[wave * kAttRows + r] = missing ? __builtin_nanf("") : l[r];
      }
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const int d = lane + n * 64;
        if (d < a.value.dim) os[(wave * kAttRows + r) * a.value.dim + d] = o[r][n];
      }
    }
    __syncthreads();
    att_write<E>(a, c, head0, rows, ms, ls, es, os);
    __syncthreads();  // LDS is free again
  }
}

// Joins the parts of split sequence blockIdx.y of the plan, a query head a workgroup: a group of 32 lanes
// takes every eighth part, four elements a lane, with maximum and sum of its own, and the groups are
// joined in LDS.
constexpr int kJoinLanes = 32, kJoinGroups = 8;

template <class E>
__global__ void __launch_bounds__(kJoinLanes * kJoinGroups)
k_kv_attention_join(AttArgs a) {
  __shared__ float ms[kJoinGroups], ls[kJoinGroups], os[kJoinGroups][kJoinLanes * 4];
  __shared__ int es[kJoinGroups];
  // all of the plan at once, also where it says that there is no such entry
  const int32_t* plan = a.plan + 2 + 3 * blockIdx.y;
  const int splits = a.plan[0], sequence = plan[0];
  const uint32_t per = (uint32_t)a.plan[1], begin = (uint32_t)plan[1], end = (uint32_t)plan[2];
  if ((int)blockIdx.y >= splits) return;
  const int share = (int)(begin / per), count = (int)((end - 1) / per) - share + 1;
  const int head = (int)blockIdx.x, lane = (int)threadIdx.x & (kJoinLanes - 1),
            g = (int)threadIdx.x / kJoinLanes, dim = a.value.dim;
  typename E::S* out = static_cast<typename E::S*>(a.value.plain) + sequence * a.value.p_token +
                       head * a.value.p_head;
  for (int d0 = 0; d0 < dim; d0 += kJoinLanes * 4) {
    // the last four overlap those before them where there are not four more
    const int d = min(d0 + lane * 4, max(dim - 4, 0));
    float m = -__builtin_inff(), l = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    int unit = -252;  // below any part's
#pragma unroll 4
    for (int i = g; i < count; i += kJoinGroups) {
      // the first share's part is its second one where the share begins with another sequence
      const int part = 2 * (share + i) + (i == 0 && begin > (uint32_t)share * per ? 1 : 0);
      const int64_t row = (int64_t)part * a.query_heads + head;
      const Pack<float, 4> s = ld<float, 4>(a.sums + row * 4);
      const float mi = s.v[0], li = s.v[1];
      const int ei = (int)s.v[2];
      const float* src = a.parts + row * dim;
      float v[4];
      if (dim >= 4) {
        __builtin_memcpy(v, src + d, sizeof(v));
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = src[min(e, dim - 1)];
      }
      const float top = __builtin_fmaxf(m, mi);
      const float keep = att_weight(m, top), w = att_weight(mi, top);
      m = top;
      l = l * keep + li * w;
      const int high = max(unit, ei);
      const float keep_o = keep * att_power(unit - high), w_o = w * att_power(ei - high);
      unit = high;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = o[e] * keep_o + v[e] * w_o;
    }
    if (lane == 0) ms[g] = m, ls[g] = l, es[g] = unit;
#pragma unroll
    for (int e = 0; e < 4; ++e) os[g][lane * 4 + e] = o[e];
    __syncthreads();
    float top = -__builtin_inff(), sum = 0.0f;
    int high = -252;
#pragma unroll
    for (int i = 0; i < kJoinGroups; ++i) {
      top = __builtin_fmaxf(top, ms[i]);
      high = max(high, es[i]);
    }
    float f[kJoinGroups];
#pragma unroll
    for (int i = 0; i < kJoinGroups; ++i) {
      f[i] = att_weight(ms[i], top);
      sum += ls[i] * f[i];
      f[i] *= att_power(es[i] - high);
    }
    const int x = (int)threadIdx.x, at = min(d0 + (x & ~3), max(dim - 4, 0)) + (x & 3);
    if (x < kJoinLanes * 4 && d0 + (x & ~3) < dim && at < dim) {
      float v = 0.0f;
#pragma unroll
      for (int i = 0; i < kJoinGroups; ++i) v += os[i][x] * f[i];
      out[at] = E::from_f(att_value(v, sum, high));
    }
    if (a.lse != nullptr && d0 == 0 && threadIdx.x == 0) {
      a.lse[(int64_t)sequence * a.query_heads + head] = att_lse(top, sum);
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------------------------
// Host side.

namespace {

// Shares: waves for the card over all of a share's key heads and blocks of sixteen query heads.  Codes
// through LDS: four waves a CU, which have two tiles each in flight (2 x 131072 positions of 8 x 128 fp8: 111
// us, 116 with eight waves and twice the parts; 48 windows of 1024 of 4 x 256: 42 and 61); else eight (37
// ragged sequences of 5 x 80 and 96 int8 to fp32: 36 us with four, 30 so).
constexpr int kLineShares = 1024, kAttShares = 2048;
int64_t target_of(int64_t shares, int64_t heads, int64_t group) {
  return std::max<int64_t>(1, shares / (heads * ((group + 15) / 16)));
}

struct Workspace {
  int64_t parts, sums, plan;  // bytes
  int64_t bytes() const { return parts + sums + plan; }
};
Workspace workspace_of(int64_t target, int64_t query_heads, int64_t dim) {
  return {2 * target * query_heads * dim * 4, 2 * target * query_heads * 16, (2 + 3 * target) * 4};
}

bool heads_ok(int64_t heads, int64_t query_heads) {
  return heads > 0 && query_heads > 0 && query_heads <= 65535 && query_heads % heads == 0;
}

// The matrix kernel for the head sizes, an index of kTileShapes; -1: none (wider than they hold, or less
// than one of their units; nor do they take a cache without a page, which they read for any wrong one).
int tile_shape(const AttArgs& a) {
  if (a.pages == 0 || a.key.dim < 16) return -1;
  for (int i = 0; i < (int)(sizeof(kTileShapes) / sizeof(kTileShapes[0])); ++i) {
    const TileShape& s = kTileShapes[i];
    if (a.key.dim <= 64 * s.kp && a.value.dim <= 16 * s.vd) return a.value.dim >= s.vd ? i : -1;
  }
  return -1;
}

// Whether tiles can go through LDS: pages of whole halves of a tile, vectors of whole chunks of 16 bytes at
// multiples of 16, a half's positions apart by less than 2^31 bytes.
bool whole_lines(const AttArgs& a, int fmt) {
  for (const KvSide* k : {&a.key, &a.value}) {
    const int64_t bytes = fmt == KV_MXFP4 ? k->dim / 2 : k->dim;
    if (bytes % 16 != 0 || !aligned(16, k->codes) || k->c_page % 16 != 0 || k->c_token % 16 != 0 ||
        k->c_head % 16 != 0 || k->c_token >= ((int64_t)1 << 31) / 16 - 1024 ||
        k->s_token >= ((int64_t)1 << 31) / 64 - 16) {
      return false;
    }
  }
  return a.page_size % (kAttTile / 2) == 0;
}

template <class E, int FMT>
int launch_of(const char* name, AttArgs a, mcop_dtype dtype, hipStream_t st) {
  const int shape = tile_shape(a), rows = shape >= 0 ? kTileRows : kAttRows;
  const bool lines = shape >= 0 && whole_lines(a, FMT);
  a.target = (int)target_of(lines ? kLineShares : kAttShares, a.heads, a.group);
  const bool joins = a.target > 1;  // one share splits nothing
  a.row_blocks = (a.group + rows - 1) / rows;
  // shares of a die times their heads and blocks, a wave each of the matrix kernels, else a workgroup
  const int64_t inner = (int64_t)a.heads * a.row_blocks, workers = (int64_t)(a.target + 7) / 8 * inner;
  const int64_t blocks = 8 * (shape >= 0 ? (workers + kAttWaves - 1) / kAttWaves : workers);
  if (blocks >= ((int64_t)1 << 31) / 256) {
    return set_error(MCOP_E_UNSUPPORTED, "%s: more rows than one launch takes (%lld workgroups)", name,
                     (long long)blocks);
  }
  a.by_inner = Divisor((uint32_t)inner);
  a.by_blocks = Divisor((uint32_t)a.row_blocks);
  const int packed = FMT == KV_MXFP4 ? 32 : 16;
  a.k_chunks = Divisor((uint32_t)std::max(1, a.key.dim / packed));
  a.v_chunks = Divisor((uint32_t)std::max(1, a.value.dim / packed));
  // of the vector kernel: maximum, sum and outputs of each row, the outputs' unit
  const size_t lds = sizeof(float) * kAttWaves * (kAttRows * (2 + (size_t)a.value.dim) + 1);
  trace_launch(name, "sequences=%d heads=%d of %d head sizes %d and %d: %s kernel, wgs=%lld, %d "
               "shares%s", a.sequences, a.heads, a.query_heads, a.key.dim, a.value.dim,
               lines ? "matrix, through LDS," : shape >= 0 ? "matrix" : "vector", (long long)blocks,
               a.target, joins ? "" : ", none split");
  const dim3 grid((unsigned)blocks), block(kAttWaves * 64);
  if (shape >= 0) {
    int rc;
    if constexpr (FMT == KV_INT8) rc = attention_tiles_int8(shape, lines, dtype, a, grid, st);
    else if constexpr (FMT == KV_FP8) rc = attention_tiles_fp8(shape, lines, dtype, a, grid, st);
    else rc = attention_tiles_mxfp4(shape, lines, dtype, a, grid, st);
    if (rc) return rc;
  } else if (std::max(a.key.dim, a.value.dim) <= 256) {
    hipLaunchKernelGGL((k_kv_attention_rows<E, FMT, 4>), grid, block, lds, st, a);
  } else {
    hipLaunchKernelGGL((k_kv_attention_rows<E, FMT, 16>), grid, block, lds, st, a);
  }
  if (int rc = check_launch(name)) return rc;
  if (!joins) return MCOP_OK;
  // each cut between two shares splits one sequence
  const dim3 pairs((unsigned)a.query_heads, (unsigned)std::min(a.sequences, a.target - 1));
  hipLaunchKernelGGL((k_kv_attention_join<E>), pairs, dim3(kJoinLanes * kJoinGroups), 0, st, a);
  return check_launch(name);
}

}  // namespace

}  // namespace mcop

extern "C" int64_t mcop_kv_cache_attention_workspace(int64_t num_heads, int64_t query_heads,
                                                     int64_t value_head_size) {
  using namespace mcop;
  if (!heads_ok(num_heads, query_heads) || value_head_size <= 0 || value_head_size > kKvMostDim) {
    return set_error(MCOP_E_INVALID, "kv_cache_attention: bad shape num_heads=%lld query_heads=%lld "
                     "head_size=%lld", (long long)num_heads, (long long)query_heads,
                     (long long)value_head_size);
  }
  return workspace_of(target_of(kAttShares, num_heads, query_heads / num_heads), query_heads,
                      value_head_size).bytes();
}

extern "C" int mcop_kv_cache_attention(const mcop_kv_side* key, const mcop_kv_side* value,
                                       mcop_dtype cache_dtype, int64_t num_pages, int64_t page_size,
                                       int64_t num_heads, int64_t query_heads,
                                       const int32_t* block_table, int64_t table_row_stride,
                                       int64_t table_columns, const int32_t* seq_lens,
                                       int64_t num_sequences, float scale, int64_t window,
                                       mcop_dtype dtype, float* lse, void* workspace,
                                       int64_t workspace_bytes, void* stream) {
  using namespace mcop;
  const char* name = "kv_cache_attention";
  if (num_sequences == 0) return MCOP_OK;
  const int fmt = format_of(cache_dtype);
  if (fmt < 0) {
    return set_error(MCOP_E_INVALID, "%s: cache dtype %d is not int8, fp8_e4m3fn or mxfp4", name,
                     (int)cache_dtype);
  }
  if (dtype != MCOP_BF16 && dtype != MCOP_F16 && dtype != MCOP_F32) {
    return set_error(MCOP_E_INVALID, "%s: dtype %d is not bf16/fp16/fp32", name, (int)dtype);
  }
  if (!key || !value) return set_error(MCOP_E_INVALID, "%s: null pointer", name);
  if (!heads_ok(num_heads, query_heads)) {
    return set_error(MCOP_E_INVALID, "%s: %lld query heads (at most 65535) are not a multiple of %lld "
                     "key heads", name, (long long)query_heads, (long long)num_heads);
  }
  if (num_pages < 0 || page_size <= 0 || page_size > INT32_MAX || num_pages > INT32_MAX ||
      num_pages * page_size > INT32_MAX) {
    return set_error(MCOP_E_INVALID, "%s: bad shape num_pages=%lld page_size=%lld (at most 2^31 - 1 "
                     "slots)", name, (long long)num_pages, (long long)page_size);
  }
  if (num_sequences < 0 || num_sequences > (1 << 24) || table_columns < 0 ||
      table_columns > INT32_MAX || table_row_stride < 0 ||
      table_row_stride > INT64_MAX / 8 / num_sequences) {
    return set_error(MCOP_E_INVALID, "%s: bad block table: %lld sequences (at most 2^24) of %lld pages",
                     name, (long long)num_sequences, (long long)table_columns);
  }
  // the kernels count tiles in 32 bits; a sequence has as many as its row of the table holds
  const int64_t capacity = std::min<int64_t>(table_columns * page_size, INT32_MAX);
  if ((capacity / kAttTile + 2) * num_sequences > INT32_MAX) {
    return set_error(MCOP_E_UNSUPPORTED, "%s: %lld sequences of up to %lld positions are 2^31 tiles of 32 "
                     "or more", name, (long long)num_sequences, (long long)capacity);
  }
  if (window < 0) return set_error(MCOP_E_INVALID, "%s: negative window", name);
  AttArgs a;
  if (int rc = side_of(name, "key", *key, fmt, num_pages, page_size, query_heads, num_sequences,
                       &a.key)) {
    return rc;
  }
  if (int rc = side_of(name, "value", *value, fmt, num_pages, page_size, query_heads, num_sequences,
                       &a.value)) {
    return rc;
  }
  if (!seq_lens || (!block_table && table_columns > 0)) {
    return set_error(MCOP_E_INVALID, "%s: null pointer", name);
  }
  const int64_t target = target_of(kAttShares, num_heads, query_heads / num_heads);
  const Workspace ws = workspace_of(target, query_heads, a.value.dim);
  if (!workspace || !aligned(16, workspace) || workspace_bytes < ws.bytes()) {
    return set_error(MCOP_E_INVALID, "%s: the workspace must be %lld bytes at a multiple of 16", name,
                     (long long)ws.bytes());
  }
  a.lse = lse;
  a.table = block_table;
  a.table_stride = table_row_stride;
  a.columns = (int)table_columns;
  a.lens = seq_lens;
  a.sequences = (int)num_sequences;
  a.pages = num_pages;
  a.page_size = (int)page_size;
  a.by_page = Divisor((uint32_t)page_size);
  a.heads = (int)num_heads;
  a.query_heads = (int)query_heads;
  a.group = (int)(query_heads / num_heads);
  a.window = (int)std::min<int64_t>(window, INT32_MAX);
  a.scale = scale * kLog2e;
  a.parts = static_cast<float*>(workspace);
  a.sums = a.parts + ws.parts / 4;
  a.plan = reinterpret_cast<int32_t*>(a.sums + ws.sums / 4);
  auto st = static_cast<hipStream_t>(stream);
  auto by_format = [&](auto e) {
    using E = decltype(e);
    if (fmt == KV_INT8) return launch_of<E, KV_INT8>(name, a, dtype, st);
    if (fmt == KV_FP8) return launch_of<E, KV_FP8>(name, a, dtype, st);
    return launch_of<E, KV_MXFP4>(name, a, dtype, st);
  };
  if (dtype == MCOP_BF16) return by_format(BF16());
  if (dtype == MCOP_F16) return by_format(F16());
  return by_format(F32());
}
