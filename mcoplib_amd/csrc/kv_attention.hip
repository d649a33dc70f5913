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
// product is a sum over the wave.  For head sizes that the matrix kernels are not built for; where they are, they
// are two to twenty times as fast (37 ragged sequences of 5 x 80 and 96 int8 to fp32: 25 us, 199 so; 64 of
// 8 x 128 int8: 66 and 1468; one of 1000 positions: 11 and 23).  A position's sums over the wave bound it.
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
    // the end of the last tile of 2^31 - 1 positions, and the position after a wave's last, are no ints
    const uint32_t from = (uint32_t)max(c.first, c.tile * kAttTile);
    const uint32_t to = min((uint32_t)c.end, (uint32_t)(c.tile + c.tiles) * kAttTile);
    bool missing = false;
    int unit = FMT == KV_MXFP4 ? 0 : kAttNoUnit;
    for (uint32_t p = from + wave; p < to; p += kAttWaves) {
      uint32_t off;
      const int page = att_page(a, c.sequence, p, &off);
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
      bool far = false;  // of the lane's 4-bit values
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
            const uint32_t byte = static_cast<const uint8_t*>(a.value.scales)[vs + (d >> 5)];
            vf[n] *= mx_value(byte);
            far = far || byte >= kMxFarByte;
          }
        }
      }
      float k_scale = a.scale, v_scale = 1.0f;
      int e = FMT == KV_MXFP4 && __builtin_amdgcn_ballot_w64(far) != 0 ? kMxUnit : unit;
      if constexpr (FMT != KV_MXFP4) {
        k_scale *= static_cast<const float*>(a.key.scales)[ks];
        v_scale = static_cast<const float*>(a.value.scales)[vs];
        e = att_unit(v_scale);
      }
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

// Joins the parts of split sequence blockIdx.y of the plan, a query head in WAVES waves, each with every
// WAVES-th part.  Lane i knows maximum, sum and unit of part i, all of a wave's at once, and what its weights
// become; then the parts' elements are added up, four a lane and of kJoinBatch parts on their way together
// (vectors of up to 128 elements: each half of the wave every second part).  The code is kept short: it is
// fetched from memory after a kernel whose reads have passed through the whole L2 (64 sequences' 128 cuts of 64
// query heads: 5.3 us; a workgroup a head with more code 7.0).
constexpr int kJoinWaves = 4, kJoinBatch = 4;  // waves of a workgroup; parts that a wave has on their way

template <class E, int WAVES>
__global__ void __launch_bounds__(kJoinWaves * 64)
k_kv_attention_join(AttArgs a) {
  // all of the plan at once, also where it says that there is no such entry
  const int32_t* plan = a.plan + 2 + 3 * blockIdx.y;
  const int splits = a.plan[0], sequence = plan[0];
  const uint32_t per = (uint32_t)a.plan[1], begin = (uint32_t)plan[1], end = (uint32_t)plan[2];
  if ((int)blockIdx.y >= splits) return;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = (int)threadIdx.x & 63;
  const int head = (int)blockIdx.x * (kJoinWaves / WAVES) + (WAVES == 1 ? wave : 0);
  if (WAVES == 1 && head >= a.query_heads) return;
  const int share = (int)(begin / per), count = (int)((end - 1) / per) - share + 1, dim = a.value.dim;
  // the first share's part is its second one where the share begins with another sequence
  const int shift = begin > (uint32_t)share * per ? 1 : 0;
  auto row_of = [&](int i) {
    return (int64_t)(2 * (share + i) + (i == 0 ? shift : 0)) * a.query_heads + head;
  };
  auto larger = [](float x, float y) { return __builtin_fmaxf(x, y); };
  auto sum_of = [](float x, float y) { return x + y; };
  const int by = WAVES == 1 ? 1 : WAVES, from = WAVES == 1 ? 0 : wave;
  const int mine = (count - from + by - 1) / by;  // parts from, from + by, ...
  const bool halves = dim <= 128;
  const int step = halves ? 2 : 1, half = halves ? lane >> 5 : 0;
  for (int d0 = 0; d0 < dim; d0 += 256) {
    // the last four overlap those before them where there are not four more; of less than four the rest is
    // what lies behind them in the workspace, and is not written
    const int d = min(d0 + (halves ? lane & 31 : lane) * 4, max(dim - 4, 0));
    float m = -__builtin_inff(), l = 0.0f, unit = -252.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int j0 = 0; j0 < mine; j0 += 64) {
      const bool is = j0 + lane < mine;
      const Pack<float, 4> s = ld<float, 4>(a.sums + row_of(from + by * min(j0 + lane, mine - 1)) * 4);
      const float mi = is ? s.v[0] : -__builtin_inff(), ui = is ? s.v[2] : -252.0f;
      const float top = larger(m, wave_reduce(mi, larger)), high = larger(unit, wave_reduce(ui, larger));
      const float keep = att_weight(m, top), w = att_weight(mi, top);
      l = l * keep + wave_reduce(is ? s.v[1] * w : 0.0f, sum_of);
      const float keep_o = keep * att_power((int)(unit - high));
      const float f = is ? w * att_power((int)(ui - high)) : 0.0f;
      m = top, unit = high;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] *= keep_o;
      const int n = min(mine - j0, 64);
      for (int j = 0; j < n; j += kJoinBatch * step) {
        Pack<float, 4> v[kJoinBatch];
        float g[kJoinBatch];
#pragma unroll
        for (int b = 0; b < kJoinBatch; ++b) {
          const int x = j + b * step + half;
          const float* src = a.parts + row_of(from + by * (j0 + min(x, n - 1))) * dim + d;
          __builtin_memcpy(v[b].v, src, sizeof(v[b].v));
          g[b] = from_lane_f(f, x & 63);
          // behind the last: that one once more, without weight
          if (x >= n) g[b] = 0.0f, v[b] = {};
        }
#pragma unroll
        for (int b = 0; b < kJoinBatch; ++b) {
#pragma unroll
          for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(v[b].v[e], g[b], o[e]);
        }
      }
    }
    if (halves) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float x, y;
        swap_halves(o[e], &x, &y);
        o[e] = x + y;
      }
    }
    if constexpr (WAVES > 1) {
      __shared__ float sums[WAVES][3];
      __shared__ Pack<float, 4> os[WAVES][64];
      if (lane == 0) sums[wave][0] = m, sums[wave][1] = l, sums[wave][2] = unit;
      os[wave][lane] = Pack<float, 4>{o[0], o[1], o[2], o[3]};
      __syncthreads();
      m = -__builtin_inff(), unit = -252.0f, l = 0.0f;
#pragma unroll
      for (int i = 0; i < WAVES; ++i) m = larger(m, sums[i][0]), unit = larger(unit, sums[i][2]);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = 0.0f;
#pragma unroll
      for (int i = 0; i < WAVES; ++i) {
        const float w = att_weight(sums[i][0], m), f = w * att_power((int)(sums[i][2] - unit));
        l += sums[i][1] * w;
        const Pack<float, 4> v = os[i][lane];
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] += v.v[e] * f;
      }
      __syncthreads();
      if (wave > 0) continue;
    }
    typename E::S* out = static_cast<typename E::S*>(a.value.plain) + sequence * a.value.p_token +
                         head * a.value.p_head + d;
    const float part = l == 0.0f ? 0.0f : 1.0f / l;
    if (half == 0) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (e < dim) out[e] = E::from_f(__builtin_ldexpf(o[e] * part, (int)unit));
      }
    }
    if (a.lse != nullptr && d0 == 0 && lane == 0) {
      a.lse[(int64_t)sequence * a.query_heads + head] = att_lse(m, l);
    }
  }
}

// ---------------------------------------------------------------------------------------------
// Host side.

namespace {

// Shares: waves for the card over all of a share's key heads and blocks of sixteen query heads.  Codes
// through LDS: four waves a CU, which have two tiles each in flight (2 x 131072 positions of 8 x 128 fp8: 109
// us, 115 with eight waves and twice the parts; 48 windows of 1024 of 4 x 256: 35 and 50); else eight (37
// ragged sequences of 5 x 80 and 96 int8 to fp32: 29 us with four, 25 so), while two workgroups are resident (83
// of 12338 in all, 7 x 129 fp8 to fp32, one workgroup a CU: 36 us with four waves a CU, 48 with eight).
constexpr int kLineShares = 1024, kAttShares = 2048;
int64_t target_of(int64_t shares, int64_t heads, int64_t group) {
  const int64_t n = shares / (heads * ((group + 15) / 16));
  // the same for every die: 68 shares of 15 heads would be 34 workgroups for some dies' 32 CUs
  return n >= 8 ? n / 8 * 8 : std::max<int64_t>(1, n);
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

// Codes through LDS with eight waves a CU: where two workgroups are resident, and either tiles are small (64
// sequences of 4000 of 8 x 64 fp8: 58 us, 71 with four; of 2000 of 8 x 128 4-bit, tiles of 5 KiB: 42 and 49) or
// shares have two sequences or more each, whose starts overlap then while few are cut (1024 of 128 of 8 x 128
// fp8: 64 us and 74; 512 of 100 int8: 37 and 43; 200 of 333 fp8, 1.6 a share, the same; 150 of 600, 1.2 a share,
// 44 and 42).  Keys of 192 and values of 128, 4-bit, tiles of 7.5 KiB: 52 and 53.
constexpr int kSmallTile = 6 * 1024;
template <class E, int FMT, int I = 0>
bool eight_waves(int shape, bool many) {
  if (shape == I) return kTwoResident<E, FMT, I> && (many || kTileBytes<FMT, I> <= kSmallTile);
  if constexpr (I < 3) return eight_waves<E, FMT, I + 1>(shape, many);
  return false;
}

template <class E, int FMT>
int launch_of(const char* name, AttArgs a, mcop_dtype dtype, hipStream_t st) {
  const int shape = tile_shape(a), rows = shape >= 0 ? kTileRows : kAttRows;
  const bool lines = shape >= 0 && whole_lines(a, FMT);
  a.target = (int)target_of(kAttShares, a.heads, a.group);
  if (shape >= 0) {
    const int four = (int)target_of(kLineShares, a.heads, a.group);
    if (lines ? !eight_waves<E, FMT>(shape, a.sequences >= 2 * four) : kTileShapes[shape].vd == 16) {
      a.target = four;
    }
  }
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
  // each cut between two shares splits one sequence; a query head in one wave while an even split has fewer
  // parts than two of its batches (a call over 64 sequences, two parts each: 66 us, 70 with four waves; over
  // 48 windows, five: 35 and 37; 37 ragged sequences with eleven: 25, 27 with one wave)
  const dim3 lanes(kJoinWaves * 64);
  const unsigned splits = (unsigned)std::min(a.sequences, a.target - 1);
  if (a.target / a.sequences < 2 * kJoinBatch) {
    const dim3 grid((unsigned)((a.query_heads + kJoinWaves - 1) / kJoinWaves), splits);
    hipLaunchKernelGGL((k_kv_attention_join<E, 1>), grid, lanes, 0, st, a);
  } else {
    hipLaunchKernelGGL((k_kv_attention_join<E, kJoinWaves>), dim3((unsigned)a.query_heads, splits), lanes, 0,
                       st, a);
  }
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
  if ((capacity / kAttTile + 2 + kAttStart) * num_sequences > INT32_MAX) {
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
