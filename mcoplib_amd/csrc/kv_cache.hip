// kv_cache.hip -- keys and values quantized as they are written to a paged cache, and read back.
//
// A vector is one token's key (or value) of one head: D elements with a scale of their own, by the
// arithmetic of the framework's per-token quantizers (per_token_quant.hip) or as 4-bit blocks
// (mxfp4.h):
//   int8   s = A / 127,                    q = sat[-127,127](rne(x * (127 / A))), A = max|x|
//   fp8    s = max(A / 448, 1/(448*512)),  q = e4m3fn(clamp(x / s, +-448))
//   mxfp4  a scale byte and 32 codes a block
// and reads back as q * s in fp32 (exact for 4-bit blocks), rounded to the output's type.
//
// Both directions are bound by HBM (three bytes an element of a 16-bit type).  A vector takes the
// fewest lanes (a power of two) that hold it at eight elements a lane, so that a wave's loads are 1 KiB
// in a row where heads and tokens lie next to each other; its absmax is a few register moves.
// Workgroups of blockIdx.y = 0 do the keys, 1 the values.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdio>

#include "../../include/mcop_norm.h"
#include "kv_side.h"
#include "launch_trace.h"
#include "mxfp4.h"

namespace mcop {

constexpr int kKvLanes = 256;

struct KvSides {
  KvSide side[2];
  int heads;
  Divisor by_heads, by_page;
};

// The eight (or, past the vector's end, fewer) elements of a unit: not WHOLE, at any alignment where there
// are eight, else one by one (all of them so, 65536 tokens of 8 x 61 int8 read in 125 us, 88 so).
template <class E, bool WHOLE>
__device__ __forceinline__ Pack<typename E::S, 8> load_unit(const typename E::S* p, int n) {
  if constexpr (WHOLE) {
    return load8<typename E::S, false, false>(p);
  } else {
    if (n >= 8) return load8<typename E::S, true, false>(p);
    Pack<typename E::S, 8> v;
#pragma unroll
    for (int e = 0; e < 8; ++e) v.v[e] = e < n ? p[e] : typename E::S(0);
    return v;
  }
}
template <class T, bool WHOLE>
__device__ __forceinline__ void store_unit(T* p, const Pack<T, 8>& v, int n) {
  if constexpr (WHOLE) {
    if constexpr (sizeof(T) == 1) st_nt<T, 8>(p, v);
    else store8<T, false>(p, v);
  } else if (n >= 8) {
    __builtin_memcpy(p, &v, sizeof(v));
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (e < n) p[e] = v.v[e];
    }
  }
}
// A dword of codes, in bytes where the cache is not aligned to it.
template <bool WHOLE>
__device__ __forceinline__ void store_dword(uint8_t* p, uint32_t v) {
  if constexpr (WHOLE) *reinterpret_cast<uint32_t*>(p) = v;
  else __builtin_memcpy(p, &v, 4);
}
template <bool WHOLE>
__device__ __forceinline__ uint32_t load_dword(const uint8_t* p) {
  uint32_t v;
  if constexpr (WHOLE) v = *reinterpret_cast<const uint32_t*>(p);
  else __builtin_memcpy(&v, p, 4);
  return v;
}

// Quantizes one vector, whose `lanes` lanes hold NU units each (left[n]: elements of unit n inside the
// vector; a unit past its end holds copies of the first, or zeros), and stores codes and scales.
// WHOLE: vectors are whole units, and every tensor's vectors are aligned to theirs.
template <class E, int FMT, bool WHOLE, int NU>
__device__ __forceinline__ void write_vector(const Pack<typename E::S, 8> (&v)[NU],
                                             const int (&left)[NU], int j, int lanes, bool store,
                                             uint8_t* dst, void* scales, int64_t s_at) {
  if constexpr (FMT == KV_MXFP4) {
    uint8_t* sd = static_cast<uint8_t*>(scales) + s_at;
#pragma unroll
    for (int n = 0; n < NU; ++n) {
      const int unit = j + n * lanes;
      // vectors are whole blocks: a block's four lanes are all inside or all past the end
      const uint32_t e = mx_scale(lanes_max(absmax8<E>(v[n]), 4));
      if (!store || left[n] <= 0) continue;
      store_dword<WHOLE>(dst + unit * 4, mx_codes8<E>(v[n], e));
      if ((unit & 3) == 0) sd[unit >> 2] = (uint8_t)e;
    }
  } else {
    float A;
    bool ordinary;  // no NaN in the vector, and A where the short forms below hold
    if constexpr (sizeof(typename E::S) == 2) {
      // the largest magnitude by its bits, two values an instruction; NaN's are above infinity's
      uint32_t m = 0;
#pragma unroll
      for (int n = 0; n < NU; ++n) {
        const Pack<uint32_t, 4> w = __builtin_bit_cast(Pack<uint32_t, 4>, v[n]);
#pragma unroll
        for (int e = 0; e < 4; ++e) m = max_u16x2(m, w.v[e] & 0x7fff7fffu);
      }
      m = lanes_max(max(m & 0xffffu, m >> 16), lanes);
      A = E::to_f((uint16_t)m);
      ordinary = A <= 0x1p100f && (FMT == KV_FP8 || A >= 0x1p-100f);
    } else {
      ordinary = false;
    }
    float f[NU][8], s;
    Codes<8> q[NU];
#pragma unroll
    for (int n = 0; n < NU; ++n) widen<E, 8>(f[n], v[n]);
    if (sizeof(typename E::S) == 2 && __builtin_amdgcn_ballot_w64(!ordinary) == 0) {
      if constexpr (FMT == KV_INT8) {
        s = div_floored<127>(A);
        const float r = rcp_in_domain(A), h = 127.0f * r;  // 127 / A, as row_ratio
        const float inv = __builtin_fmaf(__builtin_fmaf(-h, A, 127.0f), r, h);
#pragma unroll
        for (int n = 0; n < NU; ++n) q[n] = i8_codes_in_range<8>(f[n], inv);
      } else {
        s = __builtin_fmaxf(div_floored<448>(A), 1.0f / 229376.0f);
        const float inv = rcp_in_domain(s);
        // fp8_quotient_codes' bounded form; without NaN its upper clamp gives the conversion's code
#pragma unroll
        for (int n = 0; n < NU; ++n) {
          float c[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float q0 = f[n][e] * inv;
            const float r = __builtin_fmaf(-q0, s, f[n][e]);
            c[e] = __builtin_copysignf(__builtin_fmaf(r, inv, q0), f[n][e]);
          }
          q[n] = cvt_fp8<8>(c);
        }
      }
    } else {
      float m = 0.0f;  // NaN is ignored, as in a row's absmax
#pragma unroll
      for (int n = 0; n < NU; ++n) {
#pragma unroll
        for (int e = 0; e < 8; ++e) m = __builtin_fmaxf(m, __builtin_fabsf(f[n][e]));
      }
      A = __builtin_bit_cast(float, lanes_max(__builtin_bit_cast(uint32_t, m), lanes));
      float inv;
      if constexpr (FMT == KV_INT8) {
        s = row_div<127>(A);
        inv = row_ratio(127.0f, A);
      } else {
        s = __builtin_fmaxf(div_floored<448>(A), 1.0f / 229376.0f);
        inv = row_rcp(s);
      }
#pragma unroll
      for (int n = 0; n < NU; ++n) {
        if constexpr (FMT == KV_INT8) q[n] = i8_codes<-127, 8>(f[n], inv);
        else q[n] = fp8_quotient_codes<8>(f[n], s, inv, mcop_divisor_ok(s), s <= 0x1p100f);
      }
    }
#pragma unroll
    for (int n = 0; n < NU; ++n) {
      if (store && left[n] > 0) {
        store_unit<uint8_t, WHOLE>(dst + (j + n * lanes) * 8,
                                   __builtin_bit_cast(Pack<uint8_t, 8>, q[n]), left[n]);
      }
    }
    if (store && j == 0) static_cast<float*>(scales)[s_at] = s;
  }
}

// Vectors of few lanes: a vector a group of lanes, wherever its token is.  NU: units a lane.
template <class E, int FMT, bool WHOLE, int NU>
__global__ void __launch_bounds__(kKvLanes)
k_kv_cache_write(KvSides a, const int64_t* __restrict__ slots, uint32_t vectors, int64_t num_slots,
                 int page_size) {
  using S = typename E::S;
  const KvSide& k = a.side[blockIdx.y];
  const int sh = 31 - __builtin_clz((unsigned)k.lanes);
  const uint32_t i = blockIdx.x * (uint32_t)(kKvLanes >> sh) + (threadIdx.x >> sh);
  const int j = (int)threadIdx.x & (k.lanes - 1);
  const bool live = i < vectors;
  const uint32_t token = a.by_heads.quotient(live ? i : vectors - 1);
  const uint32_t head = (live ? i : vectors - 1) - token * (uint32_t)a.heads;
  const S* src = static_cast<const S*>(k.plain) + token * k.p_token + head * k.p_head;
  Pack<S, 8> v[NU];
  int left[NU];  // elements of the unit inside the vector
#pragma unroll
  for (int n = 0; n < NU; ++n) {
    const int at = (j + n * k.lanes) * 8;
    left[n] = k.dim - at;
    if constexpr (WHOLE) {
      v[n] = load_unit<E, true>(src + (left[n] > 0 ? at : 0), 8);
    } else {
      v[n] = load_unit<E, false>(src + at, left[n]);
    }
  }
  const int64_t slot = slots[token];
  const bool store = live && slot >= 0 && slot < num_slots;
  const uint32_t page = a.by_page.quotient(store ? (uint32_t)slot : 0u);
  const uint32_t off = (store ? (uint32_t)slot : 0u) - page * (uint32_t)page_size;
  uint8_t* dst = k.codes + page * k.c_page + off * k.c_token + head * k.c_head;
  const int64_t s_at = page * k.s_page + off * k.s_token + head * k.s_head;
  write_vector<E, FMT, WHOLE, NU>(v, left, j, k.lanes, store, dst, k.scales, s_at);
}

// Tokens of a wave or more: a wave takes 64 / lanes heads of TW tokens, so that everything a token stands
// for (its slot, its page, their addresses) is computed in scalar registers; with a vector a group of
// lanes that arithmetic took longer than the memory.  The waves of a token are neighbours, so that what a
// token writes is written together (apart, by blockIdx.y, 65536 tokens of 8 x 128 read in 105 us, 89
// with the heads in a loop).
__device__ __forceinline__ int uniform_int(int v) { return __builtin_amdgcn_readfirstlane(v); }

template <class E, int FMT, bool WHOLE, int NU, int TW>
__global__ void __launch_bounds__(kKvLanes)
k_kv_cache_write_tokens(KvSides a, const int64_t* __restrict__ slots, int tokens, int64_t num_slots,
                        int page_size) {
  using S = typename E::S;
  const KvSide& k = a.side[blockIdx.y];
  const int sh = 31 - __builtin_clz((unsigned)k.lanes), lane = (int)threadIdx.x & 63;
  const int j = lane & (k.lanes - 1);
  const uint32_t item = (uint32_t)uniform_int(
      (int)(blockIdx.x * (kKvLanes / 64) + (threadIdx.x >> 6)));
  const int t0 = (int)k.by_passes.quotient(item) * TW;
  const int pass = (int)(item - k.by_passes.quotient(item) * k.by_passes.d);
  if (t0 >= tokens) return;
  int left[NU], at[NU];
#pragma unroll
  for (int n = 0; n < NU; ++n) {
    at[n] = (j + n * k.lanes) * 8;
    left[n] = k.dim - at[n];
    if (WHOLE && left[n] <= 0) at[n] = 0;
  }
  const int head = pass * (64 >> sh) + (lane >> sh);
  const bool live = head < a.heads;
  const int64_t h = live ? head : 0;
  Pack<S, 8> v[TW][NU];
#pragma unroll
  for (int i = 0; i < TW; ++i) {
    const S* src = static_cast<const S*>(k.plain) + min(t0 + i, tokens - 1) * k.p_token;
#pragma unroll
    for (int n = 0; n < NU; ++n) {
      v[i][n] = load_unit<E, WHOLE>(src + (h * k.p_head + at[n]), left[n]);
    }
  }
  // lane i looks for token i: one wait for all of them
  const int mine = min(t0 + (lane < TW ? lane : 0), tokens - 1);
  const int64_t slot = slots[mine];
  const bool in = slot >= 0 && slot < num_slots;
  const uint32_t my_page = a.by_page.quotient(in ? (uint32_t)slot : 0u);
  const uint32_t my_off = (in ? (uint32_t)slot : 0u) - my_page * (uint32_t)page_size;
  int64_t dst[TW], s_at[TW];
  bool store[TW];
#pragma unroll
  for (int i = 0; i < TW; ++i) {
    store[i] = t0 + i < tokens && __builtin_amdgcn_readlane((int)in, i) != 0;
    const uint32_t page = lane_value(my_page, i), off = lane_value(my_off, i);
    dst[i] = page * k.c_page + off * k.c_token;
    s_at[i] = page * k.s_page + off * k.s_token;
  }
#pragma unroll
  for (int i = 0; i < TW; ++i) {
    if (!store[i]) continue;
    write_vector<E, FMT, WHOLE, NU>(v[i], left, j, k.lanes, live, k.codes + dst[i] + h * k.c_head,
                                    k.scales, s_at[i] + h * k.s_head);
  }
}

// Four e4m3fn codes times s.
__device__ __forceinline__ void widen_fp8(float* f, uint32_t w, float s) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  const f2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
  const f2 b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  f[0] = a[0] * s, f[1] = a[1] * s, f[2] = b[0] * s, f[3] = b[1] * s;
}

// One unit of a vector as it lies in the cache, and its values.
template <int FMT>
struct KvUnit {
  Pack<uint8_t, 8> q;
  uint32_t c, e;
  float s;
};
template <int FMT, bool WHOLE>
__device__ __forceinline__ KvUnit<FMT> load_codes(const uint8_t* src, const void* scales,
                                                  int64_t s_at, int unit, int left) {
  KvUnit<FMT> u;
  if constexpr (FMT == KV_MXFP4) {
    u.c = load_dword<WHOLE>(src + unit * 4);
    u.e = static_cast<const uint8_t*>(scales)[s_at + (unit >> 2)];
  } else {
    if constexpr (WHOLE) {
      u.q = ld<uint8_t, 8>(src + unit * 8);
    } else if (left >= 8) {
      __builtin_memcpy(&u.q, src + unit * 8, 8);
    } else {
#pragma unroll
      for (int b = 0; b < 8; ++b) u.q.v[b] = b < left ? src[unit * 8 + b] : 0;
    }
    u.s = static_cast<const float*>(scales)[s_at];
  }
  return u;
}
template <class E, int FMT>
__device__ __forceinline__ Pack<typename E::S, 8> values_of(const KvUnit<FMT>& u, bool none) {
  float f[8];
  if constexpr (FMT == KV_MXFP4) {
    mx_widen8(f, u.c, u.e);
  } else if constexpr (FMT == KV_INT8) {
#pragma unroll
    for (int b = 0; b < 8; ++b) f[b] = (float)(int8_t)u.q.v[b] * u.s;
  } else {
    const Pack<uint32_t, 2> w = __builtin_bit_cast(Pack<uint32_t, 2>, u.q);
    widen_fp8(f, w.v[0], u.s);
    widen_fp8(f + 4, w.v[1], u.s);
  }
  Pack<typename E::S, 8> o;
#pragma unroll
  for (int b = 0; b < 8; ++b) o.v[b] = E::from_f(none ? __builtin_nanf("") : f[b]);
  return o;
}

// The sequence that holds token t: how many of cu[1..n] are <= t (the wave counts together).
__device__ __forceinline__ int sequence_of(const int32_t* __restrict__ cu, int n, int64_t t) {
  int s = 0;
  for (int i = 0; i < n; i += 64) {
    const int at = i + (int)(threadIdx.x & 63);
    const bool below = at < n && cu[at + 1] <= t;
    s += (int)__builtin_popcountll(__builtin_amdgcn_ballot_w64(below));
  }
  return s;
}

// Where a token of the gathered tensors lies: 1 in the cache (at page and off), 2 nowhere (no such page),
// 0 past the last sequence.  `s` is at most the token's sequence, and becomes it.
__device__ __forceinline__ int find_token(int64_t token, int& s, const int32_t* __restrict__ cu,
                                          const int32_t* __restrict__ starts, int sequences,
                                          const int32_t* __restrict__ table, int64_t table_stride,
                                          int columns, int64_t pages, int page_size,
                                          const Divisor& by_page, uint32_t* page, uint32_t* off) {
  *page = *off = 0;
  while (s < sequences && cu[s + 1] <= token) ++s;
  if (s >= sequences) return 0;
  const int64_t p = token - cu[s] + (starts != nullptr ? starts[s] : 0);
  if (p < 0 || p > INT32_MAX) return 2;
  const uint32_t column = by_page.quotient((uint32_t)p);
  if (column >= (uint32_t)columns) return 2;
  const int32_t g = table[s * table_stride + column];
  if (g < 0 || g >= pages) return 2;
  *page = (uint32_t)g;
  *off = (uint32_t)p - column * (uint32_t)page_size;
  return 1;
}

template <class E, int FMT, bool WHOLE, int NU, int R>
__global__ void __launch_bounds__(kKvLanes)
k_kv_cache_read(KvSides a, const int32_t* __restrict__ table, int64_t table_stride, int columns,
                const int32_t* __restrict__ cu, const int32_t* __restrict__ starts, int sequences,
                uint32_t vectors, int64_t pages, int page_size) {
  using S = typename E::S;
  const KvSide& k = a.side[blockIdx.y];
  const int sh = 31 - __builtin_clz((unsigned)k.lanes);
  const uint32_t per = kKvLanes >> sh;
  const uint32_t i0 = blockIdx.x * (per * R);
  if (i0 >= vectors) return;
  const int j = (int)threadIdx.x & (k.lanes - 1);
  const int s0 = sequence_of(cu, sequences, a.by_heads.quotient(i0));
  const uint8_t* src[R];
  int64_t s_at[R];
  S* dst[R];
  int state[R];  // 0: nothing to write, 1: a value, 2: no such page
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const uint32_t i = i0 + r * per + (threadIdx.x >> sh);
    const uint32_t token = a.by_heads.quotient(i < vectors ? i : vectors - 1);
    const uint32_t head = (i < vectors ? i : vectors - 1) - token * (uint32_t)a.heads;
    int s = s0;
    uint32_t page, off;
    dst[r] = static_cast<S*>(k.plain) + token * k.p_token + head * k.p_head;
    state[r] = i >= vectors ? 0
                            : find_token(token, s, cu, starts, sequences, table, table_stride, columns,
                                         pages, page_size, a.by_page, &page, &off);
    if (i >= vectors) page = off = 0;
    src[r] = k.codes + page * k.c_page + off * k.c_token + head * k.c_head;
    s_at[r] = page * k.s_page + off * k.s_token + head * k.s_head;
  }
#pragma unroll
  for (int n = 0; n < NU; ++n) {
    const int unit = j + n * k.lanes, at = unit * 8, left = k.dim - at;
    if (left <= 0) continue;
    KvUnit<FMT> u[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (state[r] == 1) u[r] = load_codes<FMT, WHOLE>(src[r], k.scales, s_at[r], unit, left);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (state[r] == 0) continue;
      store_unit<S, WHOLE>(dst[r] + at, values_of<E, FMT>(u[r], state[r] == 2), left);
    }
  }
}

// Tokens of a wave or more, as for the write: a wave takes whole tokens, and finds them in scalar
// registers (65536 tokens of 8 x 128 int8: 112 us with a vector a group of lanes, 75 so).
template <class E, int FMT, bool WHOLE, int NU, int TW>
__global__ void __launch_bounds__(kKvLanes)
k_kv_cache_read_tokens(KvSides a, const int32_t* __restrict__ table, int64_t table_stride,
                       int columns, const int32_t* __restrict__ cu,
                       const int32_t* __restrict__ starts, int sequences, int tokens, int64_t pages,
                       int page_size) {
  using S = typename E::S;
  const KvSide& k = a.side[blockIdx.y];
  const int sh = 31 - __builtin_clz((unsigned)k.lanes), lane = (int)threadIdx.x & 63;
  const int j = lane & (k.lanes - 1);
  const uint32_t item = (uint32_t)uniform_int(
      (int)(blockIdx.x * (kKvLanes / 64) + (threadIdx.x >> 6)));
  const int t0 = (int)k.by_passes.quotient(item) * TW;
  const int pass = (int)(item - k.by_passes.quotient(item) * k.by_passes.d);
  if (t0 >= tokens) return;
  // lane i looks for token i: one way through the tables for all of them (token after token in scalar
  // registers, 65536 tokens of 8 x 128 int8 took 78 us)
  const int mine = min(t0 + (lane < TW ? lane : 0), tokens - 1);
  int s = sequence_of(cu, sequences, t0);
  uint32_t my_page, my_off;
  const int my_state = find_token(mine, s, cu, starts, sequences, table, table_stride, columns, pages,
                                  page_size, a.by_page, &my_page, &my_off);
  int64_t src[TW], s_at[TW];
  int state[TW];
#pragma unroll
  for (int i = 0; i < TW; ++i) {
    state[i] = t0 + i < tokens ? __builtin_amdgcn_readlane(my_state, i) : 0;
    const uint32_t page = lane_value(my_page, i), off = lane_value(my_off, i);
    src[i] = page * k.c_page + off * k.c_token;
    s_at[i] = page * k.s_page + off * k.s_token;
  }
  const int64_t head = pass * (64 >> sh) + (lane >> sh);
  if (head >= a.heads) return;
#pragma unroll
  for (int n = 0; n < NU; ++n) {
    const int unit = j + n * k.lanes, at = unit * 8, left = k.dim - at;
    if (left <= 0) continue;
    KvUnit<FMT> u[TW];
#pragma unroll
    for (int i = 0; i < TW; ++i) {
      if (state[i] == 1) {
        u[i] = load_codes<FMT, WHOLE>(k.codes + src[i] + head * k.c_head, k.scales,
                                      s_at[i] + head * k.s_head, unit, left);
      }
    }
#pragma unroll
    for (int i = 0; i < TW; ++i) {
      if (state[i] == 0) continue;
      S* dst = static_cast<S*>(k.plain) + (t0 + i) * k.p_token;
      store_unit<S, WHOLE>(dst + (head * k.p_head + at), values_of<E, FMT>(u[i], state[i] == 2), left);
    }
  }
}

// ---------------------------------------------------------------------------------------------
// Host side.

namespace {

// Whether a side's vectors are whole units aligned to 16 bytes (plain) and to a unit's codes.
bool whole_units(const KvSide& k, int fmt, int elem) {
  const int64_t c = fmt == KV_MXFP4 ? 4 : 8;
  return k.dim % 8 == 0 && aligned(16, k.plain) && aligned((int)c, k.codes) &&
         k.p_token * elem % 16 == 0 && k.p_head * elem % 16 == 0 && k.c_page % c == 0 &&
         k.c_token % c == 0 && k.c_head % c == 0;
}

int kv_sides(const char* name, const mcop_kv_side* key, const mcop_kv_side* value,
             mcop_dtype cache_dtype, mcop_dtype dtype, int64_t pages, int64_t page_size,
             int64_t heads, int64_t tokens, KvSides* a, int* fmt, bool* whole) {
  *fmt = format_of(cache_dtype);
  if (*fmt < 0) {
    return set_error(MCOP_E_INVALID, "%s: cache dtype %d is not int8, fp8_e4m3fn or mxfp4", name,
                     (int)cache_dtype);
  }
  if (dtype != MCOP_BF16 && dtype != MCOP_F16 && dtype != MCOP_F32) {
    return set_error(MCOP_E_INVALID, "%s: dtype %d is not bf16/fp16/fp32", name, (int)dtype);
  }
  if (!key || !value) return set_error(MCOP_E_INVALID, "%s: null pointer", name);
  if (tokens < 0 || heads <= 0 || pages < 0 || page_size <= 0 || page_size > INT32_MAX ||
      heads > INT32_MAX || pages > INT32_MAX || pages * page_size > INT32_MAX) {
    return set_error(MCOP_E_INVALID,
                     "%s: bad shape num_tokens=%lld num_heads=%lld num_pages=%lld page_size=%lld "
                     "(at most 2^31 - 1 slots)", name, (long long)tokens, (long long)heads,
                     (long long)pages, (long long)page_size);
  }
  if (tokens > (INT32_MAX - 65536) / heads) {
    return set_error(MCOP_E_UNSUPPORTED, "%s: %lld tokens of %lld heads are 2^31 vectors or more",
                     name, (long long)tokens, (long long)heads);
  }
  if (int rc = side_of(name, "key", *key, *fmt, pages, page_size, heads, tokens, &a->side[0])) {
    return rc;
  }
  if (int rc = side_of(name, "value", *value, *fmt, pages, page_size, heads, tokens,
                       &a->side[1])) {
    return rc;
  }
  a->heads = (int)heads;
  a->by_heads = Divisor((uint32_t)heads);
  a->by_page = Divisor((uint32_t)page_size);
  const int elem = dtype == MCOP_F32 ? 4 : 2;
  *whole = whole_units(a->side[0], *fmt, elem) && whole_units(a->side[1], *fmt, elem);
  return MCOP_OK;
}

// A launch takes fewer than 2^32 threads along x.
constexpr int64_t kMostBlocks = ((int64_t)1 << 32) / kKvLanes - 1;

// Workgroups for `vectors` vectors at `r` rounds a workgroup, of the side that needs more.
int64_t kv_blocks(const KvSides& a, int64_t vectors, int r) {
  const int64_t per = (int64_t)kKvLanes / std::max(a.side[0].lanes, a.side[1].lanes) * r;
  return (vectors + per - 1) / per;
}

bool two_units(const KvSides& a) { return a.side[0].dim > 512 || a.side[1].dim > 512; }

// Whether a token's vectors fill a wave on both sides; the passes over its heads, of the side that has
// more; and the workgroups for those.
bool by_tokens(const KvSides& a) {
  return (int64_t)a.heads * std::min(a.side[0].lanes, a.side[1].lanes) >= 64;
}
int64_t head_passes(const KvSides& a) {
  const int lanes = std::max(a.side[0].lanes, a.side[1].lanes);
  return ((int64_t)a.heads * lanes + 63) / 64;
}
int64_t token_blocks(const KvSides& a, int64_t tokens, int tw) {
  const int64_t items = (tokens + tw - 1) / tw * head_passes(a), waves = kKvLanes / 64;
  return (items + waves - 1) / waves;
}
// Whether a launch takes so many workgroups; sets the grid, or the error.
bool kv_grid(const char* name, int64_t blocks, dim3* grid) {
  *grid = dim3((unsigned)blocks, 2);
  if (blocks <= kMostBlocks) return true;
  set_error(MCOP_E_UNSUPPORTED, "%s: more vectors than one launch takes (%lld workgroups)", name,
            (long long)blocks);
  return false;
}
// The launch's trace line; a_wave: tokens a wave takes at a time, 0 where it takes vectors.
void trace_kv(const char* name, const KvSides& a, int64_t tokens, bool whole, int a_wave,
              const dim3& grid) {
  if (!launches_traced()) return;
  char how[48] = "a vector a group of lanes";
  if (a_wave > 0) snprintf(how, sizeof(how), "whole tokens a wave, %d at a time", a_wave);
  trace_launch(name, "tokens=%lld heads=%d head sizes %d and %d: %s, %d units a lane, %s, wgs=%u x 2",
               (long long)tokens, a.heads, a.side[0].dim, a.side[1].dim, how, two_units(a) ? 2 : 1,
               whole ? "whole units" : "any alignment", grid.x);
}
// Tokens a wave: four where that leaves 4096 waves or more, else one.
bool four_tokens(const KvSides& a, int64_t tokens) { return tokens * head_passes(a) >= 8192; }

template <class E, int FMT, bool WHOLE>
int write_of(const char* name, const KvSides& a, const int64_t* slots, int64_t vectors,
             int64_t num_slots, int page_size, hipStream_t st) {
  const dim3 block(kKvLanes);
  dim3 grid;
  const int tokens = (int)(vectors / a.heads);
  if (by_tokens(a)) {
    const bool four = four_tokens(a, tokens);
    if (!kv_grid(name, token_blocks(a, tokens, four ? 4 : 1), &grid)) return MCOP_E_UNSUPPORTED;
    trace_kv(name, a, tokens, WHOLE, four ? 4 : 1, grid);
#define MCOP_WRITE(NU, TW)                                                                       \
  hipLaunchKernelGGL((k_kv_cache_write_tokens<E, FMT, WHOLE, NU, TW>), grid, block, 0, st, a, \
                     slots, tokens, num_slots, page_size)
    if (two_units(a)) {
      if (four) MCOP_WRITE(2, 4);
      else MCOP_WRITE(2, 1);
    } else {
      if (four) MCOP_WRITE(1, 4);
      else MCOP_WRITE(1, 1);
    }
#undef MCOP_WRITE
  } else {
    if (!kv_grid(name, kv_blocks(a, vectors, 1), &grid)) return MCOP_E_UNSUPPORTED;
    trace_kv(name, a, tokens, WHOLE, 0, grid);
    if (two_units(a)) {
      hipLaunchKernelGGL((k_kv_cache_write<E, FMT, WHOLE, 2>), grid, block, 0, st, a, slots,
                         (uint32_t)vectors, num_slots, page_size);
    } else {
      hipLaunchKernelGGL((k_kv_cache_write<E, FMT, WHOLE, 1>), grid, block, 0, st, a, slots,
                         (uint32_t)vectors, num_slots, page_size);
    }
  }
  return check_launch(name);
}

template <class E, int FMT, bool WHOLE>
int read_of(const char* name, const KvSides& a, const int32_t* table, int64_t table_stride,
            int columns, const int32_t* cu, const int32_t* starts, int sequences, int64_t vectors,
            int64_t pages, int page_size, hipStream_t st) {
  const dim3 block(kKvLanes);
  dim3 grid;
  const int tokens = (int)(vectors / a.heads);
  if (by_tokens(a)) {
    const bool four = four_tokens(a, tokens);
    if (!kv_grid(name, token_blocks(a, tokens, four ? 4 : 1), &grid)) return MCOP_E_UNSUPPORTED;
    trace_kv(name, a, tokens, WHOLE, four ? 4 : 1, grid);
#define MCOP_READ(NU, TW)                                                                        \
  hipLaunchKernelGGL((k_kv_cache_read_tokens<E, FMT, WHOLE, NU, TW>), grid, block, 0, st, a,     \
                     table, table_stride, columns, cu, starts, sequences, tokens, pages, page_size)
    if (two_units(a)) {
      if (four) MCOP_READ(2, 4);
      else MCOP_READ(2, 1);
    } else {
      if (four) MCOP_READ(1, 4);
      else MCOP_READ(1, 1);
    }
#undef MCOP_READ
  } else {
    const int rounds = two_units(a) ? 1 : 4;
    if (!kv_grid(name, kv_blocks(a, vectors, rounds), &grid)) return MCOP_E_UNSUPPORTED;
    trace_kv(name, a, tokens, WHOLE, 0, grid);
    if (two_units(a)) {
      hipLaunchKernelGGL((k_kv_cache_read<E, FMT, WHOLE, 2, 1>), grid, block, 0, st, a, table,
                         table_stride, columns, cu, starts, sequences, (uint32_t)vectors, pages,
                         page_size);
    } else {
      hipLaunchKernelGGL((k_kv_cache_read<E, FMT, WHOLE, 1, 4>), grid, block, 0, st, a, table,
                         table_stride, columns, cu, starts, sequences, (uint32_t)vectors, pages,
                         page_size);
    }
  }
  return check_launch(name);
}

// f(E, FMT, WHOLE) for the launch's types.
template <class F>
int for_types(mcop_dtype dtype, int fmt, bool whole, F f) {
  auto by_form = [&](auto e, auto m) {
    return whole ? f(e, m, std::true_type()) : f(e, m, std::false_type());
  };
  auto by_format = [&](auto e) {
    if (fmt == KV_INT8) return by_form(e, std::integral_constant<int, KV_INT8>());
    if (fmt == KV_FP8) return by_form(e, std::integral_constant<int, KV_FP8>());
    return by_form(e, std::integral_constant<int, KV_MXFP4>());
  };
  if (dtype == MCOP_BF16) return by_format(BF16());
  if (dtype == MCOP_F16) return by_format(F16());
  return by_format(F32());
}

}  // namespace

}  // namespace mcop

extern "C" int mcop_kv_cache_write_quant(const mcop_kv_side* key, const mcop_kv_side* value,
                                         mcop_dtype cache_dtype, int64_t num_pages,
                                         int64_t page_size, int64_t num_heads,
                                         const int64_t* slot_mapping, int64_t num_tokens,
                                         mcop_dtype in_dtype, void* stream) {
  using namespace mcop;
  const char* name = "kv_cache_write_quant";
  KvSides a;
  int fmt;
  bool whole;
  if (num_tokens == 0) return MCOP_OK;
  if (int rc = kv_sides(name, key, value, cache_dtype, in_dtype, num_pages, page_size, num_heads,
                        num_tokens, &a, &fmt, &whole)) {
    return rc;
  }
  if (!slot_mapping) return set_error(MCOP_E_INVALID, "%s: null pointer", name);
  if (num_pages == 0) return MCOP_OK;  // no slot to write to
  auto st = static_cast<hipStream_t>(stream);
  return for_types(in_dtype, fmt, whole, [&](auto e, auto m, auto w) {
    return write_of<decltype(e), decltype(m)::value, decltype(w)::value>(
        name, a, slot_mapping, num_tokens * num_heads, num_pages * page_size, (int)page_size, st);
  });
}

extern "C" int mcop_kv_cache_read_dequant(const mcop_kv_side* key, const mcop_kv_side* value,
                                          mcop_dtype cache_dtype, int64_t num_pages,
                                          int64_t page_size, int64_t num_heads,
                                          const int32_t* block_table, int64_t table_row_stride,
                                          int64_t table_columns, const int32_t* cu_seqlens,
                                          const int32_t* seq_starts, int64_t num_sequences,
                                          int64_t num_tokens, mcop_dtype out_dtype,
                                          void* stream) {
  using namespace mcop;
  const char* name = "kv_cache_read_dequant";
  KvSides a;
  int fmt;
  bool whole;
  if (num_tokens == 0 || num_sequences == 0) return MCOP_OK;
  if (int rc = kv_sides(name, key, value, cache_dtype, out_dtype, num_pages, page_size, num_heads,
                        num_tokens, &a, &fmt, &whole)) {
    return rc;
  }
  if (num_sequences < 0 || num_sequences > INT32_MAX || table_columns < 0 ||
      table_columns > INT32_MAX || table_row_stride < 0 ||
      table_row_stride > INT64_MAX / 8 / num_sequences) {
    return set_error(MCOP_E_INVALID, "%s: bad block table: %lld sequences of %lld pages", name,
                     (long long)num_sequences, (long long)table_columns);
  }
  if (!cu_seqlens || (!block_table && table_columns > 0)) {
    return set_error(MCOP_E_INVALID, "%s: null pointer", name);
  }
  auto st = static_cast<hipStream_t>(stream);
  return for_types(out_dtype, fmt, whole, [&](auto e, auto m, auto w) {
    return read_of<decltype(e), decltype(m)::value, decltype(w)::value>(
        name, a, block_table, table_row_stride, (int)table_columns, cu_seqlens, seq_starts,
        (int)num_sequences, num_tokens * num_heads, num_pages, (int)page_size, st);
  });
}
