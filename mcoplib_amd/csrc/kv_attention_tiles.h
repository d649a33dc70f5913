// kv_attention_tiles.h -- decode attention on the matrix units (kv_attention.h has the mathematics and the
// split): a wave takes tiles of 32 positions of one key head for up to sixteen of its query heads.
//
// Both products run on v_mfma_f32_16x16x32_bf16, transposed, so that a lane keeps one query head all the
// way: S^T = K Q^T has positions in rows and query heads in columns, O^T = V^T P^T elements in rows and
// query heads in columns.  Lane (c = lane % 16, g = lane / 16) holds
//   K   position c (and 16 + c) of the tile, 16 elements from 64 kp + 16 g of each pair kp of K steps
//   S   query head c, positions 4 g + i and 16 + 4 g + i: as they come out of the first product they are
//       the second one's operand, whose eight positions a lane are taken in this order
//   V   those eight positions, VD elements from VD c: its rows for VD products, one element of each
//   O   query head c, elements VD (4 g + i) + n
// so codes go from memory to the matrix units in registers: no LDS, no barrier, and a transposition of V
// that is half an instruction an element (two positions' elements to a dword).  Vectors that are not
// whole units of 16 (K) or VD (V) elements end in a unit that overlaps the one before: its queries are zero
// where it repeats elements, and outputs that come twice are the same.
//
// Every code (int8, e4m3, e2m1 with its block's power of two) is a bf16 value.  fp32 scales stay out of
// the products: a key's multiplies its logit, a value's its weight.  Queries enter as the sum of one bf16
// (bf16), two (fp16) or three (fp32), which is exact; weights as two (to 2^-17 of themselves: a half step
// of fp16 outputs is 2^-11, of bf16 outputs 2^-9) or, for fp32, three (2^-26).
#pragma once

#include "kv_attention.h"

namespace mcop {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kTileRows = 16;  // query heads of a workgroup

template <class E>
struct AttTerms {  // bf16 terms of a query, of a weight
  static constexpr int Q = std::is_same_v<E, F32> ? 3 : (std::is_same_v<E, F16> ? 2 : 1);
  static constexpr int P = std::is_same_v<E, F32> ? 3 : 2;
};

// Two fp32 values as bf16 in a dword, and what that leaves of them.
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), bf16x2));
}
__device__ __forceinline__ uint32_t take_bf16(float& a, float& b) {
  const uint32_t u = pack_bf16(a, b);
  a -= __builtin_bit_cast(float, u << 16);
  b -= __builtin_bit_cast(float, u & 0xffff0000u);
  return u;
}
// The high halves of two dwords, the low halves.
__device__ __forceinline__ uint32_t high_halves(uint32_t lo, uint32_t hi) {
  return __builtin_amdgcn_perm(hi, lo, 0x07060302u);
}
__device__ __forceinline__ uint32_t low_halves(uint32_t lo, uint32_t hi) {
  return __builtin_amdgcn_perm(hi, lo, 0x05040100u);
}
__device__ __forceinline__ uint32_t i8_bits(uint32_t w, int byte) {  // as binary32
  return __builtin_bit_cast(uint32_t, (float)(int8_t)(w >> (8 * byte)));
}
// Codes 2 i, 2 i + 1 of the dwords at w as bf16.
template <int FMT>
__device__ __forceinline__ uint32_t code_pair(const uint32_t* w, int i, float scale) {
  if constexpr (FMT == KV_INT8) {
    return high_halves(i8_bits(w[i >> 1], (i & 1) * 2), i8_bits(w[i >> 1], (i & 1) * 2 + 1));
  } else if constexpr (FMT == KV_FP8) {
    return __builtin_bit_cast(uint32_t, i & 1 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i >> 1], 1.0f, true)
                                              : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i >> 1], 1.0f, false));
  } else {
    const uint32_t d = w[i >> 2];
    bf16x2 r;
    switch (i & 3) {
      case 0: r = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d, scale, 0); break;
      case 1: r = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d, scale, 1); break;
      case 2: r = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d, scale, 2); break;
      default: r = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d, scale, 3);
    }
    return __builtin_bit_cast(uint32_t, r);
  }
}

__device__ __forceinline__ uint32_t from_lane(uint32_t v, int lane) {
  return (uint32_t)__builtin_amdgcn_ds_bpermute(lane * 4, (int)v);
}
__device__ __forceinline__ int64_t from_lane64(int64_t v, int lane) {
  return (int64_t)((uint64_t)from_lane((uint32_t)((uint64_t)v >> 32), lane) << 32 |
                   from_lane((uint32_t)v, lane));
}
__device__ __forceinline__ float from_lane_f(float v, int lane) {
  return __builtin_bit_cast(float, from_lane(__builtin_bit_cast(uint32_t, v), lane));
}

// N bytes (2, 4, 8, 16) at any alignment.
template <int N>
__device__ __forceinline__ void load_bytes(uint32_t* w, const uint8_t* p) {
  if constexpr (N == 2) {
    uint16_t v;
    __builtin_memcpy(&v, p, 2);
    w[0] = v;
  } else {
    __builtin_memcpy(w, p, N);
  }
}
// A vector's `n` (1..8) scale bytes in two dwords: block b in byte b of the first, or from the fifth on in
// byte b - (n - 4) of the second.
__device__ __forceinline__ void load_scales8(uint32_t* w, const uint8_t* p, int n) {
  w[0] = w[1] = 0;
  if (n >= 4) {
    __builtin_memcpy(&w[0], p, 4);
    if (n > 4) __builtin_memcpy(&w[1], p + (n - 4), 4);
  } else {
    w[0] = p[0];
    if (n > 1) w[0] |= (uint32_t)p[1] << 8;
    if (n > 2) w[0] |= (uint32_t)p[2] << 16;
  }
}
// The byte selector that puts block b's scale in the top byte of v_perm(w[1], w[0]).
__device__ __forceinline__ uint32_t scale_selector(int b, int n) {
  return (uint32_t)(b < 4 ? b : 4 + b - (n - 4)) << 24 | 0x0c0c0cu;
}
__device__ __forceinline__ float scale_operand(const uint32_t* w, uint32_t selector) {
  return __builtin_bit_cast(float, __builtin_amdgcn_perm(w[1], w[0], selector) >> 1);
}

// The larger, the sum over the four lanes of a query head.
__device__ __forceinline__ float column_max(float v) {
  v = __builtin_fmaxf(v, __shfl_xor(v, 16, 64));
  return __builtin_fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ float column_sum(float v) {
  v += __shfl_xor(v, 16, 64);
  return v + __shfl_xor(v, 32, 64);
}

// What a lane knows of a tile's position lane % 32: its page (or where a wrong one was found), and its place
// on it.  Positions before the first or behind the last stand for those.
struct TilePlace {
  int page;
  uint32_t off;
};

// A tile as it lies in the cache.
template <int FMT, int KP, int VD>
struct TileCodes {
  static constexpr int KW = FMT == KV_MXFP4 ? 2 : 4;                          // dwords of 16 codes
  static constexpr int VB = FMT == KV_MXFP4 ? VD / 2 : VD, VW = (VB + 3) / 4;  // bytes, dwords of VD codes
  uint32_t k[2][KP][KW];
  uint32_t v[8][VW];
  float ks, vs;                 // scales of position lane % 32
  uint32_t kb[2], vb[2];        // the same of 4-bit blocks
};

template <class E, int FMT, int KP, int VD>
struct TileKernel {
  static constexpr int TQ = AttTerms<E>::Q, TP = AttTerms<E>::P;
  using Codes = TileCodes<FMT, KP, VD>;
  static constexpr bool MX = FMT == KV_MXFP4;

  const AttArgs& a;
  const int lane, c, g;
  const int32_t* row;                // of the table
  const uint8_t *k_base, *v_base;    // of the key head
  const void *ks_base, *vs_base;
  int first, end;
  int k_at[KP], v_at;                // bytes
  uint32_t k_sel[KP], v_sel;
  bf16x8 q[KP][2][TQ];
  f32x4 o[VD];
  float m, l;
  int unit;
  bool missing;

  __device__ __forceinline__ TileKernel(const AttArgs& args, const AttChunk& chunk, int head,
                                        int head0, int rows)
      : a(args), lane((int)threadIdx.x & 63), c(lane & 15), g(lane >> 4) {
    row = a.table + chunk.sequence * a.table_stride;
    k_base = a.key.codes + head * a.key.c_head;
    v_base = a.value.codes + head * a.value.c_head;
    const int es = MX ? 1 : 4;
    ks_base = static_cast<const uint8_t*>(a.key.scales) + head * a.key.s_head * es;
    vs_base = static_cast<const uint8_t*>(a.value.scales) + head * a.value.s_head * es;
    first = chunk.first, end = chunk.end;
    const int from = value_at(c);
    v_at = MX ? from / 2 : from;
    v_sel = MX ? scale_selector(from / kMxBlock, a.value.dim / kMxBlock) : 0;
    const typename E::S* src = static_cast<const typename E::S*>(a.key.plain) +
                               chunk.sequence * a.key.p_token +
                               (head0 + min(c, rows - 1)) * a.key.p_head;
#pragma unroll
    for (int kp = 0; kp < KP; ++kp) {
      const int nominal = kp * 64 + g * 16, at = min(nominal, a.key.dim - 16);
      k_at[kp] = MX ? at / 2 : at;
      k_sel[kp] = MX ? scale_selector(at / kMxBlock, a.key.dim / kMxBlock) : 0;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        uint32_t w[TQ][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float f[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int d = at + j * 8 + i * 2 + e;
            f[e] = d >= nominal && c < rows ? E::to_f(src[d]) : 0.0f;
          }
#pragma unroll
          for (int t = 0; t < TQ; ++t) w[t][i] = take_bf16(f[0], f[1]);
        }
#pragma unroll
        for (int t = 0; t < TQ; ++t) {
          q[kp][j][t] = __builtin_bit_cast(bf16x8, (u32x4{w[t][0], w[t][1], w[t][2], w[t][3]}));
        }
      }
    }
#pragma unroll
    for (int n = 0; n < VD; ++n) o[n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    m = -__builtin_inff(), l = 0.0f;
    unit = MX ? 0 : kAttNoUnit;
    missing = false;
  }

  // The first element of lane column r's unit of a value vector.
  __device__ __forceinline__ int value_at(int r) const { return min(r * VD, a.value.dim - VD); }

  __device__ __forceinline__ TilePlace place(int tile) const {
    const int p = min(max(tile * kAttTile + (lane & 31), first), end - 1);
    const uint32_t column = a.by_page.quotient((uint32_t)p);
    return TilePlace{row[column], (uint32_t)p - column * (uint32_t)a.page_size};
  }

  __device__ __forceinline__ void load(Codes& t, const TilePlace& at) {
    const bool none = at.page < 0 || at.page >= a.pages;
    missing |= none;
    const int64_t page = none ? 0 : at.page, off = at.off;
    const int64_t ko = page * a.key.c_page + off * a.key.c_token;
    const int64_t vo = page * a.value.c_page + off * a.value.c_token;
    const int64_t kso = page * a.key.s_page + off * a.key.s_token;
    const int64_t vso = page * a.value.s_page + off * a.value.s_token;
    if constexpr (MX) {
      load_scales8(t.kb, static_cast<const uint8_t*>(ks_base) + kso, a.key.dim / kMxBlock);
      load_scales8(t.vb, static_cast<const uint8_t*>(vs_base) + vso, a.value.dim / kMxBlock);
    } else {
      t.ks = static_cast<const float*>(ks_base)[kso];
      t.vs = static_cast<const float*>(vs_base)[vso];
    }
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const uint8_t* p = k_base + from_lane64(ko, s * 16 + c);
#pragma unroll
      for (int kp = 0; kp < KP; ++kp) load_bytes<Codes::KW * 4>(t.k[s][kp], p + k_at[kp]);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      load_bytes<Codes::VB>(t.v[e], v_base + from_lane64(vo, position(e)) + v_at);
    }
  }

  // The tile's position of element e of S, P and V.
  __device__ __forceinline__ int position(int e) const { return (e >> 2) * 16 + g * 4 + (e & 3); }

  __device__ __forceinline__ void compute(Codes& t, int tile) {
    f32x4 s[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t b[2] = {0, 0};
      if constexpr (MX) {
        b[0] = from_lane(t.kb[0], h * 16 + c);
        if (KP > 2) b[1] = from_lane(t.kb[1], h * 16 + c);
      }
      s[h] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int kp = 0; kp < KP; ++kp) {
        const float scale = MX ? scale_operand(b, k_sel[kp]) : 1.0f;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint32_t* w = t.k[h][kp] + j * (Codes::KW / 2);
          const bf16x8 k = __builtin_bit_cast(
              bf16x8, (u32x4{code_pair<FMT>(w, 0, scale), code_pair<FMT>(w, 1, scale),
                             code_pair<FMT>(w, 2, scale), code_pair<FMT>(w, 3, scale)}));
#pragma unroll
          for (int x = TQ - 1; x >= 0; --x) {  // the smallest terms first
            s[h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, q[kp][j][x], s[h], 0, 0, 0);
          }
        }
      }
    }
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      f[e] = s[e >> 2][e & 3] * (MX ? a.scale : from_lane_f(t.ks * a.scale, position(e)));
    }
    // a tile that holds positions outside [first, end): no weight, and nothing that could spoil a sum
    const bool edge = tile * kAttTile < first || tile * kAttTile + kAttTile > end;
    if (edge) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int p = tile * kAttTile + position(e);
        if (p < first || p >= end) {
          f[e] = -__builtin_inff();
#pragma unroll
          for (int x = 0; x < Codes::VW; ++x) t.v[e][x] = 0;
        }
      }
    }
    float top = __builtin_fmaxf(__builtin_fmaxf(__builtin_fmaxf(f[0], f[1]), __builtin_fmaxf(f[2], f[3])),
                                __builtin_fmaxf(__builtin_fmaxf(f[4], f[5]), __builtin_fmaxf(f[6], f[7])));
    top = __builtin_fmaxf(m, column_max(top));
    int e_max = unit;
    bool wider = false;
    if constexpr (!MX) {
      const int e = att_unit(t.vs);
      wider = __builtin_amdgcn_ballot_w64(e > unit) != 0;
      if (wider) {
        e_max = max(e, unit);
#pragma unroll
        for (int d = 1; d < 32; d *= 2) e_max = max(e_max, __shfl_xor(e_max, d, 64));
      }
    }
    if (wider || __builtin_amdgcn_ballot_w64(top > m) != 0) {
      const float keep = att_weight(m, top);
      const float keep_o = keep * att_power(unit - e_max);
      l *= keep;
#pragma unroll
      for (int n = 0; n < VD; ++n) o[n] *= keep_o;
      m = top;
      unit = e_max;
    }
    const float at = m == -__builtin_inff() ? 0.0f : m;
    const float vs = MX ? 1.0f : __builtin_ldexpf(t.vs, -unit);
    float w[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float p = __builtin_amdgcn_exp2f(f[e] - at);
      l += p;
      w[e] = MX ? p : p * from_lane_f(vs, position(e));
    }
    if (!MX && edge) {  // no 0 times a scale that is no number
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int p = tile * kAttTile + position(e);
        if (p < first || p >= end) w[e] = 0.0f;
      }
    }
    bf16x8 p[TP];
    {
      uint32_t d[TP][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int x = 0; x < TP; ++x) d[x][i] = take_bf16(w[i * 2], w[i * 2 + 1]);
      }
#pragma unroll
      for (int x = 0; x < TP; ++x) {
        p[x] = __builtin_bit_cast(bf16x8, (u32x4{d[x][0], d[x][1], d[x][2], d[x][3]}));
      }
    }
    float scale[8];
    if constexpr (MX) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        uint32_t b[2];
        b[0] = from_lane(t.vb[0], position(e));
        b[1] = VD > 8 ? from_lane(t.vb[1], position(e)) : 0;
        scale[e] = scale_operand(b, v_sel);
        if (edge) {
          const int at_p = tile * kAttTile + position(e);
          if (at_p < first || at_p >= end) scale[e] = 1.0f;
        }
      }
    }
#pragma unroll
    for (int n = 0; n < VD; n += 2) {
      uint32_t even[4], odd[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t *x = t.v[i * 2], *y = t.v[i * 2 + 1];
        if constexpr (FMT == KV_INT8) {
          even[i] = high_halves(i8_bits(x[n >> 2], n & 3), i8_bits(y[n >> 2], n & 3));
          odd[i] = high_halves(i8_bits(x[n >> 2], (n & 3) + 1), i8_bits(y[n >> 2], (n & 3) + 1));
        } else {
          const uint32_t xs = code_pair<FMT>(x, n >> 1, MX ? scale[i * 2] : 1.0f);
          const uint32_t ys = code_pair<FMT>(y, n >> 1, MX ? scale[i * 2 + 1] : 1.0f);
          even[i] = low_halves(xs, ys), odd[i] = high_halves(xs, ys);
        }
      }
      const bf16x8 v0 = __builtin_bit_cast(bf16x8, (u32x4{even[0], even[1], even[2], even[3]}));
      const bf16x8 v1 = __builtin_bit_cast(bf16x8, (u32x4{odd[0], odd[1], odd[2], odd[3]}));
#pragma unroll
      for (int x = TP - 1; x >= 0; --x) {
        o[n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v0, p[x], o[n], 0, 0, 0);
        o[n + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v1, p[x], o[n + 1], 0, 0, 0);
      }
    }
  }
};

template <class E, int FMT, int KP, int VD>
__global__ void __launch_bounds__(kAttWaves * 64)
k_kv_attention_tiles(AttArgs a) {
  // m, l [waves][16], e [waves], o [waves][rows][value.dim + 1]
  extern __shared__ float lds[];
  using K = TileKernel<E, FMT, KP, VD>;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  uint32_t flat;
  int head, block;
  att_place(a, &flat, &head, &block);
  AttChunk c;
  if (!find_chunk(a, flat, head == 0 && block == 0 && wave == 0, &c)) return;
  const int head0 = head * a.group + block * kTileRows;
  const int rows = min(kTileRows, a.group - block * kTileRows);
  K k(a, c, head, head0, rows);
  const int last = c.tile + c.tiles - 1;
  int tile = c.tile + wave;
  if (tile <= last) {
    // two tiles' codes in turn; a position's page is looked up two tiles ahead, its codes are loaded one
    typename K::Codes t[2];
    TilePlace next = k.place(min(tile + kAttWaves, last));
    k.load(t[0], k.place(tile));
    for (;;) {
      TilePlace after = k.place(min(tile + 2 * kAttWaves, last));
      if (tile + kAttWaves <= last) k.load(t[1], next);
      k.compute(t[0], tile);
      tile += kAttWaves;
      if (tile > last) break;
      next = k.place(min(tile + 2 * kAttWaves, last));
      if (tile + kAttWaves <= last) k.load(t[0], after);
      k.compute(t[1], tile);
      tile += kAttWaves;
      if (tile > last) break;
    }
  }
  const bool missing = __builtin_amdgcn_ballot_w64(k.missing) != 0;
  const float l = column_sum(k.l);
  float *ms = lds, *ls = ms + kAttWaves * kTileRows;
  int* es = reinterpret_cast<int*>(ls + kAttWaves * kTileRows);
  float* os = reinterpret_cast<float*>(es + kAttWaves);
  const int most = min(kTileRows, a.group), stride = a.value.dim + 1;
  if (k.g == 0) {
    ms[wave * kTileRows + k.c] = k.m;
    ls[wave * kTileRows + k.c] = missing ? __builtin_nanf("") : l;
  }
  if (k.lane == 0) es[wave] = k.unit;
  if (k.c < rows) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float* dst = os + (wave * most + k.c) * stride + k.value_at(k.g * 4 + i);
#pragma unroll
      for (int n = 0; n < VD; ++n) dst[n] = k.o[n][i];
    }
  }
  __syncthreads();
  att_write<E>(a, c, head0, rows, 0, a.value.dim, ms, ls, es, os, kTileRows, most, stride);
}

// The kernels' head sizes: keys of up to 64 KP and values of up to 16 VD elements, at least a unit of each.
struct TileShape {
  int kp, vd;
};
constexpr TileShape kTileShapes[] = {{1, 4}, {2, 8}, {3, 8}, {4, 16}};

// Launches the kernel of shape `shape` (an index above) on the sequences' chunks.
int attention_tiles_int8(int shape, mcop_dtype dtype, const AttArgs& a, dim3 grid, size_t lds,
                         hipStream_t st);
int attention_tiles_fp8(int shape, mcop_dtype dtype, const AttArgs& a, dim3 grid, size_t lds,
                        hipStream_t st);
int attention_tiles_mxfp4(int shape, mcop_dtype dtype, const AttArgs& a, dim3 grid, size_t lds,
                          hipStream_t st);

template <int FMT, class E>
void attention_tiles_of(int shape, const AttArgs& a, dim3 grid, size_t lds, hipStream_t st) {
  const dim3 block(kAttWaves * 64);
  switch (shape) {
    case 0: hipLaunchKernelGGL((k_kv_attention_tiles<E, FMT, 1, 4>), grid, block, lds, st, a); break;
    case 1: hipLaunchKernelGGL((k_kv_attention_tiles<E, FMT, 2, 8>), grid, block, lds, st, a); break;
    case 2: hipLaunchKernelGGL((k_kv_attention_tiles<E, FMT, 3, 8>), grid, block, lds, st, a); break;
    default: hipLaunchKernelGGL((k_kv_attention_tiles<E, FMT, 4, 16>), grid, block, lds, st, a);
  }
}
template <int FMT>
int attention_tiles_for(int shape, mcop_dtype dtype, const AttArgs& a, dim3 grid, size_t lds,
                        hipStream_t st) {
  if (dtype == MCOP_BF16) attention_tiles_of<FMT, BF16>(shape, a, grid, lds, st);
  else if (dtype == MCOP_F16) attention_tiles_of<FMT, F16>(shape, a, grid, lds, st);
  else attention_tiles_of<FMT, F32>(shape, a, grid, lds, st);
  return check_launch("kv_cache_attention");
}

}  // namespace mcop
