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
// so neither the weights nor V change lanes between the products (V's transposition is half an instruction an
// element: two positions' elements to a dword), and no wave waits for another.  Codes come through LDS, where
// they are whole lines, or straight to registers.  Vectors that are not whole units of 16 (K) or VD (V)
// elements end in a unit that overlaps the one before: its queries are zero where it repeats elements, and
// outputs that come twice are the same.
//
// What bounds it: reading the cache, for 4-bit ones also the vector units (with every tile masked, a tenth more
// instructions, 4-bit codes take 4% longer, int8 3%, fp8 the same).  2 x 131072 positions of 8 x 128 fp8 for 8
// query heads each (554 MB) take 107-114 us by card with the join, 5 TB/s, the same reads alone 90-94; 64 ragged
// sequences of 131072 in all, int8 (279 MB), 66 us; 16 of 4-bit keys of 192 and values of 128 (179 MB), 52 us.
// Vector units are 35-39% busy, the matrix units 11-16%.
//
// Every code (int8, e4m3, e2m1 with its block's power of two) is a bf16 value.  fp32 scales stay out of the
// products: a key's multiplies its logit, a value's its weight.  Queries enter as the sum of one bf16 (bf16),
// two (fp16) or three (fp32), weights as three: both exact.  Weights of two rounded terms, 2^-18 off, changed
// the last bit of one 16-bit output in 400; the third is a product more for each of two, and takes 1-2 us of a
// 4-bit cache's 52 and one of the widest heads' 35, nothing else.  Terms are cut off, not rounded, which takes
// as long: rounded ones would be infinite for the largest fp32 queries.
#pragma once

#include "kv_attention.h"

namespace mcop {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// Workgroups a CU that a kernel's registers are held to: two, where that spills none of them (16 x 131072
// positions in all of 8 x 192 and 128 mxfp4: 53 us with two, 57 with one).
constexpr int att_resident(bool fp32, int fmt, int kp, int vd, bool lines) {
  return vd == 16 || (lines && kp == 3 && fmt != KV_MXFP4 && fp32) ? 1 : 2;
}

constexpr int kTileRows = 16;    // query heads of a wave
constexpr float kAttSlack = 8.0f;  // weights are at most 2^8
// Outputs are in units of 2^0 while a tile's largest value scale has an exponent of -60..60, and until one has
// an exponent more than this above the unit's.
constexpr int kAttUnitSlack = 60;

template <class E>
struct AttTerms {  // bf16 terms of a query, of a weight
  static constexpr int Q = std::is_same_v<E, F32> ? 3 : (std::is_same_v<E, F16> ? 2 : 1);
  static constexpr int P = 3;
};

// The high halves of two dwords, the low halves.
__device__ __forceinline__ uint32_t high_halves(uint32_t lo, uint32_t hi) {
  return __builtin_amdgcn_perm(hi, lo, 0x07060302u);
}
__device__ __forceinline__ uint32_t low_halves(uint32_t lo, uint32_t hi) {
  return __builtin_amdgcn_perm(hi, lo, 0x05040100u);
}
// The leading eight bits of two values' significands as bf16 in a dword, and what that leaves of them, exactly:
// three such terms hold a binary32 value, two a binary16 one.  (Of an infinity it leaves NaN.)
__device__ __forceinline__ uint32_t take_bf16(float& a, float& b) {
  const uint32_t x = __builtin_bit_cast(uint32_t, a), y = __builtin_bit_cast(uint32_t, b);
  a -= __builtin_bit_cast(float, x & 0xffff0000u);
  b -= __builtin_bit_cast(float, y & 0xffff0000u);
  return high_halves(x, y);
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

// The larger, the sum over the four lanes of a query head.  The swaps put rows 0 and 2 of a value's four
// rows of sixteen lanes into one register and rows 1 and 3 into the other; the lower and upper halves.
__device__ __forceinline__ void swap_rows(float v, float* x, float* y) {
  const uint32_t u = __builtin_bit_cast(uint32_t, v);
  const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  *x = __builtin_bit_cast(float, (uint32_t)r[0]), *y = __builtin_bit_cast(float, (uint32_t)r[1]);
}
__device__ __forceinline__ void swap_halves(float v, float* x, float* y) {
  const uint32_t u = __builtin_bit_cast(uint32_t, v);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  *x = __builtin_bit_cast(float, (uint32_t)r[0]), *y = __builtin_bit_cast(float, (uint32_t)r[1]);
}
__device__ __forceinline__ float column_max(float v) {
  float x, y;
  swap_rows(v, &x, &y);
  swap_halves(__builtin_fmaxf(x, y), &x, &y);
  return __builtin_fmaxf(x, y);
}
__device__ __forceinline__ float column_sum(float v) {
  float x, y;
  swap_rows(v, &x, &y);
  swap_halves(x + y, &x, &y);
  return x + y;
}

// 16, 4 bytes, or one as a dword, a lane from its address to LDS at `to` + 16, 4 * lane, which the instruction
// takes from m0 (a state after its write).  The compiler sees neither what this writes nor that it is in
// flight: wait_loads() orders it.
__device__ __forceinline__ void tile_to_lds16(uint32_t to, const uint8_t* base, uint32_t off) {
  asm volatile(
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %1, %2"
      :
      : "{m0}"(to), "v"(off), "s"(base)
      : "memory");
}
__device__ __forceinline__ void tile_to_lds1(uint32_t to, const uint8_t* base, uint32_t off) {
  asm volatile(
      "s_nop 0\n\t"
      "global_load_lds_ubyte %1, %2"
      :
      : "{m0}"(to), "v"(off), "s"(base)
      : "memory");
}
__device__ __forceinline__ void tile_to_lds4(uint32_t to, const uint8_t* from) {
  asm volatile(
      "s_nop 0\n\t"
      "global_load_lds_dword %1, off"
      :
      : "{m0}"(to), "v"(from)
      : "memory");
}
// All but the wave's last LEFT loads have landed; its LDS reads are done.
template <int LEFT>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LEFT) : "memory");
}
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// A wave's query heads, its sums, and the two products of a tile, whose codes `src` gives:
//   key(h, kp, w)      sixteen codes of position 16 h + c, and key_scale(h, kp) of 4-bit ones
//   value(e, w)        VD codes of position(e), and value_scale(e) of 4-bit ones
//   ks(e), vs(e)       fp32 scales of position(e)
//   most_vs()          the lane's part of the tile's value scales
//   far(live)          whether a 4-bit one of its part is kMxFarByte or more (live: which of value_scale(e) count)
template <class E, int FMT, int KP, int VD>
struct AttWave {
  static constexpr int TQ = AttTerms<E>::Q, TP = AttTerms<E>::P;
  static constexpr bool MX = FMT == KV_MXFP4;
  static constexpr int KW = MX ? 2 : 4;                                 // dwords of 16 codes
  static constexpr int VB = MX ? VD / 2 : VD, VW = (VB + 3) / 4;        // bytes, dwords of VD codes
  // Wide fp32 kernels have no registers for a tile's values beside its keys: values are read when needed.
  static constexpr bool LATE = VD == 16 && TQ == 3;

  const AttArgs& a;
  const int lane, c, g;
  int first, end;
  Pack<typename E::S, 8> raw[KP][2];  // the queries as they were loaded
  bf16x8 q[KP][2][TQ];
  f32x4 o[VD];
  float m, l;
  int unit;

  __device__ __forceinline__ AttWave(const AttArgs& args, const AttChunk& chunk, int head0, int rows)
      : a(args), lane((int)threadIdx.x & 63), c(lane & 15), g(lane >> 4),
        first(__builtin_amdgcn_readfirstlane(chunk.first)),
        end(__builtin_amdgcn_readfirstlane(chunk.end)) {
    const typename E::S* src = static_cast<const typename E::S*>(a.key.plain) +
                               chunk.sequence * a.key.p_token +
                               (head0 + min(c, rows - 1)) * a.key.p_head;
#pragma unroll
    for (int kp = 0; kp < KP; ++kp) {
#pragma unroll
      for (int j = 0; j < 2; ++j) raw[kp][j] = load8<typename E::S, true, false>(src + key_at(kp) + j * 8);
    }
  }
  // Waits for the queries as they were loaded, before what the elements' conditions would make of the loads.
  __device__ __forceinline__ void settle() {
    constexpr int W = sizeof(raw[0][0]) / 4;
#pragma unroll
    for (int kp = 0; kp < KP; ++kp) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        Pack<uint32_t, W> w = __builtin_bit_cast(Pack<uint32_t, W>, raw[kp][j]);
#pragma unroll
        for (int i = 0; i < W; ++i) asm volatile("" : "+v"(w.v[i]));
        raw[kp][j] = __builtin_bit_cast(Pack<typename E::S, 8>, w);
      }
    }
  }
  // Takes them apart into their terms, and starts with nothing.
  __device__ __forceinline__ void begin(int rows) {
#pragma unroll
    for (int kp = 0; kp < KP; ++kp) {
      if constexpr (VD == 16) __builtin_amdgcn_sched_barrier(0);
      const int nominal = kp * 64 + g * 16, at = key_at(kp);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        uint32_t w[TQ][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float f[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            f[e] = E::to_f(raw[kp][j].v[i * 2 + e]) * (a.scale < 0.0f ? -1.0f : 1.0f);
            if (at + j * 8 + i * 2 + e < nominal || c >= rows) f[e] = 0.0f;
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
    if constexpr (VD == 16) __builtin_amdgcn_sched_barrier(0);
  }

  // The first of the lane's sixteen elements of pair kp of a key; of column r's unit of a value.
  __device__ __forceinline__ int key_at(int kp) const { return min(kp * 64 + g * 16, a.key.dim - 16); }
  __device__ __forceinline__ int value_at(int r) const { return min(r * VD, a.value.dim - VD); }
  // The tile's position of element e of S, P and V.
  __device__ __forceinline__ int position(int e) const { return (e >> 2) * 16 + g * 4 + (e & 3); }

  template <class Src>
  __device__ __forceinline__ void tile(Src& src, int t) {
    // a tile that holds positions outside [first, end): no weight, and nothing that could spoil a sum
    if (t * kAttTile < first || (uint32_t)t * kAttTile + kAttTile > (uint32_t)end) tile_of<true>(src, t);
    else tile_of<false>(src, t);
  }
  template <bool EDGE, class Src>
  __device__ __forceinline__ void tile_of(Src& src, int t) {
    // The two forms begin differently, and take keys as values of their own: else the compiler puts their
    // conversions in front of the branch, all at once, which spills the widest kernels.
    if constexpr (EDGE) asm volatile("; edge" ::: "memory");
    else asm volatile("; inside" ::: "memory");
    bool live[8];
    if constexpr (EDGE) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int p = t * kAttTile + position(e);
        live[e] = p >= first && p < end;
      }
    }
    f32x4 s[2] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
    for (int kp = 0; kp < KP; ++kp) {
      if constexpr (VD == 16) __builtin_amdgcn_sched_barrier(0);
      uint32_t w[2][KW];
      float scale[2] = {1.0f, 1.0f};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        src.key(h, kp, w[h]);
#pragma unroll
        for (int i = 0; i < KW; ++i) asm volatile("" : "+v"(w[h][i]));
        if constexpr (MX) scale[h] = src.key_scale(h, kp);
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if constexpr (VD == 16) __builtin_amdgcn_sched_barrier(0);
        bf16x8 k[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t* x = w[h] + j * (KW / 2);
          k[h] = __builtin_bit_cast(
              bf16x8, (u32x4{code_pair<FMT>(x, 0, scale[h]), code_pair<FMT>(x, 1, scale[h]),
                             code_pair<FMT>(x, 2, scale[h]), code_pair<FMT>(x, 3, scale[h])}));
        }
#pragma unroll
        for (int x = TQ - 1; x >= 0; --x) {  // the smallest terms first
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            s[h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k[h], q[kp][j][x], s[h], 0, 0, 0);
          }
        }
      }
    }
    const float by = __builtin_fabsf(a.scale);  // its sign is the queries'
    if constexpr (VD == 16) __builtin_amdgcn_sched_barrier(0);
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      f[e] = MX ? s[e >> 2][e & 3] : s[e >> 2][e & 3] * src.ks(e);
      if (EDGE) f[e] = live[e] ? f[e] : -__builtin_inff();
    }
    float top = __builtin_fmaxf(__builtin_fmaxf(__builtin_fmaxf(f[0], f[1]), __builtin_fmaxf(f[2], f[3])),
                                __builtin_fmaxf(__builtin_fmaxf(f[4], f[5]), __builtin_fmaxf(f[6], f[7])));
    top = column_max(top);
    top = top == -__builtin_inff() ? m : __builtin_fmaxf(m, top * by);
    int e_max = unit;
    bool wider = false;
    if constexpr (!MX) {
      const int p = t * kAttTile + (lane & 31);
      const int e = EDGE && (p < first || p >= end) ? kAttNoUnit : att_unit(src.most_vs());
      wider = __builtin_amdgcn_ballot_w64(e > unit + kAttUnitSlack) != 0;
      if (wider) {
        e_max = e;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) e_max = max(e_max, __shfl_xor(e_max, d, 64));
        e_max = __builtin_amdgcn_readfirstlane(e_max);
        if (e_max >= -kAttUnitSlack && e_max <= kAttUnitSlack) e_max = 0;
      }
    }
    // The reference of the weights moves when a logit is more than kAttSlack past it, a weight of 2^kAttSlack, not
    // with every new maximum: of sixteen query heads one has a new one in nearly every tile.  4-bit values of
    // any size are looked for in the same branch (1-2% of a 4-bit cache's time, 2-3% with a branch of their own).
    bool far = false;
    if constexpr (MX) far = src.template far<EDGE>(live);
    if (wider || __builtin_amdgcn_ballot_w64(top > m + kAttSlack || far) != 0) {
      if (MX && __builtin_amdgcn_ballot_w64(far) != 0) e_max = kMxUnit;
      const float keep = att_weight(m, top);
      const float keep_o = keep * att_power(unit - e_max);
      l *= keep;
#pragma unroll
      for (int n = 0; n < VD; ++n) o[n] *= keep_o;
      m = top;
      unit = e_max;
    }
    const float at = m == -__builtin_inff() ? 0.0f : m;
    float w[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float p = __builtin_amdgcn_exp2f(__builtin_fmaf(f[e], by, -at));
      if (EDGE) p = live[e] ? p : 0.0f;
      l += p;
      w[e] = MX ? p : p * src.vs(e);
      if (!MX && EDGE) w[e] = live[e] ? w[e] : 0.0f;  // no 0 times a scale that is no number
    }
    if (unit != 0) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if constexpr (MX) {
          w[e] *= att_power(-kMxUnit);
        } else {
          w[e] = EDGE && !live[e] ? 0.0f
                                  : __builtin_amdgcn_exp2f(__builtin_fmaf(f[e], by, -at)) *
                                        __builtin_ldexpf(src.vs(e), -unit);
        }
      }
    }
    if constexpr (VD == 16) __builtin_amdgcn_sched_barrier(0);
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
    uint32_t v[8][VW];
    float scale[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      src.value(e, v[e]);
      scale[e] = 1.0f;
      if constexpr (MX) scale[e] = src.value_scale(e);
      if constexpr (EDGE) {
        scale[e] = live[e] ? scale[e] : 1.0f;
#pragma unroll
        for (int x = 0; x < VW; ++x) v[e][x] = live[e] ? v[e][x] : 0;
      }
    }
#pragma unroll
    for (int n = 0; n < VD; n += 2) {
      // kernels at the end of their registers: no conversion ahead of its product
      if constexpr (VD == 16) __builtin_amdgcn_sched_barrier(0);
      uint32_t even[4], odd[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t *x = v[i * 2], *y = v[i * 2 + 1];
        if constexpr (FMT == KV_INT8) {
          even[i] = high_halves(i8_bits(x[n >> 2], n & 3), i8_bits(y[n >> 2], n & 3));
          odd[i] = high_halves(i8_bits(x[n >> 2], (n & 3) + 1), i8_bits(y[n >> 2], (n & 3) + 1));
        } else {
          const uint32_t xs = code_pair<FMT>(x, n >> 1, scale[i * 2]);
          const uint32_t ys = code_pair<FMT>(y, n >> 1, scale[i * 2 + 1]);
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

  // Writes the wave's query heads: the outputs, or of a split sequence its part.
  __device__ __forceinline__ void write(const AttChunk& ch, int head0, int rows, bool missing) {
    float sum = column_sum(l);
    if (missing || ch.missing) sum = __builtin_nanf("");
    if (c >= rows) return;
    const int query = head0 + c;
    if (g == 0) {
      if (ch.part >= 0) {
        float* dst = a.sums + ((int64_t)ch.part * a.query_heads + query) * 4;
        dst[0] = m, dst[1] = sum, dst[2] = (float)unit;
      } else if (a.lse != nullptr) {
        a.lse[(int64_t)ch.sequence * a.query_heads + query] = att_lse(m, sum);
      }
    }
    // one division a row; an element's rounding of its product is 2^-24 of it
    const float share = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int d = value_at(g * 4 + i);
      if (ch.part >= 0) {
        float* dst = a.parts + ((int64_t)ch.part * a.query_heads + query) * a.value.dim + d;
        float v[VD];
#pragma unroll
        for (int n = 0; n < VD; ++n) v[n] = o[n][i];
        __builtin_memcpy(dst, v, sizeof(v));
      } else {
        typename E::S v[VD];
#pragma unroll
        for (int n = 0; n < VD; ++n) {
          const float x = o[n][i] * share;
          v[n] = E::from_f(unit == 0 ? x : __builtin_ldexpf(x, unit));
        }
        __builtin_memcpy(static_cast<typename E::S*>(a.value.plain) + ch.sequence * a.value.p_token +
                             query * a.value.p_head + d, v, sizeof(v));
      }
    }
  }
};

// ---- Codes through LDS: pages of whole sixteens, vectors of whole 16-byte chunks at multiples of 16.
//
// A wave's loads are then whole cache lines (a lane a chunk, the chunks of a position next to each other),
// where loads in the order of the products take one request a lane: 2 x 131072 positions of 8 x 128 fp8
// took 131 us so, with the L1 busy for four fifths of it.  A half of a tile, 16 positions of one page, is
// CR chunks a position; chunk x of position r goes to place (x + r / (16 / gcd(CR, 16))) mod CR of its row, so
// that the reads of one chunk of sixteen positions fall on different banks.
struct HalfLayout {
  const Divisor& by_row;
  int row, turn;  // chunks a row; log2 of 16 / gcd(row, 16)
  __device__ __forceinline__ explicit HalfLayout(const Divisor& chunks)
      : by_row(chunks), row((int)chunks.d) {
    turn = 4 - min(4, (int)__builtin_ctz((unsigned)row));
  }
  __device__ __forceinline__ int mod(int y) const {
    return y - row * (int)by_row.quotient((uint32_t)y);
  }
  __device__ __forceinline__ int place(int r, int x) const { return r * row + mod(x + (r >> turn)); }
  // Where in the cache, from the half's start, the chunk of LDS place i (of 16 rows) lies.
  __device__ __forceinline__ uint32_t from(int i, int token) const {
    const int r = (int)by_row.quotient((uint32_t)i), turned = mod(r >> turn);
    const int y = i - r * row - turned;
    return (uint32_t)(r * token + (y < 0 ? y + row : y) * 16);
  }
};

template <int FMT, int KP, int VD>
struct LdsTile {  // loads of a half's keys, values and 4-bit blocks' scales; bytes
  static constexpr bool MX = FMT == KV_MXFP4;
  static constexpr int KN = MX ? (KP + 1) / 2 : KP, VN = MX ? (VD + 7) / 8 : (VD + 3) / 4;
  static constexpr int KS = MX ? (KP + 1) / 2 : 0, VS = MX ? (VD + 7) / 8 : 0;
  static constexpr int kScales = 1024 * (KN + VN), kHalf = kScales + 256 * (KS + VS);
  static constexpr int kBytes = 2 * kHalf + (MX ? 0 : 256);
  static constexpr int kLoads = 2 * (KN + VN + KS + VS) + (MX ? 0 : 1);
  static constexpr int kGroup = kAttWaves * 2 * kBytes;  // a workgroup's
};

template <class E, int FMT, int KP, int VD>
struct LdsSource {
  using W = AttWave<E, FMT, KP, VD>;
  using T = LdsTile<FMT, KP, VD>;
  static constexpr bool MX = W::MX;
  const AttArgs& a;
  const W& wave;
  const int32_t* row;  // of the table
  const uint8_t *k_base, *v_base, *ks_base, *vs_base;  // of the key head
  uint32_t k_from[T::KN], v_from[T::VN];  // where the lane's chunks lie in a half of the cache
  uint32_t ks_from[MX ? T::KS : 1], vs_from[MX ? T::VS : 1];  // and its scales
  int k_at[KP], v_at[4];                  // what the lane reads of a half in LDS
  int ks_at[KP], vs_at;
  // halves [base, base + 64) of the sequence: lane i knows half base + i
  int base;
  int64_t ko, vo, kso, vso;
  uint64_t none_at;  // those without a page
  bool missing;
  const uint8_t* lds;  // of the wave
  uint32_t to;
  // the tile in turn
  const uint8_t* at;
  uint32_t k[2][KP][W::KW], v[W::LATE ? 1 : 8][W::VW];
  float kscale[2][MX ? KP : 4], vscale[8], most;

  __device__ __forceinline__ LdsSource(const AttArgs& args, const W& w, const AttChunk& ch, int head,
                                       const uint8_t* mine, uint32_t mine_at)
      : a(args), wave(w), lds(mine), to(mine_at) {
    row = a.table + ch.sequence * a.table_stride;
    const int es = MX ? 1 : 4;
    k_base = a.key.codes + head * a.key.c_head;
    v_base = a.value.codes + head * a.value.c_head;
    ks_base = static_cast<const uint8_t*>(a.key.scales) + head * a.key.s_head * es;
    vs_base = static_cast<const uint8_t*>(a.value.scales) + head * a.value.s_head * es;
    const int lane = w.lane, c = w.c, g = w.g;
    const HalfLayout kl(a.k_chunks), vl(a.v_chunks);
#pragma unroll
    for (int i = 0; i < T::KN; ++i) {
      k_from[i] = kl.from(min(i * 64 + lane, 16 * kl.row - 1), (int)a.key.c_token);
    }
#pragma unroll
    for (int i = 0; i < T::VN; ++i) {
      v_from[i] = vl.from(min(i * 64 + lane, 16 * vl.row - 1), (int)a.value.c_token);
    }
    const int d = w.value_at(c), b = MX ? d / 2 : d;
#pragma unroll
    for (int i = 0; i < 4; ++i) v_at[i] = 1024 * T::KN + vl.place(g * 4 + i, b / 16) * 16 + b % 16;
#pragma unroll
    for (int kp = 0; kp < KP; ++kp) {
      const int dk = w.key_at(kp), bk = MX ? dk / 2 : dk;
      k_at[kp] = kl.place(c, bk / 16) * 16 + bk % 16;
      // a row of codes has as many chunks as blocks
      if constexpr (MX) ks_at[kp] = T::kScales + (c * kl.row + dk / kMxBlock) * 4;
    }
    if constexpr (MX) {
#pragma unroll
      for (int i = 0; i < T::KS; ++i) {
        const int x = min(i * 64 + lane, 16 * kl.row - 1), r = (int)kl.by_row.quotient((uint32_t)x);
        ks_from[i] = (uint32_t)(r * (int)a.key.s_token + x - r * kl.row);
      }
#pragma unroll
      for (int i = 0; i < T::VS; ++i) {
        const int x = min(i * 64 + lane, 16 * vl.row - 1), r = (int)vl.by_row.quotient((uint32_t)x);
        vs_from[i] = (uint32_t)(r * (int)a.value.s_token + x - r * vl.row);
      }
      vs_at = T::kScales + 256 * T::KS + (g * 4 * vl.row + d / kMxBlock) * 4;
    } else {
      ks_from[0] = (uint32_t)((lane & 15) * (int)(lane < 32 ? a.key.s_token : a.value.s_token) * 4);
    }
    missing = false;
  }

  // Looks up the pages of the halves from tile t on; those without a live position stand for their
  // neighbours.
  __device__ __forceinline__ void look_up(int t) {
    base = t * 2;
    const int p = min(max(base + wave.lane, wave.first / 16), (wave.end - 1) / 16) * 16;
    const uint32_t column = a.by_page.quotient((uint32_t)p);
    const int found = row[column];
    const bool none = found < 0 || found >= a.pages;
    const int64_t page = none ? 0 : found, off = (uint32_t)p - column * (uint32_t)a.page_size;
    ko = page * a.key.c_page + off * a.key.c_token;
    vo = page * a.value.c_page + off * a.value.c_token;
    kso = (page * a.key.s_page + off * a.key.s_token) * (MX ? 1 : 4);
    vso = (page * a.value.s_page + off * a.value.s_token) * (MX ? 1 : 4);
    none_at = __builtin_amdgcn_ballot_w64(none);
  }

  static __device__ __forceinline__ int64_t of_lane(int64_t v, int i) {
    return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), i) << 32 |
                     (uint32_t)__builtin_amdgcn_readlane((int)v, i));
  }

  // Starts the T::kLoads loads of tile t into buffer `turn`.
  __device__ __forceinline__ void load(int t, int turn) {
    if (t * 2 >= base + 64) look_up(t);
    const int i = t * 2 - base;
    missing |= (none_at >> i & 3) != 0;
    const uint32_t dst = to + turn * T::kBytes;
    const uint8_t *ks[2], *vs[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t half = dst + h * T::kHalf;
      const uint8_t* kp = k_base + of_lane(ko, i + h);
      const uint8_t* vp = v_base + of_lane(vo, i + h);
      ks[h] = ks_base + of_lane(kso, i + h), vs[h] = vs_base + of_lane(vso, i + h);
#pragma unroll
      for (int x = 0; x < T::KN; ++x) tile_to_lds16(half + x * 1024, kp, k_from[x]);
#pragma unroll
      for (int x = 0; x < T::VN; ++x) tile_to_lds16(half + (T::KN + x) * 1024, vp, v_from[x]);
#pragma unroll
      for (int x = 0; x < T::KS; ++x) tile_to_lds1(half + T::kScales + x * 256, ks[h], ks_from[x]);
#pragma unroll
      for (int x = 0; x < T::VS; ++x) {
        tile_to_lds1(half + T::kScales + (T::KS + x) * 256, vs[h], vs_from[x]);
      }
    }
    if constexpr (!MX) {
      const bool high = (wave.lane & 16) != 0;
      const uint8_t *kp = high ? ks[1] : ks[0], *vp = high ? vs[1] : vs[0];
      tile_to_lds4(dst + 2 * T::kHalf, (wave.lane < 32 ? kp : vp) + ks_from[0]);
    }
  }

  __device__ __forceinline__ void read_value(const uint8_t* tile, int e, uint32_t* w) const {
    const uint8_t* p = tile + (e >> 2) * T::kHalf + v_at[e & 3];
    if constexpr (W::VB == 2) {
      w[0] = *reinterpret_cast<const uint16_t*>(p);
    } else {
      const auto x = *reinterpret_cast<const Pack<uint32_t, W::VW>*>(p);
#pragma unroll
      for (int n = 0; n < W::VW; ++n) w[n] = x.v[n];
    }
  }

  // Reads what has landed in buffer `turn`.
  __device__ __forceinline__ void fetch(int turn) {
    at = lds + turn * T::kBytes;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint8_t* half = at + h * T::kHalf;
#pragma unroll
      for (int kp = 0; kp < KP; ++kp) {
        const auto x = *reinterpret_cast<const Pack<uint32_t, W::KW>*>(half + k_at[kp]);
#pragma unroll
        for (int i = 0; i < W::KW; ++i) k[h][kp][i] = x.v[i];
        if constexpr (MX) kscale[h][kp] = mx_operand(*reinterpret_cast<const uint32_t*>(half + ks_at[kp]));
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (!W::LATE) read_value(at, h * 4 + i, v[h * 4 + i]);
        if constexpr (MX) {
          vscale[h * 4 + i] = mx_operand(
              *reinterpret_cast<const uint32_t*>(half + vs_at + i * (int)a.v_chunks.d * 4));
        }
      }
      if constexpr (!MX) {
        const float* f = reinterpret_cast<const float*>(at + 2 * T::kHalf);
        const auto x = *reinterpret_cast<const Pack<float, 4>*>(f + h * 16 + wave.g * 4);
        const auto y = *reinterpret_cast<const Pack<float, 4>*>(f + 32 + h * 16 + wave.g * 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) kscale[h][i] = x.v[i], vscale[h * 4 + i] = y.v[i];
      }
    }
    if constexpr (!MX) most = reinterpret_cast<const float*>(at + 2 * T::kHalf)[32 + (wave.lane & 31)];
  }

  __device__ __forceinline__ void key(int h, int kp, uint32_t* w) const {
#pragma unroll
    for (int i = 0; i < W::KW; ++i) w[i] = k[h][kp][i];
  }
  __device__ __forceinline__ float key_scale(int h, int kp) const { return kscale[h][kp]; }
  __device__ __forceinline__ void value(int e, uint32_t* w) const {
    if constexpr (W::LATE) {
      read_value(at, e, w);
    } else {
#pragma unroll
      for (int i = 0; i < W::VW; ++i) w[i] = v[e][i];
    }
  }
  __device__ __forceinline__ float value_scale(int e) const { return vscale[e]; }
  template <bool EDGE>
  __device__ __forceinline__ bool far(const bool* live) const {  // slots that are not live hold anything
    uint32_t most = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      most = max(most, EDGE && !live[e] ? 0u : __builtin_bit_cast(uint32_t, vscale[e]));
    }
    return most >= kMxFarByte << 23;
  }
  __device__ __forceinline__ float ks(int e) const { return kscale[e >> 2][e & 3]; }
  __device__ __forceinline__ float vs(int e) const { return vscale[e]; }
  __device__ __forceinline__ float most_vs() const { return most; }
};

template <class E, int FMT, int KP, int VD>
__global__ void __launch_bounds__(kAttWaves * 64, att_resident(std::is_same_v<E, F32>, FMT, KP, VD, true))
k_kv_attention_lines(AttArgs a) {
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds_bytes[];  // [waves][2] tiles
  using T = LdsTile<FMT, KP, VD>;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  uint32_t share;
  int head, block;
  att_place(a, (blockIdx.x >> 3) * kAttWaves + wave, &share, &head, &block);
  const int head0 = head * a.group + block * kTileRows;
  const int rows = min(kTileRows, a.group - block * kTileRows);
  AttWalk walk(a, share, head == 0 && block == 0);
  AttChunk c;
  using W = AttWave<E, FMT, KP, VD>;
  while (walk.next(&c)) {
    W w(a, c, head0, rows);
    LdsSource<E, FMT, KP, VD> src(
        a, w, c, head, lds_bytes + wave * (2 * T::kBytes),
        (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds_bytes +
            wave * (2 * T::kBytes));
    // queries and pages are on their way together; the queries are taken apart while tiles are
    if (c.tiles > 0) src.look_up(c.tile);
    w.settle();
    wait_lds();  // of the segment before: nothing of it is in flight when its buffers are filled again
    if (c.tiles > 0) src.load(c.tile, 0);
    if (c.tiles > 1) src.load(c.tile + 1, 1);
    w.begin(rows);
    if (c.tiles > 0) {
      const int last = c.tile + c.tiles - 1;
      for (int t = c.tile, turn = 0; t <= last; ++t, turn ^= 1) {
        // a tile is taken to registers whole, so that the loads of the one after the next follow at once
        if (t < last) wait_loads<T::kLoads>();
        else wait_loads<0>();
        src.fetch(turn);
        if constexpr (W::LATE) w.tile(src, t);
        wait_lds();
        if (t + 2 <= last) src.load(t + 2, turn);
        if constexpr (!W::LATE) w.tile(src, t);
      }
    }
    w.write(c, head0, rows, src.missing);
  }
}

// ---- Codes straight to registers, at any alignment and in pages of any size.
template <class E, int FMT, int KP, int VD>
struct RegisterSource {
  using W = AttWave<E, FMT, KP, VD>;
  static constexpr bool MX = W::MX;
  const AttArgs& a;
  const W& wave;
  const int32_t* row;
  const uint8_t *k_base, *v_base;
  const void *ks_base, *vs_base;
  int v_at;
  uint32_t k_sel[KP], v_sel;
  int base, found;  // columns [base, base + 64) of the table's row: lane i knows the page of base + i
  bool missing;
  uint32_t k[2][KP][W::KW], v[W::LATE ? 1 : 8][W::VW], kb[2], vb[2];
  int64_t v_from;          // of position lane % 32
  float k_scale, v_scale;  // of position lane % 32

  __device__ __forceinline__ RegisterSource(const AttArgs& args, const W& w, const AttChunk& ch,
                                            int head)
      : a(args), wave(w) {
    row = a.table + ch.sequence * a.table_stride;
    k_base = a.key.codes + head * a.key.c_head;
    v_base = a.value.codes + head * a.value.c_head;
    const int es = MX ? 1 : 4;
    ks_base = static_cast<const uint8_t*>(a.key.scales) + head * a.key.s_head * es;
    vs_base = static_cast<const uint8_t*>(a.value.scales) + head * a.value.s_head * es;
    const int d = w.value_at(w.c);
    v_at = MX ? d / 2 : d;
    v_sel = MX ? scale_selector(d / kMxBlock, a.value.dim / kMxBlock) : 0;
#pragma unroll
    for (int kp = 0; kp < KP; ++kp) {
      k_sel[kp] = MX ? scale_selector(w.key_at(kp) / kMxBlock, a.key.dim / kMxBlock) : 0;
    }
    missing = false;
  }

  __device__ __forceinline__ void look_up(uint32_t column) {
    base = __builtin_amdgcn_readfirstlane((int)column);
    found = row[min(base + wave.lane, (int)a.by_page.quotient((uint32_t)wave.end - 1))];
    if (found >= a.pages) found = -1;
  }

  // Loads tile t; positions before the first or behind the last stand for those.
  __device__ __forceinline__ void load(int t) {
    const int p = min(max(t * kAttTile + (wave.lane & 31), wave.first), wave.end - 1);
    const uint32_t column = a.by_page.quotient((uint32_t)p);
    if (__builtin_amdgcn_readlane((int)column, 31) >= base + 64) look_up(column);
    const int g = (int)from_lane((uint32_t)found, (int)column - base);
    missing |= __builtin_amdgcn_ballot_w64(g < 0) != 0;
    const int64_t page = max(g, 0), off = (uint32_t)p - column * (uint32_t)a.page_size;
    const int64_t ko = page * a.key.c_page + off * a.key.c_token;
    const int64_t vo = page * a.value.c_page + off * a.value.c_token;
    const int64_t kso = page * a.key.s_page + off * a.key.s_token;
    const int64_t vso = page * a.value.s_page + off * a.value.s_token;
    if constexpr (MX) {
      load_scales8(kb, static_cast<const uint8_t*>(ks_base) + kso, a.key.dim / kMxBlock);
      load_scales8(vb, static_cast<const uint8_t*>(vs_base) + vso, a.value.dim / kMxBlock);
    } else {
      k_scale = static_cast<const float*>(ks_base)[kso];
      v_scale = static_cast<const float*>(vs_base)[vso];
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint8_t* p = k_base + from_lane64(ko, h * 16 + wave.c);
#pragma unroll
      for (int kp = 0; kp < KP; ++kp) {
        const int d = wave.key_at(kp);
        load_bytes<W::KW * 4>(k[h][kp], p + (MX ? d / 2 : d));
      }
    }
    v_from = vo;
    if constexpr (!W::LATE) {
#pragma unroll
      for (int e = 0; e < 8; ++e) read_value(e, v[e]);
    }
  }
  __device__ __forceinline__ void read_value(int e, uint32_t* w) const {
    load_bytes<W::VB>(w, v_base + from_lane64(v_from, wave.position(e)) + v_at);
  }

  __device__ __forceinline__ void key(int h, int kp, uint32_t* w) const {
#pragma unroll
    for (int i = 0; i < W::KW; ++i) w[i] = k[h][kp][i];
  }
  __device__ __forceinline__ float key_scale(int h, int kp) const {
    uint32_t b[2];
    b[0] = from_lane(kb[0], h * 16 + wave.c);
    b[1] = KP > 2 ? from_lane(kb[1], h * 16 + wave.c) : 0;
    return scale_operand(b, k_sel[kp]);
  }
  __device__ __forceinline__ void value(int e, uint32_t* w) const {
    if constexpr (W::LATE) {
      read_value(e, w);
    } else {
#pragma unroll
      for (int i = 0; i < W::VW; ++i) w[i] = v[e][i];
    }
  }
  __device__ __forceinline__ float value_scale(int e) const {
    uint32_t b[2];
    b[0] = from_lane(vb[0], wave.position(e));
    b[1] = VD > 8 ? from_lane(vb[1], wave.position(e)) : 0;
    return scale_operand(b, v_sel);
  }
  template <bool EDGE>
  __device__ __forceinline__ bool far(const bool*) const {  // of position lane % 32, a live one
    const uint32_t top = vb[0] & vb[0] << 1, next = VD > 8 ? vb[1] & vb[1] << 1 : 0;
    return ((top | next) & 0x80808080u) != 0;
  }
  __device__ __forceinline__ float ks(int e) const { return from_lane_f(k_scale, wave.position(e)); }
  __device__ __forceinline__ float vs(int e) const { return from_lane_f(v_scale, wave.position(e)); }
  __device__ __forceinline__ float most_vs() const { return v_scale; }
};

template <class E, int FMT, int KP, int VD>
__global__ void __launch_bounds__(kAttWaves * 64, att_resident(std::is_same_v<E, F32>, FMT, KP, VD, false))
k_kv_attention_tiles(AttArgs a) {
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  uint32_t share;
  int head, block;
  att_place(a, (blockIdx.x >> 3) * kAttWaves + wave, &share, &head, &block);
  const int head0 = head * a.group + block * kTileRows;
  const int rows = min(kTileRows, a.group - block * kTileRows);
  AttWalk walk(a, share, head == 0 && block == 0);
  AttChunk c;
  while (walk.next(&c)) {
    AttWave<E, FMT, KP, VD> w(a, c, head0, rows);
    RegisterSource<E, FMT, KP, VD> src(a, w, c, head);
    // queries and pages are on their way together
    if (c.tiles > 0) src.look_up(a.by_page.quotient((uint32_t)max(c.tile * kAttTile, c.first)));
    w.settle();
    w.begin(rows);
    for (int t = c.tile; t < c.tile + c.tiles; ++t) {
      src.load(t);
      w.tile(src, t);
    }
    w.write(c, head0, rows, src.missing);
  }
}

// The kernels' head sizes: keys of up to 64 KP and values of up to 16 VD elements, at least a unit of each.
struct TileShape {
  int kp, vd;
};
constexpr TileShape kTileShapes[] = {{1, 4}, {2, 8}, {3, 8}, {4, 16}};
// Whether a CU holds two workgroups of the kernel through LDS, by registers and LDS.
template <class E, int FMT, int I>
constexpr bool kTwoResident =
    att_resident(std::is_same_v<E, F32>, FMT, kTileShapes[I].kp, kTileShapes[I].vd, true) == 2 &&
    2 * LdsTile<FMT, kTileShapes[I].kp, kTileShapes[I].vd>::kGroup <= 160 * 1024;
template <int FMT, int I>
constexpr int kTileBytes = LdsTile<FMT, kTileShapes[I].kp, kTileShapes[I].vd>::kBytes;

// Launches the kernel of shape `shape` (an index above) on the sequences' chunks.
int attention_tiles_int8(int shape, bool lines, mcop_dtype dtype, const AttArgs& a, dim3 grid,
                         hipStream_t st);
int attention_tiles_fp8(int shape, bool lines, mcop_dtype dtype, const AttArgs& a, dim3 grid,
                        hipStream_t st);
int attention_tiles_mxfp4(int shape, bool lines, mcop_dtype dtype, const AttArgs& a, dim3 grid,
                          hipStream_t st);

template <int FMT, class E, int KP, int VD>
void attention_tiles_of(bool lines, const AttArgs& a, dim3 grid, hipStream_t st) {
  const dim3 block(kAttWaves * 64);
  if (lines) {
    hipLaunchKernelGGL((k_kv_attention_lines<E, FMT, KP, VD>), grid, block, (LdsTile<FMT, KP, VD>::kGroup), st,
                       a);
  } else {
    hipLaunchKernelGGL((k_kv_attention_tiles<E, FMT, KP, VD>), grid, block, 0, st, a);
  }
}
template <int FMT>
int attention_tiles_for(int shape, bool lines, mcop_dtype dtype, const AttArgs& a, dim3 grid,
                        hipStream_t st) {
  auto by_shape = [&](auto e) {
    using E = decltype(e);
    switch (shape) {
      case 0: attention_tiles_of<FMT, E, 1, 4>(lines, a, grid, st); break;
      case 1: attention_tiles_of<FMT, E, 2, 8>(lines, a, grid, st); break;
      case 2: attention_tiles_of<FMT, E, 3, 8>(lines, a, grid, st); break;
      default: attention_tiles_of<FMT, E, 4, 16>(lines, a, grid, st);
    }
  };
  if (dtype == MCOP_BF16) by_shape(BF16());
  else if (dtype == MCOP_F16) by_shape(F16());
  else by_shape(F32());
  return check_launch("kv_cache_attention");
}

}  // namespace mcop
