// kv_attention.h -- attention of one new token a sequence over the quantized paged cache: the arguments,
// the split of the sequences' lengths over workgroups, and how their parts are written.
//
// For sequence b, query head h and the positions P = [first, n) of the sequence (n = seq_lens[b], first =
// n - window or 0), with k_j = q_j * s_j and v_j the dequantized vectors of h's key head:
//   s_j = scale * <q, k_j>,   o = sum_j e^(s_j) v_j / sum_j e^(s_j),   lse = log sum_j e^(s_j)
// in one pass over P with the running maximum m and sum l of the softmax (in powers of two: s_j times
// log2 e).  Parts of P that were walked apart are joined by  m = max m_i,  l = sum l_i 2^(m_i - m),
// o = sum o_i 2^(m_i - m).  The o_i of int8 and fp8 caches are held in units of 2^e, the exponent of the
// largest value scale seen, so that neither a weight times a scale nor their sum leaves fp32's range where
// the values themselves do not.  An empty P gives o = 0 and lse = -inf; a position of P without a page of the
// cache makes the sequence's rows NaN.
//
// Work is split by tiles of 32 positions.  The lengths are on the device, so every workgroup finds its
// own share: all tiles of all sequences over the number of chunks aimed at (`target`) is a chunk's
// length, a sequence takes as many chunks as that asks for, and the grid has room for all (at most
// target + sequences).  So one long sequence among short ones fills the card as equal ones do, and no
// call needs lengths on the host.  Sequences of one chunk are written at once; the others write parts
// (at most 2 * target chunks, since a split sequence has more tiles than a chunk) that a second kernel
// joins, in chunk order: results do not depend on timing.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kv_side.h"
#include "rowkern.h"

namespace mcop {

constexpr int kAttTile = 32;      // positions of a tile
constexpr int kAttWaves = 4;      // of a workgroup, which share out a chunk's tiles
constexpr int kAttLeastTiles = 1; // of a chunk
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct AttArgs {
  KvSide key, value;  // plain: the queries, the outputs
  float* lse;         // [sequences][query heads], or null
  const int32_t* table;
  int64_t table_stride;
  int columns;
  const int32_t* lens;
  int sequences;
  int64_t pages;
  int page_size;
  Divisor by_page;
  int heads, group, query_heads;  // key heads, query heads of each, query heads
  int row_blocks;                 // waves (or workgroups) that a key head's query heads take
  Divisor by_inner, by_blocks;    // heads * row_blocks, row_blocks
  Divisor k_chunks, v_chunks;     // chunks of 16 bytes of a key, of a value
  int window;
  int target;
  float scale;    // times log2 e
  float* parts;   // [2 * target][query heads][value.dim]
  float* sums;    // [2 * target][query heads][4]: m, l, e
  int32_t* plan;  // the number of split sequences; then of each: sequence, first part, parts
};

struct AttChunk {
  int sequence;
  int first, end;     // the sequence's positions
  int tile, tiles;    // first tile and tiles of this chunk
  int index, count;   // of the sequence's chunks
  int part;           // where its part goes (count > 1)
  bool missing;       // longer than its row of the table
};

__device__ __forceinline__ int64_t att_capacity(const AttArgs& a) {
  const int64_t c = (int64_t)a.columns * a.page_size;
  return c < INT32_MAX ? c : INT32_MAX;
}
__device__ __forceinline__ int att_first(const AttArgs& a, int n) {
  return a.window > 0 && n > a.window ? n - a.window : 0;
}
// Tiles that hold a sequence's positions; 0 for one that is empty or longer than its table.
__device__ __forceinline__ uint32_t att_tiles(const AttArgs& a, int n) {
  if (n <= 0 || n > att_capacity(a)) return 0;
  return ((uint32_t)n + kAttTile - 1) / kAttTile - (uint32_t)att_first(a, n) / kAttTile;
}

// Inclusive sums over the wave's lanes, by register moves: within rows of 16, then across them.
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
  v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xf, 0xf, false);  // row_shr:1
  v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xf, 0xf, false);
  v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xf, 0xf, false);
  v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xf, 0xf, false);
  v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, false);  // row_bcast:15
  v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, false);  // row_bcast:31
  return v;
}
__device__ __forceinline__ uint32_t wave_total(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_readlane((int)wave_scan(v), 63);
}
// The same of values below 2^44, 22 bits at a time.
__device__ __forceinline__ uint64_t wave_total64(uint64_t v) {
  return ((uint64_t)wave_total((uint32_t)(v >> 22)) << 22) + wave_total((uint32_t)v & 0x3fffff);
}

// The chunk of number `flat`; false past the last one.  A wave works together, 64 sequences at a time.
// `plans`: this wave writes the plan of the sequence whose first chunk it finds.
__device__ __forceinline__ bool find_chunk(const AttArgs& a, uint32_t flat, bool plans, AttChunk* c) {
  const int lane = (int)threadIdx.x & 63;
  const int n0 = lane < a.sequences ? a.lens[lane] : 0;
  uint64_t total = att_tiles(a, n0);
  for (int i = 64; i < a.sequences; i += 64) {
    if (i + lane < a.sequences) total += att_tiles(a, a.lens[i + lane]);
  }
  total = wave_total64(total);
  uint32_t per = kAttLeastTiles;
  if (total > (uint64_t)a.target * kAttLeastTiles) {
    per = total >> 31 ? (uint32_t)min((total + a.target - 1) / a.target, (uint64_t)1 << 26)
                      : ((uint32_t)total - 1) / (uint32_t)a.target + 1;
  }
  uint32_t before = 0, parts_before = 0;  // chunks of earlier sequences, and their parts
  int splits = 0;
  bool found = false;
  for (int i = 0; i < a.sequences; i += 64) {
    const int n = i == 0 ? n0 : (i + lane < a.sequences ? a.lens[i + lane] : 0);
    const uint32_t t = att_tiles(a, n);
    const uint32_t k = i + lane >= a.sequences ? 0 : t <= per ? 1 : (t - 1) / per + 1;
    const uint32_t upto = wave_scan(k) + before, parts = wave_scan(k > 1 ? k : 0) + parts_before;
    const uint64_t split = __builtin_amdgcn_ballot_w64(k > 1);
    const uint64_t hit = __builtin_amdgcn_ballot_w64(k > 0 && upto > flat);
    if (!found && hit != 0) {
      found = true;
      const int at = __builtin_ctzll(hit);
      const uint32_t tiles = (uint32_t)__builtin_amdgcn_readlane((int)t, at);
      c->sequence = i + at;
      c->end = __builtin_amdgcn_readlane(n, at);
      c->count = __builtin_amdgcn_readlane((int)k, at);
      c->index = (int)flat - __builtin_amdgcn_readlane((int)(upto - k), at);
      c->part = __builtin_amdgcn_readlane((int)(parts - k), at) + c->index;
      c->missing = c->end > att_capacity(a);
      c->first = att_first(a, c->end);
      const uint32_t each = tiles / (uint32_t)c->count, more = tiles % (uint32_t)c->count;
      const uint32_t x = (uint32_t)c->index;
      c->tile = (int)((uint32_t)c->first / kAttTile + x * each + min(x, more));
      c->tiles = (int)(each + (x < more ? 1 : 0));
      if (plans && c->count > 1 && c->index == 0 && lane == 0) {
        const int rank = splits + (int)__builtin_popcountll(split & (((uint64_t)1 << at) - 1));
        a.plan[1 + 3 * rank] = c->sequence;
        a.plan[2 + 3 * rank] = c->part;
        a.plan[3 + 3 * rank] = c->count;
      }
      // the first chunk's wave goes on to count the split sequences
      if (!plans || flat != 0) return true;
    }
    splits += (int)__builtin_popcountll(split);
    before = (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
    parts_before = (uint32_t)__builtin_amdgcn_readlane((int)parts, 63);
  }
  if (plans && flat == 0 && lane == 0) a.plan[0] = splits;
  return found;
}

// A wave's place where every wave takes a chunk of one key head and block: heads and blocks of a chunk are
// neighbours, so that what lies together in the cache is read together, and chunks go round the dies.
__device__ __forceinline__ void att_wave_place(const AttArgs& a, uint32_t wave, uint32_t* flat, int* head, int* block) {
  // inner padded to whole workgroups
  const uint32_t die = blockIdx.x & 7, i = (blockIdx.x >> 3) * kAttWaves + wave;
  const uint32_t row = a.by_inner.quotient(i), inner = i - row * a.by_inner.d;
  *flat = row * 8 + die;
  *head = (int)a.by_blocks.quotient(inner);
  *block = (int)(inner - (uint32_t)*head * (uint32_t)a.row_blocks);
}

// Workgroup -> (chunk, key head, block of its query heads).  Workgroups go round the eight dies in turn,
// so those of one chunk, which share its scales' cache lines, are put on the same die.
__device__ __forceinline__ void att_place(const AttArgs& a, uint32_t* flat, int* head, int* block) {
  const uint32_t die = blockIdx.x & 7, i = blockIdx.x >> 3;
  const uint32_t row = a.by_inner.quotient(i), inner = i - row * a.by_inner.d;
  *flat = row * 8 + die;
  *head = (int)a.by_blocks.quotient(inner);
  *block = (int)(inner - (uint32_t)*head * (uint32_t)a.row_blocks);
}

// 2^(m - top), 1 where both are -inf.
__device__ __forceinline__ float att_weight(float m, float top) {
  return __builtin_amdgcn_exp2f(m - (top == -__builtin_inff() ? 0.0f : top));
}

// The unit that outputs are held in for a largest value scale: its exponent, where 2^-e is normal.
constexpr int kAttNoUnit = -126;
__device__ __forceinline__ int att_unit(float scale) {
  const int e = (int)((__builtin_bit_cast(uint32_t, scale) >> 23) & 255) - 127;
  return e < kAttNoUnit ? kAttNoUnit : (e > 126 ? 126 : e);
}
// 2^e for e of 0 down to -252.
__device__ __forceinline__ float att_power(int e) { return __builtin_ldexpf(1.0f, e); }

// A joined element of a row: its output, 0 for a row without weight.
__device__ __forceinline__ float att_value(float o, float l, int e) {
  return l == 0.0f ? 0.0f : __builtin_ldexpf(o / l, e);
}
__device__ __forceinline__ float att_lse(float m, float l) {
  return l == 0.0f ? -__builtin_inff() : (m + __builtin_amdgcn_logf(l)) * kLn2;
}

// Joins the waves' parts of `rows` query heads from LDS (m, l [kAttWaves][stride_m], e [kAttWaves], o
// [kAttWaves][stride_r][stride_o]) and writes the outputs of query heads head0.. (or, of a split sequence,
// its part) at elements d0.. of the value.
template <class E>
__device__ __forceinline__ void att_write(const AttArgs& a, const AttChunk& c, int head0, int rows,
                                          int d0, int width, const float* m, const float* l,
                                          const int* e, const float* o, int stride_m,
                                          int stride_r, int stride_o) {
  int unit = e[0];
#pragma unroll
  for (int w = 1; w < kAttWaves; ++w) unit = max(unit, e[w]);
  for (int r = 0; r < rows; ++r) {
    float top = -__builtin_inff();
#pragma unroll
    for (int w = 0; w < kAttWaves; ++w) top = __builtin_fmaxf(top, m[w * stride_m + r]);
    float f[kAttWaves], sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kAttWaves; ++w) {
      f[w] = att_weight(m[w * stride_m + r], top);
      sum += l[w * stride_m + r] * f[w];
      f[w] *= att_power(e[w] - unit);
    }
    if (c.missing) sum = __builtin_nanf("");
    const int head = head0 + r;
    for (int d = (int)threadIdx.x; d < width; d += kAttWaves * 64) {
      float v = 0.0f;
#pragma unroll
      for (int w = 0; w < kAttWaves; ++w) v += o[(w * stride_r + r) * stride_o + d] * f[w];
      if (c.count > 1) {
        a.parts[((int64_t)c.part * a.query_heads + head) * a.value.dim + d0 + d] = v;
      } else {
        static_cast<typename E::S*>(a.value.plain)[c.sequence * a.value.p_token +
                                                   head * a.value.p_head + d0 + d] =
            E::from_f(att_value(v, sum, unit));
      }
    }
    if (threadIdx.x == 0 && d0 == 0) {
      if (c.count > 1) {
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

}  // namespace mcop
