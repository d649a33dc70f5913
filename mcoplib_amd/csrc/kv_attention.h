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
// the values themselves do not; those of 4-bit caches in units of 2^48 from the first block scale of 2^65 or more
// on (kMxUnit).  An empty P gives o = 0 and lse = -inf; a position of P without a page of the
// cache makes the sequence's rows NaN.
//
// Work is split by tiles of 32 positions.  The lengths are on the device, so every wave finds its own
// share: the tiles of all sequences one after the other, cut into `target` equal shares, whatever the
// sequences' lengths (one tile at least for each, also an empty one).  A sequence's start, where a wave waits for
// its queries, its pages and its first tile in turn, counts as kAttStart tiles more: 64 ragged sequences of 131072
// in all took 71 us without, 66 so, sorted by length 81 and 66, 300 of 30 beside 64 of 1500 87 and 68; 16 equal
// ones of 8192 of a 4-bit cache, whose shares were whole eighths, 51 and 53.  A share may end one sequence, hold
// some whole and begin another: whole ones are written at once, the others as parts, of which a share has
// two at most.  A second kernel joins each sequence's parts in order: results do not depend on timing.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kv_side.h"
#include "rowkern.h"
#include "wave_scan.h"

namespace mcop {

constexpr int kAttTile = 32;  // positions of a tile
constexpr int kAttWaves = 4;  // of a workgroup
constexpr int kAttStart = 2;  // tiles that the start of a sequence counts for in the split
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
  int32_t* plan;  // split sequences, tiles a share; then of each: sequence, its first tile of all, its end
};

// The tiles of one sequence that a share holds.
struct AttChunk {
  int sequence;
  int first, end;     // the sequence's positions
  int tile, tiles;
  int part;           // where its part goes; -1: it is the whole sequence
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

// Walks the sequences of share `share`; a wave works together, 64 sequences at a time.
struct AttWalk {
  const AttArgs& a;
  const int lane;
  const bool plans;  // this wave writes the plan of the sequences that begin in its share
  const uint32_t share;
  uint32_t per, at, to, total;  // tiles a share; those of this share
  int block, splits;            // the 64 sequences in the lanes; split ones before them
  int n;
  uint32_t tiles, from;         // of the lane's sequence
  uint64_t split;

  __device__ __forceinline__ AttWalk(const AttArgs& args, uint32_t number, bool plan)
      : a(args), lane((int)threadIdx.x & 63), plans(plan), share(number) {
    n = lane < a.sequences ? a.lens[lane] : 0;
    uint32_t t = lane < a.sequences ? max(att_tiles(a, n), 1u) + kAttStart : 0;
    for (int i = 64; i < a.sequences; i += 64) {
      if (i + lane < a.sequences) t += max(att_tiles(a, a.lens[i + lane]), 1u) + kAttStart;
    }
    total = wave_total(t);
    per = (total - 1) / (uint32_t)a.target + 1;
    at = share < (uint32_t)a.target ? share * per : total;
    to = min(at + per, total);
    block = 0, splits = 0;
    enter(0);
  }
  // The sequences from `block` on to the lanes; `before`: tiles of those before.
  __device__ __forceinline__ void enter(uint32_t before) {
    tiles = block + lane < a.sequences ? max(att_tiles(a, n), 1u) : 0;
    from = wave_scan(tiles > 0 ? tiles + kAttStart : 0) - tiles + before;
    split = __builtin_amdgcn_ballot_w64(tiles > 0 && from / per != (from + tiles - 1) / per);
  }
  __device__ __forceinline__ uint32_t end_of_block() const {
    return (uint32_t)__builtin_amdgcn_readlane((int)(from + tiles), 63);
  }
  // The share's next sequence; false behind the last.
  __device__ __forceinline__ bool next(AttChunk* c) {
    if (at >= to) return false;
    while (at >= end_of_block()) {
      const uint32_t before = end_of_block();
      splits += (int)__builtin_popcountll(split);
      block += 64;
      n = block + lane < a.sequences ? a.lens[block + lane] : 0;
      enter(before);
    }
    const int i = __builtin_ctzll(__builtin_amdgcn_ballot_w64(tiles > 0 && from + tiles > at));
    const uint32_t begin = (uint32_t)__builtin_amdgcn_readlane((int)from, i);
    at = max(at, begin);
    if (at >= to) return false;  // the share ends in the sequence's start
    const uint32_t all = (uint32_t)__builtin_amdgcn_readlane((int)tiles, i);
    const uint32_t stop = min(to, begin + all);
    c->sequence = block + i;
    c->end = __builtin_amdgcn_readlane(n, i);
    c->missing = c->end > att_capacity(a);
    c->first = att_first(a, c->end);
    c->tile = (int)((uint32_t)c->first / kAttTile + at - begin);
    c->tiles = c->missing || c->end <= 0 ? 0 : (int)(stop - at);
    const bool whole = stop - at == all;
    c->part = whole ? -1 : (int)(2 * share + (at > share * per ? 1 : 0));
    if (plans && lane == 0) {
      if (!whole && at == begin) {
        int32_t* p = a.plan + 2 + 3 * (splits + (int)__builtin_popcountll(split & (((uint64_t)1 << i) - 1)));
        p[0] = c->sequence, p[1] = (int)begin, p[2] = (int)(begin + all);
      }
      if (stop == total) {  // all sequences are behind
        a.plan[0] = splits + (int)__builtin_popcountll(split);
        a.plan[1] = (int)per;
      }
    }
    at = stop;
    return true;
  }
};

// The share, key head and block of its query heads of worker `i` of the die (a wave or a workgroup; workgroups
// go round the eight dies in turn): the heads and blocks of a share are neighbours on one die, so that
// what lies together in the cache is read together.
__device__ __forceinline__ void att_place(const AttArgs& a, uint32_t i, uint32_t* share, int* head,
                                          int* block) {
  const uint32_t row = a.by_inner.quotient(i), inner = i - row * a.by_inner.d;
  *share = row * 8 + (blockIdx.x & 7);
  *head = (int)a.by_blocks.quotient(inner);
  *block = (int)(inner - (uint32_t)*head * (uint32_t)a.row_blocks);
}

// 2^(m - top), 0 where both are -inf.
__device__ __forceinline__ float att_weight(float m, float top) {
  return __builtin_amdgcn_exp2f(m - (top == -__builtin_inff() ? 0.0f : top));
}

// The unit that outputs are held in for a largest value scale: its exponent, where 2^-e is normal.
constexpr int kAttNoUnit = -126;
__device__ __forceinline__ int att_unit(float scale) {
  const int e = (int)((__builtin_bit_cast(uint32_t, scale) >> 23) & 255) - 127;
  return e < kAttNoUnit ? kAttNoUnit : (e > 126 ? 126 : e);
}
// 4-bit values: up to 6 times a block scale of 2^127, weights of at most 2^8, fewer than 2^31 of them.  Sums of scales
// below 2^65 stay below 2^107; in units of 2^48 those of any scale below 2^121, and a weight that counts beside
// others, of 2^-48 and more, keeps all terms of its products.
constexpr int kMxUnit = 48;
constexpr uint32_t kMxFarByte = 127 + 65;  // the two leading bits of a scale byte
// 2^e for e of 0 down to -252.
__device__ __forceinline__ float att_power(int e) { return __builtin_ldexpf(1.0f, e); }

// A joined element of a row: its output, 0 for a row without weight.
__device__ __forceinline__ float att_value(float o, float l, int e) {
  return l == 0.0f ? 0.0f : __builtin_ldexpf(o / l, e);
}
__device__ __forceinline__ float att_lse(float m, float l) {
  return l == 0.0f ? -__builtin_inff() : (m + __builtin_amdgcn_logf(l)) * kLn2;
}

}  // namespace mcop
