// mxfp4_mm.hip -- product of two operands of 4-bit blocks (mxfp4.h) on the matrix units:
//   out[m, n] = b(sum_k A[m, k] B[n, k] (+ bias[n])), summed in fp32.
//
// A scaled matrix instruction takes one block of each operand a lane -- 16 bytes of codes and a byte of
// a scale register -- and multiplies by both scales as it sums, so codes go from memory to the
// matrix unit as they are.  Which K a lane's block has is free as long as both operands agree.  The
// weights are the first operand: a lane then holds four consecutive n of one m.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdio>

#include "../../include/mcop_norm.h"
#include "launch_trace.h"
#include "mcop_testing.h"
#include "mxfp4.h"

namespace mcop {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kFp4 = 4;  // operand format of the matrix instructions

// VEC values of a row from column n on, of those inside its N: one store at any alignment, but at the
// row's end (memory takes vectors at any address).
template <class S, int VEC, bool NT>
__device__ __forceinline__ void store_row(S* to, const Pack<S, VEC>& v, int n, int N, bool whole) {
  if (whole) {
    if constexpr (NT) st_nt<S, VEC>(to, v);
    else st<S, VEC>(to, v);
  } else if (n + VEC <= N) {
    __builtin_memcpy(to, &v, sizeof(v));
  } else {
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      if (n + e < N) to[e] = v.v[e];
    }
  }
}

__device__ __forceinline__ i32x8 fp4_operand(i32x4 v) {
  return __builtin_shufflevector(v, v, 0, 1, 2, 3, -1, -1, -1, -1);
}

// The 16 (4 KS) scale bytes of a row from block b on, as dwords.  WHOLE: all inside the row; otherwise
// zero past its end (where the codes count as zero as well), by loads that stay inside it.
template <int KS, bool WHOLE>
__device__ __forceinline__ void scale_dwords(uint32_t (&v)[KS], const uint8_t* row, int b,
                                             int blocks) {
  if constexpr (WHOLE) {
    __builtin_memcpy(v, row + b, 4 * KS);
  } else {
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      v[s] = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t x = row[min(b + 4 * s + e, blocks - 1)];
        v[s] |= b + 4 * s + e < blocks ? x << (8 * e) : 0u;
      }
    }
  }
}

// Few rows: a workgroup makes 16 rows x 16 columns of the output, its W waves every W-th chunk of
// KS * 128 along K, straight from memory to registers, one chunk ahead; the partial sums meet in LDS
// and are added in the waves' order.  It has the shortest way to its first product, and takes operands
// of any size; what bounds it then are its loads, 64 bytes of each of 16 rows, which a CU's cache answers
// at 36 bytes a nanosecond (whole lines: 120).
// In instruction s of a chunk the lane of group g = lane / 16 has block 4 s + g, so that a load takes 64
// bytes in a row of 16 rows; its scale is byte g of the row's dword s.
template <class E, int W, int KS>
__global__ void __launch_bounds__(64 * W)
k_mxfp4_mm_rows(typename E::S* __restrict__ out, const uint8_t* __restrict__ a,
                const uint8_t* __restrict__ as, const uint8_t* __restrict__ b,
                const uint8_t* __restrict__ bs, const typename E::S* __restrict__ bias, int M, int N,
                int blocks) {
  using S = typename E::S;
  constexpr int CHUNK = 4 * KS;  // blocks
  __shared__ f32x4 part[W][64];
  const int lane = (int)threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  const int n0 = (int)blockIdx.x * 16, m0 = (int)blockIdx.y * 16;
  // b's row and a's; rows past an operand's end repeat its last
  const int64_t row[2] = {min(n0 + r, N - 1), min(m0 + r, M - 1)};
  const uint8_t* code_row[2] = {b + (row[0] * blocks + g) * 16, a + (row[1] * blocks + g) * 16};
  const uint8_t* scale_row[2] = {bs + row[0] * blocks, as + row[1] * blocks};
  f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
  struct Chunk {
    i32x4 code[2][KS];
    uint32_t scale[2][KS];
  };
  auto load = [&](Chunk& c, int k, auto whole) {  // the chunk from block k on
    constexpr bool WHOLE = decltype(whole)::value;
#pragma unroll
    for (int o = 0; o < 2; ++o) {
      scale_dwords<KS, WHOLE>(c.scale[o], scale_row[o], k, blocks);
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const int64_t at = (int64_t)(k + 4 * s) * 16;
        if constexpr (WHOLE) {
          if (o == 0) {
            c.code[o][s] = __builtin_nontemporal_load(
                reinterpret_cast<const i32x4*>(code_row[o] + at));
          } else {
            c.code[o][s] = *reinterpret_cast<const i32x4*>(code_row[o] + at);
          }
        } else {
          c.code[o][s] = i32x4{0, 0, 0, 0};
          if (k + 4 * s + g < blocks) {
            c.code[o][s] = *reinterpret_cast<const i32x4*>(code_row[o] + at);
          }
        }
      }
    }
  };
  auto multiply = [&](const Chunk& c) {
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      sum = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
          fp4_operand(c.code[0][s]), fp4_operand(c.code[1][s]), sum, kFp4, kFp4, 0,
          (int)(c.scale[0][s] >> (8 * g)), 0, (int)(c.scale[1][s] >> (8 * g)));
    }
  };
  const int whole = blocks / CHUNK;
  Chunk even, odd;
  int c = wave;
  // The order is kept as written: a chunk's loads all go out before the products of the one before (the
  // compiler would put each next to its use, and wait for it there).
  auto apart = []() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
  };
  if (c < whole) {
    load(even, c * CHUNK, std::true_type());
    while (true) {
      load(odd, min(c + W, whole - 1) * CHUNK, std::true_type());
      apart();
      multiply(even);
      apart();
      if ((c += W) >= whole) break;
      load(even, min(c + W, whole - 1) * CHUNK, std::true_type());
      apart();
      multiply(odd);
      apart();
      if ((c += W) >= whole) break;
    }
  }
  if (whole * CHUNK < blocks && wave == whole % W) {  // what is left of the rows
    load(even, whole * CHUNK, std::false_type());
    multiply(even);
  }
  part[wave][lane] = sum;
  __syncthreads();
  if (wave != 0) return;
  f32x4 v = part[0][lane];
#pragma unroll
  for (int w = 1; w < W; ++w) v += part[w][lane];
  const int m = m0 + r, n = n0 + 4 * g;  // four n of one m a lane
  if (m >= M || n >= N) return;
  Pack<S, 4> o;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (bias != nullptr) v[i] += E::to_f(bias[min(n + i, N - 1)]);
    o.v[i] = E::from_f(v[i]);
  }
  const bool quads = N % 4 == 0 && ((uintptr_t)out & (4 * sizeof(S) - 1)) == 0;
  store_row<S, 4, false>(out + (int64_t)m * N + n, o, n, N, quads);
}

// Tiles: a group of WD x WD waves makes a (32 WD FM) x (32 WD FN) tile of the output, each wave FM x FN
// products of 32 x 32; KS such groups of a workgroup share out K and add up in LDS at the end.  Codes go
// from memory to LDS in tiles of 256 along K (128 bytes a row: whole lines), D tiles in turn, without
// passing through registers; from there to registers three steps of 64 along K ahead of the products.
// In 32x32x64 instructions the lane of group g = lane / 32 takes blocks 4g..4g+3 of a tile, one a step, so
// that the scales of its row for the tile are one dword, whose bytes the instructions pick in turn.
//
// LDS: a tile's row is 8 chunks of 16 bytes, chunk c at place c ^ (row / 2 & 7): two rows span the 64
// banks, and the sixteen lanes that a 16-byte read serves at once have eight rows of each parity, which
// then take eight different places (by row & 7 there were conflicts for half of the reads' cycles).  A
// direct load writes 64 x 16 bytes in lane order (eight rows), so each lane's address is that of the
// chunk that belongs at its place.  Scales are not placed so: their rows are 32 bytes, and a dword of each of
// 32 rows falls on eight banks, some 15 cycles of conflict a read (8192 x 8192 x 8192: 16.3 M, 13% of the
// CUs' cycles).
//
// One barrier a tile (none for a group of one wave), after the first step's products: the tile's last
// operands are in registers by then, the wave waits for its part of the next tile, meets the others,
// reads on from the next tile and starts the loads of the tile D on, into the one that all have read.
// Scales that pass through registers are waited for with all other loads, every fourth tile.
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint64_t u64x2 __attribute__((ext_vector_type(2)));

constexpr int kTileK = 8;  // blocks
constexpr int kRowBytes = kTileK * 16;
// Tiles whose scales (32 bytes of a row) are read and put into LDS together, two lanes a row: a lane a
// row with 16 bytes touches a line for each lane, and those requests hold up the direct loads behind
// them; more at a time do not leave the room for two tiles of 256 x 256.
constexpr int kScaleTiles = 4, kScaleBytes = kScaleTiles * kTileK;

// 16 bytes a lane from base + off to LDS at `to` + 16 * lane, which the instruction takes from m0 (a state
// after its write).  The compiler does not see what this writes nor that it is in flight: wait_loads()
// and the barrier order it.
__device__ __forceinline__ void load_to_lds(uint32_t to, const uint8_t* base, uint32_t off) {
  asm volatile(
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %1, %2"
      :
      : "{m0}"(to), "v"(off), "s"(base)
      : "memory");
}
// The same of four bytes a lane.
__device__ __forceinline__ void load_to_lds4(uint32_t to, const uint8_t* base, uint32_t off) {
  asm volatile(
      "s_nop 0\n\t"
      "global_load_lds_dword %1, %2"
      :
      : "{m0}"(to), "v"(off), "s"(base)
      : "memory");
}
template <int LEFT>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LEFT) : "memory");
}
__device__ __forceinline__ void wait_lds() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
}
// The group's barrier, behind the wave's own LDS reads and writes: the barrier alone orders neither, and
// what is read here may be written over by the next wave that has passed it.
__device__ __forceinline__ void meet() {
  wait_lds();
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// DS: rows of scales are whole dwords, and go to LDS by direct loads too, so that no tile waits for more
// than its own (300 x 5000 x 4096: tiles of 128 x 64 three deep 11.7 us, 10.7 so; two deep every tile
// waits for all loads anyway, and 4096 x 4096 x 8192 takes 69.1 us, 71.3 so).
template <class E, int FM, int FN, int WD, int KS, int D, bool DS>
__global__ void __launch_bounds__(64 * WD * WD * KS, 1)
k_mxfp4_mm_tile(typename E::S* __restrict__ out, const uint8_t* __restrict__ a,
                const uint8_t* __restrict__ as, const uint8_t* __restrict__ b,
                const uint8_t* __restrict__ bs, const typename E::S* __restrict__ bias, int M, int N,
                int blocks, int tiles_m, int tiles) {
  using S = typename E::S;
  constexpr int GW = WD * WD, THREADS = 64 * GW * KS;  // waves of a group
  constexpr int BM = 32 * WD * FM, BN = 32 * WD * FN, ROWS = BM + BN;
  constexpr int SR = (ROWS * 2 + 64 * GW - 1) / (64 * GW);  // 16-byte scale pieces of a thread
  constexpr int TILE = ROWS * kRowBytes, SCALES = SR * 32 * GW * kScaleBytes;
  constexpr int GROUP = D * TILE + 2 * SCALES;  // LDS of a group
  constexpr int ALOADS = BM / 8 / GW, LOADS = ROWS / 8 / GW;  // direct loads of a wave and tile
  __shared__ alignas(1024) uint8_t lds_all[KS * GROUP];
  const int lane = (int)threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6) & (GW - 1);  // of its group
  const int part = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6) / GW;        // the group
  const int tid = (int)threadIdx.x & (64 * GW - 1);
  const int wm = wave % WD, wn = wave / WD;
  uint8_t* lds = lds_all + part * GROUP;
  // Workgroups go to the eight dies in turn.  Each die takes consecutive tiles of an order in bands of 8
  // along M, so that those it has at a time share rows of both operands in its L2: with tiles counted
  // along M alone 1237 x 4099 x 5152 took 36.9 us, this 30.8.  The grid is a multiple of 8.
  const int tile = (int)(blockIdx.x & 7) * (int)(gridDim.x >> 3) + (int)(blockIdx.x >> 3);
  const int band_tiles = 8 * ((N + BN - 1) / BN), band = tile / band_tiles, in = tile % band_tiles;
  const int high = min(8, tiles_m - band * 8);  // of the last band
  if (high <= 0) return;
  const int m0 = (band * 8 + in % high) * BM, n0 = in / high * BN;
  if (n0 >= N) return;
  const int64_t pitch = (int64_t)blocks * 16;

  // The group's tiles: `tiles` from block `from` on, which may pass the rows' end.  What is past it
  // counts as zero by its scales: 0 stands for 2^-127, and with that of both operands every product
  // is below binary32's range.  Its codes are read from the group's last tile, or the rows' first.
  const int start = part * tiles * kTileK;
  const int from = start < blocks ? start : 0, have = start < blocks ? blocks - start : 0;
  const int last_full = max(have - 1, 0) / kTileK;

  // Rows 0..BM-1 of the LDS tile are a's, the rest b's; a wave's first loads of eight rows are of a, the
  // rest of b.  Rows past an operand's end repeat its last.
  auto chunk_of = [&](int j) { return (lane & 7) ^ (lane >> 4) ^ (j & 1) * 4; };  // row / 2 & 7
  auto first_row = [&](int j) {
    return j < ALOADS ? (wave * ALOADS + j) * 8
                      : BM + (wave * (LOADS - ALOADS) + j - ALOADS) * 8;
  };
  uint32_t off[LOADS];
#pragma unroll
  for (int j = 0; j < LOADS; ++j) {
    const int row = first_row(j) + lane / 8;
    const int r = j < ALOADS ? min(row, M - 1 - m0) : min(row - BM, N - 1 - n0);
    off[j] = (uint32_t)(r * pitch) + chunk_of(j) * 16;
  }
  const uint8_t* abase = a + m0 * pitch + (int64_t)from * 16;
  const uint8_t* bbase = b + n0 * pitch + (int64_t)from * 16;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds;
  // Load j of tile t into buffer `to`.  Chunks past the row's end read the tile's first.
  auto load_rows = [&](int j, int t, int to) {
    const int u = min(t, last_full), c = chunk_of(j);
    const uint32_t back = c < blocks - from - u * kTileK ? 0 : c * 16;
    load_to_lds(lds0 + to * TILE + first_row(j) * kRowBytes,
                (j < ALOADS ? abase : bbase) + u * kRowBytes, off[j] - back);
  };

  // Scales of tiles 4 s to 4 s + 3: two lanes a row, 16 bytes each.  Those of the row's end may pass it,
  // and the tensor's: they are read before that, moved and masked when they are stored (looking at
  // them sooner would wait for them, and for the direct loads around them).
  i32x4 sv[SR];
  const uint8_t* srow[SR];
  int to_end[SR];  // bytes from `from` in the row to the end of its tensor, where those are few
  const int piece = (lane & 1) * 16;
#pragma unroll
  for (int k = 0; k < SR; ++k) {
    const int row = tid / 2 + 32 * GW * k;
    const int r = row < BM ? min(m0 + row, M - 1) : min(n0 + row - BM, N - 1);
    srow[k] = (row < BM ? as : bs) + (int64_t)r * blocks + from;
    to_end[k] =
        (int)min((int64_t)((row < BM ? M : N) - r) * blocks - from, (int64_t)1 << 30);
  }
  const uint8_t* asbase = as + (int64_t)m0 * blocks + from;
  const uint8_t* bsbase = bs + (int64_t)n0 * blocks + from;
  auto direct_scales = [&](int s) {  // the rows of the codes' loads, a dword a lane; past the end the first
    const int at = s * kScaleBytes + (lane & 7) * 4;
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
      load_to_lds4(lds0 + D * TILE + (s & 1) * SCALES + first_row(j) * kScaleBytes,
                   j < ALOADS ? asbase : bsbase,
                   (off[j] >> 4) - chunk_of(j) + (at < have ? at : 0));
    }
  };
  auto load_scales = [&](int s) {
    if constexpr (DS) return direct_scales(s);
    const int at = s * kScaleBytes + piece;
#pragma unroll
    for (int k = 0; k < SR; ++k) {
      __builtin_memcpy(&sv[k], srow[k] + min(at, to_end[k] - 16), 16);
    }
  };
  auto store_scales = [&](int s) {
    if constexpr (DS) return;
    if (have - s * kScaleBytes < kScaleBytes) {
      const int at = s * kScaleBytes + piece, left = min(max(have - at, 0), 16);
#pragma unroll
      for (int k = 0; k < SR; ++k) {
        const int past = max(at - (to_end[k] - 16), 0);
        const u64x2 v = __builtin_bit_cast(u64x2, sv[k]);
        uint64_t lo = past >= 8 ? v[1] : v[0], hi = past >= 8 ? 0 : v[1];
        const int bits = (past & 7) * 8;
        lo = lo >> bits | (hi << 1) << (63 - bits);
        hi >>= bits;
        if (left < 8) lo &= ((uint64_t)1 << (8 * left)) - 1;
        if (left < 16) hi &= left <= 8 ? 0 : ((uint64_t)1 << (8 * (left - 8))) - 1;
        sv[k] = __builtin_bit_cast(i32x4, u64x2{lo, hi});
      }
    }
    uint8_t* to = lds + D * TILE + (s & 1) * SCALES + tid * 16;
#pragma unroll
    for (int k = 0; k < SR; ++k) *reinterpret_cast<i32x4*>(to + k * 1024 * GW) = sv[k];
  };
  auto have_scales = [&]() {  // waits for them here and not later, when other loads are in flight
    if constexpr (DS) return;
#pragma unroll
    for (int k = 0; k < SR; ++k) asm volatile("" : "+v"(sv[k]));
  };

  const int r32 = lane & 31, g = lane >> 5;
  const int am = wm * 32 * FM + r32, bn = BM + wn * 32 * FN + r32;
  i32x4 fa[4][FM], fb[4][FN];
  int sa[2][FM], sb[2][FN];
  constexpr int OPS = FM + FN, MMS = FM * FN, LSTEPS = 3;
  // Operand o of step s: a's first, then b's; and its scales for the tile.
  auto read_codes = [&](int o, int buf, int s) {
    const int place = ((4 * g + s) ^ (r32 >> 1 & 7)) * 16 + buf * TILE;
    if (o < FM) {
      fa[s][o] = *reinterpret_cast<const i32x4*>(lds + place + (am + 32 * o) * kRowBytes);
    } else {
      fb[s][o - FM] =
          *reinterpret_cast<const i32x4*>(lds + place + (bn + 32 * (o - FM)) * kRowBytes);
    }
  };
  auto read_scales = [&](int o, int t, int into) {
    const bool in = !DS || t * kTileK + 4 * g < have;
    const int place = D * TILE + (t / kScaleTiles & 1) * SCALES + t % kScaleTiles * kTileK + 4 * g;
    if (o < FM) {
      const int v = *reinterpret_cast<const int*>(lds + place + (am + 32 * o) * kScaleBytes);
      sa[into][o] = in ? v : 0;
    } else {
      const int v = *reinterpret_cast<const int*>(lds + place + (bn + 32 * (o - FM)) * kScaleBytes);
      sb[into][o - FM] = in ? v : 0;
    }
  };
  f32x16 sum[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i) {
#pragma unroll
    for (int j = 0; j < FN; ++j) {
#pragma unroll
      for (int e = 0; e < 16; ++e) sum[i][j][e] = 0.0f;
    }
  }
  // The products of step s, with `other(q)` issued behind the q-th: the order is kept as written, so
  // that reads and loads go out between products, each in the time one takes.
  auto step = [&](auto s, auto other) {
    constexpr int ST = decltype(s)::value;
#pragma unroll
    for (int q = 0; q < MMS; ++q) {
      const int i = q / FN, j = q % FN;
      sum[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
          fp4_operand(fb[ST][j]), fp4_operand(fa[ST][i]), sum[i][j], kFp4, kFp4, ST, sb[0][j], ST,
          sa[0][i]);
      other(q);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  using S0 = std::integral_constant<int, 0>;
  using S1 = std::integral_constant<int, 1>;
  using S2 = std::integral_constant<int, 2>;
  using S3 = std::integral_constant<int, 3>;
  auto reading = [&](int q, int buf, int s) {  // the operands of step s, from the first products on
#pragma unroll
    for (int o = 0; o < OPS; ++o) {
      if (o * MMS / 2 / OPS == q) read_codes(o, buf, s);
    }
  };
  auto together = [&]() {  // the group's waves; one alone waits for itself
    if constexpr (GW > 1) meet();
    else wait_lds();
  };
  // The products so far are made before this point: they touch no memory, and without it the compiler
  // moves them behind the barrier and the branches below, to where their results are next used.
  auto here = [&]() {
#pragma unroll
    for (int i = 0; i < FM; ++i) {
#pragma unroll
      for (int j = 0; j < FN; ++j) asm volatile("" : "+a"(sum[i][j]));
    }
  };

  load_scales(0);
#pragma unroll
  for (int j = 0; j < LOADS; ++j) load_rows(j, 0, 0);
#pragma unroll
  for (int j = 0; j < LOADS; ++j) load_rows(j, 1, 1);
  have_scales();
  store_scales(0);
  wait_loads<0>();
#pragma unroll
  for (int u = 2; u < D; ++u) {
#pragma unroll
    for (int j = 0; j < LOADS; ++j) load_rows(j, u, u);
  }
  together();
#pragma unroll
  for (int o = 0; o < OPS; ++o) {
    read_codes(o, 0, 0);
    read_scales(o, 0, 0);
  }
#pragma unroll
  for (int u = 1; u < 3; ++u) {
#pragma unroll
    for (int o = 0; o < OPS; ++o) read_codes(o, 0, u);
  }
  int cur = 0;
  for (int t = 0; t + 1 < tiles; ++t) {
    const int next = cur + 1 < D ? cur + 1 : 0;
    __builtin_amdgcn_sched_barrier(0);
    step(S0(), [&](int q) { reading(q, cur, 3); });
    here();
    if constexpr (D > 2) {
      if (t % kScaleTiles == kScaleTiles - 1) {
        have_scales();
        store_scales(t / kScaleTiles + 1);
      }
      wait_loads<(D - 2) * LOADS>();
    } else {
      if (t % kScaleTiles == kScaleTiles - 1) store_scales(t / kScaleTiles + 1);
      wait_loads<0>();
      have_scales();
    }
    together();
    if (t % kScaleTiles == 0) load_scales(t / kScaleTiles + 1);
    __builtin_amdgcn_sched_barrier(0);
    auto loading = [&](int q, int s) {  // over the steps but the first
#pragma unroll
      for (int j = 0; j < LOADS; ++j) {
        if (j * LSTEPS * MMS / LOADS == q + s * MMS) load_rows(j, t + D, cur);
      }
    };
    step(S1(), [&](int q) {
      reading(q, next, 0);
#pragma unroll
      for (int o = 0; o < OPS; ++o) {
        if (o * MMS / 2 / OPS == q) read_scales(o, t + 1, 1);
      }
      loading(q, 0);
    });
    step(S2(), [&](int q) {
      reading(q, next, 1);
      loading(q, 1);
    });
    step(S3(), [&](int q) {
      reading(q, next, 2);
      loading(q, 2);
    });
#pragma unroll
    for (int i = 0; i < FM; ++i) sa[0][i] = sa[1][i];
#pragma unroll
    for (int i = 0; i < FN; ++i) sb[0][i] = sb[1][i];
    cur = next;
  }
#pragma unroll
  for (int o = 0; o < OPS; ++o) read_codes(o, cur, 3);
  step(S0(), [](int) {});
  step(S1(), [](int) {});
  step(S2(), [](int) {});
  step(S3(), [](int) {});
  wait_loads<0>();  // the loads past the last tile, before other uses of their LDS
  meet();           // every wave has read its last operands

  // A lane holds n = 8 (e / 4) + 4 g + e % 4 of m = lane % 32 of each product: 8 or 16 bytes in a row.
  // The rows are turned in LDS and stored 16 bytes a lane, whole lines in a row: as they are held, two
  // or four bytes a store, the stores took 130 of 420 us (8192 x 8192 x 8192 bf16).
  constexpr int VEC = 16 / (int)sizeof(S);
  const bool whole = N % VEC == 0 && ((uintptr_t)out & 15) == 0;
  if constexpr (KS > 1) {
    // every group's tile in fp32, added in the groups' order by all
    constexpr int LINE = BN * 4 + 16;  // 16: rows start in other banks
    static_assert(BM * LINE <= GROUP, "a group's sums fit its LDS");
#pragma unroll
    for (int i = 0; i < FM; ++i) {
#pragma unroll
      for (int j = 0; j < FN; ++j) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int c = wn * 32 * FN + 32 * j + 8 * q + 4 * g;
          *reinterpret_cast<f32x4*>(lds + (am + 32 * i) * LINE + c * 4) =
              f32x4{sum[i][j][4 * q], sum[i][j][4 * q + 1], sum[i][j][4 * q + 2],
                    sum[i][j][4 * q + 3]};
        }
      }
    }
    __syncthreads();
    constexpr int PER = BN / VEC;  // lanes a row
#pragma unroll
    for (int k = 0; k < (BM * PER + THREADS - 1) / THREADS; ++k) {
      const int at = k * THREADS + (int)threadIdx.x, r = at / PER, c = at % PER * VEC;
      const int m = m0 + r, n = n0 + c;
      if (r >= BM || m >= M || n >= N) continue;
      Pack<S, VEC> v;
#pragma unroll
      for (int h = 0; h < VEC / 4; ++h) {
        f32x4 f = *reinterpret_cast<const f32x4*>(lds_all + r * LINE + (c + 4 * h) * 4);
#pragma unroll
        for (int p = 1; p < KS; ++p) {
          f += *reinterpret_cast<const f32x4*>(lds_all + p * GROUP + r * LINE + (c + 4 * h) * 4);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (bias != nullptr) f[e] += E::to_f(bias[min(n + 4 * h + e, N - 1)]);
          v.v[4 * h + e] = E::from_f(f[e]);
        }
      }
      store_row<S, VEC, false>(out + (int64_t)m * N + n, v, n, N, whole);
    }
  } else {
    // 32 rows of each wave at a time
    constexpr int WN = 32 * FN, LINE = WN * (int)sizeof(S) + 16;
    constexpr int ADD = GW * 32 * LINE;  // the bias, behind the waves' rows
    static_assert(ADD + BN * 4 <= D * TILE, "what reuses the tiles");
    if (bias != nullptr) {
      for (int c = tid; c < BN; c += 64 * GW) {
        *reinterpret_cast<float*>(lds + ADD + c * 4) = E::to_f(bias[min(n0 + c, N - 1)]);
      }
      __syncthreads();
    }
    uint8_t* own = lds + wave * 32 * LINE;
    const int wn0 = n0 + wn * WN;
#pragma unroll
    for (int i = 0; i < FM; ++i) {
#pragma unroll
      for (int j = 0; j < FN; ++j) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int c = 32 * j + 8 * q + 4 * g;
          f32x4 f;
#pragma unroll
          for (int e = 0; e < 4; ++e) f[e] = sum[i][j][4 * q + e];
          if (bias != nullptr) {
            f += *reinterpret_cast<const f32x4*>(lds + ADD + (wn * WN + c) * 4);
          }
          Pack<S, 4> v;
#pragma unroll
          for (int e = 0; e < 4; ++e) v.v[e] = E::from_f(f[e]);
          *reinterpret_cast<Pack<S, 4>*>(own + r32 * LINE + c * sizeof(S)) = v;
        }
      }
      const int wm0 = m0 + wm * 32 * FM + 32 * i;
      constexpr int PER = WN / VEC, STEPS = 32 * PER / 64;  // lanes a row
#pragma unroll
      for (int k = 0; k < STEPS; ++k) {
        const int r = (k * 64 + lane) / PER, c = (k * 64 + lane) % PER * VEC;
        const int m = wm0 + r, n = wn0 + c;
        const Pack<S, VEC> v =
            *reinterpret_cast<const Pack<S, VEC>*>(own + r * LINE + c * sizeof(S));
        if (m < M && n < N) store_row<S, VEC, true>(out + (int64_t)m * N + n, v, n, N, whole);
      }
    }
  }
}

static int64_t tiles_of(int M, int N, int bm, int bn) {
  return (int64_t)((M + bm - 1) / bm) * ((N + bn - 1) / bn);
}

// Whether the tile kernel's 32-bit offsets and its reads of 16 scale bytes fit the operands.
static bool tiles_fit(int M, int N, int blocks) {
  return (int64_t)blocks * 16 * 256 < ((int64_t)1 << 32) && (int64_t)M * blocks >= 16 &&
         (int64_t)N * blocks >= 16;
}

template <class E, int FM, int FN, int WD, int KS, int D = 2>
static int product_tiles(typename E::S* out, const uint8_t* a, const uint8_t* as, const uint8_t* b,
                         const uint8_t* bs, const typename E::S* bias, int M, int N, int blocks,
                         bool direct, hipStream_t st) {
  constexpr int BM = 32 * WD * FM, BN = 32 * WD * FN;
  const int tm = (M + BM - 1) / BM, tn = (N + BN - 1) / BN;
  const int tiles = (blocks + kTileK * KS - 1) / (kTileK * KS);  // of a group
  const dim3 grid((unsigned)((tm * tn + 7) / 8 * 8)), block(64 * WD * WD * KS);
  if constexpr (D > 2) {
    if (direct) {
      hipLaunchKernelGGL((k_mxfp4_mm_tile<E, FM, FN, WD, KS, D, true>), grid, block, 0, st, out, a, as,
                         b, bs, bias, M, N, blocks, tm, tiles);
      return check_launch("mxfp4_scaled_mm");
    }
  }
  hipLaunchKernelGGL((k_mxfp4_mm_tile<E, FM, FN, WD, KS, D, false>), grid, block, 0, st, out, a, as, b,
                     bs, bias, M, N, blocks, tm, tiles);
  return check_launch("mxfp4_scaled_mm");
}

// The form for a product: the one of the lowest estimated time.  The estimates (us) are fits to calls of
// every form over M from 1 to 4096, N from 512 to 16384 and K from 512 to 14336 (bf16; weights of several
// sets in turn).  They know sizes only: fp32 outputs, K that is not a multiple of 256 and sizes past those
// take longer than estimated (1237 x 4099 x 5152 fp32 21.5 us estimated, 29-31 measured) and may have a
// faster form than the one chosen.  Measured (us) where one gives way to the next (M x N x K):
//   rows (16 x 16, straight from memory) and 32 x 32 of four waves: 1 x 512 x 5120 4.5 and 5.2, 1 x 8192 x
//     5120 8.2 and 7.0, 16 x 8192 x 12288 20.0 and 14.6
//   32 x 32 of four waves and of eight, whose LDS is a whole CU's: 1 x 4099 x 12288 10.0 and 8.2, 48 x 4099
//     x 5120 (two rounds) 8.0 and 11.1
//   32 x 32 and 64 x 64 of four waves, without barriers: 40 x 8192 x 14336 14.9 and 18.0, 100 x 6144 x 8192
//     15.8 and 12.1
//   the latter and 64 x 64 with barriers: 100 x 6144 x 8192 12.1 and 13.1, 64 x 16384 x 5120 12.9 and 10.3
//   64 x 64 and 128 x 64, where the latter is one round: 256 x 8192 x 5120 13.4 and 12.5, 128 x 8192 x 8192
//     16.2 and 19.1
//   128 x 64 and 128 x 128: 1024 x 4096 x 5120 23.2 and 18.0, 256 x 8192 x 5120 12.5 and 15.3
//   128 x 128 and 192 x 128, where the latter is one round: 1500 x 4096 x 4096 20.4 and 18.5, 700 x 8192 x
//     5120 23.8 and 21.8, 2048 x 4096 x 4096 (1.4 rounds) 23.1 and 32.3
//   128 x 128 and 256 x 256: 700 x 8192 x 5120 23.8 and 33.3, 2048 x 4099 x 5120 43.2 and 37.8, 4096 x 4099
//     x 5120 (272 tiles of the larger) 69.6 and 78.2
enum MmForm {
  MM_ROWS, MM_32X32_LONG, MM_32X32, MM_64X64_APART, MM_64X64, MM_128X64, MM_128X128, MM_192X128,
  MM_256X256
};

static MmForm form_of(int M, int N, int blocks) {
  auto waves = [&](int bm, int bn) {  // workgroups of such tiles a CU
    return (double)((M + bm - 1) / bm) * ((N + bn - 1) / bn) / 256.0;
  };
  auto part = [](double w) { return (w + std::ceil(w)) / 2; };  // rounds, where the last is not full
  const double k = blocks / 256.0;  // in units of K = 8192
  double w = waves(16, 16), best = 1e30;
  MmForm form = MM_ROWS;
  auto offer = [&](MmForm f, double us) {
    if (us < best && w < 65000) best = us, form = f;  // a launch takes fewer than 2^32 threads
  };
  offer(MM_ROWS, 2.9 + k * (w > 1 ? w * ((M > 16 ? 4.5 : 3) + 2.5 * k) : M == 1 ? 3.7 : 5.3));
  if (!tiles_fit(M, N, blocks)) return MM_ROWS;
  w = waves(32, 32);
  if (w <= 1) offer(MM_32X32_LONG, 3.8 + k * (2.6 + 3.7 * w * w));
  offer(MM_32X32, w <= 1   ? 3.5 + k * (4 + 2.8 * w * w)
                  : w <= 2 ? 3.2 + k * (1.5 + 2.8 * w)
                           : 2 + part(w) * (0.9 + 5.7 * k));
  w = waves(64, 64);
  if (w <= 1) {
    const double memory = 4 + ((double)M + N) * blocks * 17 / 5e6;  // its operands' way, if that is longer
    offer(MM_64X64_APART, std::max(5.2 + k * (6.2 + 1.5 * w), memory));
  }
  offer(MM_64X64, w <= 2   ? 3.2 + k * (9 + 2.5 * w)
                  : w <= 4 ? 3.5 + part(w) * (0.25 + 7.7 * k)
                           : 3.5 + part(w) * (0.6 + 7.7 * k));
  w = waves(128, 64);
  if (w <= 1) offer(MM_128X64, 3.7 + k * (10.5 + 2 * w));
  w = waves(128, 128);
  offer(MM_128X128, w <= 1   ? 5.4 + k * (13.4 + 6 * w)
                    : w <= 2 ? 4 + k * (25 + 7 * w)
                             : 3 + part(w) * (2 + 20.5 * k));
  w = waves(192, 128);
  if (w <= 1) offer(MM_192X128, 5.5 + k * (21 + 5 * w));
  w = waves(256, 256);
  offer(MM_256X256, w <= 1 ? 8 + k * (36 + 30 * w * w) : std::ceil(w) * (8.5 + 61 * k));
  return form;
}

// A product's form, whether it has three tiles in flight, and whether scales go to LDS by direct loads.
struct MmPlan {
  MmForm form;
  bool deep, direct;
};
static MmPlan plan_of(int M, int N, int blocks, bool aligned_scales) {
  MmPlan p{form_of(M, N, blocks), false, false};
  switch (p.form) {
    case MM_64X64:
      // as below; two workgroups a CU: 128 x 8192 x 8192 16.2 us, 25.4 with two tiles; 1024 x 4096 x 5120
      // (four a CU) 24.8 and 23.4
      p.deep = tiles_of(M, N, 64, 64) <= 512;
      break;
    case MM_128X128:
      // one workgroup a CU has room for a third tile in flight: 1024 x 4096 x 5120 17.7 us, 20.3 with two;
      // where two share a CU they overlap, 2048 x 4096 x 4096 23.5 us and 28.0
      p.deep = tiles_of(M, N, 128, 128) <= 256;
      break;
    case MM_128X64:
    case MM_192X128: p.deep = true; break;
    default: break;
  }
  p.direct = p.deep && blocks % 4 == 0 && aligned_scales;
  return p;
}

struct MmName {
  char text[64];
};
static MmName name_of(const MmPlan& p) {
  static const char* const forms[] = {"rows", "32x32 by eight waves", "32x32", "64x64 by waves apart",
                                      "64x64", "128x64", "128x128", "192x128", "256x256"};
  MmName n;
  snprintf(n.text, sizeof(n.text), "%s%s%s", forms[p.form], p.deep ? ", three tiles" : "",
           p.direct ? ", direct scales" : "");
  return n;
}

template <class E>
static int product(void* out, const uint8_t* a, const uint8_t* as, const uint8_t* b,
                   const uint8_t* bs, const void* bias, int M, int N, int blocks, hipStream_t st) {
  using S = typename E::S;
  auto* o = static_cast<S*>(out);
  const auto* bi = static_cast<const S*>(bias);
  const MmPlan p = plan_of(M, N, blocks, aligned(4, as, bs));
  if (launches_traced()) {
    trace_launch("mxfp4_scaled_mm", "M=%d N=%d K=%lld: %s", M, N, (long long)blocks * kMxBlock,
                 name_of(p).text);
  }
#define MCOP_TILES(...) \
  return product_tiles<E, __VA_ARGS__>(o, a, as, b, bs, bi, M, N, blocks, p.direct, st)
  switch (p.form) {
    case MM_32X32_LONG: MCOP_TILES(1, 1, 1, 8);
    case MM_32X32: MCOP_TILES(1, 1, 1, 4);
    case MM_64X64_APART: MCOP_TILES(2, 2, 1, 4);
    case MM_64X64:
      if (p.deep) MCOP_TILES(1, 1, 2, 1, 3);
      MCOP_TILES(1, 1, 2, 1);
    case MM_128X64: MCOP_TILES(2, 1, 2, 1, 3);
    case MM_128X128:
      if (p.deep) MCOP_TILES(2, 2, 2, 1, 3);
      MCOP_TILES(2, 2, 2, 1);
    case MM_192X128: MCOP_TILES(3, 2, 2, 1, 3);
    case MM_256X256: MCOP_TILES(4, 4, 2, 1);
    default: break;
  }
#undef MCOP_TILES
  const dim3 grid((unsigned)((N + 15) / 16), (unsigned)((M + 15) / 16)), block(256);
  hipLaunchKernelGGL((k_mxfp4_mm_rows<E, 4, 4>), grid, block, 0, st, o, a, as, b, bs, bi, M, N,
                     blocks);
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
  // the grid: at most 65535 workgroups along M, and fewer than 2^32 threads along N
  if (N > ((int64_t)1 << 27) || M > (int64_t)65535 * 16) {
    return set_error(MCOP_E_UNSUPPORTED, "%s: M %lld or N %lld is more than one launch takes "
                     "(%d and 2^27)", name, (long long)M, (long long)N, 65535 * 16);
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

extern "C" const char* mcop_debug_mxfp4_mm_form(int64_t M, int64_t N, int64_t K, int aligned_scales) {
  using namespace mcop;
  static thread_local MmName name;
  if (M <= 0 || N <= 0 || K <= 0 || K % kMxBlock != 0 || K > INT32_MAX ||
      N > ((int64_t)1 << 27) || M > (int64_t)65535 * 16) {
    return "";
  }
  name = name_of(plan_of((int)M, (int)N, (int)(K / kMxBlock), aligned_scales != 0));
  return name.text;
}
