// kv_pages.hip -- the pages of a paged cache between steps: copied, shared with a fork, taken for new tokens,
// given back, and moved together.
//
// The pool is three device tensors: ref_counts[p], the sequences that hold page p (0 or less: free);
// block_table, a row of pages a sequence, -1 behind the last; seq_lens, the positions of each.  Pages are
// taken the lowest free one first, in the order of the requests, so that results depend on nothing
// else.  Bookkeeping is bound by latency: a request's answer needs all requests before it and the counts up to
// its pages, so one workgroup scans both (a list of the free pages that are asked for, and where each
// request's begin), and writes the requests' rows itself where they are few and short; else a second launch
// has a workgroup for every request.  Copies are bound by HBM.
//
// Every index that comes from a tensor is checked before it is used: one outside the table, the row or the
// pool is left out.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "../../include/mcop_norm.h"
#include "launch_trace.h"
#include "rowkern.h"
#include "wave_scan.h"

namespace mcop {

// ---- Copies: a workgroup moves 16 KiB, a piece of a page or some whole pages.
constexpr int kCopyLanes = 256, kCopyUnits = 4, kCopyBytes = kCopyLanes * kCopyUnits * 16;
constexpr int kCopyTensors = 64;  // of a launch; one lane a tensor finds a workgroup's

struct CopyTensor {
  uint8_t* base;
  int64_t stride, bytes;  // from page to page; of a page
};
struct CopyArgs {
  CopyTensor t[kCopyTensors];
  uint32_t first[kCopyTensors];  // the tensor's first workgroup
  int tensors;
  const int32_t *src, *dst;
  int64_t pairs, pages;
};

typedef u32x4 u32x4_any __attribute__((aligned(1)));
__device__ __forceinline__ u32x4 load_unit(const uint8_t* p) {
  return *reinterpret_cast<const u32x4_any*>(p);
}
__device__ __forceinline__ void store_unit(uint8_t* p, const u32x4& v) {
  __builtin_nontemporal_store(v, reinterpret_cast<u32x4_any*>(p));
}

// Each lane's loads go out together: none hangs on a condition, and a lane that has nothing to move reads what
// another does (with a condition on each, 400 pages of 32 layers took 200 us; so 167, 5.2 TB/s of what is read and
// written).  Bound by HBM in both directions.
__global__ void __launch_bounds__(kCopyLanes, 8) k_kv_copy_pages(CopyArgs a) {
  const int lane = (int)threadIdx.x & 63;
  const bool mine = lane < a.tensors && a.first[lane < a.tensors ? lane : 0] <= blockIdx.x;
  const int i = (int)__builtin_popcountll(__builtin_amdgcn_ballot_w64(mine)) - 1;
  const CopyTensor t = a.t[i];
  const int64_t block = blockIdx.x - a.first[i];
  // whole units of 16 bytes of a page, and bytes behind them
  const int64_t units = t.bytes / 16;
  const int rest = (int)(t.bytes % 16);
  constexpr int kUnits = kCopyLanes * kCopyUnits;
  if (units >= kUnits) {  // a piece of one page
    const int64_t pieces = (units + kUnits - 1) / kUnits, pair = block / pieces;
    const int64_t from = a.src[pair], where = a.dst[pair], first = (block - pair * pieces) * kUnits;
    if (from < 0 || from >= a.pages || where < 0 || where >= a.pages || from == where) return;
    const uint8_t* src = t.base + from * t.stride;
    uint8_t* dst = t.base + where * t.stride;
    u32x4 v[kCopyUnits];
#pragma unroll
    for (int k = 0; k < kCopyUnits; ++k) {
      v[k] = load_unit(src + min(first + k * kCopyLanes + (int)threadIdx.x, units - 1) * 16);
    }
#pragma unroll
    for (int k = 0; k < kCopyUnits; ++k) {
      const int64_t u = first + k * kCopyLanes + (int)threadIdx.x;
      if (u < units) store_unit(dst + u * 16, v[k]);
    }
    if (first + kUnits >= units && (int)threadIdx.x < rest) {
      dst[units * 16 + threadIdx.x] = src[units * 16 + threadIdx.x];
    }
    return;
  }
  // some whole pages, a unit (or what is behind the last) a lane at a time
  const uint32_t each = (uint32_t)units + (rest > 0 ? 1 : 0);
  const int many = kUnits / (int)each;
  const int64_t pair0 = block * many;
  int64_t from[kCopyUnits], where[kCopyUnits];
  uint32_t unit[kCopyUnits];
  bool moves[kCopyUnits];
#pragma unroll
  for (int k = 0; k < kCopyUnits; ++k) {
    const uint32_t x = (uint32_t)(k * kCopyLanes) + threadIdx.x, q = x / each;
    unit[k] = x - q * each;
    const int64_t pair = pair0 + q;
    moves[k] = (int)q < many && pair < a.pairs;
    from[k] = a.src[min(pair, a.pairs - 1)], where[k] = a.dst[min(pair, a.pairs - 1)];
  }
  u32x4 v[kCopyUnits];
#pragma unroll
  for (int k = 0; k < kCopyUnits; ++k) {
    moves[k] = moves[k] && from[k] >= 0 && from[k] < a.pages && where[k] >= 0 && where[k] < a.pages &&
               from[k] != where[k];
    if (units > 0) {
      v[k] = load_unit(t.base + (moves[k] ? from[k] : 0) * t.stride +
                       min((int64_t)unit[k], units - 1) * 16);
    }
  }
#pragma unroll
  for (int k = 0; k < kCopyUnits; ++k) {
    if (!moves[k]) continue;
    const uint8_t* src = t.base + from[k] * t.stride;
    uint8_t* dst = t.base + where[k] * t.stride;
    if (unit[k] < units) {
      store_unit(dst + unit[k] * 16, v[k]);
    } else {
      for (int x = 0; x < rest; ++x) dst[units * 16 + x] = src[units * 16 + x];
    }
  }
}

// ---- The pool.
struct Pool {
  int32_t* table;
  int64_t stride;
  int rows, columns;
  int32_t *lens, *counts;
  int pages, page_size;
};

__device__ __forceinline__ int64_t pages_of(int64_t tokens, int page_size) {
  return (tokens + page_size - 1) / page_size;
}
__device__ __forceinline__ bool row_ok(const Pool& p, int row) { return row >= 0 && row < p.rows; }
__device__ __forceinline__ bool len_ok(const Pool& p, int64_t n) {  // of a row of the table, and of lens
  return n >= 0 && n <= INT32_MAX && n <= (int64_t)p.columns * p.page_size;
}

// Exclusive sum over a workgroup of 1024 threads, of values up to 2^31 - 1, where it stops; *all: the whole.
// The barriers let `lds` be used again at once.
constexpr int kScanLanes = 1 << 10, kScanWaves = kScanLanes / 64;
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t* lds, uint32_t* all) {
  const ScanAddUpTo31 op;
  const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
  const uint32_t upto = wave_scan<ScanAddUpTo31>(v);
  uint32_t before = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)upto, 0x138, 0xf, 0xf, false);  // wave_shr:1
  if (lane == 63) lds[wave] = upto;
  __syncthreads();
  // every wave sums the waves for itself
  const uint32_t sums = wave_scan<ScanAddUpTo31>(lane < kScanWaves ? lds[lane] : 0);
  __syncthreads();
  *all = (uint32_t)__builtin_amdgcn_readlane((int)sums, kScanWaves - 1);
  const uint32_t earlier = (uint32_t)__builtin_amdgcn_readlane((int)sums, wave > 0 ? wave - 1 : 0);
  return op(before, wave > 0 ? earlier : 0);
}

// What a request is: a fork of one sequence into another, or new tokens for one.
struct Requests {
  const int32_t *from, *to;  // fork: parents, children; extend: sequences, null
  const int32_t* cu;         // extend: where each one's new tokens begin
  int count;
};
struct Request {
  bool ok;             // its indexes and lengths are
  int from, to;
  int64_t old, now;    // the sequence's length before and after
  int64_t have, need;  // pages that it has (fork: shares), and needs besides
};
template <bool FORK>
__device__ __forceinline__ Request request_of(const Pool& p, const Requests& r, int i) {
  Request q = {};
  q.from = r.from[i];
  q.to = FORK ? r.to[i] : q.from;
  q.ok = row_ok(p, q.from) && row_ok(p, q.to);
  if (!q.ok) return q;
  q.old = p.lens[q.from];
  q.now = FORK ? q.old : q.old + (int64_t)r.cu[i + 1] - r.cu[i];
  q.ok = len_ok(p, q.old) && q.now >= q.old && len_ok(p, q.now);
  if (!q.ok) return q;
  q.have = FORK ? q.old / p.page_size : pages_of(q.old, p.page_size);
  q.need = pages_of(q.now, p.page_size) - q.have;
  if (FORK && q.need > 0) {  // a part-filled page that the parent has not: the child has none either
    const int32_t page = p.table[q.from * p.stride + q.have];
    if (page < 0 || page >= p.pages) q.need = 0;
  }
  return q;
}

// Workspace of a fork or an extension: found free pages; then where each request's begin in them; then
// the pages.
struct Taken {
  int32_t *found, *begin, *list;
  __host__ __device__ Taken(void* ws, int requests)
      : found(static_cast<int32_t*>(ws)), begin(found + 4), list(begin + requests) {}
};

constexpr int kScanPages = 16;  // pages a lane at a time

// The counts of sixteen pages from `first` on, and which of them are in use.
struct PageCounts {
  int32_t c[kScanPages];
  __device__ __forceinline__ void load(const int32_t* counts, int64_t first, int64_t pages) {
    if (first + kScanPages <= pages) {
      __builtin_memcpy(c, counts + first, sizeof(c));
    } else {
#pragma unroll
      for (int k = 0; k < kScanPages; ++k) c[k] = first + k < pages ? counts[first + k] : 0;
    }
  }
  __device__ __forceinline__ uint32_t used() const {
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k < kScanPages; ++k) m |= (uint32_t)(c[k] > 0) << k;
    return m;
  }
};
// The low bits that stand for pages below `end`, of sixteen from `first` on.
__device__ __forceinline__ uint32_t pages_below(int64_t first, int64_t end) {
  const int64_t n = end - first;
  return n <= 0 ? 0u : n >= kScanPages ? 0xffffu : (1u << (int)n) - 1;
}

// A request's pages, if there are enough; null else.
__device__ __forceinline__ const int32_t* pages_for(const Taken& t, const Request& q, int i) {
  const int64_t begin = t.begin[i];
  return q.need == 0 || begin + q.need <= t.found[0] ? t.list + begin : nullptr;
}

// What a request's lanes do (of a wave, some waves, or a part of one).
struct Lanes {
  int lane, all;
};

// Fork i: the child's row.
struct ForkTo {
  int32_t *src, *dst;
};
__device__ __forceinline__ void fork_row(const Pool& p, const Requests& r, const Taken& t, const ForkTo& to,
                                         int i, Lanes me) {
  const Request q = request_of<true>(p, r, i);
  if (!q.ok) {
    if (me.lane == 0) to.src[i] = to.dst[i] = -1;
    return;
  }
  const int32_t* pages = pages_for(t, q, i);
  const int32_t* from = p.table + q.from * p.stride;
  int32_t* row = p.table + q.to * p.stride;
  for (int c = me.lane; c < p.columns; c += me.all) {
    int32_t page = -1;
    if (pages != nullptr && c < q.have) {
      page = from[c];
      if (page >= 0 && page < p.pages) atomicAdd(&p.counts[page], 1);
    } else if (pages != nullptr && c < q.have + q.need) {
      page = pages[0];
    }
    row[c] = page;
  }
  if (me.lane == 0) {
    const bool copies = pages != nullptr && q.need > 0;
    to.src[i] = copies ? from[q.have] : -1;
    to.dst[i] = copies ? pages[0] : -1;
    if (copies) p.counts[pages[0]] = 1;
    p.lens[q.to] = pages != nullptr ? (int32_t)q.now : 0;
  }
}

// Sequence i that grows: its row and slots, and what lane 0 writes as its length when every lane has read the
// old one (-1: nothing); i == r.count: the slots behind the last.
struct ExtendTo {
  int64_t* slots;
  int64_t tokens;
  int32_t* starts;
};
__device__ __forceinline__ int extend_row(const Pool& p, const Requests& r, const Taken& t,
                                          const ExtendTo& to, int i, Lanes me) {
  if (i == r.count) {
    const int64_t last = max(r.cu[r.count], 0);
    for (int64_t s = last + me.lane; s < to.tokens; s += me.all) to.slots[s] = -1;
    return -1;
  }
  const Request q = request_of<false>(p, r, i);
  const int32_t* pages = q.ok ? pages_for(t, q, i) : nullptr;
  const int64_t first = max(r.cu[i], 0), end = min((int64_t)r.cu[i + 1], to.tokens);
  int32_t* row = q.ok ? p.table + q.from * p.stride : nullptr;
  for (int64_t s = first + me.lane; s < end; s += me.all) {
    int64_t slot = -1;
    if (pages != nullptr) {
      const int64_t at = q.old + s - r.cu[i], c = at / p.page_size;
      const int32_t page = c < q.have ? row[c] : pages[c - q.have];
      if (page >= 0 && page < p.pages) slot = (int64_t)page * p.page_size + at % p.page_size;
    }
    to.slots[s] = slot;
  }
  if (pages != nullptr) {
    for (int64_t k = me.lane; k < q.need; k += me.all) {
      row[q.have + k] = pages[k];
      p.counts[pages[k]] = 1;
    }
  }
  if (me.lane == 0) to.starts[i] = pages != nullptr ? (int32_t)q.old : -1;
  return pages != nullptr ? (int)q.now : -1;
}

// One workgroup: where each request's pages begin in the order of all, and the lowest free pages, as many as
// are asked for.  With ALONE also the rows, 2^log_lanes lanes a request, where a second launch would take
// longer (lanes_alone).
template <class To, bool ALONE>
__global__ void __launch_bounds__(kScanLanes)
k_kv_pages_take(Pool p, Requests r, Taken t, To to, int log_lanes) {
  constexpr bool FORK = std::is_same_v<To, ForkTo>;
  __shared__ uint32_t lds[kScanWaves];
  // the first counts are on their way while the requests are read
  const int64_t lane_first = (int64_t)threadIdx.x * kScanPages;
  PageCounts c;
  c.load(p.counts, lane_first, p.pages);
  const ScanAddUpTo31 add;  // no pool has 2^31 pages: what is past that is not there
  uint32_t asked = 0, all;
  for (int i0 = 0; i0 < r.count; i0 += kScanLanes) {
    const int i = i0 + (int)threadIdx.x;
    const uint32_t need = i < r.count ? (uint32_t)request_of<FORK>(p, r, i).need : 0;
    const uint32_t begin = add(asked, block_scan(need, lds, &all));
    if (i < r.count) t.begin[i] = (int32_t)begin;
    asked = add(asked, all);
  }
  uint32_t found = 0;
  for (int64_t p0 = 0; p0 < p.pages && found < asked; p0 += kScanLanes * kScanPages) {
    const int64_t first = p0 + lane_first;
    if (p0 > 0) c.load(p.counts, first, p.pages);
    uint32_t free = ~c.used() & pages_below(first, p.pages);
    uint32_t at = found + block_scan((uint32_t)__builtin_popcount(free), lds, &all);
    while (free != 0 && at < asked) {
      t.list[at++] = (int32_t)(first + __builtin_ctz(free));
      free &= free - 1;
    }
    found += all;
  }
  if (threadIdx.x == 0) t.found[0] = (int32_t)min(found, asked);
  if constexpr (ALONE) {
    __syncthreads();  // the lists are whole
    const Lanes me{(int)threadIdx.x & ((1 << log_lanes) - 1), 1 << log_lanes};
    const int i = (int)threadIdx.x >> log_lanes;
    if constexpr (FORK) {
      if (i < r.count) fork_row(p, r, t, to, i, me);
    } else {
      const int now = i <= r.count ? extend_row(p, r, t, to, i, me) : -1;
      __syncthreads();
      if (now >= 0 && me.lane == 0) p.lens[r.from[i]] = now;
    }
  }
}

constexpr int kRowLanes = 256;

// A workgroup a request (an extension's last one: the slots behind the last).
__global__ void __launch_bounds__(kRowLanes)
k_kv_pages_fork(Pool p, Requests r, Taken t, ForkTo to) {
  fork_row(p, r, t, to, (int)blockIdx.x, {(int)threadIdx.x, kRowLanes});
}
__global__ void __launch_bounds__(kRowLanes)
k_kv_pages_extend(Pool p, Requests r, Taken t, ExtendTo to) {
  const int now = extend_row(p, r, t, to, (int)blockIdx.x, {(int)threadIdx.x, kRowLanes});
  __syncthreads();
  if (now >= 0 && threadIdx.x == 0) p.lens[r.from[blockIdx.x]] = now;
}
// A workgroup a sequence that ends.  Its length is taken away first, so that a sequence that is named twice
// gives its pages back once.
__global__ void __launch_bounds__(kRowLanes)
k_kv_pages_free(Pool p, const int32_t* sequences) {
  __shared__ int32_t len;
  const int s = sequences[blockIdx.x];
  if (!row_ok(p, s)) return;
  if (threadIdx.x == 0) {
    const int32_t n = p.lens[s];
    len = n > 0 && len_ok(p, n) && atomicCAS(&p.lens[s], n, 0) == n ? n : 0;
  }
  __syncthreads();
  if (len <= 0) return;
  const int64_t held = pages_of(len, p.page_size);
  int32_t* row = p.table + s * p.stride;
  for (int c = (int)threadIdx.x; c < p.columns; c += kRowLanes) {
    const int32_t page = row[c];
    if (c < held && page >= 0 && page < p.pages) atomicSub(&p.counts[page], 1);
    row[c] = -1;
  }
}

// ---- Compaction: U pages are in use.  Those at U and above go to the free ones below it, the highest to the
// lowest: a page in use with b in use before it is the (U - 1 - b)-th from the end, a free page f with b in use
// before it the (f - b)-th hole.
constexpr int kMoveLanes = kScanLanes, kMovePages = 4;  // pages a lane

// A workgroup 4096 pages.  Each counts the whole pool for itself (twice: all, and those below U; the first
// 65536 pages stay in registers): 8192 pages are 32 KiB from L2, where another launch would take longer.
__global__ void __launch_bounds__(kMoveLanes)
k_kv_pages_moves(const int32_t* __restrict__ counts, int64_t pages, int32_t* src, int32_t* dst,
                 int32_t* used, int32_t* moved) {
  __shared__ uint32_t lds[kScanWaves];
  constexpr int kKept = 4;
  constexpr int64_t kRound = kMoveLanes * kScanPages;
  const int64_t mine = (int64_t)blockIdx.x * (kMoveLanes * kMovePages), half = pages / 2;
  const int64_t lane_first = (int64_t)threadIdx.x * kScanPages;
  uint32_t kept[kKept];
  uint32_t in_use = 0, before = 0;  // before this workgroup's pages
#pragma unroll
  for (int r = 0; r < kKept; ++r) {
    kept[r] = 0;
    if (r * kRound >= pages) continue;
    PageCounts c;
    c.load(counts, r * kRound + lane_first, pages);
    kept[r] = c.used();
    const uint32_t n = (uint32_t)__builtin_popcount(kept[r]);
    in_use += n;
    if (r * kRound + lane_first < mine) before += n;
  }
  for (int64_t p0 = kKept * kRound; p0 < pages; p0 += kRound) {
    PageCounts c;
    c.load(counts, p0 + lane_first, pages);
    const uint32_t n = (uint32_t)__builtin_popcount(c.used());
    in_use += n;
    if (p0 + lane_first < mine) before += n;
  }
  block_scan(in_use, lds, &in_use);
  block_scan(before, lds, &before);
  uint32_t below = 0;
#pragma unroll
  for (int r = 0; r < kKept; ++r) {
    below += __builtin_popcount(kept[r] & pages_below(r * kRound + lane_first, in_use));
  }
  for (int64_t p0 = kKept * kRound; p0 < in_use; p0 += kRound) {
    PageCounts c;
    c.load(counts, p0 + lane_first, pages);
    below += __builtin_popcount(c.used() & pages_below(p0 + lane_first, in_use));
  }
  block_scan(below, lds, &below);
  const int64_t moves = in_use - below;
  const int64_t first = mine + (int64_t)threadIdx.x * kMovePages;
  int32_t c[kMovePages];
  uint32_t here = 0, all;
#pragma unroll
  for (int k = 0; k < kMovePages; ++k) {
    c[k] = first + k < pages ? counts[first + k] : 0;
    here += c[k] > 0;
  }
  before += block_scan(here, lds, &all);
#pragma unroll
  for (int k = 0; k < kMovePages; ++k) {
    const int64_t p = first + k;
    if (p >= pages) break;
    int64_t rank = -1;
    if (c[k] > 0) {
      if (p >= in_use) {
        rank = (int64_t)in_use - 1 - before;
        src[rank] = (int32_t)p;
      }
      ++before;
    } else if (p < in_use) {
      dst[p - before] = (int32_t)p;
    }
    moved[p] = (int32_t)rank;
    // the lists have half as many places as there are pages
    if (p < half && p >= moves) src[p] = dst[p] = -1;
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) used[0] = (int32_t)in_use;
}

// The table's pages and the counts where they are now.
__global__ void __launch_bounds__(kRowLanes)
k_kv_pages_move(Pool p, const int32_t* src, const int32_t* dst, const int32_t* moved, int64_t places) {
  const int64_t i = (int64_t)blockIdx.x * kRowLanes + threadIdx.x;
  const int64_t half = p.pages / 2;
  if (i < half && src[i] >= 0) {
    p.counts[dst[i]] = p.counts[src[i]];
    p.counts[src[i]] = 0;
  }
  if (i < places) {
    const int64_t row = i / p.columns;
    int32_t* at = p.table + row * p.stride + (i - row * p.columns);
    const int32_t page = *at;
    if (page >= 0 && page < p.pages && moved[page] >= 0) *at = dst[moved[page]];
  }
}

// ---------------------------------------------------------------------------------------------
// Host side.

namespace {

// Requests, workgroups of a launch (which takes fewer than 2^32 threads, one request's more among them).
constexpr int64_t kMostCount = ((int64_t)1 << 24) - 2;

int pool_of(const char* name, const mcop_kv_pool* in, bool lens, Pool* out) {
  if (!in) return set_error(MCOP_E_INVALID, "%s: null pointer", name);
  if (in->num_rows < 0 || in->num_rows > INT32_MAX || in->table_columns < 0 ||
      in->table_columns > INT32_MAX || in->table_row_stride < 0 ||
      (in->num_rows > 0 && in->table_row_stride > INT64_MAX / 8 / in->num_rows) || in->num_pages < 0 ||
      in->num_pages > INT32_MAX || in->page_size <= 0 || in->page_size > INT32_MAX) {
    return set_error(MCOP_E_INVALID, "%s: bad pool: %lld rows of %lld pages, %lld pages of %lld tokens",
                     name, (long long)in->num_rows, (long long)in->table_columns,
                     (long long)in->num_pages, (long long)in->page_size);
  }
  if ((!in->block_table && in->num_rows > 0 && in->table_columns > 0) ||
      (lens && !in->seq_lens && in->num_rows > 0) || (!in->ref_counts && in->num_pages > 0)) {
    return set_error(MCOP_E_INVALID, "%s: null pointer", name);
  }
  *out = Pool{in->block_table, in->table_row_stride, (int)in->num_rows, (int)in->table_columns,
              in->seq_lens, in->ref_counts, (int)in->num_pages, (int)in->page_size};
  return MCOP_OK;
}

int count_ok(const char* name, int64_t n) {
  if (n < 0 || n > kMostCount) {
    return set_error(MCOP_E_INVALID, "%s: bad number of requests %lld (at most 2^24 - 2)", name,
                     (long long)n);
  }
  return MCOP_OK;
}

int workspace_ok(const char* name, const void* ws, int64_t bytes, int64_t requests, int64_t pages) {
  const int64_t need = mcop_kv_cache_pages_workspace(requests, pages);
  if (!ws || !aligned(16, ws) || bytes < need) {
    return set_error(MCOP_E_INVALID, "%s: the workspace must be %lld bytes at a multiple of 16", name,
                     (long long)need);
  }
  return MCOP_OK;
}

// Log of the lanes a request where the workgroup that takes the pages writes `requests` rows of at most
// `elements` too, kAloneSteps a lane; -1: another launch does.  Replayed from a graph, one launch against two:
// one token for each of 16 sequences 5.3 and 7.0 us, of 60 6.1 and 7.4; four forks of rows of 256 pages 5.3
// and 6.5, of 1000 (four steps a lane) 7.3 and 8.2; 16 of 250, also four steps, 7.6 and 7.1.
constexpr int kAloneSteps = 4;
int lanes_alone(int64_t requests, int64_t elements) {
  int log_lanes = 10;
  while (log_lanes >= 0 && requests << log_lanes > kScanLanes) --log_lanes;
  return log_lanes >= 0 && elements <= (int64_t)kAloneSteps << log_lanes ? log_lanes : -1;
}

}  // namespace

}  // namespace mcop

extern "C" int64_t mcop_kv_cache_pages_workspace(int64_t num_requests, int64_t num_pages) {
  using namespace mcop;
  if (num_requests < 0 || num_requests > kMostCount || num_pages < 0 || num_pages > INT32_MAX) {
    return set_error(MCOP_E_INVALID, "kv_cache_pages_workspace: %lld requests, %lld pages",
                     (long long)num_requests, (long long)num_pages);
  }
  return (4 + num_requests + num_pages) * 4;
}

extern "C" int mcop_kv_cache_copy_pages(const mcop_kv_pages* tensors, int64_t num_tensors,
                                        int64_t num_pages, const int32_t* src, const int32_t* dst,
                                        int64_t num_pairs, void* stream) {
  using namespace mcop;
  const char* name = "kv_cache_copy_pages";
  if (num_tensors < 0 || num_pages < 0 || num_pages > INT32_MAX || num_pairs < 0 ||
      num_pairs > INT32_MAX) {
    return set_error(MCOP_E_INVALID, "%s: bad shape num_tensors=%lld num_pages=%lld num_pairs=%lld", name,
                     (long long)num_tensors, (long long)num_pages, (long long)num_pairs);
  }
  if (num_tensors == 0 || num_pairs == 0 || num_pages == 0) return MCOP_OK;
  if (!tensors || !src || !dst) return set_error(MCOP_E_INVALID, "%s: null pointer", name);
  for (int64_t i = 0; i < num_tensors; ++i) {
    const mcop_kv_pages& t = tensors[i];
    if (!t.base || t.page_bytes <= 0 || t.page_stride < t.page_bytes ||
        t.page_stride > INT64_MAX / 4 / num_pages) {
      return set_error(MCOP_E_INVALID, "%s: tensor %lld: null pointer, or bad pages of %lld bytes %lld "
                       "apart", name, (long long)i, (long long)t.page_bytes, (long long)t.page_stride);
    }
  }
  auto st = static_cast<hipStream_t>(stream);
  for (int64_t i0 = 0; i0 < num_tensors; i0 += kCopyTensors) {
    CopyArgs a{};
    a.tensors = (int)std::min<int64_t>(kCopyTensors, num_tensors - i0);
    a.src = src, a.dst = dst, a.pairs = num_pairs, a.pages = num_pages;
    int64_t blocks = 0;
    constexpr int64_t kUnits = kCopyLanes * kCopyUnits;
    for (int i = 0; i < a.tensors; ++i) {
      const mcop_kv_pages& t = tensors[i0 + i];
      a.t[i] = CopyTensor{static_cast<uint8_t*>(t.base), t.page_stride, t.page_bytes};
      a.first[i] = (uint32_t)blocks;
      const int64_t units = t.page_bytes / 16;
      const int64_t per = units >= kUnits ? (units + kUnits - 1) / kUnits : 1;
      const int64_t pages = units >= kUnits ? 1 : kUnits / ((t.page_bytes + 15) / 16);
      const int64_t groups = (num_pairs + pages - 1) / pages;
      if (per > kMostCount || groups > kMostCount / per || blocks + groups * per >= kMostCount) {
        return set_error(MCOP_E_UNSUPPORTED, "%s: more bytes than one launch takes", name);
      }
      blocks += groups * per;
    }
    trace_launch(name, "%d tensors, %lld pairs, wgs=%lld", a.tensors, (long long)num_pairs,
                 (long long)blocks);
    hipLaunchKernelGGL(k_kv_copy_pages, dim3((unsigned)blocks), dim3(kCopyLanes), 0, st, a);
    if (int rc = check_launch(name)) return rc;
  }
  return MCOP_OK;
}

extern "C" int mcop_kv_cache_fork(const mcop_kv_pool* pool, const int32_t* parents,
                                  const int32_t* children, int64_t num_forks, int32_t* src,
                                  int32_t* dst, void* workspace, int64_t workspace_bytes,
                                  void* stream) {
  using namespace mcop;
  const char* name = "kv_cache_fork";
  Pool p;
  if (int rc = count_ok(name, num_forks)) return rc;
  if (num_forks == 0) return MCOP_OK;
  if (int rc = pool_of(name, pool, true, &p)) return rc;
  if (!parents || !children || !src || !dst) return set_error(MCOP_E_INVALID, "%s: null pointer", name);
  if (int rc = workspace_ok(name, workspace, workspace_bytes, num_forks, p.pages)) return rc;
  const Requests r{parents, children, nullptr, (int)num_forks};
  const Taken t(workspace, (int)num_forks);
  auto st = static_cast<hipStream_t>(stream);
  const ForkTo to{src, dst};
  const int log_lanes = lanes_alone(num_forks, p.columns);
  trace_launch(name, "%lld forks, %d pages, %s", (long long)num_forks, p.pages,
               log_lanes >= 0 ? "one launch" : "two launches");
  if (log_lanes >= 0) {
    hipLaunchKernelGGL((k_kv_pages_take<ForkTo, true>), dim3(1), dim3(kScanLanes), 0, st, p, r, t, to,
                       log_lanes);
    return check_launch(name);
  }
  hipLaunchKernelGGL((k_kv_pages_take<ForkTo, false>), dim3(1), dim3(kScanLanes), 0, st, p, r, t, to, 0);
  if (int rc = check_launch(name)) return rc;
  hipLaunchKernelGGL(k_kv_pages_fork, dim3((unsigned)num_forks), dim3(kRowLanes), 0, st, p, r, t, to);
  return check_launch(name);
}

extern "C" int mcop_kv_cache_extend(const mcop_kv_pool* pool, const int32_t* sequences,
                                    const int32_t* cu_tokens, int64_t num_sequences, int64_t* slots,
                                    int64_t num_tokens, int32_t* starts, void* workspace,
                                    int64_t workspace_bytes, void* stream) {
  using namespace mcop;
  const char* name = "kv_cache_extend";
  Pool p;
  if (int rc = count_ok(name, num_sequences)) return rc;
  if (num_tokens < 0) return set_error(MCOP_E_INVALID, "%s: bad num_tokens %lld", name, (long long)num_tokens);
  if (num_sequences == 0 && num_tokens == 0) return MCOP_OK;
  if (int rc = pool_of(name, pool, true, &p)) return rc;
  if (!cu_tokens || (num_sequences > 0 && (!sequences || !starts)) || (!slots && num_tokens > 0)) {
    return set_error(MCOP_E_INVALID, "%s: null pointer", name);
  }
  if (int rc = workspace_ok(name, workspace, workspace_bytes, num_sequences, p.pages)) return rc;
  const Requests r{sequences, nullptr, cu_tokens, (int)num_sequences};
  const Taken t(workspace, (int)num_sequences);
  auto st = static_cast<hipStream_t>(stream);
  const ExtendTo to{slots, num_tokens, starts};
  const int log_lanes = lanes_alone(num_sequences + 1, num_tokens);
  trace_launch(name, "%lld sequences, %lld tokens, %d pages, %s", (long long)num_sequences,
               (long long)num_tokens, p.pages, log_lanes >= 0 ? "one launch" : "two launches");
  if (log_lanes >= 0) {
    hipLaunchKernelGGL((k_kv_pages_take<ExtendTo, true>), dim3(1), dim3(kScanLanes), 0, st, p, r, t, to,
                       log_lanes);
    return check_launch(name);
  }
  hipLaunchKernelGGL((k_kv_pages_take<ExtendTo, false>), dim3(1), dim3(kScanLanes), 0, st, p, r, t, to, 0);
  if (int rc = check_launch(name)) return rc;
  hipLaunchKernelGGL(k_kv_pages_extend, dim3((unsigned)num_sequences + 1), dim3(kRowLanes), 0, st, p, r,
                     t, to);
  return check_launch(name);
}

extern "C" int mcop_kv_cache_free(const mcop_kv_pool* pool, const int32_t* sequences,
                                  int64_t num_sequences, void* stream) {
  using namespace mcop;
  const char* name = "kv_cache_free";
  Pool p;
  if (int rc = count_ok(name, num_sequences)) return rc;
  if (num_sequences == 0) return MCOP_OK;
  if (int rc = pool_of(name, pool, true, &p)) return rc;
  if (!sequences) return set_error(MCOP_E_INVALID, "%s: null pointer", name);
  trace_launch(name, "%lld sequences", (long long)num_sequences);
  hipLaunchKernelGGL(k_kv_pages_free, dim3((unsigned)num_sequences), dim3(kRowLanes), 0,
                     static_cast<hipStream_t>(stream), p, sequences);
  return check_launch(name);
}

extern "C" int mcop_kv_cache_compact(const mcop_kv_pool* pool, int32_t* src, int32_t* dst,
                                     int32_t* used, void* workspace, int64_t workspace_bytes,
                                     void* stream) {
  using namespace mcop;
  const char* name = "kv_cache_compact";
  Pool p;
  if (int rc = pool_of(name, pool, false, &p)) return rc;
  if (!used || (p.pages > 1 && (!src || !dst))) {
    return set_error(MCOP_E_INVALID, "%s: null pointer", name);
  }
  if (int rc = workspace_ok(name, workspace, workspace_bytes, 0, p.pages)) return rc;
  const int64_t places = (int64_t)p.rows * p.columns;
  const int64_t threads = std::max(places, (int64_t)p.pages / 2);
  if (threads >= ((int64_t)1 << 32) - kRowLanes) {
    return set_error(MCOP_E_UNSUPPORTED, "%s: a table of %lld places is more than one launch takes", name,
                     (long long)places);
  }
  int32_t* moved = static_cast<int32_t*>(workspace);
  auto st = static_cast<hipStream_t>(stream);
  constexpr int kPages = kMoveLanes * kMovePages;
  trace_launch(name, "%d pages, a table of %d x %d", p.pages, p.rows, p.columns);
  const unsigned blocks = (unsigned)std::max<int64_t>(1, ((int64_t)p.pages + kPages - 1) / kPages);
  hipLaunchKernelGGL(k_kv_pages_moves, dim3(blocks), dim3(kMoveLanes), 0, st, p.counts, (int64_t)p.pages, src,
                     dst, used, moved);
  if (int rc = check_launch(name)) return rc;
  if (threads == 0) return MCOP_OK;
  hipLaunchKernelGGL(k_kv_pages_move, dim3((unsigned)((threads + kRowLanes - 1) / kRowLanes)),
                     dim3(kRowLanes), 0, st, p, src, dst, moved, places);
  return check_launch(name);
}
