// The cache's attention and page entry points over a grid of shapes, types, alignments and strides, under
// AddressSanitizer and UndefinedBehaviorSanitizer, with device pointers that host code never dereferences
// and no device to launch on. Each call ends in a documented status: 0 where there is nothing to do,
// MCOP_E_INVALID or MCOP_E_UNSUPPORTED from the checks, or MCOP_E_LAUNCH once everything is checked and
// chosen and the launch fails; each failure leaves a message. Any sanitizer report ends the run with a
// non-zero status.
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <initializer_list>
#include <vector>

#include "../../include/mcop_norm.h"

namespace {

int g_calls = 0, g_fail = 0;
int g_status[4] = {0, 0, 0, 0};  // counts of 0, -1, -2, -3

template <class T = void>
T* dev(int slot, int mis = 0) {
  return reinterpret_cast<T*>(static_cast<uintptr_t>(0x7f0000000000ull) +
                              static_cast<uintptr_t>(slot) * 0x100000000ull + static_cast<uintptr_t>(mis));
}

void expect(int rc, bool empty, const char* what, int64_t a, int64_t b, int64_t c) {
  ++g_calls;
  const size_t len = strnlen(mcop_last_error(), 512);
  if (rc > 0 || rc < -3 || len >= 512 || (rc != MCOP_OK && len == 0) || (rc == MCOP_OK && !empty)) {
    ++g_fail;
    fprintf(stderr, "unexpected: %s %lld %lld %lld rc=%d\n", what, (long long)a, (long long)b,
            (long long)c, rc);
    return;
  }
  g_status[-rc] += 1;
}

const int64_t kFar = (int64_t)1 << 40;
const int64_t kMany[] = {0, 1, 5, 64, 3000000, (int64_t)1 << 24, ((int64_t)1 << 31) - 1, kFar};

}  // namespace

int main() {
  for (int64_t B : kMany) {
    for (int64_t heads : {(int64_t)0, (int64_t)1, (int64_t)8, (int64_t)700, kFar}) {
      for (int64_t group : {(int64_t)1, (int64_t)17, (int64_t)128, (int64_t)40000}) {
        for (int64_t D : {0, 1, 15, 16, 61, 64, 96, 192, 256, 320, 1024, 1025}) {
          for (mcop_dtype c : {MCOP_I8, MCOP_FP8_E4M3FN, MCOP_MXFP4, MCOP_F16}) {
            const int64_t queries = heads > 65536 ? heads : heads * group;
            for (int mis : {0, 3}) {
              const mcop_kv_side k{dev(0), queries * D, D,      dev(1, mis), 16 * heads * D,
                                   heads * D, D,      dev(2), 16 * heads,  heads,
                                   1,         D};
              mcop_kv_side v = k;
              v.head_size = D / 2 + 1;
              for (const mcop_kv_side* w : {&k, (const mcop_kv_side*)&v}) {
                for (mcop_dtype t : {MCOP_BF16, MCOP_F16, MCOP_F32, MCOP_I8}) {
                  const int64_t room = mcop_kv_cache_attention_workspace(heads, queries, w->head_size);
                  expect(mcop_kv_cache_attention(&k, w, c, 7, mis ? 16 : 5, heads, queries, dev<int32_t>(3),
                                                 9, mis ? 9 : 0, dev<int32_t>(4), B, 0.1f, mis * 100, t,
                                                 mis ? dev<float>(5) : nullptr, dev(6), room < 0 ? 0 : room,
                                                 nullptr),
                         B == 0, "kv_cache_attention", B, heads, D);
                }
              }
            }
          }
        }
      }
    }
  }
  for (int64_t n : kMany) {
    for (int64_t rows : kMany) {
      for (int64_t columns : kMany) {
        for (int64_t pages : kMany) {
          for (int64_t page : {(int64_t)0, (int64_t)1, (int64_t)16, kFar}) {
            const mcop_kv_pool pool{dev<int32_t>(0), columns, rows, columns, dev<int32_t>(1),
                                    dev<int32_t>(2), pages, page};
            const int64_t room = mcop_kv_cache_pages_workspace(n, pages);
            const int64_t bytes = room < 0 ? 0 : room;
            expect(mcop_kv_cache_fork(&pool, dev<int32_t>(3), dev<int32_t>(4), n, dev<int32_t>(5),
                                      dev<int32_t>(6), dev(7), bytes, nullptr),
                   n == 0, "kv_cache_fork", n, rows, pages);
            expect(mcop_kv_cache_extend(&pool, dev<int32_t>(3), dev<int32_t>(4), n, dev<int64_t>(5), columns,
                                        dev<int32_t>(6), dev(7), bytes, nullptr),
                   n == 0 && columns == 0, "kv_cache_extend", n, rows, pages);
            expect(mcop_kv_cache_free(&pool, dev<int32_t>(3), n, nullptr), n == 0, "kv_cache_free", n, rows,
                   pages);
            expect(mcop_kv_cache_compact(&pool, dev<int32_t>(3), dev<int32_t>(4), dev<int32_t>(5), dev(7),
                                         bytes, nullptr),
                   false, "kv_cache_compact", n, rows, pages);
          }
        }
      }
    }
    for (int64_t tensors : {0, 1, 63, 64, 65, 200}) {
      for (int64_t bytes : {(int64_t)0, (int64_t)1, (int64_t)15, (int64_t)16, (int64_t)16383, (int64_t)16384,
                            (int64_t)100000, kFar, INT64_MAX}) {
        std::vector<mcop_kv_pages> list((size_t)tensors, mcop_kv_pages{dev(0), bytes, bytes});
        for (int64_t pages : kMany) {
          expect(mcop_kv_cache_copy_pages(list.data(), tensors, pages, dev<int32_t>(1), dev<int32_t>(2), n,
                                          nullptr),
                 n == 0 || tensors == 0 || pages == 0, "kv_cache_copy_pages", n, bytes, pages);
        }
      }
    }
  }
  printf("calls %d: ok %d, invalid %d, unsupported %d, launch %d; unexpected %d\n", g_calls,
         g_status[0], g_status[1], g_status[2], g_status[3], g_fail);
  return g_fail == 0 ? 0 : 1;
}
