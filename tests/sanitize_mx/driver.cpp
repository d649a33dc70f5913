// The 4-bit operators' and the quantized cache's C entry points over a grid of shapes, types,
// alignments and strides, under AddressSanitizer and UndefinedBehaviorSanitizer, with device pointers
// that host code never dereferences and no device to launch on. Each call ends in a documented
// status: 0 where there is nothing to do, MCOP_E_INVALID or MCOP_E_UNSUPPORTED from the checks, or
// MCOP_E_LAUNCH once everything is checked and chosen and the launch fails; each failure leaves a
// message. Any sanitizer report ends the run with a non-zero status.
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <initializer_list>

#include "../../include/mcop_norm.h"

namespace {

int g_calls = 0, g_fail = 0;
int g_status[4] = {0, 0, 0, 0};  // counts of 0, -1, -2, -3

void* dev(int slot, int mis = 0) {
  return reinterpret_cast<void*>(static_cast<uintptr_t>(0x7f0000000000ull) +
                                 static_cast<uintptr_t>(slot) * 0x100000000ull +
                                 static_cast<uintptr_t>(mis));
}
uint8_t* bytes(int slot, int mis = 0) { return static_cast<uint8_t*>(dev(slot, mis)); }

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

const int64_t kRows[] = {0, 1, 5, 64, 300, 8192, (int64_t)1 << 20, (int64_t)1 << 31, (int64_t)1 << 40};
const int64_t kWide[] = {0, 31, 32, 96, 5152, 8192, 65536, 131104, (int64_t)1 << 24,
                         ((int64_t)1 << 31) - 32, (int64_t)1 << 40};
const mcop_dtype kAll[] = {MCOP_BF16, MCOP_F16, MCOP_F32, MCOP_I8, MCOP_FP8_E4M3FN, MCOP_MXFP4};

}  // namespace

int main() {
  for (int64_t T : kRows) {
    for (int64_t H : kWide) {
      for (mcop_dtype t : kAll) {
        for (int mis : {0, 2, 4}) {
          expect(mcop_mxfp4_quant(bytes(0), bytes(1), dev(2, mis), T, H, H + mis, t, nullptr), T == 0,
                 "mxfp4_quant", T, H, t);
          expect(mcop_mxfp4_dequant(dev(0, mis), t, bytes(1), bytes(2), T, H, nullptr), T == 0,
                 "mxfp4_dequant", T, H, t);
          for (int res = 0; res < 2; ++res) {
            expect(mcop_rms_norm_mxfp4_quant(bytes(0), bytes(1), dev(2, mis), dev(3),
                                             res ? dev(4) : nullptr, res ? dev(5) : nullptr, T, H,
                                             t, 1e-6f, nullptr),
                   T == 0, "rms_norm_mxfp4_quant", T, H, t);
          }
        }
        for (int64_t N : kRows) {
          expect(mcop_mxfp4_scaled_mm(dev(0), t, bytes(1), bytes(2), bytes(3), bytes(4, 1),
                                      T & 1 ? dev(5) : nullptr, T, N, H, nullptr),
                 T == 0 || N == 0, "mxfp4_scaled_mm", T, N, H);
        }
      }
    }
  }
  for (int64_t T : kRows) {
    for (int64_t heads : {(int64_t)0, (int64_t)1, (int64_t)2, (int64_t)8, (int64_t)100000,
                          (int64_t)1 << 26, (int64_t)1 << 30}) {
      for (int64_t D : {0, 8, 32, 61, 64, 128, 576, 1024, 1025}) {
        for (mcop_dtype c : {MCOP_I8, MCOP_FP8_E4M3FN, MCOP_MXFP4, MCOP_BF16}) {
          for (int mis : {0, 1}) {
            const mcop_kv_side k{dev(0), heads * D, D,       bytes(1, mis), 16 * heads * D,
                                 heads * D, D,      dev(2), 16 * heads,    heads,
                                 1,         D};
            mcop_kv_side v = k;
            v.head_size = D / 2 + 1;
            for (const mcop_kv_side* w : {&k, (const mcop_kv_side*)&v}) {
              for (mcop_dtype t : {MCOP_BF16, MCOP_F32, MCOP_I8}) {
                for (int64_t pages : {(int64_t)0, (int64_t)7, (int64_t)1 << 28, (int64_t)1 << 31}) {
                  expect(mcop_kv_cache_write_quant(&k, w, c, pages, 16, heads, (const int64_t*)dev(3), T,
                                                   t, nullptr),
                         T == 0 || pages == 0, "kv_cache_write_quant", T, heads, D);
                }
                for (int64_t B : {0, 1, 9}) {
                  expect(mcop_kv_cache_read_dequant(&k, w, c, 7, 16, heads, (const int32_t*)dev(3), 5, 5,
                                                    (const int32_t*)dev(4),
                                                    B & 1 ? (const int32_t*)dev(5) : nullptr, B, T, t,
                                                    nullptr),
                         T == 0 || B == 0, "kv_cache_read_dequant", T, heads, D);
                }
              }
            }
          }
        }
      }
    }
  }
  const mcop_kv_side huge{dev(0), INT64_MAX, 1, dev(1), INT64_MAX / 2, 64, 64, dev(2), 1, 1, 1, 64};
  expect(mcop_kv_cache_write_quant(&huge, &huge, MCOP_I8, 4, 16, 2, (const int64_t*)dev(3), 4, MCOP_BF16,
                                   nullptr),
         false, "kv_cache_write_quant (strides)", 4, 2, 64);
  expect(mcop_kv_cache_write_quant(nullptr, nullptr, MCOP_I8, 4, 16, 2, nullptr, 4, MCOP_BF16, nullptr),
         false, "kv_cache_write_quant (null)", 4, 2, 64);
  expect(mcop_kv_cache_read_dequant(nullptr, nullptr, MCOP_I8, 4, 16, 2, nullptr, 1, 1, nullptr, nullptr,
                                    1, 4, MCOP_BF16, nullptr),
         false, "kv_cache_read_dequant (null)", 4, 2, 64);
  printf("calls %d: ok %d, invalid %d, unsupported %d, launch %d; unexpected %d\n", g_calls,
         g_status[0], g_status[1], g_status[2], g_status[3], g_fail);
  return g_fail == 0 ? 0 : 1;
}
