// What the append kernels share: launch-time index division, read-only vector
// loads and the error bits that refuse a batch.
#pragma once

#include "common.cuh"

namespace iris {

// Division of non-negative 32-bit integers n < 2^31 by a divisor fixed at
// launch: q = (umulhi(n, m) + n) >> l with l = ceil(log2 d) and
// m = floor(2^32 (2^l - d) / d) + 1 (Granlund & Montgomery, "Division by
// Invariant Integers using Multiplication", 1994).
struct FastDiv {
  uint32_t d, m, l;
  static FastDiv make(uint32_t d) {
    FastDiv f;
    f.d = d;
    f.l = 0;
    while ((1ull << f.l) < d) ++f.l;
    f.m = static_cast<uint32_t>(((1ull << 32) * ((1ull << f.l) - d)) / d + 1);
    return f;
  }
  IRIS_DEV uint32_t div(uint32_t n) const { return (__umulhi(n, m) + n) >> l; }
};

// Batches of at most this many tokens are validated inside the append kernel
// (ranges and duplicate slots, by every CTA), with no check kernel before it.
constexpr int64_t kInlineCheckTokens = IRIS_APPEND_INLINE_CHECK_TOKENS;

// 32-byte read-only load (sm_100 vector width), 32-byte aligned address.
IRIS_DEV void ldg_nc_v8(const void* p, uint4& a, uint4& b) {
  asm volatile("ld.global.nc.v8.u32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(a.x), "=r"(a.y), "=r"(a.z), "=r"(a.w), "=r"(b.x), "=r"(b.y), "=r"(b.z), "=r"(b.w)
               : "l"(p));
}

IRIS_DEV uint4 ldg_nc_v4(const void* p) {
  uint4 r;
  asm volatile("ld.global.nc.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "l"(p));
  return r;
}

// A batch with one of these bits in the error word is not written.
constexpr int32_t kRejectBits = IRIS_ERR_SLOT_RANGE | IRIS_ERR_POS_NEGATIVE | IRIS_ERR_POS_RANGE | IRIS_ERR_DUP_SLOT;

}  // namespace iris
