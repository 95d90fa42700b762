// The page index of the INT4 paged cache, and the selection of pages by it.
//
// Bounds.  Per physical page and KV head: lo_d <= k_d <= hi_d over the page's
// stored keys k (value = nibble * group scale) in every dim d, held as 8-bit
// codes of one fp32 step: step = max_d(|lo_d|, |hi_d|) / 127, codes
// floor(lo / step) and ceil(hi / step), rounded outwards so that the codes
// still bound the keys, each division rounded once.
//
// Score.  For a query head q held in 8-bit codes c = rint(q / unit), unit =
// max|q| / 127, no key of the page has a larger (quantised) product with q
// than  sum_d max(c_d lo_d, c_d hi_d) = min(c, 0) . lo + max(c, 0) . hi:
// a product of length 2 D of whole numbers, below 2^24 for D <= 256, so its
// value does not depend on the order of its additions.  The page's score for
// a KV head is the maximum over the head's query heads of
// (sum * step) * unit, fp32.
//
// Selection.  Per sequence and KV head the max_pages highest scores, the
// first sink_pages and last recent_pages before all others, ties to the
// lowest page; written in rising order.
//
// Measured (B200, 8 KV heads of 128 dims).  Bounds of 16 sequences of up to
// 8191 tokens: 36.5 us, 3.1 TB/s, the integer and minimum pipe at two thirds:
// 7.7 instructions a key and dim, of which the product, the minimum and the
// maximum are 2 and the unpacking 2; the others are the codes' quotients, the
// finiteness of the scales and the next page's words moved to their place.
// Of one new page in each of 64 sequences 3.1 us.  Scores and selection over
// 64 sequences of up to 16384 tokens: 32.9 us, 3.7 TB/s; the scores take 26 of
// them, 23 at 5.4 TB/s behind a start of 3.5.  One sequence of 131072 tokens
// 11.1 us, two launches and their chains of dependent loads; of 524288 tokens
// 20.9, and of one page more 132: past 32768 pages a row is one CTA's, which reads
// its keys again in every round.
#include <mutex>
#include <set>
#include <utility>

#include "elem.cuh"
#include "key_range.h"

namespace iris {
namespace {

constexpr int kPage = 16;
constexpr int kBoundsCtas = 4;  // CTAs an SM of the bounds kernel: one wave (5 to 8: 1 us more for a step, no less for all)

// ------------------------------------------------------------------ bounds
struct BoundsParams {
  const uint8_t* k_data;
  const __half* k_scale;
  const int32_t* block_table;
  int64_t table_stride;
  const int32_t* seq_lens;
  const int32_t* first_token;  // NULL: every page
  int8_t* bounds;
  float* step;
  __half* values;  // NULL: not wanted
  int64_t num_pages;
  int32_t max_pages;
  int32_t kv_heads;
  int32_t* err;
};

// a / b rounded once, from r = the correctly rounded 1 / b: the first residual
// step makes the quotient faithful, the second one correctly rounded
// (Markstein 1990).
IRIS_DEV float quotient(float a, float b, float r) {
  float t = __fmul_rn(a, r);
  t = fmaf(fmaf(-t, b, a), r, t);
  return fmaf(fmaf(-t, b, a), r, t);
}

IRIS_DEV float min3(float a, float b, float c) {
  float d;
  asm("min.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
IRIS_DEV float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// The lowest bytes of four words.
IRIS_DEV uint32_t low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return prmt(prmt(a, b, 0x0040), prmt(c, d, 0x0040), 0x5410);
}

// A product of two fp16 in fp32: exact, one operation.
IRIS_DEV float product(__half a, __half b) {
  float d;
  asm("fma.rn.f32.f16 %0, %1, %2, %3;" : "=f"(d) : "h"(__half_as_ushort(a)), "h"(__half_as_ushort(b)), "f"(0.0f));
  return d;
}

// A CTA takes every gridDim.x-th of a sequence's pages, one thread per 8 dims
// of one head; the D / 8 threads of a head are adjacent lanes.  The 16 words
// and 16 scales of a thread's next page are asked for before the present one
// is worked on, so that one wave of CTAs does: more would only come and go
// where a decode step has one new page a sequence.  Two nibbles become fp16
// with two operations, a product takes one, and two tokens one three-way
// minimum and maximum: it is these that bound the kernel, not the bytes.
template <int D>
__global__ void __launch_bounds__(256, 2) bounds_kernel(const BoundsParams p) {
  constexpr int V = D / 8;
  grid_dependency_wait();
  const int b = blockIdx.y;
  const int len = __ldg(p.seq_lens + b);
  const int from = p.first_token != nullptr ? max(0, __ldg(p.first_token + b)) / kPage : 0;
  if (len <= 0) {
    if (len < 0 && blockIdx.x == 0 && threadIdx.x == 0) set_error(p.err, IRIS_ERR_SEQ_NEGATIVE);
    return;
  }
  int last = (len - 1) / kPage;
  if (last >= p.max_pages) {
    if (blockIdx.x == 0 && threadIdx.x == 0) set_error(p.err, IRIS_ERR_BLOCK_TABLE);
    last = p.max_pages - 1;
  }
  const int vecs = p.kv_heads * V;
  const int32_t* table = p.block_table + b * p.table_stride;
  const int step0 = static_cast<int>(blockDim.x), stride = static_cast<int>(gridDim.x);
  // Whole warps go round together, over the pages and over the vectors where a page has more than the CTA threads:
  // lanes past the last vector repeat it and store nothing.
  const int lane = threadIdx.x & 31;
  int next_col = from + static_cast<int>(blockIdx.x), next_i0 = static_cast<int>(threadIdx.x) - lane;
  const auto page_at = [&](int col) -> int32_t { return col <= last ? __ldg(table + col) : -1; };
  int32_t next_page = page_at(next_col), page_after = page_at(next_col + stride);
  uint32_t w[kPage];
  unsigned short sh[kPage];
  const auto load = [&]() {  // what next_col and next_i0 say
    if (next_col > last || next_page < 0 || next_page >= p.num_pages || next_i0 >= vecs) return;
    const int i = min(next_i0 + lane, vecs - 1);
    const int final_token = min(kPage, len - next_col * kPage) - 1;
    const uint32_t* src = reinterpret_cast<const uint32_t*>(p.k_data) + static_cast<int64_t>(next_page) * kPage * vecs + i;
    const unsigned short* scl = reinterpret_cast<const unsigned short*>(p.k_scale) +
                                static_cast<int64_t>(next_page) * kPage * (vecs >> 2) + (i >> 2);
#pragma unroll
    for (int t = 0; t < kPage; ++t) {  // tokens past the last one repeat it
      const int tok = min(t, final_token);
      w[t] = __ldg(src + tok * vecs);
      sh[t] = __ldg(scl + tok * (vecs >> 2));
    }
  };
  load();
  while (next_col <= last) {
    const int i0 = next_i0;
    const int64_t page = next_page;
    const bool known = page >= 0 && page < p.num_pages, here = known && i0 < vecs;
    if (!known && threadIdx.x == 0) set_error(p.err, IRIS_ERR_PAGE_ID);
    uint32_t cw[kPage];
    unsigned short cs[kPage];
#pragma unroll
    for (int t = 0; t < kPage; ++t) cw[t] = w[t], cs[t] = sh[t];
    next_i0 += step0;
    if (next_i0 >= vecs || !known) {
      next_i0 = static_cast<int>(threadIdx.x) - lane;
      next_col += stride;
      next_page = page_after;
      page_after = page_at(next_col + stride);
    }
    load();
    if (here) {
      const int i = min(i0 + lane, vecs - 1);
      const bool mine = i0 + lane < vecs;
      float lo[8], hi[8], bad = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        lo[j] = INFINITY;
        hi[j] = -INFINITY;
      }
#pragma unroll
      for (int t = 0; t < kPage; t += 2) {
        bad = fmaf(__half2float(__ushort_as_half(cs[t])), 0.0f, bad);  // NaN from a scale that is not finite
        bad = fmaf(__half2float(__ushort_as_half(cs[t + 1])), 0.0f, bad);
        float x[2][8];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t v = cw[t + e], u = v >> 8;
          const uint32_t n[4] = {int4_lo_exact(v), int4_hi_exact(v), int4_lo_exact(u), int4_hi_exact(u)};
          const __half s = __ushort_as_half(cs[t + e]);
#pragma unroll
          for (int j = 0; j < 4; ++j) {  // dims j and j + 4
            x[e][j] = product(__low2half(u32_as_h2(n[j])), s);
            x[e][j + 4] = product(__high2half(u32_as_h2(n[j])), s);
          }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          lo[j] = min3(lo[j], x[0][j], x[1][j]);
          hi[j] = max3(hi[j], x[0][j], x[1][j]);
        }
      }
      float m = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) m = max3(m, -lo[j], hi[j]);
      if (bad != bad) m = INFINITY;
#pragma unroll
      for (int o = 1; o < V; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      const bool finite = m <= 3.0e38f;
      const float step = finite ? __fdiv_rn(m, 127.0f) : INFINITY;
      const float unit = finite && step > 0.0f ? step : 1.0f;  // (a head of zeros: lo = hi = 0)
      const float r = __frcp_rn(unit);
      const float kMagic = 12582912.0f;  // 1.5 2^23: a sum's low byte is the rounded value's
      if (!finite) {
#pragma unroll
        for (int j = 0; j < 8; ++j) lo[j] = -127.0f, hi[j] = 127.0f;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        // (a quotient passes 127 by less than a step: the rounded-outward one is held to it)
        lo[j] = fmaxf(__fadd_rd(quotient(lo[j], unit, r), kMagic), kMagic - 127.0f);
        hi[j] = fminf(__fadd_ru(quotient(hi[j], unit, r), kMagic), kMagic + 127.0f);
      }
      if (mine) {
        const int h = i / V, v = i - h * V;
        const int64_t head = page * p.kv_heads + h;
        const auto bytes = [&](const float (&z)[8]) {
          uint32_t c[2];
#pragma unroll
          for (int j = 0; j < 2; ++j)
            c[j] = low_bytes(__float_as_uint(z[4 * j]), __float_as_uint(z[4 * j + 1]), __float_as_uint(z[4 * j + 2]),
                             __float_as_uint(z[4 * j + 3]));
          return make_uint2(c[0], c[1]);
        };
        uint2* out = reinterpret_cast<uint2*>(p.bounds + head * 2 * D) + v;
        out[0] = bytes(lo);
        out[V] = bytes(hi);
        if (v == 0) p.step[head] = step;
        if (p.values != nullptr) {
          const auto value = [&](const float (&z)[8], int j) {
            const float2 c = __fadd2_rn(make_float2(z[2 * j], z[2 * j + 1]), make_float2(-kMagic, -kMagic));
            const float2 x = __fmul2_rn(c, make_float2(step, step));
            return Fp16Elem::pack(x.x, x.y);
          };
          uint4* val = reinterpret_cast<uint4*>(p.values + head * 2 * D) + v;
          val[0] = make_uint4(value(lo, 0), value(lo, 1), value(lo, 2), value(lo, 3));
          val[V] = make_uint4(value(hi, 0), value(hi, 1), value(hi, 2), value(hi, 3));
        }
      }
    }
  }
}

// ------------------------------------------------------------------- score
struct ScoreParams {
  const void* query;
  const int8_t* bounds;
  const float* step;
  const int32_t* block_table;
  int64_t table_stride;
  const int32_t* seq_lens;
  uint32_t* keys;  // [B, Hkv, key_stride]: the scores as ordered integers
  int64_t key_stride;
  int64_t num_pages;
  int32_t max_pages;
  int32_t kv_heads, group;
  int32_t cta_heads;  // KV heads per CTA
  int32_t max_keep;
  int32_t* err;
};

constexpr int kScoreWarps = 8;
constexpr int kScoreStages = 2;  // units of a warp in flight and in use

// Two adjacent k-steps of m16n8k32 share one 16-byte load a lane: lane t of
// a quad holds bytes 16 t .. 16 t + 15 of a 64-byte span of its page, words 0
// and 1 of which are one product's two A registers of that page and words 2
// and 3 the next one's.  The query's codes are read with the same assignment,
// so the sum runs over the span in another order than in memory, which whole
// numbers do not mind.
IRIS_DEV void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// fp32 -> unsigned with the same order (no NaN; -0 is made +0 first).
IRIS_DEV uint32_t ordered(float f) {
  const uint32_t u = __float_as_uint(f + 0.0f);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// A ring slot: each lane's 16-byte pieces of its two pages, then their steps.
template <int D>
constexpr int kSlotBytes = 2 * (2 * D / 64 * 512 + 128);

IRIS_DEV void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
IRIS_DEV void copy4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}

// One CTA a part of one sequence's pages and some of its KV heads; its warps
// share the units, (KV head, 16 pages).  A unit's bounds are a product of 16
// rows (pages) x 8 columns (query heads; kWide, more than 8 a KV head: two of
// them); the unit after it is on its way to shared memory.
template <typename E, int D, bool kWide>
__global__ void __launch_bounds__(32 * kScoreWarps, 3) score_kernel(const ScoreParams p) {
  // codes of the query heads: [Hq][min(c, 0) : D][max(c, 0) : D], rows padded by 16 bytes; their units;
  // the warps' rings
  extern __shared__ __align__(16) uint8_t smem[];
  constexpr int kRow = 2 * D + 16;
  constexpr int kSpans = 2 * D / 64;
  grid_dependency_wait();
  grid_dependents_launch();  // the selection may come up meanwhile
  const int b = blockIdx.y;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int head0 = blockIdx.z * p.cta_heads;  // this CTA's first KV head
  const int len = __ldg(p.seq_lens + b);
  // the warp's first query heads (heads warp, warp + 8, ..) are asked for together with the length
  const int heads = p.cta_heads * p.group;
  constexpr int W = D / 64;  // words a lane
  constexpr int kAtOnce = 4;
  uint32_t q[kAtOnce][W];
  const auto load_queries = [&](int i0) {
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      const int i = i0 + j * kScoreWarps;
#pragma unroll
      for (int k = 0; k < W; ++k)
        q[j][k] = i < heads ? __ldg(static_cast<const uint32_t*>(p.query) +
                                    ((static_cast<int64_t>(b) * p.kv_heads + head0) * p.group + i) * (D / 2) + lane * W + k)
                            : 0u;
    }
  };
  load_queries(warp);
  const bool first = blockIdx.x == 0 && blockIdx.z == 0 && threadIdx.x == 0;
  if (len < 0 && first) set_error(p.err, IRIS_ERR_SEQ_NEGATIVE);
  const int64_t all = len > 0 ? (static_cast<int64_t>(len) + kPage - 1) / kPage : 0;
  if (all > p.max_pages && first) set_error(p.err, IRIS_ERR_BLOCK_TABLE);
  const int n = static_cast<int>(all < p.max_pages ? all : p.max_pages);
  const int sixteens = (n + 15) / 16, share = (sixteens + gridDim.x - 1) / gridDim.x, unit0 = blockIdx.x * share;
  if (n <= p.max_keep || unit0 >= sixteens) return;  // every page is kept, or none of these exist
  const int g = lane >> 2, t = lane & 3;
  const int count = min(share, sixteens - unit0);  // a head
  const int total = p.cta_heads * count;           // a contiguous run of them for each warp
  const int lo = total * warp / kScoreWarps, hi = total * (warp + 1) / kScoreWarps;
  // Page numbers are asked for a unit before the copies that need them.
  const int page0 = unit0 * 16 + g;  // this lane's first page; its others: 8 after it, and 16 a unit on
  const int32_t* table = p.block_table + b * p.table_stride + page0;
  const auto page_of = [&](int u, int half) -> int32_t {
    return page0 + 16 * u + 8 * half < n ? __ldg(table + 16 * u + 8 * half) : 0;
  };
  int h1 = lo / count, u1 = lo - h1 * count;  // the unit whose bounds are loaded next
  const auto advance = [&](int& h, int& u) {
    if (++u == count) {
      u = 0;
      ++h;
    }
  };
  int h = h1, u = u1;
  int32_t page[2] = {0, 0}, after[2] = {0, 0};  // its pages, and those of the unit after it
  if (lo < hi) {
    page[0] = page_of(u1, 0);
    page[1] = page_of(u1, 1);
  }
  uint8_t* codes = smem;
  float* units = reinterpret_cast<float*>(smem + heads * kRow);  // [Hq]
  // A lane copies and reads back its own 16 bytes of each span, so that a slot needs no barrier.
  uint8_t* ring = smem + (heads * (kRow + 4) + 15) / 16 * 16 + warp * kScoreStages * kSlotBytes<D> + 16 * lane;
  const int8_t* bounds = p.bounds + 16 * t;
  const uint32_t page_bytes = static_cast<uint32_t>(p.kv_heads) * (2 * D);  // (at most 2^14 heads)
  int fill = 0;  // the slot of the unit that is loaded next
  const auto load_unit = [&](int i) {
    if (i < hi) {
      const int head = head0 + h1;
      const uint32_t dst = smem_u32(ring + fill * kSlotBytes<D>);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        if (page[half] < 0 || page[half] >= p.num_pages) {
          set_error(p.err, IRIS_ERR_PAGE_ID);
          page[half] = 0;
        }
        const int8_t* src = bounds + static_cast<int64_t>(page[half]) * page_bytes + head * (2 * D);
#pragma unroll
        for (int k = 0; k < kSpans; ++k) copy16(dst + 512 * (2 * k + half), src + 64 * k);
        copy4(dst + 1024 * kSpans + 128 * half - 12 * lane, p.step + static_cast<int64_t>(page[half]) * p.kv_heads + head);
        page[half] = after[half];
      }
      advance(h1, u1);
      if (i + 2 < hi) {
        int h2 = h1, u2 = u1;
        advance(h2, u2);
        after[0] = page_of(u2, 0);
        after[1] = page_of(u2, 1);
      }
      fill = fill + 1 == kScoreStages ? 0 : fill + 1;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  if (lo + 1 < hi) {
    int h2 = h1, u2 = u1;
    advance(h2, u2);
    after[0] = page_of(u2, 0);
    after[1] = page_of(u2, 1);
  }

  // the first units' bounds, on their way while the heads are quantised
#pragma unroll
  for (int j = 0; j < kScoreStages - 1; ++j) load_unit(lo + j);

  // Quantise the query heads, four of a warp at a time.
  for (int i0 = warp; i0 < heads; i0 += kAtOnce * kScoreWarps) {
    if (i0 != warp) load_queries(i0);
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      const int i = i0 + j * kScoreWarps;
      float m = 0.0f;
      bool nan = false;
#pragma unroll
      for (int k = 0; k < W; ++k) {
        const float2 f = E::unpack(q[j][k]);
        m = fmaxf(m, fmaxf(fabsf(f.x), fabsf(f.y)));
        nan |= f.x != f.x || f.y != f.y;
      }
      if (nan) m = INFINITY;
      // magnitudes order as their bit patterns
      m = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(m)));
      // a head that is not finite scores every page alike
      const float unit = m <= 3.402823466e38f ? __fdiv_rn(m, 127.0f) : 0.0f;
      if (i < heads) {
        const bool plain = unit >= 1.0e-30f;  // its reciprocal is an ordinary number
        const float r = plain ? __frcp_rn(unit) : 0.0f;
        const auto code = [&](float x) {  // as a float, rounded half to even
          const float t = plain ? quotient(x, unit, r) : unit > 0.0f ? __fdiv_rn(x, unit) : 0.0f;
          return __fadd_rn(__fadd_rn(fminf(fmaxf(t, -127.0f), 127.0f), 12582912.0f), -12582912.0f);
        };
        const auto byte = [](float c) { return __float_as_uint(c + 12582912.0f); };
#pragma unroll
        for (int k = 0; k < W; ++k) {
          const float2 f = E::unpack(q[j][k]);
          const float x = unit > 0.0f ? code(f.x) : 0.0f, y = unit > 0.0f ? code(f.y) : 0.0f;
          uint8_t* at = codes + i * kRow + 2 * (lane * W + k);
          *reinterpret_cast<uint16_t*>(at) =
              static_cast<uint16_t>(prmt(byte(fminf(x, 0.0f)), byte(fminf(y, 0.0f)), 0x0040));
          *reinterpret_cast<uint16_t*>(at + D) =
              static_cast<uint16_t>(prmt(byte(fmaxf(x, 0.0f)), byte(fmaxf(y, 0.0f)), 0x0040));
        }
        if (lane == 0) units[i] = unit;
      }
    }
  }
  __syncthreads();

  int head = -1, use = 0;
  uint4 code[kWide ? 2 : 1][kSpans];  // codes of query head g (and g + 8): the product's column
  float unit[kWide ? 4 : 2];       // of query heads 2 t, 2 t + 1 (and 8 after them): the results' columns
  uint32_t* out = p.keys + (static_cast<int64_t>(b) * p.kv_heads + head0) * p.key_stride + unit0 * 16;
  for (int i = lo; i < hi; ++i, advance(h, u)) {
    load_unit(i + kScoreStages - 1);
    if (h != head) {
      head = h;
#pragma unroll
      for (int w = 0; w < (kWide ? 2 : 1); ++w) {
        const int hq = g + 8 * w, cols = 2 * t + 8 * w;
#pragma unroll
        for (int k = 0; k < kSpans; ++k)
          code[w][k] = hq < p.group ? *reinterpret_cast<const uint4*>(codes + (h * p.group + hq) * kRow + 16 * t + 64 * k)
                                 : make_uint4(0, 0, 0, 0);
        unit[2 * w] = cols < p.group ? units[h * p.group + cols] : 0.0f;
        unit[2 * w + 1] = cols + 1 < p.group ? units[h * p.group + cols + 1] : 0.0f;
      }
    }
    asm volatile("cp.async.wait_group %0;" ::"n"(kScoreStages - 1) : "memory");
    const uint8_t* slot = ring + use * kSlotBytes<D>;
    use = use + 1 == kScoreStages ? 0 : use + 1;
    // sums start at the bits of 1.5 2^23, so that their own are a float's: below 2^22, they come out exact
    constexpr int kStart = 0x4B400000;
    int acc[kWide ? 2 : 1][4];
#pragma unroll
    for (int w = 0; w < (kWide ? 2 : 1); ++w) acc[w][0] = acc[w][1] = acc[w][2] = acc[w][3] = kStart;
#pragma unroll
    for (int k = 0; k < kSpans; ++k) {
      const uint4 x = *reinterpret_cast<const uint4*>(slot + 1024 * k), y = *reinterpret_cast<const uint4*>(slot + 1024 * k + 512);
#pragma unroll
      for (int w = 0; w < (kWide ? 2 : 1); ++w) {
        mma_s8(acc[w], x.x, y.x, x.y, y.y, code[w][k].x, code[w][k].y);
        mma_s8(acc[w], x.z, y.z, x.w, y.w, code[w][k].z, code[w][k].w);
      }
    }
    // the maxima over the heads of pages g and g + 8
    const float s0 = *reinterpret_cast<const float*>(slot + 1024 * kSpans - 12 * lane);
    const float s1 = *reinterpret_cast<const float*>(slot + 1024 * kSpans + 128 - 12 * lane);
    const auto score = [](int sum, float step, float unit) {
      return __fmul_rn(__fmul_rn(__int_as_float(sum) - 12582912.0f, step), unit);
    };
    float m0 = -INFINITY, m1 = -INFINITY;
#pragma unroll
    for (int c = 0; c < (kWide ? 4 : 2); ++c) {
      if (2 * t + (c & 1) + 8 * (c >> 1) < p.group) {
        m0 = fmaxf(m0, score(acc[c >> 1][c & 1], s0, unit[c]));
        m1 = fmaxf(m1, score(acc[c >> 1][2 + (c & 1)], s1, unit[c]));
      }
    }
    // the first exchange leaves page g to the lanes of even t, g + 8 to the others
    const bool odd = t & 1;
    float m = fmaxf(odd ? m1 : m0, __shfl_xor_sync(0xffffffffu, odd ? m0 : m1, 1));
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
    // a page whose keys are not all finite comes before every other
    if (t < 2 && page0 + 16 * u + 8 * t < n)
      out[h * p.key_stride + 16 * u + 8 * t + g] =
          (odd ? s1 : s0) <= 3.402823466e38f ? ordered(m) : ordered(INFINITY);
  }
}

// --------------------------------------------------------------- selection
struct SelectParams {
  const uint32_t* keys;
  int64_t key_stride;
  const int32_t* seq_lens;
  int32_t* lists;   // [B, Hkv, keep]
  int32_t* counts;  // [B, Hkv]
  int32_t max_pages;
  int32_t kv_heads;
  int32_t rows;
  int32_t keep, sink, recent;
};

// What one row needs, before its keys are looked at.
struct SelectRow {
  int n, keep;  // pages there are, and pages to list
  int32_t* out;
  const uint32_t* keys;
};
IRIS_DEV SelectRow select_row(const SelectParams& p, int row) {
  const int len = __ldg(p.seq_lens + row / p.kv_heads);
  const int64_t all = len > 0 ? (static_cast<int64_t>(len) + kPage - 1) / kPage : 0;
  SelectRow r;
  r.n = static_cast<int>(all < p.max_pages ? all : p.max_pages);
  r.keep = min(p.keep, r.n);
  r.out = p.lists + static_cast<int64_t>(row) * p.keep;
  r.keys = p.keys + static_cast<int64_t>(row) * p.key_stride;
  return r;
}
// The key by which page i is chosen: kept ends above every score, 0 (below every key) past the end.
IRIS_DEV uint32_t select_key(const SelectParams& p, const SelectRow& r, int i, uint32_t stored) {
  return i >= r.n ? 0u : i < p.sink || i >= r.n - p.recent ? 0xffffffffu : stored;
}
IRIS_DEV bool scored(uint32_t key) { return key != 0u && key != 0xffffffffu; }

// The highest `keep` keys are those above a threshold, the largest one that at
// least `keep` keys reach, and the first of those equal to it.  A warp with a
// short row finds it bit by bit by counting, from the highest bit in which the
// scored keys differ at all; a count that hits `keep` ends the search.
struct Search {
  uint32_t thr;
  int bit;  // the next one to decide; -1: none
};
IRIS_DEV Search search_from(uint32_t lowest, uint32_t highest) {
  const uint32_t differ = lowest ^ highest;
  const int top = differ != 0 ? 31 - __clz(differ) : -1;
  return {top < 0 ? highest : (highest >> top >> 1) << 1 << top, top};
}

// One warp per row of up to 32 KPT pages, all keys in registers, KPT
// consecutive ones a lane: a count is a sum over the warp, no barrier.
template <int KPT>
__global__ void __launch_bounds__(128) select_warp_kernel(const SelectParams p) {
  const int lane = threadIdx.x & 31, row = blockIdx.x * 4 + (threadIdx.x >> 5);
  if (row >= p.rows) return;
  const SelectRow r = select_row(p, row);
  if (lane == 0) p.counts[row] = r.keep;
  for (int i = r.keep + lane; i < p.keep; i += 32) r.out[i] = -1;
  if (r.n <= p.keep) {
    for (int i = lane; i < r.n; i += 32) r.out[i] = i;
    grid_dependency_wait();  // (nothing here runs ahead of the kernels before)
    return;
  }
  grid_dependency_wait();  // the scores are there
  uint32_t k[KPT], lowest = 0xffffffffu, highest = 0u;
#pragma unroll
  for (int j = 0; j < KPT; j += 4) {
    const int i = lane * KPT + j;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (i < r.n) v = __ldcg(reinterpret_cast<const uint4*>(r.keys + i));  // (the row's stride is a multiple of 8)
    k[j] = select_key(p, r, i, v.x);
    k[j + 1] = select_key(p, r, i + 1, v.y);
    k[j + 2] = select_key(p, r, i + 2, v.z);
    k[j + 3] = select_key(p, r, i + 3, v.w);
  }
#pragma unroll
  for (int j = 0; j < KPT; ++j) {
    if (scored(k[j])) lowest = min(lowest, k[j]), highest = max(highest, k[j]);
  }
  lowest = __reduce_min_sync(0xffffffffu, lowest);
  highest = __reduce_max_sync(0xffffffffu, highest);
  Search f = search_from(lowest, highest);
  for (; f.bit >= 0; --f.bit) {
    const uint32_t cand = f.thr | 1u << f.bit;
    int c[4] = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < KPT; ++j) c[j & 3] += k[j] >= cand;
    const int all = __reduce_add_sync(0xffffffffu, (c[0] + c[1]) + (c[2] + c[3]));
    if (all >= r.keep) f.thr = cand;
    if (all == r.keep) break;  // exactly the wanted ones reach it
  }
  int above = 0, equal = 0;
#pragma unroll
  for (int j = 0; j < KPT; ++j) {
    above += k[j] > f.thr;
    equal += k[j] == f.thr;
  }
  const int need = r.keep - __reduce_add_sync(0xffffffffu, above);
  int a = above, e = equal;  // inclusive sums over the lanes
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, a, o), y = __shfl_up_sync(0xffffffffu, e, o);
    if (lane >= o) a += x, e += y;
  }
  int eq = e - equal, at = a - above + min(eq, need);
#pragma unroll
  for (int j = 0; j < KPT; ++j) {
    bool take = k[j] > f.thr;
    if (k[j] == f.thr) take = eq++ < need;
    if (take) r.out[at++] = lane * KPT + j;
  }
}

// The bin in which the wanted number of keys is reached, the keys in the bins
// before it and in it.
struct Bin {
  int index, before, count;
};

// What the warps of a row tell one another: an array entry a warp, in the
// shared memory of each of the row's CTAs.  put() leaves a warp's value there,
// meet() waits for all warps' (every CTA of a cluster comes to it), and then
// any warp sums the entries, or those of the warps before it.
template <int kThreads, int kCtas>
struct Board {
  static constexpr int kPerCta = kThreads / 32, kEntries = kCtas * kPerCta;
  IRIS_DEV static int rank() {
    if constexpr (kCtas == 1) return 0;
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return static_cast<int>(r);
  }
  IRIS_DEV static int entry() { return rank() * kPerCta + (threadIdx.x >> 5); }
  IRIS_DEV static void put(uint32_t* board, uint32_t v) {
    const int lane = threadIdx.x & 31;
    if constexpr (kCtas == 1) {
      if (lane == 0) board[entry()] = v;
    } else if (lane < kCtas) {
      uint32_t to;
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(smem_u32(board + entry())), "r"(lane));
      asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(to), "r"(v) : "memory");
    }
  }
  IRIS_DEV static void meet() {
    if constexpr (kCtas == 1) __syncthreads();
    else asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
  }
  // sum of the first `n` entries, in every lane
  IRIS_DEV static int sum(const uint32_t* board, int n = kEntries) {
    uint32_t v = 0;
    for (int i = threadIdx.x & 31; i < n; i += 32) v += board[i];
    return static_cast<int>(__reduce_add_sync(0xffffffffu, v));
  }
  // the first of 256 bins, over all CTAs' counts, up to which there are at least `need` keys; for a whole warp
  IRIS_DEV static Bin find(const uint32_t* bins, int need) {
    const int lane = threadIdx.x & 31;
    uint32_t c[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < kCtas; ++i) {
#pragma unroll
      for (int j = 0; j < 8; j += 4) {
        const uint32_t* at = bins + 8 * lane + j;
        uint4 v;
        if constexpr (kCtas == 1) {
          v = *reinterpret_cast<const uint4*>(at);
        } else {
          uint32_t from;
          asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(from) : "r"(smem_u32(at)), "r"(i));
          asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                       : "r"(from)
                       : "memory");
        }
        c[j] += v.x;
        c[j + 1] += v.y;
        c[j + 2] += v.z;
        c[j + 3] += v.w;
      }
    }
    int sum = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) sum += static_cast<int>(c[j]);
    int upto = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    const int who = __ffs(__ballot_sync(0xffffffffu, upto >= need)) - 1;
    Bin b = {8 * lane, upto - sum, 0};
    bool found = false;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (!found) {
        b.count = static_cast<int>(c[j]);
        found = b.before + b.count >= need;
        if (!found) {
          b.before += b.count;
          ++b.index;
        }
      }
    }
    b.index = __shfl_sync(0xffffffffu, b.index, who);
    b.before = __shfl_sync(0xffffffffu, b.before, who);
    b.count = __shfl_sync(0xffffffffu, b.count, who);
    return b;
  }
  IRIS_DEV static uint32_t lowest(const uint32_t* board) {
    uint32_t v = 0xffffffffu;
    for (int i = threadIdx.x & 31; i < kEntries; i += 32) v = min(v, board[i]);
    return __reduce_min_sync(0xffffffffu, v);
  }
  IRIS_DEV static uint32_t highest(const uint32_t* board) {
    uint32_t v = 0;
    for (int i = threadIdx.x & 31; i < kEntries; i += 32) v = max(v, board[i]);
    return __reduce_max_sync(0xffffffffu, v);
  }
};

// kCtas CTAs (a cluster) per longer row: KPT consecutive keys a thread in
// registers, or for KPT = 0 read again for every count.  The threshold is
// found with histograms over the range that it still can lie in: two or three
// rounds of one barrier, where two bits at a time took about eight (8 rows of
// 8192 pages, with the scores: 13.7 -> 10.8 us).  A row of one long sequence
// goes over several SMs.
template <int kThreads, int KPT, int kCtas>
__global__ void __launch_bounds__(kThreads) select_kernel(const SelectParams p) {
  using B = Board<kThreads, kCtas>;
  __shared__ uint32_t s_more[4][B::kEntries];
  __shared__ __align__(16) uint32_t s_bins[kRangeRounds][256];
  __shared__ Bin s_found;
  constexpr int kAll = kThreads * kCtas;
  const int row = blockIdx.x / kCtas, tid = B::rank() * kThreads + threadIdx.x, lane = threadIdx.x & 31;
  const SelectRow r = select_row(p, row);
  if (tid == 0) p.counts[row] = r.keep;
  for (int i = r.keep + tid; i < p.keep; i += kAll) r.out[i] = -1;
  if (r.n <= p.keep) {
    for (int i = tid; i < r.n; i += kAll) r.out[i] = i;
    grid_dependency_wait();  // (nothing here runs ahead of the kernels before)
    return;                  // (nor does any CTA of the row go on)
  }
  for (int i = threadIdx.x; i < kRangeRounds * 64; i += kThreads) reinterpret_cast<uint4*>(s_bins)[i] = make_uint4(0, 0, 0, 0);
  grid_dependency_wait();  // the scores are there
  const auto key_at = [&](int i) { return select_key(p, r, i, i < r.n ? __ldcg(r.keys + i) : 0u); };
  constexpr int kRegs = KPT > 0 ? KPT : 1;
  uint32_t k[kRegs];
  if constexpr (KPT > 0) {
#pragma unroll
    for (int j = 0; j < KPT; j += 4) {
      const int i = tid * KPT + j;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (i < r.n) v = __ldcg(reinterpret_cast<const uint4*>(r.keys + i));
      k[j] = select_key(p, r, i, v.x);
      k[j + 1] = select_key(p, r, i + 1, v.y);
      k[j + 2] = select_key(p, r, i + 2, v.z);
      k[j + 3] = select_key(p, r, i + 3, v.w);
    }
  }
  const auto each = [&](auto&& f) {
    if constexpr (KPT > 0) {
#pragma unroll
      for (int j = 0; j < KPT; ++j) f(tid * KPT + j, k[j]);
    } else {
      const int per = (r.n + kAll - 1) / kAll;  // consecutive keys a thread
      for (int j = 0; j < per; ++j) f(tid * per + j, key_at(tid * per + j));
    }
  };
  uint32_t lowest = 0xffffffffu, highest = 0u;
  const auto widen = [&](uint32_t x) {
    if (scored(x)) lowest = min(lowest, x), highest = max(highest, x);
  };
  if constexpr (KPT > 0) {
    each([&](int, uint32_t x) { widen(x); });
  } else {
    for (int i = tid; i < r.n; i += kAll) widen(key_at(i));
  }
  lowest = __reduce_min_sync(0xffffffffu, lowest);
  highest = __reduce_max_sync(0xffffffffu, highest);
  if constexpr (kCtas > 1) B::meet();  // the other CTAs' memory is there to write to
  B::put(s_more[0], lowest);
  B::put(s_more[1], highest);
  B::meet();
  KeyRange range = {B::lowest(s_more[0]), B::highest(s_more[1])};
  // The scored keys that are wanted lie in the range, and the last of them is to be found: 256 bins over the range,
  // counted from the top, until one bin's keys are all wanted, or all the same.
  int need = r.keep - p.sink - p.recent;  // (n > keep: the two ends do not meet)
  uint32_t thr = range.high;              // keys above it are taken, and the first `need` equal ones
  for (int round = 0; need > 0 && round < kRangeRounds; ++round) {
    const int shift = max(24 - __clz(range.high - range.low), 0);
    uint32_t* bins = s_bins[round];
    const auto count = [&](uint32_t x) {
      if (range.holds(x)) atomicAdd(bins + range.bin(x, shift), 1u);
    };
    if constexpr (KPT > 0) {
      each([&](int, uint32_t x) { count(x); });
    } else {  // in any order
      for (int i = tid; i < r.n; i += kAll) count(key_at(i));
    }
    B::meet();
    Bin bin;
    if (kCtas == 1 || threadIdx.x < 32) bin = B::find(bins, need);
    if constexpr (kCtas > 1) {
      if (threadIdx.x == 0) s_found = bin;
      __syncthreads();
      bin = s_found;  // (next written behind another meeting)
    }
    need -= bin.before;
    range.narrow(static_cast<uint32_t>(bin.index), shift);
    if (bin.count == need) {  // exactly the wanted ones
      thr = range.low - 1u;
      need = 0;
    } else if (shift == 0) {
      thr = range.low;
      break;
    }
  }
  int above = 0, equal = 0;
  each([&](int, uint32_t x) {
    above += x > thr;
    equal += x == thr;
  });
  int a = above, e = equal;  // inclusive sums over the lanes, then over the warps before
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, a, o), y = __shfl_up_sync(0xffffffffu, e, o);
    if (lane >= o) a += x, e += y;
  }
  B::put(s_more[2], __shfl_sync(0xffffffffu, a, 31));
  B::put(s_more[3], __shfl_sync(0xffffffffu, e, 31));
  B::meet();  // the last one: nothing is written to another CTA's memory after it
  a += B::sum(s_more[2], B::entry());
  e += B::sum(s_more[3], B::entry());
  int eq = e - equal, at = a - above + min(eq, need);
  each([&](int i, uint32_t x) {
    bool take = x > thr;
    if (x == thr) take = eq++ < need;
    if (take) r.out[at++] = i;
  });
}

constexpr int kMaxShared = 227 * 1024;

// Shared memory of the score kernel.
int64_t score_bytes(int64_t q_heads, int head_dim) {
  return (q_heads * (2 * head_dim + 20) + 15) / 16 * 16 +
         kScoreWarps * kScoreStages * (head_dim == 128 ? kSlotBytes<128> : kSlotBytes<64>);
}

// All the shared memory that a CTA can have, asked for once per kernel and GPU.
cudaError_t allow_shared_memory(const void* fn) {
  static std::mutex mu;
  static std::set<std::pair<const void*, int>> done;
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  std::lock_guard<std::mutex> lock(mu);
  const auto key = std::make_pair(fn, device);
  if (done.count(key) != 0) return cudaSuccess;
  e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxShared);
  if (e == cudaSuccess) done.insert(key);
  return e;
}

template <typename E>
cudaError_t launch_score(const ScoreParams& p, int head_dim, dim3 grid, cudaStream_t s) {
  const bool wide = p.group > 8;
  const int bytes = static_cast<int>(score_bytes(p.cta_heads * p.group, head_dim));
  const auto fn = head_dim == 128 ? (wide ? score_kernel<E, 128, true> : score_kernel<E, 128, false>)
                                  : (wide ? score_kernel<E, 64, true> : score_kernel<E, 64, false>);
  const cudaError_t e = allow_shared_memory(reinterpret_cast<const void*>(fn));
  if (e != cudaSuccess) return e;
  return launch_early(fn, grid, dim3(32 * kScoreWarps), static_cast<size_t>(bytes), s, p);
}

cudaError_t launch_select(const SelectParams& p, cudaStream_t s) {
  const unsigned rows = static_cast<unsigned>(p.rows), fours = (rows + 3) / 4;
  if (p.max_pages <= 256) return launch_early(select_warp_kernel<8>, fours, 128, 0, s, p);
  if (p.max_pages <= 512) return launch_early(select_kernel<64, 8, 1>, rows, 64, 0, s, p);
  if (p.max_pages <= 1024) return launch_early(select_kernel<128, 8, 1>, rows, 128, 0, s, p);
  if (p.max_pages <= 2048) return launch_early(select_kernel<256, 8, 1>, rows, 256, 0, s, p);
  if (p.max_pages <= 8192) return launch_early_clusters(select_kernel<256, 8, 4>, 4 * rows, 256, 4, 0, s, p);
  if (p.max_pages <= 32768) return launch_early_clusters(select_kernel<512, 8, 8>, 8 * rows, 512, 8, 0, s, p);
  return launch_early(select_kernel<1024, 0, 1>, rows, 1024, 0, s, p);
}

int sm_count() {
  int device = 0, n = 0;
  if (cudaGetDevice(&device) != cudaSuccess ||
      cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess || n <= 0)
    return 148;
  return n;
}

int64_t key_stride_of(int32_t max_pages) { return (static_cast<int64_t>(max_pages) + 7) / 8 * 8; }

}  // namespace
}  // namespace iris

using namespace iris;

extern "C" int iris_b200_int4_page_bounds(const void* k_data, const void* k_scale, const int32_t* block_table,
                                          int64_t block_table_stride, const int32_t* seq_lens,
                                          const int32_t* first_token, void* bounds, float* bounds_step, void* values,
                                          int32_t batch, int32_t num_kv_heads, int32_t head_dim, int64_t num_pages,
                                          int32_t page_size, int32_t max_pages_per_seq, int32_t* error_word,
                                          void* stream) {
  if (batch < 0 || num_kv_heads <= 0 || num_pages < 0 || max_pages_per_seq < 0) return IRIS_EINVAL;
  if (page_size != kPage || (head_dim != 64 && head_dim != 128)) return IRIS_EUNSUPPORTED;
  if (batch == 0) return IRIS_OK;
  if (num_pages == 0) return IRIS_EINVAL;
  if (batch > 65535 || num_kv_heads > 65536) return IRIS_EUNSUPPORTED;
  const void* ptrs[] = {k_data, k_scale, block_table, seq_lens, bounds, bounds_step};
  for (const void* q : ptrs)
    if (q == nullptr) return IRIS_EINVAL;
  if (!aligned_to(k_data, 8) || !aligned_to(k_scale, 2) || !aligned_to(bounds, 16) || !aligned_to(bounds_step, 4) ||
      !aligned_to(values, 16))
    return IRIS_EALIGN;
  BoundsParams p = {};
  p.k_data = static_cast<const uint8_t*>(k_data);
  p.k_scale = static_cast<const __half*>(k_scale);
  p.block_table = block_table;
  p.table_stride = block_table_stride;
  p.seq_lens = seq_lens;
  p.first_token = first_token;
  p.bounds = static_cast<int8_t*>(bounds);
  p.step = bounds_step;
  p.values = static_cast<__half*>(values);
  p.num_pages = num_pages;
  p.max_pages = max_pages_per_seq;
  p.kv_heads = num_kv_heads;
  p.err = error_word;
  clear_stale_cuda_error();
  const int vecs = num_kv_heads * (head_dim / 8);
  const int threads = vecs >= 256 ? 256 : (vecs + 31) / 32 * 32;
  const int64_t want = (static_cast<int64_t>(sm_count()) * kBoundsCtas + batch - 1) / batch;
  int64_t x = want < max_pages_per_seq ? want : max_pages_per_seq;
  if (x < 1) x = 1;
  const dim3 grid(static_cast<unsigned>(x), static_cast<unsigned>(batch));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = launch_early(head_dim == 128 ? bounds_kernel<128> : bounds_kernel<64>, grid,
                                     dim3(static_cast<unsigned>(threads)), 0, s, p);
  if (e != cudaSuccess) {
    record_cuda_error(e, "bounds_kernel launch");
    return IRIS_ECUDA;
  }
  return IRIS_OK;
}

extern "C" size_t iris_b200_page_select_workspace_bytes(int32_t batch, int32_t num_kv_heads,
                                                        int32_t max_pages_per_seq) {
  if (batch <= 0 || num_kv_heads <= 0 || max_pages_per_seq <= 0) return 0;
  return static_cast<size_t>(batch) * num_kv_heads * key_stride_of(max_pages_per_seq) * sizeof(uint32_t);
}

extern "C" int iris_b200_page_select(const void* query, const void* bounds, const float* bounds_step,
                                     const int32_t* block_table, int64_t block_table_stride, const int32_t* seq_lens,
                                     int32_t* page_list, int32_t* page_count, int32_t batch, int32_t num_q_heads,
                                     int32_t num_kv_heads, int32_t head_dim, int64_t num_pages, int32_t page_size,
                                     int32_t max_pages_per_seq, int32_t max_pages, int32_t sink_pages,
                                     int32_t recent_pages, int32_t dtype, void* workspace, size_t workspace_bytes,
                                     int32_t* error_word, void* stream) {
  if (batch < 0 || num_q_heads <= 0 || num_kv_heads <= 0 || num_pages < 0 || max_pages_per_seq < 0) return IRIS_EINVAL;
  if (num_q_heads % num_kv_heads != 0) return IRIS_EINVAL;
  if (max_pages <= 0 || sink_pages < 0 || recent_pages < 0 ||
      static_cast<int64_t>(sink_pages) + recent_pages > max_pages)
    return IRIS_EINVAL;
  if (dtype != IRIS_DTYPE_FP16 && dtype != IRIS_DTYPE_BF16) return IRIS_EINVAL;
  const int group = num_q_heads / num_kv_heads;
  if (page_size != kPage || (head_dim != 64 && head_dim != 128) || group > 16) return IRIS_EUNSUPPORTED;
  if (score_bytes(num_q_heads, head_dim) > kMaxShared) return IRIS_EUNSUPPORTED;  // 589 query heads of 128 dims
  if (batch == 0) return IRIS_OK;
  if (num_pages == 0) return IRIS_EINVAL;
  if (batch > 65535 || num_kv_heads > 16384 || max_pages_per_seq > (1 << 27)) return IRIS_EUNSUPPORTED;
  const void* ptrs[] = {query, bounds, bounds_step, block_table, seq_lens, page_list, page_count};
  for (const void* q : ptrs)
    if (q == nullptr) return IRIS_EINVAL;
  if (!aligned_to(query, 4) || !aligned_to(bounds, 16) || !aligned_to(bounds_step, 4)) return IRIS_EALIGN;
  const size_t need = iris_b200_page_select_workspace_bytes(batch, num_kv_heads, max_pages_per_seq);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) return IRIS_EWORKSPACE;
  if (!aligned_to(workspace, 16)) return IRIS_EALIGN;
  clear_stale_cuda_error();
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  ScoreParams p = {};
  p.query = query;
  p.bounds = static_cast<const int8_t*>(bounds);
  p.step = bounds_step;
  p.block_table = block_table;
  p.table_stride = block_table_stride;
  p.seq_lens = seq_lens;
  p.keys = static_cast<uint32_t*>(workspace);
  p.key_stride = key_stride_of(max_pages_per_seq);
  p.num_pages = num_pages;
  p.max_pages = max_pages_per_seq;
  p.kv_heads = num_kv_heads;
  p.group = group;
  p.max_keep = max_pages;
  p.err = error_word;
  // the score kernel also reports bad lengths, so it runs even where every page is kept
  // Two CTAs an SM in all, as many a sequence as there are sequences for (three: 36.7 instead of 33.0 us at 64 sequences,
  // 15.9 instead of 14.0 at one, both with the selection: what a CTA does before its first unit then costs more than
  // its loads hide).  A CTA quantises the queries of its heads before it starts, so the heads are shared out first, as
  // long as three CTAs a share of the heads are left for the pages (one sequence of 8192 pages, 64 heads: 17.9 -> 16.1).
  int want = 2 * sm_count() / batch > 1 ? 2 * sm_count() / batch : 1;
  int shares = 1;
  while (num_kv_heads % (2 * shares) == 0 && want / (2 * shares) >= 3) shares *= 2;
  want /= shares;
  p.cta_heads = num_kv_heads / shares;
  const int sixteens = (max_pages_per_seq + 15) / 16;
  const dim3 grid(static_cast<unsigned>(want < sixteens ? want : sixteens > 0 ? sixteens : 1),
                  static_cast<unsigned>(batch), static_cast<unsigned>(shares));
  cudaError_t e = dtype == IRIS_DTYPE_FP16 ? launch_score<Fp16Elem>(p, head_dim, grid, s)
                                           : launch_score<Bf16Elem>(p, head_dim, grid, s);
  if (e == cudaSuccess) {
    SelectParams q = {};
    q.keys = p.keys;
    q.key_stride = p.key_stride;
    q.seq_lens = seq_lens;
    q.lists = page_list;
    q.counts = page_count;
    q.max_pages = max_pages_per_seq;
    q.kv_heads = num_kv_heads;
    q.rows = batch * num_kv_heads;
    q.keep = max_pages;
    q.sink = sink_pages;
    q.recent = recent_pages;
    e = launch_select(q, s);
  }
  if (e != cudaSuccess) {
    record_cuda_error(e, "page selection launch");
    return IRIS_ECUDA;
  }
  return IRIS_OK;
}
