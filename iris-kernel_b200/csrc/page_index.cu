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

#include "elem.cuh"

namespace iris {
namespace {

constexpr int kPage = 16;

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

IRIS_DEV uint32_t pack_s8(const int (&v)[4]) {
  return (v[0] & 0xff) | (v[1] & 0xff) << 8 | (v[2] & 0xff) << 16 | static_cast<uint32_t>(v[3]) << 24;
}

// One CTA per page (looping), one thread per 8-dim vector of one head; the
// D / 8 threads of a head are adjacent lanes.
template <int D>
__global__ void __launch_bounds__(256) bounds_kernel(const BoundsParams p) {
  constexpr int V = D / 8;
  const int b = blockIdx.y;
  const int len = __ldg(p.seq_lens + b);
  if (len <= 0) {
    if (len < 0 && blockIdx.x == 0 && threadIdx.x == 0) set_error(p.err, IRIS_ERR_SEQ_LEN);
    return;
  }
  int last = (len - 1) / kPage;
  if (last >= p.max_pages) {
    if (blockIdx.x == 0 && threadIdx.x == 0) set_error(p.err, IRIS_ERR_BLOCK_TABLE);
    last = p.max_pages - 1;
  }
  const int from = p.first_token != nullptr ? max(0, __ldg(p.first_token + b)) / kPage : 0;
  const int vecs = p.kv_heads * V;
  for (int col = from + blockIdx.x; col <= last; col += gridDim.x) {
    const int64_t page = __ldg(p.block_table + b * p.table_stride + col);
    if (page < 0 || page >= p.num_pages) {
      if (threadIdx.x == 0) set_error(p.err, IRIS_ERR_PAGE_ID);
      continue;
    }
    const int tokens = min(kPage, len - col * kPage);
    // whole warps go round together: lanes past the last vector repeat it and store nothing
    for (int i0 = threadIdx.x & ~31; i0 < vecs; i0 += blockDim.x) {
      const int i = min(i0 + static_cast<int>(threadIdx.x & 31), vecs - 1);
      const bool mine = i0 + static_cast<int>(threadIdx.x & 31) < vecs;
      const uint32_t* src = reinterpret_cast<const uint32_t*>(p.k_data) + page * kPage * vecs + i;
      const __half* scl = p.k_scale + page * kPage * (vecs >> 2) + (i >> 2);
      uint32_t w[kPage];
      float s[kPage];
#pragma unroll
      for (int t = 0; t < kPage; ++t) {
        w[t] = t < tokens ? __ldg(src + static_cast<int64_t>(t) * vecs) : 0u;
        s[t] = t < tokens ? __half2float(__ldg(scl + static_cast<int64_t>(t) * (vecs >> 2))) : 0.0f;
      }
      float lo[8], hi[8];
      bool bad = false;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        lo[j] = INFINITY;
        hi[j] = -INFINITY;
      }
#pragma unroll
      for (int t = 0; t < kPage; ++t) {
        if (t < tokens) {
          bad |= !(fabsf(s[t]) <= 65504.0f);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float x = static_cast<float>(nibble(w[t], j)) * s[t];  // exact
            lo[j] = fminf(lo[j], x);
            hi[j] = fmaxf(hi[j], x);
          }
        }
      }
      float m = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) m = fmaxf(m, fmaxf(fabsf(lo[j]), fabsf(hi[j])));
      if (bad) m = INFINITY;
#pragma unroll
      for (int o = 1; o < V; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      const bool finite = m <= 3.0e38f;
      const float step = finite ? __fdiv_rn(m, 127.0f) : INFINITY;
      int cl[8], ch[8];
      const float r = finite && step > 0.0f ? __frcp_rn(step) : 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        cl[j] = finite ? (step > 0.0f ? max(-127, __float2int_rd(quotient(lo[j], step, r))) : 0) : -127;
        ch[j] = finite ? (step > 0.0f ? min(127, __float2int_ru(quotient(hi[j], step, r))) : 0) : 127;
        cl[j] = min(127, cl[j]);
        ch[j] = max(-127, ch[j]);
      }
      if (mine) {
        const int h = i / V, v = i - h * V;
        const int64_t head = page * p.kv_heads + h;
        const int l0[4] = {cl[0], cl[1], cl[2], cl[3]}, l1[4] = {cl[4], cl[5], cl[6], cl[7]};
        const int h0[4] = {ch[0], ch[1], ch[2], ch[3]}, h1[4] = {ch[4], ch[5], ch[6], ch[7]};
        uint2* out = reinterpret_cast<uint2*>(p.bounds + head * 2 * D) + v;
        out[0] = make_uint2(pack_s8(l0), pack_s8(l1));
        out[V] = make_uint2(pack_s8(h0), pack_s8(h1));
        if (v == 0) p.step[head] = step;
        if (p.values != nullptr) {
          uint32_t a[4], c[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            a[j] = Fp16Elem::pack(cl[2 * j] * step, cl[2 * j + 1] * step);
            c[j] = Fp16Elem::pack(ch[2 * j] * step, ch[2 * j + 1] * step);
          }
          uint4* val = reinterpret_cast<uint4*>(p.values + head * 2 * D) + v;
          val[0] = make_uint4(a[0], a[1], a[2], a[3]);
          val[V] = make_uint4(c[0], c[1], c[2], c[3]);
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
  int32_t octets;  // 8-page groups per CTA
  int32_t max_keep;
  int32_t* err;
};

constexpr int kScoreWarps = 8;

// Four adjacent k-steps of m16n8k32 share one 16-byte load a lane: lane t of
// a quad holds bytes 16 t .. 16 t + 15 of a 64-byte span, words 0 and 1 of
// which are one product's two B registers and words 2 and 3 the next one's.
// The query's codes are read with the same assignment, so the sum runs over
// the span in another order than in memory, which whole numbers do not mind.
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

// kWide: more than 8 query heads a KV head (rows 8 .. 15 of the product).
template <typename E, int D, bool kWide>
__global__ void __launch_bounds__(32 * kScoreWarps) score_kernel(const ScoreParams p) {
  // codes of the query heads: [head][min(c, 0) : D][max(c, 0) : D], rows padded by 16 bytes
  extern __shared__ __align__(16) uint8_t smem[];
  constexpr int kRow = 2 * D + 16;
  constexpr int kSpans = 2 * D / 64;
  constexpr int kRows = kWide ? 16 : 8;
  const int b = blockIdx.y;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int len = __ldg(p.seq_lens + b);
  const bool first = blockIdx.x == 0 && threadIdx.x == 0;
  if (len < 0 && first) set_error(p.err, IRIS_ERR_SEQ_LEN);
  const int64_t all = len > 0 ? (static_cast<int64_t>(len) + kPage - 1) / kPage : 0;
  if (all > p.max_pages && first) set_error(p.err, IRIS_ERR_BLOCK_TABLE);
  const int n = static_cast<int>(all < p.max_pages ? all : p.max_pages);
  const int oct0 = blockIdx.x * p.octets;
  if (n <= p.max_keep || oct0 * 8 >= n) return;  // every page is kept, or none of these exist
  uint8_t* codes = smem;
  float* units = reinterpret_cast<float*>(smem + p.kv_heads * kRows * kRow);  // [Hkv][kRows]

  // quantise the query heads, one warp a head at a time
  for (int i = warp; i < p.kv_heads * kRows; i += kScoreWarps) {
    const int h = i / kRows, g = i - h * kRows;
    constexpr int W = D / 64;  // words a lane
    uint32_t q[W];
    float m = 0.0f;
    bool nan = false;
#pragma unroll
    for (int k = 0; k < W; ++k) {
      q[k] = g < p.group ? __ldg(static_cast<const uint32_t*>(p.query) +
                                 (static_cast<int64_t>(b) * p.kv_heads * p.group + h * p.group + g) * (D / 2) + lane * W + k)
                         : 0u;
      const float2 f = E::unpack(q[k]);
      m = fmaxf(m, fmaxf(fabsf(f.x), fabsf(f.y)));
      nan |= f.x != f.x || f.y != f.y;
    }
    if (nan) m = INFINITY;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    // a head that is not finite scores every page alike
    const float unit = m <= 3.402823466e38f ? __fdiv_rn(m, 127.0f) : 0.0f;
#pragma unroll
    for (int k = 0; k < W; ++k) {
      const float2 f = E::unpack(q[k]);
      const int x = unit > 0.0f ? max(-127, min(127, __float2int_rn(__fdiv_rn(f.x, unit)))) : 0;
      const int y = unit > 0.0f ? max(-127, min(127, __float2int_rn(__fdiv_rn(f.y, unit)))) : 0;
      uint8_t* at = codes + i * kRow + 2 * (lane * W + k);
      *reinterpret_cast<uint16_t*>(at) = static_cast<uint16_t>((min(x, 0) & 0xff) | (min(y, 0) & 0xff) << 8);
      *reinterpret_cast<uint16_t*>(at + D) = static_cast<uint16_t>(max(x, 0) | max(y, 0) << 8);
    }
    if (lane == 0) units[i] = unit;
  }
  __syncthreads();

  const int g = lane >> 2, t = lane & 3;
  const int octs = min(p.octets, (n + 7) / 8 - oct0);
  // units of work: (head, octet), a contiguous run of them for each warp
  const int total = p.kv_heads * octs;
  const int lo = total * warp / kScoreWarps, hi = total * (warp + 1) / kScoreWarps;
  int head = -1;
  uint32_t a[kSpans][kWide ? 8 : 4];
  float u0 = 0.0f, u1 = 0.0f;
  for (int i = lo; i < hi; ++i) {
    const int h = i / octs, oct = oct0 + i - h * octs;
    if (h != head) {
      head = h;
      const uint8_t* row = codes + (h * kRows + g) * kRow + 16 * t;
#pragma unroll
      for (int k = 0; k < kSpans; ++k) {
        const uint4 x = *reinterpret_cast<const uint4*>(row + 64 * k);
        a[k][0] = x.x, a[k][1] = x.y, a[k][2] = x.z, a[k][3] = x.w;
        if constexpr (kWide) {
          const uint4 y = *reinterpret_cast<const uint4*>(row + 8 * kRow + 64 * k);
          a[k][4] = y.x, a[k][5] = y.y, a[k][6] = y.z, a[k][7] = y.w;
        }
      }
      u0 = units[h * kRows + g];
      u1 = kWide ? units[h * kRows + g + 8] : 0.0f;
    }
    const int col = oct * 8 + g;
    int64_t page = col < n ? __ldg(p.block_table + b * p.table_stride + col) : 0;
    if (page < 0 || page >= p.num_pages) {
      set_error(p.err, IRIS_ERR_PAGE_ID);
      page = 0;
    }
    const uint4* src = reinterpret_cast<const uint4*>(p.bounds + (page * p.kv_heads + h) * 2 * D) + t;
    uint4 w[kSpans];
#pragma unroll
    for (int k = 0; k < kSpans; ++k) w[k] = __ldg(src + 4 * k);
    const float step = __ldg(p.step + page * p.kv_heads + h);
    int acc[4] = {0, 0, 0, 0};
#pragma unroll
    for (int k = 0; k < kSpans; ++k) {
      mma_s8(acc, a[k][0], kWide ? a[k][4] : 0u, a[k][1], kWide ? a[k][5] : 0u, w[k].x, w[k].y);
      mma_s8(acc, a[k][2], kWide ? a[k][6] : 0u, a[k][3], kWide ? a[k][7] : 0u, w[k].z, w[k].w);
    }
    // acc: head g (and g + 8), pages 2 t and 2 t + 1 of the octet
    const float s0 = __shfl_sync(0xffffffffu, step, 8 * t), s1 = __shfl_sync(0xffffffffu, step, 8 * t + 4);
    float m0 = -INFINITY, m1 = -INFINITY;
    if (g < p.group) {
      m0 = __fmul_rn(__fmul_rn(static_cast<float>(acc[0]), s0), u0);
      m1 = __fmul_rn(__fmul_rn(static_cast<float>(acc[1]), s1), u0);
    }
    if (kWide && g + 8 < p.group) {
      m0 = fmaxf(m0, __fmul_rn(__fmul_rn(static_cast<float>(acc[2]), s0), u1));
      m1 = fmaxf(m1, __fmul_rn(__fmul_rn(static_cast<float>(acc[3]), s1), u1));
    }
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) {
      m0 = fmaxf(m0, __shfl_xor_sync(0xffffffffu, m0, o));
      m1 = fmaxf(m1, __shfl_xor_sync(0xffffffffu, m1, o));
    }
    if (g == 0) {
      // a page whose keys are not all finite comes before every other
      const uint32_t k0 = s0 <= 3.402823466e38f ? ordered(m0) : ordered(INFINITY);
      const uint32_t k1 = s1 <= 3.402823466e38f ? ordered(m1) : ordered(INFINITY);
      uint32_t* out = p.keys + (static_cast<int64_t>(b) * p.kv_heads + h) * p.key_stride + oct * 8 + 2 * t;
      *reinterpret_cast<uint2*>(out) = make_uint2(k0, k1);
    }
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
  int32_t keep, sink, recent;
};

// Sum of v over the CTA, in every thread.  `slot` alternates between calls so
// that one barrier a call is enough.
template <int kThreads>
IRIS_DEV int block_sum(int v, int* part, int slot) {
  v = __reduce_add_sync(0xffffffffu, v);
  if ((threadIdx.x & 31) == 0) part[slot * 32 + (threadIdx.x >> 5)] = v;
  __syncthreads();
  const int lane = threadIdx.x & 31;
  return __reduce_add_sync(0xffffffffu, lane < kThreads / 32 ? part[slot * 32 + lane] : 0);
}

// One CTA per (sequence, KV head).  The highest `keep` keys: the largest
// threshold that at least `keep` keys reach, found bit by bit from the top
// (32 counts over the CTA, keys in registers for KPT > 0, read again each
// time otherwise), then one pass that writes the keys above it and the first
// of those equal to it.
template <int kThreads, int KPT>
__global__ void __launch_bounds__(kThreads) select_kernel(const SelectParams p) {
  __shared__ int s_part[64];
  __shared__ int s_scan[32];
  const int row = blockIdx.x, b = row / p.kv_heads;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int len = __ldg(p.seq_lens + b);
  const int64_t all = len > 0 ? (static_cast<int64_t>(len) + kPage - 1) / kPage : 0;
  const int n = static_cast<int>(all < p.max_pages ? all : p.max_pages);
  int32_t* out = p.lists + static_cast<int64_t>(row) * p.keep;
  const int keep = min(p.keep, n);
  if (tid == 0) p.counts[row] = keep;
  for (int i = keep + tid; i < p.keep; i += kThreads) out[i] = -1;
  if (n <= p.keep) {
    for (int i = tid; i < n; i += kThreads) out[i] = i;
    return;
  }
  const uint32_t* keys = p.keys + static_cast<int64_t>(row) * p.key_stride;
  const auto key_at = [&](int i) -> uint32_t {  // 0 past the end: below every key
    if (i >= n) return 0u;
    return i < p.sink || i >= n - p.recent ? 0xffffffffu : __ldg(keys + i);
  };
  constexpr int kRegs = KPT > 0 ? KPT : 1;
  uint32_t k[kRegs];
  if constexpr (KPT > 0) {
#pragma unroll
    for (int j = 0; j < KPT; ++j) k[j] = key_at(tid * KPT + j);
  }
  const auto count = [&](uint32_t at_least) {
    int c = 0;
    if constexpr (KPT > 0) {
#pragma unroll
      for (int j = 0; j < KPT; ++j) c += k[j] >= at_least;
    } else {
      for (int i = tid; i < n; i += kThreads) c += key_at(i) >= at_least;
    }
    return c;
  };
  uint32_t thr = 0;
  int slot = 0;
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t cand = thr | 1u << bit;
    const int c = block_sum<kThreads>(count(cand), s_part, slot);
    slot ^= 1;
    if (c >= keep) thr = cand;
    if (c == keep) break;  // exactly the wanted ones reach it
  }
  // keys above the threshold, and how many of those equal to it come along
  const auto each = [&](auto&& f) {
    if constexpr (KPT > 0) {
#pragma unroll
      for (int j = 0; j < KPT; ++j) f(tid * KPT + j, k[j]);
    } else {
      const int per = (n + kThreads - 1) / kThreads;  // consecutive keys a thread
      for (int j = 0; j < per; ++j) f(tid * per + j, key_at(tid * per + j));
    }
  };
  int above = 0, equal = 0;
  each([&](int, uint32_t x) {
    above += x > thr;
    equal += x == thr;
  });
  const int total_above = block_sum<kThreads>(above, s_part, slot);
  slot ^= 1;
  const int need = keep - total_above;
  // exclusive scans over the threads: of `above`, then of `equal`
  int pre[2];
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const int own = which == 0 ? above : equal;
    int x = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    __syncthreads();  // the previous round's readers are done
    if (lane == 31) s_scan[warp] = x;
    __syncthreads();
    const int w = lane < kThreads / 32 && lane < warp ? s_scan[lane] : 0;
    pre[which] = x - own + __reduce_add_sync(0xffffffffu, w);
  }
  int at = pre[0] + min(pre[1], need), eq = pre[1];
  each([&](int i, uint32_t x) {
    bool take = x > thr;
    if (x == thr) take = eq++ < need;
    if (take) out[at++] = i;
  });
}

template <typename E>
cudaError_t launch_score(const ScoreParams& p, int head_dim, dim3 grid, cudaStream_t s) {
  const bool wide = p.group > 8;
  const int rows = p.kv_heads * (wide ? 16 : 8);
  const int bytes = rows * (2 * head_dim + 16) + rows * 4;
  const auto fn = head_dim == 128 ? (wide ? score_kernel<E, 128, true> : score_kernel<E, 128, false>)
                                  : (wide ? score_kernel<E, 64, true> : score_kernel<E, 64, false>);
  if (bytes > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return e;
  }
  fn<<<grid, 32 * kScoreWarps, bytes, s>>>(p);
  return cudaGetLastError();
}

cudaError_t launch_select(const SelectParams& p, int64_t rows, cudaStream_t s) {
  const unsigned blocks = static_cast<unsigned>(rows);
  if (p.max_pages <= 2048)
    select_kernel<256, 8><<<blocks, 256, 0, s>>>(p);
  else if (p.max_pages <= 8192)
    select_kernel<1024, 8><<<blocks, 1024, 0, s>>>(p);
  else if (p.max_pages <= 32768)
    select_kernel<1024, 32><<<blocks, 1024, 0, s>>>(p);
  else
    select_kernel<1024, 0><<<blocks, 1024, 0, s>>>(p);
  return cudaGetLastError();
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
  if (!aligned_to(k_data, 4) || !aligned_to(k_scale, 2) || !aligned_to(bounds, 16) || !aligned_to(bounds_step, 4) ||
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
  const int64_t want = (static_cast<int64_t>(sm_count()) * 16 + batch - 1) / batch;
  int64_t x = want < max_pages_per_seq ? want : max_pages_per_seq;
  if (x < 1) x = 1;
  const dim3 grid(static_cast<unsigned>(x), static_cast<unsigned>(batch));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (head_dim == 128)
    bounds_kernel<128><<<grid, threads, 0, s>>>(p);
  else
    bounds_kernel<64><<<grid, threads, 0, s>>>(p);
  const cudaError_t e = cudaGetLastError();
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
  if (num_kv_heads * (group > 8 ? 16 : 8) * (2 * head_dim + 20) > 200 * 1024) return IRIS_EUNSUPPORTED;
  if (batch == 0) return IRIS_OK;
  if (num_pages == 0) return IRIS_EINVAL;
  if (batch > 65535 || max_pages_per_seq > (1 << 27)) return IRIS_EUNSUPPORTED;
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
  const int octets = static_cast<int>(key_stride_of(max_pages_per_seq) / 8);
  // the score kernel also reports bad lengths, so it runs even where every page is kept
  const int want = (2 * sm_count() + batch - 1) / batch;
  p.octets = octets > 0 ? (octets + want - 1) / want : 1;
  const dim3 grid(octets > 0 ? static_cast<unsigned>((octets + p.octets - 1) / p.octets) : 1u,
                  static_cast<unsigned>(batch));
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
    q.keep = max_pages;
    q.sink = sink_pages;
    q.recent = recent_pages;
    e = launch_select(q, static_cast<int64_t>(batch) * num_kv_heads, s);
  }
  if (e != cudaSuccess) {
    record_cuda_error(e, "page selection launch");
    return IRIS_ECUDA;
  }
  return IRIS_OK;
}
