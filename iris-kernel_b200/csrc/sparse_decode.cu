// Decode attention over selected pages of the INT4 paged cache, for sm_100a.
//
// Per sequence and KV head a list of logical pages; each of the head's G
// query heads attends to those pages' tokens that lie inside the sequence:
//   x_t = scale * q . k_t,   o = sum_t 2^(x'_t - m) v_t / sum_t 2^(x'_t - m),
//   lse = m + log2(sum),  x' = x log2(e),
// in one pass, with the running maximum m and sums rescaled when m rises.
// A list without tokens gives zeros and lse = -inf.
//
// Layout.  The head's share of a page is 16 rows of D/2 packed bytes and D/16
// scale bytes, for K and V: small strided pieces, so each warp copies its own
// pages with asynchronous copies into a ring of its own (no barrier between
// warps) and keeps its own running softmax.  The copies ask L2 for 64 bytes at
// a time: a token's other heads lie next to its own, and without that were
// fetched with it (the copies alone, 64 sequences x 128 pages, 8 KV heads of
// 128 dims: 49.2 -> 40.8 us).
//
// Products run on the tensor cores with fp16 operands and fp32 accumulation:
//   S^T = K Q^T    rows = tokens, columns = query heads, one accumulator per
//                  32-dim group, the group scale applied in fp32.  A nibble n
//                  enters as the subnormal fp16 (n + 8) 2^-24, one logic
//                  operation for two; -8 sum(q) 2^-24 is added to the
//                  group's sum.  Each query head is scaled by a power of two to a
//                  largest value in [2^15, 2^16) and put back in the logits' scale:
//                  odd dims enter times 1/16, so an element keeps all its bits
//                  down to 2^-25 of the head's largest, and a step of 2^-35
//                  of it below that.
//   O^T = V^T P^T  rows = dims, columns = query heads; V as exact integers; a
//                  weight p is two fp16 terms, p * scale again two: the rounded
//                  product and, by fused multiply-adds, what it left off (22
//                  bits).  FP16 ends at 2^-24, and so would a small weight of
//                  a small scale: weights are taken up to 2^14, which leaves
//                  a term a step of 2^-38 of the largest weight, 2^-24 of it
//                  times the smallest scale.  A row in which a scale of 2 or more
//                  is seen takes them up to 2^7, and each group's scales times a
//                  power of two of its own that brings the group's largest one
//                  so far to [2^7, 2^8), 2^7 at most; its sums are divided by
//                  it when the row is done.
//                  S^T's accumulators become the fragment of P^T by a transposing
//                  move of 8 x 8 matrices, which costs less than S = Q K^T, whose
//                  accumulators are that fragment, and whose products are twice
//                  as many with up to eight heads.
// A 16-byte chunk of a page's row is one group: ldmatrix hands each lane the
// eight dims of a token that its place in K's fragment needs, and its
// transposing form four dims of two tokens, as V's fragment needs them.
//
// Work.  A step takes two pages (their products and exponentials are
// independent; maxima, votes and rescalings are shared).  All steps of all rows
// (sequence x KV head), one after another, are cut into equal runs, one a warp,
// by the lists' real lengths: every warp finishes at the same time whatever the
// batch looks like, and waits for no other.  A row inside one run is written at
// once; the parts of the others go to the workspace as (o, m, l), and a second
// kernel joins them in the order of the list.
//
// Measured (B200): 64 sequences x 128 pages of 8192 tokens, 32 + 8 heads of 128
// dims: 57.4 us, 2.6 TB/s of the bytes it needs.  DRAM moves 226 MB, 1.5 times
// those (other heads' scales share a sector), which would take 35; the rest is
// 364 instructions a page and warp at half an instruction a cycle, with three
// CTAs of 164 registers an SM.  64 and 128 query heads: 61.4 and 78.2 us.  96 x 45
// pages, 16 heads of 64 dims: 51.8 us; DRAM moves 200 MB, 2.5 times what is
// needed, which would take 31, and a page has 283 instructions.  One sequence,
// 128 pages: 11.5 us, a chain of launches and dependent loads.
#include <map>
#include <mutex>
#include <type_traits>
#include <utility>

#include "elem.cuh"

namespace iris {
namespace {

constexpr int kPage = 16;
constexpr int kWarps = 4;
constexpr int kStages = 3;  // steps in flight and in use, per warp
constexpr int kSlots = 2 * kStages;

struct SparseParams {
  const void* query;
  const uint8_t* k_data;
  const uint8_t* v_data;
  const __half* k_scale;
  const __half* v_scale;
  const int32_t* block_table;
  int64_t table_stride;
  const int32_t* seq_lens;
  const int32_t* lists;   // [B, Hkv, keep]
  const int32_t* counts;  // [B, Hkv]
  void* output;           // [B, Hq, D]
  float* lse;             // [B, Hq] or NULL
  int64_t num_pages;
  int32_t max_pages;
  int32_t kv_heads, group;
  int32_t keep;
  int32_t rows;       // B * Hkv
  int32_t min_steps;  // shortest run of a warp
  int32_t warps;
  int32_t vector_counts;  // counts is 16-byte aligned
  float* part_o;      // [2 * warps][group][D]
  float* part_ml;     // [2 * warps][group][2]
  int32_t* row_start;  // [rows + 1]: number of the row's first step; last, the length of a run
  float scale_log2;
  int32_t* err;
};

IRIS_DEV void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global.L2::64B [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
template <int N>
IRIS_DEV void cp_async_small(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global.L2::64B [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(N) : "memory");
}
IRIS_DEV void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
IRIS_DEV void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// D = A B + C for m16n8k16.  (Not volatile: a function of its operands, and the
// compiler may interleave independent ones.)
IRIS_DEV void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const float (&c)[4]) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%10, %11, %12, %13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}

IRIS_DEV void mma_f16_zero(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%10, %10, %10, %10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}

// Four 8 x 8 matrices of 16-bit elements (rows of 16 bytes); lane L gives row
// L % 8 of matrix L / 8.  (With a memory clobber: the copies' waits order them.)
IRIS_DEV void load_matrices(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
IRIS_DEV void load_matrices_transposed(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

// An 8 x 8 matrix of 16-bit elements, two adjacent ones of row lane / 4 a lane, transposed.
IRIS_DEV uint32_t transposed(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// Signed nibbles n of w as (n + 8) in place: (w ^ 8) & 15.  Read as fp16, the
// nibbles in bits 0-3 are (n + 8) 2^-24 and those in bits 4-7 (n + 8) 2^-20.
constexpr int kLutOffset = 0x48;  // (a ^ c) & b
IRIS_DEV uint32_t offset_lo(uint32_t w) { return lop3<kLutOffset>(w, 0x000f000fu, 0x00080008u); }
IRIS_DEV uint32_t offset_hi(uint32_t w) { return lop3<kLutOffset>(w, 0x00f000f0u, 0x00800080u); }

// NaN in place of an infinite scale: the key is NaN (its nibbles are zeros), but
// the offset's share of a sum may leave a rounding that is not zero, and an
// infinite logit, if negative, would pass for a weight of zero.
IRIS_DEV __half2 finite_or_nan(__half2 s) { return __hfma2(s, __half2half2(__ushort_as_half(0)), s); }

// The largest logit of a row, rounded up, has weight 2^14; with scaled values 2^7.
constexpr float kWeightExponent = 14.0f, kScaledExponent = 7.0f;
// The largest value scales a pair of groups has been made ready for, their bits
// below the exponent set.  Below 2 there is nothing to do; beyond, the factors
// for exponent fields e are 2^(22 - e), 2^7 to 2^-8.
constexpr uint32_t kPlainCap = 0x3fff3fffu;
IRIS_DEV __half2 factors_of(uint32_t cap) { return u32_as_h2(0x94009400u - (cap & 0x7c007c00u)); }
// 127 + the exponent of one's factor
IRIS_DEV uint32_t factor_of(uint32_t cap, int half, bool scaled) {
  return scaled ? 149u - ((cap >> (10 + 16 * half)) & 31u) : 127u;
}

// Steps of a row.
IRIS_DEV int steps_of(const SparseParams& p, int row) {
  return (min(max(__ldg(p.counts + row), 0), p.keep) + 1) >> 1;
}

// Number of all steps, and the row (with the number of its first step) that
// holds step `at` if there is one.  The whole warp calls it.
struct Place {
  int total, row, start;
};
IRIS_DEV int warp_scan(int x) {  // inclusive
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, d);
    if (lane >= d) x += y;
  }
  return x;
}
// run_of(total) gives this warp's first step
template <typename F>
IRIS_DEV Place locate(const SparseParams& p, F&& run_of) {
  const int lane = threadIdx.x & 31;
  const int per = (p.rows + 127) / 128 * 4;  // consecutive rows a lane, in fours
  const auto clamped = [&](int c) { return (min(max(c, 0), p.keep) + 1) >> 1; };
  int sum = 0;
  for (int i = 0; i < per; i += 64) {  // up to sixteen loads in flight
    int4 c[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const int r = lane * per + i + 4 * j;
      c[j] = make_int4(0, 0, 0, 0);
      if (i + 4 * j < per && r < p.rows) {
        if (p.vector_counts && r + 3 < p.rows) {
          c[j] = __ldg(reinterpret_cast<const int4*>(p.counts + r));
        } else {
          c[j].x = __ldg(p.counts + r);
          if (r + 1 < p.rows) c[j].y = __ldg(p.counts + r + 1);
          if (r + 2 < p.rows) c[j].z = __ldg(p.counts + r + 2);
          if (r + 3 < p.rows) c[j].w = __ldg(p.counts + r + 3);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < 16; ++j) sum += clamped(c[j].x) + clamped(c[j].y) + clamped(c[j].z) + clamped(c[j].w);
  }
  const int upto = warp_scan(sum);
  Place out;
  out.total = __shfl_sync(0xffffffffu, upto, 31);
  out.row = -1;
  out.start = 0;
  const int at = run_of(out.total);
  if (at >= out.total) return out;
  const int who = __ffs(__ballot_sync(0xffffffffu, upto > at)) - 1;
  int base = __shfl_sync(0xffffffffu, upto - sum, who);
  for (int i = 0; i < per; i += 32) {  // the rows of that lane, 32 at a time
    const int r = who * per + i + lane;
    const int n = i + lane < per && r < p.rows ? steps_of(p, r) : 0;
    const int end = base + warp_scan(n);
    const unsigned past = __ballot_sync(0xffffffffu, end > at);
    if (past != 0) {
      const int l = __ffs(past) - 1;
      out.row = who * per + i + l;
      out.start = __shfl_sync(0xffffffffu, end - n, l);
      return out;
    }
    base = __shfl_sync(0xffffffffu, end, 31);
  }
  return out;  // not reached: the lane's rows hold the step
}
IRIS_DEV int run_length(const SparseParams& p, int total, int warps) {
  return max(p.min_steps, (total + warps - 1) / warps);
}

template <int D>
struct SparseCfg {
  static constexpr int kGroups = D / 32;
  static constexpr int kData = kPage * D / 2;        // bytes of a page's head, K or V
  static constexpr int kScale = kPage * kGroups * 2;  // bytes of its scales
  static constexpr int kStage = 2 * (kData + kScale);  // one page's slot
  static constexpr int kRing = kSlots * kStage;  // per warp
  static constexpr int kChunks = D / 32;          // 16-byte chunks per row
};

// Shared memory of a warp: its ring, its row's query fragments, its slots' info.
template <int D, int kHeads>
constexpr int kWarpBytes = SparseCfg<D>::kRing + (kHeads > 8 ? 2 : 1) * SparseCfg<D>::kGroups * 512 + 64;

// Byte offset of 16-byte chunk c of row r: rows 0, 2, 4, .. would start at the
// same banks, so the chunks of a row are turned by a function of the row.
template <int D>
IRIS_DEV int chunk_at(int r, int c) {
  if constexpr (D == 128) return r * 64 + ((c ^ ((r >> 1) & 3)) << 4);
  else return r * 32 + ((c ^ ((r >> 2) & 1)) << 4);
}

// A page's slot of the ring as the warp's lanes see it: its row, and how many
// tokens from its first one lie inside the sequence (0 or less: none, or no
// such page).
struct SlotInfo {
  int32_t row, left;
};

// kHeads: 4, 8 or 16, what the group fits in.  With up to four query heads
// the columns 4 to 7 are theirs again, and the second terms of the scaled
// weights take the place of a second product (64 x 128 pages: 3 us less).
// CTAs an SM, by registers: 16 heads of 128 dims 2 (78.2 us; 3 spill: 24 more), of
// 64 dims 3 (53.0; 2 or 4: 1.4 more); fewer heads of 128 dims 3 (4 spill), of 64
// dims 5 (96 x 45 pages 51.8; 4: 0.7 more, 6: 2.5 more).
template <typename E, int D, int kHeads>
__global__ void __launch_bounds__(32 * kWarps, D == 128 ? (kHeads > 8 ? 2 : 3) : (kHeads > 8 ? 3 : 5)) sparse_decode_kernel(SparseParams p) {
  using C = SparseCfg<D>;
  constexpr int G4 = C::kGroups;
  constexpr bool kWide = kHeads > 8, kTwice = kHeads == 4;
  constexpr int kH = kWide ? 2 : 1;  // eights of query heads; a lane has logits of heads 2 t and 2 t + 1 of each
  extern __shared__ __align__(128) uint8_t smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int me = blockIdx.x * kWarps + warp;
  grid_dependency_wait();
  grid_dependents_launch();  // the joining kernel may come up meanwhile
  const Place first = locate(p, [&](int total) {
    return min(static_cast<int64_t>(me) * run_length(p, total, p.warps), static_cast<int64_t>(total));
  });
  const int length = run_length(p, first.total, p.warps);
  if (me == 0 && lane == 0) p.row_start[p.rows] = length;
  if (first.row < 0) return;  // (nothing below waits for another warp)
  const int begin = me * length, end = min(begin + length, first.total);  // below 2^30 + the run

  uint8_t* ring = smem + warp * (kWarpBytes<D, kHeads>);
  uint4* s_query = reinterpret_cast<uint4*>(ring + C::kRing);  // [half][group][lane]
  SlotInfo* info = reinterpret_cast<SlotInfo*>(ring + C::kRing + kH * G4 * 512);
  const uint32_t ring_addr = smem_u32(ring);

  // ---- copies: pages of 16 steps are looked up at a time, a page a lane ----
  int64_t my_off = -1;  // bytes from k_data to the head's share of the page; -1: nothing there
  SlotInfo my_info = {0, 0};
  const uint32_t row_bytes = static_cast<uint32_t>(p.kv_heads) * (D / 2);
  int seek_row = first.row, seek_start = first.start;  // the row of the next step to look up, or an earlier one
  const auto look_up = [&](int step) {
    const int u = min(step + (lane >> 1), end - 1);
    int row = seek_row, start = seek_start, n = steps_of(p, row);
    while (u >= start + n && row + 1 < p.rows) {
      start += n;
      n = steps_of(p, ++row);
    }
    seek_row = __shfl_sync(0xffffffffu, row, 31);
    seek_start = __shfl_sync(0xffffffffu, start, 31);
    const int entry = 2 * (u - start) + (lane & 1);
    const int b = row / p.kv_heads;
    const int len = __ldg(p.seq_lens + b);
    my_off = -1;
    my_info = {row, 0};
    if (entry >= min(__ldg(p.counts + row), p.keep)) return;
    const int col = __ldg(p.lists + static_cast<int64_t>(row) * p.keep + entry);
    if (col < 0 || static_cast<int64_t>(col) * kPage >= len) return;
    if (col >= p.max_pages) {
      set_error(p.err, IRIS_ERR_BLOCK_TABLE);
      return;
    }
    const int32_t page = __ldg(p.block_table + b * p.table_stride + col);
    if (page < 0 || page >= p.num_pages) {
      set_error(p.err, IRIS_ERR_PAGE_ID);
      return;
    }
    my_off = static_cast<int64_t>(page) * (kPage * static_cast<int64_t>(row_bytes)) + (row - b * p.kv_heads) * (D / 2);
    my_info.left = len - col * kPage;
  };
  // this lane's chunks of any page: row lane / kChunks (and 8 below it for D = 128), and one row's scales
  const int r0 = lane / C::kChunks, c0 = lane % C::kChunks;
  const uint32_t data_off = r0 * row_bytes + 16 * c0;
  const uint8_t* k_src = p.k_data + data_off;
  const uint8_t* v_src = p.v_data + data_off;
  const uint8_t* s_src = reinterpret_cast<const uint8_t*>(lane < 16 ? p.k_scale : p.v_scale) +
                         static_cast<uint32_t>(lane & 15) * p.kv_heads * (2 * G4);
  const uint32_t dst0 = chunk_at<D>(r0, c0);
  const uint32_t s_dst = 2 * C::kData + (lane >> 4) * C::kScale + (lane & 15) * 2 * G4;
  const uint8_t* k_low = k_src + 8 * row_bytes;
  const uint8_t* v_low = v_src + 8 * row_bytes;
  // starts the copies of the next step's two pages, as far as there are any
  int ahead = 0, fill = 0;  // steps asked for, and the slot pair of the next one
  const auto fetch = [&]() {
    if (begin + ahead < end) {
      const int at = ahead & 15;
      if (at == 0) look_up(begin + ahead);
      if ((lane >> 1) == at) info[2 * fill + (lane & 1)] = my_info;
#pragma unroll
      for (int pg = 0; pg < 2; ++pg) {
        const int64_t off = __shfl_sync(0xffffffffu, my_off, 2 * at + pg);
        if (off >= 0) {
          const uint32_t st = ring_addr + (2 * fill + pg) * C::kStage;
          cp_async16(st + dst0, k_src + off);
          cp_async16(st + C::kData + dst0, v_src + off);
          if constexpr (D == 128) {
            cp_async16(st + dst0 + C::kData / 2, k_low + off);
            cp_async16(st + C::kData + dst0 + C::kData / 2, v_low + off);
          }
          cp_async_small<2 * G4>(st + s_dst, s_src + (off >> 3));
        }
      }
    }
    cp_async_commit();
    ++ahead;
    fill = fill + 1 == kStages ? 0 : fill + 1;
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) fetch();

  // ---- state of the row at hand ----
  constexpr int kTiles = D / 16;  // of 16 dims; a lane has two dims of each for heads 2 t, 2 t + 1 (+ 8)
  float o[kH][kTiles][4];
  float2 m[kH], minus_base[kH], l[kH], q_sum[kH][G4], head_scale[kH];  // (l: of this lane's tokens)
  uint32_t v_cap[G4 / 2];  // of two groups each
  bool scaled = false;     // (the same in every lane)
  int cur = -1, cur_start = first.start;

  // Query fragments.  Of this lane's eight dims of a group, the first product
  // takes 0, 4, 2, 6 (nibbles in bits 0-3 of a half word), the second 1, 5, 3, 7
  // (bits 4-7, 16 times as large) times 1/16.
  const auto start_row = [&](int row) {
    __syncwarp();  // the last row's fragments have been read
#pragma unroll
    for (int k = 0; k < G4 / 2; ++k) v_cap[k] = kPlainCap;
    scaled = false;
#pragma unroll
    for (int half = 0; half < kH; ++half) {
      m[half] = make_float2(-INFINITY, -INFINITY);
      minus_base[half] = l[half] = make_float2(0.0f, 0.0f);
#pragma unroll
      for (int j = 0; j < kTiles; ++j) o[half][j][0] = o[half][j][1] = o[half][j][2] = o[half][j][3] = 0.0f;
      const int hq = kTwice ? g & 3 : g + 8 * half;
      uint4 w[G4];
      float top = 0.0f;
#pragma unroll
      for (int k = 0; k < G4; ++k) {
        w[k] = hq < p.group ? __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.query) +
                                                                   (static_cast<int64_t>(row) * p.group + hq) * D +
                                                                   32 * k + 8 * t))
                            : make_uint4(0, 0, 0, 0);
        const uint32_t v[4] = {w[k].x, w[k].y, w[k].z, w[k].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 f = E::unpack(v[j]);
          top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
        }
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const uint32_t e = min(max(__float_as_uint(top) >> 23, 15u), 254u);
      const float down = __uint_as_float((269u - e) << 23);  // 2^(15 - (e - 127))
      const auto of_columns = [&](float x) {  // head g's -> heads 2 t and 2 t + 1's
        return make_float2(__shfl_sync(0xffffffffu, x, 8 * t), __shfl_sync(0xffffffffu, x, 8 * t + 4));
      };
      head_scale[half] = of_columns((p.scale_log2 * 512.0f) * __uint_as_float(e << 23));  // 2^24 / 2^15
#pragma unroll
      for (int k = 0; k < G4; ++k) {
        const uint32_t v[4] = {w[k].x, w[k].y, w[k].z, w[k].w};  // dims (0,1) (2,3) (4,5) (6,7)
        float f[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 x = E::unpack(v[j]);
          f[2 * j] = x.x * down;
          f[2 * j + 1] = x.y * (down * 0.0625f);
        }
        const uint32_t a[4] = {Fp16Elem::pack(f[0], f[4]), Fp16Elem::pack(f[2], f[6]), Fp16Elem::pack(f[1], f[5]),
                               Fp16Elem::pack(f[3], f[7])};
        s_query[(half * G4 + k) * 32 + lane] = make_uint4(a[0], a[1], a[2], a[3]);
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 x = Fp16Elem::unpack(a[j]);
          sum += (j < 2 ? 1.0f : 16.0f) * (x.x + x.y);
        }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        q_sum[half][k] = of_columns(sum * -4.76837158203125e-07f);  // -8 2^-24
      }
    }
    // (each lane reads back only what it wrote)
  };
  // the row's outputs, or this warp's part of them
  const auto finish_row = [&]() {
    const int after = cur_start + steps_of(p, cur);
    const bool starts = cur_start >= begin, whole = starts && after <= end;
    const int64_t part = 2 * static_cast<int64_t>(me) + (starts ? 1 : 0);  // the run's first row may have begun earlier
    if (starts && lane == 0) p.row_start[cur] = cur_start;
#pragma unroll
    for (int hh = 0; hh < kH; ++hh) {
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) {
        l[hh].x += __shfl_xor_sync(0xffffffffu, l[hh].x, d);
        l[hh].y += __shfl_xor_sync(0xffffffffu, l[hh].y, d);
      }
      const float lv[2] = {l[hh].x, l[hh].y}, minus[2] = {minus_base[hh].x, minus_base[hh].y};
      float inv[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int hq = 2 * t + e + 8 * hh;
        inv[e] = lv[e] == 0.0f ? 0.0f : __fdiv_rn(1.0f, lv[e]);
        if (g == 0 && hq < p.group) {
          if (!whole)
            *reinterpret_cast<float2*>(p.part_ml + (part * p.group + hq) * 2) =
                make_float2(lv[e] == 0.0f ? -INFINITY : -minus[e], lv[e]);
          else if (p.lse != nullptr)
            p.lse[static_cast<int64_t>(cur) * p.group + hq] = lv[e] == 0.0f ? -INFINITY : log2f(lv[e]) - minus[e];
        }
      }
      if constexpr (kTwice) {  // the two terms' sums
#pragma unroll
        for (int j = 0; j < kTiles; ++j) {
#pragma unroll
          for (int e = 0; e < 4; ++e) o[hh][j][e] += __shfl_xor_sync(0xffffffffu, o[hh][j][e], 2);
        }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int head = 2 * t + e + 8 * hh;
        const float f = inv[e];
        if (head < p.group) {
#pragma unroll
          for (int k = 0; k < G4; ++k) {  // this lane's four dims of the group are adjacent
            const float down = __uint_as_float((254u - factor_of(v_cap[k >> 1], k & 1, scaled)) << 23);  // 1 / the group's factor
            const float4 v = make_float4(o[hh][2 * k][e] * down, o[hh][2 * k][2 + e] * down, o[hh][2 * k + 1][e] * down,
                                         o[hh][2 * k + 1][2 + e] * down);
            const int d = 32 * k + 4 * g;
            if (whole)
              *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.output) +
                                        (static_cast<int64_t>(cur) * p.group + head) * D + d) =
                  make_uint2(E::pack(v.x * f, v.y * f), E::pack(v.z * f, v.w * f));
            else
              *reinterpret_cast<float4*>(p.part_o + (part * p.group + head) * D + d) = v;
          }
        }
      }
    }
  };

  // this lane's row of the four 8 x 16-byte matrices (tokens 0-7 and 8-15) x (groups 0 and 1)
  const uint32_t mat = chunk_at<D>((lane & 7) + (lane & 8), (lane >> 4) & 1);
  // words of the scales of this lane's token pairs (2 t, 2 t + 1) and (2 t + 8, 2 t + 9), adjacent in
  // memory: token 2 t's groups two a word, then the next token's
  const auto scale_words = [&](const uint8_t* at, uint32_t (&w)[2][G4]) {
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      if constexpr (G4 == 4) {
        const uint4 v = *reinterpret_cast<const uint4*>(at + (2 * t + 8 * n) * 8);
        w[n][0] = v.x, w[n][1] = v.y, w[n][2] = v.z, w[n][3] = v.w;
      } else {
        const uint2 v = *reinterpret_cast<const uint2*>(at + (2 * t + 8 * n) * 4);
        w[n][0] = v.x, w[n][1] = v.y;
      }
    }
  };
  const uint32_t second_term = g < 4 ? 0u : 0xffffffffu;  // kTwice
  int slot = -2;
  for (int step = begin; step < end; ++step) {
    __syncwarp();  // every lane is done with the slots that are filled next
    fetch();
    cp_async_wait<kStages - 1>();
    __syncwarp();
    slot = slot + 2 == kSlots ? 0 : slot + 2;
    const SlotInfo i0 = info[slot], i1 = info[slot + 1];
    if (i0.row != cur) {
      if (cur >= 0) {
        finish_row();
        cur_start = step;  // (rows without steps lie between, if any)
      }
      cur = i0.row;
      start_row(cur);
    }
    const int left[2] = {i0.left, i1.left};
    if (max(left[0], left[1]) <= 0) continue;
    const uint8_t* st = ring + slot * C::kStage;
    const uint32_t st_addr = ring_addr + slot * C::kStage;

    // S^T = K Q^T, one accumulator per group, scaled in fp32 (2^-24 and the query's power of two left out)
    float2 x[kH][2][2];  // [eight][page][token g | g + 8]: heads 2 t and 2 t + 1
    {
      uint32_t ks[2][2][G4 / 2];  // [page][token][groups, two a word]
#pragma unroll
      for (int pg = 0; pg < 2; ++pg) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const uint8_t* at = st + pg * C::kStage + 2 * C::kData + (g + 8 * r) * (2 * G4);
          if constexpr (G4 == 4) {
            const uint2 v = *reinterpret_cast<const uint2*>(at);
            ks[pg][r][0] = v.x, ks[pg][r][1] = v.y;
          } else {
            ks[pg][r][0] = *reinterpret_cast<const uint32_t*>(at);
          }
        }
      }
#pragma unroll
      for (int k0 = 0; k0 < G4; k0 += 2) {
        uint32_t kw[2][4];  // [page][group k0, tokens 0-7 | 8-15, group k0 + 1, ..]
        float2 sc[2][2];    // [page][token]: of groups k0 and k0 + 1
#pragma unroll
        for (int pg = 0; pg < 2; ++pg) {
          load_matrices(kw[pg], st_addr + pg * C::kStage + (mat ^ (16 * k0)));
#pragma unroll
          for (int r = 0; r < 2; ++r) sc[pg][r] = __half22float2(finite_or_nan(u32_as_h2(ks[pg][r][k0 / 2])));
        }
#pragma unroll
        for (int k = k0; k < k0 + 2; ++k) {
          uint4 q[kH];
#pragma unroll
          for (int hh = 0; hh < kH; ++hh) q[hh] = s_query[(hh * G4 + k) * 32 + lane];
#pragma unroll
          for (int pg = 0; pg < 2; ++pg) {
            const uint32_t w0 = kw[pg][2 * (k - k0)], w1 = kw[pg][2 * (k - k0) + 1], v0 = w0 >> 8, v1 = w1 >> 8;
            const uint32_t a0[4] = {offset_lo(w0), offset_lo(w1), offset_lo(v0), offset_lo(v1)};
            const uint32_t a1[4] = {offset_hi(w0), offset_hi(w1), offset_hi(v0), offset_hi(v1)};
#pragma unroll
            for (int hh = 0; hh < kH; ++hh) {
              float acc[4];
              mma_f16_zero(acc, a0, q[hh].x, q[hh].y);
              mma_f16(acc, a1, q[hh].z, q[hh].w, acc);
#pragma unroll
              for (int r = 0; r < 2; ++r) {
                const float scale = k == k0 ? sc[pg][r].x : sc[pg][r].y;
                const float2 a = __fadd2_rn(make_float2(acc[2 * r], acc[2 * r + 1]), q_sum[hh][k]);
                const float2 scale2 = make_float2(scale, scale);
                x[hh][pg][r] = k == 0 ? __fmul2_rn(a, scale2) : __ffma2_rn(a, scale2, x[hh][pg][r]);
              }
            }
          }
        }
      }
    }
    uint32_t vs[2][2][G4];
#pragma unroll
    for (int pg = 0; pg < 2; ++pg) scale_words(st + pg * C::kStage + 2 * C::kData + C::kScale, vs[pg]);
    // and, to see the largest of them, a lane two groups of one token of a page (of each, or of its half of the lanes)
    constexpr int kLook = D == 128 ? 2 : 1;
    uint32_t look[kLook];
#pragma unroll
    for (int i = 0; i < kLook; ++i)
      look[i] = *reinterpret_cast<const uint32_t*>(st + (D == 128 ? i : lane >> 4) * C::kStage + 2 * C::kData + C::kScale +
                                                   4 * (D == 128 ? lane : lane & 15));

    // The logits, rounded to fp32 before a maximum is taken from them: a fused multiply-add would leave the largest
    // token that maximum's own rounding, which passes an exponential's range for logits from 2^30 on.
#pragma unroll
    for (int hh = 0; hh < kH; ++hh) {
#pragma unroll
      for (int pg = 0; pg < 2; ++pg) {
#pragma unroll
        for (int n = 0; n < 2; ++n) x[hh][pg][n] = __fmul2_rn(x[hh][pg][n], head_scale[hh]);
      }
    }

    // tokens past the sequence's end count for nothing, whatever their bytes hold
    if (min(left[0], left[1]) < kPage) {
#pragma unroll
      for (int i = 0; i < kLook; ++i) {
        if ((D == 128 ? lane >> 1 : lane & 15) >= (D == 128 ? left[i] : lane < 16 ? left[0] : left[1])) look[i] = 0u;
      }
#pragma unroll
      for (int pg = 0; pg < 2; ++pg) {
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const bool out0 = 2 * t + 8 * n >= left[pg], out1 = 2 * t + 8 * n + 1 >= left[pg];
#pragma unroll
          for (int hh = 0; hh < kH; ++hh) {
            if (g + 8 * n >= left[pg]) x[hh][pg][n] = make_float2(-INFINITY, -INFINITY);
          }
#pragma unroll
          for (int k = 0; k < G4 / 2; ++k) {
            if (out0) vs[pg][n][k] = 0u;
            if (out1) vs[pg][n][k + G4 / 2] = 0u;
          }
        }
      }
    }

    // running softmax; the maxima (and those of the value scales) are looked at across the tokens only when one rises
    __half2 seen = __habs2(u32_as_h2(look[0]));
    if constexpr (D == 128) seen = __hmax2(seen, __habs2(u32_as_h2(look[kLook - 1])));
    const uint32_t my_cap = D == 128 && (lane & 1) ? v_cap[G4 / 2 - 1] : v_cap[0];
    const bool grows = !__hble2(seen, u32_as_h2(my_cap));
    bool rises = grows;
    float2 top[kH];
#pragma unroll
    for (int hh = 0; hh < kH; ++hh) {
      top[hh].x = fmaxf(fmaxf(x[hh][0][0].x, x[hh][0][1].x), fmaxf(x[hh][1][0].x, x[hh][1][1].x));
      top[hh].y = fmaxf(fmaxf(x[hh][0][0].y, x[hh][0][1].y), fmaxf(x[hh][1][0].y, x[hh][1][1].y));
      rises |= top[hh].x > m[hh].x || top[hh].y > m[hh].y;
    }
    if (__any_sync(0xffffffffu, rises)) {
      if (__any_sync(0xffffffffu, grows)) {
        uint32_t cap = h2_as_u32(seen);
        // (a group with a scale that is not finite gives NaN, whatever its factor)
        if ((cap & 0x7c00u) == 0x7c00u) cap &= 0xffff0000u;
        if ((cap & 0x7c000000u) == 0x7c000000u) cap &= 0x0000ffffu;
        cap = __vmaxu2(cap, my_cap);
#pragma unroll
        for (int d = D == 128 ? 2 : 1; d < 32; d <<= 1) cap = __vmaxu2(cap, __shfl_xor_sync(0xffffffffu, cap, d));
        cap |= 0x03ff03ffu;
        uint32_t next[G4 / 2];
        bool now = false;
#pragma unroll
        for (int i = 0; i < G4 / 2; ++i) {
          next[i] = __shfl_sync(0xffffffffu, cap, i);
          now |= next[i] != kPlainCap;
        }
#pragma unroll
        for (int k = 0; k < G4; ++k) {  // the groups' sums, by their new factors over their present ones
          const float smaller = __uint_as_float(
              (127u + factor_of(next[k >> 1], k & 1, now) - factor_of(v_cap[k >> 1], k & 1, scaled)) << 23);
#pragma unroll
          for (int hh = 0; hh < kH; ++hh) {
#pragma unroll
            for (int e = 0; e < 8; ++e) o[hh][2 * k + (e >> 2)][e & 3] *= smaller;
          }
          if (k & 1) v_cap[k >> 1] = next[k >> 1];
        }
        scaled = now;
      }
      const float exponent = scaled ? kScaledExponent : kWeightExponent;
#pragma unroll
      for (int hh = 0; hh < kH; ++hh) {
        float2 to = top[hh];
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) {
          to.x = fmaxf(to.x, __shfl_xor_sync(0xffffffffu, to.x, d));
          to.y = fmaxf(to.y, __shfl_xor_sync(0xffffffffu, to.y, d));
        }
        // rounded up to a whole number, so that the exponents' base is exact (or, from 2^24 on, no further down than m)
        to = make_float2(fmaxf(ceilf(to.x), m[hh].x), fmaxf(ceilf(to.y), m[hh].y));
        const float2 base = make_float2(to.x == -INFINITY ? 0.0f : __fadd_rd(exponent, -to.x),
                                        to.y == -INFINITY ? 0.0f : __fadd_rd(exponent, -to.y));
        const float2 f = make_float2(m[hh].x == -INFINITY ? 0.0f : ex2(base.x - minus_base[hh].x),
                                     m[hh].y == -INFINITY ? 0.0f : ex2(base.y - minus_base[hh].y));
        m[hh] = to;
        minus_base[hh] = base;
        l[hh] = __fmul2_rn(l[hh], f);
#pragma unroll
        for (int j = 0; j < kTiles; ++j) {
#pragma unroll
          for (int e = 0; e < 4; e += 2) {
            const float2 v = __fmul2_rn(make_float2(o[hh][j][e], o[hh][j][e + 1]), f);
            o[hh][j][e] = v.x;
            o[hh][j][e + 1] = v.y;
          }
        }
      }
    }
#pragma unroll
    for (int hh = 0; hh < kH; ++hh) {
#pragma unroll
      for (int pg = 0; pg < 2; ++pg) {
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const float2 y = __fadd2_rn(x[hh][pg][n], minus_base[hh]);
          x[hh][pg][n] = make_float2(ex2(y.x), ex2(y.y));
          l[hh] = __fadd2_rn(l[hh], x[hh][pg][n]);
        }
      }
    }

    if (scaled) {
#pragma unroll
      for (int pg = 0; pg < 2; ++pg) {
#pragma unroll
        for (int n = 0; n < 2; ++n) {
#pragma unroll
          for (int k = 0; k < G4; ++k)
            vs[pg][n][k] = h2_as_u32(__hmul2(u32_as_h2(vs[pg][n][k]), factors_of(v_cap[k % (G4 / 2)])));
        }
      }
    }

    // O^T += V^T P^T
#pragma unroll
    for (int pg = 0; pg < 2; ++pg) {
      // Weights, rounded and the rest, turned round to head g and the token pairs (2 t, 2 t + 1), (2 t + 8, 2 t + 9);
      // kTwice: neither -ph nor the rest where the first term is wanted.
      __half2 ph[kH][2], pl[kH][2], minus[kH][2];
#pragma unroll
      for (int hh = 0; hh < kH; ++hh) {
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const __half2 h = __floats2half2_rn(x[hh][pg][n].x, x[hh][pg][n].y);
          const float2 r = __half22float2(h);
          const uint32_t hi_bits = transposed(h2_as_u32(h));
          const uint32_t lo_bits = transposed(h2_as_u32(__floats2half2_rn(x[hh][pg][n].x - r.x, x[hh][pg][n].y - r.y)));
          ph[hh][n] = u32_as_h2(hi_bits);
          pl[hh][n] = u32_as_h2(kTwice ? lo_bits & second_term : lo_bits);
          minus[hh][n] = u32_as_h2((hi_bits ^ 0x80008000u) & second_term);
        }
      }
#pragma unroll
      for (int k0 = 0; k0 < G4; k0 += 2) {
        uint32_t vw[4];  // group k0: tokens (2 t, 2 t + 1), (2 t + 8, 2 t + 9), group k0 + 1: ..
        load_matrices_transposed(vw, st_addr + pg * C::kStage + C::kData + (mat ^ (16 * k0)));
#pragma unroll
        for (int k = k0; k < k0 + 2; ++k) {
          uint32_t hi[kH][2], lo[kH][2];  // P^T: head g (and g + 8), token pairs
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            // the group's scales of the pair
            const __half2 sc = u32_as_h2(prmt(vs[pg][n][k / 2], vs[pg][n][(G4 + k) / 2], k % 2 == 0 ? 0x5410 : 0x7632));
#pragma unroll
            for (int hh = 0; hh < kH; ++hh) {
              const __half2 a = __hmul2_rn(kTwice ? minus[hh][n] : ph[hh][n], sc);
              const __half2 c = __hfma2(pl[hh][n], sc, __hfma2(ph[hh][n], sc, kTwice ? a : __hneg2(a)));
              hi[hh][n] = h2_as_u32(kTwice ? c : a);
              lo[hh][n] = h2_as_u32(c);
            }
          }
          const uint32_t v0 = vw[2 * (k - k0)], v1 = vw[2 * (k - k0) + 1];
#pragma unroll
          for (int jj = 0; jj < 2; ++jj) {  // rows g and g + 8 of the tile: dims 4 g + 2 jj and 4 g + 2 jj + 1
            const uint32_t a[4] = {int4_lo_exact(v0 >> (8 * jj)), int4_hi_exact(v0 >> (8 * jj)),
                                   int4_lo_exact(v1 >> (8 * jj)), int4_hi_exact(v1 >> (8 * jj))};
#pragma unroll
            for (int hh = 0; hh < kH; ++hh) {
              float(&acc)[4] = o[hh][2 * k + jj];
              mma_f16(acc, a, hi[hh][0], hi[hh][1], acc);
              if constexpr (!kTwice) mma_f16(acc, a, lo[hh][0], lo[hh][1], acc);
            }
          }
        }
      }
    }
  }

  finish_row();
}

// Joins the parts of the rows that no single warp had, one warp per query head;
// rows without a step are written here too.
template <typename E, int D>
__global__ void __launch_bounds__(128) sparse_join_kernel(SparseParams p) {
  constexpr int kPer = D / 32;   // dims a lane
  constexpr int kAhead = 8;      // parts loaded at a time
  using Vec = std::conditional_t<kPer == 4, float4, float2>;
  const int lane = threadIdx.x & 31;
  const int row = blockIdx.x, head = blockIdx.y * 4 + (threadIdx.x >> 5);
  const int n = steps_of(p, row);
  // The row's first step and the length of a run: with few rows from the counts, while the runs finish; otherwise
  // from what they wrote down.
  const bool few = p.rows <= 256;
  int start = 0, length = 1;
  if (few) {
    int before = 0, all = 0;
    for (int r = lane; r < p.rows; r += 32) {
      const int x = steps_of(p, r);
      all += x;
      before += r < row ? x : 0;
    }
    start = __reduce_add_sync(0xffffffffu, before);
    length = run_length(p, __reduce_add_sync(0xffffffffu, all), p.warps);
  }
  if (head == 0 && lane == 0 && __ldg(p.seq_lens + row / p.kv_heads) < 0) set_error(p.err, IRIS_ERR_SEQ_NEGATIVE);
  grid_dependency_wait();
  if (head >= p.group) return;
  const int64_t out = static_cast<int64_t>(row) * p.group + head;
  float acc[kPer];
#pragma unroll
  for (int j = 0; j < kPer; ++j) acc[j] = 0.0f;
  float top = -INFINITY, sum = 0.0f;
  if (n > 0) {
    if (!few) {
      start = __ldcg(p.row_start + row);
      length = __ldcg(p.row_start + p.rows);
    }
    const int first = start / length, parts = (start + n - 1) / length - first + 1;
    if (parts == 1) return;  // its warp wrote the outputs
    const auto part_at = [&](int i) {
      return (2 * static_cast<int64_t>(first + i) + (i == 0 ? 1 : 0)) * p.group + head;
    };
    for (int i0 = 0; i0 < parts; i0 += 32) {
      float2 ml = make_float2(-INFINITY, 0.0f);
      if (i0 + lane < parts) ml = __ldcg(reinterpret_cast<const float2*>(p.part_ml) + part_at(i0 + lane));
      const int here = min(32, parts - i0);
      float w = 0.0f;
      for (int i = 0; i < here; i += kAhead) {
        Vec v[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
          if (i + j < here)
            v[j] = __ldcg(reinterpret_cast<const Vec*>(p.part_o + part_at(i0 + i + j) * D) + lane);
        if (i == 0) {  // the weights of these up to 32 parts, while the first parts are on their way
          float m = ml.x;
#pragma unroll
          for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
          m = fmaxf(m, top);
          const float base = m == -INFINITY ? 0.0f : m, old = ex2(top - base);
          top = m;
          w = ex2(ml.x - base);
          sum = fmaf(sum, old, w * ml.y);
#pragma unroll
          for (int j = 0; j < kPer; ++j) acc[j] *= old;
        }
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
          const float f = __shfl_sync(0xffffffffu, w, i + j);
          if (i + j < here) {
            const float* x = reinterpret_cast<const float*>(&v[j]);
#pragma unroll
            for (int e = 0; e < kPer; ++e) acc[e] = fmaf(f, x[e], acc[e]);
          }
        }
      }
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  }
  const float inv = sum == 0.0f ? 0.0f : __fdiv_rn(1.0f, sum);
  uint32_t* dst = static_cast<uint32_t*>(p.output) + out * (D / 2) + lane * (kPer / 2);
#pragma unroll
  for (int j = 0; j < kPer / 2; ++j) dst[j] = E::pack(acc[2 * j] * inv, acc[2 * j + 1] * inv);
  if (lane == 0 && p.lse != nullptr) p.lse[out] = sum == 0.0f ? -INFINITY : top + log2f(sum);
}

// Warps that one launch of the kernel keeps on the current GPU (asked once per kernel and GPU).
cudaError_t resident_warps(const void* fn, int bytes, int* out) {
  static std::mutex mu;
  static std::map<std::pair<const void*, int>, int> known;
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  std::lock_guard<std::mutex> lock(mu);
  const auto key = std::make_pair(fn, device);
  auto it = known.find(key);
  if (it == known.end()) {
    int sms = 0, per_sm = 0;
    e = cudaFuncSetAttribute(fn, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
    if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, fn, 32 * kWarps, bytes);
    if (e != cudaSuccess) return e;
    it = known.emplace(key, sms * (per_sm > 0 ? per_sm : 1) * kWarps).first;
  }
  *out = it->second;
  return cudaSuccess;
}

using KernelFn = void (*)(SparseParams);
struct Kernel {
  KernelFn fn;
  KernelFn join;
  int bytes;  // of shared memory
};
template <typename E, int D, int kHeads>
Kernel kernel() {
  return {sparse_decode_kernel<E, D, kHeads>, sparse_join_kernel<E, D>, kWarps * kWarpBytes<D, kHeads>};
}
template <typename E>
Kernel kernel_of(int head_dim, int group) {
  if (head_dim == 128) return group > 8 ? kernel<E, 128, 16>() : group > 4 ? kernel<E, 128, 8>() : kernel<E, 128, 4>();
  return group > 8 ? kernel<E, 64, 16>() : group > 4 ? kernel<E, 64, 8>() : kernel<E, 64, 4>();
}
Kernel kernel_for(int dtype, int head_dim, int group) {
  return dtype == IRIS_DTYPE_FP16 ? kernel_of<Fp16Elem>(head_dim, group) : kernel_of<Bf16Elem>(head_dim, group);
}

struct SparseGrid {
  int ctas;
  size_t part_o, part_ml, bytes;  // offsets of the workspace's parts after row_start, and its size
};
cudaError_t grid_for(const Kernel& k, int64_t rows, int group, int head_dim, int64_t max_pages, int min_steps,
                     SparseGrid* out) {
  int resident = 0;
  const cudaError_t e = resident_warps(reinterpret_cast<const void*>(k.fn), k.bytes, &resident);
  if (e != cudaSuccess) return e;
  const int64_t runs = (rows * ((max_pages + 1) / 2) + min_steps - 1) / min_steps;  // at most
  const int64_t warps = runs < resident ? runs : resident;
  out->ctas = static_cast<int>((warps + kWarps - 1) / kWarps);
  const size_t parts = 2 * static_cast<size_t>(out->ctas) * kWarps * group;
  out->part_o = (static_cast<size_t>(rows + 1) * 4 + 255) / 256 * 256;
  out->part_ml = out->part_o + parts * head_dim * 4;
  out->bytes = out->part_ml + parts * 8;
  return cudaSuccess;
}

// Shortest run of a warp, in steps (one sequence of 128 pages, 8 KV heads: 11.1 us with 2; 13.1, 12.3 and 12.1 with 1,
// 3 and 4: shorter runs leave more parts to join, longer ones fewer warps).
constexpr int kMinSteps = 2;

}  // namespace
}  // namespace iris

using namespace iris;

static bool sparse_shape_ok(int32_t batch, int32_t hq, int32_t hkv, int32_t head_dim, int32_t max_pages) {
  return batch > 0 && hq > 0 && hkv > 0 && max_pages > 0 && hq % hkv == 0 && hq / hkv <= 16 &&
         (head_dim == 64 || head_dim == 128) && hkv <= (1 << 20) &&
         static_cast<int64_t>(batch) * hkv * ((static_cast<int64_t>(max_pages) + 1) / 2) < (1ll << 30);
}

extern "C" size_t iris_b200_sparse_decode_workspace_bytes(int32_t batch, int32_t num_q_heads, int32_t num_kv_heads,
                                                          int32_t head_dim, int32_t max_pages, int32_t device) {
  if (!sparse_shape_ok(batch, num_q_heads, num_kv_heads, head_dim, max_pages)) return 0;
  int before = 0;
  if (cudaGetDevice(&before) != cudaSuccess) return 0;
  if (before != device && cudaSetDevice(device) != cudaSuccess) return 0;
  const int group = num_q_heads / num_kv_heads;
  size_t bytes = 0;
  for (const int dtype : {IRIS_DTYPE_FP16, IRIS_DTYPE_BF16}) {
    SparseGrid grid;
    if (grid_for(kernel_for(dtype, head_dim, group), static_cast<int64_t>(batch) * num_kv_heads, group, head_dim,
                 max_pages, kMinSteps, &grid) != cudaSuccess) {
      bytes = 0;
      break;
    }
    if (grid.bytes > bytes) bytes = grid.bytes;
  }
  if (before != device) cudaSetDevice(before);
  return bytes;
}

extern "C" int iris_b200_int4_sparse_paged_decode(const void* query, const void* k_data, const void* v_data,
                                                  const void* k_scale, const void* v_scale, const int32_t* block_table,
                                                  int64_t block_table_stride, const int32_t* seq_lens,
                                                  const int32_t* page_list, const int32_t* page_count, void* output,
                                                  float* out_lse, int32_t batch, int32_t num_q_heads,
                                                  int32_t num_kv_heads, int32_t head_dim, int64_t num_pages,
                                                  int32_t page_size, int32_t max_pages_per_seq, int32_t max_pages,
                                                  float softmax_scale, int32_t dtype, void* workspace,
                                                  size_t workspace_bytes, int32_t* error_word, void* stream) {
  if (batch < 0 || num_q_heads <= 0 || num_kv_heads <= 0 || num_pages < 0 || max_pages_per_seq < 0 || max_pages <= 0)
    return IRIS_EINVAL;
  if (num_q_heads % num_kv_heads != 0 || !(softmax_scale > 0.0f)) return IRIS_EINVAL;
  if (dtype != IRIS_DTYPE_FP16 && dtype != IRIS_DTYPE_BF16) return IRIS_EINVAL;
  if (batch == 0) return IRIS_OK;
  if (page_size != kPage || !sparse_shape_ok(batch, num_q_heads, num_kv_heads, head_dim, max_pages))
    return IRIS_EUNSUPPORTED;
  if (num_pages == 0) return IRIS_EINVAL;
  const void* ptrs[] = {query, k_data, v_data, k_scale, v_scale, block_table, seq_lens, page_list, page_count, output};
  for (const void* q : ptrs)
    if (q == nullptr) return IRIS_EINVAL;
  if (!aligned_to(query, 16) || !aligned_to(k_data, 16) || !aligned_to(v_data, 16) || !aligned_to(k_scale, 8) ||
      !aligned_to(v_scale, 8) || !aligned_to(output, 8) || !aligned_to(out_lse, 4) || !aligned_to(workspace, 16))
    return IRIS_EALIGN;
  const int group = num_q_heads / num_kv_heads;
  const int64_t rows = static_cast<int64_t>(batch) * num_kv_heads;
  const Kernel k = kernel_for(dtype, head_dim, group);
  clear_stale_cuda_error();
  SparseGrid grid;
  cudaError_t e = grid_for(k, rows, group, head_dim, max_pages, kMinSteps, &grid);
  if (e != cudaSuccess) {
    record_cuda_error(e, "sparse_decode_kernel occupancy");
    return IRIS_ECUDA;
  }
  if (workspace == nullptr || workspace_bytes < grid.bytes) return IRIS_EWORKSPACE;
  SparseParams p = {};
  p.query = query;
  p.k_data = static_cast<const uint8_t*>(k_data);
  p.v_data = static_cast<const uint8_t*>(v_data);
  p.k_scale = static_cast<const __half*>(k_scale);
  p.v_scale = static_cast<const __half*>(v_scale);
  p.block_table = block_table;
  p.table_stride = block_table_stride;
  p.seq_lens = seq_lens;
  p.lists = page_list;
  p.counts = page_count;
  p.output = output;
  p.lse = out_lse;
  p.num_pages = num_pages;
  p.max_pages = max_pages_per_seq;
  p.kv_heads = num_kv_heads;
  p.group = group;
  p.keep = max_pages;
  p.rows = static_cast<int32_t>(rows);
  p.min_steps = kMinSteps;
  p.warps = grid.ctas * kWarps;
  p.vector_counts = aligned_to(page_count, 16) ? 1 : 0;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  p.row_start = reinterpret_cast<int32_t*>(ws);
  p.part_o = reinterpret_cast<float*>(ws + grid.part_o);
  p.part_ml = reinterpret_cast<float*>(ws + grid.part_ml);
  p.scale_log2 = static_cast<float>(static_cast<double>(softmax_scale) * 1.4426950408889634);
  p.err = error_word;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  e = launch_early(k.fn, static_cast<unsigned>(grid.ctas), 32 * kWarps, static_cast<size_t>(k.bytes), s, p);
  if (e == cudaSuccess)
    e = launch_early(k.join, dim3(static_cast<unsigned>(rows), static_cast<unsigned>((group + 3) / 4)), 128, 0, s, p);
  if (e != cudaSuccess) {
    record_cuda_error(e, "sparse_decode_kernel launch");
    return IRIS_ECUDA;
  }
  return IRIS_OK;
}
