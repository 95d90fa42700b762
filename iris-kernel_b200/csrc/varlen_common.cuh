// What attention over new tokens and its weights share: which rows a block
// has, which cached tokens they see, and what becomes of a logit.
//
// Sequence b has n_b new tokens, the last n_b of its seq_lens[b] cached ones;
// new token i is at place seq_lens[b] - n_b + i.  Row r of a (sequence, KV
// head) is its new token r / group with query head r % group of the KV head.
// A row at place `pos` sees token j iff
//   j < seq_lens[b]  and  j >= first_visible  and
//   (j < prefix_lens[b]  or  (j <= pos and (window == 0 or j > pos - window)))
// which is two runs of tokens.
#pragma once

#include "elem.cuh"
#include "umma.cuh"

namespace iris {

constexpr int kTile = 128;        // cached tokens of a tile
constexpr int kTokPage = 16;      // tokens of a page
constexpr float kLog2e = 1.4426950408889634f;

IRIS_DEV float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

struct VarlenBatch {
  const int32_t* block_table;
  int64_t bt_stride;
  const int32_t* seq_lens;
  const int32_t* cu;             // [batch + 1], or NULL: one new token a sequence
  const int32_t* prefix_lens;    // [batch] or NULL
  const int32_t* first_visible;  // [tokens] or NULL
  const float* slopes;           // [hq] or NULL
  int32_t* err;
  int64_t num_pages;
  int32_t tokens;                // rows of the query
  int32_t batch, hq, hkv, group, max_pages;
  int32_t window;                // 0: none
  float scale;                   // softmax scale
  float cap;                     // 0: none
};

// Waits of a whole warp: false (and an error) if the phase does not complete
// within the limit.  The clock is only read once a first round of polls, each of
// which the hardware may let sleep, has failed.
IRIS_DEV bool wait_all(uint64_t* bar, uint32_t parity, int32_t* err) {
  const uint32_t at = smem_u32(bar);
  bool there = false;
#pragma unroll 1
  for (int i = 0; i < 64 && !there; ++i) there = mbar_try_wait(at, parity);
  if (__all_sync(0xffffffffu, there)) return true;
  return __all_sync(0xffffffffu, mbar_wait_bounded(at, parity, err));
}

// New tokens [start, start + count) of sequence b; offsets outside the query are cut off.
struct Span {
  int32_t start, count;
};
IRIS_DEV Span new_tokens(const VarlenBatch& p, int b) {
  if (p.cu == nullptr) return {b, 1};
  const int32_t s = min(max(__ldg(p.cu + b), 0), p.tokens);
  const int32_t e = min(max(__ldg(p.cu + b + 1), s), p.tokens);
  return {s, e - s};
}

// Offsets have to rise from 0 and end inside the query (one warp looks).
IRIS_DEV void check_offsets(const VarlenBatch& p, int lane) {
  if (p.cu == nullptr) return;
  bool bad = lane == 0 && __ldg(p.cu) != 0;
  for (int b = lane; b < p.batch; b += 32) {
    const int32_t s = __ldg(p.cu + b), e = __ldg(p.cu + b + 1);
    bad |= s < 0 || e < s || e > p.tokens;
  }
  if (bad) set_error(p.err, IRIS_ERR_OFFSETS);
}

// Rows that the offsets leave over start here.
IRIS_DEV int32_t used_rows(const VarlenBatch& p) {
  return p.cu == nullptr ? min(p.batch, p.tokens) : min(max(__ldg(p.cu + p.batch), 0), p.tokens);
}

// A sequence's length n in the cache, as far as its pages go; `say` reports what is wrong with it.
IRIS_DEV int32_t cached_tokens(const VarlenBatch& p, int32_t n, int32_t count, bool say) {
  if (n < 0) {
    if (say) set_error(p.err, IRIS_ERR_SEQ_NEGATIVE);
    return 0;
  }
  if ((static_cast<int64_t>(n) + kTokPage - 1) / kTokPage > p.max_pages) {
    if (say) set_error(p.err, IRIS_ERR_BLOCK_TABLE);
    n = p.max_pages * kTokPage;
  }
  if (n > 0 && n < count && say) set_error(p.err, IRIS_ERR_QUERY_LEN);
  return n;
}

IRIS_DEV int warp_sum(int v) { return __reduce_add_sync(0xffffffffu, v); }

// Block u of the blocks of `rows` rows of all sequences with more than `over`
// and at most `most_rows` rows, heaviest first: the last block of every
// sequence, then the one before it, and so on (a block's work grows with its
// tokens' places).  One warp; false: there is no block u.  (With one new token
// a sequence the rows are the host's to choose a kernel by, and all are taken.)
struct Block {
  int32_t b, index;
  Span span;
  int32_t len;  // as the sequence's length stands, not checked
};

// Up to 32 * kHeld sequences: a lane has kHeld of them in registers (one trip to
// memory; the search that asked memory again at each step took 7000 cycles).
constexpr int kHeld = 4;
IRIS_DEV bool find_held_block(const VarlenBatch& p, int u, int rows, int64_t over, int64_t most_rows, int lane, Block* out) {
  int32_t start[kHeld], count[kHeld], len[kHeld], n[kHeld];
  int most = 0;
#pragma unroll
  for (int i = 0; i < kHeld; ++i) {
    const int b = lane + 32 * i;
    start[i] = count[i] = len[i] = 0;
    if (b < p.batch) {
      const Span s = new_tokens(p, b);
      start[i] = s.start;
      count[i] = s.count;
      len[i] = __ldg(p.seq_lens + b);
    }
  }
#pragma unroll
  for (int i = 0; i < kHeld; ++i) {
    const int64_t r = static_cast<int64_t>(count[i]) * p.group;
    n[i] = r > over && r <= most_rows ? static_cast<int32_t>((r + rows - 1) / rows) : 0;
    most = max(most, n[i]);
  }
  most = __reduce_max_sync(0xffffffffu, most);
  auto upto = [&](int depth) {  // blocks among the last `depth` of every sequence
    int x = 0;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) x += min(depth, n[i]);
    return warp_sum(x);
  };
  if (u >= upto(most)) return false;
  int lo = 0, hi = most, before = 0;  // upto(lo) = before <= u < upto(hi)
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1, x = upto(mid);
    if (x <= u) lo = mid, before = x; else hi = mid;
  }
  int left = u - before;
#pragma unroll
  for (int i = 0; i < kHeld; ++i) {
    const unsigned has = __ballot_sync(0xffffffffu, n[i] > lo);
    const int c = __popc(has);
    if (left >= 0 && left < c) {
      const int src = __fns(has, 0, left + 1);
      out->b = src + 32 * i;
      out->index = __shfl_sync(0xffffffffu, n[i], src) - 1 - lo;
      out->span = {__shfl_sync(0xffffffffu, start[i], src), __shfl_sync(0xffffffffu, count[i], src)};
      out->len = __shfl_sync(0xffffffffu, len[i], src);
      return true;
    }
    left -= c;
  }
  return false;
}

IRIS_DEV bool find_block(const VarlenBatch& p, int u, int rows, int64_t over, int64_t most_rows, int lane, Block* out) {
  if (p.cu == nullptr) {
    const int per = (p.group + rows - 1) / rows;
    out->b = u / per;
    out->index = u % per;
    if (out->b >= p.batch) return false;
    out->span = {out->b, 1};
    out->len = __ldg(p.seq_lens + out->b);
    return true;
  }
  if (p.batch <= 32 * kHeld) return find_held_block(p, u, rows, over, most_rows, lane, out);
  auto blocks = [&](int b) {
    const int64_t n = static_cast<int64_t>(new_tokens(p, b).count) * p.group;
    return n > over && n <= most_rows ? static_cast<int32_t>((n + rows - 1) / rows) : 0;
  };
  int most = 0;
  for (int b = lane; b < p.batch; b += 32) most = max(most, blocks(b));
  most = __reduce_max_sync(0xffffffffu, most);
  auto upto = [&](int depth) {
    int n = 0;
    for (int b = lane; b < p.batch; b += 32) n += min(depth, blocks(b));
    return warp_sum(n);
  };
  if (u >= upto(most)) return false;
  int lo = 0, hi = most;  // upto(lo) <= u < upto(hi)
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (upto(mid) <= u) lo = mid; else hi = mid;
  }
  int left = u - upto(lo);
  for (int base = 0; base < p.batch; base += 32) {
    const int b = base + lane;
    const int n = b < p.batch ? blocks(b) : 0;
    const unsigned has = __ballot_sync(0xffffffffu, n > lo);
    const int c = __popc(has);
    if (left < c) {
      const int src = __fns(has, 0, left + 1);
      out->b = base + src;
      out->index = __shfl_sync(0xffffffffu, n, src) - 1 - lo;
      out->span = new_tokens(p, out->b);
      out->len = __ldg(p.seq_lens + out->b);
      return true;
    }
    left -= c;
  }
  return false;
}

// The smallest first visible token of a block's rows (one warp).
IRIS_DEV int32_t first_of_block(const VarlenBatch& p, const Span& sp, int index, int rows, int lane) {
  if (p.first_visible == nullptr) return 0;
  const int64_t r0 = static_cast<int64_t>(index) * rows;
  const int i0 = static_cast<int>(r0 / p.group);
  const int i1 = static_cast<int>(min((r0 + rows - 1) / p.group, static_cast<int64_t>(sp.count - 1)));
  int32_t first = INT32_MAX;
  for (int i = i0 + lane; i <= i1; i += 32) first = min(first, __ldg(p.first_visible + sp.start + i));
  return __reduce_min_sync(0xffffffffu, first);
}

// What one row sees, as two runs [a0, a1) and [b0, b1) of tokens (a: prefix).
struct Sight {
  int32_t a0, a1, b0, b1;
};
IRIS_DEV Sight row_sight(int32_t pos, int32_t first, int32_t prefix, int32_t window, int32_t len) {
  Sight s;
  s.a0 = max(first, 0);
  s.a1 = max(min(prefix, len), 0);  // (differences of places must fit 32 bits)
  s.b0 = window > 0 ? max(s.a0, pos - window + 1) : s.a0;
  s.b1 = min(pos + 1, len);
  return s;
}

// Bits [lo, hi) of 32, bounds anywhere.
IRIS_DEV uint32_t bits_between(int lo, int hi) {
  lo = max(lo, 0);
  hi = min(hi, 32);
  if (hi <= lo) return 0u;
  return (0xffffffffu >> (32 - (hi - lo))) << lo;
}
IRIS_DEV uint32_t sight_bits(const Sight& s, int32_t base) {
  return bits_between(s.a0 - base, s.a1 - base) | bits_between(s.b0 - base, s.b1 - base);
}

// Tiles that a block's rows may see: `head` tiles from `head0` (the prefix) and `body` from `body0`.
struct Tiles {
  int32_t head0, head, body0, body;
  IRIS_DEV int32_t count() const { return head + body; }
  IRIS_DEV int32_t at(int32_t k) const { return k < head ? head0 + k : body0 + (k - head); }
};
IRIS_DEV Tiles tiles_seen(int32_t pos_lo, int32_t pos_hi, int32_t first, int32_t prefix, int32_t window, int32_t len) {
  Tiles t;
  const int32_t a0 = max(first, 0), a1 = min(prefix, len);
  const int32_t b0 = window > 0 ? max(a0, pos_lo - window + 1) : a0, b1 = min(pos_hi + 1, len);
  t.head0 = a0 / kTile;
  t.head = a1 > a0 ? (a1 + kTile - 1) / kTile - t.head0 : 0;
  t.body0 = b0 / kTile;
  t.body = b1 > b0 ? (b1 + kTile - 1) / kTile - t.body0 : 0;
  if (t.head > 0 && t.body > 0 && t.body0 < t.head0 + t.head) {  // tiles of both count once
    const int32_t end = max(t.body0 + t.body, t.head0 + t.head);
    t.body0 = t.head0 + t.head;
    t.body = end - t.body0;
  }
  return t;
}

// tanh, within a few units in the last place of 1 anywhere and relatively near
// 0: 1 - 2 / (1 + e^2x) (right at both infinities), or, where that would cancel, x
// times a polynomial in x^2 (Chebyshev's of degree 5 over |x| <= 0.6: 3e-9).
constexpr float kTanhNear = 0.6f;
IRIS_DEV float2 tanh_near(float2 x) {
  const float2 q = __fmul2_rn(x, x);
  float2 r = make_float2(-0.00585643f, -0.00585643f);
  r = __ffma2_rn(r, q, make_float2(0.02075748f, 0.02075748f));
  r = __ffma2_rn(r, q, make_float2(-0.05376992f, -0.05376992f));
  r = __ffma2_rn(r, q, make_float2(0.13331705f, 0.13331705f));
  r = __ffma2_rn(r, q, make_float2(-0.33333284f, -0.33333284f));
  r = __ffma2_rn(r, q, make_float2(1.0f, 1.0f));
  return __fmul2_rn(x, r);
}
IRIS_DEV float tanh_f(float x) {
  const float t = ex2(2.0f * kLog2e * x);
  const float far = fmaf(-2.0f, rcp(1.0f + t), 1.0f);
  return fabsf(x) < kTanhNear ? tanh_near(make_float2(x, x)).x : far;
}
// s = cap2 * tanh(s), by a whole warp; false: some lie too far out for the
// polynomial, and s is as it was.  Logits mostly lie well inside a cap, and then
// no exponential and no reciprocal is needed, whose unit (16 a cycle and SM) would
// bound the kernel.
template <int N>
IRIS_DEV bool cap_near(float (&s)[N], float cap2) {
  float most = 0.0f;
#pragma unroll
  for (int j = 0; j < N; ++j) most = fmaxf(most, fabsf(s[j]));
  if (__any_sync(0xffffffffu, most >= kTanhNear)) return false;
#pragma unroll
  for (int j = 0; j < N; j += 2) {
    const float2 y = __fmul2_rn(tanh_near(make_float2(s[j], s[j + 1])), make_float2(cap2, cap2));
    s[j] = y.x;
    s[j + 1] = y.y;
  }
  return true;
}

// Two's power as fp32, |e| < 127.
IRIS_DEV float pow2i(int e) { return __int_as_float((e + 127) << 23); }

// ---------------------------------------------------------- query rows in fp16
// A query row goes to the tensor cores as fp16 times a power of two that
// brings its largest value into [2^15, 2^16): exact for fp16 and bf16 values
// down to 2^-29 of the largest.  Within a group of 8 dims the order is 0 4 1 5
// 2 6 3 7, as the nibbles of a word come apart (stored keys have it too, so
// products do not change).  A row with a value that is not finite becomes NaN.
//
// The larger magnitude's bits of a pair, of either type.
IRIS_DEV uint32_t pair_size(uint32_t w) { return max(w & 0x7fffu, (w >> 16) & 0x7fffu); }
// From a row's largest magnitude's bits: the power to scale by (NaN: not finite), and what undoes it.
IRIS_DEV float row_power(uint32_t most, bool bf16, float* up) {
  const bool finite = most < (bf16 ? 0x7f80u : 0x7c00u);
  const float top = bf16 ? __uint_as_float(most << 16) : __half2float(__ushort_as_half(static_cast<unsigned short>(most)));
  int e = 15;
  if (finite && top > 0.0f) e = max(static_cast<int>((__float_as_uint(top) >> 23) & 255) - 127, -110);
  *up = finite ? pow2i(15 - e) : __int_as_float(0x7fffffff);
  return pow2i(e - 15);
}
IRIS_DEV uint32_t scale_pair(uint32_t w, bool bf16, float up) {
  const float2 v = bf16 ? Bf16Elem::unpack(w) : Fp16Elem::unpack(w);
  return Fp16Elem::pack(v.x * up, v.y * up);
}
// `words`: a thread's pairs as loaded; `widest` takes the largest magnitude's
// bits over the threads that share the row.  Returns the factor that undoes the power.
template <int kWords, typename F>
IRIS_DEV float scale_row_part(uint32_t (&words)[kWords], bool bf16, F&& widest) {
  uint32_t most = 0;
#pragma unroll
  for (int i = 0; i < kWords; ++i) most = max(most, pair_size(words[i]));
  float up;
  const float back = row_power(widest(most), bf16, &up);
#pragma unroll
  for (int i = 0; i < kWords; ++i) words[i] = scale_pair(words[i], bf16, up);
  return back;
}

// Eight dims (four pairs as loaded) in the order above.
IRIS_DEV uint4 order8(uint32_t w0, uint32_t w1, uint32_t w2, uint32_t w3) {
  return make_uint4(prmt(w0, w2, 0x5410), prmt(w0, w2, 0x7632), prmt(w1, w3, 0x5410), prmt(w1, w3, 0x7632));
}

// Byte offset of 16-byte chunk c (of D / 8) of row r in an operand tile of 128 rows.
IRIS_DEV uint32_t operand_at(int row, int chunk) {
  return (chunk >> 3) * (kTile * 128) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4);
}

// Page of token j as the table has it (to be checked where it is used, so that
// nothing waits for the load before), 0 past the sequence's end.
IRIS_DEV int32_t raw_page(const VarlenBatch& p, int b, int32_t j, int32_t len) {
  return j < len ? __ldg(p.block_table + b * p.bt_stride + j / kTokPage) : 0;
}
// 0 (and an error) for an id outside the cache.
IRIS_DEV int32_t checked_page(const VarlenBatch& p, int32_t id) {
  if (static_cast<uint32_t>(id) < static_cast<uint32_t>(p.num_pages)) return id;  // (num_pages fits 31 bits)
  set_error(p.err, IRIS_ERR_PAGE_ID);
  return 0;
}
IRIS_DEV int32_t page_of(const VarlenBatch& p, int b, int32_t j, int32_t len) {
  return checked_page(p, raw_page(p, b, j, len));
}

// ------------------------------------------------------- packed tiles by TMA
// A tile's packed rows of one head land as [128 tokens][D / 2 bytes], a page
// (16 rows) a copy, 16-byte chunk c of row r at c ^ ((r >> 1) & 3) (D = 128: the
// 64-byte swizzle) or c ^ ((r >> 2) & 1) (D = 64: the 32-byte one), so that a
// warp whose threads each read a row of their own meets no bank twice.  (Loads
// straight from memory, a row a thread, kept L1 57 % busy with their 32 lines
// each.)  Pages past the sequence's end are left out: what the rows held before
// has finite nibbles and counts for nothing.
template <int D>
IRIS_DEV uint32_t packed_at(int row, int chunk) {
  return row * (D / 2) + (D == 128 ? (chunk ^ ((row >> 1) & 3)) << 4 : (chunk ^ ((row >> 2) & 1)) << 4);
}
// One warp: the copies of a tile whose first token is j0; lane i < 8 has page i's
// id and issues its copy (a loop over the lanes after all, but half as long as
// one that hands the ids round).
template <int D>
IRIS_DEV void load_packed(uint8_t* dst, const CUtensorMap* map, int32_t page, int32_t j0, int32_t len, int h,
                          uint64_t* bar, int lane) {
  const int pages = min(kTile / kTokPage, (len - j0 + kTokPage - 1) / kTokPage);
  if (elect_one()) mbar_arrive_expect_tx(bar, pages * kTokPage * (D / 2));
  __syncwarp();
  if (lane < pages) tma_load_4d(dst + lane * kTokPage * (D / 2), map, 0, 0, h, page, bar);
  __syncwarp();
}

// Host: into how many chunks to cut each of `units` rows of `tiles` tiles, for a
// GPU that runs `slots` blocks at once: the one whose rounds of blocks take the
// least, a block costing `start` tiles before its first.
inline int64_t best_chunks(int64_t units, int64_t tiles, int64_t slots, int64_t start, int64_t most) {
  if (most > 1024) most = 1024;
  if (most < 1) most = 1;
  int64_t best = 1, least = INT64_MAX;
  for (int64_t n = 1; n <= most; ++n) {
    const int64_t cost = (units * n + slots - 1) / slots * ((tiles + n - 1) / n + start);
    if (cost < least) {
      least = cost;
      best = n;
    }
    if (units * n > 4 * slots) break;  // finer cuts only add starts
  }
  return best;
}

// Host: the cache [pages, 16, Hkv, D / 2] as (row bytes, 16 tokens, heads, pages), a box of one page of one head.
inline bool packed_map(CUtensorMap* map, const void* base, int dim, int hkv, int64_t num_pages) {
  using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static const Encode encode = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    const bool ok = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess &&
                    q == cudaDriverEntryPointSuccess;
    return ok ? reinterpret_cast<Encode>(f) : nullptr;
  }();
  if (encode == nullptr) return false;
  const cuuint64_t row = static_cast<cuuint64_t>(dim) / 2;
  const cuuint64_t dims[4] = {row, kTokPage, static_cast<cuuint64_t>(hkv), static_cast<cuuint64_t>(num_pages)};
  const cuuint64_t strides[3] = {row * hkv, row, row * hkv * kTokPage};
  const cuuint32_t box[4] = {static_cast<cuuint32_t>(row), kTokPage, 1u, 1u}, step[4] = {1u, 1u, 1u, 1u};
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<void*>(base), dims, strides, box, step,
                CU_TENSOR_MAP_INTERLEAVE_NONE, dim == 128 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_32B,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace iris
