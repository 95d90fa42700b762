// Attention of sequences with few rows (at most kFewRows query rows a KV head:
// single tokens, drafts).  With 128 rows to a product most of it would be
// padding, and one warp would have all the softmax; so the products are turned
// around: cached tokens are the rows, query rows the columns.
//   S [128 tokens x rows] = K Q^T   K unpacked straight into tensor memory
//                                   (thread = token = lane), Q in shared memory
//   O [dims x rows]       = V^T P^T V as it lies in shared memory (MN-major),
//                                   P in shared memory
// A thread has a token's logits in registers, then a dim's outputs; sums over
// tokens of the probabilities stay in the thread until the end.  Keys go in as
// whole numbers with an accumulator a group of 32 dims, and a token's fp32 scales
// join the sums: no product by the scale, and nothing is rounded.  Values are fp16,
// each token's scaled by a power of two of its own; probabilities are fp16 too,
// relative to the largest probability times power of the row, so values that it
// does not see, or that weigh nothing, cost the others no bits.  A product of so
// few columns takes its latency, about 140 cycles, when it adds to the one before
// it; dealt out over several accumulators (the groups; four for the outputs, that
// are added up as they are read) they follow each other without it.
// A block is two warpgroups and a warp: one group unpacks keys and makes
// probabilities (a cached token a thread), the other unpacks values (likewise) and
// adds up outputs (a dim a thread), the warp issues copies and products.  Packed
// rows come by TMA into the buffers that the groups have just emptied; two or
// three blocks an SM overlap.  Loops over a token's groups are not unrolled: the
// kernel's instructions come from a small cache too.
#pragma once

#include "varlen_common.cuh"

namespace iris {

constexpr int kFewRows = 32;

struct AttendParams {
  VarlenBatch s;
  const uint16_t* query;
  const uint8_t *k_data, *v_data;
  const uint8_t *k_scale, *v_scale;
  void* out;
  float* out_lse;    // or NULL
  // where several blocks share a row's tiles, their parts: of sequences with many rows
  float* part_o;     // [splits][tokens][hq][D]
  float* part_lse;   // [splits][tokens][hq]
  // and with few
  float* few_o;      // [batch][hkv][chunks][cols][D]
  float* few_lse;    // [batch][hkv][chunks][cols]
  int64_t q_stride;  // elements between tokens of the query
  int32_t splits;    // slots of sequences with many rows
  int32_t chunks;    // slots of sequences with few rows,
  int32_t per;       // each of so many tiles
  int32_t bf16;
  int32_t few, many; // which kernels run
};

constexpr float kRise = 7.0f;  // log2 that a row's logits may pass its reference by
constexpr float kHead = 8.0f;  // log2 of the reference's own probability
constexpr float kFarOut = 4194304.0f;  // 2^22: from there on a reference is two numbers
#define kMinusInf (-__int_as_float(0x7f800000))

// Rows that the offsets leave over: zeros.
template <int D>
IRIS_DEV void clear_unused(const AttendParams& p) {
  for (int64_t row = static_cast<int64_t>(used_rows(p.s)) * p.s.hq + blockIdx.x;
       row < static_cast<int64_t>(p.s.tokens) * p.s.hq; row += gridDim.x) {
    if (threadIdx.x < D / 2) reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(p.out) + row * D)[threadIdx.x] = 0u;
    if (threadIdx.x == 0 && p.out_lse != nullptr) p.out_lse[row] = kMinusInf;
  }
}

template <int D, int kCols>
struct FewCfg {
  static constexpr int kN = kCols <= 16 ? 16 : 32;     // columns of a product
  static constexpr int kValues = kTile * D * 2;
  static constexpr int kQuery = kN * D * 2;
  static constexpr int kProb = kN * kTile * 2;
  static constexpr int kPacked = kTile * D / 2;
  static constexpr int kSmem = 1024 + kValues + kQuery + kProb + 2 * kPacked;
  static constexpr int kSums = D / 32;                 // accumulators of a logit
  static constexpr int kParts = D / 32;                // and of an output
  static constexpr int kKeyColumns = D / 2;
  static constexpr int kUsed = kKeyColumns + kSums * kN;
  static constexpr int kColumns = kUsed <= 64 ? 64 : kUsed <= 128 ? 128 : 256;
  static constexpr int kBlocks = kCols <= 8 ? 3 : 2;   // an SM
};

struct FewShared {
  uint64_t k_here, v_here;             // packed rows have landed
  uint64_t s_done, o_done;             // products are done
  uint64_t k_ready, p_ready, v_ready;  // operands are in their places
  uint64_t o_free;                     // outputs are read
  uint64_t e_ready;                    // the values' powers are in their place
  uint32_t tmem;
  int32_t live, b, index, start, count, len, first_lo;
  int32_t v_exp[kTile];                // what a token's values were scaled down by, log2
  int32_t risen[2];                    // whether references rose in a tile
  float4 row[kFewRows];                // factor, m, the limit r + 15 (-inf before there is a reference), r
  float2 more[kFewRows];               // place, slope
  int4 sight[kFewRows];
  float warp_top[4][kFewRows];
  float fall[2][kFewRows];             // what a rise of the reference multiplies sums by
  float total[4][kFewRows];
  uint32_t spoilt[kFewRows];
  int32_t all_lo, all_hi;
};

// One warpgroup's barrier, and an "or" over it.
template <int kId>
IRIS_DEV void group_sync() { asm volatile("bar.sync %0, 128;" ::"n"(kId) : "memory"); }
template <int kId>
IRIS_DEV bool group_or(bool v) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.or.pred q, %2, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(static_cast<uint32_t>(v)), "n"(kId)
      : "memory");
  return r != 0;
}
template <int D, int kCols, bool kCap, bool kBias>
__global__ void __launch_bounds__(288, FewCfg<D, kCols>::kBlocks) varlen_few_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                      const AttendParams p) {
  using C = FewCfg<D, kCols>;
  constexpr int kGroups = D / 32, kN = C::kN, kStep = kCols < 8 ? 4 : 8;
  extern __shared__ uint8_t smem_raw[];
  __shared__ FewShared sh;
  const int group_id = threadIdx.x >> 7, tid = threadIdx.x & 127, warp = tid >> 5, lane = tid & 31;
  const int chunk = blockIdx.x % p.chunks, h = blockIdx.x / p.chunks % p.s.hkv, unit = blockIdx.x / p.chunks / p.s.hkv;
  if (threadIdx.x == 0) {
    mbar_init(&sh.s_done, 1);
    mbar_init(&sh.o_done, 1);
    mbar_init(&sh.k_here, 1);
    mbar_init(&sh.v_here, 1);
    mbar_init(&sh.k_ready, 128);
    mbar_init(&sh.p_ready, 128);
    mbar_init(&sh.v_ready, 128);
    mbar_init(&sh.o_free, 128);
    mbar_init(&sh.e_ready, 128);
    fence_barrier_init();
    sh.all_lo = 0;
    sh.all_hi = INT32_MAX;
  }
  if (threadIdx.x < kFewRows) {  // columns that no row has: computed along, and never written
    sh.spoilt[threadIdx.x] = 0;
    sh.row[threadIdx.x] = make_float4(0.0f, 0.0f, -kMinusInf, 0.0f);
    sh.more[threadIdx.x] = make_float2(0.0f, 0.0f);
    sh.sight[threadIdx.x] = make_int4(0, 0, 0, 0);
  }
  grid_dependency_wait();
  grid_dependents_launch();
  if (threadIdx.x < 32) {
    if (blockIdx.x == 0) check_offsets(p.s, lane);
    Block blk = {0, 0, {0, 0}, 0};
    const bool live = find_block(p.s, unit, kCols, 0, kFewRows, lane, &blk);
    int first = 0;
    Span sp = {0, 0};
    int32_t len = 0;
    if (live) {
      sp = blk.span;
      len = cached_tokens(p.s, blk.len, sp.count, lane == 0 && h == 0 && chunk == 0 && blk.index == 0);
      first = first_of_block(p.s, sp, blk.index, kCols, lane);
    }
    if (lane == 0) {
      sh.live = live;
      sh.b = blk.b;
      sh.index = blk.index;
      sh.start = sp.start;
      sh.count = sp.count;
      sh.len = len;
      sh.first_lo = first;
    }
  }
  if (!p.many) clear_unused<D>(p);
  __syncthreads();
  if (!sh.live) return;
  const int b = sh.b, len = sh.len, group = p.s.group;
  const int rows_all = sh.count * group, r0 = sh.index * kCols, cols = min(kCols, rows_all - r0);
  const int32_t off = len - sh.count;
  const int32_t prefix = p.s.prefix_lens != nullptr ? __ldg(p.s.prefix_lens + b) : 0;
  const Tiles tiles = tiles_seen(off + r0 / group, off + (r0 + cols - 1) / group, sh.first_lo, prefix, p.s.window, len);
  const int all = tiles.count();
  const int k0 = chunk * p.per, n = min(all - k0, p.per);
  const bool whole = p.chunks == 1;
  auto row_at = [&](int c) {  // index of column c's row in the output
    const int r = r0 + c;
    return static_cast<int64_t>(sh.start + r / group) * p.s.hq + h * group + r % group;
  };
  const int64_t part = ((static_cast<int64_t>(b) * p.s.hkv + h) * p.chunks + chunk) * kCols;
  if (n <= 0) {
    const int tid = threadIdx.x;
    if (!whole) {
      if (tid < cols) p.few_lse[part + tid] = kMinusInf;
    } else {
      for (int c = 0; c < cols; ++c) {
        if (tid < D / 2) reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(p.out) + row_at(c) * D)[tid] = 0u;
        if (tid == 0 && p.out_lse != nullptr) p.out_lse[row_at(c)] = kMinusInf;
      }
    }
    return;
  }

  uint8_t* base = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const uint32_t v_tile = smem_u32(base), q_tile = v_tile + C::kValues, p_tile = q_tile + C::kQuery;
  uint8_t *k_packed = base + C::kValues + C::kQuery + C::kProb, *v_packed = k_packed + C::kPacked;
  const uint32_t k_raw = smem_u32(k_packed), v_raw = smem_u32(v_packed);
  auto first_token = [&](int k) { return tiles.at(k0 + k) * kTile; };
  // ---- scales of the tile that is next to be unpacked: keys' by the first group, values' by the second
  const uint8_t* scales = group_id == 0 ? p.k_scale : p.v_scale;
  uint32_t sc2[kGroups / 2];
  auto fetch_scales = [&](int32_t page, int32_t j) {
    const uint8_t* x = scales + ((static_cast<int64_t>(page) * kTokPage + (j & (kTokPage - 1))) * p.s.hkv + h) * (D / 16);
    if constexpr (D == 128) {
      const uint2 v = j < len ? __ldg(reinterpret_cast<const uint2*>(x)) : make_uint2(0, 0);
      sc2[0] = v.x;
      sc2[1] = v.y;
    } else {
      sc2[0] = j < len ? __ldg(reinterpret_cast<const uint32_t*>(x)) : 0u;
    }
  };
  auto scale_bits = [&](int c) {  // of group c
    const uint32_t w = D == 128 && c >= 2 ? sc2[kGroups / 2 - 1] : sc2[0];
    return (w >> (16 * (c & 1))) & 0xffffu;
  };
  int32_t page = 0;  // of this thread's token in the tile after that, not checked yet
  if (group_id < 2) {
    fetch_scales(page_of(p.s, b, first_token(0) + tid, len), first_token(0) + tid);
    if (n > 1) page = raw_page(p.s, b, first_token(1) + tid, len);
  }

  if (threadIdx.x < 32) umma_alloc(&sh.tmem, C::kColumns);
  // ---- query rows: four threads a row
  if (group_id == 0) {
    const int c = tid >> 2, part = tid & 3;
    const bool valid = c < cols;
    const int r = r0 + (valid ? c : 0), i = r / group, g = r % group;
    const int64_t token = sh.start + i;
    const int head = h * group + g;
    constexpr int kWords = D / 8;
    uint32_t w[kWords];
#pragma unroll
    for (int x = 0; x < kWords / 4; ++x) {
      const uint4 v = *reinterpret_cast<const uint4*>(p.query + token * p.q_stride + static_cast<int64_t>(head) * D +
                                                      part * (D / 4) + 8 * x);
      w[4 * x] = v.x;
      w[4 * x + 1] = v.y;
      w[4 * x + 2] = v.z;
      w[4 * x + 3] = v.w;
    }
    const float back = scale_row_part<kWords>(w, p.bf16 != 0, [](uint32_t m) {
      m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
      return max(m, __shfl_xor_sync(0xffffffffu, m, 2));
    });
#pragma unroll
    for (int x = 0; x < kWords / 4; ++x) {
      if (!valid) break;
      const uint4 v = order8(w[4 * x], w[4 * x + 1], w[4 * x + 2], w[4 * x + 3]);
      const int ch = part * (D / 32) + x;
      sts128(q_tile + (ch >> 3) * (kN * 128) + c * 128 + (((ch & 7) ^ (c & 7)) << 4), v.x, v.y, v.z, v.w);
    }
    if (part == 0 && valid) {
      const int32_t pos = off + i;
      const Sight see = row_sight(pos, p.s.first_visible != nullptr ? __ldg(p.s.first_visible + token) : 0, prefix,
                                  p.s.window, len);
      sh.row[c] = make_float4(fminf(kCap ? p.s.scale * back / p.s.cap : p.s.scale * kLog2e * back, 1e38f), 0.0f, kMinusInf, 0.0f);
      sh.more[c] = make_float2(__int_as_float(pos), kBias ? -__ldg(p.s.slopes + head) * kLog2e : 0.0f);
      sh.sight[c] = make_int4(see.a0, see.a1, see.b0, see.b1);
      atomicMax(&sh.all_lo, see.b0);
      atomicMin(&sh.all_hi, see.b1);
    }
  }
  fence_proxy_async_shared();
  umma_fence_before();
  __syncthreads();
  umma_fence_after();
  const uint32_t tmem = sh.tmem, lanes = tmem + (static_cast<uint32_t>(warp * 32) << 16);
  const uint32_t s_at = C::kKeyColumns;
  const float cap2 = p.s.cap * kLog2e;

  bool ok = true;
  if (group_id == 2) {
    // ================ copies and products
    auto page_at = [&](int k) { return lane < 8 ? raw_page(p.s, b, first_token(k) + lane * kTokPage, len) : 0; };
    int32_t next = checked_page(p.s, page_at(0)), later = n > 1 ? page_at(1) : 0;
    load_packed<D>(k_packed, &k_map, next, first_token(0), len, h, &sh.k_here, lane);
    load_packed<D>(v_packed, &v_map, next, first_token(0), len, h, &sh.v_here, lane);
#pragma unroll 1
    for (int k = 0; k < n; ++k) {
      if (!(ok = wait_all(&sh.k_ready, k & 1, p.s.err))) break;
      if (k > 0 && !(ok = wait_all(&sh.o_free, (k - 1) & 1, p.s.err))) break;  // the sums' place is free
      if (elect_one()) {
        umma_fence_after();
#pragma unroll
        for (int x = 0; x < D / 16; ++x) {  // the groups in turn, twice
          const int g = x % kGroups, s = 2 * g + x / kGroups;
          umma_ts(tmem + s_at + g * kN, tmem + 8 * s, umma_desc(q_tile + (s >> 2) * (kN * 128) + (s & 3) * 32, 16, 1024),
                  umma_idesc(kTile, kN, false, false), x >= kGroups);
        }
        umma_commit(smem_u32(&sh.s_done));
      }
      __syncwarp();
      if (k + 1 < n) {
        next = checked_page(p.s, later);
        if (k + 2 < n) later = page_at(k + 2);
        load_packed<D>(k_packed, &k_map, next, first_token(k + 1), len, h, &sh.k_here, lane);
      }
      if (!(ok = wait_all(&sh.v_ready, k & 1, p.s.err))) break;
      if (k + 1 < n) load_packed<D>(v_packed, &v_map, next, first_token(k + 1), len, h, &sh.v_here, lane);
      if (!(ok = wait_all(&sh.p_ready, k & 1, p.s.err))) break;
      if (elect_one()) {
        umma_fence_after();
        // (64 dims: the product's other 64 rows are the same values again, column blocks 0 bytes apart)
#pragma unroll
        for (int s = 0; s < kTile / 16; ++s)
          umma_ss(tmem + s_at + (s % C::kParts) * kN, umma_desc(v_tile + s * 2048, D == 128 ? kTile * 128 : 0, 1024),
                  umma_desc(p_tile + (s >> 2) * (kN * 128) + (s & 3) * 32, 16, 1024), umma_idesc(kTile, kN, true, false),
                  s >= C::kParts);
        umma_commit(smem_u32(&sh.o_done));
      }
      __syncwarp();
    }
    if (!ok) {  // a wait gave up: copies that are under way land before the block ends
      for (uint32_t parity = 0; parity < 2; ++parity) {
        mbar_wait_bounded(&sh.k_here, parity, p.s.err);
        mbar_wait_bounded(&sh.v_here, parity, p.s.err);
      }
    }
    __syncthreads();
  } else if (group_id == 0) {
    // ================ keys and probabilities: a token a thread
    const int32_t all_lo = sh.all_lo, all_hi = sh.all_hi;
    float l[kCols];  // this thread's tokens' part of the sums
#pragma unroll
    for (int c = 0; c < kCols; ++c) l[c] = 0.0f;
#pragma unroll 1
    for (int k = 0; k < n; ++k) {
      const int32_t base_j = first_token(k), j = base_j + tid;
      // ---- keys into tensor memory (the product before has read its own: s_done)
      ok = wait_all(&sh.k_here, k & 1, p.s.err) && ok;
#pragma unroll 1
      for (int c = 0; c < kGroups; ++c) {
        const uint4 w4 = lds128(k_raw + packed_at<D>(tid, c));
        const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
        uint32_t x[16];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[4 * i] = int4_lo_exact(w[i]);
          x[4 * i + 1] = int4_hi_exact(w[i]);
          x[4 * i + 2] = int4_lo_exact(w[i] >> 8);
          x[4 * i + 3] = int4_hi_exact(w[i] >> 8);
        }
        umma_st16(lanes + 16 * c, x);
      }
      umma_wait_st();
      umma_fence_before();
      mbar_arrive(&sh.k_ready);
      float sc[kGroups];
      {
        bool odd = false;  // a scale that is not finite: NaN logits
#pragma unroll
        for (int c = 0; c < kGroups; ++c) {
          const uint32_t bits = scale_bits(c);
          odd |= (bits & 0x7fffu) >= 0x7c00u;
          sc[c] = __half2float(__ushort_as_half(static_cast<unsigned short>(bits)));
        }
        if (odd) sc[0] = __int_as_float(0x7fffffff);
      }
      if (k + 1 < n) {
        fetch_scales(checked_page(p.s, page), first_token(k + 1) + tid);
        if (k + 2 < n) page = raw_page(p.s, b, first_token(k + 2) + tid, len);
      }
      const bool full = all_lo <= base_j && base_j + kTile <= all_hi;

      // ---- logits in log2 units, -inf where a token is not seen
      ok = wait_all(&sh.s_done, k & 1, p.s.err) && ok;
      umma_fence_after();
      float y[kCols];
#pragma unroll
      for (int c0 = 0; c0 < kCols; c0 += kStep) {
        if (c0 >= cols) break;
        uint32_t v[C::kSums][kStep];
#pragma unroll
        for (int g = 0; g < C::kSums; ++g) umma_ld<kStep>(lanes + s_at + g * kN + c0, v[g]);
        umma_wait_ld();
        float x[kStep];
#pragma unroll
        for (int i = 0; i < kStep; ++i) {
          x[i] = 0.0f;
#pragma unroll
          for (int g = 0; g < C::kSums; ++g) {
            asm volatile("" : "+r"(v[g][i]));
            x[i] = fmaf(__uint_as_float(v[g][i]), sc[g], x[i]);
          }
          x[i] *= sh.row[c0 + i].x;
        }
        if (kCap && !cap_near(x, cap2)) {
#pragma unroll
          for (int i = 0; i < kStep; ++i) x[i] = cap2 * tanh_f(x[i]);
        }
#pragma unroll
        for (int i = 0; i < kStep; ++i) {
          const int c = c0 + i;
          if (kBias) x[i] = fmaf(sh.more[c].y, fabsf(static_cast<float>(__float_as_int(sh.more[c].x) - j)), x[i]);
          if (!full) {
            const int4 z = sh.sight[c];
            if (!((j >= z.x && j < z.y) || (j >= z.z && j < z.w))) x[i] = kMinusInf;
          }
          y[c] = x[i];
        }
      }
      // ---- what a token adds to a row has the size 2^(y + ve)
      ok = wait_all(&sh.e_ready, k & 1, p.s.err) && ok;
      const int ve = sh.v_exp[tid];
      const float lift = kHead + static_cast<float>(ve), unlift = pow2i(-ve - 8);
      bool rise = false;
#pragma unroll
      for (int c = 0; c < kCols; ++c) {
        if (c % kStep == 0 && c >= cols) break;
        rise |= (y[c] - sh.row[c].y) + lift > sh.row[c].z;
      }
      bool risen = false;
      if (group_or<1>(rise || !ok)) {
        // something passes its row's reference by too much: the largest of the tile is the new one.  Where that or m is far
        // out, m becomes about the largest (0, if that is not), and what lies above it is looked at again.
        bool again = false;
        float m_old = 0.0f, r_old = 0.0f;
        risen = true;
#pragma unroll 1
        for (int look = 0; ; ++look) {
          if (group_or<1>(!ok)) {
            ok = false;
            break;
          }
#pragma unroll
          for (int c = 0; c < kCols; ++c) {
            if (c >= cols) break;
            float t = (y[c] - sh.row[c].y) + static_cast<float>(ve);
#pragma unroll
            for (int x = 16; x > 0; x >>= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, x));
            if (lane == 0) sh.warp_top[warp][c] = t;
          }
          group_sync<1>();
          if (tid < cols) {
            const float4 f = sh.row[tid];
            const float t =
                fmaxf(fmaxf(sh.warp_top[0][tid], sh.warp_top[1][tid]), fmaxf(sh.warp_top[2][tid], sh.warp_top[3][tid]));
            if (look == 0) {
              m_old = f.y;
              r_old = f.z == kMinusInf ? kMinusInf : f.w;
            }
            const bool go = look == 0 ? t + kHead > f.z : again;
            again = go && look < 3 && (fabsf(t) >= kFarOut || (look == 0 && f.y != 0.0f));
            const float m = again ? (fabsf(f.y + t) >= kFarOut ? rintf(f.y + t) : 0.0f) : f.y, r = go && !again ? rintf(t) : f.w;
            sh.fall[k & 1][tid] = go ? ex2((m_old - m) + (r_old - r)) : look == 0 ? 1.0f : sh.fall[k & 1][tid];
            sh.row[tid] = make_float4(f.x, m, go && !again ? r + (kHead + kRise) : f.z, r);
          }
          group_sync<1>();
          if (!group_or<1>(again)) break;
        }
        if (!ok) break;
#pragma unroll
        for (int c = 0; c < kCols; ++c) {
          if (c >= cols) break;
          l[c] *= sh.fall[k & 1][c];
        }
      }
      if (tid == 0) sh.risen[k & 1] = risen;
      // ---- probabilities: fp16, K-major [row][token], and their sums
      if (k > 0) ok = wait_all(&sh.o_done, (k - 1) & 1, p.s.err) && ok;  // the product before has read its own
      const uint32_t p_at = p_tile + (tid >> 6) * (kN * 128) + (tid & 7) * 2, p_chunk = (tid & 63) >> 3;
#pragma unroll
      for (int c = 0; c < kCols; ++c) {
        if (c % kStep == 0 && c >= cols) break;
        const float e = ex2((y[c] - sh.row[c].y) + (lift - sh.row[c].w));
        l[c] = fmaf(e, unlift, l[c]);
        asm volatile("st.shared.u16 [%0], %1;" ::"r"(p_at + c * 128 + ((p_chunk ^ (c & 7)) << 4)),
                     "h"(__half_as_ushort(__float2half_rn(e)))
                     : "memory");
      }
      fence_proxy_async_shared();
      umma_fence_before();
      mbar_arrive(&sh.p_ready);
    }
    // sums over the tokens
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
      if (c >= cols) break;
      float t = l[c];
#pragma unroll
      for (int x = 16; x > 0; x >>= 1) t += __shfl_xor_sync(0xffffffffu, t, x);
      if (lane == 0) sh.total[warp][c] = t;
    }
    umma_fence_before();
    __syncthreads();
    umma_fence_after();
    if (warp == 0) umma_free(tmem, C::kColumns);
  } else {
    // ================ values, a token a thread, and outputs, a dim a thread
    float o[kCols];
#pragma unroll
    for (int c = 0; c < kCols; ++c) o[c] = 0.0f;
#pragma unroll 1
    for (int k = 0; k <= n; ++k) {
      if (k > 0) {  // the outputs of the tile before (whose product has then read the values)
        if (!(ok = wait_all(&sh.o_done, (k - 1) & 1, p.s.err))) break;
        umma_fence_after();
        if (sh.risen[(k - 1) & 1]) {
#pragma unroll
          for (int c = 0; c < kCols; ++c) {
            if (c >= cols) break;
            o[c] *= sh.fall[(k - 1) & 1][c];
          }
        }
#pragma unroll
        for (int c0 = 0; c0 < kCols; c0 += kStep) {
          if (c0 >= cols) break;
          uint32_t v[C::kParts][kStep];
#pragma unroll
          for (int g = 0; g < C::kParts; ++g) umma_ld<kStep>(lanes + s_at + g * kN + c0, v[g]);
          umma_wait_ld();
#pragma unroll
          for (int i = 0; i < kStep; ++i) {
            float t = 0.0f;
#pragma unroll
            for (int g = 0; g < C::kParts; ++g) {
              asm volatile("" : "+r"(v[g][i]));
              t += __uint_as_float(v[g][i]);
            }
            o[c0 + i] += t;
          }
        }
        umma_fence_before();
        mbar_arrive(&sh.o_free);
        if (k == n) break;
      }
      // a power of two for each token (the powers before have been read: the product that they went into is done)
      uint32_t bad = 0, most = 0;
#pragma unroll
      for (int c = 0; c < kGroups; ++c) {
        const uint32_t mag = scale_bits(c) & 0x7fffu;
        if (mag >= 0x7c00u) bad |= 1u << c; else most = max(most, mag);
      }
      const int e = static_cast<int>(most >> 10);
      const float up = pow2i(27 - e);
      sh.v_exp[tid] = e - 27;
      mbar_arrive(&sh.e_ready);
      if (bad != 0) {
        const int32_t j = first_token(k) + tid;
        for (int c = 0; c < cols; ++c) {
          const int4 z = sh.sight[c];
          if ((j >= z.x && j < z.y) || (j >= z.z && j < z.w)) atomicOr(&sh.spoilt[c], bad);
        }
      }
      if (!(ok = wait_all(&sh.v_here, k & 1, p.s.err))) break;
#pragma unroll 1
      for (int c = 0; c < kGroups; ++c) {
        const uint4 w4 = lds128(v_raw + packed_at<D>(tid, c));
        const float f =
            (bad >> c) & 1u ? 0.0f : __half2float(__ushort_as_half(static_cast<unsigned short>(scale_bits(c)))) * up;
        const __half2 s = u32_as_h2(Fp16Elem::pack(f, f));
        const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
          sts128(v_tile + operand_at(tid, 4 * c + i), h2_as_u32(__hmul2(u32_as_h2(int4_lo_exact(w[i])), s)),
                 h2_as_u32(__hmul2(u32_as_h2(int4_hi_exact(w[i])), s)),
                 h2_as_u32(__hmul2(u32_as_h2(int4_lo_exact(w[i] >> 8)), s)),
                 h2_as_u32(__hmul2(u32_as_h2(int4_hi_exact(w[i] >> 8)), s)));
      }
      fence_proxy_async_shared();
      mbar_arrive(&sh.v_ready);
      if (k + 1 < n) {
        fetch_scales(checked_page(p.s, page), first_token(k + 1) + tid);
        if (k + 2 < n) page = raw_page(p.s, b, first_token(k + 2) + tid, len);
      }
    }
    umma_fence_before();
    __syncthreads();
    umma_fence_after();
    const int dim = (tid & ~7) + ((tid & 1) << 2) + ((tid >> 1) & 3);
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
      if (c >= cols) break;
      const float sum = (sh.total[0][c] + sh.total[1][c]) + (sh.total[2][c] + sh.total[3][c]);
      const float lse = sum == 0.0f ? kMinusInf : sh.row[c].y + (sh.row[c].w + lg2(sum));
      float v = sum == 0.0f ? 0.0f : o[c] * (1.0f / 256.0f) / sum;
      if ((sh.spoilt[c] >> (dim / 32)) & 1u) v = __int_as_float(0x7fffffff);
      const int64_t row = row_at(c);
      if (whole) {
        if (tid < D)
          static_cast<uint16_t*>(p.out)[row * D + dim] =
              static_cast<uint16_t>(p.bf16 ? Bf16Elem::pack(v, v) : Fp16Elem::pack(v, v));
        if (tid == 0 && p.out_lse != nullptr) p.out_lse[row] = lse;
      } else {
        if (tid < D) p.few_o[(part + c) * D + dim] = v;
        if (tid == 0) p.few_lse[part + c] = lse;
      }
    }
  }
}

// Joins the parts of a row: `parts` of them, `stride` rows apart.  One warp.
template <int D>
IRIS_DEV void join_row(const AttendParams& p, const float* part_o, const float* part_lse, int parts, int64_t stride,
                       int64_t row, int lane) {
  float top = kMinusInf;
  for (int s = lane; s < parts; s += 32) top = fmaxf(top, __ldcg(part_lse + s * stride));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  const float zero = top == kMinusInf ? 0.0f : top;
  float acc[D / 32] = {}, total = 0.0f;
#pragma unroll 4
  for (int s = 0; s < parts; ++s) {
    const float part = __ldcg(part_lse + s * stride);
    if (part == kMinusInf) continue;  // it saw nothing
    const float w = ex2(part - zero);
    total += w;
    const float* o = part_o + s * stride * D + lane * (D / 32);
#pragma unroll
    for (int j = 0; j < D / 32; ++j) acc[j] = fmaf(w, __ldcg(o + j), acc[j]);
  }
  const float norm = total == 0.0f ? 0.0f : 1.0f / total;
  uint32_t* dst = reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(p.out) + row * D) + lane * (D / 64);
#pragma unroll
  for (int j = 0; j < D / 64; ++j) {
    const float a = acc[2 * j] * norm, b = acc[2 * j + 1] * norm;
    dst[j] = p.bf16 ? Bf16Elem::pack(a, b) : Fp16Elem::pack(a, b);
  }
  if (lane == 0 && p.out_lse != nullptr) p.out_lse[row] = total == 0.0f ? kMinusInf : zero + lg2(total);
}

// A block a (sequence with few rows, KV head), a warp a row.
template <int D>
__global__ void __launch_bounds__(128) varlen_few_join_kernel(const AttendParams p, int cols) {
  grid_dependency_wait();
  grid_dependents_launch();
  const int b = blockIdx.x / p.s.hkv, h = blockIdx.x % p.s.hkv;
  const Span sp = new_tokens(p.s, b);
  const int64_t rows = static_cast<int64_t>(sp.count) * p.s.group;
  if (rows > cols) return;
  const int64_t part = static_cast<int64_t>(blockIdx.x) * p.chunks * cols;
  for (int c = threadIdx.x >> 5; c < rows; c += 4)
    join_row<D>(p, p.few_o + (part + c) * D, p.few_lse + part + c, p.chunks, cols,
                static_cast<int64_t>(sp.start + c / p.s.group) * p.s.hq + h * p.s.group + c % p.s.group, threadIdx.x & 31);
}

}  // namespace iris
