// The attention weight that each cached token received, added up beside the
// cache: iris_b200_int4_paged_attention_mass.
//
// mass[page, head, slot] of a KV head is decay * its old value (0 from
// first_token on) plus the sum over the sequence's query rows and the KV head's
// query heads of 2^(logit - lse).  Products are turned around against the
// attention's: cached tokens are the rows (a thread a token), query rows the
// columns, so a token's sum stays in one thread and no order of additions
// depends on timing.  Stored nibbles go to the tensor cores as whole numbers,
// one accumulator a group of 32 dims, and a token's fp32 scales join them
// afterwards: nothing is rounded but the fp32 sums, whose losses are made good.
//
// A block is 128 threads that unpack a tile of 128 tokens into tensor memory
// (thread = token = lane) and then take its columns, 16 query rows a product; the
// packed rows of the next tile are on their way meanwhile (TMA).  Four blocks an SM
// (their keys and sums fill its tensor memory) overlap each other.
#include "varlen_common.cuh"

namespace iris {
namespace {

constexpr int kCols = 16;       // query rows of a product
// Query rows that stay in shared memory.  More are loaded again for every tile, 16 at a time, visible or not: 2100 us for
// all rows of two prompts of 4096 tokens (32 heads over 8 of 128), where the last 32 tokens' of 8 x 8191 take 90.
constexpr int kResident = 128;
constexpr int kSlots = kResident / kCols;

struct MassParams {
  VarlenBatch s;
  const uint16_t* query;
  const float* lse;  // [tokens, hq]
  const uint8_t* k_data;
  const uint8_t* k_scale;
  float* mass;       // [pages, hkv, 16]
  const int32_t* first_token;  // [batch] or NULL: 0
  int64_t q_stride;
  float decay;
  int32_t bf16;
  int32_t per;       // tiles of a block
  int32_t chunks;    // blocks of a (sequence, KV head)
  int32_t slots;     // column tiles in shared memory
};

template <int D>
struct MassCfg {
  static constexpr int kQuery = kCols * D * 2;
  static constexpr int kPacked = kTile * D / 2;
  static constexpr int kMeta = kCols * (8 + 8 + 16);  // a row: factor and lse (two rows a vector), place and slope, sight
  static constexpr int kSumColumn = D / 2;            // tensor memory: keys, then D / 32 groups x 16 columns of sums
  static constexpr int kColumns = D;
  static int smem(int slots) { return 1024 + slots * (kQuery + kMeta) + kPacked; }
};

struct MassShared {
  uint64_t here, done;
  uint32_t tmem;
  int32_t all_lo[kSlots], all_hi[kSlots];  // tokens that every row of a slot sees (without the prefix)
  int32_t any_lo[kSlots], any_hi[kSlots];  // between them lies all that any row sees
};

IRIS_DEV float min_nan(float a, float b) {  // NaN stays NaN
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// A slot's rows in shared memory.
struct MassRows {
  float4* f;     // [8] factors of two rows, minus their lse
  float2* more;  // [16] place, slope
  int4* sight;   // [16]
};

// Query rows r0 .. r0 + 16 into a slot: eight threads a row.
template <int D, bool kCap, bool kBias>
IRIS_DEV void load_columns(const MassParams& p, MassShared& sh, const Span& sp, int b, int len, int h, int r0, int rows,
                           uint32_t q_tile, const MassRows& to, int slot, int tid) {
  constexpr int kWords = D / 16;  // a thread's pairs
  const int row = tid >> 3, part = tid & 7, r = r0 + row;
  const bool valid = r < rows;
  const int i = valid ? r / p.s.group : 0, g = valid ? r % p.s.group : 0;
  const int64_t token = sp.start + i;
  const int head = h * p.s.group + g;
  uint32_t w[kWords] = {};
  if (valid) {
    const uint4* src = reinterpret_cast<const uint4*>(p.query + token * p.q_stride + static_cast<int64_t>(head) * D +
                                                      part * (D / 8));
#pragma unroll
    for (int c = 0; c < kWords / 4; ++c) {
      const uint4 v = src[c];
      w[4 * c] = v.x;
      w[4 * c + 1] = v.y;
      w[4 * c + 2] = v.z;
      w[4 * c + 3] = v.w;
    }
  }
  const float back = scale_row_part<kWords>(w, p.bf16 != 0, [](uint32_t m) {
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
    return max(m, __shfl_xor_sync(0xffffffffu, m, 4));
  });
#pragma unroll
  for (int c = 0; c < kWords / 4; ++c) {
    const uint4 v = order8(w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]);
    const int chunk = part * (D / 64) + c;
    sts128(q_tile + (chunk >> 3) * (kCols * 128) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4), v.x, v.y, v.z, v.w);
  }
  if (part == 0) {
    Sight see = {0, 0, 0, 0};
    float factor = 0.0f, lse = 0.0f, slope = 0.0f;
    int32_t pos = 0;
    if (valid) {
      pos = len - sp.count + i;
      lse = __ldg(p.lse + token * p.s.hq + head);
      factor = fminf(kCap ? p.s.scale * back / p.s.cap : p.s.scale * kLog2e * back, 1e38f);
      slope = kBias ? -__ldg(p.s.slopes + head) * kLog2e : 0.0f;
      if (lse != -__int_as_float(0x7f800000))  // (a row that saw nothing gives nothing)
        see = row_sight(pos, p.s.first_visible != nullptr ? __ldg(p.s.first_visible + token) : 0,
                        p.s.prefix_lens != nullptr ? __ldg(p.s.prefix_lens + b) : 0, p.s.window, len);
    }
    float* f = reinterpret_cast<float*>(to.f + row / 2);
    f[row & 1] = factor;
    f[2 + (row & 1)] = -lse;
    to.more[row] = make_float2(__int_as_float(pos), slope);
    to.sight[row] = make_int4(see.a0, see.a1, see.b0, see.b1);
    atomicMax(&sh.all_lo[slot], see.b0);
    atomicMin(&sh.all_hi[slot], see.b1);
    if (see.a1 > see.a0) {
      atomicMin(&sh.any_lo[slot], see.a0);
      atomicMax(&sh.any_hi[slot], see.a1);
    }
    if (see.b1 > see.b0) {
      atomicMin(&sh.any_lo[slot], see.b0);
      atomicMax(&sh.any_hi[slot], see.b1);
    }
  }
}
IRIS_DEV void clear_slots(MassShared& sh, int slots, int tid) {
  __syncthreads();  // what they held is read
  if (tid < slots) {
    sh.all_lo[tid] = 0;
    sh.all_hi[tid] = INT32_MAX;
    sh.any_lo[tid] = INT32_MAX;
    sh.any_hi[tid] = 0;
  }
  __syncthreads();
}
IRIS_DEV void slots_done() {
  fence_proxy_async_shared();
  __syncthreads();
}

template <int D, bool kCap, bool kBias>
__global__ void __launch_bounds__(128, 4) attention_mass_kernel(const __grid_constant__ CUtensorMap k_map, const MassParams p) {
  using C = MassCfg<D>;
  constexpr int kGroups = D / 32;
  extern __shared__ uint8_t smem_raw[];
  __shared__ MassShared sh;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int chunk = blockIdx.x % p.chunks, h = blockIdx.x / p.chunks % p.s.hkv, b = blockIdx.x / p.chunks / p.s.hkv;
  if (tid == 0) {
    mbar_init(&sh.here, 1);
    mbar_init(&sh.done, 1);
    fence_barrier_init();
  }
  grid_dependency_wait();
  grid_dependents_launch();
  if (blockIdx.x == 0 && warp == 0) check_offsets(p.s, lane);
  const Span sp = new_tokens(p.s, b);
  const int len = cached_tokens(p.s, __ldg(p.s.seq_lens + b), sp.count, tid == 0 && h == 0 && chunk == 0);
  const int tiles = (len + kTile - 1) / kTile;
  const int k0 = chunk * p.per, n = min(p.per, tiles - k0);
  if (n <= 0) return;
  __syncthreads();  // (the barriers are ready)

  uint8_t* base = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const uint32_t q_tiles = smem_u32(base);
  uint8_t* packed = base + p.slots * C::kQuery;
  const uint32_t raw = smem_u32(packed);
  float4* row_f = reinterpret_cast<float4*>(packed + C::kPacked);
  float2* row_more = reinterpret_cast<float2*>(row_f + p.slots * kCols / 2);
  int4* row_sight_ = reinterpret_cast<int4*>(row_more + p.slots * kCols);
  auto rows_of = [&](int slot) {
    return MassRows{row_f + slot * kCols / 2, row_more + slot * kCols, row_sight_ + slot * kCols};
  };

  auto first = [&](int k) { return (k0 + k) * kTile; };
  auto page_at = [&](int k) { return lane < 8 ? raw_page(p.s, b, first(k) + lane * kTokPage, len) : 0; };
  uint32_t sc2[kGroups / 2];  // scales of the tile that is next
  auto fetch = [&](int32_t page, int32_t j) {
    const uint8_t* x = p.k_scale + ((static_cast<int64_t>(page) * kTokPage + (j & (kTokPage - 1))) * p.s.hkv + h) * (D / 16);
    if constexpr (D == 128) {
      const uint2 v = j < len ? __ldg(reinterpret_cast<const uint2*>(x)) : make_uint2(0, 0);
      sc2[0] = v.x;
      sc2[1] = v.y;
    } else {
      sc2[0] = j < len ? __ldg(reinterpret_cast<const uint32_t*>(x)) : 0u;
    }
  };
  int32_t copy_page = 0;  // (warp 0) of the tile whose copies are next, not checked yet
  if (warp == 0) {
    load_packed<D>(packed, &k_map, checked_page(p.s, page_at(0)), first(0), len, h, &sh.here, lane);
    if (n > 1) copy_page = page_at(1);
  }
  // This thread's token's page.  An id outside the cache is read as page 0, whose weights are others': none is written.
  auto in_cache = [&](int32_t id) { return static_cast<uint32_t>(id) < static_cast<uint32_t>(p.s.num_pages); };
  int32_t page = raw_page(p.s, b, first(0) + tid, len);
  bool good = in_cache(page);
  page = checked_page(p.s, page);
  fetch(page, first(0) + tid);
  int32_t later = n > 1 ? raw_page(p.s, b, first(1) + tid, len) : 0;
  if (warp == 0) umma_alloc(&sh.tmem, C::kColumns);
  umma_fence_before();
  __syncthreads();
  umma_fence_after();
  const uint32_t tmem = sh.tmem, lanes = tmem + (static_cast<uint32_t>(warp * 32) << 16);
  const int rows = sp.count * p.s.group, col_tiles = (rows + kCols - 1) / kCols;
  const bool resident = col_tiles <= p.slots;
  if (resident) {
    clear_slots(sh, col_tiles, tid);
#pragma unroll 2
    for (int q = 0; q < col_tiles; ++q)
      load_columns<D, kCap, kBias>(p, sh, sp, b, len, h, q * kCols, rows, q_tiles + q * C::kQuery, rows_of(q), q, tid);
    slots_done();
  }
  const int32_t fresh = p.first_token != nullptr ? __ldg(p.first_token + b) : 0;
  const float cap2 = p.s.cap * kLog2e;
  uint32_t phase = 0;
  bool ok = true;
#pragma unroll 1
  for (int k = 0; ok && k < n; ++k) {
    const int32_t base_j = first(k), j = base_j + tid;
    float* slot_mass = p.mass + (static_cast<int64_t>(page) * p.s.hkv + h) * kTokPage + j % kTokPage;
    const bool writes = j < len && good;
    const float old = writes && j < fresh ? *slot_mass : 0.0f;
    float sc[kGroups];
    {
      bool odd = false;  // a scale that is not finite makes the token's logits NaN
#pragma unroll
      for (int c = 0; c < kGroups; ++c) {
        const uint32_t bits = (sc2[c / 2] >> (16 * (c & 1))) & 0xffffu;
        odd |= (bits & 0x7fffu) >= 0x7c00u;
        sc[c] = __half2float(__ushort_as_half(static_cast<unsigned short>(bits)));
      }
      if (odd) sc[0] = __int_as_float(0x7fffffff);
    }
    if (k + 1 < n) {
      good = in_cache(later);
      page = checked_page(p.s, later);
      fetch(page, first(k + 1) + tid);
      if (k + 2 < n) later = raw_page(p.s, b, first(k + 2) + tid, len);
    }
    ok = wait_all(&sh.here, k & 1, p.s.err);
#pragma unroll
    for (int c = 0; c < kGroups; ++c) {
      const uint4 w4 = lds128(raw + packed_at<D>(tid, c));
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
    if (!(ok = __syncthreads_and(ok))) break;
    // Sums of 16 rows' weights, and the sum of those with what its additions lost (Kahan's method): a whole prompt's rows are
    // thousands of weights, and in one running sum of fp32 the losses add up (2.6e-4 of 26 for 190 rows of 33 heads).
    float2 total = make_float2(0.0f, 0.0f), lost = make_float2(0.0f, 0.0f);
    bool loaded = k + 1 >= n;  // the next tile's copies are under way
#pragma unroll 1
    for (int q = 0; q < col_tiles; ++q) {
      const int slot = resident ? q : 0;
      if (!resident) {
        clear_slots(sh, 1, tid);
        load_columns<D, kCap, kBias>(p, sh, sp, b, len, h, q * kCols, rows, q_tiles, rows_of(0), 0, tid);
        slots_done();
      }
      if (sh.any_hi[slot] <= base_j || sh.any_lo[slot] >= base_j + kTile) continue;  // no row sees the tile
      if (warp == 0) {
        if (elect_one()) {
          umma_fence_after();
#pragma unroll
          for (int x = 0; x < D / 16; ++x) {  // the groups in turn, twice: a product does not wait for the one before it
            const int g = x % kGroups, s = 2 * g + x / kGroups;
            umma_ts(tmem + C::kSumColumn + g * kCols, tmem + 8 * s,
                    umma_desc(q_tiles + slot * C::kQuery + (s >> 2) * (kCols * 128) + (s & 3) * 32, 16, 1024),
                    umma_idesc(kTile, kCols, false, false), x >= kGroups);
          }
          umma_commit(smem_u32(&sh.done));
        }
        __syncwarp();
        if (!loaded) {
          load_packed<D>(packed, &k_map, checked_page(p.s, copy_page), first(k + 1), len, h, &sh.here, lane);
          if (k + 2 < n) copy_page = page_at(k + 2);
        }
      }
      loaded = true;
      ok = wait_all(&sh.done, phase, p.s.err);
      phase ^= 1;
      umma_fence_after();
      const bool full = sh.all_lo[slot] <= base_j && base_j + kTile <= sh.all_hi[slot];
      const MassRows at = rows_of(slot);
      const int cols = min(kCols, rows - q * kCols);
      float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
      for (int c0 = 0; c0 < kCols; c0 += 8) {
        if (c0 >= cols) break;
        uint32_t v[kGroups][8];
#pragma unroll
        for (int c = 0; c < kGroups; ++c) umma_ld8(lanes + C::kSumColumn + c * kCols + c0, v[c]);
        umma_wait_ld();
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          float2 s = make_float2(0.0f, 0.0f);
#pragma unroll
          for (int c = 0; c < kGroups; ++c) {
            asm volatile("" : "+r"(v[c][i]), "+r"(v[c][i + 1]));
            s = __ffma2_rn(make_float2(__uint_as_float(v[c][i]), __uint_as_float(v[c][i + 1])), make_float2(sc[c], sc[c]), s);
          }
          const float4 f = at.f[(c0 + i) / 2];
          float2 y;
          if (kCap || kBias) {
            y = __fmul2_rn(s, make_float2(f.x, f.y));
            if (kCap) y = make_float2(cap2 * tanh_f(y.x), cap2 * tanh_f(y.y));
            if (kBias) {
              const float2 a = at.more[c0 + i], d = at.more[c0 + i + 1];
              y.x = fmaf(a.y, fabsf(static_cast<float>(__float_as_int(a.x) - j)), y.x);
              y.y = fmaf(d.y, fabsf(static_cast<float>(__float_as_int(d.x) - j)), y.y);
            }
            y = __fadd2_rn(y, make_float2(f.z, f.w));
          } else {
            y = __ffma2_rn(s, make_float2(f.x, f.y), make_float2(f.z, f.w));
          }
          float2 e = make_float2(ex2(min_nan(y.x, 0.0f)), ex2(min_nan(y.y, 0.0f)));  // (a weight is at most 1)
          if (!full) {
            const int4 a = at.sight[c0 + i], d = at.sight[c0 + i + 1];
            if (!((j >= a.x && j < a.y) || (j >= a.z && j < a.w))) e.x = 0.0f;
            if (!((j >= d.x && j < d.y) || (j >= d.z && j < d.w))) e.y = 0.0f;
          }
          sum = __fadd2_rn(sum, e);
        }
      }
      {
        const float2 more = __fadd2_rn(sum, make_float2(-lost.x, -lost.y)), now = __fadd2_rn(total, more),
                     taken = __fadd2_rn(now, make_float2(-total.x, -total.y));
        lost = __fadd2_rn(taken, make_float2(-more.x, -more.y));
        total = now;
      }
      umma_fence_before();
      if (!(ok = __syncthreads_and(ok))) break;  // the sums are read: the next product may overwrite them
    }
    if (!loaded && warp == 0) {
      load_packed<D>(packed, &k_map, checked_page(p.s, copy_page), first(k + 1), len, h, &sh.here, lane);
      if (k + 2 < n) copy_page = page_at(k + 2);
    }
    if (ok && writes) *slot_mass = fmaf(old, p.decay, total.x + total.y);
  }
  if (!ok) {  // a wait gave up: copies that are under way land before the block ends
    for (uint32_t parity = 0; parity < 2; ++parity) mbar_wait_bounded(&sh.here, parity, p.s.err);
  }
  umma_fence_before();
  __syncthreads();
  umma_fence_after();
  if (warp == 0) umma_free(tmem, C::kColumns);
}

template <int D, bool kCap, bool kBias>
cudaError_t launch_mass(const MassParams& p, int64_t grid, cudaStream_t stream) {
  auto fn = attention_mass_kernel<D, kCap, kBias>;
  CUtensorMap k;
  if (!packed_map(&k, p.k_data, D, p.s.hkv, p.s.num_pages)) return cudaErrorInvalidValue;
  const int smem = MassCfg<D>::smem(p.slots);
  static_assert(kSlots == 8, "48 KB hold every slot: no attribute is needed");
  return launch_early(fn, dim3(static_cast<unsigned>(grid)), dim3(128), smem, stream, k, p);
}
template <int D>
cudaError_t launch_mass(const MassParams& p, int64_t grid, cudaStream_t stream) {
  const bool cap = p.s.cap > 0.0f, bias = p.s.slopes != nullptr;
  if (cap && bias) return launch_mass<D, true, true>(p, grid, stream);
  if (cap) return launch_mass<D, true, false>(p, grid, stream);
  if (bias) return launch_mass<D, false, true>(p, grid, stream);
  return launch_mass<D, false, false>(p, grid, stream);
}

}  // namespace
}  // namespace iris

using namespace iris;

extern "C" int iris_b200_int4_paged_attention_mass(
    const void* query, int64_t query_stride, const float* lse, const void* k_data, const void* k_scale,
    const int32_t* block_table, int64_t block_table_stride, const int32_t* seq_lens, const int32_t* cu_seqlens,
    const float* slopes, const int32_t* prefix_lens, const int32_t* first_visible, const int32_t* first_token, float* mass,
    int64_t tokens, int32_t batch, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, int64_t num_pages,
    int32_t page_size, int32_t max_pages_per_seq, int32_t window, float logit_cap, float softmax_scale, float decay,
    int32_t dtype, int32_t* error_word, void* stream) {
  if (tokens < 0 || batch < 0 || num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads != 0 || window < 0 ||
      !(logit_cap >= 0.0f && logit_cap <= 1e20f) || !(softmax_scale > 0.0f) || (dtype != IRIS_DTYPE_FP16 && dtype != IRIS_DTYPE_BF16))
    return IRIS_EINVAL;
  if (page_size != kTokPage || (head_dim != 64 && head_dim != 128)) return IRIS_EUNSUPPORTED;
  if (cu_seqlens == nullptr && tokens != batch) return IRIS_EINVAL;
  if (batch == 0) return tokens == 0 ? IRIS_OK : IRIS_EINVAL;
  if (num_pages <= 0 || max_pages_per_seq <= 0) return IRIS_EINVAL;
  if (k_data == nullptr || k_scale == nullptr || block_table == nullptr || seq_lens == nullptr || mass == nullptr ||
      (tokens > 0 && (query == nullptr || lse == nullptr)))
    return IRIS_EINVAL;
  const int32_t group = num_q_heads / num_kv_heads;
  if (tokens * group > INT32_MAX / 2 || num_pages > INT32_MAX || max_pages_per_seq > INT32_MAX / 2 / kTokPage)
    return IRIS_EUNSUPPORTED;
  if (!aligned_to(query, 16) || query_stride % 8 != 0 || !aligned_to(k_data, 16) || !aligned_to(k_scale, 8) ||
      !aligned_to(mass, 4))
    return IRIS_EALIGN;
  MassParams p = {};
  p.s.block_table = block_table;
  p.s.bt_stride = block_table_stride;
  p.s.seq_lens = seq_lens;
  p.s.cu = cu_seqlens;
  p.s.prefix_lens = prefix_lens;
  p.s.first_visible = first_visible;
  p.s.slopes = slopes;
  p.s.err = error_word;
  p.s.num_pages = num_pages;
  p.s.tokens = static_cast<int32_t>(tokens);
  p.s.batch = batch;
  p.s.hq = num_q_heads;
  p.s.hkv = num_kv_heads;
  p.s.group = group;
  p.s.max_pages = max_pages_per_seq;
  p.s.window = window < (1 << 30) ? window : 0;
  p.s.scale = softmax_scale;
  p.s.cap = logit_cap;
  p.query = static_cast<const uint16_t*>(query);
  p.lse = lse;
  p.k_data = static_cast<const uint8_t*>(k_data);
  p.k_scale = static_cast<const uint8_t*>(k_scale);
  p.mass = mass;
  p.first_token = first_token;
  p.q_stride = query_stride;
  p.decay = decay;
  p.bf16 = dtype == IRIS_DTYPE_BF16;
  const int64_t tiles = (static_cast<int64_t>(max_pages_per_seq) * kTokPage + kTile - 1) / kTile;
  const int64_t units = static_cast<int64_t>(batch) * num_kv_heads;
  // a block's start is about three tiles long, and as much again where it has many query rows to load
  const int64_t chunks = best_chunks(units, tiles, 148 * 4, cu_seqlens == nullptr && group <= kCols ? 3 : 6, tiles);
  p.per = static_cast<int32_t>((tiles + chunks - 1) / chunks);
  p.chunks = static_cast<int32_t>((tiles + p.per - 1) / p.per);
  const int64_t most = cu_seqlens == nullptr ? group : static_cast<int64_t>(tokens) * group;
  p.slots = most >= kResident ? kSlots : static_cast<int32_t>((most + kCols - 1) / kCols);
  if (p.slots < 1) p.slots = 1;
  const int64_t grid = units * p.chunks;
  if (grid > INT32_MAX) return IRIS_EUNSUPPORTED;
  clear_stale_cuda_error();
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = head_dim == 128 ? launch_mass<128>(p, grid, st) : launch_mass<64>(p, grid, st);
  if (e != cudaSuccess) return record_cuda_error(e, "attention_mass"), IRIS_ECUDA;
  return IRIS_OK;
}
