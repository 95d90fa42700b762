// Reading the INT4 paged cache back: the keys and values of every sequence's
// tokens, dequantised (value = nibble * group scale, one rounding to the
// output type), as dense rows one sequence after another.
//
// A copy: per token and head 1.125 D bytes in and 4 D bytes out.  The heads of
// a token are contiguous in the cache and in the output, so a token is one
// row of R = Hkv D dims.  A CTA takes a tile of consecutive output rows; one
// warp finds the first row's sequence and, a lane a row, the rows' places in
// the cache; then all pass over the tile's 8-dim vectors: four packed bytes
// in, one 16-byte store out (or eight and 32), consecutive lanes on consecutive
// vectors.  8 x 8192 tokens of 8 heads of 128 dims: 53.2 us, 5.8 TB/s (90 % of a
// plain copy), DRAM bound; 517 tokens of 8 heads of 64 dims: 2.4 us, launch and dependent loads.
#include <type_traits>

#include "elem.cuh"

namespace iris {
namespace {

constexpr int kThreads = 256;
constexpr int kTile = 16;  // most output rows per CTA

struct GatherParams {
  const uint8_t* k_data;
  const uint8_t* v_data;
  const __half* k_scale;
  const __half* v_scale;
  const int32_t* block_table;
  int64_t table_stride;
  const int32_t* cu_seqlens;
  const int32_t* first_token;  // NULL: every sequence from its token 0
  void* key;
  void* value;
  int64_t num_tokens;
  int64_t num_pages;
  int32_t batch;
  int32_t max_pages;
  int32_t vecs;  // 8-dim vectors per token: Hkv D / 8
  int32_t page_size;
  int32_t tile;  // output rows per CTA
  int32_t* err;
};

// The last sequence whose offset is <= n.  The whole warp calls it: 32 offsets
// are tried at a time, so that a thousand sequences take two loads in a row.
IRIS_DEV int sequence_of(const GatherParams& p, int64_t n) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = p.batch;
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) >> 5, at = lo + lane * step;
    const bool below = at < hi && static_cast<int64_t>(__ldg(p.cu_seqlens + at)) <= n;
    const unsigned mask = __ballot_sync(0xffffffffu, below);
    const int k = mask != 0 ? 31 - __clz(mask) : 0;
    lo += k * step;
    hi = min(hi, lo + step);
  }
  return lo;
}

// Cache row (page * page_size + offset) of output row n, -1 if it has none;
// `seq`: the sequence of a row at or before it.
IRIS_DEV int64_t row_of(const GatherParams& p, int64_t n, int seq) {
  const int64_t total = __ldg(p.cu_seqlens + p.batch);
  if (n >= total) return -1;  // past the last sequence: zeros
  int64_t start = __ldg(p.cu_seqlens + seq), end = __ldg(p.cu_seqlens + seq + 1);
  while (n >= end && seq + 1 < p.batch) {
    start = end;
    end = __ldg(p.cu_seqlens + ++seq + 1);
  }
  const int64_t from = p.first_token != nullptr ? __ldg(p.first_token + seq) : 0;
  if (start < 0 || n < start || n >= end || end > total || from < 0) {
    set_error(p.err, IRIS_ERR_OFFSETS);
    return -1;
  }
  const int64_t at = from + n - start, col = at / p.page_size;
  if (col >= p.max_pages) {
    set_error(p.err, IRIS_ERR_BLOCK_TABLE);
    return -1;
  }
  const int64_t page = __ldg(p.block_table + seq * p.table_stride + col);
  if (page < 0 || page >= p.num_pages) {
    set_error(p.err, IRIS_ERR_PAGE_ID);
    return -1;
  }
  return page * p.page_size + at % p.page_size;
}

// Eight nibbles times their scale, rounded once to the output type.  A pair's
// nibbles become 1024 + u and 1024 + 16 u in fp16 (u = nibble + 8, by setting
// the exponent over them), one fused step makes them exact whole numbers.
// FP16: their product with the scale is that type's own; BF16: it is exact in
// fp32 (14 bits) and rounded from there.
template <typename E>
IRIS_DEV uint4 dequant8(uint32_t w, __half scale) {
  w ^= 0x88888888u;
  const uint32_t lo = __byte_perm(w, 0u, 0x1010), hi = __byte_perm(w, 0u, 0x3232);
  const uint32_t u[4] = {lo, lo >> 8, hi, hi >> 8};
  uint32_t x[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 q = __hfma2(u32_as_h2((u[i] & 0x00F0000Fu) | 0x64006400u), u32_as_h2(0x2C003C00u) /* 1/16, 1 */,
                              u32_as_h2(0xD480E408u) /* -72, -1032 */);
    if constexpr (E::kFp16) {
      x[i] = h2_as_u32(__hmul2(q, __half2half2(scale)));
    } else {
      const float2 f = __half22float2(q);
      const float s = __half2float(scale);
      x[i] = E::pack(__fmul_rn(f.x, s), __fmul_rn(f.y, s));
    }
  }
  return make_uint4(x[0], x[1], x[2], x[3]);
}

// 32 bytes, 32-byte aligned.
IRIS_DEV void store32(void* p, const uint4& a, const uint4& b) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(a.x), "r"(a.y), "r"(a.z),
               "r"(a.w), "r"(b.x), "r"(b.y), "r"(b.z), "r"(b.w)
               : "memory");
}

// kWide: 16 dims a thread and one 32-byte store, where everything is aligned to
// that: 65536 tokens of 8 heads of 128 dims 58.2 -> 53.2 us.  (A second vector
// of each tensor on the way takes 52.7, but 8192 tokens then 2 us more.)
template <typename E, bool kWide>
__global__ void __launch_bounds__(kThreads) gather_kernel(const GatherParams p) {
  __shared__ int64_t s_row[kTile];
  grid_dependency_wait();
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * p.tile;
  const int rows = static_cast<int>(p.num_tokens - n0 < p.tile ? p.num_tokens - n0 : p.tile);
  if (threadIdx.x < 32) {
    const int seq = sequence_of(p, n0);
    if (threadIdx.x < rows) s_row[threadIdx.x] = row_of(p, n0 + threadIdx.x, seq);
  } else if (blockIdx.x == 0) {  // the other warps of one CTA meanwhile: the offsets rise from 0
    for (int i = static_cast<int>(threadIdx.x) - 32; i < p.batch; i += kThreads - 32) {
      const int from = __ldg(p.cu_seqlens + i), to = __ldg(p.cu_seqlens + i + 1);
      if (to < from || (i == 0 && from != 0)) set_error(p.err, IRIS_ERR_OFFSETS);
    }
  }
  constexpr int kVecs = kWide ? 2 : 1;
  const int units = p.vecs / kVecs;
  const int down = kThreads / units, along = kThreads - down * units;  // from a thread's unit to its next one
  int r = threadIdx.x / units, v = threadIdx.x - r * units;
  __syncthreads();
  using Word = std::conditional_t<kWide, uint2, uint32_t>;
  while (r < rows) {
    Word kw = {}, vw = {};
    __half ks = __ushort_as_half(0), vs = ks;
    const int64_t src = s_row[r], dst = (n0 + r) * units + v;
    if (src >= 0) {
      const int64_t at = src * units + v, scale = at * kVecs >> 2;
      kw = __ldg(reinterpret_cast<const Word*>(p.k_data) + at);
      vw = __ldg(reinterpret_cast<const Word*>(p.v_data) + at);
      ks = __ldg(p.k_scale + scale);
      vs = __ldg(p.v_scale + scale);
    }
    if constexpr (kWide) {
      store32(static_cast<char*>(p.key) + 32 * dst, dequant8<E>(kw.x, ks), dequant8<E>(kw.y, ks));
      store32(static_cast<char*>(p.value) + 32 * dst, dequant8<E>(vw.x, vs), dequant8<E>(vw.y, vs));
    } else {
      static_cast<uint4*>(p.key)[dst] = dequant8<E>(kw, ks);
      static_cast<uint4*>(p.value)[dst] = dequant8<E>(vw, vs);
    }
    r += down;
    v += along;
    if (v >= units) {
      v -= units;
      ++r;
    }
  }
}

}  // namespace
}  // namespace iris

using namespace iris;

extern "C" int iris_b200_int4_paged_gather(const void* k_data, const void* v_data, const void* k_scale,
                                           const void* v_scale, const int32_t* block_table, int64_t block_table_stride,
                                           const int32_t* cu_seqlens, const int32_t* first_token, void* key,
                                           void* value, int64_t num_tokens, int32_t batch, int32_t num_kv_heads,
                                           int32_t head_dim, int64_t num_pages, int32_t page_size,
                                           int32_t max_pages_per_seq, int32_t dtype, int32_t* error_word,
                                           void* stream) {
  if (num_tokens < 0 || batch < 0 || num_kv_heads <= 0 || page_size <= 0 || num_pages < 0 || max_pages_per_seq < 0)
    return IRIS_EINVAL;
  if (dtype != IRIS_DTYPE_FP16 && dtype != IRIS_DTYPE_BF16) return IRIS_EINVAL;
  if (head_dim <= 0 || head_dim % 32 != 0 || head_dim > 512) return IRIS_EUNSUPPORTED;
  if (num_tokens == 0) return IRIS_OK;
  if (batch == 0) return IRIS_EINVAL;
  if (static_cast<int64_t>(num_kv_heads) * head_dim > (1 << 24)) return IRIS_EUNSUPPORTED;
  if (num_tokens > (1ll << 30)) return IRIS_EUNSUPPORTED;
  const void* ptrs[] = {k_data, v_data, k_scale, v_scale, block_table, cu_seqlens, key, value};
  for (const void* q : ptrs)
    if (q == nullptr) return IRIS_EINVAL;
  if (!aligned_to(key, 16) || !aligned_to(value, 16) || !aligned_to(k_data, 4) || !aligned_to(v_data, 4) ||
      !aligned_to(k_scale, 2) || !aligned_to(v_scale, 2))
    return IRIS_EALIGN;
  GatherParams p = {};
  p.k_data = static_cast<const uint8_t*>(k_data);
  p.v_data = static_cast<const uint8_t*>(v_data);
  p.k_scale = static_cast<const __half*>(k_scale);
  p.v_scale = static_cast<const __half*>(v_scale);
  p.block_table = block_table;
  p.table_stride = block_table_stride;
  p.cu_seqlens = cu_seqlens;
  p.first_token = first_token;
  p.key = key;
  p.value = value;
  p.num_tokens = num_tokens;
  p.num_pages = num_pages;
  p.batch = batch;
  p.max_pages = max_pages_per_seq;
  p.vecs = num_kv_heads * (head_dim / 8);
  p.page_size = page_size;
  p.err = error_word;
  // Rows per CTA: one vector a thread at least; then more, as long as 1024 CTAs
  // are left to fill the machine.  With 1, 2, 4, 8 and 16 rows of 1024 dims an
  // append of 64 tokens and its read back take 7.2, 7.4, 8.0, 9.2 and 11.5 us, of
  // 8192 tokens 65.4, 59.7, 57.7, 56.5 and 57.8; reading 65536 tokens takes 114,
  // 80, 63, 58.6 and 58.1.
  p.tile = 1;
  while (p.tile < kTile && (p.tile * p.vecs < kThreads ||
                            (2 * p.tile * p.vecs <= 8 * kThreads && num_tokens >= 1024 * 2ll * p.tile)))
    p.tile *= 2;
  clear_stale_cuda_error();
  const unsigned blocks = static_cast<unsigned>((num_tokens + p.tile - 1) / p.tile);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool wide = aligned_to(key, 32) && aligned_to(value, 32) && aligned_to(k_data, 8) && aligned_to(v_data, 8);
  const auto fn = dtype == IRIS_DTYPE_FP16 ? (wide ? gather_kernel<Fp16Elem, true> : gather_kernel<Fp16Elem, false>)
                                           : (wide ? gather_kernel<Bf16Elem, true> : gather_kernel<Bf16Elem, false>);
  const cudaError_t e = launch_early(fn, blocks, kThreads, 0, s, p);
  if (e != cudaSuccess) {
    record_cuda_error(e, "gather_kernel launch");
    return IRIS_ECUDA;
  }
  return IRIS_OK;
}
