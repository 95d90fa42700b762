// Rotary positions with several axes + group-32 symmetric INT4 quantisation +
// paged append, for sm_100a; optionally the queries (and keys) rotated too.
//
// A token of an image or a video has a position on each of A axes (time,
// height, width, ...).  Frequency i of the rotary half turns by the token's
// position on axis a(i): with x1 = x[i], x2 = x[i + R/2] (R = rotary_dim),
//   y1 = x1 cos[p_a(i)][i] - x2 sin[p_a(i)][i]
//   y2 = x2 cos[p_a(i)][i] + x1 sin[p_a(i)][i]
// and dims >= R pass through.  The products of two 16-bit values are exact in
// fp32, so y carries one fp32 rounding; it is not rounded to 16 bits before
// it is quantised.  Per 32-dim group: scale = fp16(min(max(amax / 7, 2^-14),
// 65504)), q = clamp(rint(y / scale), -7, 7), divisions rounded once.  A group
// that holds an infinity or NaN stores that as its scale and zero nibbles, so
// that reading it back gives NaN.
//
// The work is a copy with arithmetic on the way: per token 2 Hkv D (and Hq D)
// 16-bit values in, 1.125 Hkv D bytes (and Hq D values) out.  One CTA takes
// one token, a thread one 8-dim vector of the row: the rotary rows of the
// token are read, and their axes blended, once per thread and used for all
// the rows (keys, values, queries) that the thread passes over.  A group is
// four adjacent lanes; its absmax takes two shuffles.
#include "append_common.cuh"
#include "elem.cuh"

namespace iris {
namespace {

constexpr int kMaxAxes = IRIS_MROPE_MAX_AXES;
constexpr int kMaxFreqs = 256;  // head_dim <= 512
constexpr int kThreads = 256;

struct MropeParams {
  const void* key;
  const void* value;
  const void* query;
  void* query_out;
  void* key_out;
  int64_t key_stride, value_stride, query_stride;  // elements between tokens
  const int32_t* positions;
  int64_t positions_stride;  // between axes
  const int32_t* slots;
  const void* cos_cache;
  const void* sin_cache;
  uint8_t* k_data;
  uint8_t* v_data;
  __half* k_scale;
  __half* v_scale;
  int64_t num_tokens;
  int64_t max_position;
  int64_t num_slots;
  int32_t axes;
  int32_t kv_heads, q_heads;
  int32_t vecs;         // 8-dim vectors per row
  int32_t rotary_vecs;  // of them rotated
  int32_t* err;
  uint32_t axis_map[kMaxFreqs / 16];  // two bits per frequency
};

// Error bits of one token's slot and positions.
IRIS_DEV int32_t token_bits(const MropeParams& p, int32_t slot, int64_t tok) {
  int32_t bits = static_cast<int64_t>(slot) >= p.num_slots ? IRIS_ERR_SLOT_RANGE : 0;
  for (int a = 0; a < p.axes; ++a) {
    const int32_t pos = __ldg(p.positions + a * p.positions_stride + tok);
    if (pos < 0) bits |= IRIS_ERR_POS_NEGATIVE;
    else if (static_cast<int64_t>(pos) >= p.max_position) bits |= IRIS_ERR_POS_RANGE;
  }
  return bits;
}

// Validation of a large batch before the append: ranges, and one bit per slot
// for duplicates.  The append's launch overlaps it.
__global__ void __launch_bounds__(kThreads) mrope_check_kernel(const MropeParams p, uint32_t* __restrict__ bitmap) {
  grid_dependents_launch();
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (i >= p.num_tokens) return;
  const int32_t slot = __ldg(p.slots + i);
  if (slot < 0) return;
  int32_t bits = token_bits(p, slot, i);
  if (!(bits & IRIS_ERR_SLOT_RANGE)) {
    const uint32_t bit = 1u << (slot & 31);
    if (atomicOr(bitmap + (slot >> 5), bit) & bit) bits |= IRIS_ERR_DUP_SLOT;
  }
  if (bits) set_error(p.err, bits);
}

// The same for at most kInlineCheckTokens tokens, by every CTA of the append.
IRIS_DEV bool check_small_batch(const MropeParams& p) {
  __shared__ __align__(16) int32_t s_slot[kInlineCheckTokens];
  const int T = static_cast<int>(p.num_tokens), T4 = (T + 3) & ~3;
  int32_t bits = 0;
  for (int i = threadIdx.x; i < T4; i += blockDim.x) {
    const int32_t s = i < T ? __ldg(p.slots + i) : -1;
    if (s >= 0) bits |= token_bits(p, s, i);
    s_slot[i] = s;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < T; i += blockDim.x) {
    const int32_t s = s_slot[i];
    if (s < 0) continue;
    int hits = 0;
    for (int j = 0; j < T4; j += 4) {
      const int4 v = *reinterpret_cast<const int4*>(s_slot + j);
      hits += (v.x == s) + (v.y == s) + (v.z == s) + (v.w == s);
    }
    if (hits > 1) bits |= IRIS_ERR_DUP_SLOT;
  }
  if (blockIdx.x == 0 && blockIdx.y == 0 && bits) set_error(p.err, bits);
  return __syncthreads_or(bits != 0);
}

// cos / sin of eight frequencies, each from the row of its own axis.  `code`
// holds the eight axes, two bits each; one load if they are all the same.
template <typename E>
IRIS_DEV void blend_rows(const MropeParams& p, int64_t tok, int fv, float (&c)[8], float (&s)[8]) {
  const uint32_t code = (p.axis_map[fv >> 1] >> (16 * (fv & 1))) & 0xffffu;
  const int64_t width = static_cast<int64_t>(p.rotary_vecs) * 4;  // R / 2
  uint32_t cw[4] = {0, 0, 0, 0}, sw[4] = {0, 0, 0, 0};
  for (int a = 0; a < p.axes; ++a) {
    const uint32_t same = code ^ (0x5555u * static_cast<uint32_t>(a));  // 00 where the axis is a
    const uint32_t other = (same | (same >> 1)) & 0x5555u;              // bit 2j set where it is not
    if (other == 0x5555u) continue;
    const int64_t row = __ldg(p.positions + a * p.positions_stride + tok);
    const char* cb = static_cast<const char*>(p.cos_cache) + (row * width + 8 * fv) * 2;
    const char* sb = static_cast<const char*>(p.sin_cache) + (row * width + 8 * fv) * 2;
    const uint4 cv = ldg_nc_v4(cb), sv = ldg_nc_v4(sb);
    const uint32_t ci[4] = {cv.x, cv.y, cv.z, cv.w}, si[4] = {sv.x, sv.y, sv.z, sv.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t m = ((other >> (4 * j)) & 1u ? 0u : 0x0000ffffu) | ((other >> (4 * j + 2)) & 1u ? 0u : 0xffff0000u);
      cw[j] |= ci[j] & m;
      sw[j] |= si[j] & m;
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 a = E::unpack(cw[j]), b = E::unpack(sw[j]);
    c[2 * j] = a.x;
    c[2 * j + 1] = a.y;
    s[2 * j] = b.x;
    s[2 * j + 1] = b.y;
  }
}

template <typename E>
IRIS_DEV void unpack8(const uint4& w, float (&x)[8]) {
  const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 f = E::unpack(v[j]);
    x[2 * j] = f.x;
    x[2 * j + 1] = f.y;
  }
}

// Eight fp32 values of a group of four lanes -> fp16 group scale and this
// lane's packed word.  y / scale is rounded as the IEEE division rounds it: r
// is the correctly rounded reciprocal, t = x r is off by at most 1.5 ulp, and
// one residual step (Markstein 1990) leaves an error of 2^-23 ulp before the
// last rounding, while a quotient of a 24-bit by an 11-bit number that is no
// rounding midpoint stays 2^-12 ulp away from one.
IRIS_DEV uint32_t quant8(const float (&x)[8], uint32_t quad, __half& scale16) {
  float m = 0.0f;
  bool nan = false;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    m = fmaxf(m, fabsf(x[j]));  // skips NaN
    nan |= x[j] != x[j];
  }
  if (nan) m = __int_as_float(0x7fffffff);  // as an integer above every magnitude
  // magnitudes order as their bit patterns, NaN on top
  uint32_t b = __float_as_uint(m);
  b = max(b, __shfl_xor_sync(quad, b, 1));
  b = max(b, __shfl_xor_sync(quad, b, 2));
  m = __uint_as_float(b);
  if (!(m <= 3.402823466e38f)) {  // an infinity or NaN in the group
    scale16 = __float2half_rn(m);
    return 0u;
  }
  const float s = fminf(fmaxf(__fdiv_rn(m, 7.0f), 6.103515625e-05f), 65504.0f);
  scale16 = __float2half_rn(s);
  const float sc = __half2float(scale16), r = __frcp_rn(sc);
  uint32_t z[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float t = __fmul_rn(x[j], r);
    const float q = fmaf(fmaf(-t, sc, x[j]), r, t);
    // 2^23 + 16: rounds half to even, low four bits are the nibble
    z[j] = __float_as_uint(__fadd_rn(fminf(fmaxf(q, -7.0f), 7.0f), 8388624.0f));
  }
  const uint32_t ev = __byte_perm(__byte_perm(z[0], z[2], 0x0040), __byte_perm(z[4], z[6], 0x0040), 0x5410);
  const uint32_t od = __byte_perm(__byte_perm(z[1], z[3], 0x0040), __byte_perm(z[5], z[7], 0x0040), 0x5410);
  return (ev & 0x0F0F0F0Fu) | ((od << 4) & 0xF0F0F0F0u);
}

template <typename E>
IRIS_DEV uint4 pack8(const float (&x)[8]) {
  return make_uint4(E::pack(x[0], x[1]), E::pack(x[2], x[3]), E::pack(x[4], x[5]), E::pack(x[6], x[7]));
}

// gridDim = (tokens, row splits).  kSmall: at most kInlineCheckTokens tokens,
// validated here; otherwise the check kernel before this launch did it.
template <typename E, bool kSmall>
__global__ void __launch_bounds__(kThreads) mrope_append_kernel(const MropeParams p) {
  const int v = threadIdx.x % p.vecs;  // vector within the row
  const int per_pass = blockDim.x / p.vecs;
  const int64_t tok = blockIdx.x;
  const int rows = 2 * p.kv_heads + p.q_heads;
  const int32_t slot = __ldg(p.slots + tok);
  bool rejected = false;
  if constexpr (kSmall) rejected = check_small_batch(p);
  // A token with a bad slot or position: never touch memory outside the cache
  // or the tables.  (The check has recorded its bits.)
  const bool live = slot >= 0 && token_bits(p, slot, tok) == 0;
  const int half = p.rotary_vecs / 2;  // vectors of the rotary half
  const bool turns = live && v < p.rotary_vecs;
  const bool low = v < half;
  const int fv = low ? v : v - half;
  float c[8], s[8];
  if (turns) blend_rows<E>(p, tok, fv, c, s);
  const uint32_t quad = 0xFu << (threadIdx.x & 28);
  if constexpr (!kSmall) grid_dependency_wait();
  if (rejected || (p.err != nullptr && (*reinterpret_cast<volatile int32_t*>(p.err) & kRejectBits) != 0)) return;
  const int64_t D = 8ll * p.vecs;
  for (int r = threadIdx.x / p.vecs + per_pass * blockIdx.y; r < rows; r += per_pass * gridDim.y) {
    const bool is_v = r >= p.kv_heads && r < 2 * p.kv_heads, is_q = r >= 2 * p.kv_heads;
    const int h = is_q ? r - 2 * p.kv_heads : is_v ? r - p.kv_heads : r;
    const char* base = static_cast<const char*>(is_q ? p.query : is_v ? p.value : p.key);
    const int64_t stride = is_q ? p.query_stride : is_v ? p.value_stride : p.key_stride;
    char* out = static_cast<char*>(is_q ? p.query_out : is_v ? nullptr : p.key_out);
    if (out != nullptr) out += ((tok * (is_q ? p.q_heads : p.kv_heads) + h) * D + 8 * v) * 2;
    if (!live) {  // padding: its rotated rows are zeros
      if (out != nullptr) *reinterpret_cast<uint4*>(out) = make_uint4(0, 0, 0, 0);
      continue;
    }
    const char* row = base + (tok * stride + h * D) * 2;
    float x[8];
    unpack8<E>(ldg_nc_v4(row + 16 * v), x);
    if (!is_v && turns) {
      float o[8];
      unpack8<E>(ldg_nc_v4(row + 16 * (low ? v + half : v - half)), o);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float t = __fmul_rn(o[j], s[j]), u = __fmul_rn(x[j], c[j]);  // both exact
        x[j] = low ? __fsub_rn(u, t) : __fadd_rn(u, t);
      }
    }
    if (out != nullptr) *reinterpret_cast<uint4*>(out) = pack8<E>(x);
    if (!is_q) {
      __half scale;
      const uint32_t word = quant8(x, quad, scale);
      const int64_t cache_row = static_cast<int64_t>(slot) * p.kv_heads + h;
      *reinterpret_cast<uint32_t*>((is_v ? p.v_data : p.k_data) + cache_row * (D / 2) + 4 * v) = word;
      if ((v & 3) == 0) (is_v ? p.v_scale : p.k_scale)[cache_row * (D / 32) + (v >> 2)] = scale;
    }
  }
}

template <typename E>
cudaError_t launch_mrope(const MropeParams& p, uint32_t* bitmap, size_t bitmap_bytes, cudaStream_t stream) {
  const int threads = kThreads / p.vecs * p.vecs;
  const int rows = 2 * p.kv_heads + p.q_heads, per_pass = threads / p.vecs;
  const int passes = (rows + per_pass - 1) / per_pass;
  cudaLaunchConfig_t cfg = {};
  cfg.stream = stream;
  cfg.blockDim = dim3(threads);
  if (p.num_tokens <= kInlineCheckTokens) {
    cfg.gridDim = dim3(static_cast<unsigned>(p.num_tokens), static_cast<unsigned>(passes));
    return cudaLaunchKernelEx(&cfg, mrope_append_kernel<E, true>, p);
  }
  cudaError_t e = bitmap_bytes > 0 ? cudaMemsetAsync(bitmap, 0, bitmap_bytes, stream) : cudaSuccess;
  if (e != cudaSuccess) return e;
  mrope_check_kernel<<<static_cast<unsigned>((p.num_tokens + kThreads - 1) / kThreads), kThreads, 0, stream>>>(p, bitmap);
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute attr[1];  // starts while the check kernel finishes
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cfg.gridDim = dim3(static_cast<unsigned>(p.num_tokens), 1);
  return cudaLaunchKernelEx(&cfg, mrope_append_kernel<E, false>, p);
}

}  // namespace
}  // namespace iris

using namespace iris;

extern "C" int iris_b200_mrope_int4_paged_append(
    const void* key, int64_t key_stride, const void* value, int64_t value_stride, const void* query,
    int64_t query_stride, const int32_t* positions, int64_t positions_stride, const int32_t* sections,
    int32_t num_axes, int32_t interleaved, const int32_t* slot_mapping, const void* cos_cache, const void* sin_cache,
    void* k_data, void* v_data, void* k_scale, void* v_scale, void* query_out, void* key_out, int64_t num_tokens,
    int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, int32_t rotary_dim, int64_t max_position,
    int64_t num_pages, int32_t page_size, int32_t dtype, void* workspace, size_t workspace_bytes, int32_t* error_word,
    void* stream) {
  if (num_tokens < 0 || num_kv_heads <= 0 || num_q_heads < 0 || page_size <= 0 || num_pages < 0 || max_position < 0)
    return IRIS_EINVAL;
  if (dtype != IRIS_DTYPE_FP16 && dtype != IRIS_DTYPE_BF16) return IRIS_EINVAL;
  if (sections == nullptr || num_axes < 1 || num_axes > kMaxAxes) return IRIS_EINVAL;
  if (head_dim <= 0 || head_dim % 64 != 0 || head_dim > 512) return IRIS_EUNSUPPORTED;
  if (rotary_dim <= 0 || rotary_dim > head_dim || rotary_dim % 16 != 0) return IRIS_EUNSUPPORTED;
  MropeParams p = {};
  int32_t left[kMaxAxes], sum = 0;
  for (int a = 0; a < num_axes; ++a) {
    if (sections[a] < 0 || sections[a] > rotary_dim / 2) return IRIS_EINVAL;
    left[a] = sections[a];
    sum += sections[a];
  }
  if (sum != rotary_dim / 2) return IRIS_EINVAL;
  for (int i = 0, a = 0; i < sum; ++i) {
    while (left[a] == 0) a = (a + 1) % num_axes;
    p.axis_map[i >> 4] |= static_cast<uint32_t>(a) << (2 * (i & 15));
    --left[a];
    if (interleaved) a = (a + 1) % num_axes;
  }
  if (num_tokens == 0) return IRIS_OK;
  if (num_tokens >= (1ll << 31) || num_pages * page_size >= (1ll << 31)) return IRIS_EUNSUPPORTED;
  if ((num_q_heads > 0) != (query != nullptr) || (query != nullptr) != (query_out != nullptr)) return IRIS_EINVAL;
  const void* ptrs[] = {key, value, positions, slot_mapping, cos_cache, sin_cache, k_data, v_data, k_scale, v_scale};
  for (const void* q : ptrs)
    if (q == nullptr) return IRIS_EINVAL;
  const void* wide[] = {key, value, query, cos_cache, sin_cache, query_out, key_out};
  for (const void* q : wide)
    if (!aligned_to(q, 16)) return IRIS_EALIGN;
  if (key_stride % 8 != 0 || value_stride % 8 != 0 || query_stride % 8 != 0) return IRIS_EALIGN;
  if (!aligned_to(k_data, 4) || !aligned_to(v_data, 4) || !aligned_to(k_scale, 2) || !aligned_to(v_scale, 2))
    return IRIS_EALIGN;
  const size_t need = num_tokens <= kInlineCheckTokens ? 0 : iris_b200_append_check_workspace_bytes(num_pages, page_size);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) return IRIS_EWORKSPACE;
  if (need > 0 && !aligned_to(workspace, 4)) return IRIS_EALIGN;
  p.key = key;
  p.value = value;
  p.query = query;
  p.query_out = query_out;
  p.key_out = key_out;
  p.key_stride = key_stride;
  p.value_stride = value_stride;
  p.query_stride = query_stride;
  p.positions = positions;
  p.positions_stride = positions_stride;
  p.slots = slot_mapping;
  p.cos_cache = cos_cache;
  p.sin_cache = sin_cache;
  p.k_data = static_cast<uint8_t*>(k_data);
  p.v_data = static_cast<uint8_t*>(v_data);
  p.k_scale = static_cast<__half*>(k_scale);
  p.v_scale = static_cast<__half*>(v_scale);
  p.num_tokens = num_tokens;
  p.max_position = max_position;
  p.num_slots = num_pages * page_size;
  p.axes = num_axes;
  p.kv_heads = num_kv_heads;
  p.q_heads = num_q_heads;
  p.vecs = head_dim / 8;
  p.rotary_vecs = rotary_dim / 8;
  p.err = error_word;
  clear_stale_cuda_error();
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = dtype == IRIS_DTYPE_FP16
                            ? launch_mrope<Fp16Elem>(p, static_cast<uint32_t*>(workspace), need, s)
                            : launch_mrope<Bf16Elem>(p, static_cast<uint32_t*>(workspace), need, s);
  if (e != cudaSuccess) {
    record_cuda_error(e, "mrope_append_kernel launch");
    return IRIS_ECUDA;
  }
  return IRIS_OK;
}
