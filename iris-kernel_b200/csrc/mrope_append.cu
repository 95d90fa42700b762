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
// 16-bit values in, 1.125 Hkv D bytes (and Hq D values) out.  A token takes
// row_lanes x D / 8 threads, a thread one 8-dim vector of every row_lanes-th
// head (in large batches of whole turning groups two vectors, the ones that
// turn together, by half as many threads): the token's rotary rows are read,
// and their axes blended, once per thread and used for all its keys and
// queries.  A group is four adjacent lanes; its absmax takes two shuffles.
// Arithmetic goes two values at a time.
// 8192 tokens of 32 + 2 x 8 heads of 128 dims, three axes dealt out in turn,
// rotated keys wanted: 55 us with the check and the read back of the cache,
// bound by the latency of its loads and by issue; 64 tokens of them 7.4 us with
// the read back, chains of dependent loads.
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
  int32_t row_lanes;    // threads of a token that share a vector
  int32_t vecs;         // 8-dim vectors per row
  int32_t rotary_vecs;  // of them rotated
  int32_t* err;
  uint32_t axis_map[kMaxFreqs / 16];  // two bits per frequency
};

// Error bits of one token's slot and positions; a token without a slot has
// none.  (All its positions are asked for at once, whatever the slot is.)
IRIS_DEV int32_t token_bits(const MropeParams& p, int32_t slot, int64_t tok) {
  int32_t pos[kMaxAxes];
#pragma unroll
  for (int a = 0; a < kMaxAxes; ++a) pos[a] = a < p.axes ? __ldg(p.positions + a * p.positions_stride + tok) : 0;
  int32_t bits = static_cast<int64_t>(slot) >= p.num_slots ? IRIS_ERR_SLOT_RANGE : 0;
#pragma unroll
  for (int a = 0; a < kMaxAxes; ++a) {
    if (a < p.axes) {
      if (pos[a] < 0) bits |= IRIS_ERR_POS_NEGATIVE;
      else if (static_cast<int64_t>(pos[a]) >= p.max_position) bits |= IRIS_ERR_POS_RANGE;
    }
  }
  return slot >= 0 ? bits : 0;
}

// Validation of a large batch before the append: ranges, and one bit per slot
// for duplicates.  The append's launch overlaps it.
__global__ void __launch_bounds__(kThreads) mrope_check_kernel(const MropeParams p, uint32_t* __restrict__ bitmap) {
  grid_dependency_wait();
  grid_dependents_launch();  // the append may come up meanwhile
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (i >= p.num_tokens) return;
  const int32_t slot = __ldg(p.slots + i);
  int32_t bits = token_bits(p, slot, i);
  if (slot < 0) return;
  if (!(bits & IRIS_ERR_SLOT_RANGE)) {
    const uint32_t bit = 1u << (slot & 31);
    if (atomicOr(bitmap + (slot >> 5), bit) & bit) bits |= IRIS_ERR_DUP_SLOT;
  }
  if (bits) set_error(p.err, bits);
}

// The same for batches of up to kPairwiseTokens tokens without a bitmap, and
// so without a workspace or clearing one: every slot is held against all the
// others, by eight lanes a token.  (Every CTA of the append looking all slots up
// in a hash table of its own instead, without this launch: 1021 tokens 9.2 us
// instead of 7.5.)
constexpr int64_t kPairwiseTokens = 2048;
__global__ void __launch_bounds__(kThreads) mrope_check_pairs_kernel(const MropeParams p) {
  __shared__ __align__(16) int32_t s_slot[kPairwiseTokens];
  grid_dependency_wait();
  grid_dependents_launch();  // the append may come up meanwhile
  const int T = static_cast<int>(p.num_tokens), T4 = (T + 3) & ~3;
  for (int i = threadIdx.x; i < T4; i += kThreads) s_slot[i] = i < T ? __ldg(p.slots + i) : -1;
  const int i = (blockIdx.x * kThreads + threadIdx.x) >> 3, part = threadIdx.x & 7;
  const int32_t slot = i < T ? __ldg(p.slots + i) : -1;
  int32_t bits = 0;
  if (slot >= 0 && part == 0) bits = token_bits(p, slot, i);
  __syncthreads();
  if (slot < 0) return;  // all eight lanes of the token
  int hits = 0;
  for (int j = 4 * part; j < T4; j += 32) {
    const int4 v = *reinterpret_cast<const int4*>(s_slot + j);
    hits += (v.x == slot) + (v.y == slot) + (v.z == slot) + (v.w == slot);
  }
  const unsigned mates = 0xFFu << (threadIdx.x & 24);  // the token's lanes, which all came here
  if (__reduce_add_sync(mates, hits) > 1 && static_cast<int64_t>(slot) < p.num_slots) bits |= IRIS_ERR_DUP_SLOT;
  if (part == 0 && bits) set_error(p.err, bits);
}

// The same for at most kInlineCheckTokens tokens, by every CTA of the append.
IRIS_DEV bool check_small_batch(const MropeParams& p) {
  __shared__ __align__(16) int32_t s_slot[kInlineCheckTokens];
  const int T = static_cast<int>(p.num_tokens), T4 = (T + 3) & ~3;
  int32_t bits = 0;
  for (int i = threadIdx.x; i < T4; i += blockDim.x) {
    const int32_t s = i < T ? __ldg(p.slots + i) : -1;
    if (i < T) bits |= token_bits(p, s, i);
    s_slot[i] = s;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < T; i += blockDim.x) {
    const int32_t s = s_slot[i];
    if (s < 0 || static_cast<int64_t>(s) >= p.num_slots) continue;
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
IRIS_DEV void blend_rows(const MropeParams& p, int64_t tok, int fv, float2 (&c)[4], float2 (&s)[4]) {
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
    c[j] = E::unpack(cw[j]);
    s[j] = E::unpack(sw[j]);
  }
}

template <typename E>
IRIS_DEV void unpack8(const uint4& w, float2 (&x)[4]) {
  x[0] = E::unpack(w.x);
  x[1] = E::unpack(w.y);
  x[2] = E::unpack(w.z);
  x[3] = E::unpack(w.w);
}
template <typename E>
IRIS_DEV uint4 pack8(const float2 (&x)[4]) {
  return make_uint4(E::pack(x[0].x, x[0].y), E::pack(x[1].x, x[1].y), E::pack(x[2].x, x[2].y), E::pack(x[3].x, x[3].y));
}

// max(|a|, |b|, |c|), NaN if one of them is.
IRIS_DEV float absmax3(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(fabsf(a)), "f"(fabsf(b)), "f"(fabsf(c)));
  return d;
}

// Eight fp32 values of a group of four lanes -> fp16 group scale and this
// lane's packed word.  y / scale is rounded as the IEEE division rounds it: r
// is the correctly rounded reciprocal, t = x r is off by at most 1.5 ulp, and
// one residual step (Markstein 1990) leaves an error of 2^-23 ulp before the
// last rounding, while a quotient of a 24-bit by an 11-bit number that is no
// rounding midpoint stays 2^-12 ulp away from one.  amax / 7 takes two such
// steps, its first quotient then being faithful whatever amax is.
IRIS_DEV uint32_t quant8(const float2 (&x)[4], uint32_t quad, __half& scale16) {
  float m = absmax3(x[0].x, x[0].y, x[1].x);
  m = absmax3(m, x[1].y, x[2].x);
  m = absmax3(m, x[2].y, x[3].x);
  m = absmax3(m, x[3].y, __shfl_xor_sync(quad, absmax3(m, x[3].y, 0.0f), 1));
  m = absmax3(m, 0.0f, __shfl_xor_sync(quad, m, 2));
  if (!(m <= 3.402823466e38f)) {  // an infinity or NaN in the group
    scale16 = __float2half_rn(m);
    return 0u;
  }
  const float r7 = 0.142857149f;  // fp32(1 / 7)
  float s = m * r7;
  s = fmaf(fmaf(-s, 7.0f, m), r7, s);
  s = fmaf(fmaf(-s, 7.0f, m), r7, s);
  scale16 = __float2half_rn(fminf(fmaxf(s, 6.103515625e-05f), 65504.0f));
  const float sc = __half2float(scale16), r = __frcp_rn(sc);
  const float2 r2 = make_float2(r, r), ns2 = make_float2(-sc, -sc);
  float2 q[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 t = __fmul2_rn(x[j], r2);
    q[j] = __ffma2_rn(__ffma2_rn(t, ns2, x[j]), r2, t);
  }
  if (s > 65504.0f) {  // only then can a quotient pass 7 by more than a rounding
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      q[j].x = fminf(fmaxf(q[j].x, -7.0f), 7.0f);
      q[j].y = fminf(fmaxf(q[j].y, -7.0f), 7.0f);
    }
  }
  const float2 magic = make_float2(8388624.0f, 8388624.0f);  // 2^23 + 16: rounds half to even, low four bits the nibble
  uint32_t z[8];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 v = __fadd2_rn(q[j], magic);
    z[2 * j] = __float_as_uint(v.x);
    z[2 * j + 1] = __float_as_uint(v.y);
  }
  const uint32_t ev = __byte_perm(__byte_perm(z[0], z[2], 0x0040), __byte_perm(z[4], z[6], 0x0040), 0x5410);
  const uint32_t od = __byte_perm(__byte_perm(z[1], z[3], 0x0040), __byte_perm(z[5], z[7], 0x0040), 0x5410);
  return (ev & 0x0F0F0F0Fu) | ((od << 4) & 0xF0F0F0F0u);
}

// kSmall: at most kInlineCheckTokens tokens, one a CTA, validated here;
// otherwise the check kernel before this launch did it.  The first keys (with
// few tokens the first values and queries too) are asked for before anything
// else is looked at: they depend on neither the slot nor the positions.  With
// few tokens the check comes next, whose loads do not wait for one another, so
// that a thread's own slot and positions are then at hand (64 tokens: 9.0 ->
// 7.9 us).  With many tokens more warps on an SM do more than more loads a
// thread: with 64 registers a thread 8192 tokens take 62.3 us, with 85 68.4
// and with 48 73.5.
template <typename E, bool kSmall, bool kPaired>
__global__ void __launch_bounds__(kThreads, kSmall ? 2 : 4) mrope_append_kernel(const MropeParams p) {
  if constexpr (kSmall) grid_dependency_wait();
  constexpr int kBatch = kPaired ? 1 : 2;  // heads whose vectors a thread has on the way, of each kind
  const int units = kPaired ? p.vecs / 2 : p.vecs;
  const int per_token = p.row_lanes * units;
  const int here = threadIdx.x / per_token, in_token = threadIdx.x - here * per_token;
  const int row = in_token / units, unit = in_token - row * units;  // first head, and place within the head
  const int64_t tok = static_cast<int64_t>(blockIdx.x) * (blockDim.x / per_token) + here;
  const bool there = tok < p.num_tokens;  // (the last CTA's threads past the end go along with the checks)
  const int64_t at = there ? tok : 0;
  const int half = p.rotary_vecs / 2;  // vectors of the rotary half
  // this thread's vector v and, `mate` vectors on, the one that turns with it (of the dims that do not turn, their other half's)
  const bool rotary = unit < (kPaired ? half : p.rotary_vecs), low = kPaired || unit < half;
  const int v = kPaired && !rotary ? unit + half : unit;
  const int mate = kPaired && !rotary ? (p.vecs - p.rotary_vecs) / 2 : low ? half : -half;
  const int64_t D2 = 16ll * p.vecs;         // bytes of a head
  const int64_t stride = D2 * p.row_lanes;  // bytes to this thread's next head
  const char* key = static_cast<const char*>(p.key) + at * p.key_stride * 2 + row * D2 + 16 * v;
  const char* value = static_cast<const char*>(p.value) + at * p.value_stride * 2 + row * D2 + 16 * v;
  const char* query = static_cast<const char*>(p.query) + at * p.query_stride * 2 + row * D2 + 16 * v;
  if constexpr (!kSmall) {
    // the token's values and queries go to L2 while its keys are worked on (8192 tokens: 78 -> 69 us)
    if (in_token == 0 && there) {
      prefetch_l2_bulk(static_cast<const char*>(p.value) + at * p.value_stride * 2, static_cast<uint32_t>(D2 * p.kv_heads));
      if (p.q_heads > 0)
        prefetch_l2_bulk(static_cast<const char*>(p.query) + at * p.query_stride * 2, static_cast<uint32_t>(D2 * p.q_heads));
    }
  }
  // vectors of heads h, h + row_lanes, .. of a tensor, and if wanted their mates
  const auto load = [&](const char* src, int h, int heads, bool mates, uint4 (&x)[kBatch], uint4 (&o)[kBatch]) {
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      if (h + j * p.row_lanes < heads) {
        x[j] = ldg_nc_v4(src + j * stride);
        if (kPaired || mates) o[j] = ldg_nc_v4(src + j * stride + 16 * mate);
      }
    }
  };
  uint4 kx[kBatch], ko[kBatch];
  load(key, row, p.kv_heads, rotary, kx, ko);
  uint4 vx[kBatch], vo[kBatch], qx[kBatch], qo[kBatch];
  if constexpr (kSmall) {
    load(value, row, p.kv_heads, false, vx, vo);
    load(query, row, p.q_heads, rotary, qx, qo);
  }
  bool rejected = false;
  int32_t pending = 0;
  if constexpr (kSmall) {  // before the token's own slot: that and its positions then come from L1
    if (p.err != nullptr) pending = *reinterpret_cast<volatile int32_t*>(p.err);
    rejected = check_small_batch(p);
  }
  const int32_t slot = there ? __ldg(p.slots + tok) : -1;
  // A token with a bad slot or position: never touch memory outside the cache
  // or the tables.  (The check records its bits.)
  const bool live = token_bits(p, slot, at) == 0 && slot >= 0;
  float2 c[4], s[4];
  if (live && rotary) {
    blend_rows<E>(p, tok, low ? v : v - half, c, s);
    if (low) {
#pragma unroll
      for (int j = 0; j < 4; ++j) s[j] = make_float2(-s[j].x, -s[j].y);
    }
  }
  if constexpr (!kSmall) {
    grid_dependency_wait();
    if (p.err != nullptr) pending = *reinterpret_cast<volatile int32_t*>(p.err);
  }
  if (rejected || (pending & kRejectBits) != 0) return;
  if (!there) return;
  const uint32_t quad = 0xFu << (threadIdx.x & 28);

  // x cos + mate (-+ sin): both products are exact, one rounding in all.  Paired: the mate's, too.
  const auto turn = [&](const uint4& xw, const uint4& ow, float2 (&x)[4], float2 (&o)[4]) {
    unpack8<E>(xw, x);
    if (kPaired || rotary) unpack8<E>(ow, o);
    if (rotary) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 xs = __fmul2_rn(x[j], s[j]);
        x[j] = __ffma2_rn(x[j], c[j], __fmul2_rn(o[j], s[j]));
        if constexpr (kPaired) o[j] = __ffma2_rn(o[j], c[j], make_float2(-xs.x, -xs.y));
      }
    }
  };
  const int64_t cache_row = static_cast<int64_t>(slot) * p.kv_heads;
  const auto store = [&](const float2 (&x)[4], int64_t vec, uint8_t* data, __half* scales) {
    __half scale;
    const uint32_t word = quant8(x, quad, scale);
    reinterpret_cast<uint32_t*>(data)[vec] = word;
    if ((unit & 3) == 0) scales[vec >> 2] = scale;
  };

  char* out = p.key_out != nullptr ? static_cast<char*>(p.key_out) + (at * p.kv_heads + row) * D2 + 16 * v : nullptr;
  for (int h = row; h < p.kv_heads; h += kBatch * p.row_lanes) {
    if (h != row) load(key, h, p.kv_heads, rotary, kx, ko);
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int hh = h + j * p.row_lanes;
      if (hh < p.kv_heads) {
        uint4* to = reinterpret_cast<uint4*>(out + j * stride);
        if (live) {
          float2 x[4], o[4];
          turn(kx[j], ko[j], x, o);
          const int64_t vec = (cache_row + hh) * p.vecs + v;
          if (out != nullptr) *to = pack8<E>(x);
          store(x, vec, p.k_data, p.k_scale);
          if constexpr (kPaired) {
            if (out != nullptr) to[mate] = pack8<E>(o);
            store(o, vec + mate, p.k_data, p.k_scale);
          }
        } else if (out != nullptr) {  // padding: its rotated rows are zeros
          *to = make_uint4(0, 0, 0, 0);
          if constexpr (kPaired) to[mate] = make_uint4(0, 0, 0, 0);
        }
      }
    }
    key += kBatch * stride;
    if (out != nullptr) out += kBatch * stride;
  }
  if (live) {
    for (int h = row; h < p.kv_heads; h += kBatch * p.row_lanes) {
      if (!kSmall || h != row) load(value, h, p.kv_heads, false, vx, vo);
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const int hh = h + j * p.row_lanes;
        if (hh < p.kv_heads) {
          float2 x[4];
          const int64_t vec = (cache_row + hh) * p.vecs + v;
          unpack8<E>(vx[j], x);
          store(x, vec, p.v_data, p.v_scale);
          if constexpr (kPaired) {
            unpack8<E>(vo[j], x);
            store(x, vec + mate, p.v_data, p.v_scale);
          }
        }
      }
      value += kBatch * stride;
    }
  }
  out = static_cast<char*>(p.query_out) + (at * p.q_heads + row) * D2 + 16 * v;
  for (int h = row; h < p.q_heads; h += kBatch * p.row_lanes) {
    if (!kSmall || h != row) load(query, h, p.q_heads, rotary, qx, qo);
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      if (h + j * p.row_lanes < p.q_heads) {
        float2 x[4], o[4];
        uint4 word = make_uint4(0, 0, 0, 0), other = word;
        if (live) {
          turn(qx[j], qo[j], x, o);
          word = pack8<E>(x);
          if constexpr (kPaired) other = pack8<E>(o);
        }
        uint4* to = reinterpret_cast<uint4*>(out + j * stride);
        *to = word;
        if constexpr (kPaired) to[mate] = other;
      }
    }
    query += kBatch * stride;
    out += kBatch * stride;
  }
}

// Threads of a token of a large batch that share a vector.  More of them read
// and blend the token's rotary rows more often, fewer walk longer over its
// heads: 8192 tokens as above take 68.4, 66.1, 62.3 and 74.9 us with 2, 4, 8
// and 16, 1021 tokens of 3 x 16 heads 26.7, 20.5, 16.4 and 17.5.
constexpr int kRowLanes = 8;

template <typename E>
cudaError_t launch_mrope(MropeParams& p, uint32_t* bitmap, size_t bitmap_bytes, cudaStream_t stream) {
  if (p.num_tokens <= kInlineCheckTokens) {  // few tokens: as many threads on each as fit
    p.row_lanes = kThreads / p.vecs;
    return launch_early(mrope_append_kernel<E, true, false>, static_cast<unsigned>(p.num_tokens), p.row_lanes * p.vecs, 0,
                        stream, p);
  }
  // Vectors in pairs where whole groups turn with whole groups (8192 tokens: 69 -> 62 us); with few tokens the
  // longer work of a thread costs more than its loads (64 tokens: 14.4 -> 15.0 us).
  const bool paired = p.rotary_vecs % 8 == 0;
  const int units = paired ? p.vecs / 2 : p.vecs;
  p.row_lanes = kThreads / units < kRowLanes ? kThreads / units : kRowLanes;
  const int threads = kThreads / (p.row_lanes * units) * (p.row_lanes * units);
  const int64_t tokens = threads / (p.row_lanes * units);  // a CTA
  cudaError_t e = cudaSuccess;
  if (p.num_tokens <= kPairwiseTokens) {
    e = launch_early(mrope_check_pairs_kernel, static_cast<unsigned>((8 * p.num_tokens + kThreads - 1) / kThreads),
                     kThreads, 0, stream, p);
  } else {
    if (bitmap_bytes > 0) e = cudaMemsetAsync(bitmap, 0, bitmap_bytes, stream);
    if (e == cudaSuccess)
      e = launch_early(mrope_check_kernel, static_cast<unsigned>((p.num_tokens + kThreads - 1) / kThreads), kThreads, 0,
                       stream, p, bitmap);
  }
  if (e != cudaSuccess) return e;
  // comes up while the check finishes
  return launch_early(paired ? mrope_append_kernel<E, false, true> : mrope_append_kernel<E, false, false>,
                      static_cast<unsigned>((p.num_tokens + tokens - 1) / tokens), threads, 0, stream, p);
}

}  // namespace
}  // namespace iris

using namespace iris;

extern "C" size_t iris_b200_mrope_append_workspace_bytes(int64_t num_tokens, int64_t num_pages, int32_t page_size) {
  if (num_tokens <= kPairwiseTokens || num_pages <= 0 || page_size <= 0) return 0;
  return iris_b200_append_check_workspace_bytes(num_pages, page_size);
}

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
  if (num_kv_heads > (1 << 16) || num_q_heads > (1 << 16)) return IRIS_EUNSUPPORTED;
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
  const size_t need = iris_b200_mrope_append_workspace_bytes(num_tokens, num_pages, page_size);
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
