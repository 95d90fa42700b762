// Attention of new tokens over the INT4 paged cache (prompts, chunks of
// prompts, drafts, single tokens): the public form is
// iris_b200_int4_paged_varlen_attention.
//
// A block owns up to 128 * kTiles rows (new token x query head) of one KV head
// and walks the tiles of 128 cached tokens that any of them sees.  Its warps:
//   * softmax warps, two threads a row (64 columns each), eight warps a row tile:
//     scores from tensor memory, mask, cap and bias, running maximum and sum in
//     registers, probabilities back to tensor memory as the next product's operand;
//   * four or eight unpacking warps, a cached token a thread: packed rows (TMA)
//     and scales become swizzled fp16 tiles;
//   * one warp that issues the products: S = Q K^T (both operands in shared
//     memory, K-major) and O += P V (P in tensor memory, V as it lies, MN-major);
//   * one warp that issues the copies.
// Two row tiles take turns: one's softmax runs while the other's products do.
// A row's scores are read twice, 32 columns at a time (maximum, then
// probabilities): all at once would not fit the registers, and what is spilled
// here misses the few kilobytes of L1 that are left (740 us against 506 for two
// prompts of 4096 tokens when that was tried).  Some spills remain, 40 to 230 bytes
// read a thread, most of them with a cap or a bias.
//
// Roundings.  A stored key or value is nibble * scale: 15 bits, where fp16 has 11.
// Values are rounded.  Keys are not, as the log-sum-exp of a row with few tokens
// would show it (1e-4 of a logit): their scale is split into its upper 8 bits and
// the rest, and two exact fp16 tiles follow each other in the product.  (The
// second one's products take 50 of the 432 us of two prompts of 4096 tokens; there
// is a second tile's store as well, and with 128 dims no second key buffer.)
//
// Each run of 32 tokens is first scaled by a power of two that brings its largest
// scale into [2^12, 2^13), so that neither large scales overflow nor small ones
// lose bits; a key's into [2^11, 2^12), as its upper 8 bits may round up and -8
// times 2^13 is past fp16 (keys stay exact down to 2^-25 of the run's largest
// scale).  Runs whose tokens' values lie further apart than 2^8 give each token a
// power of its own.  The power goes into the logit's factor (keys) and the
// probability's exponent (values).
//
// Probabilities are fp16, at 2^8 for the largest that a token adds to the row, its
// probability times its values' power.  So values that the row does not see, or
// that weigh nothing, cost the others no bits; relative to the largest probability
// and to all tokens' largest value they cost them all from a factor of 2^25 on (two
// prompts of 4096 tokens took 422 us then).  Logits, statistics and sums are fp32.
#include "varlen_few.cuh"

namespace iris {
namespace {

template <int D, int kTiles>
struct Cfg {
  static constexpr int kOperand = kTile * D * 2;       // one fp16 tile
  static constexpr int kPacked = kTile * D / 2;        // one packed tile
  static constexpr int kKeySlots = D == 128 ? 1 : 2;   // of two tiles
  static constexpr int kOperands = kTiles + 2 * kKeySlots + 2;
  static constexpr int kSmem = 1024 + kOperands * kOperand + 3 * kPacked;  // two packed slots of keys, one of values
  static constexpr int kColumns = kTiles == 2 ? 512 : 256;
  static constexpr int kOutColumn = kTiles * kTile;    // first column of O
  static constexpr int kSoftWarps = 8 * kTiles;
  static constexpr int kMmaWarp = kSoftWarps + (kTiles == 2 ? 4 : 8), kCopyWarp = kMmaWarp + 1;
  static constexpr int kThreads = 32 * (kMmaWarp + 4);  // (two warps idle: registers move by warpgroups)
  // Registers a thread: launched with 80 (kTiles 2: 768 x 80 = 61,440) or 96 (640 x 96 = 61,440), then shared out as
  // 512 x 88 + 128 x 72 + 128 x 56 = 61,440 or 256 x 136 + 256 x 72 + 128 x 56 = 60,416.
  static constexpr int kSoftRegs = kTiles == 2 ? 88 : 136, kUnpackRegs = 72, kIssueRegs = 56;
};

struct Shared {
  uint64_t raw_full[3], raw_empty[3];  // packed tiles: two slots of keys, one of values
  uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2];
  uint64_t s_full[2], p_full[2], o_full[2], drain;
  uint32_t tmem;
  alignas(16) int32_t k_exp[4][4], v_exp[4][4];  // [tile & 3][run of 32 tokens]
  alignas(8) uint32_t v_any[2][4];   // 1: a run has values that are not finite; 2: its tokens have powers of their own
  uint8_t v_bad[2][kTile];           // which groups of a token's
  float v_own[2][kTile];             // a token's own power
  float top[2][2][2][kTile];         // [tile & 1][row tile][half]: a row's largest logit; at the end its sum
  float back[2][kTile];              // undoes the query row's power of two
  uint32_t spoilt[2][kTile];         // groups of dims with a visible value that is not finite
  // the block's work
  int32_t b, index, start, count, len, first_lo;
  int32_t live;
};

// Tokens of a run share a power where their largest scales lie this many powers of two apart or less.
constexpr int kSpread = 8;

// ------------------------------------------------------------------ unpacking
// One tile of keys or values, with its scales.  False: a wait gave up.
template <int D, bool keys>
IRIS_DEV bool unpack_tile(const AttendParams& p, Shared& sh, int k, const uint32_t (&sc)[D / 64], uint32_t packed,
                        uint32_t operands, int tid) {
  using C = Cfg<D, 1>;
  constexpr int kGroups = D / 32;
  const int warp = tid >> 5, lane = tid & 31;
  const int st = keys ? k % C::kKeySlots : k & 1, slot = keys ? k & 1 : 2;
  const uint32_t round = keys ? k / C::kKeySlots & 1 : (k >> 1) & 1;
  // what the run of 32 tokens is scaled by, and what is not finite
  uint32_t most = 0, bad = 0;
#pragma unroll
  for (int c = 0; c < kGroups; ++c) {
    const uint32_t mag = (sc[c / 2] >> (16 * (c & 1))) & 0x7fffu;
    if (mag >= 0x7c00u) bad |= 1u << c; else most = max(most, mag);
  }
  int e = static_cast<int>(__reduce_max_sync(0xffffffffu, most) >> 10);
  const int run_e = e;
  bool wide = false;
  if (!keys) {
    const int own = static_cast<int>(most >> 10);
    wide = run_e - static_cast<int>(__reduce_min_sync(0xffffffffu, most != 0 ? own : 31)) > kSpread;
    if (wide) e = own;
  }
  constexpr int kUp = keys ? 26 : 27;
  const float up = pow2i(kUp - e);
  if (!wait_all(&sh.raw_full[slot], keys ? (k >> 1) & 1 : k & 1, p.s.err)) return false;
  if (!wait_all(keys ? &sh.k_empty[st] : &sh.v_empty[st], round ^ 1, p.s.err)) return false;
  if (keys) {
    if (lane == 0) sh.k_exp[k & 3][warp] = e - kUp;
  } else {
    const bool any = __any_sync(0xffffffffu, bad != 0);
    if (lane == 0) {
      sh.v_exp[k & 3][warp] = run_e - kUp;
      sh.v_any[st][warp] = static_cast<uint32_t>(any) | (wide ? 2u : 0u);
    }
    if (wide) sh.v_own[st][tid] = static_cast<float>(e - kUp);
    if (any) sh.v_bad[st][tid] = static_cast<uint8_t>(bad);
  }
  const uint32_t src = packed + slot * C::kPacked, dst = operands + st * (keys ? 2 : 1) * C::kOperand;
#pragma unroll 1
  for (int c = 0; c < kGroups; ++c) {
    const uint4 w4 = lds128(src + packed_at<D>(tid, c));
    const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
    const uint32_t bits = (D == 128 && c >= 2 ? sc[kGroups / 2 - 1] : sc[0]) >> (16 * (c & 1));
    const float v = __half2float(__ushort_as_half(static_cast<unsigned short>(bits))) * up;
    float top = v;
    if (keys) {  // its upper 8 bits (Veltkamp's split), and what is left
      const float t = __fmul_rn(v, 65537.0f);
      top = __fsub_rn(t, __fsub_rn(t, v));
    }
    const bool odd = (bad >> c) & 1u;
    const __half2 s = u32_as_h2(odd ? (keys ? 0x7fff7fffu : 0u) : Fp16Elem::pack(top, top)),
                  r = u32_as_h2(odd ? 0u : Fp16Elem::pack(v - top, v - top));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 n0 = u32_as_h2(int4_lo_exact(w[i])), n1 = u32_as_h2(int4_hi_exact(w[i])),
                    n2 = u32_as_h2(int4_lo_exact(w[i] >> 8)), n3 = u32_as_h2(int4_hi_exact(w[i] >> 8));
      const uint32_t at = dst + operand_at(tid, 4 * c + i);
      sts128(at, h2_as_u32(__hmul2(n0, s)), h2_as_u32(__hmul2(n1, s)), h2_as_u32(__hmul2(n2, s)), h2_as_u32(__hmul2(n3, s)));
      if (keys)
        sts128(at + C::kOperand, h2_as_u32(__hmul2(n0, r)), h2_as_u32(__hmul2(n1, r)), h2_as_u32(__hmul2(n2, r)),
               h2_as_u32(__hmul2(n3, r)));
    }
  }
  fence_proxy_async_shared();
  mbar_arrive(keys ? &sh.k_full[st] : &sh.v_full[st]);
  mbar_arrive(&sh.raw_empty[slot]);
  return true;
  }

// kKeys, kValues: what this warpgroup unpacks (both: in turn).
template <int D, bool kKeys, bool kValues>
IRIS_DEV void unpack_tiles(const AttendParams& p, Shared& sh, const Tiles& tiles, int k0, int n, int b, int len, int h,
                           uint32_t packed, uint32_t k_tiles, uint32_t v_tiles, int tid) {
  constexpr int kGroups = D / 32;
  auto token = [&](int k) { return tiles.at(k0 + k) * kTile + tid; };
  uint32_t sc2[2][kGroups / 2];  // the scales of the tile that is next
  auto fetch = [&](const uint8_t* scales, int32_t page, int32_t j, uint32_t (&s)[kGroups / 2]) {
    const uint8_t* x = scales + ((static_cast<int64_t>(page) * kTokPage + (j & (kTokPage - 1))) * p.s.hkv + h) * (D / 16);
    if constexpr (D == 128) {
      const uint2 v = j < len ? __ldg(reinterpret_cast<const uint2*>(x)) : make_uint2(0, 0);
      s[0] = v.x;
      s[1] = v.y;
    } else {
      s[0] = j < len ? __ldg(reinterpret_cast<const uint32_t*>(x)) : 0u;
    }
  };
  int32_t page = page_of(p.s, b, token(0), len);
  if (kKeys) fetch(p.k_scale, page, token(0), sc2[0]);
  if (kValues) fetch(p.v_scale, page, token(0), sc2[1]);
  page = n > 1 ? raw_page(p.s, b, token(1), len) : 0;
#pragma unroll 1
  for (int k = 0; k < n; ++k) {
    uint32_t now[2][kGroups / 2];
#pragma unroll
    for (int i = 0; i < kGroups / 2; ++i) now[0][i] = sc2[0][i], now[1][i] = sc2[1][i];
    if (k + 1 < n) {
      const int32_t id = checked_page(p.s, page);
      if (kKeys) fetch(p.k_scale, id, token(k + 1), sc2[0]);
      if (kValues) fetch(p.v_scale, id, token(k + 1), sc2[1]);
      if (k + 2 < n) page = raw_page(p.s, b, token(k + 2), len);
    }
    if (kKeys && !unpack_tile<D, true>(p, sh, k, now[0], packed, k_tiles, tid)) break;
    if (kValues && !unpack_tile<D, false>(p, sh, k, now[1], packed, v_tiles, tid)) break;
  }
}

// --------------------------------------------------------------------- copies
template <int D>
IRIS_DEV void issue_copies(const AttendParams& p, const CUtensorMap* k_map, const CUtensorMap* v_map, Shared& sh,
                           const Tiles& tiles, int k0, int n, int b, int len, int h, uint8_t* packed, int lane) {
  constexpr int kPacked = kTile * D / 2;
  auto first = [&](int k) { return tiles.at(k0 + k) * kTile; };
  auto page_at = [&](int k) { return lane < 8 ? raw_page(p.s, b, first(k) + lane * kTokPage, len) : 0; };
  int32_t later = page_at(0);
  int k = 0;
#pragma unroll 1
  for (; k < n; ++k) {
    const int32_t page = checked_page(p.s, later);
    if (k + 1 < n) later = page_at(k + 1);
    const int st = k & 1;
    if (!wait_all(&sh.raw_empty[st], ((k >> 1) & 1) ^ 1, p.s.err)) break;
    load_packed<D>(packed + st * kPacked, k_map, page, first(k), len, h, &sh.raw_full[st], lane);
    if (!wait_all(&sh.raw_empty[2], (k & 1) ^ 1, p.s.err)) break;
    load_packed<D>(packed + 2 * kPacked, v_map, page, first(k), len, h, &sh.raw_full[2], lane);
  }
  if (k < n)  // a wait gave up: copies that are under way land before the block ends
    for (int i = 0; i < 6; ++i) mbar_wait_bounded(&sh.raw_full[i % 3], i / 3, p.s.err);
}

// ------------------------------------------------------------------- products
template <int D, int kTiles>
IRIS_DEV void issue_products(const AttendParams& p, Shared& sh, int n, int active, uint32_t q_tiles, uint32_t k_tiles,
                             uint32_t v_tiles, uint32_t tmem) {
  using C = Cfg<D, kTiles>;
  constexpr uint32_t kScores = umma_idesc(kTile, kTile, false, false), kOut = umma_idesc(kTile, D, false, true);
  auto scores = [&](int i, int k) {
    if (elect_one()) {
      const uint32_t q = umma_fresh(umma_desc_low(q_tiles + i * C::kOperand, 16)),
                     kk = umma_fresh(umma_desc_low(k_tiles + k % C::kKeySlots * 2 * C::kOperand, 16));
#pragma unroll
      for (int x = 0; x < 2 * D / 16; ++x) {
        const int s = x % (D / 16);
        const uint32_t at = ((s >> 2) * (kTile * 128) + (s & 3) * 32) >> 4;
        umma_ss(tmem + i * kTile, umma_desc_from(q + at, 1024),
                umma_desc_from(kk + at + (x < D / 16 ? 0 : C::kOperand >> 4), 1024), kScores, x > 0);
      }
      umma_commit(smem_u32(&sh.s_full[i]));
      if (i == active - 1) umma_commit(smem_u32(&sh.k_empty[k % C::kKeySlots]));
    }
    __syncwarp();
  };
  bool ok = wait_all(&sh.k_full[0], 0, p.s.err);
  if (ok) {
    umma_fence_after();
    for (int i = 0; i < active; ++i) scores(i, 0);
  }
  for (int k = 0; ok && k < n; ++k) {
    ok = wait_all(&sh.v_full[k & 1], (k >> 1) & 1, p.s.err);
    for (int i = 0; ok && i < active; ++i) {
      ok = wait_all(&sh.p_full[i], k & 1, p.s.err);
      if (!ok) break;
      umma_fence_after();
      if (elect_one()) {
        const uint32_t v = umma_fresh(umma_desc_low(v_tiles + (k & 1) * C::kOperand, kTile * 128));
#pragma unroll
        for (int s = 0; s < kTile / 16; ++s)
          umma_ts(tmem + C::kOutColumn + i * D, tmem + i * kTile + 8 * s + (s < 4 ? 0 : 32), umma_desc_from(v + (s * 2048 >> 4), 1024), kOut,
                  k > 0 || s > 0);
        umma_commit(smem_u32(&sh.o_full[i]));
        if (i == active - 1) umma_commit(smem_u32(&sh.v_empty[k & 1]));
      }
      __syncwarp();
      if (k + 1 < n) {
        if (i == 0) ok = wait_all(&sh.k_full[(k + 1) % C::kKeySlots], (k + 1) / C::kKeySlots & 1, p.s.err);
        if (!ok) break;
        umma_fence_after();
        scores(i, k + 1);
      }
    }
  }
  // everything issued is done before the block lets go of its memory
  if (elect_one()) umma_commit(smem_u32(&sh.drain));
  __syncwarp();
  wait_all(&sh.drain, 0, p.s.err);
}

// -------------------------------------------------------------------- softmax
// 32 columns of this thread's lane.
IRIS_DEV void load_scores(uint32_t at, float (&s)[32]) {
  umma_ld32(at, reinterpret_cast<uint32_t*>(s));
  umma_wait_ld();
#pragma unroll
  for (int j = 0; j < 32; ++j) asm volatile("" : "+f"(s[j]));
}

template <int D, int kTiles, bool kCap, bool kBias>
IRIS_DEV void softmax_rows(const AttendParams& p, Shared& sh, const Tiles& tiles, int k0, int n, int rows, int h, int tile,
                           uint32_t q_tiles, uint32_t tmem, int split, int warp, int lane) {
  using C = Cfg<D, kTiles>;
  constexpr bool kMod = kCap || kBias;
  const int half = warp >> 2, quarter = warp & 3;
  const int local = quarter * 32 + lane;  // row of the row tile
  const int r = sh.index * (kTile * kTiles) + tile * kTile + local;
  const bool valid = r < rows;
  const int i = valid ? r / p.s.group : 0, g = valid ? r % p.s.group : 0;
  const int token = sh.start + i, head = h * p.s.group + g;
  const int32_t pos = sh.len - sh.count + i;
  Sight sight = {0, 0, 0, 0};
  if (valid) {
    const int32_t prefix = p.s.prefix_lens != nullptr ? __ldg(p.s.prefix_lens + sh.b) : 0;
    const int32_t first = p.s.first_visible != nullptr ? __ldg(p.s.first_visible + token) : 0;
    sight = row_sight(pos, first, prefix, p.s.window, sh.len);
  }
  if (n > 0) {  // the tile's query rows: four threads a row, 64 rows at a time
    constexpr int kWords = D / 8;
#pragma unroll
    for (int r0 = 0; r0 < kTile; r0 += 64) {
      const int row = r0 + (warp * 32 + lane) / 4, part = lane & 3;
      const int rr = min(sh.index * (kTile * kTiles) + tile * kTile + row, rows - 1);
      const int64_t at = (sh.start + rr / p.s.group) * p.q_stride + static_cast<int64_t>(h * p.s.group + rr % p.s.group) * D;
      const uint4* src = reinterpret_cast<const uint4*>(p.query + at + part * (D / 4));
      uint32_t w[kWords];
#pragma unroll
      for (int c = 0; c < kWords / 4; ++c) {
        const uint4 v = src[c];
        w[4 * c] = v.x;
        w[4 * c + 1] = v.y;
        w[4 * c + 2] = v.z;
        w[4 * c + 3] = v.w;
      }
      const float undo = scale_row_part<kWords>(w, p.bf16 != 0, [](uint32_t m) {
        m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
        return max(m, __shfl_xor_sync(0xffffffffu, m, 2));
      });
      if (part == 0) sh.back[tile][row] = undo;
      const uint32_t dst = q_tiles + tile * C::kOperand;
#pragma unroll
      for (int c = 0; c < kWords / 4; ++c) {
        const uint4 v = order8(w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]);
        sts128(dst + operand_at(row, part * (D / 32) + c), v.x, v.y, v.z, v.w);
      }
    }
  }
  if (half == 0) sh.spoilt[tile][local] = 0;
  fence_proxy_async_shared();
  asm volatile("bar.sync 1, %0;" ::"n"(C::kSoftWarps * 32 + 32) : "memory");  // with the warp of the products

  const uint32_t lanes = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
  const uint32_t s_at = lanes + tile * kTile + half * 64, o_at = lanes + C::kOutColumn + tile * D + half * (D / 2);
  const bool busy = __any_sync(0xffffffffu, valid);
  const float back = n > 0 ? sh.back[tile][local] : 1.0f;
  const float unit = fminf(kCap ? p.s.scale * back / p.s.cap : p.s.scale * kLog2e * back, 1e38f);  // (0 times it is 0)
  const float cap2 = p.s.cap * kLog2e;
  const float slope2 = kBias ? -__ldg(p.s.slopes + head) * kLog2e : 0.0f;
  auto meet = [&] { asm volatile("bar.sync %0, 64;" ::"r"(2 + tile * 4 + quarter) : "memory"); };  // the rows' two warps
  // Probabilities stand relative to 2^(m + ref): what a token adds to the row, 2^(logit + its values' power), is near or
  // below that.  m is 0 unless the logits lie far out, where whole numbers as small as ref have no room beside them.
  float m = 0.0f, ref = kMinusInf, l = 0.0f;
  bool ok = true;
#pragma unroll 1
  for (int k = 0; k < n; ++k) {
    // (once a wait has given up no other is made, but the two warps go on meeting)
    ok = ok && wait_all(&sh.s_full[tile], k & 1, p.s.err);
    ok = ok && wait_all(&sh.v_full[k & 1], (k >> 1) & 1, p.s.err);
    umma_fence_after();
    if (busy) {
      const int32_t base = tiles.at(k0 + k) * kTile + half * 64;
      const int4 ve = *reinterpret_cast<const int4*>(sh.v_exp[k & 3]);
      const int2 ke = *reinterpret_cast<const int2*>(sh.k_exp[k & 3] + 2 * half);
      const float f[2] = {fmaxf(unit * pow2i(ke.x), 1.17549435e-38f), fmaxf(unit * pow2i(ke.y), 1.17549435e-38f)};
      const int ves[2] = {half ? ve.z : ve.x, half ? ve.w : ve.y};
      const uint2 any2 = *reinterpret_cast<const uint2*>(&sh.v_any[k & 1][2 * half]);
      const uint32_t any[2] = {any2.x, any2.y};
      const bool full = !valid || (sight.b0 <= base && base + 64 <= sight.b1) || (sight.a0 <= base && base + 64 <= sight.a1);
      const bool masked = !__all_sync(0xffffffffu, full);
      // the largest that a token of run c adds, from the logits in tensor memory as they now are
      auto largest = [&](int c) {
        float s[32], t = kMinusInf;
        load_scores(s_at + 32 * c, s);
        const float* own = sh.v_own[k & 1] + 64 * half + 32 * c;
#pragma unroll
        for (int j = 0; j < 32; ++j)
          t = fmaxf(t, ((kMod ? s[j] : __fmul_rn(s[j], f[c])) - m) + (any[c] & 2 ? own[j] : static_cast<float>(ves[c])));
        return t;
      };
      // ---- the largest that a token adds; with a mask, a cap or a bias the logits go back as they now are
      float top = kMinusInf;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float s[32];
        load_scores(s_at + 32 * c, s);
        if (kMod) {
#pragma unroll
          for (int j = 0; j < 32; ++j) s[j] *= f[c];
          if (kCap && !cap_near(s, cap2)) {  // 16 at a time, through tensor memory: there are no registers for more
#pragma unroll 1
            for (int q = 0; q < 32; q += 16) {
              float x[16];
              umma_ld16(s_at + 32 * c + q, reinterpret_cast<uint32_t*>(x));
              umma_wait_ld();
#pragma unroll
              for (int j = 0; j < 16; ++j) {
                asm volatile("" : "+f"(x[j]));
                x[j] = cap2 * tanh_f(x[j] * f[c]);
              }
              umma_st16(s_at + 32 * c + q, reinterpret_cast<const uint32_t*>(x));
            }
            umma_wait_st();
            load_scores(s_at + 32 * c, s);
          }
          if (kBias) {
            const float d0 = static_cast<float>(pos - base - 32 * c);
#pragma unroll
            for (int j = 0; j < 32; ++j) s[j] = fmaf(slope2, fabsf(d0 - j), s[j]);
          }
        }
        if (masked) {
          const uint32_t bits = valid ? sight_bits(sight, base + 32 * c) : ~0u;
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (!((bits >> j) & 1u)) s[j] = kMinusInf;
        }
        if (kMod || masked) umma_st32(s_at + 32 * c, reinterpret_cast<const uint32_t*>(s));
        float t0 = s[0], t1 = s[1];
#pragma unroll
        for (int j = 2; j < 32; j += 2) {
          t0 = fmaxf(t0, s[j]);
          t1 = fmaxf(t1, s[j + 1]);
        }
        t0 = fmaxf(t0, t1);
        if (!(any[c] & 2)) top = fmaxf(top, ((kMod ? t0 : __fmul_rn(t0, f[c])) - m) + static_cast<float>(ves[c]));
      }
      if (kMod || masked) umma_wait_st();
      if ((any[0] | any[1]) & 2) {
#pragma unroll 1
        for (int c = 0; c < 2; ++c)
          if (any[c] & 2) top = fmaxf(top, largest(c));
      }
      auto share = [&] {  // the larger of the two halves' (uniform over a row's two warps from there on)
        sh.top[k & 1][tile][half][local] = top;
        meet();
        top = fmaxf(top, sh.top[k & 1][tile][half ^ 1][local]);
      };
      share();
      // raise the row's reference where something passes it by too much
      const bool rise = top > ref + kRise;  // (also from -inf)
      if (__any_sync(0xffffffffu, rise)) {
        const float m_old = m, ref_old = ref;
        bool out = rise && (m != 0.0f || fabsf(top) >= kFarOut);
#pragma unroll 1
        for (int look = 0; look < 3 && __any_sync(0xffffffffu, out); ++look) {  // m about there, or 0, and a look at the rest
          if (out) m = fabsf(m + top) >= kFarOut ? rintf(m + top) : 0.0f;
          const float before = top;
          top = fmaxf(largest(0), largest(1));
          meet();  // what was shared is read
          share();
          if (!out) top = before;
          out = out && fabsf(top) >= kFarOut;
        }
        if (rise) ref = rintf(top);
        const float by = rise ? ex2((m_old - m) + (ref_old - ref)) : 1.0f;
        if (k > 0) {
          ok = ok && wait_all(&sh.o_full[tile], (k - 1) & 1, p.s.err);
          umma_fence_after();
#pragma unroll 1
          for (int c = 0; c < D / 64; ++c) {
            float o[32];
            load_scores(o_at + 32 * c, o);
#pragma unroll
            for (int j = 0; j < 32; ++j) o[j] *= by;
            umma_st32(o_at + 32 * c, reinterpret_cast<const uint32_t*>(o));
          }
          l *= by;
        }
      }
      const float off = ref == kMinusInf ? 0.0f : ref;  // (a row that sees nothing yet)
      const bool far = __any_sync(0xffffffffu, m != 0.0f);
      // ---- probabilities and their sum
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float s[32];
        load_scores(s_at + 32 * c, s);
        float add = kHead + static_cast<float>(ves[c]) - off, by = f[c], unlift = pow2i(-ves[c] - 8);
        if (far || (any[c] & 2)) {  // (m comes off rounded products: one that is not rounded would be another logit)
#pragma unroll
          for (int j = 0; j < 32; ++j) s[j] = (kMod ? s[j] : __fmul_rn(s[j], by)) - m;
          by = 1.0f;
        }
        if (any[c] & 2) {  // tokens with powers of their own
          const float* own = sh.v_own[k & 1] + 64 * half + 32 * c;
          add = kHead - off;
          unlift = 0.0f;
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            l += ex2(s[j] - off);
            s[j] += own[j];
          }
        }
        float2 sum = make_float2(0.0f, 0.0f);
        uint32_t w[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          float2 y = make_float2(s[2 * j], s[2 * j + 1]);
          y = kMod ? __fadd2_rn(y, make_float2(add, add)) : __ffma2_rn(y, make_float2(by, by), make_float2(add, add));
          y.x = ex2(y.x);
          y.y = ex2(y.y);
          sum = __fadd2_rn(sum, y);
          w[j] = Fp16Elem::pack(y.x, y.y);
        }
        l = fmaf(sum.x + sum.y, unlift, l);
        umma_st16(s_at + 16 * c, w);  // over this thread's own scores, which are read
      }
      if ((any[0] | any[1]) & 1) {
#pragma unroll 1
        for (int c = 0; c < 2; ++c) {
          if (!(any[c] & 1)) continue;
          uint32_t hit = 0;
          for (uint32_t left = valid ? sight_bits(sight, base + 32 * c) : 0u; left != 0; left &= left - 1)
            hit |= sh.v_bad[k & 1][64 * half + 32 * c + __ffs(left) - 1];
          if (hit != 0) atomicOr(&sh.spoilt[tile][local], hit);
        }
      }
      umma_wait_st();
    }
    umma_fence_before();
    mbar_arrive(&sh.p_full[tile]);
  }
  // the row's output: half the dims each
  if (ok && n > 0) {
    ok = wait_all(&sh.o_full[tile], (n - 1) & 1, p.s.err);
    umma_fence_after();
  }
  sh.top[n & 1][tile][half][local] = l;
  if (!busy) return;
  meet();
  if (!ok) return;
  l += sh.top[n & 1][tile][half ^ 1][local];
  const uint32_t spoilt = sh.spoilt[tile][local];
  const bool whole = p.splits == 1;
  const int64_t row = static_cast<int64_t>(token) * p.s.hq + head;
  const float norm = l == 0.0f ? 0.0f : (1.0f / 256.0f) / l;
#pragma unroll 1
  for (int c = 0; c < D / 64; ++c) {
    const int group = half * (D / 64) + c;  // of 32 dims
    float v[32];
    if (n > 0) load_scores(o_at + 32 * c, v);
#pragma unroll
    for (int j = 0; j < 32; ++j) {
      v[j] = n > 0 && l != 0.0f ? v[j] * norm : 0.0f;
      if ((spoilt >> group) & 1u) v[j] = __int_as_float(0x7fffffff);
    }
    if (!valid) continue;
#pragma unroll
    for (int q = 0; q < 4; ++q) {  // 8 dims, back in their order
      const float* x = v + 8 * q;
      if (whole) {
        uint4 w;
        if (p.bf16)
          w = make_uint4(Bf16Elem::pack(x[0], x[2]), Bf16Elem::pack(x[4], x[6]), Bf16Elem::pack(x[1], x[3]),
                         Bf16Elem::pack(x[5], x[7]));
        else
          w = make_uint4(Fp16Elem::pack(x[0], x[2]), Fp16Elem::pack(x[4], x[6]), Fp16Elem::pack(x[1], x[3]),
                         Fp16Elem::pack(x[5], x[7]));
        reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + row * D)[4 * group + q] = w;
      } else {
        float4* dst = reinterpret_cast<float4*>(p.part_o + (static_cast<int64_t>(split) * p.s.tokens * p.s.hq + row) * D);
        dst[2 * (4 * group + q)] = make_float4(x[0], x[2], x[4], x[6]);
        dst[2 * (4 * group + q) + 1] = make_float4(x[1], x[3], x[5], x[7]);
      }
    }
  }
  if (!valid || half != 0) return;
  const float lse = l == 0.0f ? kMinusInf : m + (ref + lg2(l));
  if (!whole)
    p.part_lse[static_cast<int64_t>(split) * p.s.tokens * p.s.hq + row] = lse;
  else if (p.out_lse != nullptr)
    p.out_lse[row] = lse;
}

static_assert(Cfg<128, 2>::kSmem + sizeof(Shared) <= 227 * 1024, "a block's shared memory");

template <int D, int kTiles, bool kCap, bool kBias>
__global__ void __launch_bounds__(Cfg<D, kTiles>::kThreads, 1)
    varlen_attention_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                            const AttendParams p) {
  using C = Cfg<D, kTiles>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ Shared sh;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int unit = blockIdx.x / (p.s.hkv * p.splits);
  const int h = blockIdx.x / p.splits % p.s.hkv, split = blockIdx.x % p.splits;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.k_full[i], 128);
      mbar_init(&sh.v_full[i], 128);
      mbar_init(&sh.k_empty[i], 1);
      mbar_init(&sh.v_empty[i], 1);
      mbar_init(&sh.s_full[i], 1);
      mbar_init(&sh.p_full[i], 256);
      mbar_init(&sh.o_full[i], 1);
    }
    for (int i = 0; i < 3; ++i) {
      mbar_init(&sh.raw_full[i], 1);
      mbar_init(&sh.raw_empty[i], 128);
    }
    mbar_init(&sh.drain, 1);
    fence_barrier_init();
  }
  grid_dependency_wait();
  grid_dependents_launch();
  if (warp == 0) {
    if (blockIdx.x == 0) check_offsets(p.s, lane);
    Block blk = {0, 0, {0, 0}, 0};
    const bool live = find_block(p.s, unit, kTile * kTiles, p.few ? kFewRows : 0, INT64_MAX, lane, &blk);
    int first = 0;
    Span sp = {0, 0};
    int32_t len = 0;
    if (live) {
      sp = blk.span;
      len = cached_tokens(p.s, blk.len, sp.count, lane == 0 && h == 0 && split == 0 && blk.index == 0);
      first = first_of_block(p.s, sp, blk.index, kTile * kTiles, lane);
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
  clear_unused<D>(p);
  __syncthreads();
  if (!sh.live) return;
  if (warp == C::kMmaWarp) umma_alloc(&sh.tmem, C::kColumns);
  umma_fence_before();
  __syncthreads();
  umma_fence_after();
  const uint32_t tmem = sh.tmem;

  const int rows = sh.count * p.s.group;
  const int r0 = sh.index * (kTile * kTiles), r1 = min(r0 + kTile * kTiles, rows);
  const int active = r1 - r0 > kTile ? 2 : 1;
  const int32_t off = sh.len - sh.count;
  const int32_t prefix = p.s.prefix_lens != nullptr ? __ldg(p.s.prefix_lens + sh.b) : 0;
  const Tiles tiles =
      tiles_seen(off + r0 / p.s.group, off + (r1 - 1) / p.s.group, sh.first_lo, prefix, p.s.window, sh.len);
  const int64_t all = tiles.count();
  const int k0 = static_cast<int>(all * split / p.splits), n = static_cast<int>(all * (split + 1) / p.splits) - k0;

  uint8_t* base = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const uint32_t q_tiles = smem_u32(base), k_tiles = q_tiles + kTiles * C::kOperand, v_tiles = k_tiles + 2 * C::kKeySlots * C::kOperand;
  uint8_t* packed = base + C::kOperands * C::kOperand;
  if (warp < C::kSoftWarps) {
    regs_take<C::kSoftRegs>();
    const int tile = warp >> 3;
    if (tile < active) {
      softmax_rows<D, kTiles, kCap, kBias>(p, sh, tiles, k0, n, rows, h, tile, q_tiles, tmem, split, warp & 7, lane);
    } else {
      asm volatile("bar.sync 1, %0;" ::"n"(C::kSoftWarps * 32 + 32) : "memory");
    }
  } else if (warp < C::kMmaWarp) {
    regs_give<C::kUnpackRegs>();
    const int tid = (threadIdx.x - C::kSoftWarps * 32) & 127;
    if (n > 0) {
      const uint32_t raw = smem_u32(packed);
      if (kTiles == 2)
        unpack_tiles<D, true, true>(p, sh, tiles, k0, n, sh.b, sh.len, h, raw, k_tiles, v_tiles, tid);
      else if (warp < C::kSoftWarps + 4)
        unpack_tiles<D, true, false>(p, sh, tiles, k0, n, sh.b, sh.len, h, raw, k_tiles, v_tiles, tid);
      else
        unpack_tiles<D, false, true>(p, sh, tiles, k0, n, sh.b, sh.len, h, raw, k_tiles, v_tiles, tid);
    }
  } else {
    regs_give<C::kIssueRegs>();
    if (warp == C::kMmaWarp) {
      asm volatile("bar.sync 1, %0;" ::"n"(C::kSoftWarps * 32 + 32) : "memory");
      if (n > 0) issue_products<D, kTiles>(p, sh, n, active, q_tiles, k_tiles, v_tiles, tmem);
    } else if (warp == C::kCopyWarp && n > 0) {
      issue_copies<D>(p, &k_map, &v_map, sh, tiles, k0, n, sh.b, sh.len, h, packed, lane);
    }
  }
  umma_fence_before();
  __syncthreads();
  umma_fence_after();
  if (warp == C::kMmaWarp) umma_free(tmem, C::kColumns);
}

// Joins the parts of rows whose tiles several blocks shared: a warp a row.
template <int D>
__global__ void __launch_bounds__(256) varlen_join_kernel(const AttendParams p) {
  grid_dependency_wait();
  grid_dependents_launch();
  const int64_t rows = static_cast<int64_t>(used_rows(p.s)) * p.s.hq;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (row >= rows) return;
  if (p.few) {  // the other kernel's rows are not here; the row's sequence is the last that starts at or before it
    const int32_t token = static_cast<int32_t>(row / p.s.hq);
    int lo = 0, hi = p.s.batch;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (__ldg(p.s.cu + mid) <= token) lo = mid; else hi = mid;
    }
    if (static_cast<int64_t>(new_tokens(p.s, lo).count) * p.s.group <= kFewRows) return;
  }
  join_row<D>(p, p.part_o + row * D, p.part_lse + row, p.splits, static_cast<int64_t>(p.s.tokens) * p.s.hq, row,
              threadIdx.x & 31);
}

// ----------------------------------------------------------------------- host
constexpr int kFewTiles = 2;  // blocks of few rows: each of so many tiles or more
constexpr int kFewStart = 6;  // ... and costing about so many before the first

int sm_count(int device) {
  static int known[64] = {};
  if (device < 0 || device >= 64) return 148;
  if (known[device] == 0) {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess || n <= 0) n = 148;
    known[device] = n;
  }
  return known[device];
}

// Rows, places and page offsets are 32-bit numbers in the kernels.
bool too_long(int64_t tokens, int32_t group, int32_t max_pages) {
  return tokens > INT32_MAX / 2 / group || max_pages > INT32_MAX / 2 / kTokPage;
}

// Which kernels run, and how the work is cut.
//
// Sequences of at most kFewRows rows go to varlen_few_kernel, the others to
// varlen_attention_kernel.  With one new token a sequence the host knows which;
// with offsets both are launched unless all rows together are few (an empty
// launch costs 2 to 5 us; one kernel for both would give single tokens 128-row
// products, 837 us where the other takes a sixth of it at 64 x 4096).
struct Plan {
  bool few, many;
  int tiles;               // row tiles of a block (many)
  int64_t many_blocks, few_blocks;
  int32_t splits, chunks, per;
  int cols;                // columns of a block (few)
  int64_t many_parts, few_parts;  // rows of parts in the workspace
};
Plan plan(int64_t tokens, int32_t batch, int32_t group, bool offsets, int32_t hkv, int32_t max_pages, int32_t window,
          bool prefix, int sms) {
  Plan r = {};
  const int64_t rows = tokens * group;
  r.few = offsets || group <= kFewRows;
  r.many = offsets ? rows > kFewRows : group > kFewRows;
  int64_t tiles = (static_cast<int64_t>(max_pages) * kTokPage + kTile - 1) / kTile;  // that a block may see
  const int64_t all_tiles = tiles;
  if (window > 0 && !prefix) tiles = tiles < window / kTile + 4 ? tiles : window / kTile + 4;
  r.splits = r.chunks = 1;
  const int64_t some = batch < tokens ? batch : tokens;
  if (r.many) {
    // two row tiles a block where sequences have more than 128 rows on average
    r.tiles = offsets && rows > 128 * static_cast<int64_t>(batch) ? 2 : 1;
    const int64_t each = 128 * r.tiles;
    r.many_blocks = offsets ? rows / each + some : batch * ((group + each - 1) / each);
    // blocks that share a row's tiles: as many as bring a block to every SM, each with four tiles or more
    const int64_t want = sms / (r.many_blocks * hkv), most = tiles / 4;
    const int64_t n = want < most ? want : most;
    r.splits = static_cast<int32_t>(n < 1 ? 1 : n);
  }
  if (r.few) {
    const int64_t most_rows = offsets ? (rows < kFewRows ? rows : kFewRows) : group;
    r.cols = most_rows <= 4 ? 4 : most_rows <= 8 ? 8 : most_rows <= 16 ? 16 : 32;
    r.few_blocks = offsets ? some : batch;  // (kFewRows rows are one block)
    if (offsets && r.cols < kFewRows) r.few_blocks = some;
    // (when they were chosen, 64 x 4096 tokens: two chunks 137 us, four 154; 16 x 5 drafts over 4096: two 98 us, five 122)
    const int64_t slots = static_cast<int64_t>(sms) * (r.cols <= 8 ? 3 : 2);
    const int64_t n = best_chunks(r.few_blocks * hkv, tiles, slots, kFewStart, (tiles + kFewTiles - 1) / kFewTiles);
    r.per = static_cast<int32_t>((all_tiles < tiles ? all_tiles : tiles) + n - 1) / static_cast<int32_t>(n);
    // a window's tiles are an estimate from above; a prefix may add to it, so chunks cover all tiles there
    const int64_t cover = window > 0 && !prefix ? tiles : all_tiles;
    r.chunks = static_cast<int32_t>((cover + r.per - 1) / r.per);
  }
  r.many_parts = r.many && r.splits > 1 ? r.splits * rows * hkv : 0;
  r.few_parts = r.few && r.chunks > 1 ? static_cast<int64_t>(r.chunks) * batch * hkv * r.cols : 0;
  return r;
}

template <int D, int kTiles, bool kCap, bool kBias>
cudaError_t launch_attend(const AttendParams& p, int64_t grid, cudaStream_t stream) {
  auto fn = varlen_attention_kernel<D, kTiles, kCap, kBias>;
  static thread_local uint64_t ready = 0;  // GPUs that know the kernel's shared memory
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  if (device >= 64 || !((ready >> device) & 1)) {
    e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<D, kTiles>::kSmem);
    if (e != cudaSuccess) return e;
    if (device < 64) ready |= 1ull << device;
  }
  CUtensorMap k, v;
  if (!packed_map(&k, p.k_data, D, p.s.hkv, p.s.num_pages) || !packed_map(&v, p.v_data, D, p.s.hkv, p.s.num_pages))
    return cudaErrorInvalidValue;
  return launch_early(fn, dim3(static_cast<unsigned>(grid)), dim3(Cfg<D, kTiles>::kThreads), Cfg<D, kTiles>::kSmem, stream,
                      k, v, p);
}

template <int D, int kCols, bool kCap, bool kBias>
cudaError_t launch_few(const AttendParams& p, int64_t grid, cudaStream_t stream) {
  auto fn = varlen_few_kernel<D, kCols, kCap, kBias>;
  static thread_local uint64_t ready = 0;
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  if (device >= 64 || !((ready >> device) & 1)) {
    e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, FewCfg<D, kCols>::kSmem);
    if (e != cudaSuccess) return e;
    if (device < 64) ready |= 1ull << device;
  }
  CUtensorMap k, v;
  const int64_t pages = p.s.num_pages;
  if (!packed_map(&k, p.k_data, D, p.s.hkv, pages) || !packed_map(&v, p.v_data, D, p.s.hkv, pages))
    return cudaErrorInvalidValue;
  return launch_early(fn, dim3(static_cast<unsigned>(grid)), dim3(288), FewCfg<D, kCols>::kSmem, stream, k, v, p);
}
template <int D, int kCols>
cudaError_t launch_few(const AttendParams& p, int64_t grid, cudaStream_t stream) {
  const bool cap = p.s.cap > 0.0f, bias = p.s.slopes != nullptr;
  if (cap && bias) return launch_few<D, kCols, true, true>(p, grid, stream);
  if (cap) return launch_few<D, kCols, true, false>(p, grid, stream);
  if (bias) return launch_few<D, kCols, false, true>(p, grid, stream);
  return launch_few<D, kCols, false, false>(p, grid, stream);
}

template <int D>
cudaError_t launch_few(const AttendParams& p, int cols, int64_t grid, cudaStream_t stream) {
  if (cols == 4) return launch_few<D, 4>(p, grid, stream);
  if (cols == 8) return launch_few<D, 8>(p, grid, stream);
  if (cols == 16) return launch_few<D, 16>(p, grid, stream);
  return launch_few<D, 32>(p, grid, stream);
}

template <int D, int kTiles>
cudaError_t launch_attend(const AttendParams& p, int64_t grid, cudaStream_t stream) {
  const bool cap = p.s.cap > 0.0f, bias = p.s.slopes != nullptr;
  if (cap && bias) return launch_attend<D, kTiles, true, true>(p, grid, stream);
  if (cap) return launch_attend<D, kTiles, true, false>(p, grid, stream);
  if (bias) return launch_attend<D, kTiles, false, true>(p, grid, stream);
  return launch_attend<D, kTiles, false, false>(p, grid, stream);
}

}  // namespace
}  // namespace iris

using namespace iris;

extern "C" size_t iris_b200_varlen_attention_workspace_bytes(int64_t tokens, int32_t batch, int32_t num_q_heads,
                                                             int32_t num_kv_heads, int32_t head_dim,
                                                             int32_t max_pages_per_seq, int32_t window, int32_t has_prefix,
                                                             int32_t has_offsets, int32_t device) {
  // (what the operator refuses, or is done with at once, needs none; the plan is only right for the rest)
  if (tokens <= 0 || batch <= 0 || num_kv_heads <= 0 || num_q_heads <= 0 || num_q_heads % num_kv_heads != 0 ||
      (head_dim != 64 && head_dim != 128) || max_pages_per_seq <= 0 || window < 0 ||
      too_long(tokens, num_q_heads / num_kv_heads, max_pages_per_seq) || (has_offsets == 0 && tokens != batch))
    return 0;
  const Plan r = plan(tokens, batch, num_q_heads / num_kv_heads, has_offsets != 0, num_kv_heads, max_pages_per_seq, window,
                      has_prefix != 0, sm_count(device));
  return static_cast<size_t>(r.many_parts + r.few_parts) * (head_dim + 1) * 4;
}

extern "C" int iris_b200_int4_paged_varlen_attention(
    const void* query, int64_t query_stride, const void* k_data, const void* v_data, const void* k_scale,
    const void* v_scale, const int32_t* block_table, int64_t block_table_stride, const int32_t* seq_lens,
    const int32_t* cu_seqlens, const float* slopes, const int32_t* prefix_lens, const int32_t* first_visible, void* output,
    float* out_lse, int64_t tokens, int32_t batch, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
    int64_t num_pages, int32_t page_size, int32_t max_pages_per_seq, int32_t window, float logit_cap, float softmax_scale,
    int32_t dtype, void* workspace, size_t workspace_bytes, int32_t* error_word, void* stream) {
  if (tokens < 0 || batch < 0 || num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads != 0 || window < 0 ||
      !(logit_cap >= 0.0f && logit_cap <= 1e20f) || !(softmax_scale > 0.0f) || (dtype != IRIS_DTYPE_FP16 && dtype != IRIS_DTYPE_BF16))
    return IRIS_EINVAL;
  if (page_size != kTokPage || (head_dim != 64 && head_dim != 128)) return IRIS_EUNSUPPORTED;
  if (cu_seqlens == nullptr && tokens != batch) return IRIS_EINVAL;
  if (tokens == 0) return IRIS_OK;
  if (batch == 0 || num_pages <= 0 || max_pages_per_seq <= 0) return IRIS_EINVAL;
  if (query == nullptr || k_data == nullptr || v_data == nullptr || k_scale == nullptr || v_scale == nullptr ||
      block_table == nullptr || seq_lens == nullptr || output == nullptr)
    return IRIS_EINVAL;
  const int32_t group = num_q_heads / num_kv_heads;
  if (too_long(tokens, group, max_pages_per_seq) || num_pages > INT32_MAX) return IRIS_EUNSUPPORTED;
  if (!aligned_to(query, 16) || query_stride % 8 != 0 || !aligned_to(k_data, 16) || !aligned_to(v_data, 16) ||
      !aligned_to(k_scale, 8) || !aligned_to(v_scale, 8) || !aligned_to(output, 16))
    return IRIS_EALIGN;
  const bool offsets = cu_seqlens != nullptr;
  int device = 0;
  clear_stale_cuda_error();
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return record_cuda_error(e, "cudaGetDevice"), IRIS_ECUDA;
  const Plan r = plan(tokens, batch, group, offsets, num_kv_heads, max_pages_per_seq, window, prefix_lens != nullptr,
                      sm_count(device));
  const int64_t many_grid = r.many_blocks * num_kv_heads * r.splits, few_grid = r.few_blocks * num_kv_heads * r.chunks;
  if (many_grid > INT32_MAX || few_grid > INT32_MAX) return IRIS_EUNSUPPORTED;
  const int64_t parts = r.many_parts + r.few_parts;
  if (parts > 0 && (workspace == nullptr || workspace_bytes < static_cast<size_t>(parts) * (head_dim + 1) * 4))
    return IRIS_EWORKSPACE;
  if (parts > 0 && !aligned_to(workspace, 16)) return IRIS_EALIGN;
  AttendParams p = {};
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
  p.k_data = static_cast<const uint8_t*>(k_data);
  p.v_data = static_cast<const uint8_t*>(v_data);
  p.k_scale = static_cast<const uint8_t*>(k_scale);
  p.v_scale = static_cast<const uint8_t*>(v_scale);
  p.out = output;
  p.out_lse = out_lse;
  p.part_o = static_cast<float*>(workspace);
  p.few_o = p.part_o + r.many_parts * head_dim;
  p.part_lse = p.part_o + parts * head_dim;
  p.few_lse = p.part_lse + r.many_parts;
  p.q_stride = query_stride;
  p.splits = r.splits;
  p.chunks = r.chunks;
  p.per = r.per;
  p.few = r.few;
  p.many = r.many;
  p.bf16 = dtype == IRIS_DTYPE_BF16;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (r.many) {
    if (head_dim == 128)
      e = r.tiles == 2 ? launch_attend<128, 2>(p, many_grid, st) : launch_attend<128, 1>(p, many_grid, st);
    else
      e = r.tiles == 2 ? launch_attend<64, 2>(p, many_grid, st) : launch_attend<64, 1>(p, many_grid, st);
    if (e != cudaSuccess) return record_cuda_error(e, "varlen_attention"), IRIS_ECUDA;
  }
  if (r.few) {
    e = head_dim == 128 ? launch_few<128>(p, r.cols, few_grid, st) : launch_few<64>(p, r.cols, few_grid, st);
    if (e != cudaSuccess) return record_cuda_error(e, "varlen_few"), IRIS_ECUDA;
  }
  if (r.few_parts > 0) {
    const dim3 grid(static_cast<unsigned>(static_cast<int64_t>(batch) * num_kv_heads));
    e = head_dim == 128 ? launch_early(varlen_few_join_kernel<128>, grid, dim3(128), 0, st, p, r.cols)
                        : launch_early(varlen_few_join_kernel<64>, grid, dim3(128), 0, st, p, r.cols);
    if (e != cudaSuccess) return record_cuda_error(e, "varlen_few_join"), IRIS_ECUDA;
  }
  if (r.many_parts > 0) {
    const dim3 grid(static_cast<unsigned>((tokens * num_q_heads + 7) / 8));
    e = head_dim == 128 ? launch_early(varlen_join_kernel<128>, grid, dim3(256), 0, st, p)
                        : launch_early(varlen_join_kernel<64>, grid, dim3(256), 0, st, p);
    if (e != cudaSuccess) return record_cuda_error(e, "varlen_join"), IRIS_ECUDA;
  }
  return IRIS_OK;
}
