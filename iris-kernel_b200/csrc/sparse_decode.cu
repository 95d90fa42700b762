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
// pages with 16-byte asynchronous copies into a ring of its own (no barrier
// between warps) and keeps its own running softmax.  Products run on the
// tensor cores with fp32 accumulation:
//   S = Q K^T  rows = query heads, columns = tokens; K as the exact integers
//              in the query's 16-bit type, one accumulator per 32-dim group,
//              the group scale applied in fp32;
//   O = P V    rows = query heads, columns = dims; V as the exact integers in
//              bf16; p * scale is split into two bf16 terms (16 bits, and
//              fp32's range).  With G <= 8 the second term fills the product's
//              idle rows 8 .. 15 at no cost; otherwise it takes a second
//              product.
// The warps' partial results meet in shared memory, over a cluster of up to 8
// CTAs where few rows have to fill the GPU, and each CTA writes its share of
// the outputs.
#include "elem.cuh"

namespace iris {
namespace {

constexpr int kPage = 16;
constexpr int kWarps = 4;
constexpr int kStages = 4;

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
  float scale_log2;
  int32_t* err;
};

IRIS_DEV void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
template <int N>
IRIS_DEV void cp_async_small(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(N) : "memory");
}
IRIS_DEV void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
IRIS_DEV void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

IRIS_DEV void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
IRIS_DEV void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The signed nibbles in bits 0-3 and 16-19 of w as two bf16: 0x4300 | n ^ 8 is
// 128 + (n + 8) (one lop3, as for fp16 in common.cuh), minus 136 exactly.
IRIS_DEV uint32_t nibbles_bf16(uint32_t w) {
  const uint32_t biased = lop3<kLutMagic>(w, 0x000f000fu, 0x43084308u);
  const __nv_bfloat162 v =
      __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&biased), __floats2bfloat162_rn(136.0f, 136.0f));
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Eight nibbles of a word as four pairs (0,4) (1,5) (2,6) (3,7) of the type.
IRIS_DEV void pairs(const Fp16Elem&, uint32_t w, uint32_t (&o)[4]) {
  o[0] = int4_lo_exact(w);
  o[1] = int4_hi_exact(w);
  o[2] = int4_lo_exact(w >> 8);
  o[3] = int4_hi_exact(w >> 8);
}
IRIS_DEV void pairs(const Bf16Elem&, uint32_t w, uint32_t (&o)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) o[j] = nibbles_bf16(w >> (4 * j));
}
IRIS_DEV void mma_qk(const Fp16Elem&, float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  mma_f16(d, a, b0, b1);
}
IRIS_DEV void mma_qk(const Bf16Elem&, float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  mma_bf16(d, a, b0, b1);
}

IRIS_DEV uint32_t map_to_rank(uint32_t addr, uint32_t rank) {
  uint32_t out;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(out) : "r"(addr), "r"(rank));
  return out;
}
IRIS_DEV float ld_cluster(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
IRIS_DEV void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
IRIS_DEV uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}

template <int D>
struct SparseCfg {
  static constexpr int kGroups = D / 32;
  static constexpr int kData = kPage * D / 2;        // bytes of a page's head, K or V
  static constexpr int kScale = kPage * kGroups * 2;  // bytes of its scales
  static constexpr int kStage = 2 * (kData + kScale);
  static constexpr int kRing = kStages * kStage;  // per warp
  static constexpr int kChunks = D / 32;          // 16-byte chunks per row
};

// Byte offset of 16-byte chunk c of row r: rows 0, 2, 4, .. would start at the
// same banks, so the chunks of a row are turned by a function of the row.
template <int D>
IRIS_DEV int chunk_at(int r, int c) {
  if constexpr (D == 128) return r * 64 + ((c ^ ((r >> 1) & 3)) << 4);
  else return r * 32 + ((c ^ ((r >> 2) & 1)) << 4);
}

// Output records: per warp and query head, fp32 [D + 2]: o, m, l.
template <typename E, int D, bool kWide>
__global__ void __launch_bounds__(32 * kWarps) sparse_decode_kernel(const SparseParams p, int splits) {
  using C = SparseCfg<D>;
  constexpr int kHeads = kWide ? 16 : 8;
  constexpr int G4 = C::kGroups;
  extern __shared__ __align__(128) uint8_t smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int row = blockIdx.x / splits;  // sequence * Hkv + head
  const int split = splits > 1 ? static_cast<int>(cluster_rank()) : 0;
  const int b = row / p.kv_heads, h = row - b * p.kv_heads;
  const int len = __ldg(p.seq_lens + b);
  if (len < 0 && h == 0 && split == 0 && threadIdx.x == 0) set_error(p.err, IRIS_ERR_SEQ_LEN);
  const int count = min(max(__ldg(p.counts + row), 0), p.keep);
  const int workers = splits * kWarps, me = split * kWarps + warp;
  const int mine = count > me ? (count - me + workers - 1) / workers : 0;  // pages me, me + workers, ..
  const int32_t* list = p.lists + static_cast<int64_t>(row) * p.keep;

  const uint32_t ring = smem_u32(smem) + warp * C::kRing;
  int32_t* stage_col = reinterpret_cast<int32_t*>(smem + kWarps * C::kRing) + warp * kStages;
  int32_t my_col = -1;   // this lane's page of the current 32: logical
  int64_t my_page = -1;  // and physical, -1 where there is none
  const auto look_up = [&](int at) {
    my_col = -1;
    my_page = -1;
    if (at >= mine) return;
    const int col = __ldg(list + me + static_cast<int64_t>(at) * workers);
    if (col < 0 || static_cast<int64_t>(col) * kPage >= len) return;
    if (col >= p.max_pages) {
      set_error(p.err, IRIS_ERR_BLOCK_TABLE);
      return;
    }
    const int64_t page = __ldg(p.block_table + b * p.table_stride + col);
    if (page < 0 || page >= p.num_pages) {
      set_error(p.err, IRIS_ERR_PAGE_ID);
      return;
    }
    my_col = col;
    my_page = page;
  };
  // starts the copies of the warp's page i, or of nothing where there is none
  const auto fetch = [&](int i) {
    if (i < mine) {
      if ((i & 31) == 0) look_up(i + lane);
      const int64_t page = __shfl_sync(0xffffffffu, my_page, i & 31);
      const int32_t col = __shfl_sync(0xffffffffu, my_col, i & 31);
      if (lane == 0) stage_col[i % kStages] = col;
      if (page >= 0) {
        const uint32_t st = ring + (i % kStages) * C::kStage;
        const int64_t row0 = page * kPage * p.kv_heads + h;
        const uint8_t* kd = p.k_data + row0 * (D / 2);
        const uint8_t* vd = p.v_data + row0 * (D / 2);
        const int64_t step = static_cast<int64_t>(p.kv_heads) * (D / 2);
#pragma unroll
        for (int j = lane; j < kPage * C::kChunks; j += 32) {
          const int r = j / C::kChunks, c = j % C::kChunks;
          const int at = chunk_at<D>(r, c);
          cp_async16(st + at, kd + r * step + 16 * c);
          cp_async16(st + C::kData + at, vd + r * step + 16 * c);
        }
        const int r = lane & 15;
        const __half* sc = (lane < 16 ? p.k_scale : p.v_scale) + (row0 + static_cast<int64_t>(r) * p.kv_heads) * G4;
        cp_async_small<2 * G4>(st + 2 * C::kData + (lane >> 4) * C::kScale + r * 2 * G4, sc);
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) fetch(i);

  // query fragments, in the pair order of the unpacked nibbles
  uint32_t qa[G4][2][4];
#pragma unroll
  for (int k = 0; k < G4; ++k) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      uint4 w = make_uint4(0, 0, 0, 0);
      const int hq = g + 8 * half;
      if ((half == 0 || kWide) && hq < p.group)
        w = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.query) +
                                                 (static_cast<int64_t>(row) * p.group + hq) * D + 32 * k + 8 * t));
      // words hold dims (0,1) (2,3) (4,5) (6,7) of this lane's eight
      qa[k][0][half] = prmt(w.x, w.z, 0x5410);      // dims 0, 4
      qa[k][0][half + 2] = prmt(w.x, w.z, 0x7632);  // dims 1, 5
      qa[k][1][half] = prmt(w.y, w.w, 0x5410);      // dims 2, 6
      qa[k][1][half + 2] = prmt(w.y, w.w, 0x7632);  // dims 3, 7
    }
  }

  constexpr int kTiles = D / 8;
  float o[kTiles][4];
#pragma unroll
  for (int j = 0; j < kTiles; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;
  constexpr int kH = kWide ? 2 : 1;  // query heads a lane: g, g + 8
  float m[kH], l[kH];
#pragma unroll
  for (int a = 0; a < kH; ++a) {
    m[a] = -INFINITY;
    l[a] = 0.0f;
  }
  const uint32_t v_sel = g < 4 ? 0x5410u : 0x7632u;

  for (int i = 0; i < mine; ++i) {
    __syncwarp();  // every lane is done with the stage that is filled next
    fetch(i + kStages - 1);
    cp_async_wait<kStages - 1>();
    __syncwarp();
    const int col = stage_col[i % kStages];
    if (col < 0) continue;
    const uint32_t st = ring + (i % kStages) * C::kStage;

    // scales of this lane's tokens 2 t, 2 t + 1, 2 t + 8, 2 t + 9
    float ks[4][G4], vs[4][G4];
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      const int tok = 2 * t + (a & 1) + 8 * (a >> 1);
      const uint32_t at = st + 2 * C::kData + tok * 2 * G4;
#pragma unroll
      for (int k = 0; k < G4; k += 2) {
        const float2 x = __half22float2(u32_as_h2(lds32(at + 2 * k)));
        const float2 y = __half22float2(u32_as_h2(lds32(at + C::kScale + 2 * k)));
        ks[a][k] = x.x, ks[a][k + 1] = x.y;
        vs[a][k] = y.x, vs[a][k + 1] = y.y;
      }
    }

    // S = Q K^T, one accumulator per group, scaled in fp32
    float x[kH][4];  // [head][token]
#pragma unroll
    for (int a = 0; a < kH; ++a) x[a][0] = x[a][1] = x[a][2] = x[a][3] = 0.0f;
#pragma unroll
    for (int k = 0; k < G4; ++k) {
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        uint32_t kw[4];
        pairs(E{}, lds32(st + chunk_at<D>(8 * n + g, k) + 4 * t), kw);
        float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        mma_qk(E{}, acc, qa[k][0], kw[0], kw[1]);
        mma_qk(E{}, acc, qa[k][1], kw[2], kw[3]);
        x[0][2 * n] = fmaf(acc[0], ks[2 * n][k], x[0][2 * n]);
        x[0][2 * n + 1] = fmaf(acc[1], ks[2 * n + 1][k], x[0][2 * n + 1]);
        if constexpr (kWide) {
          x[kH - 1][2 * n] = fmaf(acc[2], ks[2 * n][k], x[kH - 1][2 * n]);
          x[kH - 1][2 * n + 1] = fmaf(acc[3], ks[2 * n + 1][k], x[kH - 1][2 * n + 1]);
        }
      }
    }

    // running softmax; tokens past the sequence's end count for nothing, whatever their bytes hold
    const int left = len - col * kPage;  // > 0
    if (left < kPage) {
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        if (2 * t + (a & 1) + 8 * (a >> 1) >= left) {
#pragma unroll
          for (int hh = 0; hh < kH; ++hh) x[hh][a] = -INFINITY;
#pragma unroll
          for (int k = 0; k < G4; ++k) vs[a][k] = 0.0f;
        }
      }
    }
    float alpha[kH];
    bool moved = false;
#pragma unroll
    for (int hh = 0; hh < kH; ++hh) {
#pragma unroll
      for (int a = 0; a < 4; ++a) x[hh][a] *= p.scale_log2;
      float top = fmaxf(fmaxf(x[hh][0], x[hh][1]), fmaxf(x[hh][2], x[hh][3]));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      top = fmaxf(top, m[hh]);
      const float base = top == -INFINITY ? 0.0f : top;
      alpha[hh] = ex2(m[hh] - base);
      moved |= top != m[hh];
      m[hh] = top;
      float sum = 0.0f;
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        x[hh][a] = ex2(x[hh][a] - base);
        sum += x[hh][a];
      }
      l[hh] = fmaf(l[hh], alpha[hh], sum);
    }
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int j = 0; j < kTiles; ++j) {
        o[j][0] *= alpha[0];
        o[j][1] *= alpha[0];
        o[j][2] *= alpha[kH - 1];
        o[j][3] *= alpha[kH - 1];
      }
    }

    // O += P V
#pragma unroll
    for (int k = 0; k < G4; ++k) {
      uint32_t hi[4], lo[4];  // A registers: (head g | g + 8) x (tokens 2 t, 2 t + 1 | 2 t + 8, 2 t + 9)
#pragma unroll
      for (int hh = 0; hh < kH; ++hh) {
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const float u = x[hh][2 * n] * vs[2 * n][k], v = x[hh][2 * n + 1] * vs[2 * n + 1][k];
          const uint32_t w = Bf16Elem::pack(u, v);
          const float2 r = Bf16Elem::unpack(w);
          hi[2 * n + hh] = w;
          lo[2 * n + hh] = Bf16Elem::pack(u - r.x, v - r.y);
        }
      }
      if constexpr (!kWide) {  // the second terms are rows 8 .. 15
        hi[1] = lo[0];
        hi[3] = lo[2];
      }
      uint32_t w[4];
#pragma unroll
      for (int a = 0; a < 4; ++a)
        w[a] = lds32(st + C::kData + chunk_at<D>(2 * t + (a & 1) + 8 * (a >> 1), k) + 4 * (g & 3));
      const uint32_t v0 = prmt(w[0], w[1], v_sel), v1 = prmt(w[2], w[3], v_sel);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t b0 = nibbles_bf16(v0 >> (4 * j)), b1 = nibbles_bf16(v1 >> (4 * j));
        mma_bf16(o[4 * k + j], hi, b0, b1);
        if constexpr (kWide) mma_bf16(o[4 * k + j], lo, b0, b1);
      }
    }
  }

  // ---- join the warps' partial results ----
  cp_async_wait<0>();
  __syncthreads();  // the rings are free: [warp][head][D] outputs, then [warp][head] (m, l)
  float* part_o = reinterpret_cast<float*>(smem);
  float* part_ml = part_o + kWarps * kHeads * D;
#pragma unroll
  for (int hh = 0; hh < kH; ++hh) {
    l[hh] += __shfl_xor_sync(0xffffffffu, l[hh], 1);
    l[hh] += __shfl_xor_sync(0xffffffffu, l[hh], 2);
    const int head = warp * kHeads + g + 8 * hh;
#pragma unroll
    for (int k = 0; k < G4; ++k) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {  // column 2 t + e of the tiles: dims 32 k + at .. at + 3
        const int n = 2 * t + e;
        float4 v;
        float* f = reinterpret_cast<float*>(&v);
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = kWide ? o[4 * k + j][2 * hh + e] : o[4 * k + j][e] + o[4 * k + j][2 + e];
        *reinterpret_cast<float4*>(part_o + head * D + 32 * k + 8 * (n & 3) + 4 * (n >> 2)) = v;
      }
    }
    if (t == 0) {
      part_ml[2 * head] = m[hh];
      part_ml[2 * head + 1] = l[hh];
    }
  }
  if (splits > 1) cluster_barrier();
  else __syncthreads();
  float* weight = reinterpret_cast<float*>(smem + kWarps * (C::kRing + kStages * 4));  // [head][record]
  const uint32_t o_addr = smem_u32(part_o), ml_addr = smem_u32(part_ml);
  const int records = splits * kWarps;  // at most 32
  for (int head = warp; head < p.group; head += kWarps) {
    float mr = -INFINITY, lr = 0.0f;
    if (lane < records) {
      const uint32_t at = map_to_rank(ml_addr, lane / kWarps) + 8 * ((lane % kWarps) * kHeads + head);
      mr = ld_cluster(at);
      lr = ld_cluster(at + 4);
    }
    float top = mr;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    const float w = ex2(mr - (top == -INFINITY ? 0.0f : top));
    float sum = w * lr;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    weight[head * 32 + lane] = sum == 0.0f ? 0.0f : __fdiv_rn(w, sum);
    if (lane == 0 && split == 0 && p.lse != nullptr)
      p.lse[static_cast<int64_t>(row) * p.group + head] = sum == 0.0f ? -INFINITY : top + log2f(sum);
  }
  __syncthreads();
  uint32_t* out = static_cast<uint32_t*>(p.output) + static_cast<int64_t>(row) * p.group * (D / 2);
  for (int i = split * 32 * kWarps + threadIdx.x; i < p.group * (D / 2); i += splits * 32 * kWarps) {
    const int head = i / (D / 2), d = i % (D / 2) * 2;
    float a = 0.0f, c = 0.0f;
    for (int r = 0; r < records; ++r) {
      const float w = weight[head * 32 + r];
      const uint32_t at = map_to_rank(o_addr, r / kWarps) + 4 * (((r % kWarps) * kHeads + head) * D + d);
      a = fmaf(w, ld_cluster(at), a);
      c = fmaf(w, ld_cluster(at + 4), c);
    }
    out[i] = E::pack(a, c);
  }
  if (splits > 1) cluster_barrier();  // nobody leaves while its memory is read
}

template <typename E, int D, bool kWide>
cudaError_t launch(const SparseParams& p, int64_t rows, int splits, cudaStream_t s) {
  const int bytes = kWarps * (SparseCfg<D>::kRing + kStages * 4) + 16 * 32 * 4;
  const auto fn = sparse_decode_kernel<E, D, kWide>;
  if (bytes > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return e;
  }
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(splits);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(rows * splits));
  cfg.blockDim = dim3(32 * kWarps);
  cfg.dynamicSmemBytes = static_cast<size_t>(bytes);
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = splits > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, fn, p, splits);
}

template <typename E>
cudaError_t launch_any(const SparseParams& p, int head_dim, int64_t rows, int splits, cudaStream_t s) {
  const bool wide = p.group > 8;
  if (head_dim == 128)
    return wide ? launch<E, 128, true>(p, rows, splits, s) : launch<E, 128, false>(p, rows, splits, s);
  return wide ? launch<E, 64, true>(p, rows, splits, s) : launch<E, 64, false>(p, rows, splits, s);
}

}  // namespace
}  // namespace iris

using namespace iris;

extern "C" int iris_b200_int4_sparse_paged_decode(const void* query, const void* k_data, const void* v_data,
                                                  const void* k_scale, const void* v_scale, const int32_t* block_table,
                                                  int64_t block_table_stride, const int32_t* seq_lens,
                                                  const int32_t* page_list, const int32_t* page_count, void* output,
                                                  float* out_lse, int32_t batch, int32_t num_q_heads,
                                                  int32_t num_kv_heads, int32_t head_dim, int64_t num_pages,
                                                  int32_t page_size, int32_t max_pages_per_seq, int32_t max_pages,
                                                  float softmax_scale, int32_t dtype, int32_t* error_word,
                                                  void* stream) {
  if (batch < 0 || num_q_heads <= 0 || num_kv_heads <= 0 || num_pages < 0 || max_pages_per_seq < 0 || max_pages <= 0)
    return IRIS_EINVAL;
  if (num_q_heads % num_kv_heads != 0 || !(softmax_scale > 0.0f)) return IRIS_EINVAL;
  if (dtype != IRIS_DTYPE_FP16 && dtype != IRIS_DTYPE_BF16) return IRIS_EINVAL;
  const int group = num_q_heads / num_kv_heads;
  if (page_size != kPage || (head_dim != 64 && head_dim != 128) || group > 16) return IRIS_EUNSUPPORTED;
  const int64_t rows = static_cast<int64_t>(batch) * num_kv_heads;
  if (rows == 0) return IRIS_OK;
  if (num_pages == 0) return IRIS_EINVAL;
  if (rows > (1 << 27)) return IRIS_EUNSUPPORTED;
  const void* ptrs[] = {query, k_data, v_data, k_scale, v_scale, block_table, seq_lens, page_list, page_count, output};
  for (const void* q : ptrs)
    if (q == nullptr) return IRIS_EINVAL;
  if (!aligned_to(query, 16) || !aligned_to(k_data, 16) || !aligned_to(v_data, 16) || !aligned_to(k_scale, 8) ||
      !aligned_to(v_scale, 8) || !aligned_to(output, 4) || !aligned_to(out_lse, 4))
    return IRIS_EALIGN;
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
  p.scale_log2 = static_cast<float>(static_cast<double>(softmax_scale) * 1.4426950408889634);
  p.err = error_word;
  int splits = 1;
  while (splits < 8 && rows * splits < 444 && max_pages > splits * kWarps) splits *= 2;
  clear_stale_cuda_error();
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = dtype == IRIS_DTYPE_FP16 ? launch_any<Fp16Elem>(p, head_dim, rows, splits, s)
                                                 : launch_any<Bf16Elem>(p, head_dim, rows, splits, s);
  if (e != cudaSuccess) {
    record_cuda_error(e, "sparse_decode_kernel launch");
    return IRIS_ECUDA;
  }
  return IRIS_OK;
}
