// The cache kept to a budget: iris_b200_int4_paged_evict.
//
// A (sequence, KV head) with more than `budget` tokens keeps its first
// `sink`, its last `recent` and, of those between, the heaviest (ties to the
// lowest index; NaN counts as +inf).  Order matters to nothing in attention but
// recency, so few rows move: kept tokens in front of heavy = budget - recent
// stay, the kept ones behind fill the holes there, both in rising order, and
// the last `recent` follow in order.
//
// One thread-block cluster a (sequence, KV head), each block a run of its
// tokens: weights are read once into shared memory as keys whose order is that
// of unsigned numbers; three histograms over the cluster (11, 11 and 10 bits)
// find the lightest key that stays; ranks by block scans and the cluster's
// counts; rows are copied by the whole cluster between its barriers.
#include <cooperative_groups.h>

#include "varlen_common.cuh"

namespace iris {
namespace {

namespace cg = cooperative_groups;

constexpr int kEvictThreads = 512;
constexpr int kEvictWarps = kEvictThreads / 32;
constexpr int kBins = 2048;
constexpr int kMostKeys = 40960;  // keys of a block that stay in shared memory

struct EvictParams {
  uint8_t *k_data, *v_data, *k_scale, *v_scale;
  float* mass;
  const int32_t* block_table;
  int64_t bt_stride;
  const int32_t* seq_lens;
  int32_t* new_lens;
  int32_t* kept;     // [batch, hkv, budget] or NULL
  int32_t* late;     // workspace [batch * hkv][2][budget - recent]: tokens that move, places they move to
  int32_t* err;
  int64_t num_pages;
  int32_t batch, hkv, max_pages, budget, sink, recent;
  int32_t keys;      // keys of a block in shared memory
};

// The order of weights as that of unsigned numbers; -0 is 0, NaN is +inf.
IRIS_DEV uint32_t weight_key(float w) {
  if (w != w) w = __int_as_float(0x7f800000);
  const uint32_t u = __float_as_uint(w + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

struct EvictShared {
  alignas(16) uint32_t bins[3][kBins];
  int32_t warp_sums[kEvictWarps];
  int32_t equal, moving, holes;  // of this block's run
  int32_t bad;                   // a page id outside the cache
  uint32_t pick[2];              // this round's bin, and how many keys above it stay in question
};

// Exclusive sum over the block and its total.
IRIS_DEV int block_scan(int v, int32_t* sums, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();  // sums of the call before are read
  if (lane == 31) sums[warp] = x;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < kEvictWarps; ++i) {
    const int s = sums[i];
    before += i < warp ? s : 0;
    all += s;
  }
  *total = all;
  return before + x - v;
}

template <int D>
struct EvictRow {
  static constexpr int kVectors = D / 32;  // 16-byte vectors of packed keys (or values)
  static constexpr int kLanes = 2 * kVectors;  // threads that carry a row
};

// This thread's part of a row: a vector of the packed data, a scale pair or the weight.
struct Part {
  uint4 data;
  uint2 scale;
  float mass;
};
template <int D>
IRIS_DEV Part read_part(const EvictParams& p, int64_t row, int h, int sub) {
  constexpr int kV = EvictRow<D>::kVectors;
  const int64_t r = row * p.hkv + h;
  const bool value = sub >= kV;
  Part x;
  x.data = *reinterpret_cast<const uint4*>((value ? p.v_data : p.k_data) + r * (D / 2) + (sub % kV) * 16);
  x.scale = make_uint2(0, 0);
  if (sub % kV == 0) {
    const uint8_t* s = (value ? p.v_scale : p.k_scale) + r * (D / 16);
    if constexpr (D == 128)
      x.scale = *reinterpret_cast<const uint2*>(s);
    else
      x.scale.x = *reinterpret_cast<const uint32_t*>(s);
  }
  x.mass = sub == 1 ? p.mass[(row / kTokPage * p.hkv + h) * kTokPage + row % kTokPage] : 0.0f;
  return x;
}
template <int D>
IRIS_DEV void write_part(const EvictParams& p, int64_t row, int h, int sub, const Part& x) {
  constexpr int kV = EvictRow<D>::kVectors;
  const int64_t r = row * p.hkv + h;
  const bool value = sub >= kV;
  *reinterpret_cast<uint4*>((value ? p.v_data : p.k_data) + r * (D / 2) + (sub % kV) * 16) = x.data;
  if (sub % kV == 0) {
    uint8_t* s = (value ? p.v_scale : p.k_scale) + r * (D / 16);
    if constexpr (D == 128)
      *reinterpret_cast<uint2*>(s) = x.scale;
    else
      *reinterpret_cast<uint32_t*>(s) = x.scale.x;
  }
  if (sub == 1) p.mass[(row / kTokPage * p.hkv + h) * kTokPage + row % kTokPage] = x.mass;
}

template <int D>
__global__ void __launch_bounds__(kEvictThreads, 2) evict_kernel(const EvictParams p) {
  extern __shared__ uint32_t keys[];
  __shared__ EvictShared sh;
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = static_cast<int>(cluster.block_rank()), size = static_cast<int>(cluster.num_blocks());
  const int pair = blockIdx.x / size, b = pair / p.hkv, h = pair % p.hkv;
  const int tid = threadIdx.x;
  grid_dependency_wait();
  grid_dependents_launch();
  const int32_t raw = __ldg(p.seq_lens + b);
  const bool wrong = raw < 0 || (static_cast<int64_t>(raw) + kTokPage - 1) / kTokPage > p.max_pages;
  if (tid == 0 && rank == 0 && h == 0) {
    if (raw < 0) set_error(p.err, IRIS_ERR_SEQ_NEGATIVE);
    else if (wrong) set_error(p.err, IRIS_ERR_BLOCK_TABLE);
  }
  const int len = wrong ? 0 : raw, budget = p.budget;
  int32_t* kept = p.kept != nullptr ? p.kept + static_cast<int64_t>(pair) * budget : nullptr;
  const int32_t* table = p.block_table + b * p.bt_stride;
  auto row_of = [&](int j) { return static_cast<int64_t>(__ldg(table + j / kTokPage)) * kTokPage + j % kTokPage; };

  // a block's run of tokens: whole pages
  const int pages = (len + kTokPage - 1) / kTokPage;
  const int j0 = static_cast<int>(static_cast<int64_t>(pages) * rank / size) * kTokPage;
  const int j1 = min(len, static_cast<int>(static_cast<int64_t>(pages) * (rank + 1) / size) * kTokPage);
  auto meet = [&] {  // of the cluster's blocks
    if (size == 1) __syncthreads(); else cluster.sync();
  };
  auto stay = [&](bool bad) {  // nothing to do, or nothing that may be touched
    if (kept != nullptr)
      for (int i = rank * kEvictThreads + tid; i < budget; i += size * kEvictThreads) kept[i] = i < len ? i : -1;
    if (tid == 0 && rank == 0 && h == 0) p.new_lens[b] = wrong || bad ? raw : len;
  };
  auto id_ok = [&](int32_t id) { return static_cast<uint32_t>(id) < static_cast<uint32_t>(p.num_pages); };
  if (len <= budget) {
    bool bad = false;  // (page ids are looked at all the same)
    for (int c = j0 / kTokPage + tid; c * kTokPage < j1; c += kEvictThreads) bad |= !id_ok(__ldg(table + c));
    if (bad) set_error(p.err, IRIS_ERR_PAGE_ID);
    stay(false);
    return;
  }
  if (tid == 0) sh.bad = 0;
  for (int i = tid; i < 3 * kBins; i += kEvictThreads) (&sh.bins[0][0])[i] = 0;
  __syncthreads();
  const int sink = p.sink, recent = p.recent, heavy = budget - recent, last = len - recent;
  const int want = heavy - sink;  // tokens of [sink, last) that stay
  const bool cached = j1 - j0 <= p.keys;
  auto key_at = [&](int j) {
    return cached ? keys[j - j0]
                  : weight_key(p.mass[(static_cast<int64_t>(__ldg(table + j / kTokPage)) * p.hkv + h) * kTokPage + j % kTokPage]);
  };
  const int c0 = max(j0, sink), c1 = min(j1, last);  // this block's tokens in question
  // the weights' keys, their first histogram, and a look at every page id
#pragma unroll 4
  for (int j = j0 + 4 * tid; j < j1; j += 4 * kEvictThreads) {
    const int32_t id = __ldg(table + j / kTokPage);
    if (!id_ok(id)) {
      set_error(p.err, IRIS_ERR_PAGE_ID);
      sh.bad = 1;
      continue;
    }
    const float4 w =
        *reinterpret_cast<const float4*>(p.mass + (static_cast<int64_t>(id) * p.hkv + h) * kTokPage + j % kTokPage);
    const uint32_t k4[4] = {weight_key(w.x), weight_key(w.y), weight_key(w.z), weight_key(w.w)};
    if (cached) *reinterpret_cast<uint4*>(keys + (j - j0)) = make_uint4(k4[0], k4[1], k4[2], k4[3]);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (j + i >= c0 && j + i < c1) atomicAdd(&sh.bins[0][k4[i] >> 21], 1u);
  }
  meet();
  bool bad = false;
  for (int r = 0; r < size; ++r) bad |= *cluster.map_shared_rank(&sh.bad, r) != 0;
  if (bad) {  // the sequence stays as it is (its other heads see the same pages)
    stay(true);
    meet();
    return;
  }
  if (tid == 0 && rank == 0 && h == 0) p.new_lens[b] = budget;
  // the lightest key that stays: `low`, of which the first `ties` in the cluster's order stay
  uint32_t low = 0;
  int ties = 0;
  if (want > 0) {
    int left = want;  // keys at or above the prefix found so far that still have to be picked
#pragma unroll 1
    for (int round = 0; round < 3; ++round) {
      const int shift = round == 0 ? 21 : round == 1 ? 10 : 0, width = round == 2 ? 10 : 11;
      uint32_t* bins = sh.bins[round];
      if (round > 0) {
        for (int j = c0 + tid; j < c1; j += kEvictThreads) {
          const uint32_t key = key_at(j);
          if ((key >> (shift + width)) == (low >> (shift + width)))
            atomicAdd(&bins[(key >> shift) & ((1u << width) - 1)], 1u);
        }
        meet();
      }
      // from the top bin down: four bins a thread, summed over the cluster
      constexpr int kEach = kBins / kEvictThreads;
      static_assert(kEach == 4, "a thread's bins are one load");
      int n[kEach] = {}, mine = 0;
      for (int r = 0; r < size; ++r) {
        const uint4 v = reinterpret_cast<const uint4*>(cluster.map_shared_rank(bins, r))[kBins / kEach - 1 - tid];
        n[0] += static_cast<int>(v.w);
        n[1] += static_cast<int>(v.z);
        n[2] += static_cast<int>(v.y);
        n[3] += static_cast<int>(v.x);
      }
#pragma unroll
      for (int i = 0; i < kEach; ++i) mine += n[i];
      int total, above = block_scan(mine, sh.warp_sums, &total);
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        if (above < left && left <= above + n[i]) {
          sh.pick[0] = kBins - 1 - (tid * kEach + i);
          sh.pick[1] = left - above;
        }
        above += n[i];
      }
      __syncthreads();
      low |= sh.pick[0] << shift;
      left = static_cast<int>(sh.pick[1]);
      __syncthreads();
    }
    ties = left;
  }
  // how many of a block's tokens have that key: ties go to the lowest index
  int count = 0, total;
  for (int j = c0 + tid; want > 0 && j < c1; j += kEvictThreads) count += key_at(j) == low;
  block_scan(count, sh.warp_sums, &total);
  if (tid == 0) sh.equal = total;
  meet();
  int equal_before = 0;
  for (int r = 0; r < rank; ++r) equal_before += *cluster.map_shared_rank(&sh.equal, r);
  // ranks: a thread takes `each` tokens in a row, in whole sweeps of the block
  constexpr int kEach = 8;
  auto chosen = [&](uint32_t key, int equal_rank) { return want > 0 && (key > low || (key == low && equal_rank < ties)); };
  int32_t* moving = p.late + static_cast<int64_t>(pair) * 2 * heavy;
  int32_t* holes = moving + heavy;
  // twice over the run: the counts first, then the lists at the places the counts of the blocks before give (once where
  // one sweep is the whole run: what the first time found is still there)
  const bool once = c1 - c0 <= kEvictThreads * kEach;
  int move_at = 0, hole_at = 0, both = 0;  // (counts of a sweep: moves below, holes above 16 bits)
  uint32_t in = 0;
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {
    int equal_at = equal_before, moves = 0, gaps = 0, before_m = 0, before_g = 0;
    for (int s = c0; s < c1; s += kEvictThreads * kEach) {
      const int a = s + tid * kEach, e = min(a + kEach, c1);
      if (pass == 0 || !once) {
        uint32_t key[kEach];
        int equals = 0;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
          key[i] = a + i < e && want > 0 ? key_at(a + i) : 0u;
          equals += a + i < e && key[i] == low && want > 0;
        }
        int all;
        int eq = equal_at + block_scan(equals, sh.warp_sums, &all);
        equal_at += all;
        int mine = 0;
        in = 0;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
          if (a + i >= e) continue;
          const bool yes = chosen(key[i], eq);
          eq += key[i] == low && want > 0;
          in |= static_cast<uint32_t>(yes) << i;
          mine += (yes && a + i >= heavy) + ((!yes && a + i < heavy) << 16);
        }
        both = block_scan(mine, sh.warp_sums, &all);
        before_m = moves;
        before_g = gaps;
        moves += all & 0xffff;
        gaps += all >> 16;
      }
      if (pass == 1) {
        int m = move_at + before_m + (both & 0xffff), g = hole_at + before_g + (both >> 16);
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
          if (a + i >= e) continue;
          const bool yes = (in >> i) & 1u;
          if (yes && a + i >= heavy) moving[m++] = a + i;
          if (!yes && a + i < heavy) holes[g++] = a + i;
          if (yes && a + i < heavy && kept != nullptr) kept[a + i] = a + i;
        }
      }
    }
    if (pass == 0) {
      if (tid == 0) {
        sh.moving = moves;
        sh.holes = gaps;
      }
      meet();
      for (int r = 0; r < rank; ++r) {
        move_at += *cluster.map_shared_rank(&sh.moving, r);
        hole_at += *cluster.map_shared_rank(&sh.holes, r);
      }
    }
  }
  int n = 0;
  for (int r = 0; r < size; ++r) n += *cluster.map_shared_rank(&sh.moving, r);
  if (kept != nullptr) {
    for (int i = rank * kEvictThreads + tid; i < sink; i += size * kEvictThreads) kept[i] = i;
    for (int i = rank * kEvictThreads + tid; i < recent; i += size * kEvictThreads) kept[heavy + i] = last + i;
  }
  if (size > 1) __threadfence();
  meet();

  // kept tokens from behind into the holes: sources and targets do not meet
  constexpr int kLanes = EvictRow<D>::kLanes, kRows = kEvictThreads / kLanes;
  const int sub = tid % kLanes, unit = rank * kRows + tid / kLanes;
  constexpr int kDeep = 4;
#pragma unroll 1
  for (int i0 = unit; i0 < n; i0 += kDeep * size * kRows) {
    int src[kDeep], dst[kDeep];
    Part x[kDeep];
#pragma unroll
    for (int d = 0; d < kDeep; ++d) {
      const int i = i0 + d * size * kRows;
      src[d] = i < n ? __ldcg(moving + i) : -1;
      dst[d] = i < n ? __ldcg(holes + i) : 0;
    }
#pragma unroll
    for (int d = 0; d < kDeep; ++d)
      if (src[d] >= 0) x[d] = read_part<D>(p, row_of(src[d]), h, sub);
#pragma unroll
    for (int d = 0; d < kDeep; ++d) {
      if (src[d] < 0) continue;
      write_part<D>(p, row_of(dst[d]), h, sub, x[d]);
      if (sub == 0 && kept != nullptr) kept[dst[d]] = src[d];
    }
  }
  // then the recent ones, in steps: all of a step's rows are read before any is written, and a step's targets lie at
  // or before its own sources, so no later step reads what it wrote
#pragma unroll 1
  for (int i0 = 0; i0 < recent; i0 += size * kRows * kDeep) {
    meet();  // what this step overwrites has been read
    Part x[kDeep];
#pragma unroll
    for (int d = 0; d < kDeep; ++d) {
      const int i = i0 + d * size * kRows + unit;
      if (i < recent) x[d] = read_part<D>(p, row_of(last + i), h, sub);
    }
    meet();
#pragma unroll
    for (int d = 0; d < kDeep; ++d) {
      const int i = i0 + d * size * kRows + unit;
      if (i < recent) write_part<D>(p, row_of(heavy + i), h, sub, x[d]);
    }
  }
  meet();  // (no block leaves while another reads its shared memory)
}

// Blocks of a cluster: enough for two an SM, each with 1024 tokens or more.
int cluster_of(int64_t pairs, int64_t most_tokens) {
  int size = 1;
  while (size < 8 && pairs * size * 2 <= 296 && most_tokens / (size * 2) >= 1024) size *= 2;
  return size;
}

template <int D>
cudaError_t launch_evict(EvictParams p, cudaStream_t stream) {
  const int64_t pairs = static_cast<int64_t>(p.batch) * p.hkv, tokens = static_cast<int64_t>(p.max_pages) * kTokPage;
  const int size = cluster_of(pairs, tokens);
  const int64_t run = ((p.max_pages + size - 1) / size) * static_cast<int64_t>(kTokPage);
  p.keys = static_cast<int32_t>(run < kMostKeys ? run : kMostKeys);
  const size_t smem = static_cast<size_t>(p.keys) * 4;
  const cudaError_t e = cudaFuncSetAttribute(evict_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostKeys * 4);
  if (e != cudaSuccess) return e;
  return launch_early_clusters(evict_kernel<D>, dim3(static_cast<unsigned>(pairs * size)), dim3(kEvictThreads),
                               static_cast<unsigned>(size), smem, stream, p);
}

// Bytes that an argument covers.
struct Range {
  const void* at;
  uint64_t bytes;
  bool meets(const Range& o) const {
    const uintptr_t a = reinterpret_cast<uintptr_t>(at), b = reinterpret_cast<uintptr_t>(o.at);
    return bytes > 0 && o.bytes > 0 && (a < b ? b - a < bytes : a - b < o.bytes);
  }
};

}  // namespace
}  // namespace iris

using namespace iris;

extern "C" size_t iris_b200_evict_workspace_bytes(int32_t batch, int32_t num_kv_heads, int32_t budget, int32_t recent_tokens) {
  if (batch <= 0 || num_kv_heads <= 0 || budget <= recent_tokens) return 0;
  return static_cast<size_t>(batch) * num_kv_heads * 2 * (budget - recent_tokens) * 4;
}

extern "C" int iris_b200_int4_paged_evict(void* k_data, void* v_data, void* k_scale, void* v_scale, float* mass,
                                          const int32_t* block_table, int64_t block_table_stride, const int32_t* seq_lens,
                                          int32_t* new_lens, int32_t* kept, int32_t batch, int32_t num_kv_heads,
                                          int32_t head_dim, int64_t num_pages, int32_t page_size, int32_t max_pages_per_seq,
                                          int32_t budget, int32_t sink_tokens, int32_t recent_tokens, void* workspace,
                                          size_t workspace_bytes, int32_t* error_word, void* stream) {
  if (batch < 0 || num_kv_heads <= 0 || budget <= 0 || sink_tokens < 0 || recent_tokens < 0 || sink_tokens > budget ||
      recent_tokens > budget - sink_tokens)
    return IRIS_EINVAL;
  if (page_size != kTokPage || (head_dim != 64 && head_dim != 128)) return IRIS_EUNSUPPORTED;
  if (batch == 0) return IRIS_OK;
  if (num_pages <= 0 || max_pages_per_seq <= 0) return IRIS_EINVAL;
  if (k_data == nullptr || v_data == nullptr || k_scale == nullptr || v_scale == nullptr || mass == nullptr ||
      block_table == nullptr || seq_lens == nullptr || new_lens == nullptr)
    return IRIS_EINVAL;
  if (num_pages > INT32_MAX || max_pages_per_seq > INT32_MAX / 2 / kTokPage ||
      static_cast<int64_t>(batch) * num_kv_heads > INT32_MAX / 8)
    return IRIS_EUNSUPPORTED;
  if (!aligned_to(k_data, 16) || !aligned_to(v_data, 16) || !aligned_to(k_scale, 8) || !aligned_to(v_scale, 8) ||
      !aligned_to(mass, 16))
    return IRIS_EALIGN;
  // (a table that holds no more than the budget has nothing to move)
  const size_t need = budget >= max_pages_per_seq * kTokPage
                          ? 0 : iris_b200_evict_workspace_bytes(batch, num_kv_heads, budget, recent_tokens);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) return IRIS_EWORKSPACE;
  if (!aligned_to(workspace, 4)) return IRIS_EALIGN;
  // Clusters of other heads read lengths and tables after the first has written: neither output may lie in what is read,
  // or in the other one.
  const uint64_t heads = num_kv_heads, rows = static_cast<uint64_t>(num_pages) * kTokPage * heads, sequences = batch;
  const uint64_t table = (sequences - 1) * static_cast<uint64_t>(block_table_stride > 0 ? block_table_stride : 0) + max_pages_per_seq;
  const Range read[] = {{seq_lens, sequences * 4}, {block_table, table * 4}, {mass, rows * 4},
                        {k_data, rows * (head_dim / 2)}, {v_data, rows * (head_dim / 2)}, {k_scale, rows * (head_dim / 16)},
                        {v_scale, rows * (head_dim / 16)}, {workspace, need}};
  const Range lens_out = {new_lens, sequences * 4}, kept_out = {kept, kept != nullptr ? sequences * heads * budget * 4 : 0};
  if (lens_out.meets(kept_out)) return IRIS_EINVAL;
  for (const Range& r : read)
    if (lens_out.meets(r) || kept_out.meets(r)) return IRIS_EINVAL;
  EvictParams p = {};
  p.k_data = static_cast<uint8_t*>(k_data);
  p.v_data = static_cast<uint8_t*>(v_data);
  p.k_scale = static_cast<uint8_t*>(k_scale);
  p.v_scale = static_cast<uint8_t*>(v_scale);
  p.mass = mass;
  p.block_table = block_table;
  p.bt_stride = block_table_stride;
  p.seq_lens = seq_lens;
  p.new_lens = new_lens;
  p.kept = kept;
  p.late = static_cast<int32_t*>(workspace);
  p.err = error_word;
  p.num_pages = num_pages;
  p.batch = batch;
  p.hkv = num_kv_heads;
  p.max_pages = max_pages_per_seq;
  p.budget = budget;
  p.sink = sink_tokens;
  p.recent = recent_tokens;
  clear_stale_cuda_error();
  const cudaError_t e = head_dim == 128 ? launch_evict<128>(p, static_cast<cudaStream_t>(stream))
                                        : launch_evict<64>(p, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return record_cuda_error(e, "evict"), IRIS_ECUDA;
  return IRIS_OK;
}
