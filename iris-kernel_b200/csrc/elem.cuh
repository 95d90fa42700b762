// The two 16-bit element types of keys, values and queries, behind one
// interface: pairs packed in a 32-bit word, converted to and from fp32.
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"

namespace iris {

struct Fp16Elem {
  static constexpr bool kFp16 = true;
  IRIS_DEV static float2 unpack(uint32_t w) { return __half22float2(u32_as_h2(w)); }
  IRIS_DEV static uint32_t pack(float lo, float hi) { return h2_as_u32(__floats2half2_rn(lo, hi)); }
};

struct Bf16Elem {
  static constexpr bool kFp16 = false;
  IRIS_DEV static float2 unpack(uint32_t w) {  // a bf16 is the upper half of its fp32
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  IRIS_DEV static uint32_t pack(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
};

// Signed nibble i (0..7) of a packed word.
IRIS_DEV int nibble(uint32_t w, int i) { return static_cast<int>(w << (28 - 4 * i)) >> 28; }

// Launches a kernel that may come up while the kernel before it in the stream
// drains (a programmatic dependent launch).  The kernel calls
// grid_dependency_wait() before it reads or writes anything; a kernel that
// itself lets a second one come up early does so after that wait, so that the
// second one, too, finds what came before both.
template <typename... P, typename... A>
cudaError_t launch_early_clusters(void (*fn)(P...), dim3 grid, dim3 block, unsigned cluster, size_t smem,
                                  cudaStream_t stream, A&&... args) {
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, fn, static_cast<A&&>(args)...);
}
template <typename... P, typename... A>
cudaError_t launch_early(void (*fn)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, A&&... args) {
  return launch_early_clusters(fn, grid, block, 1, smem, stream, static_cast<A&&>(args)...);
}

inline bool aligned_to(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

}  // namespace iris
