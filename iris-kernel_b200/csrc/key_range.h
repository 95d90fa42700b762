// The range of keys that the threshold of a selection lies in, and the
// 256 bins over it that one round of the search counts.  Plain integers, the
// same on the host and on the GPU.
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define IRIS_HOST_DEV __host__ __device__ __forceinline__
#else
#define IRIS_HOST_DEV inline
#endif

namespace iris {

// A round leaves at most 2^24, 2^16, 2^8 and then one key of the range.
constexpr int kRangeRounds = 4;

struct KeyRange {
  uint32_t low, high;  // both of them in it; low <= high

  IRIS_HOST_DEV bool holds(uint32_t key) const { return key - low <= high - low; }
  // A bin is 2^shift keys wide, with the smallest shift whose 256 bins reach from high to low.
  IRIS_HOST_DEV uint32_t bin(uint32_t key, int shift) const { return (high - key) >> shift; }
  // To the keys of one of its bins, counted from the top.  The last bin ends at
  // low, which may be nearer to 0 than a bin is wide: nothing is subtracted past it.
  IRIS_HOST_DEV void narrow(uint32_t index, int shift) {
    high -= index << shift;
    const uint32_t width = (1u << shift) - 1u;
    if (high - low > width) low = high - width;
  }
};

}  // namespace iris
