// A list of N units in n nearly equal parts, in 32-bit arithmetic: the first N mod n parts have one unit more.
#pragma once

namespace mts {

struct Parts {
  unsigned size, longer;       // units of a part; parts with one more
  __device__ __forceinline__ Parts(int N, int n) : size(unsigned(N) / unsigned(n)), longer(unsigned(N) % unsigned(n)) {}
  __device__ __forceinline__ int begin(int i) const { return int(size * unsigned(i) + min(unsigned(i), longer)); }
  __device__ __forceinline__ int owner(int u) const {
    const unsigned head = longer * (size + 1);
    return int(unsigned(u) < head ? unsigned(u) / (size + 1) : longer + (unsigned(u) - head) / size);
  }
};
// The same for a power of two of parts.
template <int n>
__device__ __forceinline__ int part_begin(int N, int i) { return N / n * i + min(i, N % n); }

}  // namespace mts
