// A line of tiles cut into equal stretches: the numbers alone, for the kernels and for the host.
#pragma once

#include <stdint.h>

namespace vpg {

struct Stretches {
  int units, heads;  // tiles of a head's line; the heads' lines lie one behind the other
  int count, per;    // stretches there is room for, tiles of each
};

__host__ __device__ inline Stretches cut(int units, int heads, int count, int least) {
  const int64_t all = static_cast<int64_t>(units) * heads + count - 1;
  const int per = all >> 31 ? static_cast<int>(all / count) : static_cast<int>(all) / count;
  return {units, heads, count, per > least ? per : least};
}

// Whether 32 bits hold where every stretch begins: those of numbers below count begin at most count * least behind the line.
__host__ __device__ inline bool small(const Stretches& s) { return static_cast<int64_t>(s.units) * s.heads < 1ll << 30; }

// Whether stretch w begins within the line. (Callers ask for numbers far behind the last one: count refuses them, their
// product with per may have passed 2^31.)
template <class Index>
__host__ __device__ inline bool begins(const Stretches& s, int w) {
  return w < s.count && static_cast<Index>(w) * s.per < static_cast<Index>(s.units) * s.heads;
}

}  // namespace vpg
