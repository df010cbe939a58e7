// The states of a beam search's slots in their parents' order, in place: slot b W + w takes what slot
// b W + parents[b][w] held before, up to lengths[b] positions.
//
// A thread owns a 16-byte column of a request's slots: it loads the column from every slot that becomes a parent,
// then stores it to their children. Whatever the permutation, nothing is overwritten before it is read, with no
// second buffer, no order of copies and no barrier, and a parent with several children is read once. Slots that
// are their own parent are left alone.
//
// Bound by the HBM: caches of 16 x 4 beams (2.2 GB read and written) 411 us, 5.3 TB/s; matrices of 16 x 8 beams, nearly all
// of which move, 284 us, 5.2 TB/s (a 4 GiB copy reaches 4.78). Steps of 512 columns: of 1024, 434 and 306 us.
#pragma once

#include "common.cuh"

namespace vo {

using namespace vs;

constexpr int kMaxReorderBeams = 32;  // (a parent's children are bits of a word)
constexpr int kReorderThreads = 256;
constexpr int kReorderColumns = 512;  // a workgroup's step
constexpr int kOuterDims = 3;

// One tensor: `rows` (the outer dimensions' product) runs of contiguous bytes a slot. The lengths limit the run
// (length_dim = kOuterDims; `unit` bytes a position), an outer dimension (its index), or nothing (-1).
struct StateDesc {
  char* base;
  int64_t slot_stride;
  int64_t stride[kOuterDims];
  int64_t run;
  int64_t unit;
  int32_t size[kOuterDims];
  int32_t length_dim;
  int32_t max_length;
  int32_t reserved;
};

typedef u32x4_t u32x4_byte_t __attribute__((aligned(1)));
typedef uint32_t u32_byte_t __attribute__((aligned(1)));

template <class T>
__device__ __forceinline__ T ld_col(const char* p) {
  return *(const __attribute__((address_space(1))) T*)p;
}
template <class T>
__device__ __forceinline__ void st_col(char* p, T v) {
  *(__attribute__((address_space(1))) T*)p = v;
}

// A column of type T at p in every slot of the request from slot Q on: loaded from the parents, all the loads ahead of
// the first store, then stored to each one's children (bits of slots; all of it uniform). By recursion: an array that
// a loop fills under conditions stays one value of all its registers to the compiler, copied at each of them.
template <int Q, int WMAX, class T>
__device__ __forceinline__ void move_column(char* p, int64_t slot_stride, const uint32_t* children) {
  if constexpr (Q < WMAX) {
    T v;
    if (children[Q]) v = ld_col<T>(p + Q * slot_stride);
    move_column<Q + 1, WMAX, T>(p, slot_stride, children);
#pragma unroll 1
    for (uint32_t m = children[Q]; m; m &= m - 1) st_col<T>(p + (__ffs(m) - 1) * slot_stride, v);
  }
}

template <int WMAX>
__global__ __launch_bounds__(kReorderThreads) void k_reorder(const StateDesc* descs, const int32_t* parents,
                                                             const int32_t* lengths, int W) {
  const StateDesc& s = as_global(descs)[blockIdx.y];
  const int b = blockIdx.z;
  uint32_t children[WMAX] = {};
  uint32_t moved = 0;
  for (int w = 0; w < W; ++w) {
    const int q = as_global(parents)[b * W + w];
    if (q == w) continue;  // (and of any other value than a slot: the slot keeps its state)
#pragma unroll
    for (int k = 0; k < WMAX; ++k) children[k] |= k < W && q == k ? 1u << w : 0u;
    moved |= q >= 0 && q < W;
  }
  if (!moved) return;
  uint32_t n0 = s.size[0], n1 = s.size[1], n2 = s.size[2];
  int64_t run = s.run;
  if (s.length_dim >= 0) {
    int len = as_global(lengths)[b];
    len = len < 0 ? 0 : (len < s.max_length ? len : s.max_length);
    if (s.length_dim == kOuterDims) run = len * s.unit;
    if (s.length_dim == 0) n0 = len;
    if (s.length_dim == 1) n1 = len;
    if (s.length_dim == 2) n2 = len;
  }
  const uint32_t cols = static_cast<uint32_t>((run + 15) >> 4);  // columns a run
  const uint32_t rows = n0 * n1 * n2;
  const uint32_t all = rows * cols;
  char* base = as_global(s.base) + static_cast<int64_t>(b) * W * s.slot_stride;
#pragma unroll 1
  for (uint32_t t = blockIdx.x * kReorderColumns; t < all; t += gridDim.x * kReorderColumns) {
#pragma unroll 1
    for (uint32_t i = t + threadIdx.x; i < min(t + kReorderColumns, all); i += kReorderThreads) {
      uint32_t row = 0, col = i;
      int64_t off = 0;
      if (rows > 1) {  // (uniform)
        row = i / cols;
        col = i - row * cols;
        uint32_t i0 = row / (n1 * n2);
        row -= i0 * (n1 * n2);
        const uint32_t i1 = row / n2;
        off = i0 * s.stride[0] + i1 * s.stride[1] + (row - i1 * n2) * s.stride[2];
      }
      char* p = base + off + (static_cast<int64_t>(col) << 4);
      const int64_t left = run - (static_cast<int64_t>(col) << 4);
      if (left >= 16) {
        move_column<0, WMAX, u32x4_byte_t>(p, s.slot_stride, children);
      } else {  // (a run's end)
        int k = 0;
#pragma unroll 1
        for (; k + 4 <= left; k += 4) move_column<0, WMAX, u32_byte_t>(p + k, s.slot_stride, children);
#pragma unroll 1
        for (; k < left; ++k) move_column<0, WMAX, uint8_t>(p + k, s.slot_stride, children);
      }
    }
  }
}

}  // namespace vo
