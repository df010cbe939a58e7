// Rows of logits in segments held in registers, for the operators over whole vocabularies.
#pragma once

#include "common.cuh"

namespace vo {

using namespace vs;

constexpr float kLog2e = 1.44269504088896341f;

__device__ __forceinline__ bool finite_f(float x) { return fabsf(x) < __builtin_inff(); }

// One v_maximum3_f32: a NaN is the result of any NaN. (fmaxf costs an instruction more for each operand that may be
// a signalling NaN.)
__device__ __forceinline__ float max3_nan(float x, float y, float z) {
  return __builtin_elementwise_maximum(__builtin_elementwise_maximum(x, y), z);
}
__device__ __forceinline__ float max_nan(float x, float y) { return __builtin_elementwise_maximum(x, y); }

// One 16-byte vector's elements as fp32.
template <class Tin>
struct Vec;
template <>
struct Vec<uint16_t> {
  static constexpr int kElems = 8;
  static constexpr uint32_t kNegInf = 0xFF80FF80u;
  static __device__ __forceinline__ void unpack(const uint4& d, float* x) {
    const uint32_t w[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[2 * j] = __uint_as_float(w[j] << 16);
      x[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
    }
  }
  // The same by byte permutes: to the compiler other values, which it does not keep from an earlier unpack on.
  static __device__ __forceinline__ void unpack_again(const uint4& d, float* x) {
    const uint32_t w[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[2 * j] = __uint_as_float(__builtin_amdgcn_perm(w[j], 0u, 0x05040C0Cu));
      x[2 * j + 1] = __uint_as_float(__builtin_amdgcn_perm(w[j], 0u, 0x07060C0Cu));
    }
  }
  // The largest element; NaN if there is one.
  static __device__ __forceinline__ float largest(const uint4& d) {
    float x[kElems];
    unpack(d, x);
    return max3_nan(max3_nan(x[0], x[1], x[2]), max3_nan(x[3], x[4], x[5]), max_nan(x[6], x[7]));
  }
};
template <>
struct Vec<float> {
  static constexpr int kElems = 4;
  static constexpr uint32_t kNegInf = 0xFF800000u;
  static __device__ __forceinline__ void unpack(const uint4& d, float* x) {
    x[0] = __uint_as_float(d.x);
    x[1] = __uint_as_float(d.y);
    x[2] = __uint_as_float(d.z);
    x[3] = __uint_as_float(d.w);
  }
  static __device__ __forceinline__ void unpack_again(const uint4& d, float* x) { unpack(d, x); }
  static __device__ __forceinline__ float largest(const uint4& d) {
    float x[kElems];
    unpack(d, x);
    return max_nan(max3_nan(x[0], x[1], x[2]), x[3]);
  }
};

// Element h of a word, and the word with -inf in its place (E elements a vector: two or one a word).
template <int E>
__device__ __forceinline__ float word_value(uint32_t w, int h) {
  return __uint_as_float(E == 4 ? w : h ? w & 0xFFFF0000u : w << 16);
}
template <int E>
__device__ __forceinline__ uint32_t strike_word(uint32_t w, int h) {
  return E == 4 ? 0xFF800000u : h ? (w & 0xFFFFu) | 0xFF800000u : (w & 0xFFFF0000u) | 0xFF80u;
}

// New registers to the compiler: it unpacks a vector again in the next pass rather than keep its elements.
template <int NV>
__device__ __forceinline__ void forget(uint4* d) {
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    u32x4_t v = __builtin_bit_cast(u32x4_t, d[j]);
    asm volatile("" : "+v"(v));
    d[j] = make_uint4(v.x, v.y, v.z, v.w);
  }
}

// NV vectors a thread of the segment that starts at element `first`: vector j of thread t holds the elements
// from first + (j * threads + t) * kElems. What lies past V reads as -inf.
template <class Tin, int NV, int THREADS>
__device__ __forceinline__ void load_segment(const Tin* row, int V, int first, uint4* d) {
  constexpr int E = Vec<Tin>::kElems;
  const int at = first + static_cast<int>(threadIdx.x) * E;
  if (first + NV * THREADS * E <= V) {  // (uniform)
#pragma unroll
    for (int j = 0; j < NV; ++j) d[j] = ld_row16(row + at + j * THREADS * E);
    return;
  }
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int i = at + j * THREADS * E;
    uint4 v = make_uint4(Vec<Tin>::kNegInf, Vec<Tin>::kNegInf, Vec<Tin>::kNegInf, Vec<Tin>::kNegInf);
    if (i + E <= V) {
      v = ld_row16(row + i);
    } else if (i < V) {  // (the row's last vector)
      uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if (i + e >= V) continue;
        if constexpr (sizeof(Tin) == 2) {
          const uint32_t h = ld_global(reinterpret_cast<const uint16_t*>(row) + i + e);
          w[e >> 1] = (e & 1) ? (w[e >> 1] & 0xFFFFu) | (h << 16) : (w[e >> 1] & 0xFFFF0000u) | h;
        } else {
          w[e] = __float_as_uint(ld_global(reinterpret_cast<const float*>(row) + i + e));
        }
      }
      v = make_uint4(w[0], w[1], w[2], w[3]);
    }
    d[j] = v;
  }
}

__device__ __forceinline__ float wave_max_f(float x) {
  return dpp::reduce(x, [](float p, float q) { return fmaxf(p, q); });
}

}  // namespace vo
