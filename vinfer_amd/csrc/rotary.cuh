// Rotation of queries and keys by their positions, and keys and values into their slots.
//
// Pair (x1, x2) of a token at position p turns by a = p f_j:
//   y1 = m (x1 cos a - x2 sin a), y2 = m (x2 cos a + x1 sin a)
// a is taken in 64 bits and brought to turns there (a / 2 pi less its nearest whole number), so that its sine and
// cosine are right to fp32 at any position. Each element is read and written once, products and sums are fp32, and
// the result is rounded once to the elements' type. Bound by HBM for many tokens, by latency for few: the angles of a
// workgroup's tokens are worked out once, in LDS, for all heads.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace vpg {

template <class T>
struct alignas(16) Vec8 {
  T x[8];
};

// Division by a number known to the host: floor(n / d) for n < 2^31.
struct Div {
  uint32_t mul;
  int shift, d;
};
__device__ __forceinline__ int div_of(int n, Div v) {
  return v.d == 1 ? n : static_cast<int>(__umulhi(static_cast<uint32_t>(n), v.mul) >> v.shift);
}

struct RotateArgs {
  const void *q, *k, *v;
  int64_t q_stride, k_stride, v_stride, q_head, k_head, v_head;
  void *out_q, *k_pages, *v_pages;
  int64_t page_stride, place_stride, head_stride;
  const int32_t *positions, *slots;
  const double* freq;
  float magnitude;
  int N, heads, kv_heads, D, dim;
  int64_t n_slots;
  int shift;
  int tokens;  // of a workgroup
  int items;   // of a token
  Div per_head, tail;  // items of a query's or key's head, of a value's
};

constexpr int kRotateThreads = 256;
constexpr int kRotateTokens = 4;  // of a workgroup, at most

// E: elements of an access, 8 (all addresses are multiples of 16 bytes, and halves' pairs lie in whole vectors) or 1.
// An item is, of queries and keys, where pairs lie in halves: E pairs of the turned part, or E elements of the rest;
// else E elements of a head.
template <class T, int E, bool INTERLEAVED>
__global__ __launch_bounds__(kRotateThreads) void k_rotate(RotateArgs a) {
  __shared__ float2 s_turn[kRotateTokens][128];
  __shared__ int s_pos[kRotateTokens], s_slot[kRotateTokens];
  const int tid = threadIdx.x;
  const int token0 = blockIdx.x * a.tokens, n = min(a.tokens, a.N - token0), half = a.dim / 2;
  if (tid < n) {
    s_pos[tid] = a.positions[token0 + tid];
    s_slot[tid] = a.slots[token0 + tid];
  }
  for (int i = tid; i < n * half; i += kRotateThreads) {
    const int t = i / half, j = i - t * half;
    const double turns = a.positions[token0 + t] * a.freq[j] * 0.15915494309189533577;
    float sin_a, cos_a;
    sincospif(static_cast<float>(2.0 * (turns - rint(turns))), &sin_a, &cos_a);
    s_turn[t][j] = make_float2(a.magnitude * cos_a, a.magnitude * sin_a);
  }
  __syncthreads();
  auto load = [](const T* p, float (&x)[E]) {
    if constexpr (E == 8) {
      const Vec8<T> w = *reinterpret_cast<const Vec8<T>*>(p);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = static_cast<float>(w.x[e]);
    } else {
      x[0] = static_cast<float>(*p);
    }
  };
  auto store = [](T* p, const float (&x)[E]) {
    if constexpr (E == 8) {
      Vec8<T> w;
#pragma unroll
      for (int e = 0; e < 8; ++e) w.x[e] = static_cast<T>(x[e]);
      *reinterpret_cast<Vec8<T>*>(p) = w;
    } else {
      *p = static_cast<T>(x[0]);
    }
  };
  const int turned = a.heads + a.kv_heads, n_turned = turned * a.per_head.d;
  for (int t = 0; t < n; ++t) {
    const int pos = s_pos[t];
    const int64_t slot = pos < 0 || s_slot[t] < 0 || s_slot[t] >= a.n_slots ? -1 : s_slot[t];
    const int64_t token = token0 + t;
    const int64_t at_page = (slot >> a.shift) * a.page_stride + (slot & ((1 << a.shift) - 1)) * a.place_stride;
    for (int i = blockIdx.y * kRotateThreads + tid; i < a.items; i += gridDim.y * kRotateThreads) {
      if (i >= n_turned) {  // values
        const int r = i - n_turned, h = div_of(r, a.tail), e = (r - h * a.tail.d) * E;
        if (slot < 0) continue;
        float x[E];
        load(static_cast<const T*>(a.v) + token * a.v_stride + h * a.v_head + e, x);
        store(static_cast<T*>(a.v_pages) + at_page + h * a.head_stride + e, x);
        continue;
      }
      const int h = div_of(i, a.per_head), c = i - h * a.per_head.d;
      const bool query = h < a.heads;
      if (!query && slot < 0) continue;
      const T* from = query ? static_cast<const T*>(a.q) + token * a.q_stride + h * a.q_head
                            : static_cast<const T*>(a.k) + token * a.k_stride + (h - a.heads) * a.k_head;
      T* to = query ? static_cast<T*>(a.out_q) + (token * a.heads + h) * a.D
                    : static_cast<T*>(a.k_pages) + at_page + (h - a.heads) * a.head_stride;
      if (pos < 0) {  // (a query: keys without a slot are gone)
        const float zero[E] = {};
        if (INTERLEAVED || c * E >= half) {
          store(to + c * E + (INTERLEAVED ? 0 : half), zero);
        } else {
          store(to + c * E, zero);
          store(to + half + c * E, zero);
        }
        continue;
      }
      if constexpr (INTERLEAVED) {
        const int e0 = c * E;
        float x[E], y[E];
        load(from + e0, x);
        if constexpr (E == 8) {
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            const bool turn = e0 + e < a.dim;
            const float2 w = s_turn[t][min((e0 + e) / 2, 127)];
            y[e] = turn ? x[e] * w.x - x[e + 1] * w.y : x[e];
            y[e + 1] = turn ? x[e + 1] * w.x + x[e] * w.y : x[e + 1];
          }
        } else {
          y[0] = x[0];
          if (e0 < a.dim) {
            float other[1];
            load(from + (e0 ^ 1), other);
            const float2 w = s_turn[t][e0 / 2];
            y[0] = e0 & 1 ? x[0] * w.x + other[0] * w.y : x[0] * w.x - other[0] * w.y;
          }
        }
        store(to + e0, y);
      } else if (c * E < half) {
        const int j = c * E;
        float x1[E], x2[E], y1[E], y2[E];
        load(from + j, x1);
        load(from + half + j, x2);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float2 w = s_turn[t][j + e];
          y1[e] = x1[e] * w.x - x2[e] * w.y;
          y2[e] = x2[e] * w.x + x1[e] * w.y;
        }
        store(to + j, y1);
        store(to + half + j, y2);
      } else {
        float x[E];
        load(from + half + c * E, x);
        store(to + half + c * E, x);
      }
    }
  }
}

}  // namespace vpg
