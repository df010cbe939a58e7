// Rotation of queries and keys by their positions, and keys and values into their slots.
//
// Pair (x1, x2) of a token at position p turns by a = p f_j:
//   y1 = m (x1 cos a - x2 sin a), y2 = m (x2 cos a + x1 sin a)
// a is taken in 64 bits and brought to turns there (a / 2 pi less its nearest whole number), so that its sine and
// cosine are right to fp32 up to position 2^28 (then a's own rounding, a 2^-53, shows). Each element is read and written
// once, products and sums are fp32, and the result is rounded once to the elements' type. Bound by HBM for many tokens (16384 of 48 heads of 128, 403 MB: 74 us, 5.4
// TB/s, as a copy, pairs of either kind; rows at odd addresses, an element at a time, 163 in halves and 241 in pairs; heads of 192
// in halves, which are not exchanged, 139, 4.3 TB/s), by latency for few (4 tokens 3 us): a token's angles are worked
// out once, in LDS, for all heads.
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
  int items;  // of a token
  Div per_head, tail;  // items of a query's or key's head, of a value's
};

constexpr int kRotateThreads = 256;

// How a head's pairs lie, and how a thread comes by both of one:
enum Pairs {
  kHalves,      // (j, j + dim / 2): it takes E of each half
  kExchanged,   // the same, from the lane that has the other half: whole heads lie in a wave, eight elements a lane. All
                // lanes' accesses are one run then: 16384 tokens of 48 heads of 128 74 us, against 89
  kAdjacent     // (2j, 2j + 1)
};

// A workgroup takes a token (and, where there are few, some of its items: gridDim.y of them share it). E: elements of an
// access, 8 (all addresses are multiples of 16 bytes, and halves' pairs lie in whole vectors) or 1. An item is E elements of
// a head, but with kHalves, of queries and keys, E pairs of the turned part, or E elements of the rest.
template <class T, int E, Pairs PAIRS>
__global__ __launch_bounds__(kRotateThreads) void k_rotate(RotateArgs a) {
  __shared__ float2 s_turn[128];
  const int tid = threadIdx.x, half = a.dim / 2;
  const int64_t token = blockIdx.x;
  const int pos = a.positions[token], place = a.slots[token];
  for (int j = tid; j < half; j += kRotateThreads) {
    const double turns = pos * a.freq[j] * 0.15915494309189533577;
    float sin_a, cos_a;
    sincospif(static_cast<float>(2.0 * (turns - rint(turns))), &sin_a, &cos_a);
    s_turn[j] = make_float2(a.magnitude * cos_a, a.magnitude * sin_a);
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
  const int n_turned = (a.heads + a.kv_heads) * a.per_head.d;
  const int64_t slot = pos < 0 || place < 0 || place >= a.n_slots ? -1 : place;
  const int64_t at_page = (slot >> a.shift) * a.page_stride + (slot & ((1 << a.shift) - 1)) * a.place_stride;
  // (whole waves go round together: lanes exchange halves)
  for (int first = blockIdx.y * kRotateThreads; first < a.items; first += gridDim.y * kRotateThreads) {
    const int i = first + tid;
    const bool value = i >= n_turned;
    const int r = value ? i - n_turned : i;
    const int h = div_of(r, value ? a.tail : a.per_head), c = r - h * (value ? a.tail.d : a.per_head.d);
    const bool query = !value && h < a.heads, there = i < a.items && (query || slot >= 0);
    const T* from = static_cast<const T*>(value ? a.v : query ? a.q : a.k) + token * (value ? a.v_stride : query ? a.q_stride : a.k_stride) +
                    (value || query ? h : h - a.heads) * (value ? a.v_head : query ? a.q_head : a.k_head);
    T* to = query ? static_cast<T*>(a.out_q) + (token * a.heads + h) * a.D
                  : static_cast<T*>(value ? a.v_pages : a.k_pages) + at_page + (value ? h : h - a.heads) * a.head_stride;
    if constexpr (PAIRS == kExchanged) {
      float x[E] = {}, other[E];
      if (there) load(from + c * E, x);
      const int h8 = half / E, lane = tid & 63, partner = value || c >= 2 * h8 ? lane : c < h8 ? lane + h8 : lane - h8;
#pragma unroll
      for (int e = 0; e < E; e += 2) {  // (two to a word, as they came)
        typedef T Two __attribute__((ext_vector_type(2)));
        const Two mine = {static_cast<T>(x[e]), static_cast<T>(x[e + 1])};
        const Two got = __builtin_bit_cast(Two, __shfl(__builtin_bit_cast(int, mine), partner));
        other[e] = static_cast<float>(got[0]);
        other[e + 1] = static_cast<float>(got[1]);
      }
      if (partner != lane) {
        const float sign = c < h8 ? -1.0f : 1.0f;
        const int j = (c < h8 ? c : c - h8) * E;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float2 w = s_turn[j + e];
          x[e] = x[e] * w.x + sign * (other[e] * w.y);
        }
      }
      if (pos < 0)
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = 0.0f;
      if (there) store(to + c * E, x);
      continue;
    }
    if (!there) continue;
    if (value) {
      float x[E];
      load(from + c * E, x);
      store(to + c * E, x);
      continue;
    }
    if (pos < 0) {  // (a query: keys without a slot are gone)
      const float zero[E] = {};
      if (PAIRS == kAdjacent || c * E >= half) {
        store(to + c * E + (PAIRS == kAdjacent ? 0 : half), zero);
      } else {
        store(to + c * E, zero);
        store(to + half + c * E, zero);
      }
      continue;
    }
    if constexpr (PAIRS == kAdjacent) {
      const int e0 = c * E;
      float x[E], y[E];
      load(from + e0, x);
      if constexpr (E == 8) {
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          const bool turn = e0 + e < a.dim;
          const float2 w = s_turn[min((e0 + e) / 2, 127)];
          y[e] = turn ? x[e] * w.x - x[e + 1] * w.y : x[e];
          y[e + 1] = turn ? x[e + 1] * w.x + x[e] * w.y : x[e + 1];
        }
      } else {
        y[0] = x[0];
        if (e0 < a.dim) {
          float other[1];
          load(from + (e0 ^ 1), other);
          const float2 w = s_turn[e0 / 2];
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
        const float2 w = s_turn[j + e];
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

}  // namespace vpg
