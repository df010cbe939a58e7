// Attention of sequences in groups that share a prefix, over pages.
//
// The rows that read a run of keys lie side by side: all of a group's (sequence, token, query head) rows of a key head
// on its prefix, a sequence's (token, query head) rows on its own keys. A segment is up to kRows such rows on one run
// of keys; per key head the segments' tiles of kKeys keys make one long line, all heads' lines are cut into as many
// equal stretches as workgroups fit the chip, and each workgroup walks one stretch (the plan, made once a step). So
// any mix of long and short keys, few and many rows, fills the chip evenly. Rows whose keys fall into several
// stretches leave each one's maximum, sum and products (fp32), joined by a second kernel in the stretches' order.
//
// A tile: S^T = K Q^T by 32x32x16 matrix products (a lane holds one row's scores: maxima and sums stay in the lane
// and its partner 32 lanes on), running maximum and sum, P rounded to the values' type, O^T += V^T P^T with V read
// from LDS transposed, which brings its keys in the order in which the scores lie in a lane: P never leaves the
// registers. Next tiles' keys and values come through registers into the other half of LDS while a tile is computed.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "tables.cuh"

namespace vpg {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr int kRows = 128;  // of a segment: 32 a wave
constexpr int kWaves = 4;

// Keys of a tile: as many as two halves of LDS hold with two workgroups a CU.
constexpr int tile_keys(int head_dim) { return head_dim > 128 ? 32 : 64; }

struct Shape {
  int S, B, T, H, Hkv, D, shift, M, MP;
  int G, rows, own_tiles, max_prefix, keys, wgs;  // query heads a key head; T G; a sequence's segments; the prefixes'
};

// A segment: `rows` rows from row0 of those that sequences from seq0 on make, on a run of keys.
struct alignas(16) Segment {
  int table;  // a sequence's, or ~group's
  int seq0, row0, rows;
  int keys, tiles, unit, index;  // positions there are; the tiles seen; where they begin in a head's line; which of its kind
};
constexpr int kAlone = 1 << 30;  // in rows: no other segment has these rows

struct Head {
  int units, n_prefix, n_own, per_wg;  // tiles of a head's line; segments; tiles of a workgroup
};

// The plan in memory, all of 4-byte words.
struct Plan {
  Head* head;
  int2* start;      // [wgs]: a workgroup's first segment, and the tile in it
  int* own;         // [S own_tiles]: segments of the sequences, -1 where there are no keys
  int* group;       // [S]: a sequence's group, or -1
  int* prefix;      // [B]: a group's first segment, or -1
  Segment* segments;
};
__host__ __device__ inline Plan plan_at(const Shape& s, void* p) {
  char* c = static_cast<char*>(p);
  auto up = [](size_t x) { return (x + 255) & ~static_cast<size_t>(255); };
  Plan r;
  r.head = reinterpret_cast<Head*>(c);
  size_t at = 256;
  r.start = reinterpret_cast<int2*>(c + at);
  at += up(static_cast<size_t>(s.wgs) * 8);
  r.own = reinterpret_cast<int*>(c + at);
  at += up(static_cast<size_t>(s.S) * s.own_tiles * 4);
  r.group = reinterpret_cast<int*>(c + at);
  at += up(static_cast<size_t>(s.S) * 4);
  r.prefix = reinterpret_cast<int*>(c + at);
  at += up(static_cast<size_t>(s.B) * 4);
  r.segments = reinterpret_cast<Segment*>(c + at);
  return r;
}
inline size_t plan_bytes(const Shape& s) {
  const Plan p = plan_at(s, nullptr);
  return reinterpret_cast<size_t>(p.segments) + (static_cast<size_t>(s.max_prefix) + static_cast<size_t>(s.S) * s.own_tiles) * sizeof(Segment);
}

__global__ __launch_bounds__(kTableThreads) void k_plan(Shape z, const int32_t* __restrict__ lengths,
                                                        const int32_t* __restrict__ prefix_lengths,
                                                        const int32_t* __restrict__ group_starts, void* mem) {
  __shared__ int part[kTableThreads / 64];
  const Plan plan = plan_at(z, mem);
  const int tid = threadIdx.x;
  const int64_t max_own = min(static_cast<int64_t>(z.M) << z.shift, static_cast<int64_t>(INT32_MAX) - 64);
  const int64_t max_prefix = min(static_cast<int64_t>(z.MP) << z.shift, static_cast<int64_t>(INT32_MAX) - 64);
  int segments = 0, units = 0;
  for (int base = 0; base < z.B; base += kTableThreads) {  // the groups' prefixes
    const int g = base + tid;
    int seq0 = 0, n = 0, len = 0, total;
    if (g < z.B) {
      seq0 = clampi(group_starts[g], 0, z.S);
      n = max(clampi(group_starts[g + 1], 0, z.S) - seq0, 0);
      len = static_cast<int>(min(static_cast<int64_t>(max(prefix_lengths[g], 0)), max_prefix));
    }
    const int64_t rows = static_cast<int64_t>(n) * z.rows;
    const int tiles = (len + z.keys - 1) / z.keys;
    int mine = tiles ? static_cast<int>((rows + kRows - 1) / kRows) : 0;
    const int first = segments + scan_exclusive<int>(mine, part, total);
    segments += total;
    if (first + mine > z.max_prefix) mine = 0;  // (group_starts that do not ascend)
    const int unit = units + scan_exclusive<int>(mine * tiles, part, total);
    units += total;
    if (g < z.B) plan.prefix[g] = mine ? first : -1;
    for (int i = 0; i < mine; ++i) {
      Segment s;
      s.table = ~g;
      s.seq0 = seq0;
      s.row0 = i * kRows;
      s.rows = static_cast<int>(min(rows - static_cast<int64_t>(i) * kRows, static_cast<int64_t>(kRows)));
      s.keys = len;
      s.tiles = tiles;
      s.unit = unit + i * tiles;
      s.index = first + i;
      plan.segments[first + i] = s;
    }
  }
  segments = min(segments, z.max_prefix);
  const int n_prefix = segments;
  for (int s = tid; s < z.S; s += kTableThreads) {
    int g = -1;
    if (z.B) {
      g = find(group_starts, z.B, s);
      if (s < group_starts[g] || s >= group_starts[g + 1]) g = -1;
    }
    plan.group[s] = g;
  }
  __syncthreads();
  const int n_items = z.S * z.own_tiles;
  int own = 0;
  for (int base = 0; base < n_items; base += kTableThreads) {  // the sequences' own keys
    const int item = base + tid;
    int s = 0, row0 = 0, rows = 0, len = 0, tiles = 0, total;
    if (item < n_items) {
      s = item / z.own_tiles;
      row0 = (item - s * z.own_tiles) * kRows;
      rows = min(z.rows - row0, kRows);
      len = static_cast<int>(min(static_cast<int64_t>(max(lengths[s], 0)), max_own));
      const int seen = min(len, len - z.T + 1 + (row0 + rows - 1) / z.G);  // by the last row
      tiles = seen > 0 ? (seen + z.keys - 1) / z.keys : 0;
    }
    const int index = own + scan_exclusive<int>(tiles > 0, part, total);
    own += total;
    const int unit = units + scan_exclusive<int>(tiles, part, total);
    units += total;
    if (item < n_items) plan.own[item] = tiles ? n_prefix + index : -1;
    if (tiles) {
      const int g = plan.group[s];
      Segment w;
      w.table = s;
      w.seq0 = s;
      w.row0 = row0;
      w.rows = rows | (g < 0 || plan.prefix[g] < 0 ? kAlone : 0);
      w.keys = len;
      w.tiles = tiles;
      w.unit = unit;
      w.index = index;
      plan.segments[n_prefix + index] = w;
    }
  }
  const int64_t all = static_cast<int64_t>(units) * z.Hkv;
  const int per_wg = static_cast<int>((all + z.wgs - 1) / z.wgs);
  if (tid == 0) *plan.head = Head{units, n_prefix, own, per_wg};
  __syncthreads();
  for (int w = tid; w < z.wgs; w += kTableThreads) {
    const int64_t u = static_cast<int64_t>(w) * per_wg;
    if (u >= all) continue;
    const int at = static_cast<int>(u % units);
    int lo = 0;
    const int n = n_prefix + own;
    for (int step = 1 << (31 - __clz(n)); step; step >>= 1)
      if (lo + step < n && plan.segments[lo + step].unit <= at) lo += step;
    plan.start[w] = make_int2(lo, at - plan.segments[lo].unit);
  }
}

struct AttendArgs {
  Shape z;
  int pages;
  float scale;  // log2 e in it
  const void* q;
  int64_t q_stride, q_token, q_head;
  const void *k, *v;
  int64_t page_stride, place_stride, head_stride;
  const int32_t *tables, *prefix_tables;
  int64_t table_stride, prefix_table_stride;
  void* out;
  void* plan;
  // Partial results, by rows: those of segments that a workgroup began or ended within (two a workgroup, cut_rows
  // each), then those of whole segments of sequences, own_rows each, and of prefixes, prefix_rows each.
  float* o;    // [..][D]
  float2* ml;  // maximum (in powers of 2) and sum
  int64_t own_at, prefix_at;
  int cut_rows, own_rows, prefix_rows;
};

// Where the rows of segment g of head h are that stretch w has from `tile` on.
__device__ __forceinline__ int64_t partial_row(const AttendArgs& a, const Head& head, const Segment& g, int h, int w, bool whole, bool from_start) {
  if (!whole) return static_cast<int64_t>(2 * w + from_start) * a.cut_rows;
  if (g.table < 0) return a.prefix_at + (static_cast<int64_t>(h) * head.n_prefix + g.index) * a.prefix_rows;
  return a.own_at + (static_cast<int64_t>(h) * head.n_own + g.index) * a.own_rows;
}

// Workgroups of neighbouring stretches on one XCD: its L2 serves those that read the same keys.
__device__ __forceinline__ int stretch_of(int block, int wgs) { return (block & 7) * (wgs >> 3) + (block >> 3); }

template <class T>
struct Mma;
template <>
struct Mma<__bf16> {
  typedef bf16x8 V8;
  static __device__ __forceinline__ f32x16 mma(V8 a, V8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
template <>
struct Mma<_Float16> {
  typedef f16x8 V8;
  static __device__ __forceinline__ f32x16 mma(V8 a, V8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};

__device__ __forceinline__ float other_half(float x) { return __shfl_xor(x, 32); }

// DP: the head's elements, rounded up to a multiple of 32.
template <class T, int DP>
__global__ __launch_bounds__(kWaves * 64, DP > 192 ? 1 : 2) void k_attend(AttendArgs a) {
  typedef typename Mma<T>::V8 V8;
  constexpr int kKeys = tile_keys(DP), CH = DP / 8, kThreads = kWaves * 64;
  constexpr int kLoads = kKeys * CH / kThreads;  // 16-byte pieces of keys (and of values) that a thread brings
  static_assert(kKeys * CH % kThreads == 0, "a tile is whole pieces of every thread");
  // Rows 16 bytes longer: 16 keys' pieces lie in 16 different groups of banks. The values' rows are 16 words on, modulo
  // 64, so that four keys' 64 bytes (a transposed read of half a wave) fill the banks.
  constexpr int kStrideK = DP + 8, kStrideV = DP % 64 ? DP : DP + 32;
  __shared__ __align__(16) T s_k[2][kKeys * kStrideK];
  __shared__ __align__(16) T s_v[2][kKeys * kStrideV];
  const Shape& z = a.z;
  const Plan plan = plan_at(z, a.plan);
  const Head head = *plan.head;
  const int w = stretch_of(blockIdx.x, z.wgs);
  const int64_t all = static_cast<int64_t>(head.units) * z.Hkv, u0 = static_cast<int64_t>(w) * head.per_wg;
  if (u0 >= all) return;
  int left = static_cast<int>(min(static_cast<int64_t>(head.per_wg), all - u0));
  int h = static_cast<int>(u0 / head.units);
  const int2 start = plan.start[w];
  int seg = start.x, tile = start.y;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int col = lane & 31, half = lane >> 5;
  const int n_segments = head.n_prefix + head.n_own;

  for (; left > 0; ++seg, tile = 0) {
    if (seg == n_segments) {
      seg = 0;
      ++h;
    }
    const Segment g = plan.segments[seg];
    const int n = min(left, g.tiles - tile);
    left -= n;
    const bool prefix = g.table < 0;
    const int n_rows = g.rows & (kAlone - 1);
    const bool busy = wave * 32 < n_rows;

    // this lane's row: its queries, and the keys that it sees
    const int r = wave * 32 + col;
    const bool valid = r < n_rows;
    V8 q[DP / 16];
    int limit = 0;
    if (busy) {
      const int R = g.row0 + (valid ? r : 0);
      const int in = R / z.rows, rest = R - in * z.rows, t = rest / z.G, gq = rest - t * z.G;
      const T* from = static_cast<const T*>(a.q) + (g.seq0 + in) * a.q_stride + t * a.q_token + (h * z.G + gq) * a.q_head;
      limit = prefix ? g.keys : min(g.keys, g.keys - z.T + t + 1);
#pragma unroll
      for (int c = 0; c < DP / 16; ++c) {
        const int d = c * 16 + half * 8;
        if (d < z.D) q[c] = *reinterpret_cast<const V8*>(from + d);
        else q[c] = V8{};
      }
    }
    const int least = prefix ? g.keys : min(g.keys, g.keys - z.T + 1 + (g.row0 + wave * 32) / z.G);  // of the wave's rows

    const int32_t* table = prefix ? a.prefix_tables + static_cast<int64_t>(~g.table) * a.prefix_table_stride
                                  : a.tables + static_cast<int64_t>(g.table) * a.table_stride;
    const T* k_head = static_cast<const T*>(a.k) + h * a.head_stride;
    const T* v_head = static_cast<const T*>(a.v) + h * a.head_stride;
    V8 k_in[kLoads], v_in[kLoads];
    auto fetch = [&](int tile_at) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int piece = tid + i * kThreads, key = piece / CH, c = piece % CH;
        const int j = min(tile_at * kKeys + key, g.keys - 1);  // (keys past the last are the last once more)
        const int page = clampi(table[j >> z.shift], 0, a.pages - 1);
        const int64_t at = page * a.page_stride + (j & ((1 << z.shift) - 1)) * a.place_stride + c * 8;
        if (c * 8 < z.D) {
          k_in[i] = *reinterpret_cast<const V8*>(k_head + at);
          v_in[i] = *reinterpret_cast<const V8*>(v_head + at);
        } else {
          k_in[i] = V8{};
          v_in[i] = V8{};
        }
      }
    };
    auto put = [&](int b) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int piece = tid + i * kThreads, key = piece / CH, c = piece % CH;
        *reinterpret_cast<V8*>(&s_k[b][key * kStrideK + c * 8]) = k_in[i];
        *reinterpret_cast<V8*>(&s_v[b][key * kStrideV + c * 8]) = v_in[i];
      }
    };

    float m = -INFINITY, l = 0.0f;
    f32x16 o[DP / 32];
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) o[d] = f32x16{};
    fetch(tile);
    __syncthreads();  // (the segment before is read)
    put(0);
    if (n > 1) fetch(tile + 1);
    __syncthreads();
    for (int it = 0; it < n; ++it) {
      const int b = it & 1, key0 = (tile + it) * kKeys;
      if (busy) {
        f32x16 s[kKeys / 32];
        float most = -INFINITY;
#pragma unroll
        for (int kk = 0; kk < kKeys / 32; ++kk) {
          s[kk] = f32x16{};
#pragma unroll
          for (int c = 0; c < DP / 16; ++c) {
            const V8 kv = *reinterpret_cast<const V8*>(&s_k[b][(kk * 32 + col) * kStrideK + c * 16 + half * 8]);
            s[kk] = Mma<T>::mma(kv, q[c], s[kk]);
          }
        }
        if (key0 + kKeys > least) {
#pragma unroll
          for (int kk = 0; kk < kKeys / 32; ++kk)
#pragma unroll
            for (int i = 0; i < 16; ++i)
              if (key0 + kk * 32 + 8 * (i / 4) + 4 * half + i % 4 >= limit) s[kk][i] = -INFINITY;
        }
#pragma unroll
        for (int kk = 0; kk < kKeys / 32; ++kk)
#pragma unroll
          for (int i = 0; i < 16; ++i) most = fmaxf(most, s[kk][i]);
        most = fmaxf(most, other_half(most)) * a.scale;
        if (__any(most > m)) {
          const float now = fmaxf(m, most), by = now == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - now);
          m = now;
          l *= by;
#pragma unroll
          for (int d = 0; d < DP / 32; ++d) o[d] *= by;
        }
        const float from = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int kk = 0; kk < kKeys / 32; ++kk) {
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            s[kk][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kk][i], a.scale, -from));
            l += s[kk][i];
          }
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            V8 p;
#pragma unroll
            for (int i = 0; i < 8; ++i) p[i] = static_cast<T>(s[kk][8 * c + i]);
            const T* v0 = &s_v[b][(kk * 32 + c * 16 + 4 * half + (lane & 15) / 4) * kStrideV + (lane >> 4 & 1) * 16 + (lane & 3) * 4];
#pragma unroll
            for (int d = 0; d < DP / 32; ++d) {
              typedef __attribute__((address_space(3))) s16x4* Lds;
              const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(v0 + d * 32));
              const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(v0 + d * 32 + 8 * kStrideV));
              const V8 vv = __builtin_bit_cast(V8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
              o[d] = Mma<T>::mma(vv, p, o[d]);
            }
          }
        }
      }
      if (it + 1 < n) {
        put(b ^ 1);
        if (it + 2 < n) fetch(tile + it + 2);
      }
      __syncthreads();
    }
    l += other_half(l);
    if (!valid || !busy) continue;
    const int R = g.row0 + r;
    if ((g.rows & kAlone) && n == g.tiles) {
      const int t = R / z.G, gq = R - t * z.G;
      T* to = static_cast<T*>(a.out) + ((static_cast<int64_t>(g.seq0) * z.T + t) * z.H + h * z.G + gq) * z.D;
      const float by = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
      for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int at = d * 32 + 8 * i + 4 * half;
          if (at < z.D) {
            typedef T T4 __attribute__((ext_vector_type(4)));
            T4 y;
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = static_cast<T>(o[d][4 * i + e] * by);
            *reinterpret_cast<T4*>(to + at) = y;
          }
        }
      continue;
    }
    const int64_t row = partial_row(a, head, g, h, w, n == g.tiles, tile == 0) + r;
    float* to = a.o + row * z.D;
    if (half == 0) a.ml[row] = make_float2(m, l);
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int at = d * 32 + 8 * i + 4 * half;
        if (at < z.D) *reinterpret_cast<f32x4*>(to + at) = f32x4{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
      }
  }
}

// A wave joins a row's stretches: o = sum_i 2^(m_i - m) o_i / sum_i 2^(m_i - m) l_i.
template <class T, int DP>
__global__ __launch_bounds__(256) void k_join(AttendArgs a) {
  const Shape& z = a.z;
  const int lane = threadIdx.x & 63;
  const int64_t id = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (id >= static_cast<int64_t>(z.S) * z.T * z.H) return;
  const int hq = static_cast<int>(id % z.H), st = static_cast<int>(id / z.H), t = st % z.T, s = st / z.T;
  const int h = hq / z.G, r = t * z.G + hq % z.G;
  const Plan plan = plan_at(z, a.plan);
  const Head head = *plan.head;
  T* to = static_cast<T*>(a.out) + id * z.D;
  constexpr int E = (DP + 63) / 64;
  const int own = plan.own[s * z.own_tiles + r / kRows], grp = plan.group[s];
  const int pre = grp < 0 ? -1 : plan.prefix[grp];
  Segment g{};
  if (own >= 0) g = plan.segments[own];
  if (own < 0 || g.keys - z.T + t + 1 <= 0) {  // no token
    for (int d = lane; d < z.D; d += 64) to[d] = static_cast<T>(0.0f);
    return;
  }
  auto stretches = [&](const Segment& x, int& first) {
    const int64_t u = static_cast<int64_t>(h) * head.units + x.unit;
    first = static_cast<int>(u / head.per_wg);
    return static_cast<int>((u + x.tiles - 1) / head.per_wg) - first + 1;
  };
  int first_own, first_pre = 0, n_pre = 0, r_pre = 0;
  const int n_own = stretches(g, first_own);
  if (pre < 0 && n_own == 1) return;  // (written already)
  Segment p{};
  if (pre >= 0) {
    const int R = (s - plan.segments[pre].seq0) * z.rows + r;
    p = plan.segments[pre + R / kRows];
    n_pre = stretches(p, first_pre);
    r_pre = R % kRows;
  }
  const int n = n_pre + n_own;
  auto row_of = [&](int i) {  // the prefix's stretches, then the sequence's own
    const bool is_pre = i < n_pre;
    if (!is_pre) i -= n_pre;
    return is_pre ? partial_row(a, head, p, h, first_pre + i, n_pre == 1, i == 0) + r_pre
                  : partial_row(a, head, g, h, first_own + i, n_own == 1, i == 0) + r % kRows;
  };
  float most = -INFINITY;
  for (int i = lane; i < n; i += 64) {
    most = fmaxf(most, a.ml[row_of(i)].x);
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) most = fmaxf(most, __shfl_xor(most, d));
  if (most == -INFINITY) most = 0.0f;
  float total = 0.0f, o[E] = {};
  for (int base = 0; base < n; base += 64) {
    float by = 0.0f;
    if (base + lane < n) {
      const float2 ml = a.ml[row_of(base + lane)];
      by = ml.y == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(ml.x - most);
      total += by * ml.y;
    }
    const int m = min(n - base, 64);
#pragma unroll 4
    for (int i = 0; i < m; ++i) {
      const float f = __shfl(by, i);
      const float* from = a.o + row_of(base + i) * z.D;
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (lane + 64 * e < z.D) o[e] += f * from[lane + 64 * e];
    }
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) total += __shfl_xor(total, d);
  const float by = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (lane + 64 * e < z.D) to[lane + 64 * e] = static_cast<T>(o[e] * by);
}

}  // namespace vpg
