// Attention of sequences in groups that share a prefix, over pages.
//
// The rows that read a run of keys lie side by side: all of a group's (sequence, token, query head) rows of a key head
// on its prefix, a sequence's (token, query head) rows on its own keys. A segment is some of these rows on one run of
// keys, in tiles. Two kinds are kept apart: wide segments (up to 128 rows where there are more than 32) are a
// workgroup's, 32 rows a wave on one tile of 64 keys; narrow ones (up to 32 rows) are a wave's alone, in tiles of 32
// keys. Per key head the segments' tiles make one long line; all heads' lines of a kind are cut into as many equal
// stretches as workgroups (waves) fit the chip, and each walks its own (the plan, made once a step): any mix of long
// and short keys, few and many rows, fills the chip evenly. Rows whose keys fall into several stretches leave each
// one's maximum, sum and products (fp32), joined by a second kernel in the stretches' order.
//
// A tile: S^T = K Q^T by 32x32x16 matrix products (a lane holds one row's scores: maxima and sums stay in the lane
// and its partner 32 lanes on), running maximum and sum, O^T += V^T P^T with V read from LDS transposed, which brings its keys
// in the order in which the scores lie in a lane: P never leaves the registers. P is rounded to the values' type, the only
// one that their product takes (a second product for what the rounding leaves would cost half as much again); the sum is taken
// of the rounded weights, so that their common error cancels. Against 64 bits the outputs are off by 0.0019 to 0.0020 of
// their size in bf16 (fp16 0.00023), where weights in fp32 leave the output's own rounding, 0.0017 (0.00021). The next tile's
// keys and values are on their way to registers while a tile is computed; their pages are looked up a tile before that, by
// scalar loads.
//
// Bound by HBM where rows are few: 4 sequences of 100000 positions with 5 tokens each (64 query, 8 key heads of 128, 1.15
// GB) 211 us, 5.4 TB/s; 64 requests of 4 beams behind up to 8192 positions (1.2 GB) 243 us, 4.9 TB/s. By matrix and vector
// instructions where a prefix has many: 192 sequences behind 32768 positions 103 GFLOP in 142 us, 720 TFLOP/s (heads of 64
// 600, of 256 540; four prompts' 384 tokens behind 4000 positions, heads of 256, 600). By chains of loads where there is little
// of both: 4 beams behind 1000 positions 12 us and 6 to join. Pages of fewer than 16 positions are looked up lane by lane in front
// of each load: the 64 requests 424 us a layer with pages of 8, and as much with pages of 4.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "stretches.cuh"
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

constexpr int kRows = 128;  // of a wide segment: 32 a wave
constexpr int kNarrow = 32;  // of a narrow one
constexpr int kWaves = 4;
constexpr int kWideKeys = 64, kNarrowKeys = 32;  // of a tile
constexpr int kRun = 16;                         // keys that a page is looked up for

struct Shape {
  int S, B, T, H, Hkv, D, shift, M, MP;
  int G, rows, own_tiles, wgs;     // query heads a key head; T G; a sequence's segments; workgroups
  int max_wide, max_narrow;        // segments there are room for
};

// A segment: `rows` rows from row0 of those that sequences from seq0 on make, on a run of keys.
struct alignas(16) Segment {
  int table;  // a sequence's, or ~group's
  int seq0, row0, rows;
  int keys, tiles, unit, index;  // positions there are; the tiles seen; where they begin in a head's line; which of its kind
};
constexpr int kAlone = 1 << 30;  // in rows: no other segment has these rows

// What a row's joining needs: of its sequence's segment, and of its group's first.
struct alignas(16) Place {
  int keys, tiles, unit, index;  // keys 0: there are none
};
struct alignas(16) PrefixPlace {
  int tiles, unit, index, row0;  // tiles 0: none; row0: the sequence's first row, or ~that where the group is wide
};

struct alignas(16) Start {  // of a stretch
  int segment, tile, head, lead;  // lead: places before the tile
  Segment first;  // the segment
};

struct alignas(16) Lines {
  int wide_units, n_wide, wide_per;        // tiles of a head's line, segments, tiles of a stretch
  int narrow_units, n_narrow, narrow_per;
  int n_narrow_prefix, n_narrow_own;
};

struct Plan {
  Lines* lines;
  Start *wide_start, *narrow_start;  // [wgs], [wgs kWaves]
  Place* own;                        // [S own_tiles]
  PrefixPlace* prefix;               // [S]
  int4* group;                       // [B]: a group's prefix segments: tiles, unit, index, wide
  Segment *wide, *narrow;
};
__host__ __device__ inline Plan plan_at(const Shape& s, void* p, size_t* bytes = nullptr) {
  char* c = static_cast<char*>(p);
  size_t at = 0;
  auto take = [&](size_t n) {
    char* r = c + at;
    at += (n + 255) & ~static_cast<size_t>(255);
    return r;
  };
  Plan r;
  r.lines = reinterpret_cast<Lines*>(take(sizeof(Lines)));
  r.wide_start = reinterpret_cast<Start*>(take(s.wgs * sizeof(Start)));
  r.narrow_start = reinterpret_cast<Start*>(take(s.wgs * kWaves * sizeof(Start)));
  r.own = reinterpret_cast<Place*>(take(static_cast<size_t>(s.S) * s.own_tiles * sizeof(Place)));
  r.prefix = reinterpret_cast<PrefixPlace*>(take(s.S * sizeof(PrefixPlace)));
  r.group = reinterpret_cast<int4*>(take(s.B * sizeof(int4)));
  r.wide = reinterpret_cast<Segment*>(take(static_cast<size_t>(s.max_wide) * sizeof(Segment)));
  r.narrow = reinterpret_cast<Segment*>(take(static_cast<size_t>(s.max_narrow) * sizeof(Segment)));
  if (bytes) *bytes = at;
  return r;
}

// A segment costs its tiles and what its beginning takes (its queries' and first keys' way from memory, its results'):
// about as long as the next two tiles' at full bandwidth. A line has this many places before each segment's first tile.
constexpr int kLead = 2;

constexpr int kLeast = 2;  // tiles of a narrow stretch at least: joining more of them takes longer than a tile more
constexpr int kHeld = 2048;  // segments and groups whose numbers a plan's making holds in LDS

// Where a line's stretches begin. `unit`: the segments' first tiles.
template <class Index>
__device__ __forceinline__ void write_starts(const Segment* segments, const int* held, int n, const Stretches& line, Start* out) {
  for (int w = threadIdx.x; begins<Index>(line, w); w += kTableThreads) {
    const Index u = static_cast<Index>(w) * line.per;
    Start s;
    s.head = static_cast<int>(u / line.units);
    const int at = static_cast<int>(u - static_cast<Index>(s.head) * line.units);
    int lo = 0;
    if (n <= kHeld) {
      lo = find(held, n, at + kLead);
    } else {
      for (int step = 1 << (31 - __clz(n)); step; step >>= 1)
        if (lo + step < n && segments[lo + step].unit <= at + kLead) lo += step;
    }
    s.segment = lo;
    s.first = segments[lo];
    s.tile = max(at - s.first.unit, 0);
    s.lead = max(s.first.unit - at, 0);
    out[w] = s;
  }
}

// One workgroup: the groups' segments, then the sequences' own, then the stretches' beginnings; prefix sums and searches in
// LDS. A chain of loads and barriers: 7 us for one request, 16 for 256 sequences in 64 groups.
__global__ __launch_bounds__(kTableThreads) void k_plan(Shape z, const int32_t* __restrict__ lengths,
                                                        const int32_t* __restrict__ prefix_lengths,
                                                        const int32_t* __restrict__ group_starts, void* mem) {
  __shared__ unsigned part1[1][kTableThreads / 64], part4[4][kTableThreads / 64], part2[2][kTableThreads / 64];
  __shared__ int s_wide[kHeld], s_narrow[kHeld], s_start[kHeld];
  __shared__ int4 s_group[kHeld];
  const Plan plan = plan_at(z, mem);
  const int tid = threadIdx.x;
  const int64_t max_own = min(static_cast<int64_t>(z.M) << z.shift, static_cast<int64_t>(INT32_MAX) - 64);
  const int64_t max_prefix = min(static_cast<int64_t>(z.MP) << z.shift, static_cast<int64_t>(INT32_MAX) - 64);
  const bool own_narrow = z.rows <= kNarrow, held = z.B < kHeld;
  const int* starts = held ? s_start : group_starts;
  int4* groups = held ? s_group : plan.group;
  // (the first round's own lengths are on their way meanwhile)
  const int n_items = z.S * z.own_tiles;
  const int s_first = tid < n_items ? tid / z.own_tiles : 0;
  const int len_first = tid < n_items ? lengths[s_first] : 0;
  int sequences = 0, n_wide = 0, n_narrow = 0, wide_units = 0, narrow_units = 0;
  for (int base = 0; base < z.B; base += kTableThreads) {  // the groups' prefixes
    const int g = base + tid;
    int seq0 = 0, n = 0, len = 0;
    if (g < z.B) {
      const int from = group_starts[g], to = group_starts[g + 1];
      if (held) {
        s_start[g] = from;
        if (g == z.B - 1) s_start[z.B] = to;
      }
      seq0 = clampi(from, 0, z.S);
      n = max(clampi(to, 0, z.S) - seq0, 0);
      len = static_cast<int>(min(static_cast<int64_t>(max(prefix_lengths[g], 0)), max_prefix));
    }
    unsigned before[1] = {static_cast<unsigned>(n)}, total1[1];
    scan_exclusive<1>(before, total1, part1, Add{});
    if (sequences + static_cast<int64_t>(before[0]) + n > z.S) n = 0;  // (group_starts that do not ascend)
    sequences = static_cast<int>(min(static_cast<unsigned>(sequences) + total1[0], static_cast<unsigned>(z.S) + 1));
    const int64_t rows = static_cast<int64_t>(n) * z.rows;
    const bool is_wide = rows > kNarrow;
    const int keys = is_wide ? kWideKeys : kNarrowKeys, tiles = (len + keys - 1) / keys;
    const int wide = tiles && is_wide ? static_cast<int>((rows + kRows - 1) / kRows) : 0;
    const int narrow = tiles && rows && !is_wide;
    unsigned x[4] = {static_cast<unsigned>(wide), static_cast<unsigned>(wide) * (tiles + kLead), static_cast<unsigned>(narrow),
                     narrow ? static_cast<unsigned>(tiles + kLead) : 0u}, total[4];
    scan_exclusive<4>(x, total, part4, Add{});
    const int first_wide = n_wide + x[0], wide_unit = wide_units + x[1] + kLead, first_narrow = n_narrow + x[2];
    const int narrow_unit = narrow_units + x[3] + kLead;
    n_wide += total[0];
    wide_units += total[1];
    n_narrow += total[2];
    narrow_units += total[3];
    if (g < z.B) groups[g] = make_int4(wide || narrow ? tiles : 0, wide ? wide_unit : narrow_unit, wide ? first_wide : first_narrow, wide != 0);
    for (int i = 0; i < wide + narrow; ++i) {
      Segment s;
      s.table = ~g;
      s.seq0 = seq0;
      s.row0 = i * kRows;
      s.rows = static_cast<int>(min(rows - static_cast<int64_t>(i) * kRows, static_cast<int64_t>(kRows)));
      s.keys = len;
      s.tiles = tiles;
      s.unit = wide ? wide_unit + i * (tiles + kLead) : narrow_unit;
      s.index = wide ? first_wide + i : first_narrow;
      (wide ? plan.wide : plan.narrow)[s.index] = s;
      if (s.index < kHeld) (wide ? s_wide : s_narrow)[s.index] = s.unit;
    }
  }
  const int n_narrow_prefix = n_narrow, keys = own_narrow ? kNarrowKeys : kWideKeys;
  __syncthreads();
  int n_own = own_narrow ? n_narrow : n_wide, units = own_narrow ? narrow_units : wide_units, own = 0;
  for (int base = 0; base < n_items; base += kTableThreads) {  // the sequences' own keys
    const int item = base + tid;
    int s = 0, row0 = 0, rows = 0, len = 0, tiles = 0;
    PrefixPlace p{0, 0, 0, 0};
    if (item < n_items) {
      s = item / z.own_tiles;
      row0 = (item - s * z.own_tiles) * kRows;
      rows = min(z.rows - row0, kRows);
      len = static_cast<int>(min(static_cast<int64_t>(max(base ? lengths[s] : len_first, 0)), max_own));
      const int seen = min(len, len - z.T + 1 + (row0 + rows - 1) / z.G);  // by the last row
      tiles = seen > 0 ? (seen + keys - 1) / keys : 0;
      if (z.B) {
        const int g = find(starts, z.B, s), seq0 = max(starts[g], 0);
        if (s >= seq0 && s < starts[g + 1]) {
          const int4 q = groups[g];
          p = PrefixPlace{q.x, q.y, q.z, q.w ? ~((s - seq0) * z.rows) : (s - seq0) * z.rows};
        }
      }
      if (!row0) plan.prefix[s] = p;
    }
    unsigned x[2] = {tiles > 0, tiles ? static_cast<unsigned>(tiles + kLead) : 0u}, total[2];
    scan_exclusive<2>(x, total, part2, Add{});
    const int at = x[0], segment = n_own + at, index = own_narrow ? own + at : segment, unit = units + x[1] + kLead;
    n_own += total[0];
    own += total[0];
    units += total[1];
    if (item < n_items) plan.own[item] = Place{tiles ? len : 0, tiles, unit, index};
    if (tiles) {
      Segment w;
      w.table = s;
      w.seq0 = s;
      w.row0 = row0;
      w.rows = rows | (p.tiles ? 0 : kAlone);
      w.keys = len;
      w.tiles = tiles;
      w.unit = unit;
      w.index = index;
      (own_narrow ? plan.narrow : plan.wide)[segment] = w;
      if (segment < kHeld) (own_narrow ? s_narrow : s_wide)[segment] = unit;
    }
  }
  if (own_narrow) {
    n_narrow = n_own;
    narrow_units = units;
  } else {
    n_wide = n_own;
    wide_units = units;
  }
  const Stretches wide_line = cut(wide_units, z.Hkv, z.wgs, 1), narrow_line = cut(narrow_units, z.Hkv, z.wgs * kWaves, kLeast);
  if (tid == 0)
    *plan.lines = Lines{wide_units, n_wide, wide_line.per, narrow_units, n_narrow, narrow_line.per, n_narrow_prefix, own_narrow ? own : 0};
  __syncthreads();
  auto write = [&](const Segment* segments, const int* unit, int n, const Stretches& line, Start* out) {
    if (small(line)) write_starts<int>(segments, unit, n, line, out);
    else write_starts<int64_t>(segments, unit, n, line, out);
  };
  write(plan.wide, s_wide, n_wide, wide_line, plan.wide_start);
  write(plan.narrow, s_narrow, n_narrow, narrow_line, plan.narrow_start);
}

struct AttendArgs {
  Shape z;
  int pages;
  float scale;  // log2 e in it
  const void* q;
  int64_t q_stride, q_token, q_head;
  const void *k, *v;
  uint32_t page_bytes, place_bytes;
  int64_t head_stride;
  const int32_t *tables, *prefix_tables;
  int64_t table_stride, prefix_table_stride;
  void* out;
  void* plan;
  // Partial results, by rows: those of segments that a stretch began or ended within (two a stretch, 128 and narrow_rows
  // each), then those of whole segments.
  float* o;    // [..][D]
  float2* ml;  // maximum (in powers of 2) and sum
  int64_t narrow_cut_at, wide_at, prefix_at, own_at;
  int narrow_rows, own_rows;
};

// Where the rows of a segment of head h are that stretch w has.
__device__ __forceinline__ int64_t partial_row(const AttendArgs& a, const Lines& n, bool wide, bool prefix, int index, int h, int w,
                                               bool whole, bool from_start) {
  if (wide) return (whole ? a.wide_at : 0) + (whole ? static_cast<int64_t>(h) * n.n_wide + index : 2 * w + from_start) * kRows;
  if (!whole) return a.narrow_cut_at + static_cast<int64_t>(2 * w + from_start) * a.narrow_rows;
  return prefix ? a.prefix_at + (static_cast<int64_t>(h) * n.n_narrow_prefix + index) * a.narrow_rows
                : a.own_at + (static_cast<int64_t>(h) * n.n_narrow_own + index) * a.own_rows;
}

// Workgroups of neighbouring stretches on one XCD: its L2 serves those that read the same keys.
__device__ __forceinline__ int stretch_of(int block, int wgs) { return (block & 7) * (wgs >> 3) + (block >> 3); }

// f(0), .., f(N - 1), each with its number as a constant: registers are told apart by numbers that the compiler knows.
template <int I>
struct Number {
  static constexpr int value = I;
};
template <int N, int I = 0, class F>
__device__ __forceinline__ void each(F&& f) {
  if constexpr (I < N) {
    f(Number<I>{});
    each<N, I + 1>(f);
  }
}

template <class T>
struct Mma;
template <>
struct Mma<__bf16> {
  typedef bf16x8 V8;
  static __device__ __forceinline__ f32x16 mma(V8 a, V8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ float add_pair(int x, float sum) {
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, x), bf16x2{1.0f, 1.0f}, sum, false);
  }
};
template <>
struct Mma<_Float16> {
  typedef f16x8 V8;
  static __device__ __forceinline__ f32x16 mma(V8 a, V8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ float add_pair(int x, float sum) {
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, x), f16x2{1.0f, 1.0f}, sum, false);
  }
};

__device__ __forceinline__ float other_half(float x) {  // the partner's, 32 lanes on
  const auto both = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x), false, false);
  return __builtin_bit_cast(float, (threadIdx.x & 32) ? both[0] : both[1]);
}

__device__ __forceinline__ float rounded_apart(float x, float scale, float from) {  // x scale, rounded, less `from`
#pragma clang fp contract(off)
  return x * scale - from;
}

// What the plan and the tables hold, by scalar loads: nothing writes them while a kernel runs.
template <class X>
__device__ __forceinline__ X uniform(const X* p) {
  static_assert(sizeof(X) % 4 == 0, "words");
  typedef const __attribute__((address_space(4))) int* Words;
  Words w = (Words)(reinterpret_cast<uintptr_t>(p));
  X x;
  int* to = reinterpret_cast<int*>(&x);
#pragma unroll
  for (unsigned i = 0; i < sizeof(X) / 4; ++i) to[i] = w[i];
  return x;
}

// What lanes of a wave wrote to LDS, read by its other lanes: a wave's accesses stay in order, the compiler has to know.
__device__ __forceinline__ void wave_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  asm volatile("" ::: "memory");
}

// A tile's layout in LDS. Keys' rows are 16 bytes longer: 16 keys' pieces lie in 16 different groups of banks. The values'
// rows are 16 or 48 words on, modulo 64, so that four keys' 64 bytes (a transposed read of half a wave) fill the banks.
template <int DP>
struct Layout {
  static constexpr int kStrideK = DP + 8, kStrideV = DP % 64 ? DP : DP + 32;
  static constexpr int kPieces = DP <= 64 ? 8 : DP <= 128 ? 16 : 32;  // lanes of a key's 16-byte pieces
  static constexpr int kAtOnce = 64 / kPieces;                        // keys of an access
};

typedef int i32x4 __attribute__((ext_vector_type(4)));

// A segment's keys and values of a head on their way: KEYS of them by this wave, 16 at a time from their page (a scalar
// base, the lanes' offsets the same for all; what a lane has not of a head's elements lies past the range: 0).
// SMALL: pages of fewer than 16 keys (a place of its own for each key of each lane).
template <class T, int DP, int KEYS, bool SMALL>
struct Stage {
  typedef typename Mma<T>::V8 V8;
  typedef Layout<DP> L;
  static constexpr int kLoads = KEYS / L::kAtOnce, kGroups = KEYS / kRun, kVariants = kRun / L::kAtOnce;
  static constexpr uint32_t kRange = 0x80000000u;
  V8 k[kLoads], v[kLoads];
  uint32_t offset[kVariants];
  const int32_t* table;
  const T *k_head, *v_head;
  int last;  // key
  struct Pages {
    uint64_t at[kGroups];  // bytes from a head's first page
  };

  __device__ __forceinline__ void begin(const AttendArgs& a, const Segment& g, int h) {
    table = g.table < 0 ? a.prefix_tables + static_cast<int64_t>(~g.table) * a.prefix_table_stride
                        : a.tables + static_cast<int64_t>(g.table) * a.table_stride;
    k_head = static_cast<const T*>(a.k) + h * a.head_stride;
    v_head = static_cast<const T*>(a.v) + h * a.head_stride;
    last = g.keys - 1;
    const int lane = threadIdx.x & 63, in = lane / L::kPieces, c = lane % L::kPieces;
#pragma unroll
    for (int i = 0; i < kVariants; ++i) offset[i] = place(a, i * L::kAtOnce + in, c);
  }
  static __device__ __forceinline__ uint32_t place(const AttendArgs& a, int key, int c) {
    return c * 8 < a.z.D ? static_cast<uint32_t>(key) * a.place_bytes + c * 16 : kRange;
  }
  // Where the keys from key0 on lie (keys past the last: the last run once more).
  __device__ __forceinline__ Pages look_up(const AttendArgs& a, int key0) const {
    Pages p;
    if (SMALL) return p;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      const int first = min(key0 + kRun * g, last & ~(kRun - 1));
      const unsigned page = clampi(uniform(table + (first >> a.z.shift)), 0, a.pages - 1);
      p.at[g] = static_cast<uint64_t>(page) * a.page_bytes + static_cast<unsigned>(first & ((1 << a.z.shift) - 1)) * a.place_bytes;
    }
    return p;
  }
  static __device__ __forceinline__ V8 load(const T* base, uint64_t at, uint32_t off) {
    char* p = const_cast<char*>(reinterpret_cast<const char*>(base)) + at;
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(p, 0, kRange, 0x00027000);
    return __builtin_bit_cast(V8, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0));
  }
  // x[..] = what the keys from key0 on have at `head`: the keys themselves or their values.
  __device__ __forceinline__ void fetch(V8 (&x)[kLoads], const T* head, const Pages& p, const AttendArgs& a, int key0) const {
    const int lane = threadIdx.x & 63, in = lane / L::kPieces, c = lane % L::kPieces;
    if constexpr (!SMALL) {
      if (key0 + KEYS <= last + 1) {
#pragma unroll
        for (int g = 0; g < kGroups; ++g)
#pragma unroll
          for (int i = 0; i < kVariants; ++i) x[g * kVariants + i] = load(head, p.at[g], offset[i]);
      } else {
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
          const int first = min(key0 + kRun * g, last & ~(kRun - 1));
#pragma unroll
          for (int i = 0; i < kVariants; ++i) x[g * kVariants + i] = load(head, p.at[g], place(a, min(i * L::kAtOnce + in, last - first), c));
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int key = min(key0 + i * L::kAtOnce + in, last);
        const unsigned page = clampi(table[key >> a.z.shift], 0, a.pages - 1);
        const char* at = reinterpret_cast<const char*>(head) + static_cast<uint64_t>(page) * a.page_bytes +
                         static_cast<unsigned>(key & ((1 << a.z.shift) - 1)) * a.place_bytes + c * 16;
        x[i] = c * 8 < a.z.D ? *reinterpret_cast<const V8*>(at) : V8{};
      }
    }
  }
  template <int STRIDE>
  __device__ __forceinline__ void put(const V8 (&x)[kLoads], T* to) const {
    const int lane = threadIdx.x & 63, in = lane / L::kPieces, c = lane % L::kPieces;
    if (DP % (L::kPieces * 8) != 0 && c * 8 >= DP) return;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) *reinterpret_cast<V8*>(to + (i * L::kAtOnce + in) * STRIDE + c * 8) = x[i];
  }
  __device__ __forceinline__ void put_keys(T* s_k) const { put<L::kStrideK>(k, s_k); }
  __device__ __forceinline__ void put_values(T* s_v) const { put<L::kStrideV>(v, s_v); }
};

// A wave's 32 rows: a lane has row `lane % 32`, with its partner 32 lanes on.
template <class T, int DP>
struct Rows {
  typedef typename Mma<T>::V8 V8;
  typedef Layout<DP> L;
  V8 q[DP / 16];
  f32x16 o[DP / 32];
  float m, l;
  int limit;  // the keys before it are seen
  bool far;   // a maximum of the wave's rows is past kFar
  // Scores' differences from the maximum are taken in one step, s scale - m, from the exact product: it is off by what rounding
  // the maximum's own product left, at most 1/2 up to here, and by the same for all keys. Past it that factor would leave
  // the weights' type (fp16 from 2^27, fp32 from 2^31), and the product is rounded first.
  static constexpr float kFar = 0x1p24f;

  __device__ __forceinline__ void begin(const AttendArgs& a, const Segment& g, int h, int r, bool valid) {
    const Shape& z = a.z;
    const int half = (threadIdx.x & 63) >> 5;
    const int R = g.row0 + (valid ? r : 0);
    const int in = R / z.rows, rest = R - in * z.rows, t = rest / z.G, gq = rest - t * z.G;
    const T* from = static_cast<const T*>(a.q) + (g.seq0 + in) * a.q_stride + t * a.q_token + (h * z.G + gq) * a.q_head;
    limit = g.table < 0 ? g.keys : min(g.keys, g.keys - z.T + t + 1);
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) {
      const int d = c * 16 + half * 8;
      if (d < z.D) q[c] = *reinterpret_cast<const V8*>(from + d);
      else q[c] = V8{};
    }
    // (here, not in the tiles' loop, where the wait would be one for the next tile's loads too)
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) asm volatile("" : "+v"(q[c]));
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) o[d] = f32x16{};
    m = -INFINITY;
    l = 0.0f;
    far = false;
  }

  // Operands of the products: 32 keys' elements 16 c and on; 16 keys' (of a block of 32, `c`) elements 32 d and on.
  static __device__ __forceinline__ V8 key_part(const T* s_k, int c) {
    const int lane = threadIdx.x & 63;
    return *reinterpret_cast<const V8*>(s_k + (lane & 31) * L::kStrideK + (lane >> 5) * 8 + c * 16);
  }
  static __device__ __forceinline__ V8 value_part(const T* s_v, int c, int d) {
    typedef __attribute__((address_space(3))) s16x4* Lds;
    const int lane = threadIdx.x & 63;
    const T* at = s_v + (4 * (lane >> 5) + (lane & 15) / 4 + c * 16) * L::kStrideV + (lane >> 4 & 1) * 16 + (lane & 3) * 4 + d * 32;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(at));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(at + 8 * L::kStrideV));
    return __builtin_bit_cast(V8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  }

  // A pair of weights is worked out here (the compiler would put it behind all products, next to its use) and summed, as
  // rounded.
  __device__ __forceinline__ void pin_pair(V8& w, int i) {
    i32x4 x = __builtin_bit_cast(i32x4, w);
    int y = x[i];
    asm volatile("" : "+v"(y));
    x[i] = y;
    w = __builtin_bit_cast(V8, x);
    l = Mma<T>::add_pair(y, l);
  }

  // A block of 32 keys in a pipeline of three: the next block's scores (QK), this block's weights, and the products of
  // the last block's weights and values (PV). Matrix and vector instructions are independent of each other and
  // alternate.
  //
  // The order of the reads of LDS and of the products is the one written here (kOrder lets only scalar and vector
  // arithmetic move past it): left to itself the compiler reads a product's operand right before it and waits. Reads
  // are kAhead products ahead.
  template <bool QK, bool PV>
  __device__ __forceinline__ void step(f32x16& s, V8 (&p)[2], const T* s_k, const T* s_v, int key0, int least, float scale) {
    constexpr int kOrder = 0, kAhead = 4, DT = DP / 32, N = (QK ? DP / 16 : 0) + (PV ? 2 * DT : 0);
    const int half = (threadIdx.x & 63) >> 5;
    // (the scores' products, each of which waits for the one before, alternate with the values', which do not)
    auto part = [&](auto f) {
      constexpr int i = QK && PV ? f.value / 2 : f.value;
      if constexpr (QK && !(PV && f.value % 2)) return key_part(s_k, i);
      else return value_part(s_v, i / DT, i % DT);
    };
    V8 parts[kAhead];
    each<(N < kAhead ? N : kAhead)>([&](auto f) { parts[f.value] = part(f); });
    __builtin_amdgcn_sched_barrier(kOrder);
    if (key0 + 32 > least) {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (key0 + 8 * (i / 4) + 4 * half + i % 4 >= limit) s[i] = -INFINITY;
    }
    float most = s[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) most = fmaxf(most, s[i]);
    most = fmaxf(most, other_half(most)) * scale;
    // (weights of up to 2^8 instead of 1: the sums are fp32, and hardly a block moves the maximum by more)
    const bool up = __any(most > m + 8.0f);
    float by = 1.0f;
    if (up || far) {
      const float now = up ? fmaxf(m, most) : m;
      by = now == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - now);
      m = now;
      l *= by;
      far = __any(fabsf(m) > kFar && m != -INFINITY);
      if (far) {
        const float back = 1.0f / scale, from = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = rounded_apart(s[i], scale, from) * back;
      }
    }
    const float from = far || m == -INFINITY ? 0.0f : m;
    f32x16 next{};
    V8 w[2];
    auto weights = [&](auto from_pair, auto to_pair) {
      each<to_pair.value - from_pair.value>([&](auto j) {
        constexpr int i = from_pair.value + j.value;
        w[i / 4][i % 4 * 2] = static_cast<T>(__builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * i], scale, -from)));
        w[i / 4][i % 4 * 2 + 1] = static_cast<T>(__builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * i + 1], scale, -from)));
        pin_pair(w[i / 4], i % 4);
      });
    };
    each<N>([&](auto f) {
      __builtin_amdgcn_sched_barrier(kOrder);
      constexpr int i = QK && PV ? f.value / 2 : f.value;
      if constexpr (QK && !(PV && f.value % 2)) next = Mma<T>::mma(parts[f.value % kAhead], q[i], next);
      else o[i % DT] = Mma<T>::mma(parts[f.value % kAhead], p[i / DT], o[i % DT]);
      if constexpr (f.value + kAhead < N) parts[f.value % kAhead] = part(Number<f.value + kAhead>{});
      weights(Number<8 * f.value / N>{}, Number<8 * (f.value + 1) / N>{});
    });
    if constexpr (N == 0) weights(Number<0>{}, Number<8>{});
    __builtin_amdgcn_sched_barrier(kOrder);
    if (up) {
#pragma unroll
      for (int d = 0; d < DT; ++d) o[d] *= by;
    }
    p[0] = w[0];
    p[1] = w[1];
    if (QK) s = next;
  }
  __device__ __forceinline__ void first_scores(f32x16& s, const T* s_k) {
    s = f32x16{};
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) s = Mma<T>::mma(key_part(s_k, c), q[c], s);
  }
  __device__ __forceinline__ void last_values(const V8 (&p)[2], const T* s_v) {
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int d = 0; d < DP / 32; ++d) o[d] = Mma<T>::mma(value_part(s_v, c, d), p[c], o[d]);
  }
  // A block alone.
  __device__ __forceinline__ void block(const T* s_k, const T* s_v, int key0, int least, float scale) {
    f32x16 s;
    V8 p[2];
    first_scores(s, s_k);
    step<false, false>(s, p, s_k, s_v, key0, least, scale);
    last_values(p, s_v);
  }

  // The rows' outputs where no other stretch has any of them, else their part.
  __device__ __forceinline__ void end(const AttendArgs& a, const Lines& lines, const Segment& g, bool wide, int h, int w, int r,
                                      bool valid, bool whole, bool from_start) {
    const Shape& z = a.z;
    const int half = (threadIdx.x & 63) >> 5;
    l += other_half(l);
    if (!valid) return;
    if (whole && (g.rows & kAlone)) {
      const int R = g.row0 + r, t = R / z.G, gq = R - t * z.G;
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
      return;
    }
    const int64_t row = partial_row(a, lines, wide, g.table < 0, g.index, h, w, whole, from_start) + r;
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
};

// DP: the head's elements, rounded up to a width there is.
template <class T, int DP, bool SMALL>
__global__ __launch_bounds__(kWaves * 64, DP > 128 ? 1 : 2) void k_attend(AttendArgs a) {
  typedef Layout<DP> L;
  typedef typename Mma<T>::V8 V8;
  constexpr int kWideK = kWideKeys * L::kStrideK, kWideV = kWideKeys * L::kStrideV;
  constexpr int kWaveK = kNarrowKeys * L::kStrideK, kWaveV = kNarrowKeys * L::kStrideV;
  constexpr int kWords = 2 * (kWideK + kWideV) > kWaves * (kWaveK + kWaveV) ? 2 * (kWideK + kWideV) : kWaves * (kWaveK + kWaveV);
  __shared__ __align__(16) T lds[kWords];
  const Shape& z = a.z;
  const Plan plan = plan_at(z, a.plan);
  const Lines lines = uniform(plan.lines);
  // 256 workgroups (one a CU) for wide segments, 256 for narrow ones, and so on: where there are both, a CU has one that
  // computes beside one that waits for memory. (Workgroups for both in turn take 30 registers more, which are not there.)
  const int block = blockIdx.x, group = stretch_of((block >> 9) * 256 + (block & 255), z.wgs);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  auto places_of = [&](int units, int per, int w) {  // of a stretch
    const int64_t left = static_cast<int64_t>(units) * z.Hkv - static_cast<int64_t>(w) * per;
    return static_cast<int>(min(max(left, static_cast<int64_t>(0)), static_cast<int64_t>(per)));
  };

  if (!(block & 256)) {  // wide segments: the workgroup's
    const Start start = uniform(plan.wide_start + group);
    // (a stretch behind the line has no places, and its start holds nothing)
    const int places = places_of(lines.wide_units, lines.wide_per, group);
    int left = places ? places - start.lead : 0, h = start.head, seg = start.segment, tile = start.tile;
    Segment g = start.first;
    if (left > 0) {
      T *s_k = lds, *s_v = lds + 2 * kWideK;
      constexpr int kShare = kWideKeys / kWaves;  // keys that a wave brings
      T *put_k = s_k + wave * kShare * L::kStrideK, *put_v = s_v + wave * kShare * L::kStrideV;
      for (;; tile = 0) {
        const int next = seg + 1 == lines.n_wide ? 0 : seg + 1;
        const Segment following = uniform(plan.wide + next);
        const int n = min(left, g.tiles - tile), n_rows = g.rows & (kAlone - 1);
        left -= n;
        const int r = wave * 32 + (lane & 31);
        const bool busy = wave * 32 < n_rows, valid = r < n_rows;
        Stage<T, DP, kShare, SMALL> in;
        typedef typename Stage<T, DP, kShare, SMALL>::Pages Pages;
        in.begin(a, g, h);
        const int key0 = tile * kWideKeys, mine = key0 + wave * kShare;
        // Keys of tile t + 1 and values of tile t go to LDS between the two blocks of tile t: what they take the place of
        // was read before the barrier in tile t - 1.
        const Pages pages = in.look_up(a, mine);
        in.fetch(in.k, in.k_head, pages, a, mine);
        in.fetch(in.v, in.v_head, pages, a, mine);
        Pages ahead = in.look_up(a, mine + kWideKeys);
        Rows<T, DP> rows;
        if (busy) rows.begin(a, g, h, r, valid);
        const int least = g.table < 0 ? g.keys : min(g.keys, g.keys - z.T + 1 + (g.row0 + wave * 32) / z.G);  // of the wave's rows
        __syncthreads();  // (the segment before is read)
        in.put_keys(put_k);
        if (n > 1) in.fetch(in.k, in.k_head, ahead, a, mine + kWideKeys);
        __syncthreads();
        auto keys_of = [&](int t) { return s_k + (t & 1) * kWideK; };
        auto values_of = [&](int t) { return s_v + (t & 1) * kWideV; };
        auto middle = [&](int t) {
          in.put_values(put_v + (t & 1) * kWideV);
          if (t + 1 < n) {
            in.put_keys(put_k + ((t + 1) & 1) * kWideK);
            const Pages next = in.look_up(a, mine + (t + 2) * kWideKeys);
            in.fetch(in.v, in.v_head, ahead, a, mine + (t + 1) * kWideKeys);
            in.fetch(in.k, in.k_head, next, a, mine + (t + 2) * kWideKeys);  // (behind the last tile: its last keys again)
            ahead = next;
          }
          __syncthreads();
        };
        constexpr int kSecondK = 32 * L::kStrideK, kSecondV = 32 * L::kStrideV;
        if (busy) {
          f32x16 s;
          V8 p[2];
          rows.first_scores(s, s_k);
          rows.template step<true, false>(s, p, s_k + kSecondK, s_v, key0, least, a.scale);
          middle(0);
          for (int t = 0; t + 1 < n; ++t) {
            const int key = key0 + t * kWideKeys;
            rows.template step<true, true>(s, p, keys_of(t + 1), values_of(t), key + 32, least, a.scale);
            rows.template step<true, true>(s, p, keys_of(t + 1) + kSecondK, values_of(t) + kSecondV, key + 64, least, a.scale);
            middle(t + 1);
          }
          rows.template step<false, true>(s, p, s_k, values_of(n - 1), key0 + (n - 1) * kWideKeys + 32, least, a.scale);
          rows.last_values(p, values_of(n - 1) + kSecondV);
        } else {
          for (int t = 0; t < n; ++t) middle(t);
        }
        if (busy) rows.end(a, lines, g, true, h, group, r, valid, n == g.tiles, tile == 0);
        left -= kLead;
        if (left <= 0) break;
        if (!next) ++h;
        seg = next;
        g = following;
      }
    }
  } else {  // narrow segments: each wave's
    const int w = group * kWaves + wave;
    const Start start = uniform(plan.narrow_start + w);
    // (a stretch behind the line has no places, and its start holds nothing)
    const int places = places_of(lines.narrow_units, lines.narrow_per, w);
    int left = places ? places - start.lead : 0, h = start.head, seg = start.segment, tile = start.tile;
    Segment g = start.first;
    if (left > 0) {
      T *s_k = lds + wave * (kWaveK + kWaveV), *s_v = s_k + kWaveK;
      for (;; tile = 0) {
        const int next = seg + 1 == lines.n_narrow ? 0 : seg + 1;
        const Segment following = uniform(plan.narrow + next);
        const int n = min(left, g.tiles - tile), n_rows = g.rows & (kAlone - 1);
        left -= n;
        const int r = lane & 31;
        const bool valid = r < n_rows;
        Stage<T, DP, kNarrowKeys, SMALL> in;
        typedef typename Stage<T, DP, kNarrowKeys, SMALL>::Pages Pages;
        in.begin(a, g, h);
        const int key0 = tile * kNarrowKeys;
        const Pages pages = in.look_up(a, key0);
        in.fetch(in.k, in.k_head, pages, a, key0);
        in.fetch(in.v, in.v_head, pages, a, key0);
        Pages ahead = in.look_up(a, key0 + kNarrowKeys);
        Rows<T, DP> rows;
        rows.begin(a, g, h, r, valid);
        const int least = g.table < 0 ? g.keys : min(g.keys, g.keys - z.T + 1 + g.row0 / z.G);
        for (int it = 0; it < n; ++it) {
          const int key = key0 + it * kNarrowKeys;
          wave_order();  // (the tile before is read)
          in.put_keys(s_k);
          in.put_values(s_v);
          if (it + 1 < n) {
            in.fetch(in.k, in.k_head, ahead, a, key + kNarrowKeys);
            in.fetch(in.v, in.v_head, ahead, a, key + kNarrowKeys);
            ahead = in.look_up(a, key + 2 * kNarrowKeys);
          }
          wave_order();
          rows.block(s_k, s_v, key, least, a.scale);
        }
        rows.end(a, lines, g, false, h, w, r, valid, n == g.tiles, tile == 0);
        left -= kLead;
        if (left <= 0) break;
        if (!next) ++h;
        seg = next;
        g = following;
      }
    }
  }
}

// WAVES waves join a row's stretches: o = sum_i 2^(m_i - m) o_i / sum_i 2^(m_i - m) l_i. (Where there are few rows, one
// has many stretches: 16 waves take them at once. A sequence of 30000 positions, 8 key heads: attention and joining 65 us with
// one wave a row, 33 with 16.) Bound by its three loads one behind the other: 6 us for 128 rows, 13 for 8192.
template <class T, int DP, int WAVES>
__global__ __launch_bounds__(WAVES == 1 ? 256 : WAVES * 64) void k_join(AttendArgs a) {
  const Shape& z = a.z;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), share = WAVES == 1 ? 0 : wave;
  const unsigned id = WAVES == 1 ? (blockIdx.y * kGridX + blockIdx.x) * 4 + wave : blockIdx.x;
  if (id >= static_cast<unsigned>(z.S) * z.T * z.H) return;
  const unsigned st = id / static_cast<unsigned>(z.H);
  const int hq = static_cast<int>(id - st * z.H), s = static_cast<int>(st / static_cast<unsigned>(z.T)), t = static_cast<int>(st) - s * z.T;
  const int h = hq / z.G, r = t * z.G + hq % z.G;
  const Plan plan = plan_at(z, a.plan);
  const Lines lines = uniform(plan.lines);
  const Place own = uniform(plan.own + static_cast<int64_t>(s) * z.own_tiles + r / kRows);
  const PrefixPlace pre = uniform(plan.prefix + s);
  T* to = static_cast<T*>(a.out) + static_cast<int64_t>(id) * z.D;
  constexpr int E = DP > 128 ? 4 : DP > 64 ? 2 : 1;  // elements of a lane, side by side
  typedef float V __attribute__((ext_vector_type(E)));
  const bool mine = lane * E < z.D;
  auto write = [&](V x) {
    typedef T TV __attribute__((ext_vector_type(E)));
    TV y;
#pragma unroll
    for (int e = 0; e < E; ++e) y[e] = static_cast<T>(x[e]);
    if (mine && !share) *reinterpret_cast<TV*>(to + lane * E) = y;
  };
  if (own.keys - z.T + t + 1 <= 0) return write(V{});  // no token
  const bool own_wide = z.rows > kNarrow, pre_wide = pre.row0 < 0;
  auto stretches = [&](bool wide, int unit, int tiles, int& first) {
    const uint64_t u = static_cast<uint64_t>(h) * (wide ? lines.wide_units : lines.narrow_units) + unit, last = u + tiles - 1;
    const unsigned per = wide ? lines.wide_per : lines.narrow_per;
    const bool small = last >> 32 == 0;
    first = static_cast<int>(small ? static_cast<unsigned>(u) / per : u / per);
    return static_cast<int>(small ? static_cast<unsigned>(last) / per : last / per) - first + 1;
  };
  int first_own, first_pre = 0, n_pre = 0;
  const int n_own = stretches(own_wide, own.unit, own.tiles, first_own);
  if (!pre.tiles && n_own == 1) return;  // (written already)
  const int R = (pre_wide ? ~pre.row0 : pre.row0) + r, segment = pre_wide ? R / kRows : 0;
  if (pre.tiles) n_pre = stretches(pre_wide, pre.unit + segment * (pre.tiles + kLead), pre.tiles, first_pre);
  const int n = n_pre + n_own;
  auto row_of = [&](int i) {  // the prefix's stretches, then the sequence's own
    if (i < n_pre)
      return partial_row(a, lines, pre_wide, true, pre.index + segment, h, first_pre + i, n_pre == 1, i == 0) + (pre_wide ? R % kRows : R);
    i -= n_pre;
    return partial_row(a, lines, own_wide, false, own.index, h, first_own + i, n_own == 1, i == 0) + r % kRows;
  };
  if (n <= 8) {  // all at once: what each stretch says of the row by scalar loads
    if (share) return;
    V x[8];
    float2 ml[8];
    each<8>([&](auto i) {
      x[i.value] = V{};
      ml[i.value] = make_float2(-INFINITY, 0.0f);
      if (i.value < n) {
        const int64_t row = row_of(i.value);
        ml[i.value] = uniform(a.ml + row);
        if (mine) x[i.value] = *reinterpret_cast<const V*>(a.o + row * z.D + lane * E);
      }
    });
    float most = -INFINITY, total = 0.0f;
    each<8>([&](auto i) { most = fmaxf(most, ml[i.value].x); });
    if (most == -INFINITY) most = 0.0f;
    V o = {};
    each<8>([&](auto i) {
      const float by = ml[i.value].y == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(ml[i.value].x - most);
      total += by * ml[i.value].y;
      o += by * x[i.value];
    });
    return write(o * (total == 0.0f ? 0.0f : 1.0f / total));
  }
  const int each_wave = (n + WAVES - 1) / WAVES, begin = share * each_wave, end = min(begin + each_wave, n);
  float most = -INFINITY;
  for (int i = begin + lane; i < end; i += 64) most = fmaxf(most, a.ml[row_of(i)].x);
#pragma unroll
  for (int d = 32; d; d >>= 1) most = fmaxf(most, __shfl_xor(most, d));
  const float from = most == -INFINITY ? 0.0f : most;
  float total = 0.0f;
  V o = {};
  for (int base = begin; base < end; base += 64) {
    float by = 0.0f;
    if (base + lane < end) {
      const float2 ml = a.ml[row_of(base + lane)];
      by = ml.y == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(ml.x - from);
      total += by * ml.y;
    }
    const int m = min(end - base, 64);
    for (int i = 0; i < m; i += 16) {
      V x[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        x[j] = V{};
        if (i + j < m && mine) x[j] = *reinterpret_cast<const V*>(a.o + row_of(base + i + j) * z.D + lane * E);
      }
#pragma unroll
      for (int j = 0; j < 16; ++j) o += __shfl(by, min(i + j, 63)) * x[j];
    }
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) total += __shfl_xor(total, d);
  if constexpr (WAVES > 1) {
    __shared__ V s_o[WAVES][64];
    __shared__ float2 s_ml[WAVES];
    s_o[wave][lane] = o;
    if (!lane) s_ml[wave] = make_float2(most, total);
    __syncthreads();
    if (share) return;
    float all = -INFINITY;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) all = fmaxf(all, s_ml[w].x);
    if (all == -INFINITY) all = 0.0f;
    total = 0.0f;
    o = V{};
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const float2 ml = s_ml[w];
      const float by = ml.y == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(ml.x - all);
      total += by * ml.y;
      o += by * s_o[w][lane];
    }
  }
  write(o * (total == 0.0f ? 0.0f : 1.0f / total));
}

}  // namespace vpg
