// Beam search's selection: for each request the n best continuations over its W beams and the whole
// vocabulary, by score[w] + log_softmax(x[w])[v].
//
// Two launches. k_beam_part: one workgroup a segment of a row, held in registers, so that a row is read
// once. A lane's maximum gives a bound: the n-th largest of a wave's 64 lane maxima (n <= 64) is at most the
// segment's n-th largest logit, and few elements reach the largest of the four waves' bounds (about
// 64 ln(64 / (64 - n)) a wave where the logits come in any order); above n = 8 the n-th largest of the workgroup's 256
// lane maxima is taken, with about as many elements above it as n. The vectors that hold one go to LDS, their
// elements' exponentials are taken in fp64 and added in fixed point, and those that reach the bound are ranked by
// counting: the first n are the segment's candidates in order. The other vectors, all below the bound, add their
// fp32 exponentials. So neither do the large terms lose precision nor does the order of the list, which varies,
// show in the sum: the beams of a request are compared across their rows by these sums. (The fp32 terms: two roundings of
// the exponent, v_exp_f32's ulp and a thread's sum of at most 64 are 46 2^-23 of the sum at most, 13.2 being the mean
// distance from the maximum that 524288 ids allow. In fp32, because their issue bounds the launch.)
// k_beam_merge: one workgroup a request. The rows' normalisers from the segments' sums; lane maxima of the segments'
// candidates' scores bound the request's n-th best in the same way; the few candidates that reach it are ranked.
//
// Measured on an MI355X: 64 x 4 rows of 151936 bf16 logits, n = 8: 20.7 us, 3.8 TB/s; 24 x 16 rows of 262144, n = 16: 39.5,
// 5.1 TB/s: vector issue, 700 to 713 instructions a wave of which 324 are an element's own (8 vectors a thread: fewer leave more
// waves with the same overhead, 23 and 56 us with 4). The merges 5.4 and 10.0; n = 32 and 64 of the former in all 29 and 36 us.
//
// A row with a NaN, an infinite maximum or no finite logit has no candidates, nor have logits of -inf.
// Rows of finished beams and of beams whose score is not finite are not read.
#pragma once

#include "rows.cuh"

namespace vo {

constexpr int kMaxBeams = 64;
constexpr int kMaxPick = 64;        // most continuations a request: a lane each
constexpr int kPartThreads = 256;
constexpr int kPartWaves = kPartThreads / kWave;
constexpr int kPartVecs = 512;      // a segment's vectors that hold candidates
constexpr int kPartList = 512;      // its candidates before they are ranked
constexpr int kMergeList = 1024;    // a request's
constexpr int kMergeMaxThreads = 1024;
constexpr int kMergeHeads = 512;
constexpr int kAhead = 4;           // entries that a thread loads at once
constexpr double kFix = 2251799813685248.0;  // 2^51
static_assert(kPartVecs * 8 * kFix < 18446744073709551616.0, "a sum of all listed elements' terms holds in 64 bits");

struct BeamArgs {
  const void* logits;  // row (b, w) at b * rstride + w * bstride
  int64_t rstride, bstride;
  int B, W, V, n;
  int S;               // segments a row, at most 64
  const float* scores;      // [B, W]
  const uint8_t* finished;  // [B, W] or null
  int pad, keep;
  uint32_t row_magic, list_magic;  // for divisions by S n and n
  u64* keys;           // [B W, S, n] the segments' candidates, descending (0: none)
  double* sums;        // [B W, S] sums of exp(x - max)
  float* maxs;         // [B W, S]
  float* out_scores;   // [B, n]
  int32_t* out_beams;
  int32_t* out_tokens;
};

// The n-th largest of the wave's 64 N keys, N a lane, with the bits below LOW cleared: at most the key itself. A step
// is scalar but for its compares.
template <int LOW, int N>
__device__ __forceinline__ uint32_t wave_nth_floor_of(const uint32_t* keys, int n) {
  uint32_t t = 0;
#pragma unroll
  for (int b = 31; b >= LOW; --b) {
    const uint32_t c = t | (1u << b);
    int count = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) count += __popcll(__ballot(keys[i] >= c));
    if (count >= n) t = c;
  }
  return t;
}
template <int LOW>
__device__ __forceinline__ uint32_t wave_nth_floor(uint32_t key, int n) {
  return wave_nth_floor_of<LOW, 1>(&key, n);
}

// How many of the first c words are larger than k, and how many equal it; the words behind them, up to a multiple of
// kRankStep, are 0. (kRankStep words a step: one at a time each read would wait for the last.)
constexpr int kRankStep = 8;
__device__ __forceinline__ uint32_t rank_of(const u64* words, uint32_t c, u64 k, uint32_t* equal) {
  uint32_t r = 0, e = 0;
#pragma unroll 1
  for (uint32_t j = 0; j < c; j += kRankStep) {
    u64 x[kRankStep];
#pragma unroll
    for (int i = 0; i < kRankStep; ++i) x[i] = words[j + i];
#pragma unroll
    for (int i = 0; i < kRankStep; ++i) {
      r += x[i] > k;
      e += x[i] == k;
    }
  }
  *equal = e;
  return r;
}

__device__ __forceinline__ u64 pack_key(float x, int id) {
  return (static_cast<u64>(key_of(x)) << 32) | (0xFFFFFFFFu - static_cast<uint32_t>(id));
}
__device__ __forceinline__ float key_value(u64 k) { return val_of(static_cast<uint32_t>(k >> 32)); }
__device__ __forceinline__ int key_id(u64 k) { return static_cast<int>(0xFFFFFFFFu - static_cast<uint32_t>(k)); }

// A term e in [0, 1] of a sum whose order varies: rint(e 2^51).
__device__ __forceinline__ u64 fixed(double e) { return static_cast<u64>(__builtin_rint(e * kFix)); }

struct PartShared {
  uint4 vec[kPartVecs];  // the vectors with an element at or above the bound
  int32_t vid[kPartVecs];  // their first ids
  u64 list[kPartList + kRankStep];  // those elements
  double wsum[kPartWaves];
  u64 wfix[kPartWaves];
  float wmax[kPartWaves];
  uint32_t wtau[kPartWaves];
  uint32_t lane_max[kPartThreads];
  uint32_t wcnt[kPartWaves];
  uint32_t vecs, count;
};

// f(x, id) for each of this thread's elements of the segment, read again.
template <class Tin, int NV, class F>
__device__ __forceinline__ void each_again(const Tin* row, int V, int first, F f) {
  constexpr int E = Vec<Tin>::kElems;
#pragma unroll 1
  for (int j = 0; j < NV; ++j) {
    const int at = first + j * kPartThreads * E;
    uint4 d;
    load_segment<Tin, 1, kPartThreads>(row, V, at, &d);
    float x[E];
    Vec<Tin>::unpack(d, x);
#pragma unroll
    for (int e = 0; e < E; ++e) f(x[e], at + static_cast<int>(threadIdx.x) * E + e);
  }
}

// Segments with more elements at or above the bound than the list takes (equal logits, or few lanes with a
// finite one): the n-th largest key, ids included, bit by bit between the bound and the largest key (a count of the
// segment each, read again from the cache: held in registers, its keys would take 238 a lane, and the ordinary segments'
// occupancy; 256 constant rows of 151936 bf16 logits 215 us in all, random ones 24), and this thread's part of the whole segment's sum.
template <class Tin, int NV>
__device__ __forceinline__ double part_crowded(const Tin* row, int V, int first, int n, float ref, uint32_t bound,
                                               PartShared& sh) {
  constexpr int kSpan = NV * kPartThreads * Vec<Tin>::kElems;
  const int w = threadIdx.x / kWave;
  auto total = [&](uint32_t c) {
    c = wave_sum(c);
    __syncthreads();
    if (lane_id() == 0) sh.wcnt[w] = c;
    __syncthreads();
    uint32_t t = 0;
#pragma unroll
    for (int i = 0; i < kPartWaves; ++i) t += sh.wcnt[i];
    return t;
  };
  double s = 0.0;
  uint32_t c = 0;
  each_again<Tin, NV>(row, V, first, [&](float x, int) {
    s += static_cast<double>(__builtin_amdgcn_exp2f((x - ref) * kLog2e));
    c += finite_f(x);
  });
  const uint32_t live = total(c);
  const uint32_t want = live < static_cast<uint32_t>(n) ? live : static_cast<uint32_t>(n);
  u64 kn = 0;
  if (live > want) {  // (uniform)
    uint32_t have = 0xFFFFFFFFu;
    auto step = [&](int b) {
      const u64 cand = kn | (1ull << b);
      c = 0;
      each_again<Tin, NV>(row, V, first, [&](float x, int id) { c += finite_f(x) && pack_key(x, id) >= cand; });
      c = total(c);
      if (c >= want) {
        kn = cand;
        have = c;
      }
    };
    // the value: the bits that the bound and the largest share are its own, unless the largest alone is enough
    const uint32_t top = key_of(ref);
    c = 0;
    each_again<Tin, NV>(row, V, first, [&](float x, int) { c += x == ref; });
    if (total(c) >= want) {
      kn = static_cast<u64>(top) << 32;
    } else {
      constexpr int kLow = sizeof(Tin) == 2 ? 16 : 0;  // (bf16: the bits below repeat the sign)
      const uint32_t differ = top ^ bound;
      int b = differ ? 31 - __clz(differ) : -1;
      kn = static_cast<u64>(b < 31 ? top >> (b + 1) << (b + 1) : 0u) << 32;
#pragma unroll 1
      for (; b >= kLow && have != want; --b) step(32 + b);
      if (kLow && !(kn >> 63)) kn |= 0xFFFFull << 32;
    }
    // the id: likewise, within the segment
    if (have != want) {
      const uint32_t high = 0xFFFFFFFFu - static_cast<uint32_t>(first);
      int b = 31 - __clz(high ^ (high - (kSpan - 1)));
      kn |= high >> (b + 1) << (b + 1);
#pragma unroll 1
      for (; b >= 0 && have != want; --b) step(b);
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) sh.count = 0;
  __syncthreads();
  each_again<Tin, NV>(row, V, first, [&](float x, int id) {
    if (finite_f(x) && pack_key(x, id) >= kn) {
      const uint32_t at = atomicAdd(&sh.count, 1u);
      if (at < kPartList) sh.list[at] = pack_key(x, id);
    }
  });
  __syncthreads();
  return s;
}

// MANY: the n-th largest of all the workgroup's lane maxima, not of a wave's: fewer elements reach it.
template <class Tin, int NV, bool MANY>
__global__ __launch_bounds__(kPartThreads) void k_beam_part(BeamArgs a) {
  constexpr int E = Vec<Tin>::kElems;
  __shared__ PartShared sh;
  const int tid = threadIdx.x, w = tid / kWave;
  // (a grid of segments, beams and requests)
  const int seg = blockIdx.x, row = blockIdx.z * a.W + blockIdx.y;
  const int64_t part = static_cast<int64_t>(row) * a.S + seg;
  const float score = a.scores[row];
  const int finished = a.finished ? a.finished[row] : 0;  // (both loads at once)
  if (!finite_f(score) || finished) return;  // (uniform)
  const Tin* p = as_global(static_cast<const Tin*>(a.logits)) + blockIdx.z * a.rstride + blockIdx.y * a.bstride;
  const int first = seg * NV * kPartThreads * E;
  uint4 d[NV];
  load_segment<Tin, NV, kPartThreads>(p, a.V, first, d);
  if (tid == 0) sh.vecs = sh.count = 0;
  exp_table_init();
  float lm = -__builtin_inff();
  float vm[NV];  // each vector's largest
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    vm[j] = Vec<Tin>::largest(d[j]);
    lm = max_nan(lm, vm[j]);
    __builtin_amdgcn_sched_barrier(0);  // (a vector at a time: 64 registers)
  }
  // (NaN where the wave holds one: wave_max_f passes NaNs over)
  const float wm = __ballot(lm != lm) ? __builtin_nanf("") : wave_max_f(lm);
  forget<NV>(d);
  if constexpr (MANY) {
    sh.lane_max[tid] = key_of(lm);
  } else {
    const uint32_t tau = wave_nth_floor<16>(key_of(lm), a.n);
    if (lane_id() == 0) sh.wtau[w] = tau;
  }
  if (lane_id() == 0) sh.wmax[w] = wm;
  __syncthreads();
  float M = sh.wmax[0];
#pragma unroll
  for (int i = 1; i < kPartWaves; ++i) M = max_nan(M, sh.wmax[i]);
  uint32_t tk = 0;
  if constexpr (MANY) {
    uint32_t k[kPartWaves];
#pragma unroll
    for (int i = 0; i < kPartWaves; ++i) k[i] = sh.lane_max[i * kWave + lane_id()];
    tk = wave_nth_floor_of<16, kPartWaves>(k, a.n);
  } else {
#pragma unroll
    for (int i = 0; i < kPartWaves; ++i) tk = max(tk, sh.wtau[i]);
  }
  const float ref = M == -__builtin_inff() ? 0.0f : M;  // (no finite logit: exp(-inf - 0) = 0)
  // (a bound below every finite number takes all of them, and never -inf)
  constexpr float kLowest = -3.4028234663852886e38f;
  const float bound = tk <= key_of(kLowest) ? kLowest : val_of(tk);
  // The few vectors that reach the bound go to the list, and out of this thread's sum. (A NaN reaches none, and
  // stays in the sum.)
  const float refl = ref * kLog2e;
  float s = 0.0f;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    if (vm[j] >= bound) {
      const uint32_t at = atomicAdd(&sh.vecs, 1u);
      if (at < kPartVecs) {
        sh.vec[at] = d[j];
        sh.vid[at] = first + (j * kPartThreads + tid) * E;
      }
      d[j] = make_uint4(Vec<Tin>::kNegInf, Vec<Tin>::kNegInf, Vec<Tin>::kNegInf, Vec<Tin>::kNegInf);
    }
    float x[E];
    Vec<Tin>::unpack(d[j], x);
#pragma unroll
    for (int e = 0; e < E; ++e) s += __builtin_amdgcn_exp2f(__builtin_fmaf(x[e], kLog2e, -refl));
    __builtin_amdgcn_sched_barrier(0);
  }
  double sd = s;
  __syncthreads();
  const uint32_t nv = sh.vecs;
  u64 fx = 0;
  if (nv <= kPartVecs) {  // (uniform)
    for (uint32_t i = tid; i < nv * E; i += kPartThreads) {
      const int e = i % E;
      const float x = word_value<E>(reinterpret_cast<const uint32_t*>(&sh.vec[i / E])[e * 4 / E], e & 1);
      if (x >= bound) {
        const uint32_t at = atomicAdd(&sh.count, 1u);
        if (at < kPartList) sh.list[at] = pack_key(x, sh.vid[i / E] + e);
      }
      fx += fixed(exp_nonpos(static_cast<double>(x) - static_cast<double>(ref)));
    }
  }
  __syncthreads();
  // A segment with a NaN or an infinite largest has no candidates (nor has its row), and its lane maxima bound nothing: it never
  // counts as crowded, and its list is dropped.
  const bool live = finite_f(M);  // (uniform, as all here)
  uint32_t c = live ? sh.count : 0;
  // (or logits so large that the reference's rounding would be all of the sum: masks of the type's lowest value, say)
  const bool crowded = live && (nv > kPartVecs || c > kPartList || fabsf(M) > 65536.0f);
  if (crowded) {
    sd = part_crowded<Tin, NV>(p, a.V, first, a.n, ref, tk, sh);
    fx = 0;
    c = min(sh.count, static_cast<uint32_t>(kPartList));  // (n at most)
  }
  // ranks by counting (keys differ)
  const uint32_t n = static_cast<uint32_t>(a.n);
  u64* out = a.keys + part * a.n;
  if (tid < kRankStep) sh.list[c + tid] = 0;
  __syncthreads();
  for (uint32_t i = tid; i < c; i += kPartThreads) {
    const u64 k = sh.list[i];
    uint32_t equal = 0;
    const uint32_t r = rank_of(sh.list, c, k, &equal);
    if (r < n) out[r] = k;
  }
  for (uint32_t i = c + tid; i < n; i += kPartThreads) out[i] = 0;
  sd = wave_sum(sd);
  fx = wave_sum(fx);
  if (lane_id() == 0) {
    sh.wsum[w] = sd;
    sh.wfix[w] = fx;
  }
  __syncthreads();
  if (tid == 0) {
    double t = 0.0;
    u64 f = 0;
#pragma unroll
    for (int i = 0; i < kPartWaves; ++i) {
      t += sh.wsum[i];
      f += sh.wfix[i];
    }
    // (x kLog2e - refl = (x - ref) kLog2e + (ref kLog2e - refl): the latter, refl's rounding, is exact in fp64)
    if (!crowded) t *= exp((refl - static_cast<double>(ref) * static_cast<double>(kLog2e)) * 0.6931471805599453);
    a.sums[part] = t + static_cast<double>(f) * (1.0 / kFix);
    a.maxs[part] = M;
  }
}

// ---- the request's best ---------------------------------------------------------------------------
struct MergeShared {
  u64 sk[kMergeList + kRankStep];  // a candidate's score, ordered
  u64 tb[kMergeList];  // what decides between equal scores
  uint32_t head[kMergeHeads];  // the upper words of the lists' first scores, lists that share one by their largest
  double top[kMaxBeams], logs[kMaxBeams];  // a row's largest logit, and the log of its sum against it
  double score[kMaxBeams];
  u64 rsk[kMergeMaxThreads / kWave], rtb[kMergeMaxThreads / kWave];
  float ch_score[kMaxPick];
  int32_t ch_beam[kMaxPick], ch_token[kMaxPick];
  int32_t kind[kMaxBeams];  // 0: no candidates, 1: its row's, 2: finished
  uint32_t count, bound;
};

// i / d for i d < 2^32, with magic = 2^32 / d + 1 (host).
__device__ __forceinline__ int quotient(int i, int d, uint32_t magic) {
  return d == 1 ? i : static_cast<int>(__umulhi(static_cast<uint32_t>(i), magic));
}

__device__ __forceinline__ u64 ordered(double x) {
  const u64 b = static_cast<u64>(__double_as_longlong(x + 0.0));
  return (b >> 63) ? ~b : (b | (1ull << 63));
}
__device__ __forceinline__ double unordered(u64 k) {
  return __longlong_as_double(static_cast<long long>((k >> 63) ? (k & ~(1ull << 63)) : ~k));
}
// Equal scores: the lower beam, then the larger logit, then the lower id.
__device__ __forceinline__ u64 tie_word(int beam, u64 key) {
  return (static_cast<u64>(kMaxBeams - 1 - beam) << 52) | ((key >> 32) << 20) | (key & 0xFFFFFull);
}

// The score of entry e, whose key is k, of list l (of W S lists, S a beam), ordered, and its tie word; 0 where
// there is none.
__device__ __forceinline__ u64 merge_score(const MergeShared& sh, int w, bool first, u64 k, u64* tb) {
  const int kind = sh.kind[w];
  if (kind == 1) {
    *tb = tie_word(w, k);
    return k ? ordered((static_cast<double>(key_value(k)) - sh.top[w]) - sh.logs[w] + sh.score[w]) : 0;
  }
  *tb = tie_word(w, pack_key(0.0f, 0));
  return kind == 2 && first ? ordered(sh.score[w]) : 0;
}
// The upper words of ordered fp64 scores order them too, coarsely: the first launch's bound by lane maxima again.
__global__ __launch_bounds__(kMergeMaxThreads) void k_beam_merge(BeamArgs a) {
  __shared__ MergeShared sh;
  const int tid = threadIdx.x, wave = tid / kWave, lane = lane_id(), nt = blockDim.x, nw = nt / kWave;
  const int b = blockIdx.x;
  const int W = a.W, S = a.S, n = a.n;
  // A thread an entry of the segments' lists, kAhead of them at once, and the first ones ahead of the rows' sums.
  const u64* keys = a.keys + static_cast<int64_t>(b) * W * S * n;
  const int total = W * S * n;
  auto load = [&](int i) { return i < total ? ld_global(keys + i) : 0; };
  auto score_of = [&](int i, u64 k, u64* tb) -> u64 {
    if (i >= total) return 0;
    const int w = quotient(i, S * n, a.row_magic);
    return merge_score(sh, w, i == w * S * n, k, tb);
  };
  u64 ahead[kAhead], sk[kAhead], tb[kAhead];
#pragma unroll
  for (int e = 0; e < kAhead; ++e) ahead[e] = load(tid + e * nt);
  for (int w = wave; w < W; w += nw) {
    const int row = b * W + w;
    // (all loads at once; a row that was not read has left whatever the workspace held)
    const float sc = a.scores[row];
    const int finished = a.finished ? a.finished[row] : 0;
    const float m = lane < S ? ld_global(a.maxs + static_cast<int64_t>(row) * S + lane) : -__builtin_inff();
    const double sum = lane < S ? ld_global(a.sums + static_cast<int64_t>(row) * S + lane) : 0.0;
    int kind = 0;
    double l = 0.0;
    const float M = wave_max_f(m);
    if (finite_f(sc)) {
      if (finished) {
        kind = 2;
      } else {
        l = log(wave_sum(sum * exp(static_cast<double>(m) - static_cast<double>(M))));
        kind = finite_f(M) && l - l == 0.0 ? 1 : 0;
      }
    }
    if (lane == 0) {
      sh.kind[w] = kind;
      sh.top[w] = M;
      sh.logs[w] = l;
      sh.score[w] = sc;
    }
  }
  if (tid < n) {
    sh.ch_score[tid] = -__builtin_inff();
    sh.ch_beam[tid] = -1;
    sh.ch_token[tid] = -1;
  }
  if (tid == 0) sh.count = 0;
  for (int i = tid; i < kMergeHeads; i += nt) sh.head[i] = 0;
  __syncthreads();
  // the lists' first entries, as many of each as there is room for, bound the n-th best: the n-th largest of the two
  // largest values of 64 lanes
  const int lists = W * S;
  auto head = [&](int i, u64 score) {
    const int l = quotient(i, n, a.list_magic), at = l + (i - l * n) * lists;
    if (score && (at < kMergeHeads || at < lists))
      atomicMax(&sh.head[at % kMergeHeads], static_cast<uint32_t>(score >> 32));
  };
#pragma unroll
  for (int e = 0; e < kAhead; ++e) {
    sk[e] = score_of(tid + e * nt, ahead[e], &tb[e]);
    head(tid + e * nt, sk[e]);
  }
  for (int i = tid + kAhead * nt; i < total; i += kAhead * nt) {
    u64 k[kAhead], t;
#pragma unroll
    for (int e = 0; e < kAhead; ++e) k[e] = load(i + e * nt);
#pragma unroll
    for (int e = 0; e < kAhead; ++e) head(i + e * nt, score_of(i + e * nt, k[e], &t));
  }
  __syncthreads();
  if (wave == 0) {
    uint32_t h = 0, h1 = 0;
#pragma unroll
    for (int i = 0; i < kMergeHeads / kWave; ++i) {
      const uint32_t x = sh.head[lane + i * kWave];
      h1 = max(h1, min(h, x));
      h = max(h, x);
    }
    const uint32_t two[2] = {h, h1};
    h = wave_nth_floor_of<8, 2>(two, n);
    if (lane == 0) sh.bound = max(h, 1u);
  }
  __syncthreads();
  const uint32_t bound = sh.bound;
  auto take = [&](u64 score, u64 t) {
    if (static_cast<uint32_t>(score >> 32) < bound) return;
    const uint32_t at = atomicAdd(&sh.count, 1u);
    if (at < kMergeList) {
      sh.sk[at] = score;
      sh.tb[at] = t;
    }
  };
#pragma unroll
  for (int e = 0; e < kAhead; ++e) take(sk[e], tb[e]);
  for (int i = tid + kAhead * nt; i < total; i += kAhead * nt) {
    u64 k[kAhead], t;
#pragma unroll
    for (int e = 0; e < kAhead; ++e) k[e] = load(i + e * nt);
#pragma unroll
    for (int e = 0; e < kAhead; ++e) {
      const u64 score = score_of(i + e * nt, k[e], &t);
      take(score, t);
    }
  }
  __syncthreads();
  const uint32_t c = sh.count;
  auto choose = [&](uint32_t r, u64 sk, u64 t) {
    const int w = kMaxBeams - 1 - static_cast<int>(t >> 52);
    sh.ch_score[r] = static_cast<float>(unordered(sk));
    sh.ch_beam[r] = w;
    sh.ch_token[r] = sh.kind[w] == 2 ? a.pad : static_cast<int>(0xFFFFFu - static_cast<uint32_t>(t & 0xFFFFFull));
  };
  if (c <= kWave) {
    // (the first wave alone, a candidate a lane)
    if (wave != 0) return;
    const u64 score = lane < static_cast<int>(c) ? sh.sk[lane] : 0;
    const u64 t = lane < static_cast<int>(c) ? sh.tb[lane] : 0;
    uint32_t r = 0;
    for (uint32_t j = 0; j < c; ++j) {
      const u64 other = readlane64(score, j);
      r += other > score || (other == score && readlane64(t, j) > t);
    }
    if (score && r < static_cast<uint32_t>(n)) choose(r, score, t);
    wave_lds_sync();
  } else if (c <= kMergeList) {
    if (tid < kRankStep) sh.sk[c + tid] = 0;  // (below every score)
    __syncthreads();
    for (uint32_t i = tid; i < c; i += nt) {
      const u64 score = sh.sk[i], t = sh.tb[i];
      uint32_t equal = 0, r = rank_of(sh.sk, c, score, &equal);
      if (equal > 1)
        for (uint32_t j = 0; j < c; ++j) r += sh.sk[j] == score && sh.tb[j] > t;
      if (r < static_cast<uint32_t>(n)) choose(r, score, t);
    }
  } else {
    // (thousands of equal scores: the best one after the last, n times)
    u64 psk = ~0ull, ptb = ~0ull;
    for (int r = 0; r < n; ++r) {
      u64 bsk = 0, btb = 0;
      for (int i = tid; i < total; i += nt) {
        u64 t;
        const u64 score = score_of(i, load(i), &t);
        if (!score || !(score < psk || (score == psk && t < ptb))) continue;
        if (score > bsk || (score == bsk && t > btb)) {
          bsk = score;
          btb = t;
        }
      }
      u64 m = wave_max_u64(bsk);
      u64 mt = wave_max_u64(bsk == m ? btb : 0);
      if (lane == 0) {
        sh.rsk[wave] = m;
        sh.rtb[wave] = mt;
      }
      __syncthreads();
      m = 0;
      mt = 0;
      for (int i = 0; i < nw; ++i) {
        const u64 x = sh.rsk[i], y = sh.rtb[i];
        if (x > m || (x == m && y > mt)) {
          m = x;
          mt = y;
        }
      }
      if (!m) break;  // (uniform)
      if (tid == 0) choose(r, m, mt);
      psk = m;
      ptb = mt;
      __syncthreads();
    }
  }
  if (c > kWave) {
    __syncthreads();
    if (wave != 0) return;
  }
  // A lane a choice. keep_slots (n = W): the first child of each parent takes the parent's place, the others the
  // free places in their order, the empty ones behind them.
  const bool mine = lane < n;
  const int beam = mine ? lds_peek(&sh.ch_beam[lane]) : -1;
  int place = lane;
  if (a.keep) {
    u64 taken = 0;
    bool stays = false;
    for (int i = 0; i < n; ++i) {
      const int bi = __builtin_amdgcn_readlane(beam, i);
      if (bi >= 0 && !((taken >> bi) & 1)) {
        taken |= 1ull << bi;
        stays = stays || i == lane;
      }
    }
    const uint32_t skip = lanes_below(__ballot(mine && !stays));
    uint32_t free = 0;
    for (int i = 0; i < n; ++i) {
      if ((taken >> i) & 1) continue;
      if (free++ == skip) place = i;
    }
    if (stays) place = beam;
  }
  if (mine) {
    const int64_t at = static_cast<int64_t>(b) * n + place;
    a.out_scores[at] = lds_peek(&sh.ch_score[lane]);
    a.out_beams[at] = beam;
    a.out_tokens[at] = lds_peek(&sh.ch_token[lane]);
  }
}

}  // namespace vo
