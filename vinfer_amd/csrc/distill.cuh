// The distillation loss on a teacher's top entries, and its gradient in the student's logits x.
//
// With z = x / T, q = softmax(z) and the teacher's probabilities p_k of the entries' ids:
//   loss = sum_k p_k (log p_k - log q_k)            (+ rest (log rest - log q_rest) where the rest counts)
//   d loss / d z_j = mass q_j - p_j                 listed j, mass = sum_k p_k (+ rest)
//                  = mass q_j (- rest q_j / q_rest) the others
// rest = 1 - sum_k p_k and q_rest = 1 - sum_k q_k, each taken without that subtraction where it would cancel: the
// ids' logits are left out of the vocabulary's sum, S = sum over the others of exp(z - m) with m their largest,
// so that q_rest = S exp(m - lse) however small it is, and the others' gradient is exp(z_j - m) times one number
// A = mass exp(m - lse) - rest / S a row.
//
// k_distill_part: a segment's m and S, its logits held in registers, the listed ones struck out by a bitmap of
// the segment. k_distill_row: a wave a row, in fp64: the loss, m, A and the listed entries' gradients.
// k_distill_grad: a segment's gradient. Rows of weight 0 are not read: their loss and gradient are 0. So are their A and listed
// gradients, and what is 0 there stays 0 in a backward pass, whatever the row's logits and later weight hold (0 times an
// infinite or NaN exponential would be NaN, and the m of a row that was not read says nothing of it).
// Measured on an MI355X: 2048 rows of 151936 bf16 logits, 64 entries: the segments 105.4 us, 5.9 TB/s; the rows 8.6, a chain of
// dependent loads and fp64 functions.
#pragma once

#include "rows.cuh"

namespace vo {

constexpr int kDistillThreads = 256;
constexpr int kDistillWaves = kDistillThreads / kWave;

struct DistillArgs {
  const void* x;  // row t at t * stride
  int64_t stride;
  int T, V, K, S;
  const int32_t* ids;     // [T, K]; outside [0, V): no entry
  const float* teacher;   // [T, K]
  const float* weights;   // [T] or null (1)
  double inv;  // 1 / temperature
  float c;     // log2(e) / temperature
  int tail;
  float* maxs;    // [T, S]
  double* sums;   // [T, S]
  float* states;  // [T, 2 + K] m, A, the entries' gradients
  float* loss;    // [T]
  void* grad;     // row t at t * gstride
  int64_t gstride;
};

// The segment's listed ids as a bitmap, cleared and filled by the workgroup (a barrier at its end).
template <int ELEMS>
__device__ __forceinline__ void mark_listed(const int32_t* ids, int K, int V, int first, uint32_t* bits) {
  for (int i = threadIdx.x; i < ELEMS / 32; i += kDistillThreads) bits[i] = 0;
  __syncthreads();
  for (int k = threadIdx.x; k < K; k += kDistillThreads) {
    const int64_t i = static_cast<int64_t>(ld_global(ids + k)) - first;
    if (i >= 0 && i < ELEMS && i < V - first) atomicOr(&bits[i >> 5], 1u << (i & 31));
  }
  __syncthreads();
}

// Strikes the marked elements out of the registers (-inf).
template <class Tin, int NV>
__device__ __forceinline__ void strike_listed(const uint32_t* bits, uint4* d) {
  constexpr int E = Vec<Tin>::kElems;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const uint32_t at = (j * kDistillThreads + threadIdx.x) * E;
    const uint32_t m = (bits[at >> 5] >> (at & 31)) & ((1u << E) - 1);
    if (m) {
      uint32_t w[4] = {d[j].x, d[j].y, d[j].z, d[j].w};
#pragma unroll
      for (int e = 0; e < E; ++e)
        if ((m >> e) & 1) w[e * 4 / E] = strike_word<E>(w[e * 4 / E], e & 1);
      d[j] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

template <class Tin, int NV>
__global__ __launch_bounds__(kDistillThreads) void k_distill_part(DistillArgs a) {
  constexpr int E = Vec<Tin>::kElems;
  constexpr int kElems = NV * kDistillThreads * E;
  __shared__ uint32_t bits[kElems / 32];
  __shared__ float wmax[kDistillWaves];
  __shared__ double wsum[kDistillWaves];
  const int row = blockIdx.x / a.S, seg = blockIdx.x % a.S;
  if (a.weights && a.weights[row] == 0.0f) return;  // (uniform)
  const int first = seg * kElems;
  uint4 d[NV];
  load_segment<Tin, NV, kDistillThreads>(as_global(static_cast<const Tin*>(a.x)) + row * a.stride, a.V, first, d);
  mark_listed<kElems>(a.ids + static_cast<int64_t>(row) * a.K, a.K, a.V, first, bits);
  strike_listed<Tin, NV>(bits, d);
  float m = -__builtin_inff();
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    float x[E];
    Vec<Tin>::unpack(d[j], x);
#pragma unroll
    for (int e = 0; e < E; ++e) m = fmaxf(m, x[e]);
  }
  forget<NV>(d);
  m = wave_max_f(m);
  const float ref = m == -__builtin_inff() ? 0.0f : m;
  const float c = a.c;
  float s = 0.0f;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    float x[E];
    Vec<Tin>::unpack(d[j], x);
#pragma unroll
    for (int e = 0; e < E; ++e) s += __builtin_amdgcn_exp2f((x[e] - ref) * c);
  }
  const double t = wave_sum(static_cast<double>(s));
  if (lane_id() == 0) {
    wmax[threadIdx.x / kWave] = m;
    wsum[threadIdx.x / kWave] = t;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    float M = wmax[0];
    for (int i = 1; i < kDistillWaves; ++i) M = fmaxf(M, wmax[i]);
    double S = 0.0;
    // (a wave without a finite logit has the sum 0, or NaN for a NaN)
    for (int i = 0; i < kDistillWaves; ++i)
      S += wmax[i] == M ? wsum[i] : wsum[i] * exp((static_cast<double>(wmax[i]) - M) * a.inv);
    a.maxs[blockIdx.x] = M;
    a.sums[blockIdx.x] = S;
  }
}

__device__ __forceinline__ double wave_max_d(double x) {
  return dpp::reduce(x, [](double p, double q) { return p > q ? p : q; });
}

template <class Tin>
__device__ __forceinline__ double logit(const Tin* p) {
  if constexpr (sizeof(Tin) == 2) return bf16_to_f32(ld_global(p));
  else return ld_global(p);
}

// A wave's row from the segments' sums: m and A (in every lane), the loss (lane 0) and the listed entries' gradients
// (to `listed`, K of them). ONE: at most an entry a lane, loaded once and ahead of the rest.
struct RowNumbers {
  float m, A;
  double loss;
};
template <class Tin, bool ONE>
__device__ __forceinline__ RowNumbers row_numbers(const DistillArgs& a, int row, float* listed) {
  const int lane = lane_id();
  const double inv = a.inv;
  const double ninf = -static_cast<double>(__builtin_inff());
  const float* ms = as_global(a.maxs) + static_cast<int64_t>(row) * a.S;
  const double* ss = as_global(a.sums) + static_cast<int64_t>(row) * a.S;
  const int32_t* ids = as_global(a.ids) + static_cast<int64_t>(row) * a.K;
  const float* teacher = as_global(a.teacher) + static_cast<int64_t>(row) * a.K;
  const Tin* x = as_global(static_cast<const Tin*>(a.x)) + row * a.stride;
  // f(k, is there an entry, the teacher's value, the logit)
  int id = -1;
  double tv = 0.0, xv = 0.0;
  auto load = [&](int k) {
    id = k < a.K ? ld_global(ids + k) : -1;
    tv = k < a.K ? ld_global(teacher + k) : 0.0f;
    const bool has = static_cast<uint32_t>(id) < static_cast<uint32_t>(a.V);
    xv = has ? logit(x + id) : 0.0;
    return has;
  };
  const float m1 = lane < a.S ? ms[lane] : -__builtin_inff();  // (at most 64 segments)
  const double s1 = lane < a.S ? ss[lane] : 0.0;
  bool has1 = false;
  if constexpr (ONE) has1 = load(lane);
  auto each = [&](auto f) {
    if constexpr (ONE) {
      f(lane, has1);
    } else {
      for (int k = lane; k < a.K; k += kWave) f(k, load(k));
    }
  };
  const float mf = wave_max_f(m1);
  const double m = mf;
  const double S = wave_sum(m1 == mf ? s1 : s1 * exp((m1 - m) * inv));
  // the teacher's normaliser and the listed logits' largest
  double tm = ninf, lm = ninf;
  each([&](int, bool has) {
    if (!has) return;
    tm = tv > tm ? tv : tm;
    lm = xv > lm ? xv : lm;
  });
  tm = wave_max_d(tm);
  lm = wave_max_d(lm);
  const double xm = lm > m ? lm : m;
  double ts = 0.0, xs = 0.0;
  each([&](int, bool has) {
    if (!has) return;
    ts += exp(a.tail ? tv : (tv - tm) * inv);
    xs += exp((xv - xm) * inv);
  });
  ts = wave_sum(ts);
  xs = wave_sum(xs);
  const bool none = tm == ninf;  // (no entry, or all of probability 0)
  // Nothing to learn from: no entry, or (tail) none that either side gives a probability. Its numbers are 0 whatever its logits hold.
  const bool empty = none && (!a.tail || (lm == ninf && xs == 0.0));
  // (differences of logits before anything else: beside logits of 1e38 an lse would lose log S)
  const double lts = a.tail ? 0.0 : log(ts);
  const double em = m == ninf ? 0.0 : exp((m - xm) * inv);
  const double total = (m == ninf ? S : S * em) + xs;
  const double ltotal = log(total);
  const double rest = a.tail ? fmax(0.0, 1.0 - ts) : 0.0;
  const double mass = a.tail ? ts + rest : (none ? 0.0 : 1.0);
  double loss = 0.0;
  each([&](int k, bool has) {
    float g = 0.0f;
    if (has && !empty) {
      const double lp = a.tail ? tv : (tv - tm) * inv - lts;
      const double lq = (xv - xm) * inv - ltotal;
      const double p = none ? 0.0 : exp(lp);
      if (p != 0.0) loss += p * (lp - lq);
      g = static_cast<float>(exp(lq) * mass - p);
    }
    if (k < a.K) listed[k] = g;
  });
  loss = wave_sum(loss);
  if (rest > 0.0 && !empty) loss += rest * (log(rest) - ((m == ninf ? ninf : (m - xm) * inv) + log(S) - ltotal));
  double A = 0.0;
  if ((m != ninf || S != 0.0) && !empty) A = mass * em / total - (rest > 0.0 ? rest / S : 0.0);
  return RowNumbers{mf, static_cast<float>(A), loss};
}

template <class Tin, bool ONE>
__global__ __launch_bounds__(kDistillThreads) void k_distill_row(DistillArgs a) {
  const int row = blockIdx.x * kDistillWaves + threadIdx.x / kWave;
  if (row >= a.T) return;
  const int lane = lane_id();
  const float weight = a.weights ? as_global(a.weights)[row] : 1.0f;
  float* st = as_global(a.states) + static_cast<int64_t>(row) * (2 + a.K);
  if (weight == 0.0f) {
    for (int k = lane; k < a.K; k += kWave) st[2 + k] = 0.0f;
    if (lane == 0) {
      a.loss[row] = 0.0f;
      st[0] = 0.0f;
      st[1] = 0.0f;
    }
    return;
  }
  const RowNumbers n = row_numbers<Tin, ONE>(a, row, st + 2);
  if (lane == 0) {
    a.loss[row] = static_cast<float>(weight * n.loss);
    st[0] = n.m;
    st[1] = n.A;
  }
}

typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));
// Two fp32 values rounded to bf16 (to nearest, ties to even: one v_cvt_pk_bf16_f32).
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{lo, hi}, bf16x2_t));
}

typedef u32x4_t u32x4_row_t __attribute__((aligned(2)));
__device__ __forceinline__ void st_row16(void* p, uint4 v) {
  *(__attribute__((address_space(1))) u32x4_row_t*)p = u32x4_t{v.x, v.y, v.z, v.w};
}

// (past the cache: gradients of a batch larger than it)
__device__ __forceinline__ void st_row16_nt(void* p, uint4 v) {
  __builtin_nontemporal_store(u32x4_t{v.x, v.y, v.z, v.w}, (__attribute__((address_space(1))) u32x4_row_t*)p);
}

// A vector's gradients, factor exp2((x - ref) c), packed.
template <class Tin>
__device__ __forceinline__ uint4 grad_vector(const uint4& d, float ref, float c, float factor) {
  constexpr int E = Vec<Tin>::kElems;
  float x[E];
  Vec<Tin>::unpack_again(d, x);
#pragma unroll
  for (int e = 0; e < E; ++e) x[e] = factor * __builtin_amdgcn_exp2f((x[e] - ref) * c);
  if constexpr (E == 8)
    return make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
  else
    return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
}

template <class Tin>
__device__ __forceinline__ void store_elem(Tin* p, float v) {
  if constexpr (sizeof(Tin) == 2) *(__attribute__((address_space(1))) uint16_t*)p = static_cast<uint16_t>(pack_bf16(v, v));
  else *(__attribute__((address_space(1))) float*)p = v;
}

// Stores vector v at element i of a row of V.
template <class Tin>
__device__ __forceinline__ void store_vector(Tin* row, int V, int i, const uint4& v) {
  constexpr int E = Vec<Tin>::kElems;
  if (i + E <= V) {
    st_row16(row + i, v);
    return;
  }
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int e = 0; e < E; ++e) {
    if (i + e >= V) continue;
    if constexpr (E == 8)
      *(__attribute__((address_space(1))) uint16_t*)(row + i + e) = static_cast<uint16_t>(w[e >> 1] >> (16 * (e & 1)));
    else
      *(__attribute__((address_space(1))) uint32_t*)(row + i + e) = w[e];
  }
}

// ROW: the row's numbers are worked out here, by each segment's first wave while the logits are on their way (at most
// an entry a lane), and the first segment writes the loss: a launch less, for few rows.
template <class Tin, int NV, bool ROW>
__global__ __launch_bounds__(kDistillThreads) void k_distill_grad(DistillArgs a) {
  constexpr int E = Vec<Tin>::kElems;
  constexpr int kElems = NV * kDistillThreads * E;
  __shared__ float listed[kWave], numbers[2];
  const int row = blockIdx.x / a.S, seg = blockIdx.x % a.S;
  const int first = seg * kElems;
  const float weight = a.weights ? a.weights[row] : 1.0f;
  Tin* g = as_global(static_cast<Tin*>(a.grad)) + row * a.gstride;
  const int at = first + static_cast<int>(threadIdx.x) * E;
  if (weight == 0.0f) {  // (uniform)
#pragma unroll
    for (int j = 0; j < NV; ++j) store_vector<Tin>(g, a.V, at + j * kDistillThreads * E, make_uint4(0, 0, 0, 0));
    if (ROW && seg == 0 && threadIdx.x == 0) a.loss[row] = 0.0f;
    return;
  }
  uint4 d[NV];
  load_segment<Tin, NV, kDistillThreads>(as_global(static_cast<const Tin*>(a.x)) + row * a.stride, a.V, first, d);
  const float* st = as_global(a.states) + static_cast<int64_t>(row) * (2 + a.K);
  float m, A;
  if constexpr (ROW) {
    if (threadIdx.x < kWave) {
      const RowNumbers n = row_numbers<Tin, true>(a, row, listed);
      if (threadIdx.x == 0) {
        numbers[0] = n.m;
        numbers[1] = n.A;
        if (seg == 0) a.loss[row] = static_cast<float>(weight * n.loss);
      }
    }
    lds_barrier();
    m = numbers[0];
    A = numbers[1];
  } else {
    m = st[0];
    A = st[1];
  }
  const float ref = m == -__builtin_inff() ? 0.0f : m;
  const float scale = static_cast<float>(weight * a.inv);
  const float factor = scale * A;
  const float c = a.c;
  const bool zero = A == 0.0f;  // (uniform)
#pragma unroll
  for (int j = 0; j < NV; ++j)
    store_vector<Tin>(g, a.V, at + j * kDistillThreads * E,
                      zero ? make_uint4(0, 0, 0, 0) : grad_vector<Tin>(d[j], ref, c, factor));
  __syncthreads();  // (the listed gradients go over what the vectors stored there)
  const int32_t* ids = a.ids + static_cast<int64_t>(row) * a.K;
  for (int k = threadIdx.x; k < a.K; k += kDistillThreads) {
    const int id = ld_global(ids + k);
    if (id >= first && id < a.V && id - first < kElems) {
      const float l = ROW ? listed[k] : st[2 + k];
      store_elem<Tin>(g + id, l == 0.0f ? 0.0f : scale * l);
    }
  }
}

// ---- loss and gradient of many rows in one pass -----------------------------------------------------------
// A workgroup holds a whole row: NS vectors a thread in registers, and a row's last V % E elements one a thread. Rows
// follow one another (grid-strided, those of weight 0 passed over). As a row's gradients are stored, the next row's
// logits are loaded into the registers that become free, and kBehind vectors later they are added to the next row's
// sum: a row is read once, and a CU reads, writes and computes at once. Loads and stores there are unconditional (the
// lanes past the row's end repeat its last vector), so that the waits count them. One barrier a row: the waves' sums,
// and the next row's listed ids' bits (three bitmaps take turns: one is cleared a barrier before it is used again).
// After it the last row's listed gradients go over what its vectors stored there.
//
// A wave's sum is against the largest of its first vectors, not of its row: nothing has to be known of a vector before
// it is added. Where that was far off (a sum outside 2^-40 .. 2^60) the wave adds up again against its largest.
// exp(x / T - ref / T) is one fma and v_exp_f32: 2^(x c - fl(ref c)), c = fl(log2(e) / T) (host); the rounding of ref c is
// put right in the sum, in fp64. A bf16 gradient's factor goes into the exponent too (off by 2^-16 at most). Where
// ref c is past 2^8 (logits in the hundreds, or a cold temperature) differences are taken first, in slower loops.
//
// 4096 rows of 151936 bf16 logits, an eighth of weight 0: 496 us, 4.7 TB/s of logits and gradients (in segments, which read
// the logits twice, 660); 1000 fp32 rows of 50257: 86 us. Vector issue takes 20 of a row's 31 us on its CU. Of the choices, in an
// earlier form: the sum 8 vectors behind the loads 551 us, 4 570, 2 587; gradients stored past the cache 70 us for 1000 fp32
// rows whose logits are partly in it, through it 93.
constexpr int kBehind = 8;
constexpr float kMostExponent = 256.0f;

template <int WAVES>
struct HeldShared {
  float m[2][WAVES];  // a wave's reference, and its sum
  double s[2][WAVES];
  double tm[2][WAVES], ts[2][WAVES];  // its entries': the teacher's largest and sum,
  double xm[2][WAVES], xs[2][WAVES];  // the listed logits' largest and sum
  double loss[2][WAVES];
};

template <class Tin, int THREADS, int NS, int ROWS>  // ROWS workgroups a CU
__global__ __launch_bounds__(THREADS, ROWS * THREADS / 256) void k_distill_held(DistillArgs a) {
  constexpr int E = Vec<Tin>::kElems;
  constexpr int kWavesHere = THREADS / kWave;
  constexpr int kBits = (THREADS * NS * E + E + 31) / 32;
  constexpr double kLn2 = 0.6931471805599453;
  __shared__ uint32_t bits[3][kBits];
  __shared__ HeldShared<kWavesHere> sh;
  const int tid = threadIdx.x, lane = lane_id(), w = uniform_i(tid / kWave);
  const int V = a.V, K = a.K, nvec = V / E;
  const int left = nvec * E + tid;  // this thread's element of the row's end, if below V
  const double inv = a.inv;
  const double ninf = -static_cast<double>(__builtin_inff());
  const float c = a.c;

  auto row_of = [&](int r) { return as_global(static_cast<const Tin*>(a.x)) + r * a.stride; };
  auto grad_of = [&](int r) { return as_global(static_cast<Tin*>(a.grad)) + r * a.gstride; };
  auto weight_of = [&](int r) { return a.weights ? as_global(a.weights)[r] : 1.0f; };
  auto element = [&](const Tin* p) { return static_cast<float>(logit(p)); };
  auto listed = [&](int id) { return static_cast<uint32_t>(id) < static_cast<uint32_t>(V); };
  auto id_of = [&](int r) { return ld_global(a.ids + static_cast<int64_t>(r) * K + tid); };
  auto teacher_of = [&](int r) { return ld_global(a.teacher + static_cast<int64_t>(r) * K + tid); };
  // Vector j of this thread: bytes from a uniform base, and the offset of the lane (made anew each time, or the loops
  // would keep them all in registers).
  const uint32_t most = (nvec - 1) * 16, t16 = tid * 16;
  auto anew = [&]() {
    uint32_t t = t16;
    asm volatile("" : "+v"(t));
    return t;
  };
  auto base = [&](int j) { return min(static_cast<uint32_t>(j * THREADS * 16), most); };
  auto offset = [&](int j) { return min(anew(), most - base(j)); };
  auto own = [&](int j) { return anew() + j * THREADS * 16 <= most; };  // (not a repetition)
  auto vector_at = [&](const Tin* p, int j) { return ld_row16(reinterpret_cast<const char*>(p) + base(j) + offset(j)); };

  // The first row from r on (in steps of the grid) whose weight is not 0, T for none; the ones passed over get their
  // zeros.
  auto live_from = [&](int r) {
    for (; r < a.T && weight_of(r) == 0.0f; r += gridDim.x) {
      char* g = reinterpret_cast<char*>(grad_of(r));
#pragma unroll 1
      for (uint32_t o = t16; o <= most; o += THREADS * 16) st_row16_nt(g + o, make_uint4(0, 0, 0, 0));
      if (left < V) store_elem<Tin>(grad_of(r) + left, 0.0f);
      if (tid == 0) a.loss[r] = 0.0f;
    }
    return min(r, a.T);
  };

  uint4 d[NS];
  float end = -__builtin_inff();  // the row's end's element
  float ref = 0.0f, refc = 0.0f, s = 0.0f;  // a wave's reference, a thread's sum
  // Strikes the listed elements out of the row's vector j of this thread.
  auto strike_marked = [&](uint4& v, int j, const uint32_t* marked) {
    const uint32_t at = (base(j) + offset(j)) / 16;
    const uint8_t* bytes = reinterpret_cast<const uint8_t*>(marked);
    const uint32_t marks = E == 8 ? bytes[at] : (bytes[at >> 1] >> ((at & 1) * 4)) & 15u;
    if (marks) {
      uint32_t q[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int e = 0; e < E; ++e)
        if ((marks >> e) & 1) q[e * 4 / E] = strike_word<E>(q[e * 4 / E], e & 1);
      v = make_uint4(q[0], q[1], q[2], q[3]);
    }
  };
  // Vector j without its listed elements joins the sum.
  auto add = [&](int j, const uint32_t* marked) {
    strike_marked(d[j], j, marked);
    if (j == 0) {
      const float m = wave_max_f(Vec<Tin>::largest(d[j]));
      ref = fabsf(m) * c < kMostExponent ? m : 0.0f;  // (0: far off, mostly)
      refc = uniform_f(ref * c);
      s = 0.0f;
    }
    float x[E], t = 0.0f;
    Vec<Tin>::unpack(d[j], x);
#pragma unroll
    for (int e = 0; e < E; ++e) t += __builtin_amdgcn_exp2f(__builtin_fmaf(x[e], c, -refc));
    s += own(j) ? t : 0.0f;
    asm volatile("" : "+v"(s));  // (here, not where the sum is used)
  };
  auto add_end = [&](const uint32_t* marked) {
    if (left < V && (marked[left >> 5] >> (left & 31)) & 1) end = -__builtin_inff();
    s += __builtin_amdgcn_exp2f(__builtin_fmaf(end, c, -refc));
  };

  int r = live_from(blockIdx.x);
  if (r >= a.T) return;  // (uniform)
  for (int i = tid; i < kBits; i += THREADS) bits[0][i] = bits[1][i] = bits[2][i] = 0;
  __syncthreads();
  int next = live_from(r + gridDim.x);
  int now = 0, next_bits = 1, free_bits = 2;
  int id = -1, id1 = -1;
  float tv = 0.0f, xv = 0.0f, tv1 = 0.0f;
  {
    const Tin* p = row_of(r);
    if (tid < K) {
      id = id_of(r);
      tv = teacher_of(r);
    }
#pragma unroll
    for (int j = 0; j < NS; ++j) d[j] = vector_at(p, j);
    if (left < V) end = element(p + left);
    if (listed(id)) {
      xv = element(p + id);
      atomicOr(&bits[0][id >> 5], 1u << (id & 31));
    }
  }
  if (next < a.T && tid < K) {
    id1 = id_of(next);
    tv1 = teacher_of(next);
  }
  lds_barrier();
#pragma unroll
  for (int j = 0; j < NS; ++j) {
    add(j, bits[0]);
    __builtin_amdgcn_sched_barrier(0);
  }
  add_end(bits[0]);
  // the row before: what is stored once its gradients are
  int last = -1, last_id = -1, par = 0;
  float last_g = 0.0f;
  double last_rest = 0.0;
  auto finish_last = [&](int buffer) {
    if (last_id >= 0) store_elem<Tin>(grad_of(last) + last_id, last_g);
    if (tid == 0) {
      double t = last_rest;
      for (int i = 0; i < kWavesHere; ++i) t += sh.loss[buffer][i];
      a.loss[last] = static_cast<float>(weight_of(last) * t);
    }
  };

  for (;; par ^= 1) {
    const bool has = listed(id);
    const bool more = next < a.T;  // (uniform)
    // the next row's listed ids, and their logits
    float xv1 = 0.0f;
    if (more && listed(id1)) {
      atomicOr(&bits[next_bits][id1 >> 5], 1u << (id1 & 31));
      xv1 = element(row_of(next) + id1);
    }
    double sd = wave_sum(static_cast<double>(s));
    if (sd > 0x1p-40 && sd < 0x1p60) {  // (uniform over the wave)
      sd *= 1.0 + kLn2 * (refc - static_cast<double>(ref) * static_cast<double>(c));
    } else {
      // (read again: rolled loops, no registers)
      const Tin* p = row_of(r);
      float m = end;
#pragma unroll 1
      for (int j = 0; j < NS; ++j) {
        uint4 v = vector_at(p, j);
        strike_marked(v, j, bits[now]);
        m = max_nan(m, Vec<Tin>::largest(v));
      }
      ref = wave_max_f(m);
      const float z = ref == -__builtin_inff() ? 0.0f : ref;
      s = __builtin_amdgcn_exp2f((end - z) * c);
#pragma unroll 1
      for (int j = 0; j < NS; ++j) {
        uint4 v = vector_at(p, j);
        strike_marked(v, j, bits[now]);
        float x[E], t = 0.0f;
        Vec<Tin>::unpack(v, x);
#pragma unroll
        for (int e = 0; e < E; ++e) t += __builtin_amdgcn_exp2f((x[e] - z) * c);
        s += own(j) ? t : 0.0f;
      }
      sd = wave_sum(static_cast<double>(s));
    }
    if (w * kWave < K) {  // (uniform)
      const double tm = wave_max_d(has ? static_cast<double>(tv) : ninf);
      const double xm = wave_max_d(has ? static_cast<double>(xv) : ninf);
      __builtin_amdgcn_sched_barrier(0);
      // (-inf adds nothing, also where a wave's entries have nothing else)
      const double ts = wave_sum(!has || tv == ninf ? 0.0 : exp(a.tail ? static_cast<double>(tv) : (tv - tm) * inv));
      __builtin_amdgcn_sched_barrier(0);
      const double xs = wave_sum(!has || xv == ninf ? 0.0 : exp((xv - xm) * inv));
      __builtin_amdgcn_sched_barrier(0);
      if (lane == 0) {
        sh.tm[par][w] = tm;
        sh.ts[par][w] = ts;
        sh.xm[par][w] = xm;
        sh.xs[par][w] = xs;
      }
    }
    if (lane == 0) {
      sh.m[par][w] = ref;
      sh.s[par][w] = sd;
    }
    const int after = more ? live_from(next + gridDim.x) : a.T;
    __syncthreads();
    if (last >= 0) finish_last(par ^ 1);
    if (has) bits[now][id >> 5] = 0;
    // the row's numbers, in every wave: a lane a wave's part
    const bool part = lane < kWavesHere;
    const float mw = part ? sh.m[par][lane] : -__builtin_inff();
    const float mf = wave_max_f(mw);
    const double m = mf;
    double S = part ? sh.s[par][lane] : 0.0;
    __builtin_amdgcn_sched_barrier(0);
    S = wave_sum(mw == mf ? S : S * exp((mw - m) * inv));
    __builtin_amdgcn_sched_barrier(0);
    double tm = sh.tm[par][0], ts = sh.ts[par][0], xm = sh.xm[par][0], xs = sh.xs[par][0];
    if (K > kWave) {  // (uniform)
      const bool entries = lane * kWave < K;  // (waves that have some)
      const double tw = entries ? sh.tm[par][lane] : ninf, xw = entries ? sh.xm[par][lane] : ninf;
      tm = wave_max_d(tw);
      xm = wave_max_d(xw);
      ts = entries ? sh.ts[par][lane] : 0.0;
      xs = entries ? sh.xs[par][lane] : 0.0;
      __builtin_amdgcn_sched_barrier(0);
      ts = wave_sum(a.tail || tw == tm ? ts : ts * exp((tw - tm) * inv));
      __builtin_amdgcn_sched_barrier(0);
      xs = wave_sum(xw == xm ? xs : xs * exp((xw - xm) * inv));
    }
    __builtin_amdgcn_sched_barrier(0);
    const bool empty = tm == ninf && (!a.tail || (xm == ninf && xs == 0.0));  // (as in row_numbers)
    // (against the larger of the two largest)
    double em = 1.0;
    if (xm > m) {
      em = m == ninf ? 0.0 : exp((m - xm) * inv);
    } else {
      xs = xm == ninf ? xs : xs * exp((xm - m) * inv);
      xm = m;
    }
    const double total = (m == ninf ? S : S * em) + xs;
    __builtin_amdgcn_sched_barrier(0);
    const bool none = tm == ninf;
    const double rest = a.tail ? fmax(0.0, 1.0 - ts) : 0.0;
    const double mass = a.tail ? ts + rest : (none ? 0.0 : 1.0);
    double A = 0.0;
    if ((m != ninf || S != 0.0) && !empty) A = mass * em / total - (rest > 0.0 ? rest / S : 0.0);
    __builtin_amdgcn_sched_barrier(0);
    const float scale = static_cast<float>(weight_of(r) * inv);
    const bool huge = !(fabsf(mf) * c < kMostExponent) && mf != -__builtin_inff();  // (uniform)
    const bool clear = empty && S - S != 0.0;  // (an infinite or NaN logit, whose 0 it is to be as well)
    const float zero = uniform_f(huge || mf == -__builtin_inff() ? 0.0f : mf);
    float factor = uniform_f(scale * static_cast<float>(A));
    // the gradients out, the next row in, and its sum
    {
      Tin* g = grad_of(r);
      char* gb = reinterpret_cast<char*>(g);
      float zeroc = uniform_f(zero * c);
      uint32_t sign = 0;
      if constexpr (E == 8) {
        sign = __float_as_uint(factor) & 0x80000000u;
        sign = uniform_u(sign | (sign >> 16));
        zeroc = uniform_f(zeroc - __builtin_amdgcn_logf(fabsf(factor)));
      } else {
        factor = uniform_f(factor * static_cast<float>(1.0 + kLn2 * (zeroc - static_cast<double>(zero) * static_cast<double>(c))));
      }
      auto gradient = [&](const uint4& v) {
        float x[E];
        Vec<Tin>::unpack_again(v, x);
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[e], c, -zeroc));
        if constexpr (E == 8) {
          return make_uint4(pack_bf16(x[0], x[1]) ^ sign, pack_bf16(x[2], x[3]) ^ sign, pack_bf16(x[4], x[5]) ^ sign,
                            pack_bf16(x[6], x[7]) ^ sign);
        } else {
          return make_uint4(__float_as_uint(factor * x[0]), __float_as_uint(factor * x[1]),
                            __float_as_uint(factor * x[2]), __float_as_uint(factor * x[3]));
        }
      };
      if (left < V) {
        const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(end, c, -zeroc));
        store_elem<Tin>(g + left, E == 8 ? __uint_as_float(__float_as_uint(e) ^ (sign & 0x80000000u)) : factor * e);
      }
      if (more) {
        const Tin* p = row_of(next);
        if (left < V) end = element(p + left);
        const uint32_t* marked = bits[next_bits];
#pragma unroll
        for (int j = 0; j < NS + kBehind; ++j) {
          if (j < NS) {
            const uint32_t at = offset(j);
            st_row16_nt(gb + base(j) + at, gradient(d[j]));
            d[j] = ld_row16(reinterpret_cast<const char*>(p) + base(j) + at);
          }
          __builtin_amdgcn_sched_barrier(0);
          if (j >= kBehind) add(j - kBehind, marked);
          __builtin_amdgcn_sched_barrier(0);
        }
        add_end(marked);
      } else {
#pragma unroll
        for (int j = 0; j < NS; ++j) {
          st_row16_nt(gb + base(j) + offset(j), gradient(d[j]));
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      if (huge || clear) {  // (the gradients again, from differences)
        const float f = scale * static_cast<float>(A);
#pragma unroll 1
        for (int j = 0; j < NS; ++j)
          st_row16_nt(gb + base(j) + offset(j),
                      clear ? make_uint4(0, 0, 0, 0) : grad_vector<Tin>(vector_at(row_of(r), j), mf, c, f));
        if (left < V)
          store_elem<Tin>(g + left, clear ? 0.0f : f * __builtin_amdgcn_exp2f((element(row_of(r) + left) - mf) * c));
      }
    }
    // the listed gradients and the loss, stored after the next barrier
    last = r;
    last_id = has ? id : -1;
    if (w * kWave < K) {  // (uniform)
      const double lts = a.tail ? 0.0 : log(ts);
      const double ltotal = log(total);
      double loss = 0.0;
      if (has) {
        const double lp = a.tail ? static_cast<double>(tv) : (tv - tm) * inv - lts;
        const double lq = (xv - xm) * inv - ltotal;
        const double q = none ? 0.0 : exp(lp);
        if (q != 0.0) loss = q * (lp - lq);
        last_g = empty ? 0.0f : scale * static_cast<float>(exp(lq) * mass - q);
      }
      loss = wave_sum(loss);
      if (lane == 0) sh.loss[par][w] = loss;
      last_rest = rest > 0.0 && !empty ? rest * (log(rest) - ((m == ninf ? ninf : (m - xm) * inv) + log(S) - ltotal)) : 0.0;
    } else if (lane == 0) {
      sh.loss[par][w] = 0.0;
    }
    if (!more) break;
    id = id1;
    tv = tv1;
    xv = xv1;
    r = next;
    next = after;
    id1 = -1;
    if (next < a.T && tid < K) {
      id1 = id_of(next);
      tv1 = teacher_of(next);
    }
    const int t = now;
    now = next_bits;
    next_bits = free_bits;
    free_bits = t;
  }
  __syncthreads();
  finish_last(par);
}

}  // namespace vo
