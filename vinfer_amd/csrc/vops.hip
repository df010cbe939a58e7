// C ABI of libvops.so (declared in include/vops.h).
#include <hip/hip_runtime.h>

#include <atomic>
#include <cstdarg>
#include <cstdio>
#include <cstring>

#include "../../include/vops.h"
#include "beam.cuh"
#include "distill.cuh"
#include "reorder.cuh"

namespace {

thread_local char g_err[512];

int fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
int fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof g_err, fmt, ap);
  va_end(ap);
  return code;
}

int hip_fail(hipError_t e, const char* what) { return fail(VOPS_E_HIP, "%s: %s", what, hipGetErrorString(e)); }

int launched(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? VOPS_OK : hip_fail(e, what);
}

constexpr int kMaxDevices = 64;
std::atomic<int> g_dev_ok[kMaxDevices];  // 0 unknown, 1 gfx950

int check_device(int dev, char* why, size_t n) {
  if (dev >= 0 && dev < kMaxDevices && g_dev_ok[dev].load() == 1) return VOPS_OK;
  int count = 0;
  hipError_t e = hipGetDeviceCount(&count);
  if (e != hipSuccess || count == 0) {
    if (why && n) snprintf(why, n, "no HIP device available");
    return VOPS_E_DEVICE;
  }
  if (dev < 0 || dev >= count) {
    if (why && n) snprintf(why, n, "device %d out of range (%d devices)", dev, count);
    return VOPS_E_DEVICE;
  }
  hipDeviceProp_t prop;
  e = hipGetDeviceProperties(&prop, dev);
  if (e != hipSuccess) {
    if (why && n) snprintf(why, n, "hipGetDeviceProperties: %s", hipGetErrorString(e));
    return VOPS_E_HIP;
  }
  if (std::strncmp(prop.gcnArchName, "gfx950", 6) != 0) {
    if (why && n) snprintf(why, n, "needs a gfx950 (MI355X) GPU, device %d is %s", dev, prop.gcnArchName);
    return VOPS_E_DEVICE;
  }
  if (dev < kMaxDevices) g_dev_ok[dev].store(1);
  return VOPS_OK;
}

int check_current_device() {
  int dev = 0;
  const hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return hip_fail(e, "hipGetDevice");
  char why[256];
  const int rc = check_device(dev, why, sizeof why);
  return rc ? fail(rc, "%s", why) : VOPS_OK;
}

size_t align_up(size_t x) { return (x + 255) & ~static_cast<size_t>(255); }

int check_workspace(const void* p, size_t given, size_t need) {
  if (given < need || (need && !p)) return fail(VOPS_E_WORKSPACE, "workspace of %zu bytes given, %zu needed", given, need);
  if (reinterpret_cast<uintptr_t>(p) & 255u) return fail(VOPS_E_WORKSPACE, "workspace must be 256-byte aligned");
  return VOPS_OK;
}

static_assert(VOPS_MAX_BEAMS <= vo::kMaxBeams && VOPS_MAX_CONTINUATIONS <= vo::kMaxPick && VOPS_MAX_VOCAB <= 1 << 20 &&
                  VOPS_MAX_REORDER_BEAMS <= vo::kMaxReorderBeams,
              "what is checked here is what the kernels hold (an id takes 20 bits of a selection's tie word)");

constexpr int kVecElems[2] = {8, 4};  // elements of a 16-byte vector, by dtype

// The 16-byte vectors a thread of 256 holds (a power of two up to 8): as many as leave the launch `fill`
// workgroups, and at least what keeps a row's segments to 64 (a lane each where they are joined). Where the chip is
// full, longer segments are faster: 2048 rows' losses (151936 ids) 107 us with 8 vectors, 140 with 4, 181 with 2.
int segment_vectors(int dtype, int64_t rows, int64_t V, int64_t fill) {
  const int64_t unit = 256 * kVecElems[dtype];
  int nv = 8;
  while (nv > 1 && rows * ((V + nv * unit - 1) / (nv * unit)) < fill && (V + nv / 2 * unit - 1) / (nv / 2 * unit) <= 64)
    nv /= 2;
  return nv;
}
int segments(int dtype, int nv, int64_t V) {
  const int64_t e = static_cast<int64_t>(nv) * 256 * kVecElems[dtype];
  return static_cast<int>((V + e - 1) / e);
}

constexpr int64_t kFillWorkgroups = 1024;
// Above this many continuations a segment's bound is taken over its whole workgroup, at and below it over each wave.
// (64 x 4 x 151936 bf16 logits in all, per wave and per workgroup: n = 1 22.9 and 24.0 us, 4 23.5 and 24.0, 8 25.4 and
// 25.0; bounds of a wave alone 39 us at n = 32 and 71 at 64, of the workgroup 30 and 37)
constexpr int kManyContinuations = 8;

struct BeamLayout {
  int nv, S;
  size_t keys, sums, maxs, total;
};
BeamLayout beam_layout(int dtype, int64_t B, int64_t W, int64_t V, int64_t n) {
  BeamLayout L;
  L.nv = segment_vectors(dtype, B * W, V, kFillWorkgroups);
  L.S = segments(dtype, L.nv, V);
  const size_t parts = static_cast<size_t>(B * W) * L.S;
  L.keys = 0;
  L.sums = align_up(parts * n * 8);
  L.maxs = align_up(L.sums + parts * 8);
  L.total = align_up(L.maxs + parts * 4);
  return L;
}

struct DistillLayout {
  int nv, S;
  size_t sums, maxs, states, total;
};
DistillLayout distill_layout(int dtype, int64_t T, int64_t V, int64_t K) {
  DistillLayout L;
  L.nv = segment_vectors(dtype, T, V, kFillWorkgroups);
  L.S = segments(dtype, L.nv, V);
  const size_t parts = static_cast<size_t>(T) * L.S;
  L.sums = 0;
  L.maxs = align_up(parts * 8);
  L.states = align_up(L.maxs + parts * 4);
  L.total = align_up(L.states + static_cast<size_t>(T) * (2 + K) * 4);
  return L;
}

bool beam_sizes_ok(int32_t dtype, int32_t B, int32_t W, int32_t V, int32_t n) {
  return (dtype == VOPS_BF16 || dtype == VOPS_F32) && B >= 0 && B <= 65535 && W >= 1 && W <= VOPS_MAX_BEAMS && V >= 1 &&
         V <= VOPS_MAX_VOCAB && n >= 1 && n <= VOPS_MAX_CONTINUATIONS;
}

bool distill_sizes_ok(int32_t dtype, int32_t T, int32_t V, int32_t K) {
  return (dtype == VOPS_BF16 || dtype == VOPS_F32) && T >= 0 && V >= 1 && V <= VOPS_MAX_VOCAB && K >= 1 &&
         K <= VOPS_MAX_ENTRIES;
}

// f(std::integral_constant-like tag) for nv in {1, 2, 4, 8}
template <int N>
struct Nv {
  static constexpr int value = N;
};
// Loss and gradient with whole rows held: from this many rows, or where a row is short enough for one workgroup to be
// no slower than the segments' launches. Measured, held against segments (us): bf16 rows of 151936, 32 of them
// 22.7 / 17.4, 64 23.0 / 23.2, 128 28.7 / 30.2, 512 72.8 / 98.2; of 32000, 32 10.1 / 16.2, 1024 34.8 / 46.0; fp32 rows
// of 50257, 32 12.7 / 14.5, 256 25.7 / 30.9.
constexpr int kHeldRows = 64;
constexpr int kHeldVectors = 8192;  // (16-byte vectors of a row)
constexpr int kHeldVocab = 4096;
constexpr int kHeldEntries = 512;  // (a thread each)
constexpr int kFewRows = 192;      // (their numbers are worked out by each segment of the gradient: 16 rows of 151936 15.4 -> 11.2 us)

template <class F>
void with_nv(int nv, F f) {
  if (nv == 8) f(Nv<8>{});
  else if (nv == 4) f(Nv<4>{});
  else if (nv == 2) f(Nv<2>{});
  else f(Nv<1>{});
}

int distill_common(const vops_distill_args* a) {
  if (!a) return fail(VOPS_E_ARG, "args is NULL");
  if (a->dtype != VOPS_BF16 && a->dtype != VOPS_F32)
    return fail(VOPS_E_DTYPE, "unsupported dtype %d (VOPS_BF16=0, VOPS_F32=1)", a->dtype);
  if (a->flags & ~VOPS_DISTILL_TAIL) return fail(VOPS_E_ARG, "flags must be 0 or VOPS_DISTILL_TAIL, got %u", a->flags);
  if (!distill_sizes_ok(a->dtype, a->rows, a->vocab, a->entries))
    return fail(VOPS_E_ARG, "rows must be >= 0, vocab in [1, %d], entries in [1, %d], got %d, %d, %d", VOPS_MAX_VOCAB,
                VOPS_MAX_ENTRIES, a->rows, a->vocab, a->entries);
  if (a->row_stride < 0 || (a->out_grad && a->grad_stride < a->vocab))
    return fail(VOPS_E_ARG, "row_stride must be >= 0 and grad_stride >= vocab");
  if (!(a->temperature >= VOPS_MIN_TEMPERATURE && a->temperature <= VOPS_MAX_TEMPERATURE))
    return fail(VOPS_E_ARG, "temperature must be in [%g, %g], got %g", VOPS_MIN_TEMPERATURE,
                VOPS_MAX_TEMPERATURE, a->temperature);
  if (a->rows > 0 && (!a->student || !a->ids)) return fail(VOPS_E_ARG, "student and ids must be set");
  const uintptr_t mask = a->dtype == VOPS_BF16 ? 1u : 3u;
  if ((reinterpret_cast<uintptr_t>(a->student) | reinterpret_cast<uintptr_t>(a->out_grad)) & mask)
    return fail(VOPS_E_ARG, "student and out_grad must be aligned to their elements");
  return VOPS_OK;
}

vo::DistillArgs distill_args(const vops_distill_args* a, int S) {
  vo::DistillArgs d;
  std::memset(&d, 0, sizeof d);
  d.x = a->student;
  d.stride = a->row_stride;
  d.T = a->rows;
  d.V = a->vocab;
  d.K = a->entries;
  d.S = S;
  d.ids = a->ids;
  d.teacher = a->teacher;
  d.weights = a->weights;
  d.inv = 1.0 / a->temperature;
  d.c = static_cast<float>(1.4426950408889634 / a->temperature);
  d.tail = (a->flags & VOPS_DISTILL_TAIL) != 0;
  d.loss = a->out_loss;
  d.grad = a->out_grad;
  d.gstride = a->grad_stride;
  return d;
}

constexpr int kHeldMostVectors = 1024 * 19;  // (of the last VO_HELD below)

// Whether loss and gradient go by the held form.
bool held(const vops_distill_args* a) {
  return a->out_grad && !a->states && (a->rows >= kHeldRows || a->vocab <= kHeldVectors * kVecElems[a->dtype]) &&
         a->vocab >= kHeldVocab && a->entries <= kHeldEntries && a->vocab / kVecElems[a->dtype] <= kHeldMostVectors;
}

// Its launch: the first of these whose registers take a row.
template <class Tin>
void launch_held(const vo::DistillArgs& k, hipStream_t st) {
  const int nvec = k.V / vo::Vec<Tin>::kElems;
#define VO_HELD(THREADS, NS, ROWS_A_CU)                                                                  \
  if (nvec <= THREADS * NS) {                                                                            \
    const int grid = k.T < 256 * ROWS_A_CU ? k.T : 256 * ROWS_A_CU;                                      \
    hipLaunchKernelGGL((vo::k_distill_held<Tin, THREADS, NS, ROWS_A_CU>), dim3(grid), dim3(THREADS), 0, st, k);     \
    return;                                                                                              \
  }
  VO_HELD(512, 8, 3)
  VO_HELD(512, 16, 2)
  VO_HELD(512, 20, 2)
  VO_HELD(1024, 13, 1)
  VO_HELD(1024, 16, 1)
  VO_HELD(1024, 19, 1)
#undef VO_HELD
}

// (a launch has fewer than 2^32 threads in a dimension, and a segment has a workgroup)
int grid_ok(int64_t workgroups) {
  static_assert(VOPS_MAX_DISTILL_SEGMENTS * int64_t(vo::kDistillThreads) < (int64_t(1) << 32), "");
  return workgroups <= VOPS_MAX_DISTILL_SEGMENTS
             ? VOPS_OK
             : fail(VOPS_E_ARG, "too many rows for one call: %lld segments, at most %d", static_cast<long long>(workgroups),
                    VOPS_MAX_DISTILL_SEGMENTS);
}

}  // namespace

extern "C" {

int vops_abi_version(void) { return VOPS_ABI_VERSION; }

int vops_query(int device, char* why, size_t n) {
  if (why && n) why[0] = 0;
  return check_device(device, why, n);
}

const char* vops_last_error(void) { return g_err; }

size_t vops_beam_workspace_bytes(int32_t dtype, int32_t requests, int32_t beams, int32_t vocab, int32_t n) {
  return beam_sizes_ok(dtype, requests, beams, vocab, n) ? beam_layout(dtype, requests, beams, vocab, n).total : 0;
}

int vops_beam_select(const vops_beam_args* a, void* stream) {
  g_err[0] = 0;
  if (!a) return fail(VOPS_E_ARG, "args is NULL");
  if (a->dtype != VOPS_BF16 && a->dtype != VOPS_F32)
    return fail(VOPS_E_DTYPE, "unsupported logits dtype %d (VOPS_BF16=0, VOPS_F32=1)", a->dtype);
  if (!beam_sizes_ok(a->dtype, a->requests, a->beams, a->vocab, a->n))
    return fail(VOPS_E_ARG, "requests must be in [0, 65535], beams in [1, %d], vocab in [1, %d], n in [1, %d], got %d, %d, %d, %d",
                VOPS_MAX_BEAMS, VOPS_MAX_VOCAB, VOPS_MAX_CONTINUATIONS, a->requests, a->beams, a->vocab, a->n);
  if (a->flags & ~VOPS_BEAM_KEEP_SLOTS) return fail(VOPS_E_ARG, "flags must be 0 or VOPS_BEAM_KEEP_SLOTS, got %u", a->flags);
  if ((a->flags & VOPS_BEAM_KEEP_SLOTS) && a->n != a->beams)
    return fail(VOPS_E_ARG, "VOPS_BEAM_KEEP_SLOTS needs n (%d) = beams (%d)", a->n, a->beams);
  if (a->request_stride < 0 || a->beam_stride < 0) return fail(VOPS_E_ARG, "strides must be >= 0");
  if (a->requests == 0) return VOPS_OK;
  if (!a->logits || !a->scores || !a->out_scores || !a->out_beams || !a->out_tokens)
    return fail(VOPS_E_ARG, "logits, scores, out_scores, out_beams and out_tokens must be set");
  if (reinterpret_cast<uintptr_t>(a->logits) & (a->dtype == VOPS_BF16 ? 1u : 3u))
    return fail(VOPS_E_ARG, "logits must be aligned to their elements");
  const BeamLayout L = beam_layout(a->dtype, a->requests, a->beams, a->vocab, a->n);
  if (int rc = check_workspace(a->workspace, a->workspace_bytes, L.total)) return rc;
  if (int rc = check_current_device()) return rc;
  char* ws = static_cast<char*>(a->workspace);
  vo::BeamArgs k;
  k.logits = a->logits;
  k.rstride = a->request_stride;
  k.bstride = a->beam_stride;
  k.B = a->requests;
  k.W = a->beams;
  k.V = a->vocab;
  k.n = a->n;
  k.S = L.S;
  k.scores = a->scores;
  k.finished = a->finished;
  k.pad = a->pad_id;
  k.keep = (a->flags & VOPS_BEAM_KEEP_SLOTS) != 0;
  k.row_magic = static_cast<uint32_t>((uint64_t(1) << 32) / (static_cast<uint64_t>(L.S) * a->n)) + 1u;
  k.list_magic = static_cast<uint32_t>((uint64_t(1) << 32) / static_cast<uint64_t>(a->n)) + 1u;
  k.keys = reinterpret_cast<vs::u64*>(ws + L.keys);
  k.sums = reinterpret_cast<double*>(ws + L.sums);
  k.maxs = reinterpret_cast<float*>(ws + L.maxs);
  k.out_scores = a->out_scores;
  k.out_beams = a->out_beams;
  k.out_tokens = a->out_tokens;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid(L.S, a->beams, a->requests);
  with_nv(L.nv, [&](auto nv) {
    constexpr int N = decltype(nv)::value;
    const bool bf = a->dtype == VOPS_BF16, many = a->n > kManyContinuations;
    const dim3 block(vo::kPartThreads);
    if (bf && many) hipLaunchKernelGGL((vo::k_beam_part<uint16_t, N, true>), grid, block, 0, st, k);
    else if (bf) hipLaunchKernelGGL((vo::k_beam_part<uint16_t, N, false>), grid, block, 0, st, k);
    else if (many) hipLaunchKernelGGL((vo::k_beam_part<float, N, true>), grid, block, 0, st, k);
    else hipLaunchKernelGGL((vo::k_beam_part<float, N, false>), grid, block, 0, st, k);
  });
  if (int rc = launched("launch k_beam_part")) return rc;
  // (4 entries a thread, if 16 waves have as many)
  const int64_t entries = static_cast<int64_t>(a->beams) * L.S * a->n;
  const int threads = entries <= 1024 ? 256 : entries <= 2048 ? 512 : 1024;
  hipLaunchKernelGGL(vo::k_beam_merge, dim3(a->requests), dim3(threads), 0, st, k);
  return launched("launch k_beam_merge");
}

int64_t vops_state_columns(const vops_state* s) {
  if (!s || !s->data || s->run < 1 || s->slot_stride < 0 || s->length_dim < -1 || s->length_dim > 3) return -1;
  if (s->length_dim == 3 && (s->unit < 1 || s->max_length < 1 || s->unit * s->max_length != s->run)) return -1;
  int64_t rows = 1;
  for (int i = 0; i < 3; ++i) {
    if (s->size[i] < 1 || s->stride[i] < 0) return -1;
    if (s->length_dim == i && s->max_length != s->size[i]) return -1;
    rows *= s->size[i];
    if (rows >= (int64_t(1) << 31)) return -1;
  }
  const int64_t cols = (s->run + 15) / 16;
  if (cols >= (int64_t(1) << 31) || rows * cols >= (int64_t(1) << 31)) return -1;
  return rows * cols;
}

int vops_reorder(const vops_state* states, int32_t n_states, int64_t max_columns, int32_t requests, int32_t beams,
                 const int32_t* parents, const int32_t* lengths, void* stream) {
  g_err[0] = 0;
  if (n_states < 0 || n_states > 65535) return fail(VOPS_E_ARG, "n_states must be in [0, 65535], got %d", n_states);
  if (requests < 0 || requests > 65535) return fail(VOPS_E_ARG, "requests must be in [0, 65535], got %d", requests);
  if (beams < 1 || beams > VOPS_MAX_REORDER_BEAMS)
    return fail(VOPS_E_ARG, "beams must be in [1, %d], got %d", VOPS_MAX_REORDER_BEAMS, beams);
  if (max_columns < 0 || max_columns >= (int64_t(1) << 31))
    return fail(VOPS_E_ARG, "max_columns must be in [0, 2^31), got %lld", static_cast<long long>(max_columns));
  if (n_states == 0 || requests == 0 || beams == 1 || max_columns == 0) return VOPS_OK;
  if (!states || !parents) return fail(VOPS_E_ARG, "states and parents must be set");
  if (int rc = check_current_device()) return rc;
  static_assert(sizeof(vo::StateDesc) == sizeof(vops_state), "one layout");
  // (as many workgroups a state and request as its columns need, up to 65536 in all: with 16384, caches of 16 x 4
  // beams take 434 us against 411, 16 x 8 beams' matrices 306 against 285)
  int64_t x = (max_columns + vo::kReorderColumns - 1) / vo::kReorderColumns;
  const int64_t most = 65536 / (static_cast<int64_t>(n_states) * requests);
  if (x > most) x = most < 1 ? 1 : most;
  const dim3 grid(static_cast<unsigned>(x), n_states, requests);
  const auto* d = reinterpret_cast<const vo::StateDesc*>(states);
  hipStream_t st = static_cast<hipStream_t>(stream);
#define VO_REORDER(N) hipLaunchKernelGGL(vo::k_reorder<N>, grid, dim3(vo::kReorderThreads), 0, st, d, parents, lengths, beams)
  if (beams <= 4) VO_REORDER(4);
  else if (beams <= 8) VO_REORDER(8);
  else if (beams <= 16) VO_REORDER(16);
  else VO_REORDER(32);
#undef VO_REORDER
  return launched("launch k_reorder");
}

size_t vops_distill_workspace_bytes(int32_t dtype, int32_t rows, int32_t vocab, int32_t entries) {
  return distill_sizes_ok(dtype, rows, vocab, entries) ? distill_layout(dtype, rows, vocab, entries).total : 0;
}

int vops_distill(const vops_distill_args* a, void* stream) {
  g_err[0] = 0;
  if (int rc = distill_common(a)) return rc;
  if (a->rows == 0) return VOPS_OK;
  if (!a->teacher || !a->out_loss) return fail(VOPS_E_ARG, "teacher and out_loss must be set");
  const DistillLayout L = distill_layout(a->dtype, a->rows, a->vocab, a->entries);
  if (int rc = check_workspace(a->workspace, a->workspace_bytes, L.total)) return rc;
  const int64_t parts = static_cast<int64_t>(a->rows) * L.S;
  const bool in_one = held(a);  // (in strides over the rows)
  if (int rc = in_one ? VOPS_OK : grid_ok(parts)) return rc;
  if (int rc = check_current_device()) return rc;
  char* ws = static_cast<char*>(a->workspace);
  vo::DistillArgs k = distill_args(a, L.S);
  k.sums = reinterpret_cast<double*>(ws + L.sums);
  k.maxs = reinterpret_cast<float*>(ws + L.maxs);
  k.states = a->states ? a->states : reinterpret_cast<float*>(ws + L.states);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const bool bf = a->dtype == VOPS_BF16;
  if (in_one) {
    if (bf) launch_held<uint16_t>(k, st);
    else launch_held<float>(k, st);
    return launched("launch k_distill_held");
  }
  const dim3 grid(static_cast<unsigned>(parts)), block(vo::kDistillThreads);
  const dim3 rows((a->rows + vo::kDistillWaves - 1) / vo::kDistillWaves);
  with_nv(L.nv, [&](auto nv) {
    constexpr int N = decltype(nv)::value;
    if (bf) hipLaunchKernelGGL((vo::k_distill_part<uint16_t, N>), grid, block, 0, st, k);
    else hipLaunchKernelGGL((vo::k_distill_part<float, N>), grid, block, 0, st, k);
  });
  if (int rc = launched("launch k_distill_part")) return rc;
  const bool one = a->entries <= vs::kWave;
  const bool in_grad = a->out_grad && !a->states && one && a->rows < kFewRows;
  if (!in_grad) {
    if (bf && one) hipLaunchKernelGGL((vo::k_distill_row<uint16_t, true>), rows, block, 0, st, k);
    else if (bf) hipLaunchKernelGGL((vo::k_distill_row<uint16_t, false>), rows, block, 0, st, k);
    else if (one) hipLaunchKernelGGL((vo::k_distill_row<float, true>), rows, block, 0, st, k);
    else hipLaunchKernelGGL((vo::k_distill_row<float, false>), rows, block, 0, st, k);
    if (int rc = launched("launch k_distill_row")) return rc;
  }
  if (!a->out_grad) return VOPS_OK;
  with_nv(L.nv, [&](auto nv) {
    constexpr int N = decltype(nv)::value;
    if (bf && in_grad) hipLaunchKernelGGL((vo::k_distill_grad<uint16_t, N, true>), grid, block, 0, st, k);
    else if (bf) hipLaunchKernelGGL((vo::k_distill_grad<uint16_t, N, false>), grid, block, 0, st, k);
    else if (in_grad) hipLaunchKernelGGL((vo::k_distill_grad<float, N, true>), grid, block, 0, st, k);
    else hipLaunchKernelGGL((vo::k_distill_grad<float, N, false>), grid, block, 0, st, k);
  });
  return launched("launch k_distill_grad");
}

int vops_distill_grad(const vops_distill_args* a, void* stream) {
  g_err[0] = 0;
  if (int rc = distill_common(a)) return rc;
  if (a->rows == 0) return VOPS_OK;
  if (!a->states || !a->out_grad) return fail(VOPS_E_ARG, "states and out_grad must be set");
  const DistillLayout L = distill_layout(a->dtype, a->rows, a->vocab, a->entries);
  const int64_t parts = static_cast<int64_t>(a->rows) * L.S;
  if (int rc = grid_ok(parts)) return rc;
  if (int rc = check_current_device()) return rc;
  vo::DistillArgs k = distill_args(a, L.S);
  k.states = a->states;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(parts)), block(vo::kDistillThreads);
  with_nv(L.nv, [&](auto nv) {
    constexpr int N = decltype(nv)::value;
    if (a->dtype == VOPS_BF16) hipLaunchKernelGGL((vo::k_distill_grad<uint16_t, N, false>), grid, block, 0, st, k);
    else hipLaunchKernelGGL((vo::k_distill_grad<float, N, false>), grid, block, 0, st, k);
  });
  return launched("launch k_distill_grad");
}

}  // extern "C"
