// C ABI of libvpaged.so (declared in include/vpaged.h).
#include <hip/hip_runtime.h>

#include <atomic>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <cstring>

#include "../../include/vpaged.h"
#include "attend.cuh"
#include "rotary.cuh"
#include "tables.cuh"

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

int hip_fail(hipError_t e, const char* what) { return fail(VPAGED_E_HIP, "%s: %s", what, hipGetErrorString(e)); }

int launched(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? VPAGED_OK : hip_fail(e, what);
}

constexpr int kMaxDevices = 64;
std::atomic<int> g_dev_ok[kMaxDevices];  // 0 unknown, 1 gfx950

int check_device(int dev, char* why, size_t n) {
  if (dev >= 0 && dev < kMaxDevices && g_dev_ok[dev].load() == 1) return VPAGED_OK;
  int count = 0;
  hipError_t e = hipGetDeviceCount(&count);
  if (e != hipSuccess || count == 0) {
    if (why && n) snprintf(why, n, "no HIP device available");
    return VPAGED_E_DEVICE;
  }
  if (dev < 0 || dev >= count) {
    if (why && n) snprintf(why, n, "device %d out of range (%d devices)", dev, count);
    return VPAGED_E_DEVICE;
  }
  hipDeviceProp_t prop;
  e = hipGetDeviceProperties(&prop, dev);
  if (e != hipSuccess) {
    if (why && n) snprintf(why, n, "hipGetDeviceProperties: %s", hipGetErrorString(e));
    return VPAGED_E_HIP;
  }
  if (std::strncmp(prop.gcnArchName, "gfx950", 6) != 0) {
    if (why && n) snprintf(why, n, "needs a gfx950 (MI355X) GPU, device %d is %s", dev, prop.gcnArchName);
    return VPAGED_E_DEVICE;
  }
  if (dev < kMaxDevices) g_dev_ok[dev].store(1);
  return VPAGED_OK;
}

int check_current_device() {
  int dev = 0;
  const hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return hip_fail(e, "hipGetDevice");
  char why[256];
  const int rc = check_device(dev, why, sizeof why);
  return rc ? fail(rc, "%s", why) : VPAGED_OK;
}

int check_memory(const char* name, const void* p, size_t given, size_t need) {
  if (given < need || (need && !p)) return fail(VPAGED_E_WORKSPACE, "%s of %zu bytes given, %zu needed", name, given, need);
  if (reinterpret_cast<uintptr_t>(p) & 255u) return fail(VPAGED_E_WORKSPACE, "%s must be 256-byte aligned", name);
  return VPAGED_OK;
}

bool power_of_two(int64_t x) { return x > 0 && !(x & (x - 1)); }
bool page_size_ok(int64_t x) { return power_of_two(x) && x <= VPAGED_MAX_PAGE_SIZE; }
int log2_of(int x) { return 31 - __builtin_clz(static_cast<unsigned>(x)); }

vpg::Div div_by(int d) {  // (d >= 1; exact below 2^31)
  vpg::Div r{0, 0, d};
  if (d > 1) {
    r.shift = 31 - __builtin_clz(static_cast<unsigned>(d - 1));  // ceil(log2 d) - 1
    r.mul = static_cast<uint32_t>(((1ull << (32 + r.shift)) + d - 1) / d);
  }
  return r;
}

// Up to this many tokens the workgroup that takes the pages writes the slots too; more are written over the chip.
constexpr int kFewTokens = 8192;

int check_tables(const vpaged_tables* t) {
  if (!t) return fail(VPAGED_E_ARG, "tables is NULL");
  if (t->sequences < 0 || t->sequences > VPAGED_MAX_SEQUENCES || t->max_pages < 1 || t->pages < 1 ||
      static_cast<int64_t>(t->sequences) * t->max_pages >= 1ll << 31)
    return fail(VPAGED_E_ARG, "sequences must be in [0, %d], max_pages and pages >= 1, sequences * max_pages < 2^31, got %d, %d, %d",
                VPAGED_MAX_SEQUENCES, t->sequences, t->max_pages, t->pages);
  if (!page_size_ok(t->page_size) || static_cast<int64_t>(t->pages) * t->page_size >= 1ll << 31)
    return fail(VPAGED_E_ARG, "page_size must be a power of two up to %d, pages * page_size < 2^31, got %d and %d pages",
                VPAGED_MAX_PAGE_SIZE, t->page_size, t->pages);
  if (t->sequences && (!t->tables || !t->lengths || !t->free_pages || !t->free_count))
    return fail(VPAGED_E_ARG, "tables, lengths, free_pages and free_count must be set");
  return VPAGED_OK;
}

vpg::Tables tables_of(const vpaged_tables* t) {
  return {t->tables, t->lengths, t->free_pages, t->free_count, t->sequences, t->max_pages, t->pages, log2_of(t->page_size)};
}

constexpr int kCus = 256;

// LDS and registers hold two workgroups a CU for heads of up to 128 elements.
bool shape_of(const vpaged_shape* a, vpg::Shape& z) {
  if (!a || a->sequences < 0 || a->sequences > VPAGED_MAX_SEQUENCES || a->groups < 0 || a->groups > VPAGED_MAX_SEQUENCES ||
      a->queries < 1 || a->queries > VPAGED_MAX_QUERIES || a->kv_heads < 1 || a->heads < 1 || a->heads > VPAGED_MAX_HEADS ||
      a->heads % a->kv_heads || a->head_dim < 8 || a->head_dim > VPAGED_MAX_HEAD_DIM || a->head_dim % 8 ||
      !page_size_ok(a->page_size) || a->max_pages < 1 || (a->groups > 0 && a->max_prefix_pages < 1))
    return false;
  z.S = a->sequences;
  z.B = a->groups;
  z.T = a->queries;
  z.H = a->heads;
  z.Hkv = a->kv_heads;
  z.D = a->head_dim;
  z.shift = log2_of(a->page_size);
  z.M = a->max_pages;
  z.MP = a->groups > 0 ? a->max_prefix_pages : 0;
  z.G = z.H / z.Hkv;
  const int64_t rows = static_cast<int64_t>(z.T) * z.G, own = (rows + vpg::kRows - 1) / vpg::kRows;
  const bool own_narrow = rows <= vpg::kNarrow;
  // (a wide group has more than kNarrow rows)
  const int64_t all = static_cast<int64_t>(z.S) * rows, groups = all / (vpg::kNarrow + 1);
  const int64_t wide = (z.B ? (z.B < groups ? z.B : groups) + all / vpg::kRows : 0) + (own_narrow ? 0 : z.S * own);
  const int64_t narrow = z.B + (own_narrow ? z.S : 0);
  z.wgs = kCus * (z.D > 128 ? 1 : 2);
  // (32 bits number a head's tiles, a stretch's of all heads' tiles, and the segments' rows)
  const int64_t pages = z.M > z.MP ? z.M : z.MP;
  const double tiles = static_cast<double>(wide + narrow) * static_cast<double>((pages << z.shift) / vpg::kNarrowKeys + 1 + vpg::kLead);
  if (rows >= 1ll << 24 || z.S * rows >= 1ll << 31 || z.S * own >= 1ll << 31 || tiles >= 2147483648.0 ||
      tiles * z.Hkv >= 2147483647.0 * z.wgs)
    return false;
  z.rows = static_cast<int>(rows);
  z.own_tiles = static_cast<int>(own);
  z.max_wide = static_cast<int>(wide);
  z.max_narrow = static_cast<int>(narrow);
  return true;
}

struct AttendLayout {
  int narrow_rows, own_rows;
  int64_t narrow_cut_at, wide_at, prefix_at, own_at, rows;
  size_t ml, total;
};
AttendLayout attend_layout(const vpg::Shape& z) {
  AttendLayout L;
  const int64_t group = z.B ? static_cast<int64_t>(z.S) * z.rows : z.rows;  // (all sequences in one)
  L.narrow_rows = group < vpg::kNarrow ? static_cast<int>(group) : vpg::kNarrow;
  L.own_rows = z.rows < vpg::kNarrow ? z.rows : vpg::kNarrow;
  L.narrow_cut_at = z.max_wide ? 2ll * z.wgs * vpg::kRows : 0;
  L.wide_at = L.narrow_cut_at + (z.max_narrow ? 2ll * z.wgs * vpg::kWaves * L.narrow_rows : 0);
  // (whole segments leave parts only where there are prefixes)
  L.prefix_at = L.wide_at + (z.B ? static_cast<int64_t>(z.max_wide) * z.Hkv * vpg::kRows : 0);
  L.own_at = L.prefix_at + static_cast<int64_t>(z.B) * z.Hkv * L.narrow_rows;
  L.rows = L.own_at + (z.B && z.rows <= vpg::kNarrow ? static_cast<int64_t>(z.S) * z.Hkv * L.own_rows : 0);
  L.ml = static_cast<size_t>(L.rows) * z.D * 4;
  L.ml = (L.ml + 255) & ~static_cast<size_t>(255);
  L.total = L.ml + static_cast<size_t>(L.rows) * 8;
  return L;
}

size_t plan_bytes(const vpg::Shape& z) {
  size_t n;
  vpg::plan_at(z, nullptr, &n);
  return n;
}

const char* const kShapeRule =
    "the shape is refused: sequences and groups in [0, 65536], queries in [1, 65536], heads a multiple of kv_heads up to 1024, head_dim a "
    "multiple of 8 in [8, 256], page_size a power of two up to 4096, tables of at least a page, fewer than 2^31 rows and tiles of a head, and "
    "of all heads' tiles fewer than 2^31 for each of 256 workgroups";

// f(a tag whose ::value is the head's elements rounded up) for a head of D
template <int N>
struct Width {
  static constexpr int value = N;
};
template <class F>
void with_width(int D, F f) {
  if (D <= 64) f(Width<64>{});
  else if (D <= 96) f(Width<96>{});
  else if (D <= 128) f(Width<128>{});
  else if (D <= 192) f(Width<192>{});
  else f(Width<256>{});
}

// Up to this many rows of outputs (a sequence's token's head each) 16 waves join one: the longest has few others beside it.
constexpr int kFewRows = 512;

template <class T>
int attend(const vpg::AttendArgs& d, hipStream_t stream) {
  const int64_t rows = static_cast<int64_t>(d.z.S) * d.z.T * d.z.H, fours = (rows + 3) / 4;
  const dim3 join(static_cast<unsigned>(fours < vpg::kGridX ? fours : vpg::kGridX), static_cast<unsigned>((fours + vpg::kGridX - 1) / vpg::kGridX));
  with_width(d.z.D, [&](auto w) {
    constexpr int DP = decltype(w)::value;
    const dim3 grid(2 * d.z.wgs), block(vpg::kWaves * 64);
    if ((1 << d.z.shift) < vpg::kRun) vpg::k_attend<T, DP, true><<<grid, block, 0, stream>>>(d);
    else vpg::k_attend<T, DP, false><<<grid, block, 0, stream>>>(d);
    if (rows <= kFewRows) vpg::k_join<T, DP, 16><<<dim3(static_cast<unsigned>(rows)), dim3(1024), 0, stream>>>(d);
    else vpg::k_join<T, DP, 1><<<join, dim3(256), 0, stream>>>(d);
  });
  return launched("vpaged_attend");
}

template <class T>
void rotate(const vpg::RotateArgs& r, bool vectors, vpg::Pairs pairs, dim3 grid, hipStream_t stream) {
  const dim3 block(vpg::kRotateThreads);
  if (vectors && pairs == vpg::kAdjacent) vpg::k_rotate<T, 8, vpg::kAdjacent><<<grid, block, 0, stream>>>(r);
  else if (vectors && pairs == vpg::kExchanged) vpg::k_rotate<T, 8, vpg::kExchanged><<<grid, block, 0, stream>>>(r);
  else if (vectors) vpg::k_rotate<T, 8, vpg::kHalves><<<grid, block, 0, stream>>>(r);
  else if (pairs == vpg::kAdjacent) vpg::k_rotate<T, 1, vpg::kAdjacent><<<grid, block, 0, stream>>>(r);
  else vpg::k_rotate<T, 1, vpg::kHalves><<<grid, block, 0, stream>>>(r);
}

}  // namespace

extern "C" {

int vpaged_abi_version(void) { return VPAGED_ABI_VERSION; }

int vpaged_query(int device, char* why, size_t n) { return check_device(device, why, n); }

const char* vpaged_last_error(void) { return g_err; }

size_t vpaged_extend_workspace_bytes(int32_t sequences, int32_t tokens) {
  if (sequences < 0 || tokens <= kFewTokens) return 0;
  return (2 * static_cast<size_t>(sequences) + 1) * 4;
}

int vpaged_extend(const vpaged_tables* t, const int32_t* counts, int32_t tokens, int32_t* out_slots, int32_t* out_positions,
                  int32_t* out_sequences, uint8_t* out_served, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_tables(t)) return rc;
  if (tokens < 0 || tokens > VPAGED_MAX_TOKENS) return fail(VPAGED_E_ARG, "tokens must be in [0, %d], got %d", VPAGED_MAX_TOKENS, tokens);
  if (!t->sequences && !tokens) return VPAGED_OK;
  if ((t->sequences && (!counts || !out_served)) || (tokens && (!out_slots || !out_positions || !out_sequences)))
    return fail(VPAGED_E_ARG, "counts and the outputs must be set");
  if (!t->sequences) return fail(VPAGED_E_ARG, "tokens without sequences");
  if (int rc = check_memory("workspace", workspace, workspace_bytes, vpaged_extend_workspace_bytes(t->sequences, tokens))) return rc;
  if (int rc = check_current_device()) return rc;
  const vpg::Tables d = tables_of(t);
  const auto s = static_cast<hipStream_t>(stream);
  int32_t* ws = static_cast<int32_t*>(workspace);
  if (tokens <= kFewTokens) {
    vpg::k_extend<true><<<1, vpg::kTableThreads, 0, s>>>(d, counts, tokens, out_slots, out_positions, out_sequences, out_served, ws);
  } else {
    vpg::k_extend<false><<<1, vpg::kTableThreads, 0, s>>>(d, counts, tokens, out_slots, out_positions, out_sequences, out_served, ws);
    vpg::k_tokens<<<static_cast<unsigned>((static_cast<int64_t>(tokens) + 255) / 256), 256, 0, s>>>(d, tokens, out_slots, out_positions,
                                                                                                 out_sequences, ws);
  }
  return launched("vpaged_extend");
}

int vpaged_shrink(const vpaged_tables* t, const int32_t* lengths, void* stream) {
  if (int rc = check_tables(t)) return rc;
  if (!t->sequences) return VPAGED_OK;
  if (!lengths) return fail(VPAGED_E_ARG, "lengths must be set");
  if (int rc = check_current_device()) return rc;
  vpg::k_shrink<<<1, vpg::kTableThreads, 0, static_cast<hipStream_t>(stream)>>>(tables_of(t), lengths);
  return launched("vpaged_shrink");
}

int vpaged_rotate_store(const vpaged_rotate_args* a, void* stream) {
  if (!a) return fail(VPAGED_E_ARG, "args is NULL");
  if (a->dtype != VPAGED_BF16 && a->dtype != VPAGED_F16)
    return fail(VPAGED_E_DTYPE, "unsupported dtype %d (VPAGED_BF16=0, VPAGED_F16=1)", a->dtype);
  if (a->tokens < 0 || a->heads < 0 || a->heads > VPAGED_MAX_HEADS || a->kv_heads < 0 || a->kv_heads > VPAGED_MAX_HEADS ||
      a->head_dim < 1 || a->head_dim > VPAGED_MAX_HEAD_DIM)
    return fail(VPAGED_E_ARG, "tokens must be >= 0, heads and kv_heads in [0, %d], head_dim in [1, %d], got %d, %d, %d, %d",
                VPAGED_MAX_HEADS, VPAGED_MAX_HEAD_DIM, a->tokens, a->heads, a->kv_heads, a->head_dim);
  if (a->dim < 0 || a->dim > a->head_dim || a->dim % 2)
    return fail(VPAGED_E_ARG, "dim must be even and in [0, head_dim], got %d of %d", a->dim, a->head_dim);
  if (!page_size_ok(a->page_size) || a->pages < 0 || static_cast<int64_t>(a->pages) * a->page_size >= 1ll << 31)
    return fail(VPAGED_E_ARG, "page_size must be a power of two up to %d, pages * page_size < 2^31, got %d and %d pages",
                VPAGED_MAX_PAGE_SIZE, a->page_size, a->pages);
  if (!std::isfinite(a->magnitude)) return fail(VPAGED_E_ARG, "magnitude must be finite");
  if (!a->tokens || (!a->heads && !a->kv_heads)) return VPAGED_OK;
  if ((a->heads && (!a->q || !a->out_q)) || (a->kv_heads && (!a->k || !a->v || (a->pages && (!a->k_pages || !a->v_pages)))) ||
      !a->positions || !a->slots || (a->dim && !a->frequencies))
    return fail(VPAGED_E_ARG, "q, k, v, out_q, the pages, positions, slots and frequencies must be set");
  if (int rc = check_current_device()) return rc;
  const int half = a->dim / 2;
  vpg::RotateArgs r{a->q, a->k, a->v, a->q_stride, a->k_stride, a->v_stride, a->q_head_stride, a->k_head_stride, a->v_head_stride,
                    a->out_q, a->k_pages, a->v_pages, a->page_stride, a->place_stride, a->head_stride, a->positions, a->slots,
                    a->frequencies, a->magnitude, a->tokens, a->heads, a->kv_heads, a->head_dim, a->dim,
                    static_cast<int64_t>(a->pages) * a->page_size, log2_of(a->page_size), 0, {}, {}};
  // 16-byte accesses where every head's row begins and ends on one, and halves' pairs are eight apart in both.
  int64_t all = a->head_dim | (a->interleaved ? 0 : half);
  if (a->heads) all |= a->q_stride | a->q_head_stride;
  if (a->kv_heads) all |= a->k_stride | a->k_head_stride | a->v_stride | a->v_head_stride | a->page_stride | a->place_stride | a->head_stride;
  const uintptr_t at = reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->k) | reinterpret_cast<uintptr_t>(a->v) |
                       reinterpret_cast<uintptr_t>(a->out_q) | reinterpret_cast<uintptr_t>(a->k_pages) | reinterpret_cast<uintptr_t>(a->v_pages);
  const bool vectors = all % 8 == 0 && at % 16 == 0;
  const int E = vectors ? 8 : 1;
  const vpg::Pairs pairs = a->interleaved ? vpg::kAdjacent
                           : vectors && half && power_of_two(a->head_dim) ? vpg::kExchanged
                                                                         : vpg::kHalves;
  const int per_head = (pairs == vpg::kHalves ? a->head_dim - half : a->head_dim) / E;
  r.per_head = div_by(per_head);
  r.tail = div_by(a->head_dim / E);
  r.items = (a->heads + a->kv_heads) * per_head + a->kv_heads * (a->head_dim / E);
  // A workgroup a token; where those are few, a token's items over several.
  const int rounds = (r.items + vpg::kRotateThreads - 1) / vpg::kRotateThreads;
  int y = a->tokens >= 4 * kCus ? 1 : (4 * kCus + a->tokens - 1) / a->tokens;
  if (y > rounds) y = rounds;
  const auto s = static_cast<hipStream_t>(stream);
  for (int left = a->tokens; left > 0; left -= vpg::kGridX) {
    r.N = left < vpg::kGridX ? left : vpg::kGridX;
    const dim3 grid(static_cast<unsigned>(r.N), static_cast<unsigned>(y));
    if (a->dtype == VPAGED_BF16) rotate<__bf16>(r, vectors, pairs, grid, s);
    else rotate<_Float16>(r, vectors, pairs, grid, s);
    // (elements of two bytes; a power of two of them keeps the alignment)
    const auto on = [&](const void* p, int64_t stride) { return static_cast<const char*>(p) + 2 * stride * vpg::kGridX; };
    if (left > vpg::kGridX) {
      r.q = on(r.q, r.q_stride);
      r.k = on(r.k, r.k_stride);
      r.v = on(r.v, r.v_stride);
      r.out_q = static_cast<char*>(r.out_q) + 2 * static_cast<int64_t>(r.heads) * r.D * vpg::kGridX;
      r.positions += vpg::kGridX;
      r.slots += vpg::kGridX;
    }
  }
  return launched("vpaged_rotate_store");
}

size_t vpaged_plan_bytes(const vpaged_shape* shape) {
  vpg::Shape z;
  return shape_of(shape, z) ? plan_bytes(z) : 0;
}

int vpaged_plan(const vpaged_shape* shape, const int32_t* lengths, const int32_t* prefix_lengths, const int32_t* group_starts,
                void* plan, size_t bytes, void* stream) {
  vpg::Shape z;
  if (!shape_of(shape, z)) return fail(VPAGED_E_ARG, "%s", kShapeRule);
  if (!z.S) return VPAGED_OK;
  if (!lengths || (z.B && (!prefix_lengths || !group_starts)))
    return fail(VPAGED_E_ARG, "lengths, and with groups prefix_lengths and group_starts, must be set");
  if (int rc = check_memory("plan", plan, bytes, plan_bytes(z))) return rc;
  if (int rc = check_current_device()) return rc;
  vpg::k_plan<<<1, vpg::kTableThreads, 0, static_cast<hipStream_t>(stream)>>>(z, lengths, prefix_lengths, group_starts, plan);
  return launched("vpaged_plan");
}

size_t vpaged_attend_workspace_bytes(const vpaged_shape* shape) {
  vpg::Shape z;
  return shape_of(shape, z) && z.S ? attend_layout(z).total : 0;
}

int vpaged_attend(const vpaged_attend_args* a, void* stream) {
  if (!a) return fail(VPAGED_E_ARG, "args is NULL");
  if (a->shape.dtype != VPAGED_BF16 && a->shape.dtype != VPAGED_F16)
    return fail(VPAGED_E_DTYPE, "unsupported dtype %d (VPAGED_BF16=0, VPAGED_F16=1)", a->shape.dtype);
  vpg::AttendArgs d{};
  if (!shape_of(&a->shape, d.z)) return fail(VPAGED_E_ARG, "%s", kShapeRule);
  // (normal; scores are fp32)
  if (!(a->scale >= 0x1p-126f && a->scale <= 0x1p64f)) return fail(VPAGED_E_ARG, "scale must be in [2^-126, 2^64], got %g", a->scale);
  if (!d.z.S) return VPAGED_OK;
  if (a->pages < 1 || static_cast<int64_t>(a->pages) * a->shape.page_size >= 1ll << 31)
    return fail(VPAGED_E_ARG, "pages must be >= 1 and pages * page_size < 2^31, got %d", a->pages);
  if (!a->q || !a->k_pages || !a->v_pages || !a->tables || !a->out || (d.z.B && !a->prefix_tables))
    return fail(VPAGED_E_ARG, "q, the pages, the tables and out must be set");
  if ((a->q_stride | a->q_token_stride | a->q_head_stride | a->page_stride | a->place_stride | a->head_stride) % 8 ||
      (reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->k_pages) | reinterpret_cast<uintptr_t>(a->v_pages) |
       reinterpret_cast<uintptr_t>(a->out)) % 16)
    return fail(VPAGED_E_ARG, "q, the pages and out must be 16-byte aligned, with strides of multiples of 8 elements");
  // (offsets within a page, and a page's bytes, in 32 bits)
  if ((a->page_stride | a->place_stride | a->head_stride) < 0 || a->page_stride >= 1ll << 31 ||
      a->place_stride * (a->shape.page_size > vpg::kRun ? a->shape.page_size : vpg::kRun) >= 1ll << 30)
    return fail(VPAGED_E_ARG, "strides of the pages must be >= 0, page_stride below 2^31, a page's positions below 2^30 elements");
  if (a->table_stride < 0 || (d.z.B && a->prefix_table_stride < 0)) return fail(VPAGED_E_ARG, "table strides must be >= 0");
  const AttendLayout L = attend_layout(d.z);
  if (!a->plan || reinterpret_cast<uintptr_t>(a->plan) & 255u) return fail(VPAGED_E_WORKSPACE, "plan must be set and 256-byte aligned");
  if (int rc = check_memory("workspace", a->workspace, a->workspace_bytes, L.total)) return rc;
  if (static_cast<int64_t>(d.z.S) * d.z.T * d.z.H >= 1ll << 31) return fail(VPAGED_E_ARG, "2^31 rows of outputs, or more");
  if (int rc = check_current_device()) return rc;
  d.pages = a->pages;
  d.scale = static_cast<float>(a->scale * 1.4426950408889634);
  d.q = a->q;
  d.q_stride = a->q_stride;
  d.q_token = a->q_token_stride;
  d.q_head = a->q_head_stride;
  d.k = a->k_pages;
  d.v = a->v_pages;
  d.page_bytes = static_cast<uint32_t>(a->page_stride * 2);
  d.place_bytes = static_cast<uint32_t>(a->place_stride * 2);
  d.head_stride = a->head_stride;
  d.tables = a->tables;
  d.prefix_tables = a->prefix_tables;
  d.table_stride = a->table_stride;
  d.prefix_table_stride = a->prefix_table_stride;
  d.out = a->out;
  d.plan = const_cast<void*>(a->plan);
  d.o = static_cast<float*>(a->workspace);
  d.ml = reinterpret_cast<float2*>(static_cast<char*>(a->workspace) + L.ml);
  d.narrow_cut_at = L.narrow_cut_at;
  d.wide_at = L.wide_at;
  d.prefix_at = L.prefix_at;
  d.own_at = L.own_at;
  d.narrow_rows = L.narrow_rows;
  d.own_rows = L.own_rows;
  return a->shape.dtype == VPAGED_BF16 ? attend<__bf16>(d, static_cast<hipStream_t>(stream))
                                       : attend<_Float16>(d, static_cast<hipStream_t>(stream));
}

}  // extern "C"
