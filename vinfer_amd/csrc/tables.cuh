// Page tables from the sequences' lengths: pages taken from a stack, tokens' slots, and pages given back.
//
// With len_s the sequences' lengths and c_s their new positions, sequence s needs
//   need_s = ceil((len_s + c_s) / P) - ceil(len_s / P)
// pages; the i-th page of the whole call (sequences in order) is the i-th from the stack's top, so two prefix sums
// (of c and of need) give every page and every token its place. Bound by latency: one workgroup scans, takes the
// pages and, where there are few tokens, writes them too; nothing waits between workgroups. 256 sequences' step 5 us, and 3
// to take it back; 96 prompts of 150 K tokens in 4500 pages 10 us and 4 for the tokens.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace vpg {

constexpr int kTableThreads = 1024;
// Workgroups over a grid's first dimension (a launch has fewer than 2^32 threads in one): more go on in another, or in another
// launch where that is rare and the kernel short (a second dimension in k_rotate costs 4 tokens' 3.15 us 0.24).
constexpr int kGridX = 1 << 20;

struct Tables {
  int32_t* tables;
  int32_t* lengths;
  int32_t* free_pages;
  int32_t* free_count;
  int S, M, pages, shift;
};

__device__ __forceinline__ int clampi(int x, int lo, int hi) { return min(max(x, lo), hi); }

// The inclusive prefix of x over a wave's lanes (`add` any associative sum whose zero is 0), by moves between lanes.
template <class F>
__device__ __forceinline__ unsigned scan_wave(unsigned x, F add) {
#define VPG_STEP(ctrl, rows) x = add(x, static_cast<unsigned>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), ctrl, rows, 0xf, false)))
  VPG_STEP(0x111, 0xf);  // one lane down a row of 16, two, four, eight
  VPG_STEP(0x112, 0xf);
  VPG_STEP(0x114, 0xf);
  VPG_STEP(0x118, 0xf);
  VPG_STEP(0x142, 0xa);  // each row's last lane to the next row
  VPG_STEP(0x143, 0xc);  // lane 31 to the upper half
#undef VPG_STEP
  return x;
}

// Exclusive prefixes of K numbers over the workgroup, and their totals (every thread). `part`: K words a wave.
template <int K, class F>
__device__ __forceinline__ void scan_exclusive(unsigned (&x)[K], unsigned (&total)[K], unsigned (&part)[K][kTableThreads / 64], F add) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  unsigned inc[K];
#pragma unroll
  for (int k = 0; k < K; ++k) inc[k] = scan_wave(x[k], add);
  __syncthreads();  // (part may still be read from an earlier scan)
  if (lane == 63)
#pragma unroll
    for (int k = 0; k < K; ++k) part[k][wave] = inc[k];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < K; ++k) {
    // (each row of 16 lanes has the waves' sums; a wave takes its own from the lane of its number)
    const unsigned sums = scan_wave(lane < kTableThreads / 64 ? part[k][lane] : 0u, add);
    total[k] = __builtin_amdgcn_readlane(sums, kTableThreads / 64 - 1);
    const unsigned before = wave ? __builtin_amdgcn_readlane(sums, __builtin_amdgcn_readfirstlane(wave) - 1) : 0u;
    const unsigned left = static_cast<unsigned>(__builtin_amdgcn_update_dpp(0, static_cast<int>(inc[k]), 0x138, 0xf, 0xf, false));  // the lane below's
    x[k] = add(before, lane ? left : 0u);
  }
}
struct Add {
  __device__ __forceinline__ unsigned operator()(unsigned a, unsigned b) const { return a + b; }
};
struct AddUpTo {  // (both at most cap <= 2^31)
  unsigned cap;
  __device__ __forceinline__ unsigned operator()(unsigned a, unsigned b) const { return min(a + b, cap); }
};

// The last of the n ascending starts that is <= i (starts[0] <= i).
template <class T>
__device__ __forceinline__ int find(const T* starts, int n, T i) {
  int lo = 0;
  for (int step = 1 << (31 - __clz(n)); step; step >>= 1)
    if (lo + step < n && starts[lo + step] <= i) lo += step;
  return lo;
}

// The token's slot and place; the tables' entries of this call are written.
__device__ __forceinline__ void write_token(const Tables& t, int i, int s, int position, int32_t* slots,
                                            int32_t* positions, int32_t* sequences) {
  const int page = t.tables[static_cast<int64_t>(s) * t.M + (position >> t.shift)];
  slots[i] = static_cast<int>((static_cast<unsigned>(page) << t.shift) + (position & ((1 << t.shift) - 1)));
  positions[i] = position;
  sequences[i] = s;
}

// SELF: this kernel writes the tokens. Else it leaves starts and bases for k_tokens: ws[0..S) a sequence's first token
// (at most N), ws[S..2S) its length before, or -1 where its tokens are none.
template <bool SELF>
__global__ __launch_bounds__(kTableThreads) void k_extend(Tables t, const int32_t* __restrict__ counts, int N,
                                                          int32_t* __restrict__ slots, int32_t* __restrict__ positions,
                                                          int32_t* __restrict__ sequences, uint8_t* __restrict__ served,
                                                          int32_t* __restrict__ ws) {
  __shared__ unsigned part[1][kTableThreads / 64];
  __shared__ int s_page[kTableThreads], s_have[kTableThreads], s_token[kTableThreads], s_base[kTableThreads];
  const int tid = threadIdx.x;
  const int P = 1 << t.shift;
  const int64_t cap = min(static_cast<int64_t>(t.M) << t.shift, static_cast<int64_t>(INT32_MAX));
  const int n_free = clampi(*t.free_count, 0, t.pages);
  const unsigned none = static_cast<unsigned>(N) + 1;  // (what lies past the call's tokens)
  unsigned tokens_before = 0;
  int pages_before = 0, taken = 0;
  for (int base = 0; base < t.S; base += kTableThreads) {
    const int s = base + tid;
    int64_t len = 0, c = 0;
    if (s < t.S) {
      len = t.lengths[s];
      len = len < 0 ? 0 : len > cap ? cap : len;
      c = max(counts[s], 0);
    }
    unsigned scan[1] = {static_cast<unsigned>(min(c, static_cast<int64_t>(none)))}, sum[1];
    scan_exclusive<1>(scan, sum, part, AddUpTo{none});
    const unsigned start = min(tokens_before + scan[0], none), tokens_after = min(tokens_before + sum[0], none);
    const int64_t have = (len + P - 1) >> t.shift, want = (len + c + P - 1) >> t.shift;
    const bool fits = len + c <= cap && start + c <= N;
    const int need = fits ? static_cast<int>(want - have) : 0;
    scan[0] = need;
    scan_exclusive<1>(scan, sum, part, Add{});
    const int first = scan[0], all_pages = sum[0];  // (within this round)
    const bool ok = fits && (need == 0 || pages_before + first + need <= n_free);
    s_page[tid] = first;
    s_have[tid] = ok ? static_cast<int>(have) : -1;
    s_token[tid] = static_cast<int>(min(start, static_cast<unsigned>(N)));
    s_base[tid] = ok ? static_cast<int>(len) : -1;
    if (s < t.S) {
      served[s] = ok;
      if (ok && c) t.lengths[s] = static_cast<int>(len + c);
      if (!SELF) {
        ws[s] = s_token[tid];
        ws[t.S + s] = s_base[tid];
      }
    }
    scan[0] = ok ? need : 0;
    scan_exclusive<1>(scan, sum, part, Add{});  // (its barriers also publish the arrays)
    taken += static_cast<int>(sum[0]);
    const int n = min(t.S - base, kTableThreads);
    for (int i = tid; i < all_pages && pages_before + i < n_free; i += kTableThreads) {
      const int k = find(s_page, n, i);
      if (s_have[k] >= 0)
        t.tables[static_cast<int64_t>(base + k) * t.M + s_have[k] + (i - s_page[k])] = t.free_pages[n_free - 1 - (pages_before + i)];
    }
    if (SELF) {
      __syncthreads();  // (the tables' new entries, seen by this workgroup)
      const int to = static_cast<int>(min(tokens_after, static_cast<unsigned>(N)));
      for (int i = static_cast<int>(min(tokens_before, static_cast<unsigned>(N))) + tid; i < to; i += kTableThreads) {
        const int k = find(s_token, n, i);
        if (s_base[k] >= 0) {
          write_token(t, i, base + k, s_base[k] + (i - s_token[k]), slots, positions, sequences);
        } else {
          slots[i] = positions[i] = sequences[i] = -1;
        }
      }
    }
    tokens_before = tokens_after;
    pages_before += all_pages;
    __syncthreads();
  }
  if (SELF)
    for (int i = static_cast<int>(min(tokens_before, static_cast<unsigned>(N))) + tid; i < N; i += kTableThreads)
      slots[i] = positions[i] = sequences[i] = -1;
  if (tid == 0) {
    *t.free_count = n_free - taken;
    if (!SELF) ws[2 * t.S] = static_cast<int>(min(tokens_before, static_cast<unsigned>(N)));
  }
}

__global__ __launch_bounds__(256) void k_tokens(Tables t, int N, int32_t* __restrict__ slots,
                                                int32_t* __restrict__ positions, int32_t* __restrict__ sequences,
                                                const int32_t* __restrict__ ws) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= N) return;
  if (i < ws[2 * t.S]) {
    const int s = find(ws, t.S, i);
    if (ws[t.S + s] >= 0) return write_token(t, i, s, ws[t.S + s] + (i - ws[s]), slots, positions, sequences);
  }
  slots[i] = positions[i] = sequences[i] = -1;
}

__global__ __launch_bounds__(kTableThreads) void k_shrink(Tables t, const int32_t* __restrict__ to) {
  __shared__ unsigned part[1][kTableThreads / 64];
  __shared__ int s_page[kTableThreads], s_keep[kTableThreads];
  const int tid = threadIdx.x;
  const int P = 1 << t.shift;
  const int64_t cap = min(static_cast<int64_t>(t.M) << t.shift, static_cast<int64_t>(INT32_MAX));
  const int n_free = clampi(*t.free_count, 0, t.pages);
  auto cut = [&](int s, int& keep, int& drop) {  // the sequence's new length
    int64_t len = t.lengths[s];
    len = len < 0 ? 0 : len > cap ? cap : len;
    const int64_t now = min(len, static_cast<int64_t>(max(to[s], 0)));
    keep = static_cast<int>((now + P - 1) >> t.shift);
    drop = static_cast<int>((len + P - 1) >> t.shift) - keep;
    return static_cast<int>(now);
  };
  int total = 0;
  if (t.S > kTableThreads) {  // the whole call's pages first: they are laid from the last one down
    int sum = 0, keep, drop;
    for (int s = tid; s < t.S; s += kTableThreads) {
      cut(s, keep, drop);
      sum += drop;
    }
    unsigned scan[1] = {static_cast<unsigned>(sum)}, all[1];
    scan_exclusive<1>(scan, all, part, Add{});
    total = static_cast<int>(all[0]);
  }
  int before = 0;
  for (int base = 0; base < t.S; base += kTableThreads) {
    const int s = base + tid;
    int keep = 0, drop = 0, now = 0;
    if (s < t.S) now = cut(s, keep, drop);
    unsigned scan[1] = {static_cast<unsigned>(drop)}, sum[1];
    scan_exclusive<1>(scan, sum, part, Add{});
    const int all = static_cast<int>(sum[0]);
    if (t.S <= kTableThreads) total = all;
    s_page[tid] = static_cast<int>(scan[0]);
    s_keep[tid] = keep;
    if (s < t.S) t.lengths[s] = now;
    __syncthreads();
    const int n = min(t.S - base, kTableThreads);
    for (int i = tid; i < all; i += kTableThreads) {
      const int k = find(s_page, n, i);
      const int64_t at = static_cast<int64_t>(n_free) + total - 1 - (before + i);
      if (at >= 0 && at < t.pages)  // (more pages than there are: tables that no call of extend wrote)
        t.free_pages[at] = t.tables[static_cast<int64_t>(base + k) * t.M + s_keep[k] + (i - s_page[k])];
    }
    before += all;
    __syncthreads();
  }
  if (tid == 0) *t.free_count = min(n_free + total, t.pages);
}

}  // namespace vpg
