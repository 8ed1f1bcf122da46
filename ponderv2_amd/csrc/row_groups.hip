// Rows by id: the stable order of n rows by an integer id and the offset of every id's rows in it - what the gradient
// of an embedding (embedding.hip) and the products with per-group weights (grouped_linear.hip) need.
//
// A stable radix sort, least significant digit first, of key(i) = id if 0 <= id < G, else G (so rows without a group
// come last, in row order).  Digits of up to 10 bits: one pass for G < 1024, two up to 2^20.  A pass is
//   count    every block's histogram of its 512 to 4096 keys,
//   scan     one block per digit over the blocks' counts (few counts: every block of the next kernel adds them itself),
//   scatter  every wave walks its quarter of the block's keys in order, 64 at a time; lanes with equal digits find each
//            other by one ballot per digit bit, and a lane's place is (start of the digit) + (earlier blocks and waves) +
//            (earlier rounds and equal lanes below it, known from counting).
// One LDS update for all equal lanes: with a handful of groups (or the few frequent ids of a vocabulary) an atomic per key
// would queue at a handful of addresses.
// Sums of counts are whole numbers, so nothing depends on the order in which blocks or threads run.  Bound by latency: a pass
// moves 16 bytes a key, and blocks are as small as keeps 256 CUs busy.  Up to 4096 rows one workgroup does all passes in LDS
// in a single launch.  Measured on MI355X: 64 ids 3.4 us; 32 768 ids over 65 536 rows 28 us in a graph, 32 as separate
// launches; 1 000 003 ids over 50 021 groups 57 us (count 6.5, scan 4.4, scatter 14.4 per pass, offsets 7; 12.2 MB at the rate
// of a copy are 2.4).
#include "common.h"
#include "sorted_search.h"

namespace {

constexpr int kThreads = 256;
constexpr int kMaxTile = 4096;     // most keys per block of the multi-block sort
// counts that every block adds up itself (32768 ids, 16 groups, 2048 counts: 7.3 us in all against 9.0 with a scan launch;
// 131072 ids, 8192 counts: 8.6 against 9.3; 92001 ids, 36 groups, 11520 counts: 10.7 against 9.7)
constexpr int kFewCounts = 8192;
constexpr int kMaxBits = 10;
constexpr int kMaxDigits = 1 << kMaxBits;
// rows that one workgroup sorts in LDS (1500 ids, 16 groups: 5.5 us against 7.0 by many workgroups, 1000 groups: 7.9 against
// 12.6; 4096 ids, 16 groups: 7.7 against 7.1, 1000 groups: 11.5 against 12.3)
constexpr int kSmall = 4096;
constexpr int kSmallThreads = 1024;
constexpr int kSmallBits = 8;

__device__ __forceinline__ int key_of(const void* index, int is64, int64_t i, int n_groups) {
  const int64_t id = is64 ? ((const int64_t*)index)[i] : (int64_t)((const int32_t*)index)[i];
  return (id >= 0 && id < n_groups) ? (int)id : n_groups;
}

// lanes of `active` that hold the same digit as this one
__device__ __forceinline__ uint64_t same_digit(int digit, int bits, uint64_t active) {
  uint64_t m = active;
  for (int b = 0; b < bits; ++b) {
    const uint64_t set = __ballot((digit >> b) & 1);
    m &= ((digit >> b) & 1) ? set : ~set;
  }
  return m;
}

__device__ __forceinline__ int wave_inclusive_scan(int v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int t = __shfl_up(v, d);
    if (lane >= d) v += t;
  }
  return v;
}

// exclusive scan over the block's threads; *total: the sum
template <int THREADS>
__device__ __forceinline__ int block_exclusive_scan(int v, int* s_wave, int* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int inc = wave_inclusive_scan(v);
  __syncthreads();
  if (lane == 63) s_wave[wave] = inc;
  __syncthreads();
  int before = 0, sum = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) {
    if (w < wave) before += s_wave[w];
    sum += s_wave[w];
  }
  *total = sum;
  return before + inc - v;
}

struct Source {      // keys of a pass: the caller's ids (first pass) or the previous pass's keys
  const void* index;
  int is64;
  const int32_t* keys;
  int n_groups;
  __device__ __forceinline__ int operator()(int64_t i) const {
    return keys ? keys[i] : key_of(index, is64, i, n_groups);
  }
};

// counts[digit] += number of lanes that hold it, for the lanes with `ok`; counts belongs to this wave alone.  Returns how
// many keys with the digit came before this lane's.
__device__ __forceinline__ int count_lanes(volatile int* counts, int digit, int bits, bool ok) {
  const uint64_t mine = same_digit(digit, bits, __ballot(ok));
  const int below = __popcll(mine & ((1ull << (threadIdx.x & 63)) - 1));
  const int before = ok ? counts[digit] : 0;
  __builtin_amdgcn_wave_barrier();
  if (ok && below == 0) counts[digit] = before + __popcll(mine);
  __builtin_amdgcn_wave_barrier();
  return before + below;
}

// The block of keys that a workgroup takes.  Workgroups are dealt to the 8 XCDs in turn; each XCD takes a contiguous eighth
// of the blocks, so that the short runs which neighbouring blocks write for a digit meet in one L2 (a million ids: counting
// 8.3 -> 6.5 us, scattering 14.7 -> 14.4).
__device__ __forceinline__ int block_of(int n_blocks) {
  const int x = blockIdx.x & 7;
  return x * (n_blocks >> 3) + min(x, n_blocks & 7) + (int)(blockIdx.x >> 3);
}

// hist[digit][block], or [block][digit] with `by_block`; ROUNDS of 64 keys per wave
template <int ROUNDS>
__global__ __launch_bounds__(kThreads) void count_kernel(Source src, int64_t n, int shift, int bits, int n_blocks,
                                                         bool by_block, int32_t* __restrict__ hist) {
  constexpr int kWaves = kThreads / 64;
  __shared__ int s_count[kWaves][kMaxDigits];
  const int digits = 1 << bits, mask = digits - 1;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, block = block_of(n_blocks);
  const int64_t base = ((int64_t)block * kWaves + wave) * ROUNDS * 64 + lane;
  int key[ROUNDS];
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) key[r] = base + r * 64 < n ? src(base + r * 64) : -1;
  for (int d = lane; d < digits; d += 64) s_count[wave][d] = 0;
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) count_lanes(s_count[wave], (key[r] >> shift) & mask, bits, base + r * 64 < n);
  __syncthreads();
  for (int d = threadIdx.x; d < digits; d += kThreads) {
    int sum = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) sum += s_count[w][d];
    hist[by_block ? (int64_t)block * digits + d : (int64_t)d * n_blocks + block] = sum;
  }
}

// one block per digit: hist[d][.] -> its exclusive prefix, totals[d]
__global__ __launch_bounds__(kThreads) void scan_kernel(int32_t* __restrict__ hist, int n_blocks,
                                                        int32_t* __restrict__ totals) {
  __shared__ int s_wave[kThreads / 64];
  int32_t* row = hist + (int64_t)blockIdx.x * n_blocks;
  int run = 0;
  for (int b = 0; b < n_blocks; b += kThreads) {
    const int i = b + threadIdx.x;
    const int v = i < n_blocks ? row[i] : 0;
    int sum;
    const int before = block_exclusive_scan<kThreads>(v, s_wave, &sum);
    if (i < n_blocks) row[i] = run + before;
    run += sum;
  }
  if (threadIdx.x == 0) totals[blockIdx.x] = run;
}

// offsets != nullptr (the sort's only pass): offsets[g] = start of digit g, g <= n_groups.  totals == nullptr: hist holds
// the blocks' counts [block][digit], not their prefix.
template <int ROUNDS>
__global__ __launch_bounds__(kThreads) void scatter_kernel(Source src, const int32_t* __restrict__ order_in, int64_t n,
                                                           int shift, int bits, int n_blocks,
                                                           const int32_t* __restrict__ hist,
                                                           const int32_t* __restrict__ totals,
                                                           int32_t* __restrict__ keys_out,
                                                           int32_t* __restrict__ order_out,
                                                           int32_t* __restrict__ offsets, int n_groups) {
  constexpr int kWaves = kThreads / 64;
  __shared__ int s_at[kWaves][kMaxDigits];
  __shared__ int s_before[kMaxDigits], s_total[kMaxDigits];   // of a digit: in earlier blocks, in all blocks
  __shared__ int s_wave[kWaves];
  const int digits = 1 << bits, mask = digits - 1;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, block = block_of(n_blocks);
  const int64_t base = ((int64_t)block * kWaves + wave) * ROUNDS * 64 + lane;
  int key[ROUNDS], row[ROUNDS], rank[ROUNDS];   // rank: among the wave's keys with the same digit
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    const int64_t i = base + r * 64;
    key[r] = i < n ? src(i) : -1;
    row[r] = i < n && order_in ? order_in[i] : (int32_t)i;
  }
  if (totals) {
    for (int d = threadIdx.x; d < digits; d += kThreads) {
      s_before[d] = hist[(int64_t)d * n_blocks + block];
      s_total[d] = totals[d];
    }
  } else {
    // digits next to each other in the threads; fewer than 256 digits: the blocks split over the threads as well
    for (int d = threadIdx.x; d < digits; d += kThreads) s_before[d] = s_total[d] = 0;
    __syncthreads();
    const int parts = max(1, kThreads / digits);
    for (int d = threadIdx.x % digits; d < digits; d += kThreads) {
      int before = 0, all = 0;
#pragma unroll 8
      for (int b = threadIdx.x / digits; b < n_blocks; b += parts) {
        const int c = hist[(int64_t)b * digits + d];
        all += c;
        before += b < block ? c : 0;
      }
      if (all) atomicAdd(&s_total[d], all);
      if (before) atomicAdd(&s_before[d], before);
    }
  }
  for (int d = lane; d < digits; d += 64) s_at[wave][d] = 0;
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) rank[r] = count_lanes(s_at[wave], (key[r] >> shift) & mask, bits, base + r * 64 < n);
  __syncthreads();
  // s_at[w][d]: counts -> the place of wave w's first key with digit d
  int start = 0;
  for (int d0 = 0; d0 < digits; d0 += kThreads) {
    const int d = d0 + threadIdx.x;
    int sum;
    const int before = block_exclusive_scan<kThreads>(d < digits ? s_total[d] : 0, s_wave, &sum) + start;
    start += sum;
    if (d < digits) {
      if (offsets && block == 0 && d <= n_groups) offsets[d] = before;
      int at = before + s_before[d];
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const int c = s_at[w][d];
        s_at[w][d] = at;
        at += c;
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    if (base + r * 64 >= n) continue;
    const int at = s_at[wave][(key[r] >> shift) & mask] + rank[r];
    order_out[at] = row[r];
    if (keys_out) keys_out[at] = key[r];
  }
}

__global__ __launch_bounds__(kThreads) void offsets_kernel(const int32_t* __restrict__ keys, int64_t n, int n_groups,
                                                           int32_t* __restrict__ offsets) {
  const int64_t stride = (int64_t)gridDim.x * kThreads;
  for (int64_t g = (int64_t)blockIdx.x * kThreads + threadIdx.x; g <= n_groups; g += stride)
    offsets[g] = pv2::lower_bound(keys, (int)n, (int)g);
}

// All passes of at most kSmall keys in one workgroup; every wave owns a contiguous share of the positions.
__global__ __launch_bounds__(kSmallThreads) void small_kernel(Source src, int n, int key_bits, int n_groups,
                                                              int32_t* __restrict__ keys_out,
                                                              int32_t* __restrict__ order_out,
                                                              int32_t* __restrict__ offsets) {
  constexpr int kWaves = kSmallThreads / 64, kDigits = 1 << kSmallBits;
  __shared__ int s_key[2][kSmall];
  __shared__ int s_row[2][kSmall];
  __shared__ int s_at[kWaves][kDigits];
  __shared__ int s_wave[kWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int rounds = (n + kSmallThreads - 1) / kSmallThreads;   // of 64 keys per wave
  for (int i = tid; i < n; i += kSmallThreads) {
    s_key[0][i] = src(i);
    s_row[0][i] = i;
  }
  int cur = 0;
  for (int shift = 0; shift < key_bits; shift += kSmallBits, cur ^= 1) {
    const int bits = min(kSmallBits, key_bits - shift), mask = (1 << bits) - 1;
    for (int d = tid; d < kWaves * kDigits; d += kSmallThreads) s_at[d / kDigits][d % kDigits] = 0;
    __syncthreads();
    int rank[kSmall / kSmallThreads];
#pragma unroll
    for (int r = 0; r < kSmall / kSmallThreads; ++r) {
      const int i = (wave * rounds + r) * 64 + lane;
      const bool ok = r < rounds && i < n;
      if (r < rounds) rank[r] = count_lanes(s_at[wave], ok ? (s_key[cur][i] >> shift) & mask : 0, bits, ok);
    }
    __syncthreads();
    int count = 0;
    if (tid < kDigits)
      for (int w = 0; w < kWaves; ++w) count += s_at[w][tid];
    int sum;
    int at = block_exclusive_scan<kSmallThreads>(count, s_wave, &sum);
    if (tid < kDigits)
      for (int w = 0; w < kWaves; ++w) {
        const int c = s_at[w][tid];
        s_at[w][tid] = at;
        at += c;
      }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kSmall / kSmallThreads; ++r) {
      const int i = (wave * rounds + r) * 64 + lane;
      if (r < rounds && i < n) {
        const int key = s_key[cur][i], place = s_at[wave][(key >> shift) & mask] + rank[r];
        s_key[cur ^ 1][place] = key;
        s_row[cur ^ 1][place] = s_row[cur][i];
      }
    }
    __syncthreads();
  }
  __syncthreads();
  for (int i = tid; i < n; i += kSmallThreads) {
    order_out[i] = s_row[cur][i];
    if (keys_out) keys_out[i] = s_key[cur][i];
  }
  if (offsets)
    for (int g = tid; g <= n_groups; g += kSmallThreads) offsets[g] = pv2::lower_bound(s_key[cur], n, g);
}

// cumulative row counts (B,) -> offsets [B + 1], never decreasing and within 0 .. n whatever the counts hold.  One wave: the
// scenes of a batch are few (up to 64: 1.5 us; 1000 take 7, 4096 23, 65536 355)
__global__ __launch_bounds__(64) void offsets_from_counts_kernel(const void* cumulative, int is64, int n_groups,
                                                                 int64_t n, int32_t* __restrict__ offsets) {
  const int lane = threadIdx.x;
  int run = 0;
  if (lane == 0) offsets[0] = 0;
  for (int g0 = 0; g0 < n_groups; g0 += 64) {
    const int g = g0 + lane;
    int64_t v = 0;
    if (g < n_groups) v = is64 ? ((const int64_t*)cumulative)[g] : (int64_t)((const int32_t*)cumulative)[g];
    int c = (int)(v < 0 ? 0 : v > n ? n : v);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int t = __shfl_up(c, d);
      if (lane >= d) c = max(c, t);
    }
    c = max(c, run);
    if (g < n_groups) offsets[g + 1] = c;
    run = __shfl(c, 63);
  }
}

bool few_offsets(int64_t n_groups) { return n_groups <= 8 * kSmallThreads; }   // more are searched by many blocks

// 512, 1024 or 4096 keys per block.  (32768 ids, 65536 groups: 28 us with 512, 34 with 1024; 262144 ids, 50021 groups: 33
// and 36; 1000003: 66 and 58; four million, 1000 groups: 88 with 1024, 72 with 4096)
int tile_of(int64_t n) { return n > (1 << 21) ? 4096 : n > (1 << 18) ? 1024 : 512; }

int bits_for(int64_t n_groups) {   // keys 0 .. n_groups
  int b = 1;
  while (b < 31 && (1ll << b) <= n_groups) ++b;
  return b;
}

}  // namespace

extern "C" {

int64_t pv2_row_groups_workspace_ints(int64_t n, int64_t n_groups) {
  if (n <= 0 || n_groups <= 0) return 0;
  if (n <= kSmall) return few_offsets(n_groups) ? 0 : n;
  const int64_t n_blocks = (n + tile_of(n) - 1) / tile_of(n);
  return 3 * n + kMaxDigits * (n_blocks + 1);
}

int pv2_row_groups(const void* index, int index_is_64, int64_t n, int64_t n_groups, int32_t* order, int32_t* offsets,
                   int32_t* sorted_ids, int32_t* workspace, pv2_stream_t stream) {
  PV2_REQUIRE(offsets && n >= 0 && n < (1ll << 31) - kMaxTile, "row_groups: bad row count");
  PV2_REQUIRE(n_groups >= 1 && n_groups <= (1ll << 30), "row_groups: bad group count");
  PV2_REQUIRE(n == 0 || (index && order), "row_groups: null pointer");
  PV2_REQUIRE(workspace || pv2_row_groups_workspace_ints(n, n_groups) == 0, "row_groups: no workspace");
  hipStream_t s = (hipStream_t)stream;
  if (n == 0) return pv2::zero_words(offsets, n_groups + 1, s);
  Source src{index, index_is_64, nullptr, (int)n_groups};
  const int key_bits = bits_for(n_groups);
  if (n <= kSmall) {
    const bool inside = few_offsets(n_groups);
    int32_t* keys = sorted_ids ? sorted_ids : inside ? nullptr : workspace;
    hipLaunchKernelGGL(small_kernel, dim3(1), dim3(kSmallThreads), 0, s, src, (int)n, key_bits, (int)n_groups, keys,
                       order, inside ? offsets : nullptr);
    if (!inside)
      hipLaunchKernelGGL(offsets_kernel, dim3(pv2::grid_for(n_groups + 1, kThreads)), dim3(kThreads), 0, s, keys, n,
                         (int)n_groups, offsets);
    return pv2::check_launch("row_groups");
  }
  const int tile = tile_of(n);
  const int n_blocks = (int)((n + tile - 1) / tile);
  const int passes = (key_bits + kMaxBits - 1) / kMaxBits;
  const int bits = (key_bits + passes - 1) / passes;
  int32_t* keys[2] = {workspace, workspace + n};
  int32_t* other = workspace + 2 * n;
  int32_t* hist = workspace + 3 * n;
  int32_t* totals = hist + (int64_t)kMaxDigits * n_blocks;
  const int32_t* order_in = nullptr;
  for (int p = 0; p < passes; ++p) {
    const bool last = p == passes - 1;
    int32_t* order_out = ((passes - 1 - p) & 1) ? other : order;
    int32_t* keys_out = last ? (sorted_ids ? sorted_ids : passes > 1 ? keys[p & 1] : nullptr) : keys[p & 1];
    const int shift = p * bits, digits = 1 << bits;
    const bool few = (int64_t)digits * n_blocks <= kFewCounts;
#define PV2_PASS(ROUNDS)                                                                                              \
  do {                                                                                                                \
    hipLaunchKernelGGL(count_kernel<ROUNDS>, dim3(n_blocks), dim3(kThreads), 0, s, src, n, shift, bits, n_blocks, few, \
                       hist);                                                                                         \
    if (!few) hipLaunchKernelGGL(scan_kernel, dim3(digits), dim3(kThreads), 0, s, hist, n_blocks, totals);             \
    hipLaunchKernelGGL(scatter_kernel<ROUNDS>, dim3(n_blocks), dim3(kThreads), 0, s, src, order_in, n, shift, bits,    \
                       n_blocks, hist, few ? nullptr : totals, keys_out, order_out, passes == 1 ? offsets : nullptr,   \
                       (int)n_groups);                                                                                \
  } while (0)
    if (tile == 512) PV2_PASS(2);
    else if (tile == 1024) PV2_PASS(4);
    else PV2_PASS(16);
#undef PV2_PASS
    src.keys = keys_out;
    order_in = order_out;
  }
  if (passes > 1)
    hipLaunchKernelGGL(offsets_kernel, dim3(pv2::grid_for(n_groups + 1, kThreads)), dim3(kThreads), 0, s, src.keys, n,
                       (int)n_groups, offsets);
  return pv2::check_launch("row_groups");
}

int pv2_row_offsets(const void* cumulative, int is_64, int64_t n_groups, int64_t n, int32_t* offsets,
                    pv2_stream_t stream) {
  PV2_REQUIRE(cumulative && offsets, "row_offsets: null pointer");
  PV2_REQUIRE(n >= 0 && n < (1ll << 31) - kMaxTile && n_groups >= 1 && n_groups <= (1ll << 30), "row_offsets: bad shape");
  hipLaunchKernelGGL(offsets_from_counts_kernel, dim3(1), dim3(64), 0, (hipStream_t)stream, cumulative, is_64,
                     (int)n_groups, n, offsets);
  return pv2::check_launch("row_offsets");
}

}  // extern "C"
