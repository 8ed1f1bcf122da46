// Linear layers with weights of their own for each group of rows (experts, datasets, scenes):
//     Y[r] = X[r] W[g(r)]^T + b[g(r)],   dX[r] = dY[r] W[g(r)],   dW[g] = dY_g^T X_g,   db[g] = sum of dY_g.
// The rows of a group are order[offsets[g]] .. order[offsets[g + 1] - 1] (order == nullptr: the positions themselves), so
// rows are read and written where they lie and nothing is permuted in memory.  Sizes of groups are known on the device
// only: grids cover the most tiles that M rows in G groups can need, a workgroup finds its group with one wave scan over
// the offsets and workgroups past the last tile leave.
//
// Types: bf16 and fp16 run on their MFMA, fp32 as six bf16 MFMAs over three exact pieces of each operand
// (mfma_split.h); accumulation is fp32, results are rounded once.
//
// rows_kernel          Y and dX: a 128-row x 128-column tile per workgroup, four waves of 64 x 64; fp32, and 16-bit operands
//                      whose rows are not aligned to 16 bytes.  Operands go through registers (where fp32 is split).
// rows_direct_kernel   the same for aligned 16-bit operands, memory -> LDS directly: 256 x 256 (waves of 64 x 128) or
//                      128 x 128.
// wgrad_kernel,        dW and db: a 128 x 128 (256) tile of one group's dW; long groups are split over rows into items
// wgrad_direct_kernel  whose fp32 partial results a second launch adds in order (no atomics); a group of one item has
//                      none.  db is summed from the fragments of dY, alone where dW is not asked for.
// few_rows_kernel      Y for a handful of rows (serving): bound by reading the weights once; 16 output columns per
//                      workgroup, the reduction split over its four waves, operands straight from memory to registers.
//
// Measured on MI355X (a library product of 8192^3 reaches 1374 TFLOP/s in bf16, of 4096^3 137 in fp32):
//   bf16, 16 groups of 2048 rows, 1024 x 1024   Y 77 us (892 TFLOP/s), dX 87 - 92, dW and db 102 - 105, db alone 26;
//                                               ragged groups 98 - 106, 102 - 111, 110 - 117, 28
//                                               (one library product of all rows with one weight: 58)
//   bf16, one group of 32 768, 4096 -> 1024     Y 280 - 307 us, dX 325, dW and db 1180 (256 workgroups in all), db alone 27
//   bf16, 16 ragged groups, 1023 x 1023         Y 137 us, dX 176, dW and db 322, db alone 50 (rows not aligned)
//   fp32, 16 groups of 2048, 1024 x 1024        Y 365 - 390 us (180 TFLOP/s), dX 370, dW and db 455, db alone 28
//                                               (library: Y 482, dX 562)
//   fp32, 3 groups of 92 417 rows, 96 -> 512    Y 75 us, dX 80, dW and db 95, of them 11 to join, db alone 41; within a
//                                               training step 90, 78, 103 (library, one weight: Y 125)
//   8 rows over 16 groups, 1024 -> 2048         bf16 Y 9 us (27 MB of weights: 5 us at the rate of a copy), dX 28; fp32 15, 113
// What bounds the 16-bit products: loads into LDS and products overlap only in part.  Alone, with everything else taken out,
// products take 157 us and loads 196 of 280 (4096 -> 1024); three stages of 256 x 128 or 32-deep steps three ahead, which
// wait less but load more, are slower (364 and 350).  The 256 CUs hold 512 tiles of 256 x 256 in two rounds; a few more, as
// ragged groups make, cost most of a third.
#include <type_traits>

#include "common.h"
#include "mfma_split.h"

namespace {

using pv2::f32x16;
typedef unsigned short u16;
typedef u16 u16x4 __attribute__((ext_vector_type(4)));
typedef u16 u16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int kThreads = 256;
constexpr int kTile = 128;   // rows and columns of an output tile

// rows of any alignment: gfx950 loads and stores vectors at element alignment
struct __attribute__((packed, aligned(2))) Any16 { uint4 v; };
struct __attribute__((packed, aligned(2))) Any8 { uint2 v; };

template <typename H>
struct Half {
  typedef u16 E;
  typedef H Type;
  static constexpr int kPlanes = 1, kDepth = 64;   // depth: reduction steps staged at a time
  struct Raw { uint4 v; };                         // eight elements
  static __device__ __forceinline__ Raw zero() { return {make_uint4(0u, 0u, 0u, 0u)}; }
  static __device__ __forceinline__ Raw load(const E* p, int count) {
    if (count >= 8) return {reinterpret_cast<const Any16*>(p)->v};
    u16x8 t;
#pragma unroll
    for (int j = 0; j < 8; ++j) t[j] = j < count ? p[j] : (u16)0;
    return {__builtin_bit_cast(uint4, t)};
  }
  static __device__ __forceinline__ void stage(u16* lds, int, const Raw& r) { *reinterpret_cast<uint4*>(lds) = r.v; }
  static __device__ __forceinline__ f32x16 mfma(const u16x8* a, const u16x8* b, f32x16 c) { return H::mfma(a[0], b[0], c); }
  static __device__ __forceinline__ float sum(const u16x8& f) {
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) s += H::to_float(f[j]);
    return s;
  }
  static __device__ __forceinline__ float to_float(E v) { return H::to_float(v); }
  static __device__ __forceinline__ E from_float(float v) { return H::from_float(v); }
  static __device__ __forceinline__ void put4(E* lds, const float* v) {
    u16x4 t;
#pragma unroll
    for (int j = 0; j < 4; ++j) t[j] = H::from_float(v[j]);
    *reinterpret_cast<u16x4*>(lds) = t;
  }
  static __device__ __forceinline__ void store4(E* p, const float* v, int count) {
    if (count >= 4) {
      u16x4 t;
#pragma unroll
      for (int j = 0; j < 4; ++j) t[j] = H::from_float(v[j]);
      reinterpret_cast<Any8*>(p)->v = __builtin_bit_cast(uint2, t);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < count) p[j] = H::from_float(v[j]);
    }
  }
};

struct Bf {
  static __device__ __forceinline__ f32x16 mfma(u16x8 a, u16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4 mfma16(u16x8 a, u16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ float to_float(u16 v) { return __uint_as_float((unsigned)v << 16); }
  static __device__ __forceinline__ u16 from_float(float v) { return __builtin_bit_cast(u16, (__bf16)v); }
};

struct Hf {
  static __device__ __forceinline__ f32x16 mfma(u16x8 a, u16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4 mfma16(u16x8 a, u16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ float to_float(u16 v) { return (float)__builtin_bit_cast(_Float16, v); }
  static __device__ __forceinline__ u16 from_float(float v) { return __builtin_bit_cast(u16, (_Float16)v); }
};

struct Full {   // fp32: three bf16 planes in LDS
  typedef float E;
  static constexpr int kPlanes = 3, kDepth = 32;
  struct Raw { float4 lo, hi; };
  static __device__ __forceinline__ Raw zero() { return {make_float4(0, 0, 0, 0), make_float4(0, 0, 0, 0)}; }
  static __device__ __forceinline__ Raw load(const E* p, int count) {
    struct __attribute__((packed, aligned(4))) Any { float4 v; };
    if (count >= 8) return {reinterpret_cast<const Any*>(p)->v, reinterpret_cast<const Any*>(p + 4)->v};
    float t[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) t[j] = j < count ? p[j] : 0.f;
    return {make_float4(t[0], t[1], t[2], t[3]), make_float4(t[4], t[5], t[6], t[7])};
  }
  static __device__ __forceinline__ void stage(u16* lds, int plane, const Raw& r) {
    const pv2::Split8 s = pv2::split8(r.lo, r.hi);
#pragma unroll
    for (int i = 0; i < 3; ++i) *reinterpret_cast<uint4*>(lds + i * plane) = __builtin_bit_cast(uint4, s.p[i]);
  }
  static __device__ __forceinline__ f32x16 mfma(const u16x8* a, const u16x8* b, f32x16 c) {
#define PV2_TERM(i, j) c = Bf::mfma(a[i], b[j], c);
    PV2_SPLIT_TERMS(PV2_TERM)
#undef PV2_TERM
    return c;
  }
  static __device__ __forceinline__ float sum(const u16x8& f) { return Half<Bf>::sum(f); }
  static __device__ __forceinline__ float to_float(E v) { return v; }
  static __device__ __forceinline__ E from_float(float v) { return v; }
  static __device__ __forceinline__ void put4(E* lds, const float* v) {
    *reinterpret_cast<float4*>(lds) = make_float4(v[0], v[1], v[2], v[3]);
  }
  static __device__ __forceinline__ void store4(E* p, const float* v, int count) {
    struct __attribute__((packed, aligned(4))) Any { float4 v; };
    if (count >= 4) {
      reinterpret_cast<Any*>(p)->v = make_float4(v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < count) p[j] = v[j];
    }
  }
};

// ---- operand tiles in LDS, in 16-byte chunks of eight 16-bit elements; chunks are permuted within a row so that the
// rows that one read instruction touches lie in different banks
// "along": 128 rows, the reduction (kDepth) along the row
template <int DEPTH>
__device__ __forceinline__ int along_swizzle(int row) { return DEPTH == 64 ? ((row >> 1) & 7) : ((row >> 2) & 3); }
template <int DEPTH>
__device__ __forceinline__ u16x8 along_fragment(const u16* tile, int row, int chunk) {
  return *reinterpret_cast<const u16x8*>(tile + row * DEPTH + ((chunk ^ along_swizzle<DEPTH>(row)) << 3));
}
// "across": kDepth rows of the reduction, 128 columns along the row; read through the transposing LDS read: lane t of a
// 16-lane group points at row t / 4, columns 4 (t % 4) .. of a 4 x 16 block and receives column t of it
__device__ __forceinline__ int across_swizzle(int row) { return (row & 3) << 2; }
__device__ __forceinline__ u16x8 across_fragment(const u16* tile, int step, int block, int lane) {
  typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
  const int g = lane >> 4, t = lane & 15;
  const int row = step * 16 + 8 * (g >> 1) + (t >> 2);
  const int chunk = block * 4 + 2 * (g & 1) + ((t & 3) >> 1);
  const u16* p0 = tile + row * kTile + ((chunk ^ across_swizzle(row)) << 3) + 4 * (t & 1);
  const u16* p1 = tile + (row + 4) * kTile + ((chunk ^ across_swizzle(row + 4)) << 3) + 4 * (t & 1);
  const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p0);
  const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p1);
  u16x8 v;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    v[j] = (u16)lo[j];
    v[4 + j] = (u16)hi[j];
  }
  return v;
}

struct Item {
  int group;       // n_groups: the rows of no group; -1: no such item
  int first, last; // positions
  int number, of;  // which of the group's items this is
  int slab;        // of the items of groups that have more than one: which this is
};

// The item of workgroup `id` when every group's rows are cut into pieces of `unit` (`empty`: a group without rows has one
// item, and the rows of no group have none), and its tile of `tiles`.  By a whole wave.  Workgroups are dealt to the 8
// XCDs in turn; each XCD takes a contiguous eighth of the items, tile by tile, so that its L2 holds few groups' weights
// and an item's rows are read into one L2 only (items dealt in turn instead: 124 -> 100 us for 32768 rows, 16 groups,
// 1024 x 1024, bf16).
__device__ __forceinline__ Item find_item(const int32_t* __restrict__ offsets, int n_groups, int n_rows, int unit,
                                          bool empty, int id, int tiles, int* tile) {
  const int lane = threadIdx.x & 63;
  int from = 0, to = 0, count = 0, upto = 0;
  auto scan = [&](int g0) {   // counts of groups g0 .. g0 + 63 and their prefix sums
    const int g = g0 + lane;
    from = to = 0;
    if (g <= n_groups) {
      from = offsets[g];
      to = g < n_groups ? offsets[g + 1] : n_rows;
    }
    count = (to - from + unit - 1) / unit;
    if (empty) count = g < n_groups ? max(count, 1) : 0;
    upto = count;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int t = __shfl_up(upto, d);
      if (lane >= d) upto += t;
    }
    return __shfl(upto, 63);
  };
  int total = 0;
  for (int g0 = 0; g0 <= n_groups; g0 += 64) total += scan(g0);
  const int per_xcd = (total + 7) / 8, k = id / 8 / tiles;
  const int item = id % 8 * per_xcd + k;
  *tile = id / 8 % tiles;
  Item it = {-1, 0, 0, 0, 0, 0};
  if (k >= per_xcd || item >= total) return it;
  int run = 0, single = 0;   // items of the groups before; how many of those groups have one item only
  for (int g0 = 0; g0 <= n_groups; g0 += 64) {
    const int sum = n_groups < 64 ? total : scan(g0);   // (one round: it is there already)
    const uint64_t past = __ballot(run + upto > item), ones = __ballot(count == 1);
    if (past) {
      const int l = __ffsll((unsigned long long)past) - 1;
      it.of = __shfl(count, l);
      it.number = item - (run + __shfl(upto, l) - it.of);
      it.slab = item - single - __popcll(ones & ((1ull << l) - 1));
      it.group = g0 + l;
      const int f = __shfl(from, l), t = __shfl(to, l);
      // (a group's items of a weight gradient are about equal: whole steps of 32 rows, the last one may be empty)
      const int piece = empty ? ((t - f + it.of - 1) / it.of + 31) / 32 * 32 : unit;
      it.first = f + it.number * piece;
      it.last = min(t, it.first + piece);
      return it;
    }
    run += sum;
    single += __popcll(ones);
  }
  return it;
}

// An output tile leaves through LDS, so that rows are written in whole cache lines (an accumulator register holds one
// element of 32 different rows).  `buffer`: 64 rows of kOutRow elements, this wave's 64 columns (tile columns 64 wc ..) of
// its rows 32 b .. of each half: row 32 wr + i of the buffer is row 64 wr + 32 b + i of the tile.
template <typename E, int COLS = kTile>
constexpr int kOutRow = COLS + 16 / sizeof(E);
// the buffer's ROWS rows of COLS elements -> dst(row)[0 .. count), by the whole workgroup; dst: nullptr for no such row
template <int ROWS, int COLS, int THREADS = kThreads, typename E, typename Dst>
__device__ __forceinline__ void write_rows(const E* buffer, int count, Dst dst) {
  constexpr int N = 16 / sizeof(E), kPerRow = COLS / N;
#pragma unroll 4
  for (int q = threadIdx.x; q < ROWS * kPerRow; q += THREADS) {
    const int row = q / kPerRow, col = q % kPerRow * N;
    E* p = dst(row);
    if (p == nullptr || col >= count) continue;
    const E* src = buffer + row * kOutRow<E, COLS> + col;
    if (col + N <= count) {
      reinterpret_cast<Any16*>(p + col)->v = *reinterpret_cast<const uint4*>(src);
    } else {
      for (int j = 0; j < count - col; ++j) p[col + j] = src[j];
    }
  }
}

template <class P>
__device__ __forceinline__ float load_bias(const typename P::E* __restrict__ bias, int group, int n_groups, int col,
                                           int cols) {
  return bias && group < n_groups && col < cols ? P::to_float(bias[(int64_t)group * cols + col]) : 0.f;
}

// A tile's chunks, held by the workgroup's threads between memory and LDS
template <class P>
constexpr int kChunks = kTile * P::kDepth / 8 / kThreads;
// LDS of both operands' tiles or half an fp32 output tile, in 16-bit elements
template <class P>
constexpr int kLds = 2 * P::kPlanes * kTile * P::kDepth > 64 * kOutRow<float> * 2 ? 2 * P::kPlanes * kTile * P::kDepth
                                                                                  : 64 * kOutRow<float> * 2;

// Blocks of 32 columns that a wave computes when `left` columns remain: 96 columns are three of a tile's four.  Waves trade
// the halves of a tile from one workgroup of a CU to its next (256 CUs), so that no SIMD always has the shorter one.
__device__ __forceinline__ int blocks_of_32(int left) { return left <= 0 ? 0 : left <= 32 ? 1 : 2; }

// WACROSS: the weights' reduction runs across their rows (dX: W is [reduction, columns]) instead of along them (Y)
template <class P, bool WACROSS>
__global__ __launch_bounds__(kThreads, 3) void rows_kernel(
    const typename P::E* __restrict__ x, int64_t ldx, const typename P::E* __restrict__ w, int64_t w_group,
    int64_t ldw, const typename P::E* __restrict__ bias, const int32_t* __restrict__ order,
    const int32_t* __restrict__ offsets, int n_rows, int n_groups, int cols, int depth, int n_tiles,
    typename P::E* __restrict__ y) {
  typedef typename P::E E;
  constexpr int D = P::kDepth, PL = P::kPlanes, kPlane = kTile * D, U = kChunks<P>;
  __shared__ __attribute__((aligned(16))) u16 s_all[kLds<P>];
  u16 *s_w = s_all, *s_x = s_all + PL * kPlane;
  __shared__ int s_row[kTile];
  __shared__ __attribute__((aligned(16))) float s_bias[kTile];
  int tile;
  const Item it = find_item(offsets, n_groups, n_rows, kTile, false, blockIdx.x, n_tiles, &tile);
  if (it.group < 0) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int c0 = tile * kTile;
  if (tid < kTile) {
    const int p = it.first + tid;
    s_row[tid] = p < it.last ? (order ? order[p] : p) : -1;
    s_bias[tid] = load_bias<P>(bias, it.group, n_groups, c0 + tid, cols);
  }
  __syncthreads();
  if (it.group == n_groups) {   // rows of no group: zeros
    const float zero[4] = {0.f, 0.f, 0.f, 0.f};
    for (int q = tid; q < kTile * kTile / 4; q += kThreads) {
      const int r = s_row[q / (kTile / 4)], col = c0 + q % (kTile / 4) * 4;
      if (r >= 0 && col < cols) P::store4(y + (int64_t)r * cols + col, zero, cols - col);
    }
    return;
  }
  const E* wg = w + it.group * w_group;

  typename P::Raw rw[U], rx[U];
  const E* xp[U];
  int xc[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int q = tid + u * kThreads, row = q / (D / 8);
    const int r = s_row[row];
    xc[u] = r >= 0 ? ((q % (D / 8)) ^ along_swizzle<D>(row)) * 8 : -1;
    xp[u] = x + (int64_t)max(r, 0) * ldx + max(xc[u], 0);
  }
  auto load = [&](int k0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int q = tid + u * kThreads;
      const int left = depth - k0 - xc[u];
      rx[u] = xc[u] >= 0 && left > 0 ? P::load(xp[u] + k0, left) : P::zero();
      if (WACROSS) {
        const int row = q / (kTile / 8), k = k0 + row, col = c0 + ((q % (kTile / 8)) ^ across_swizzle(row)) * 8;
        rw[u] = k < depth && col < cols ? P::load(wg + (int64_t)k * ldw + col, cols - col) : P::zero();
      } else {
        const int row = q / (D / 8), col = c0 + row, k = k0 + ((q % (D / 8)) ^ along_swizzle<D>(row)) * 8;
        rw[u] = k < depth && col < cols ? P::load(wg + (int64_t)col * ldw + k, depth - k) : P::zero();
      }
    }
  };

  f32x16 acc[2][2];
#pragma unroll
  for (int a = 0; a < 2; ++a)
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int q = 0; q < 16; ++q) acc[a][b][q] = 0.f;
  const int i = lane & 31, h = lane >> 5;
  const int wc = (wave ^ (blockIdx.x >> 8)) & 1, wr = wave >> 1;   // the wave's 64 columns and rows
  const int blocks = blocks_of_32(cols - c0 - wc * 64);

  load(0);
  for (int k0 = 0; k0 < depth; k0 += D) {
    __syncthreads();
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int q = tid + u * kThreads;
      P::stage(s_x + q * 8, kPlane, rx[u]);
      P::stage(s_w + q * 8, kPlane, rw[u]);
    }
    __syncthreads();
    if (k0 + D < depth) load(k0 + D);
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
      u16x8 fw[2][PL], fx[2][PL];
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int p = 0; p < PL; ++p) fx[b][p] = along_fragment<D>(s_x + p * kPlane, wr * 64 + b * 32 + i, 2 * s + h);
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        if (a >= blocks) break;
#pragma unroll
        for (int p = 0; p < PL; ++p)
          fw[a][p] = WACROSS ? across_fragment(s_w + p * kPlane, s, wc * 2 + a, lane)
                             : along_fragment<D>(s_w + p * kPlane, wc * 64 + a * 32 + i, 2 * s + h);
#pragma unroll
        for (int b = 0; b < 2; ++b) acc[a][b] = P::mfma(fw[a], fx[b], acc[a][b]);
      }
    }
  }

  E* out = reinterpret_cast<E*>(s_all);
#pragma unroll
  for (int b = 0; b < 2; ++b) {
    __syncthreads();   // the operands, or the first half of the tile, have been read
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int col = wc * 64 + a * 32 + 8 * q + 4 * h;
        const float4 add = *reinterpret_cast<const float4*>(s_bias + col);
        const float v[4] = {acc[a][b][4 * q] + add.x, acc[a][b][4 * q + 1] + add.y, acc[a][b][4 * q + 2] + add.z,
                            acc[a][b][4 * q + 3] + add.w};
        P::put4(out + (wr * 32 + i) * kOutRow<E> + col, v);
      }
    __syncthreads();
    write_rows<64, kTile>(out, cols - c0, [&](int row) -> E* {
      const int r = s_row[(row >> 5) * 64 + b * 32 + (row & 31)];
      return r < 0 ? nullptr : y + (int64_t)r * cols + c0;
    });
  }
}

// dW[g][n][k] over one item's rows.  The item is the whole group: written in the weights' type; else fp32 partials.
// WEIGHTS false: db alone, x is not read (tiles_in is 1, items as for one column of x).
template <class P, bool WEIGHTS>
__global__ __launch_bounds__(kThreads, 3) void wgrad_kernel(
    const typename P::E* __restrict__ dy, int64_t ldy, const typename P::E* __restrict__ x, int64_t ldx,
    const int32_t* __restrict__ order, const int32_t* __restrict__ offsets, int n_rows, int n_groups, int n_out,
    int n_in, int unit, int tiles_out, int tiles_in, typename P::E* __restrict__ dw, typename P::E* __restrict__ db,
    float* __restrict__ dw_part, float* __restrict__ db_part) {
  typedef typename P::E E;
  constexpr int D = P::kDepth, PL = P::kPlanes, kPlane = kTile * D, U = kChunks<P>;
  __shared__ __attribute__((aligned(16))) u16 s_all[kLds<P>];
  u16 *s_x = s_all, *s_g = s_all + PL * kPlane;
  int tile;
  const Item it = find_item(offsets, n_groups, n_rows, unit, true, blockIdx.x, tiles_out * tiles_in, &tile);
  if (it.group < 0) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int n0 = tile / tiles_in * kTile, k0 = tile % tiles_in * kTile;
  const int i = lane & 31, h = lane >> 5;
  const int wk = (wave ^ (blockIdx.x >> 8)) & 1, wn = wave >> 1;
  const int blocks = blocks_of_32(n_in - k0 - wk * 64);
  const bool sum_bias = db != nullptr && k0 == 0 && wk == 0;

  typename P::Raw rx[U], rg[U];
  int row_of[U];
  auto load_rows = [&](int p0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int p = p0 + (tid + u * kThreads) / (kTile / 8);
      row_of[u] = p < it.last ? (order ? order[p] : p) : -1;
    }
  };
  auto load = [&]() {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int q = tid + u * kThreads, row = q / (kTile / 8);
      const int col = ((q % (kTile / 8)) ^ across_swizzle(row)) * 8;
      const int64_t r = row_of[u];
      if (WEIGHTS) rx[u] = r >= 0 && k0 + col < n_in ? P::load(x + r * ldx + k0 + col, n_in - k0 - col) : P::zero();
      rg[u] = r >= 0 && n0 + col < n_out ? P::load(dy + r * ldy + n0 + col, n_out - n0 - col) : P::zero();
    }
  };

  f32x16 acc[2][2];
  float bias_sum[2] = {0.f, 0.f};   // of this lane's column and its reduction steps
#pragma unroll
  for (int b = 0; b < 2; ++b)
#pragma unroll
    for (int q = 0; q < 16; ++q) acc[0][b][q] = acc[1][b][q] = 0.f;

  load_rows(it.first);
  load();
  load_rows(it.first + D);
  for (int p0 = it.first; p0 < it.last; p0 += D) {
    __syncthreads();
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int q = tid + u * kThreads;
      if (WEIGHTS) P::stage(s_x + q * 8, kPlane, rx[u]);
      P::stage(s_g + q * 8, kPlane, rg[u]);
    }
    __syncthreads();
    if (p0 + D < it.last) {
      load();
      load_rows(p0 + 2 * D);
    }
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
      u16x8 fx[2][PL], fg[2][PL];
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int p = 0; p < PL; ++p) fg[b][p] = across_fragment(s_g + p * kPlane, s, wn * 2 + b, lane);
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        if (!WEIGHTS || a >= blocks) break;
#pragma unroll
        for (int p = 0; p < PL; ++p) fx[a][p] = across_fragment(s_x + p * kPlane, s, wk * 2 + a, lane);
#pragma unroll
        for (int b = 0; b < 2; ++b) acc[a][b] = P::mfma(fx[a], fg[b], acc[a][b]);
      }
      if (sum_bias) {
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int p = PL - 1; p >= 0; --p) bias_sum[b] += P::sum(fg[b][p]);
      }
    }
  }

  const bool whole = it.of == 1;
  auto leave = [&](auto* out, auto* base) {
    typedef std::remove_pointer_t<decltype(out)> O;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      __syncthreads();
#pragma unroll
      for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float v[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j] = acc[a][b][4 * q + j];
          O* at = out + (wn * 32 + i) * kOutRow<O> + wk * 64 + a * 32 + 8 * q + 4 * h;
          if constexpr (sizeof(O) == 4) Full::put4(at, v);
          else P::put4(at, v);
        }
      __syncthreads();
      write_rows<64, kTile>(out, n_in - k0, [&](int row) -> O* {
        const int n = n0 + (row >> 5) * 64 + b * 32 + (row & 31);
        return n < n_out ? base + (int64_t)n * n_in + k0 : nullptr;
      });
    }
  };
  const int64_t size = (int64_t)n_out * n_in;
  if (!WEIGHTS) {}
  else if (whole) leave(reinterpret_cast<E*>(s_all), dw + it.group * size);
  else leave(reinterpret_cast<float*>(s_all), dw_part + it.slab * size);
  if (sum_bias) {
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const float sum = bias_sum[b] + __shfl_xor(bias_sum[b], 32);
      const int n = n0 + wn * 64 + b * 32 + i;
      if (h != 0 || n >= n_out) continue;
      if (whole) db[(int64_t)it.group * n_out + n] = P::from_float(sum);
      else db_part[(int64_t)it.slab * n_out + n] = sum;
    }
  }
}

// ---- 16-bit operands whose rows are aligned to 16 bytes: memory -> LDS without registers in between.  Steps of 32 go
// through three LDS buffers, two steps ahead of the products; a wave waits for its own loads of the next step (vmcnt
// counts them) and for its reads of this one before the barrier that ends the step.  A chunk that is not there (a row
// past the group, a column past the matrix, a step past the end) comes from a page of zeros, so that every step has the
// same loads.
constexpr int kStep = 32, kBuffers = 3;   // of the weight gradient
__device__ uint4 g_zeros[4];   // never written

template <int N>
__device__ __forceinline__ void wait_for_loads() {   // all but the last N; and for all LDS reads
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0070 | (N & 15) | ((N >> 4) << 14));
  asm volatile("" ::: "memory");
}
__device__ __forceinline__ void barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
// 16 bytes per lane: the wave's 1 KB of LDS at `lds` (the same for all lanes), lane by lane
__device__ __forceinline__ void load_to_lds(const u16* p, u16* lds) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) unsigned*)p,
                                   (__attribute__((address_space(3))) unsigned*)lds, 16, 0, 0);
}

// a lane's place in the chunks of an "along" / "across" tile of 32 reduction steps and its fragments
constexpr int kDeep = 64;   // reduction steps of the row products' tiles
__device__ __forceinline__ int along_row(int q) { return q / (kDeep / 8); }
__device__ __forceinline__ int along_chunk(int q) { return (q % (kDeep / 8)) ^ along_swizzle<kDeep>(q / (kDeep / 8)); }
template <int COLS>
__device__ __forceinline__ int across_row(int q) { return q / (COLS / 8); }
template <int COLS>
__device__ __forceinline__ int across_chunk(int q) { return (q % (COLS / 8)) ^ across_swizzle(q / (COLS / 8)); }

// Fragments are read in assembly: for its own LDS reads the compiler would wait for every load into LDS, those two steps
// ahead as well.  Each block waits for its reads itself.
typedef u16 u16x4v __attribute__((ext_vector_type(4)));
__device__ __forceinline__ unsigned lds_address(const void* p) {
  return (unsigned)(uintptr_t)(__attribute__((address_space(3))) const void*)p;
}
__device__ __forceinline__ u16x8 glue(u16x4v lo, u16x4v hi) { return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7); }

// an "along" tile: N blocks of 32 rows, 4 KB apart
template <int N>
__device__ __forceinline__ void read_along(unsigned at, u16x8* f) {
  static_assert(N == 2, "");
  asm volatile("ds_read_b128 %0, %2\n\tds_read_b128 %1, %2 offset:4096\n\ts_waitcnt lgkmcnt(0)"
               : "=&v"(f[0]), "=&v"(f[1])
               : "v"(at)
               : "memory");
}
// an "along" tile's two blocks together with N of another
template <int N>
__device__ __forceinline__ void read_along2(unsigned at, unsigned at2, u16x8* f, u16x8* f2) {
  static_assert(N == 2 || N == 4, "");
  if constexpr (N == 2)
    asm volatile("ds_read_b128 %0, %4\n\tds_read_b128 %2, %5\n\tds_read_b128 %1, %4 offset:4096\n\t"
                 "ds_read_b128 %3, %5 offset:4096\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(f[0]), "=&v"(f[1]), "=&v"(f2[0]), "=&v"(f2[1])
                 : "v"(at), "v"(at2)
                 : "memory");
  else
    asm volatile("ds_read_b128 %0, %6\n\tds_read_b128 %1, %6 offset:4096\n\tds_read_b128 %2, %7\n\t"
                 "ds_read_b128 %3, %7 offset:4096\n\tds_read_b128 %4, %7 offset:8192\n\t"
                 "ds_read_b128 %5, %7 offset:12288\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(f[0]), "=&v"(f[1]), "=&v"(f2[0]), "=&v"(f2[1]), "=&v"(f2[2]), "=&v"(f2[3])
                 : "v"(at), "v"(at2)
                 : "memory");
}
// N blocks of 32 columns of an "across" tile with rows of ROW bytes: two transposing reads each, four rows apart
template <int N, int OFF, int ROW>
__device__ __forceinline__ void read_across(const unsigned* at, u16x8* f) {
  u16x4v a[N], b[N];
  if constexpr (N == 2)
    asm volatile("ds_read_b64_tr_b16 %0, %4 offset:%6\n\tds_read_b64_tr_b16 %2, %4 offset:%7\n\t"
                 "ds_read_b64_tr_b16 %1, %5 offset:%6\n\tds_read_b64_tr_b16 %3, %5 offset:%7\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(a[0]), "=&v"(a[1]), "=&v"(b[0]), "=&v"(b[1])
                 : "v"(at[0]), "v"(at[1]), "n"(OFF), "n"(OFF + 4 * ROW)
                 : "memory");
  else
    asm volatile("ds_read_b64_tr_b16 %0, %8 offset:%12\n\tds_read_b64_tr_b16 %4, %8 offset:%13\n\t"
                 "ds_read_b64_tr_b16 %1, %9 offset:%12\n\tds_read_b64_tr_b16 %5, %9 offset:%13\n\t"
                 "ds_read_b64_tr_b16 %2, %10 offset:%12\n\tds_read_b64_tr_b16 %6, %10 offset:%13\n\t"
                 "ds_read_b64_tr_b16 %3, %11 offset:%12\n\tds_read_b64_tr_b16 %7, %11 offset:%13\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(a[0]), "=&v"(a[1]), "=&v"(a[2]), "=&v"(a[3]), "=&v"(b[0]), "=&v"(b[1]), "=&v"(b[2]), "=&v"(b[3])
                 : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "n"(OFF), "n"(OFF + 4 * ROW)
                 : "memory");
#pragma unroll
  for (int n = 0; n < N; ++n) f[n] = glue(a[n], b[n]);
}
// where a lane reads: block `block` of a tile (first step)
__device__ __forceinline__ unsigned along_at(const u16* tile, int row, int chunk) {
  return lds_address(tile + row * kDeep + ((chunk ^ along_swizzle<kDeep>(row)) << 3));
}
template <int COLS>
__device__ __forceinline__ unsigned across_at(const u16* tile, int block, int lane) {
  const int g = lane >> 4, t = lane & 15;
  const int row = 8 * (g >> 1) + (t >> 2);   // (row + 4 and row + 16 have the same swizzle)
  const int chunk = (block * 4 + 2 * (g & 1) + ((t & 3) >> 1)) ^ across_swizzle(row);
  return lds_address(tile + row * COLS + (chunk << 3) + 4 * (t & 1));
}

// ROWS x COLS outputs per workgroup of ROWS / 32 waves, each with 64 rows and half of the columns
template <class H, bool WACROSS, int ROWS, int COLS>
__global__ __launch_bounds__(2 * ROWS, 2) void rows_direct_kernel(
    const u16* __restrict__ x, int64_t ldx, const u16* __restrict__ w, int64_t w_group, int64_t ldw,
    const u16* __restrict__ bias, const int32_t* __restrict__ order, const int32_t* __restrict__ offsets, int n_rows,
    int n_groups, int cols, int depth, int n_tiles, u16* __restrict__ y) {
  typedef Half<H> P;
  constexpr int T = 2 * ROWS, A = COLS / 64, UX = ROWS * kDeep / 8 / T, UW = COLS * kDeep / 8 / T;
  constexpr int kBuffer = (ROWS + COLS) * kDeep;
  constexpr int kOut = ROWS * kOutRow<u16, COLS>;
  __shared__ __attribute__((aligned(1024))) u16 s_all[2 * kBuffer > kOut ? 2 * kBuffer : kOut];   // (addresses are XORed)
  __shared__ int s_row[ROWS];
  __shared__ __attribute__((aligned(16))) float s_bias[COLS];
  int tile;
  const Item it = find_item(offsets, n_groups, n_rows, ROWS, false, blockIdx.x, n_tiles, &tile);
  if (it.group < 0) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c0 = tile * COLS;
  if (tid < ROWS) {
    const int p = it.first + tid;
    s_row[tid] = p < it.last ? (order ? order[p] : p) : -1;
  }
  if (tid < COLS) s_bias[tid] = load_bias<P>(bias, it.group, n_groups, c0 + tid, cols);
  __syncthreads();
  if (it.group == n_groups) {   // rows of no group: zeros
    const float zero[4] = {0.f, 0.f, 0.f, 0.f};
    for (int q = tid; q < ROWS * COLS / 4; q += T) {
      const int r = s_row[q / (COLS / 4)], col = c0 + q % (COLS / 4) * 4;
      if (r >= 0 && col < cols) P::store4(y + (int64_t)r * cols + col, zero, cols - col);
    }
    return;
  }
  // This thread's chunks of a step, as bytes from the operands' beginnings: those move on by themselves, and a load takes no
  // arithmetic.  A row past the group repeats the tile's first one and a column past the matrix the last one: what they
  // give is not written.
  unsigned xo[UX], wo[UW];
#pragma unroll
  for (int u = 0; u < UX; ++u) {
    const int q = tid + u * T, r = s_row[along_row(q)];
    xo[u] = (unsigned)(((int64_t)(r >= 0 ? r : s_row[0]) * ldx + along_chunk(q) * 8) * 2);
  }
#pragma unroll
  for (int u = 0; u < UW; ++u) {
    const int q = tid + u * T;
    wo[u] = (unsigned)((WACROSS ? across_row<COLS>(q) * ldw + min(c0 + across_chunk<COLS>(q) * 8, cols - 8)
                                : min(c0 + along_row(q), cols - 1) * ldw + along_chunk(q) * 8) * 2);
  }
  const char *xk = reinterpret_cast<const char*>(x), *wk = reinterpret_cast<const char*>(w + it.group * w_group);
  const int64_t w_add = (WACROSS ? kDeep * ldw : kDeep) * 2;
  int left = depth;   // reduction steps that are not loaded yet
  // chunks FROM .. TO - 1 of the next step: x's, then the weights'
  auto issue = [&](u16* to, auto from, auto until) {
    to += wave * 64 * 8;
    if (left >= kDeep) {
#pragma unroll
      for (int u = decltype(from)::value; u < decltype(until)::value; ++u)
        load_to_lds((const u16*)(u < UX ? xk + xo[u < UX ? u : 0] : wk + wo[u < UX ? 0 : u - UX]), to + u * T * 8);
    } else {   // the last, shorter step: zeros past the end
      const u16* zeros = reinterpret_cast<const u16*>(g_zeros);
#pragma unroll
      for (int u = decltype(from)::value; u < decltype(until)::value; ++u) {
        const int q = tid + (u < UX ? u : u - UX) * T;
        const int k = u >= UX && WACROSS ? across_row<COLS>(q) : along_chunk(q) * 8;
        load_to_lds(k < left ? (const u16*)(u < UX ? xk + xo[u < UX ? u : 0] : wk + wo[u < UX ? 0 : u - UX]) : zeros,
                    to + u * T * 8);
      }
    }
  };
  auto move_on = [&]() {
    left -= kDeep;
    xk += kDeep * 2;
    wk += w_add;
  };
  static_assert(UX * T * 8 == ROWS * kDeep && UX + UW == 8, "");
  using std::integral_constant;

  f32x16 acc[A][2];
#pragma unroll
  for (int a = 0; a < A; ++a)
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int q = 0; q < 16; ++q) acc[a][b][q] = 0.f;
  const int i = lane & 31, h = lane >> 5;
  const int wc = wave & 1, wr = wave >> 1;
  const bool busy = wr * 64 < it.last - it.first;   // (the last tile of a group: no products for rows that are not there)
  unsigned x_at = along_at(s_all, wr * 64 + i, h);
  unsigned w_at = WACROSS ? across_at<COLS>(s_all + ROWS * kDeep, wc * A, lane)
                          : along_at(s_all + ROWS * kDeep, wc * A * 32 + i, h);
  int other = kBuffer;   // where the buffer that is not read now begins, from the one that is
  u16* next = s_all;
  issue(next, integral_constant<int, 0>(), integral_constant<int, 8>());
  move_on();
  wait_for_loads<0>();
  barrier();
  for (int k0 = 0; k0 < depth; k0 += kDeep) {
    next += other;
    auto quarter = [&](auto part) {
      constexpr int s = decltype(part)::value;
      // the loads of the next step go out in threes: a wave that issues all eight first starts its products late
      constexpr int kFrom = s * 3 < 8 ? s * 3 : 8, kUntil = s * 3 + 3 < 8 ? s * 3 + 3 : 8;
      if (left > 0) issue(next, integral_constant<int, kFrom>(), integral_constant<int, kUntil>());
      if (!busy) return;
      u16x8 fw[A], fx[2];
      if constexpr (WACROSS) {
        unsigned at[A];
#pragma unroll
        for (int a = 0; a < A; ++a) at[a] = w_at ^ (a << 6);   // (block a: four chunks on)
        read_along<2>(x_at ^ (s << 5), fx);
        read_across<A, s * 16 * COLS * 2, COLS * 2>(at, fw);
      } else {
        read_along2<A>(x_at ^ (s << 5), w_at ^ (s << 5), fx, fw);
      }
#pragma unroll
      for (int a = 0; a < A; ++a)
#pragma unroll
        for (int b = 0; b < 2; ++b) acc[a][b] = H::mfma(fw[a], fx[b], acc[a][b]);
    };
    quarter(std::integral_constant<int, 0>());
    quarter(std::integral_constant<int, 1>());
    quarter(std::integral_constant<int, 2>());
    quarter(std::integral_constant<int, 3>());
    move_on();
    x_at += other * 2;
    w_at += other * 2;
    other = -other;
    wait_for_loads<0>();
    barrier();
  }

#pragma unroll
  for (int b = 0; b < 2; ++b)
#pragma unroll
    for (int a = 0; a < A; ++a)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int col = (wc * A + a) * 32 + 8 * q + 4 * h;
        const float4 add = *reinterpret_cast<const float4*>(s_bias + col);
        const float v[4] = {acc[a][b][4 * q] + add.x, acc[a][b][4 * q + 1] + add.y, acc[a][b][4 * q + 2] + add.z,
                            acc[a][b][4 * q + 3] + add.w};
        P::put4(s_all + (wr * 64 + b * 32 + i) * kOutRow<u16, COLS> + col, v);
      }
  __syncthreads();
  write_rows<ROWS, COLS, T>(s_all, cols - c0, [&](int row) -> u16* {
    const int r = s_row[row];
    return r < 0 ? nullptr : y + (int64_t)r * cols + c0;
  });
}

// dW of one item as wgrad_kernel: 128 rows n x COLS columns k; the item's row numbers pass through LDS, kSegment at a time
constexpr int kSegment = 60 * kStep;
template <class H, int COLS>
__global__ __launch_bounds__(kThreads, 2) void wgrad_direct_kernel(
    const u16* __restrict__ dy, int64_t ldy, const u16* __restrict__ x, int64_t ldx, const int32_t* __restrict__ order,
    const int32_t* __restrict__ offsets, int n_rows, int n_groups, int n_out, int n_in, int unit, int tiles_out,
    int tiles_in, u16* __restrict__ dw, u16* __restrict__ db, float* __restrict__ dw_part,
    float* __restrict__ db_part) {
  typedef Half<H> P;
  constexpr int A = COLS / 64, UG = kTile * kStep / 8 / kThreads, UX = COLS * kStep / 8 / kThreads;
  constexpr int kBuffer = (kTile + COLS) * kStep;
  constexpr int kOut = 64 * kOutRow<float, COLS> * 2;
  __shared__ __attribute__((aligned(16))) u16 s_all[kBuffers * kBuffer > kOut ? kBuffers * kBuffer : kOut];
  __shared__ int s_row[kSegment];
  int tile;
  const Item it = find_item(offsets, n_groups, n_rows, unit, true, blockIdx.x, tiles_out * tiles_in, &tile);
  if (it.group < 0) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n0 = tile / tiles_in * kTile, k0 = tile % tiles_in * COLS;
  const int i = lane & 31, h = lane >> 5;
  const int wk = wave & 1, wn = wave >> 1;
  const bool sum_bias = db != nullptr && k0 == 0 && wk == 0;
  const u16* zeros = reinterpret_cast<const u16*>(g_zeros);

  const int gcol = n0 + across_chunk<kTile>(tid) * 8, xcol = k0 + across_chunk<COLS>(tid) * 8;
  static_assert(kThreads / (kTile / 8) % 4 == 0 && kThreads / (COLS / 8) % 4 == 0, "the same swizzle for all chunks");
  int segment_rows = 0, at = 0;   // rows of this segment and position of the next step in it
  // the row numbers of the next step's chunks, read a step ahead (positions past the segment: any, not used)
  int g_row[UG], x_row[UX];
  auto next_rows = [&]() {
    const int last = kSegment - kStep;
    const unsigned from = lds_address(s_row + min(at, last));
    const unsigned ga = from + across_row<kTile>(tid) * 4, xa = from + across_row<COLS>(tid) * 4;
    constexpr int G = kThreads / (kTile / 8) * 4, X = kThreads / (COLS / 8) * 4;
    if constexpr (UX == 4)
      asm volatile("ds_read_b32 %0, %6\n\tds_read_b32 %1, %6 offset:%8\n\tds_read_b32 %2, %7\n\tds_read_b32 %3, %7 offset:%9\n\t"
                   "ds_read_b32 %4, %7 offset:%10\n\tds_read_b32 %5, %7 offset:%11\n\ts_waitcnt lgkmcnt(0)"
                   : "=&v"(g_row[0]), "=&v"(g_row[1]), "=&v"(x_row[0]), "=&v"(x_row[1]), "=&v"(x_row[2]), "=&v"(x_row[3])
                   : "v"(ga), "v"(xa), "n"(G), "n"(X), "n"(2 * X), "n"(3 * X)
                   : "memory");
    else
      asm volatile("ds_read_b32 %0, %4\n\tds_read_b32 %1, %4 offset:%6\n\tds_read_b32 %2, %5\n\tds_read_b32 %3, %5 offset:%7\n\t"
                   "s_waitcnt lgkmcnt(0)"
                   : "=&v"(g_row[0]), "=&v"(g_row[1]), "=&v"(x_row[0]), "=&v"(x_row[1])
                   : "v"(ga), "v"(xa), "n"(G), "n"(X)
                   : "memory");
  };
  auto issue = [&](int buffer) {
    u16* to = s_all + buffer * kBuffer + wave * 64 * 8;
#pragma unroll
    for (int u = 0; u < UG; ++u) {
      const bool ok = at + across_row<kTile>(tid + u * kThreads) < segment_rows && gcol < n_out;
      load_to_lds(ok ? dy + (int64_t)g_row[u] * ldy + gcol : zeros, to + u * kThreads * 8);
    }
#pragma unroll
    for (int u = 0; u < UX; ++u) {
      const bool ok = at + across_row<COLS>(tid + u * kThreads) < segment_rows && xcol < n_in;
      load_to_lds(ok ? x + (int64_t)x_row[u] * ldx + xcol : zeros, to + kTile * kStep + u * kThreads * 8);
    }
    at += kStep;
    next_rows();
  };

  f32x16 acc[A][2];
  float bias_sum[2] = {0.f, 0.f};
#pragma unroll
  for (int b = 0; b < 2; ++b)
#pragma unroll
    for (int q = 0; q < 16; ++q)
#pragma unroll
      for (int a = 0; a < A; ++a) acc[a][b][q] = 0.f;
  unsigned g_at[2], x_at[A];
#pragma unroll
  for (int b = 0; b < 2; ++b) g_at[b] = across_at<kTile>(s_all, wn * 2 + b, lane);
#pragma unroll
  for (int a = 0; a < A; ++a) x_at[a] = across_at<COLS>(s_all + kTile * kStep, wk * A + a, lane);
  auto step = [&](auto buffer, int next) {
    constexpr int kAt = decltype(buffer)::value * kBuffer * 2;
    u16x8 fx[A], fg[2];
    auto products = [&]() {
#pragma unroll
      for (int a = 0; a < A; ++a)
#pragma unroll
        for (int b = 0; b < 2; ++b) acc[a][b] = H::mfma(fx[a], fg[b], acc[a][b]);
      if (sum_bias) {
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          bias_sum[b] += P::sum(fg[b]);
          asm volatile("" : "+v"(bias_sum[b]));   // (summed now: the compiler would keep the fragments for later)
        }
      }
    };
    issue(next);
    read_across<2, kAt, kTile * 2>(g_at, fg);
    read_across<A, kAt, COLS * 2>(x_at, fx);
    products();
    read_across<2, kAt + 16 * kTile * 2, kTile * 2>(g_at, fg);
    read_across<A, kAt + 16 * COLS * 2, COLS * 2>(x_at, fx);
    products();
    wait_for_loads<UG + UX>();
    barrier();
  };
  for (int first = it.first; first < it.last; first += kSegment) {
    segment_rows = min(kSegment, it.last - first);
    at = 0;
    for (int p = tid; p < segment_rows; p += kThreads) s_row[p] = order ? order[first + p] : first + p;
    __syncthreads();
    next_rows();
    issue(0);
    issue(1);
    wait_for_loads<UG + UX>();
    barrier();
    for (int done = 0;; ) {
      step(std::integral_constant<int, 0>(), 2);
      if ((done += kStep) >= segment_rows) break;
      step(std::integral_constant<int, 1>(), 0);
      if ((done += kStep) >= segment_rows) break;
      step(std::integral_constant<int, 2>(), 1);
      if ((done += kStep) >= segment_rows) break;
    }
    wait_for_loads<0>();
    barrier();
  }

  const bool whole = it.of == 1;
  auto leave = [&](auto* out, auto* base) {
    typedef std::remove_pointer_t<decltype(out)> O;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      __syncthreads();
#pragma unroll
      for (int a = 0; a < A; ++a)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float v[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j] = acc[a][b][4 * q + j];
          O* to = out + (wn * 32 + i) * kOutRow<O, COLS> + (wk * A + a) * 32 + 8 * q + 4 * h;
          if constexpr (sizeof(O) == 4) Full::put4(to, v);
          else P::put4(to, v);
        }
      __syncthreads();
      write_rows<64, COLS>(out, n_in - k0, [&](int row) -> O* {
        const int n = n0 + (row >> 5) * 64 + b * 32 + (row & 31);
        return n < n_out ? base + (int64_t)n * n_in + k0 : nullptr;
      });
    }
  };
  const int64_t size = (int64_t)n_out * n_in;
  if (whole) leave(s_all, dw + it.group * size);
  else leave(reinterpret_cast<float*>(s_all), dw_part + it.slab * size);
  if (sum_bias) {
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const float sum = bias_sum[b] + __shfl_xor(bias_sum[b], 32);
      const int n = n0 + wn * 64 + b * 32 + i;
      if (h != 0 || n >= n_out) continue;
      if (whole) db[(int64_t)it.group * n_out + n] = H::from_float(sum);
      else db_part[(int64_t)it.slab * n_out + n] = sum;
    }
  }
}

// the groups of more than one item: the sum of their partial results, in order; elements 0 .. size - 1 are dW's, the
// next n_out are db's
template <class P>
__global__ __launch_bounds__(kThreads) void join_kernel(const int32_t* __restrict__ offsets, int n_rows, int n_groups,
                                                        int unit, int64_t size, int n_out, int chunks,
                                                        const float* __restrict__ dw_part,
                                                        const float* __restrict__ db_part,
                                                        typename P::E* __restrict__ dw,
                                                        typename P::E* __restrict__ db) {
  const int64_t id = blockIdx.x;
  const int g = (int)(id / chunks);
  const int from = offsets[g], to = offsets[g + 1];
  const int count = (to - from + unit - 1) / unit;
  if (count <= 1) return;
  // the group's first partial result: all items of the groups before it that have more than one
  __shared__ int s_base[kThreads / 64];
  int base = 0;
  for (int f = threadIdx.x; f < g; f += kThreads) {
    const int items = (offsets[f + 1] - offsets[f] + unit - 1) / unit;
    base += items > 1 ? items : 0;
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) base += __shfl_xor(base, d);
  if ((threadIdx.x & 63) == 0) s_base[threadIdx.x >> 6] = base;
  __syncthreads();
  base = s_base[0] + s_base[1] + s_base[2] + s_base[3];
  const int64_t total = size + (db ? n_out : 0);
  for (int64_t e = (id % chunks) * kThreads + threadIdx.x; e < total; e += (int64_t)chunks * kThreads) {
    const bool of_w = e < size;
    const float* src = of_w ? dw_part + (int64_t)base * size + e : db_part + (int64_t)base * n_out + (e - size);
    const int64_t step = of_w ? size : n_out;
    float sum = 0.f;
#pragma unroll 8
    for (int c = 0; c < count; ++c) sum += src[c * step];
    if (of_w) dw[(int64_t)g * size + e] = P::from_float(sum);
    else db[(int64_t)g * n_out + (e - size)] = P::from_float(sum);
  }
}

// ---- a handful of rows: 16 columns x 16 rows per workgroup
template <class P>
struct Few;
template <typename H>
struct Few<Half<H>> {
  static constexpr int kStep = 32, kVec = 8;   // reduction steps per round and per lane
  static __device__ __forceinline__ f32x4 mfma(const uint4& a, const uint4& b, f32x4 c) {
    return H::mfma16(__builtin_bit_cast(u16x8, a), __builtin_bit_cast(u16x8, b), c);
  }
};
template <>
struct Few<Full> {   // v_mfma_f32_16x16x4_f32: lane group h holds step h, the same 4 h + j for both operands
  static constexpr int kStep = 16, kVec = 4;
  static __device__ __forceinline__ f32x4 mfma(const uint4& a, const uint4& b, f32x4 c) {
    const f32x4 fa = __builtin_bit_cast(f32x4, a), fb = __builtin_bit_cast(f32x4, b);
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(fa[j], fb[j], c, 0, 0, 0);
    return c;
  }
};

// 16 bytes at p, the elements past `count` zero
template <typename E>
__device__ __forceinline__ uint4 load16(const E* p, int count) {
  constexpr int N = 16 / sizeof(E);
  if (count >= N) return reinterpret_cast<const Any16*>(p)->v;
  typedef E V __attribute__((ext_vector_type(N)));
  V t;
#pragma unroll
  for (int j = 0; j < N; ++j) t[j] = j < count ? p[j] : (E)0;
  return __builtin_bit_cast(uint4, t);
}

template <class P>
__global__ __launch_bounds__(kThreads) void few_rows_kernel(
    const typename P::E* __restrict__ x, int64_t ldx, const typename P::E* __restrict__ w, int64_t w_group,
    int64_t ldw, const typename P::E* __restrict__ bias, const int32_t* __restrict__ order,
    const int32_t* __restrict__ offsets, int n_rows, int n_groups, int cols, int depth, int n_tiles,
    typename P::E* __restrict__ y) {
  typedef typename P::E E;
  typedef Few<P> F;
  constexpr int U = 4;
  __shared__ f32x4 s_part[kThreads / 64][64];
  int tile;
  const Item it = find_item(offsets, n_groups, n_rows, 16, false, blockIdx.x, n_tiles, &tile);
  if (it.group < 0) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int i = lane & 15, h = lane >> 4;
  const int c0 = tile * 16;
  const int p = it.first + i;
  const int r = p < it.last ? (order ? order[p] : p) : -1;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  if (it.group < n_groups) {
    const int wcol = c0 + i;
    const E* wp = w + it.group * w_group + (int64_t)(wcol < cols ? wcol : 0) * ldw;
    const E* xp = x + (int64_t)max(r, 0) * ldx;
    const int span = U * F::kStep;
    for (int k0 = wave * span; k0 < depth; k0 += span * (kThreads / 64)) {
      uint4 a[U], b[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int k = k0 + u * F::kStep + h * F::kVec, left = depth - k;
        a[u] = wcol < cols && left > 0 ? load16(wp + k, left) : make_uint4(0u, 0u, 0u, 0u);
        b[u] = r >= 0 && left > 0 ? load16(xp + k, left) : make_uint4(0u, 0u, 0u, 0u);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) acc = F::mfma(a[u], b[u], acc);
    }
  }
  s_part[wave][lane] = acc;
  __syncthreads();
  if (wave == 0) {
#pragma unroll
    for (int v = 1; v < kThreads / 64; ++v) acc += s_part[v][lane];
    const int col = c0 + 4 * h;
    if (r >= 0 && col < cols) {
      float v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[j] = acc[j];
        if (bias && it.group < n_groups && col + j < cols)
          v[j] += P::to_float(bias[(int64_t)it.group * cols + col + j]);
      }
      P::store4(y + (int64_t)r * cols + col, v, cols - col);
    }
  }
}

typedef Half<Bf> PBf;
typedef Half<Hf> PHf;

int tiles_of(int64_t n, int tile) { return (int)((n + tile - 1) / tile); }

// the most items that `rows` rows in `groups` groups and the rows of no group can make
int64_t most_items(int64_t rows, int64_t groups, int unit) {
  return rows / unit + (rows < groups + 1 ? rows : groups + 1);
}

constexpr int64_t kMostBlocks = 1 << 24;   // of 256 threads: a grid has fewer than 2^32

// Serving: so few items of 16 rows that reading the weights is what takes the time.  Measured with 1024 x 1024 bf16 weights,
// this kernel against tiles: 16 groups, 8 rows 6 us against 15, 128 rows 10 against 17, 256 rows 13 against 17; one group,
// 64 rows 7 against 15; 64 groups, 64 rows 20 against 22, 256 rows (80 items) 27 against 24, 512 rows 29 against 24.
bool few_rows(int64_t rows, int64_t groups) {
  return rows <= 256 && rows / 16 + (rows < groups ? rows : groups) <= 72;
}

bool aligned16(const void* p, int64_t a, int64_t b, int elem) {
  return (uintptr_t)p % 16 == 0 && a * elem % 16 == 0 && b * elem % 16 == 0;
}

// Columns of a weight gradient's 16-bit tile: 256 where that pads no more than 128 would (32768 rows, 16 groups, 1024 x
// 1024: 95 us against 114 with 128; 131072, 8, 256 x 256: 55 against 58; 32768, 1, 512 -> 2048: 130 against 202).
int wgrad_cols(int n_in) { return tiles_of(n_in, 128) % 2 ? 128 : 256; }

// Tiles of 256 x 256 (bf16, 32768 rows, 16 groups, 1024 x 1024: 75 us against 90 with 128 x 128) where they fill the 256
// CUs and pad no columns; else 128 x 128 (8192 rows: 26 us against 34).
bool large_tiles(int64_t rows, int cols) {
  return tiles_of(cols, 128) % 2 == 0 && rows / 256 * tiles_of(cols, 256) >= 256;
}

template <class P, bool WACROSS>
int launch_rows(const void* x, int64_t ldx, const void* w, int64_t w_group, int64_t ldw, const void* bias,
                const int32_t* order, const int32_t* offsets, int64_t rows, int64_t groups, int cols, int depth,
                void* y, hipStream_t s) {
  typedef typename P::E E;
  const int few_tiles = tiles_of(cols, 16);
  const int64_t few_blocks = (most_items(rows, groups, 16) + 7) / 8 * 8 * few_tiles;
  if (!WACROSS && few_rows(rows, groups) && few_blocks < kMostBlocks) {
    hipLaunchKernelGGL((few_rows_kernel<P>), dim3((unsigned)few_blocks), dim3(kThreads), 0, s, (const E*)x, ldx,
                       (const E*)w, w_group, ldw, (const E*)bias, order, offsets, (int)rows, (int)groups, cols, depth,
                       few_tiles, (E*)y);
    return pv2::check_launch("grouped_linear");
  }
  // 16-byte aligned rows; operands whose bytes 32 bits count
  const bool direct = sizeof(E) == 2 && aligned16(x, ldx, depth, 2) && aligned16(w, ldw, w_group, 2) &&
                      (!WACROSS || cols % 8 == 0) && rows * ldx < (1ll << 31) && (WACROSS ? depth : cols) * ldw < (1ll << 31);
  const int size = direct && large_tiles(rows, cols) ? 256 : 128;
  const int tiles = tiles_of(cols, size);
  const int64_t blocks = (most_items(rows, groups, size) + 7) / 8 * 8 * tiles;
  PV2_REQUIRE(blocks < kMostBlocks / (size / 128), "grouped_linear: too many tiles");
  if constexpr (sizeof(E) == 2) {
    if (direct) {
#define PV2_DIRECT(ROWS, COLS)                                                                                       \
  hipLaunchKernelGGL((rows_direct_kernel<typename P::Type, WACROSS, ROWS, COLS>), dim3((unsigned)blocks),            \
                     dim3(2 * ROWS), 0, s, (const E*)x, ldx, (const E*)w, w_group, ldw, (const E*)bias, order, offsets, \
                     (int)rows, (int)groups, cols, depth, tiles, (E*)y)
      if (size == 256) PV2_DIRECT(256, 256);
      else PV2_DIRECT(128, 128);
#undef PV2_DIRECT
      return pv2::check_launch("grouped_linear");
    }
  }
  hipLaunchKernelGGL((rows_kernel<P, WACROSS>), dim3((unsigned)blocks), dim3(kThreads), 0, s, (const E*)x, ldx,
                     (const E*)w, w_group, ldw, (const E*)bias, order, offsets, (int)rows, (int)groups, cols, depth,
                     tiles, (E*)y);
  return pv2::check_launch("grouped_linear");
}

struct Split {   // of the weight gradient
  int unit;
  int64_t items, slabs;   // most items; most of them that leave a partial result: those of groups of more than `unit` rows
};

// Writing and reading an item's partial result costs as much as the products of some 700 rows (16-bit) or 150 (fp32), and
// two (16-bit) or three workgroups fit on a CU: long items and one round of 256 workgroups for the former, two of 256 for
// the latter.  (bf16, 32768 ragged rows, 16 groups, 1024 x 1024: 95 us; with twice as many items 126 and 28 to join them.)
Split split_of(int dtype, int64_t rows, int64_t groups, int n_out, int n_in) {
  const bool full = dtype == PV2_F32;
  const int64_t tiles = (int64_t)tiles_of(n_out, kTile) * tiles_of(n_in, full ? kTile : wgrad_cols(n_in));
  const int64_t want = ((full ? 512 : 256) + tiles - 1) / tiles;
  int64_t unit = (rows + want - 1) / want;
  const int64_t least = full ? 256 : 1024;
  if (unit < least) unit = least;
  unit = (unit + 63) / 64 * 64;
  // a group of r rows has c = 1 + (r - 1) / unit items: the (r - 1) / unit of all groups add up to `more` at most, and no
  // more groups than that have two items or more
  const int64_t more = rows > 0 ? (rows - 1) / unit : 0;
  return {(int)unit, rows / unit + groups, more + (more < groups ? more : groups)};
}

template <class P>
int launch_wgrad(const void* dy, int64_t ldy, const void* x, int64_t ldx, const int32_t* order,
                 const int32_t* offsets, int64_t rows, int64_t groups, int n_out, int n_in, float* ws, void* dw,
                 void* db, hipStream_t s) {
  typedef typename P::E E;
  const bool weights = dw != nullptr;
  const Split sp = split_of(sizeof(E) == 4 ? PV2_F32 : PV2_BF16, rows, groups, n_out, weights ? n_in : 1);
  const bool direct = sizeof(E) == 2 && weights && aligned16(dy, ldy, n_out, 2) && aligned16(x, ldx, n_in, 2);
  const int tile_cols = direct ? wgrad_cols(n_in) : kTile;
  const int to = tiles_of(n_out, kTile), ti = weights ? tiles_of(n_in, tile_cols) : 1;
  const int64_t blocks = (sp.items + 7) / 8 * 8 * to * ti;
  PV2_REQUIRE(blocks < kMostBlocks, "grouped_linear: too many tiles");
  const int64_t size = weights ? (int64_t)n_out * n_in : 0;
  const bool parts = rows > sp.unit;
  PV2_REQUIRE(!parts || ws, "grouped_linear: no workspace");
  float* db_part = parts ? ws + sp.slabs * size : nullptr;
#define PV2_WGRAD(kernel)                                                                                            \
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(kThreads), 0, s, (const E*)dy, ldy, (const E*)x, ldx, order, \
                     offsets, (int)rows, (int)groups, n_out, n_in, sp.unit, to, ti, (E*)dw, (E*)db, ws, db_part)
  if (!weights) {
    PV2_WGRAD((wgrad_kernel<P, false>));
  } else if constexpr (sizeof(E) == 2) {
    if (!direct) PV2_WGRAD((wgrad_kernel<P, true>));
    else if (tile_cols == 256) PV2_WGRAD((wgrad_direct_kernel<typename P::Type, 256>));
    else PV2_WGRAD((wgrad_direct_kernel<typename P::Type, 128>));
  } else {
    PV2_WGRAD((wgrad_kernel<P, true>));
  }
#undef PV2_WGRAD
  if (parts) {
    int64_t chunks = (size + (weights ? 0 : n_out) + kThreads - 1) / kThreads;
    const int64_t most = 1 + 4096 / groups;
    if (chunks > most) chunks = most;
    hipLaunchKernelGGL((join_kernel<P>), dim3((unsigned)(groups * chunks)), dim3(kThreads), 0, s, offsets, (int)rows,
                       (int)groups, sp.unit, size, n_out, (int)chunks, ws, db_part, (E*)dw, (E*)db);
  }
  return pv2::check_launch("grouped_linear_wgrad");
}

int check_shapes(int64_t rows, int64_t groups, int n_out, int n_in) {
  PV2_REQUIRE(rows >= 1 && rows < (1ll << 30) && groups >= 1 && groups <= 4096, "grouped_linear: bad shape");
  PV2_REQUIRE(n_out >= 1 && n_in >= 1 && n_out < (1 << 24) && n_in < (1 << 24), "grouped_linear: bad shape");
  return PV2_OK;
}

}  // namespace

#define PV2_BY_TYPE(dtype, call, what)                         \
  switch (dtype) {                                             \
    case PV2_F32: return call(Full);                           \
    case PV2_BF16: return call(PBf);                           \
    case PV2_F16: return call(PHf);                            \
  }                                                            \
  PV2_REQUIRE(false, what ": bad element type")

extern "C" {

int pv2_grouped_linear_forward(const void* x, int dtype, int64_t rows, int n_in, int64_t x_stride, const void* weight,
                               int64_t weight_group_stride, int64_t weight_row_stride, int64_t groups, int n_out,
                               const void* bias_or_null, const int32_t* order_or_null, const int32_t* offsets,
                               void* out, pv2_stream_t stream) {
  PV2_REQUIRE(x && weight && offsets && out, "grouped_linear_forward: null pointer");
  const int st = check_shapes(rows, groups, n_out, n_in);
  if (st != PV2_OK) return st;
#define PV2_CALL(P) (launch_rows<P, false>(x, x_stride, weight, weight_group_stride, weight_row_stride, bias_or_null, \
                                           order_or_null, offsets, rows, groups, n_out, n_in, out, (hipStream_t)stream))
  PV2_BY_TYPE(dtype, PV2_CALL, "grouped_linear_forward");
#undef PV2_CALL
}

int pv2_grouped_linear_grad_input(const void* grad_out, int dtype, int64_t rows, int n_out, int64_t grad_stride,
                                  const void* weight, int64_t weight_group_stride, int64_t weight_row_stride,
                                  int64_t groups, int n_in, const int32_t* order_or_null, const int32_t* offsets,
                                  void* grad_x, pv2_stream_t stream) {
  PV2_REQUIRE(grad_out && weight && offsets && grad_x, "grouped_linear_grad_input: null pointer");
  const int st = check_shapes(rows, groups, n_out, n_in);
  if (st != PV2_OK) return st;
#define PV2_CALL(P) (launch_rows<P, true>(grad_out, grad_stride, weight, weight_group_stride, weight_row_stride, nullptr, \
                                          order_or_null, offsets, rows, groups, n_in, n_out, grad_x, (hipStream_t)stream))
  PV2_BY_TYPE(dtype, PV2_CALL, "grouped_linear_grad_input");
#undef PV2_CALL
}

int64_t pv2_grouped_linear_workspace_floats(int dtype, int64_t rows, int64_t groups, int n_out, int n_in) {
  if (rows < 1 || groups < 1 || n_out < 1 || n_in < 1) return 0;
  const Split sp = split_of(dtype, rows, groups, n_out, n_in);
  return sp.slabs * ((int64_t)n_out * n_in + n_out);
}

int64_t pv2_grouped_linear_bias_workspace_floats(int dtype, int64_t rows, int64_t groups, int n_out) {
  if (rows < 1 || groups < 1 || n_out < 1) return 0;
  return split_of(dtype, rows, groups, n_out, 1).slabs * n_out;
}

int pv2_grouped_linear_grad_weight(const void* grad_out, int dtype, int64_t rows, int n_out, int64_t grad_stride,
                                   const void* x, int n_in, int64_t x_stride, int64_t groups,
                                   const int32_t* order_or_null, const int32_t* offsets, float* workspace,
                                   void* grad_weight_or_null, void* grad_bias_or_null, pv2_stream_t stream) {
  PV2_REQUIRE(grad_out && offsets && (grad_weight_or_null ? x : grad_bias_or_null),
              "grouped_linear_grad_weight: null pointer");
  const int st = check_shapes(rows, groups, n_out, n_in);
  if (st != PV2_OK) return st;
#define PV2_CALL(P) (launch_wgrad<P>(grad_out, grad_stride, x, x_stride, order_or_null, offsets, rows, groups, n_out, \
                                     n_in, workspace, grad_weight_or_null, grad_bias_or_null, (hipStream_t)stream))
  PV2_BY_TYPE(dtype, PV2_CALL, "grouped_linear_grad_weight");
#undef PV2_CALL
}

}  // extern "C"
