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
// rows_kernel      Y and dX: a 128-row x 128-column tile per workgroup, four waves of 64 x 64.
// wgrad_kernel     dW and db: a 128 x 128 tile of one group's dW; long groups are split over rows into items whose fp32
//                  partial results a second launch adds in order (no atomics).  db rides along as a product with ones.
// few_rows_kernel  Y for a handful of rows (serving): bound by reading the weights once; 16 output columns per
//                  workgroup, the reduction split over its four waves, operands straight from memory to registers.
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
  static __device__ __forceinline__ u16x8 ones() { return (u16x8)(H::kOne); }
  static __device__ __forceinline__ float to_float(E v) { return H::to_float(v); }
  static __device__ __forceinline__ E from_float(float v) { return H::from_float(v); }
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
  static constexpr u16 kOne = 0x3f80;
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
  static constexpr u16 kOne = 0x3c00;
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
  static __device__ __forceinline__ u16x8 ones() { return (u16x8)(Bf::kOne); }
  static __device__ __forceinline__ float to_float(E v) { return v; }
  static __device__ __forceinline__ E from_float(float v) { return v; }
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
__device__ __forceinline__ int along_swizzle(int row) { return DEPTH == 64 ? (row & 7) : ((row >> 1) & 3); }
template <int DEPTH>
__device__ __forceinline__ u16x8 along_fragment(const u16* tile, int row, int chunk) {
  return *reinterpret_cast<const u16x8*>(tile + row * DEPTH + ((chunk ^ along_swizzle<DEPTH>(row)) << 3));
}
// "across": kDepth rows of the reduction, 128 columns along the row; read through the transposing LDS read: lane t of a
// 16-lane group points at row t / 4, columns 4 (t % 4) .. of a 4 x 16 block and receives column t of it
__device__ __forceinline__ int across_swizzle(int row) { return (row & 7) << 1; }
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
  int base;        // the group's first item
};

// Item `item` when every group's rows are cut into pieces of `unit` (`empty`: a group without rows has one item, and
// the rows of no group have none).  By a whole wave.
__device__ __forceinline__ Item find_item(const int32_t* __restrict__ offsets, int n_groups, int n_rows, int unit,
                                          bool empty, int item) {
  const int lane = threadIdx.x & 63;
  Item it = {-1, 0, 0, 0, 0, 0};
  int run = 0;
  for (int g0 = 0; g0 <= n_groups; g0 += 64) {
    const int g = g0 + lane;
    int from = 0, to = 0;
    if (g <= n_groups) {
      from = offsets[g];
      to = g < n_groups ? offsets[g + 1] : n_rows;
    }
    int count = (to - from + unit - 1) / unit;
    if (empty) count = g < n_groups ? max(count, 1) : 0;
    int upto = count;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int t = __shfl_up(upto, d);
      if (lane >= d) upto += t;
    }
    const uint64_t past = __ballot(run + upto > item);
    if (past) {
      const int l = __ffsll((unsigned long long)past) - 1;
      it.of = __shfl(count, l);
      it.base = run + __shfl(upto, l) - it.of;
      it.number = item - it.base;
      it.group = g0 + l;
      const int f = __shfl(from, l), t = __shfl(to, l);
      it.first = f + it.number * unit;
      it.last = min(t, it.first + unit);
      return it;
    }
    run += __shfl(upto, 63);
  }
  return it;
}

// Workgroups are dealt to the 8 XCDs in turn; an XCD takes whole items, tile by tile, so that an item's rows are read
// into one L2 only.
__device__ __forceinline__ void item_and_tile(int id, int tiles, int* item, int* tile) {
  *item = id / (8 * tiles) * 8 + id % 8;
  *tile = id / 8 % tiles;
}

// A tile's chunks, held by the workgroup's threads between memory and LDS
template <class P>
constexpr int kChunks = kTile * P::kDepth / 8 / kThreads;

// WACROSS: the weights' reduction runs across their rows (dX: W is [reduction, columns]) instead of along them (Y)
template <class P, bool WACROSS>
__global__ __launch_bounds__(kThreads, P::kPlanes == 1 ? 2 : 2) void rows_kernel(
    const typename P::E* __restrict__ x, int64_t ldx, const typename P::E* __restrict__ w, int64_t w_group,
    int64_t ldw, const typename P::E* __restrict__ bias, const int32_t* __restrict__ order,
    const int32_t* __restrict__ offsets, int n_rows, int n_groups, int cols, int depth, int n_tiles,
    typename P::E* __restrict__ y) {
  typedef typename P::E E;
  constexpr int D = P::kDepth, PL = P::kPlanes, kPlane = kTile * D, U = kChunks<P>;
  __shared__ __attribute__((aligned(16))) u16 s_w[PL * kPlane];
  __shared__ __attribute__((aligned(16))) u16 s_x[PL * kPlane];
  __shared__ int s_row[kTile];
  int item, tile;
  item_and_tile(blockIdx.x, n_tiles, &item, &tile);
  const Item it = find_item(offsets, n_groups, n_rows, kTile, false, item);
  if (it.group < 0) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int c0 = tile * kTile;
  if (tid < kTile) {
    const int p = it.first + tid;
    s_row[tid] = p < it.last ? (order ? order[p] : p) : -1;
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
  const int wc = wave & 1, wr = wave >> 1;   // the wave's 64 columns and rows

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
        for (int p = 0; p < PL; ++p) {
          fx[b][p] = along_fragment<D>(s_x + p * kPlane, wr * 64 + b * 32 + i, 2 * s + h);
          fw[b][p] = WACROSS ? across_fragment(s_w + p * kPlane, s, wc * 2 + b, lane)
                             : along_fragment<D>(s_w + p * kPlane, wc * 64 + b * 32 + i, 2 * s + h);
        }
#pragma unroll
      for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int b = 0; b < 2; ++b) acc[a][b] = P::mfma(fw[a], fx[b], acc[a][b]);
    }
  }

#pragma unroll
  for (int b = 0; b < 2; ++b) {
    const int r = s_row[wr * 64 + b * 32 + i];
    if (r < 0) continue;
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int col = c0 + wc * 64 + a * 32 + 8 * q + 4 * h;
        if (col >= cols) continue;
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          v[j] = acc[a][b][4 * q + j];
          if (bias && col + j < cols) v[j] += P::to_float(bias[(int64_t)it.group * cols + col + j]);
        }
        P::store4(y + (int64_t)r * cols + col, v, cols - col);
      }
  }
}

// dW[g][n][k] over one item's rows.  The item is the whole group: written in the weights' type; else fp32 partials.
template <class P>
__global__ __launch_bounds__(kThreads, 2) void wgrad_kernel(
    const typename P::E* __restrict__ dy, int64_t ldy, const typename P::E* __restrict__ x, int64_t ldx,
    const int32_t* __restrict__ order, const int32_t* __restrict__ offsets, int n_rows, int n_groups, int n_out,
    int n_in, int unit, int tiles_out, int tiles_in, typename P::E* __restrict__ dw, typename P::E* __restrict__ db,
    float* __restrict__ dw_part, float* __restrict__ db_part) {
  typedef typename P::E E;
  constexpr int D = P::kDepth, PL = P::kPlanes, kPlane = kTile * D, U = kChunks<P>;
  __shared__ __attribute__((aligned(16))) u16 s_x[PL * kPlane];
  __shared__ __attribute__((aligned(16))) u16 s_g[PL * kPlane];
  int item, tile;
  item_and_tile(blockIdx.x, tiles_out * tiles_in, &item, &tile);
  const Item it = find_item(offsets, n_groups, n_rows, unit, true, item);
  if (it.group < 0) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int n0 = tile / tiles_in * kTile, k0 = tile % tiles_in * kTile;
  const int i = lane & 31, h = lane >> 5;
  const int wk = wave & 1, wn = wave >> 1;
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
      rx[u] = r >= 0 && k0 + col < n_in ? P::load(x + r * ldx + k0 + col, n_in - k0 - col) : P::zero();
      rg[u] = r >= 0 && n0 + col < n_out ? P::load(dy + r * ldy + n0 + col, n_out - n0 - col) : P::zero();
    }
  };

  f32x16 acc[2][2], acc_b[2];
#pragma unroll
  for (int b = 0; b < 2; ++b)
#pragma unroll
    for (int q = 0; q < 16; ++q) acc[0][b][q] = acc[1][b][q] = acc_b[b][q] = 0.f;

  load_rows(it.first);
  load();
  load_rows(it.first + D);
  for (int p0 = it.first; p0 < it.last; p0 += D) {
    __syncthreads();
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int q = tid + u * kThreads;
      P::stage(s_x + q * 8, kPlane, rx[u]);
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
        for (int p = 0; p < PL; ++p) {
          fx[b][p] = across_fragment(s_x + p * kPlane, s, wk * 2 + b, lane);
          fg[b][p] = across_fragment(s_g + p * kPlane, s, wn * 2 + b, lane);
        }
#pragma unroll
      for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int b = 0; b < 2; ++b) acc[a][b] = P::mfma(fx[a], fg[b], acc[a][b]);
      if (sum_bias) {
        const u16x8 one = P::ones();
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int p = PL - 1; p >= 0; --p) {
            // (a product with 1.0 is exact: the sum of the pieces is the column's sum)
            if constexpr (PL == 1) acc_b[b] = P::mfma(&one, &fg[b][p], acc_b[b]);
            else acc_b[b] = Bf::mfma(one, fg[b][p], acc_b[b]);
          }
      }
    }
  }

  const bool whole = it.of == 1;
#pragma unroll
  for (int b = 0; b < 2; ++b) {
    const int n = n0 + wn * 64 + b * 32 + i;
    if (n >= n_out) continue;
    if (sum_bias && h == 0) {
      if (whole) db[(int64_t)it.group * n_out + n] = P::from_float(acc_b[b][0]);
      else db_part[(int64_t)item * n_out + n] = acc_b[b][0];
    }
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int k = k0 + wk * 64 + a * 32 + 8 * q + 4 * h;
        if (k >= n_in) continue;
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = acc[a][b][4 * q + j];
        if (whole) P::store4(dw + ((int64_t)it.group * n_out + n) * n_in + k, v, n_in - k);
        else Full::store4(dw_part + ((int64_t)item * n_out + n) * n_in + k, v, n_in - k);
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
  // the group's first item: all items of the groups before it
  __shared__ int s_base[kThreads / 64];
  int base = 0;
  for (int f = threadIdx.x; f < g; f += kThreads) base += max(1, (offsets[f + 1] - offsets[f] + unit - 1) / unit);
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
  const int item = blockIdx.x / n_tiles, tile = blockIdx.x % n_tiles;
  const Item it = find_item(offsets, n_groups, n_rows, 16, false, item);
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

constexpr int64_t kMostBlocks = 1 << 24;   // of 256 threads

// Serving: few rows to a group on average, so that the weights are what is read.
bool few_rows(int64_t rows, int64_t groups) { return rows <= 16 || rows <= 4 * groups; }

template <class P, bool WACROSS>
int launch_rows(const void* x, int64_t ldx, const void* w, int64_t w_group, int64_t ldw, const void* bias,
                const int32_t* order, const int32_t* offsets, int64_t rows, int64_t groups, int cols, int depth,
                void* y, hipStream_t s) {
  typedef typename P::E E;
  if (!WACROSS && few_rows(rows, groups)) {
    const int tiles = tiles_of(cols, 16);
    const int64_t blocks = most_items(rows, groups, 16) * tiles;
    PV2_REQUIRE(blocks < kMostBlocks, "grouped_linear: too many tiles");
    hipLaunchKernelGGL((few_rows_kernel<P>), dim3((unsigned)blocks), dim3(kThreads), 0, s, (const E*)x, ldx,
                       (const E*)w, w_group, ldw, (const E*)bias, order, offsets, (int)rows, (int)groups, cols, depth,
                       tiles, (E*)y);
    return pv2::check_launch("grouped_linear");
  }
  const int tiles = tiles_of(cols, kTile);
  const int64_t blocks = (most_items(rows, groups, kTile) + 7) / 8 * 8 * tiles;
  PV2_REQUIRE(blocks < kMostBlocks, "grouped_linear: too many tiles");
  hipLaunchKernelGGL((rows_kernel<P, WACROSS>), dim3((unsigned)blocks), dim3(kThreads), 0, s, (const E*)x, ldx,
                     (const E*)w, w_group, ldw, (const E*)bias, order, offsets, (int)rows, (int)groups, cols, depth,
                     tiles, (E*)y);
  return pv2::check_launch("grouped_linear");
}

struct Split {   // of the weight gradient
  int unit;
  int64_t items;
};

// About 512 workgroups where the rows allow it: two to a CU.
Split split_of(int64_t rows, int64_t groups, int n_out, int n_in) {
  const int64_t tiles = (int64_t)tiles_of(n_out, kTile) * tiles_of(n_in, kTile);
  const int64_t want = (512 + tiles - 1) / tiles;
  int64_t unit = (rows + want - 1) / want;
  if (unit < 256) unit = 256;
  unit = (unit + 63) / 64 * 64;
  return {(int)unit, rows / unit + groups};
}

template <class P>
int launch_wgrad(const void* dy, int64_t ldy, const void* x, int64_t ldx, const int32_t* order,
                 const int32_t* offsets, int64_t rows, int64_t groups, int n_out, int n_in, float* ws, void* dw,
                 void* db, hipStream_t s) {
  typedef typename P::E E;
  const Split sp = split_of(rows, groups, n_out, n_in);
  const int to = tiles_of(n_out, kTile), ti = tiles_of(n_in, kTile);
  const int64_t blocks = (sp.items + 7) / 8 * 8 * to * ti;
  PV2_REQUIRE(blocks < kMostBlocks, "grouped_linear: too many tiles");
  const int64_t size = (int64_t)n_out * n_in;
  const bool parts = rows > sp.unit;
  PV2_REQUIRE(!parts || ws, "grouped_linear: no workspace");
  float* db_part = parts ? ws + sp.items * size : nullptr;
  hipLaunchKernelGGL((wgrad_kernel<P>), dim3((unsigned)blocks), dim3(kThreads), 0, s, (const E*)dy, ldy, (const E*)x,
                     ldx, order, offsets, (int)rows, (int)groups, n_out, n_in, sp.unit, to, ti, (E*)dw, (E*)db, ws,
                     db_part);
  if (parts) {
    int64_t chunks = (size + kThreads - 1) / kThreads;
    const int64_t most = 1 + 4096 / groups;
    if (chunks > most) chunks = most;
    hipLaunchKernelGGL((join_kernel<P>), dim3((unsigned)(groups * chunks)), dim3(kThreads), 0, s, offsets, (int)rows,
                       (int)groups, sp.unit, size, n_out, (int)chunks, ws, db_part, (E*)dw, (E*)db);
  }
  return pv2::check_launch("grouped_linear_wgrad");
}

int check_shapes(int64_t rows, int64_t groups, int n_out, int n_in) {
  PV2_REQUIRE(rows >= 1 && rows < (1ll << 30) && groups >= 1 && groups < (1 << 20), "grouped_linear: bad shape");
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

int64_t pv2_grouped_linear_workspace_floats(int64_t rows, int64_t groups, int n_out, int n_in) {
  if (rows < 1 || groups < 1 || n_out < 1 || n_in < 1) return 0;
  const Split sp = split_of(rows, groups, n_out, n_in);
  return rows > sp.unit ? sp.items * ((int64_t)n_out * n_in + n_out) : 0;
}

int pv2_grouped_linear_grad_weight(const void* grad_out, int dtype, int64_t rows, int n_out, int64_t grad_stride,
                                   const void* x, int n_in, int64_t x_stride, int64_t groups,
                                   const int32_t* order_or_null, const int32_t* offsets, float* workspace,
                                   void* grad_weight, void* grad_bias_or_null, pv2_stream_t stream) {
  PV2_REQUIRE(grad_out && x && offsets && grad_weight, "grouped_linear_grad_weight: null pointer");
  const int st = check_shapes(rows, groups, n_out, n_in);
  if (st != PV2_OK) return st;
#define PV2_CALL(P) (launch_wgrad<P>(grad_out, grad_stride, x, x_stride, order_or_null, offsets, rows, groups, n_out, \
                                     n_in, workspace, grad_weight, grad_bias_or_null, (hipStream_t)stream))
  PV2_BY_TYPE(dtype, PV2_CALL, "grouped_linear_grad_weight");
#undef PV2_CALL
}

}  // extern "C"
