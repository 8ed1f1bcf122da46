// Embedding lookup  y[i] = scale * W[id_i]  (a row of zeros where the id is outside the table) and its gradient
// dW[v] = scale * sum over {i : id_i = v} of dY[i],  fp32 / bf16 / fp16, sums in fp32, one rounding at the end.
//
// Both are bound by memory: the lookup moves n C elements out and the distinct rows in, the gradient n C in and V C
// out.  The gradient sorts the tokens (row_groups.hip) instead of adding to dW with atomics: every element of dW is
// summed in a fixed order and written exactly once, rows that no token names included, so nothing has to be cleared
// first and a class that holds most of the tokens costs no contention.
//   pieces   one wave per kPiece sorted tokens and column slab: an id with more than kPiece tokens leaves the sum of
//            its tokens in this piece in a partial row (a piece has at most two such ids: its first and its last);
//   rows     every row of dW: nothing / at most kPiece tokens / its partial rows, in order.
#include <type_traits>

#include "common.h"

namespace {

constexpr int kThreads = 256;
constexpr int kPiece = 128;

struct F32 {
  typedef float type;
  static __device__ __forceinline__ float to(float v) { return v; }
  static __device__ __forceinline__ float from(float v) { return v; }
};
struct B16 {
  typedef __bf16 type;
  static __device__ __forceinline__ float to(__bf16 v) { return (float)v; }
  static __device__ __forceinline__ __bf16 from(float v) { return (__bf16)v; }   // to nearest even
};
struct H16 {
  typedef _Float16 type;
  static __device__ __forceinline__ float to(_Float16 v) { return (float)v; }
  static __device__ __forceinline__ _Float16 from(float v) { return (_Float16)v; }
};

template <typename T, int VEC>
struct Vec {
  typedef typename T::type E;
  typedef E type __attribute__((ext_vector_type(VEC)));
  static __device__ __forceinline__ void load(const E* p, float* v) {
    const type t = *reinterpret_cast<const type*>(p);
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[j] = T::to(t[j]);
  }
  static __device__ __forceinline__ void store(E* p, const float* v) {
    type t;
#pragma unroll
    for (int j = 0; j < VEC; ++j) t[j] = T::from(v[j]);
    *reinterpret_cast<type*>(p) = t;
  }
};
template <typename T>
struct Vec<T, 1> {
  typedef typename T::type E;
  static __device__ __forceinline__ void load(const E* p, float* v) { v[0] = T::to(*p); }
  static __device__ __forceinline__ void store(E* p, const float* v) { *p = T::from(v[0]); }
};

// `lanes` (a power of two) threads per row, VEC elements each
template <typename T, int VEC>
__global__ __launch_bounds__(kThreads) void lookup_kernel(const void* __restrict__ index, int is64, int64_t n,
                                                          const typename T::type* __restrict__ w, int64_t rows, int c,
                                                          int64_t ldw, float scale, int lanes,
                                                          typename T::type* __restrict__ y) {
  const int per_block = kThreads / lanes;
  const int col0 = (threadIdx.x & (lanes - 1)) * VEC;
  const int64_t stride = (int64_t)gridDim.x * per_block;
  for (int64_t i = (int64_t)blockIdx.x * per_block + threadIdx.x / lanes; i < n; i += stride) {
    const int64_t id = is64 ? ((const int64_t*)index)[i] : (int64_t)((const int32_t*)index)[i];
    const bool ok = id >= 0 && id < rows;
    const typename T::type* src = w + (ok ? id : 0) * ldw;
    for (int col = col0; col < c; col += lanes * VEC) {
      float v[VEC];
      if (ok) {
        Vec<T, VEC>::load(src + col, v);
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[j] *= scale;
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[j] = 0.f;
      }
      Vec<T, VEC>::store(y + i * c + col, v);
    }
  }
}

// acc[j] += sum of dY[order[p]][col + j], p = p0 + r, p0 + r + R, .. < p1
template <typename T, int VEC>
__device__ __forceinline__ void sum_rows(const typename T::type* __restrict__ dy, int64_t ldy,
                                         const int32_t* __restrict__ order, int p0, int p1, int r, int R, int col,
                                         bool ok, float* acc) {
  constexpr int U = 8;
  int p = p0 + r;
  for (; p + (U - 1) * R < p1; p += U * R) {
    int64_t row[U];
#pragma unroll
    for (int u = 0; u < U; ++u) row[u] = order[p + u * R];
    float v[U][VEC];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (ok) {
        Vec<T, VEC>::load(dy + row[u] * ldy + col, v[u]);
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[u][j] = 0.f;
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < VEC; ++j) acc[j] += v[u][j];
  }
  for (; p < p1; p += R) {
    const int64_t row = order[p];
    float v[VEC];
    if (ok) {
      Vec<T, VEC>::load(dy + row * ldy + col, v);
#pragma unroll
      for (int j = 0; j < VEC; ++j) acc[j] += v[j];
    }
  }
}

// sum over the 64 / lanes parts of a wave, lowest part first in every pair: the same order every time
template <int VEC>
__device__ __forceinline__ void join_parts(float* acc, int lanes) {
  for (int d = lanes; d < 64; d <<= 1)
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[j] += __shfl_xor(acc[j], d);
}

template <typename T, int VEC>
__global__ __launch_bounds__(kThreads) void pieces_kernel(const typename T::type* __restrict__ dy, int64_t ldy, int c,
                                                          const int32_t* __restrict__ order,
                                                          const int32_t* __restrict__ ids,
                                                          const int32_t* __restrict__ offsets, int n, int rows,
                                                          int lanes, int slabs, float* __restrict__ partial) {
  const int lane = threadIdx.x & 63;
  const int col_lane = lane & (lanes - 1), r = lane / lanes, R = 64 / lanes;
  const int64_t units = ((int64_t)n + kPiece - 1) / kPiece * slabs;
  for (int64_t unit = (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6); unit < units;
       unit += (int64_t)gridDim.x * (kThreads / 64)) {
    const int piece = (int)(unit / slabs), slab = (int)(unit % slabs);
    const int p0 = piece * kPiece, p1 = (int)min((int64_t)n, (int64_t)p0 + kPiece);
    const int col = (slab * lanes + col_lane) * VEC;
    const bool ok = col < c;
    const int first = ids[p0], last = ids[p1 - 1];
#pragma unroll
    for (int side = 0; side < 2; ++side) {
      const int id = side ? last : first;
      if (id >= rows || (side && last == first)) continue;
      const int from = offsets[id], to = offsets[id + 1];
      if (to - from <= kPiece) continue;
      float acc[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
      sum_rows<T, VEC>(dy, ldy, order, max(p0, from), min(p1, to), r, R, col, ok, acc);
      join_parts<VEC>(acc, lanes);
      if (ok && r == 0) Vec<F32, VEC>::store(partial + (2 * (int64_t)piece + side) * c + col, acc);
    }
  }
}

// WAVES waves share a row (few rows) or each has one (many).  At most kPiece tokens: their rows of dY, else the
// partial rows of the pieces that they lie in.
template <typename T, int VEC, int WAVES>
__global__ __launch_bounds__(WAVES == 1 ? kThreads : WAVES * 64) void rows_kernel(
    const typename T::type* __restrict__ dy, int64_t ldy, int c, const int32_t* __restrict__ order,
    const int32_t* __restrict__ offsets, int64_t rows, int lanes, int slabs, const float* __restrict__ partial,
    float scale, typename T::type* __restrict__ dw) {
  __shared__ float s_sum[WAVES == 1 ? 1 : WAVES][WAVES == 1 ? 1 : 64 * VEC];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int col_lane = lane & (lanes - 1), R = 64 / lanes * (WAVES == 1 ? 1 : WAVES);
  const int r = lane / lanes + (WAVES == 1 ? 0 : wave * (64 / lanes));
  const int64_t units = rows * slabs;
  const int64_t stride = (int64_t)gridDim.x * (WAVES == 1 ? kThreads / 64 : 1);
  for (int64_t unit = WAVES == 1 ? (int64_t)blockIdx.x * (kThreads / 64) + wave : blockIdx.x; unit < units;
       unit += stride) {
    const int64_t v = unit / slabs;
    const int col = ((int)(unit % slabs) * lanes + col_lane) * VEC;
    const bool ok = col < c;
    const int from = offsets[v], to = offsets[v + 1];
    float acc[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
    if (to - from <= kPiece) {
      sum_rows<T, VEC>(dy, ldy, order, from, to, r, R, col, ok, acc);
    } else {
      const int first = from / kPiece, count = (to - 1) / kPiece - first + 1;
      for (int p = r; p < count; p += R) {
        // the piece that a run begins in holds it as its last id, unless the run begins with the piece
        const int64_t slot = 2 * (int64_t)(first + p) + (p == 0 && from % kPiece != 0);
        float t[VEC];
        if (ok) {
          Vec<F32, VEC>::load(partial + slot * c + col, t);
#pragma unroll
          for (int j = 0; j < VEC; ++j) acc[j] += t[j];
        }
      }
    }
    join_parts<VEC>(acc, lanes);
    if (WAVES > 1) {
      if (lane < lanes) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) s_sum[wave][lane * VEC + j] = acc[j];
      }
      __syncthreads();
      if (wave == 0 && lane < lanes) {
        for (int w = 1; w < WAVES; ++w)
#pragma unroll
          for (int j = 0; j < VEC; ++j) acc[j] += s_sum[w][lane * VEC + j];
      }
      __syncthreads();
    }
    if (ok && lane < lanes && (WAVES == 1 || wave == 0)) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) acc[j] *= scale;
      Vec<T, VEC>::store(dw + v * c + col, acc);
    }
  }
}

bool vectors_fit(const void* a, const void* b, int c, int64_t ld, int elem) {
  const int64_t bytes = (int64_t)elem;
  return ((uintptr_t)a % 16 == 0) && ((uintptr_t)b % 16 == 0) && (c * bytes) % 16 == 0 && (ld * bytes) % 16 == 0;
}

int lanes_for(int c, int vec) {
  int lanes = 1;
  while (lanes < 64 && lanes * vec < c) lanes <<= 1;
  return lanes;
}

int64_t align8(int64_t n) { return (n + 7) & ~(int64_t)7; }   // ints: 32 bytes

unsigned blocks_for(int64_t units) {   // four waves a block; the kernels' loops take what a grid cannot hold
  const int64_t blocks = (units + 3) / 4;
  return (unsigned)(blocks < (1 << 20) ? blocks : (1 << 20));
}

struct Layout {   // of the backward's workspace, in ints
  int64_t order, ids, offsets, partial, sort, end;
};
Layout layout_of(int64_t n, int64_t rows, int c) {
  Layout l;
  l.order = 0;
  l.ids = align8(n);
  l.offsets = l.ids + align8(n);
  l.partial = l.offsets + align8(rows + 1);
  l.sort = l.partial + align8(2 * ((n + kPiece - 1) / kPiece) * c);
  l.end = l.sort + pv2_row_groups_workspace_ints(n, rows);
  return l;
}

template <typename T>
int forward(const void* index, int is64, int64_t n, const void* w, int64_t rows, int c, int64_t ldw, float scale,
            void* y, hipStream_t s) {
  typedef typename T::type E;
  constexpr int V = 16 / sizeof(E);
  if (vectors_fit(w, y, c, ldw, sizeof(E))) {
    const int lanes = lanes_for(c, V);
    hipLaunchKernelGGL((lookup_kernel<T, V>), dim3(pv2::grid_for(n * lanes, kThreads)), dim3(kThreads), 0, s, index,
                       is64, n, (const E*)w, rows, c, ldw, scale, lanes, (E*)y);
  } else {
    const int lanes = lanes_for(c, 1);
    hipLaunchKernelGGL((lookup_kernel<T, 1>), dim3(pv2::grid_for(n * lanes, kThreads)), dim3(kThreads), 0, s, index,
                       is64, n, (const E*)w, rows, c, ldw, scale, lanes, (E*)y);
  }
  return pv2::check_launch("embedding_forward");
}

template <typename T, int VEC>
int backward(const int32_t* ws, const Layout& l, int64_t n, int64_t rows, const void* dy, int c, int64_t ldy,
             float scale, void* dw, hipStream_t s) {
  typedef typename T::type E;
  const int lanes = lanes_for(c, VEC);
  const int slabs = (c + lanes * VEC - 1) / (lanes * VEC);
  const int32_t *order = ws + l.order, *ids = ws + l.ids, *offsets = ws + l.offsets;
  float* partial = (float*)(ws + l.partial);
  if (n > kPiece) {
    const int64_t units = (n + kPiece - 1) / kPiece * slabs;
    hipLaunchKernelGGL((pieces_kernel<T, VEC>), dim3(blocks_for(units)), dim3(kThreads), 0, s, (const E*)dy, ldy, c,
                       order, ids, offsets, (int)n, (int)rows, lanes, slabs, partial);
  }
  const int64_t units = rows * slabs;
  // fewer units than the 1024 SIMDs hold waves: 16 waves to a unit, which shortens its chain of dependent reads
  if (units < 4096) {
    hipLaunchKernelGGL((rows_kernel<T, VEC, 16>), dim3((unsigned)units), dim3(1024), 0, s, (const E*)dy, ldy, c, order,
                       offsets, rows, lanes, slabs, partial, scale, (E*)dw);
  } else {
    hipLaunchKernelGGL((rows_kernel<T, VEC, 1>), dim3(blocks_for(units)), dim3(kThreads), 0, s, (const E*)dy, ldy, c,
                       order, offsets, rows, lanes, slabs, partial, scale, (E*)dw);
  }
  return pv2::check_launch("embedding_backward");
}

}  // namespace

extern "C" {

int pv2_embedding_forward(const void* index, int index_is_64, int64_t n, const void* weight, int dtype, int64_t rows,
                          int c, int64_t row_stride, float scale, void* out, pv2_stream_t stream) {
  PV2_REQUIRE(index && weight && out, "embedding_forward: null pointer");
  PV2_REQUIRE(n > 0 && rows > 0 && c > 0 && row_stride >= 0, "embedding_forward: bad shape");
  hipStream_t s = (hipStream_t)stream;
  switch (dtype) {
    case PV2_F32: return forward<F32>(index, index_is_64, n, weight, rows, c, row_stride, scale, out, s);
    case PV2_BF16: return forward<B16>(index, index_is_64, n, weight, rows, c, row_stride, scale, out, s);
    case PV2_F16: return forward<H16>(index, index_is_64, n, weight, rows, c, row_stride, scale, out, s);
  }
  PV2_REQUIRE(false, "embedding_forward: bad element type");
}

int64_t pv2_embedding_backward_workspace_ints(int64_t n, int64_t rows, int c) {
  return layout_of(n, rows, c).end;
}

int pv2_embedding_backward(const void* index, int index_is_64, int64_t n, const void* grad_out, int dtype, int64_t rows,
                           int c, int64_t grad_row_stride, float scale, int32_t* workspace, void* grad_weight,
                           pv2_stream_t stream) {
  PV2_REQUIRE(grad_weight && workspace && (n == 0 || (index && grad_out)), "embedding_backward: null pointer");
  PV2_REQUIRE(n >= 0 && rows > 0 && c > 0 && grad_row_stride >= 0, "embedding_backward: bad shape");
  PV2_REQUIRE((uintptr_t)workspace % 32 == 0, "embedding_backward: workspace not aligned to 32 bytes");
  hipStream_t s = (hipStream_t)stream;
  const Layout l = layout_of(n, rows, c);
  const int st = pv2_row_groups(index, index_is_64, n, rows, workspace + l.order, workspace + l.offsets,
                                workspace + l.ids, workspace + l.sort, stream);
  if (st != PV2_OK) return st;
  const int elem = dtype == PV2_F32 ? 4 : 2;
  const bool vec = vectors_fit(grad_out, grad_weight, c, grad_row_stride, elem);
  switch (dtype) {
    case PV2_F32:
      return vec ? backward<F32, 4>(workspace, l, n, rows, grad_out, c, grad_row_stride, scale, grad_weight, s)
                 : backward<F32, 1>(workspace, l, n, rows, grad_out, c, grad_row_stride, scale, grad_weight, s);
    case PV2_BF16:
      return vec ? backward<B16, 8>(workspace, l, n, rows, grad_out, c, grad_row_stride, scale, grad_weight, s)
                 : backward<B16, 1>(workspace, l, n, rows, grad_out, c, grad_row_stride, scale, grad_weight, s);
    case PV2_F16:
      return vec ? backward<H16, 8>(workspace, l, n, rows, grad_out, c, grad_row_stride, scale, grad_weight, s)
                 : backward<H16, 1>(workspace, l, n, rows, grad_out, c, grad_row_stride, scale, grad_weight, s);
  }
  PV2_REQUIRE(false, "embedding_backward: bad element type");
}

}  // extern "C"
