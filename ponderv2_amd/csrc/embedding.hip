// Embedding lookup  y[i] = scale * W[id_i]  (a row of zeros where the id is outside the table) and its gradient
// dW[v] = scale * sum over {i : id_i = v} of dY[i],  fp32 / bf16 / fp16, sums in fp32, one rounding at the end.
//
// Both are bound by memory: the lookup moves n C elements out and the distinct rows in, the gradient n C in and V C
// out.  The gradient sorts the tokens (row_groups.hip) instead of adding to dW with atomics: every element of dW is
// summed in a fixed order and written exactly once, rows that no token names included, so nothing has to be cleared
// first and a class that holds most of the tokens costs no contention.
//   pieces   32 sorted tokens each, `lanes` threads per piece and column slab: adds up the tokens id after id; an id
//            that lies within the piece is written to dW, one that crosses its borders leaves a partial row (at most
//            two of a piece do: the first and the last);
//   blocks   32 pieces each: the sums of those partial rows, for ids of more than 1024 tokens;
//   rows     every other row of dW: zeros, or the sum of at most 33 partial rows of pieces, or of those of blocks.
// So all waves have the same work and few dependent reads, whatever the ids' frequencies.  (One wave per row of dW instead
// of per piece: the ids of 2 .. 32 tokens, neighbours in a vocabulary, made a few waves last 80 us.)
// Measured on MI355X (copy 5.1 TB/s): 92 001 ids over 36 rows of 512 fp32, lookup 32 us (188 MB written), gradient 84 us
// (pieces 54 - 188 MB read while the lookup's writes still drain -, sort 13, joins 13); 32 768 ids over 65 536 rows of 1024 bf16,
// lookup 26 us, gradient 94 us (sort 33, pieces 21, blocks 8, rows 32: 112 MB of zeros).
#include <type_traits>

#include "common.h"

namespace {

constexpr int kThreads = 256;
constexpr int kPiece = 32;
constexpr int kBlock = 32 * kPiece;
constexpr int kMaxWidth = 1 << 30;   // columns and what a workgroup adds to them stay below 2^31

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
  static __device__ __forceinline__ type raw(const E* p) { return *reinterpret_cast<const type*>(p); }
  static __device__ __forceinline__ void open(const type& t, float* v) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[j] = T::to(t[j]);
  }
  static __device__ __forceinline__ void load(const E* p, float* v) { open(raw(p), v); }
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
  typedef E type;
  static __device__ __forceinline__ type raw(const E* p) { return *p; }
  static __device__ __forceinline__ void open(const type& t, float* v) { v[0] = T::to(t); }
  static __device__ __forceinline__ void load(const E* p, float* v) { open(raw(p), v); }
  static __device__ __forceinline__ void store(E* p, const float* v) { *p = T::from(v[0]); }
};

// `lanes` (a power of two) threads per row, VEC elements each; four rows at a time, so that their ids and then their
// elements are loaded together
template <typename T, int VEC>
__global__ __launch_bounds__(kThreads) void lookup_kernel(const void* __restrict__ index, int is64, int64_t n,
                                                          const typename T::type* __restrict__ w, int64_t rows, int c,
                                                          int64_t ldw, float scale, int lanes,
                                                          typename T::type* __restrict__ y) {
  constexpr int U = 4;
  const int per_block = kThreads / lanes;
  const int col0 = (threadIdx.x & (lanes - 1)) * VEC;
  const int64_t stride = (int64_t)gridDim.x * per_block;
  for (int64_t i0 = (int64_t)blockIdx.x * per_block + threadIdx.x / lanes; i0 < n; i0 += U * stride) {
    int64_t id[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t i = i0 + u * stride;
      id[u] = -1;
      if (i < n) id[u] = is64 ? ((const int64_t*)index)[i] : (int64_t)((const int32_t*)index)[i];
    }
    for (int col = col0; col < c; col += lanes * VEC) {
      float v[U][VEC];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (id[u] >= 0 && id[u] < rows) {
          Vec<T, VEC>::load(w + id[u] * ldw + col, v[u]);
        } else {
#pragma unroll
          for (int j = 0; j < VEC; ++j) v[u][j] = 0.f;
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t i = i0 + u * stride;
        if (i >= n) continue;
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[u][j] = id[u] >= 0 && id[u] < rows ? v[u][j] * scale : 0.f;
        Vec<T, VEC>::store(y + i * c + col, v[u]);
      }
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

// The partial row of the part (of `size` positions) that `part` numbers, for the id whose tokens begin at `from`: a part
// holds the id as its last one if the id's tokens begin inside it, else as its first.
__device__ __forceinline__ int64_t slot_of(int part, int from, int size) {
  return 2 * (int64_t)part + (part == from / size && from % size != 0);
}

// acc[j] += sum of the partial rows of parts a .. b - 1 (of `size` positions), of the id that begins at `from`; parts
// a + r, a + r + R, ..
template <int VEC>
__device__ __forceinline__ void sum_parts(const float* __restrict__ partial, int c, int a, int b, int from, int size,
                                          int r, int R, int col, bool ok, float* acc) {
  constexpr int U = 8;
  for (int p = a + r; p < b; p += U * R) {
    float v[U][VEC];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (ok && p + u * R < b) {
        Vec<F32, VEC>::load(partial + slot_of(p + u * R, from, size) * c + col, v[u]);
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
}

template <typename T, int VEC>
__global__ __launch_bounds__(kThreads) void pieces_kernel(const typename T::type* __restrict__ dy, int64_t ldy, int c,
                                                          const int32_t* __restrict__ order,
                                                          const int32_t* __restrict__ ids, int n, int rows, int lanes,
                                                          int slabs, float scale, float* __restrict__ partial,
                                                          typename T::type* __restrict__ dw) {
  constexpr int U = 16;   // tokens whose rows are loaded together
  typedef typename Vec<T, VEC>::type Raw;
  const int col_lane = threadIdx.x & (lanes - 1), per_block = kThreads / lanes;
  const int64_t units = ((int64_t)n + kPiece - 1) / kPiece * slabs;
  for (int64_t unit = (int64_t)blockIdx.x * per_block + threadIdx.x / lanes; unit < units;
       unit += (int64_t)gridDim.x * per_block) {
    const int piece = (int)(unit / slabs);
    const int col = ((int)(unit % slabs) * lanes + col_lane) * VEC;
    if (col >= c) continue;
    const int p0 = piece * kPiece, p1 = (int)min((int64_t)n, (int64_t)p0 + kPiece);
    const int before = p0 > 0 ? ids[p0 - 1] : -1, after = p1 < n ? ids[p1] : -1;
    float acc[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
    int id = ids[p0], begin = p0;
    auto leave = [&](bool last) {   // the tokens from `begin` on are all of this piece that the id has
      if (id < rows) {
        if ((begin > p0 || before != id) && !(last && after == id)) {
          float v[VEC];
#pragma unroll
          for (int j = 0; j < VEC; ++j) v[j] = acc[j] * scale;
          Vec<T, VEC>::store(dw + (int64_t)id * c + col, v);
        } else {
          Vec<F32, VEC>::store(partial + (2 * (int64_t)piece + (begin > p0)) * c + col, acc);
        }
      }
#pragma unroll
      for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
    };
    for (int p = p0; p < p1; p += U) {
      // (whole groups of four: both lists have room for them behind their last entry)
      int tok[U], row[U];
#pragma unroll
      for (int q = 0; q < U / 4; ++q) {
        int4 a = make_int4(0, 0, 0, 0), b = a;
        if (p + 4 * q < p1) {
          a = *reinterpret_cast<const int4*>(order + p + 4 * q);
          b = *reinterpret_cast<const int4*>(ids + p + 4 * q);
        }
        row[4 * q] = a.x, row[4 * q + 1] = a.y, row[4 * q + 2] = a.z, row[4 * q + 3] = a.w;
        tok[4 * q] = b.x, tok[4 * q + 1] = b.y, tok[4 * q + 2] = b.z, tok[4 * q + 3] = b.w;
      }
      Raw v[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        v[u] = p + u < p1 && tok[u] < rows ? Vec<T, VEC>::raw(dy + (int64_t)row[u] * ldy + col) : (Raw)(0);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (p + u >= p1) break;
        if (tok[u] != id) {
          leave(false);
          id = tok[u];
          begin = p + u;
        }
        float x[VEC];
        Vec<T, VEC>::open(v[u], x);
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[j] += x[j];
      }
    }
    leave(true);
  }
}

// of every block of pieces, the sums of the partial rows of its first and last id, where they have more than kBlock tokens
template <int VEC>
__global__ __launch_bounds__(kThreads) void blocks_kernel(int c, const int32_t* __restrict__ ids,
                                                          const int32_t* __restrict__ offsets, int n, int rows,
                                                          int lanes, int slabs, const float* __restrict__ in,
                                                          float* __restrict__ out) {
  const int lane = threadIdx.x & 63;
  const int col_lane = lane & (lanes - 1), r = lane / lanes, R = 64 / lanes;
  const int64_t units = ((int64_t)n + kBlock - 1) / kBlock * slabs;
  for (int64_t unit = (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6); unit < units;
       unit += (int64_t)gridDim.x * (kThreads / 64)) {
    const int part = (int)(unit / slabs), slab = (int)(unit % slabs);
    const int p0 = part * kBlock, p1 = (int)min((int64_t)n, (int64_t)p0 + kBlock);
    const int col = (slab * lanes + col_lane) * VEC;
    const bool ok = col < c;
    const int first = ids[p0], last = ids[p1 - 1];
#pragma unroll
    for (int side = 0; side < 2; ++side) {
      const int id = side ? last : first;
      if (id >= rows || (side && last == first)) continue;
      const int from = offsets[id], to = offsets[id + 1];
      if (to - from <= kBlock) continue;
      const int a = max(p0, from), b = min(p1, to);
      float acc[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
      sum_parts<VEC>(in, c, a / kPiece, (b - 1) / kPiece + 1, from, kPiece, r, R, col, ok, acc);
      join_parts<VEC>(acc, lanes);
      if (ok && r == 0) Vec<F32, VEC>::store(out + (2 * (int64_t)part + side) * c + col, acc);
    }
  }
}

// the rows of dW that pieces_kernel has not written; `lanes` threads per row and column slab, ROWS rows in turn
template <typename T, int VEC, int ROWS>
__global__ __launch_bounds__(kThreads) void rows_kernel(int c, const int32_t* __restrict__ offsets, int64_t rows,
                                                        int lanes, int slabs, const float* __restrict__ pieces,
                                                        const float* __restrict__ blocks, float scale,
                                                        typename T::type* __restrict__ dw) {
  const int col_lane = threadIdx.x & (lanes - 1), per_block = kThreads / lanes;
  const int64_t units = (rows + ROWS - 1) / ROWS * slabs;
  for (int64_t unit = (int64_t)blockIdx.x * per_block + threadIdx.x / lanes; unit < units;
       unit += (int64_t)gridDim.x * per_block) {
    const int64_t v0 = unit / slabs * ROWS;
    const int col = ((int)(unit % slabs) * lanes + col_lane) * VEC;
    if (col >= c) continue;
    int at[ROWS + 1];
#pragma unroll
    for (int j = 0; j <= ROWS; ++j) at[j] = offsets[min(v0 + j, rows)];
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
      if (v0 + j >= rows) break;
      const int from = at[j], to = at[j + 1];
      if (to > from && from / kPiece == (to - 1) / kPiece) continue;
      float acc[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) acc[e] = 0.f;
      if (to - from > kBlock)
        sum_parts<VEC>(blocks, c, from / kBlock, (to - 1) / kBlock + 1, from, kBlock, 0, 1, col, true, acc);
      else if (to > from)
        sum_parts<VEC>(pieces, c, from / kPiece, (to - 1) / kPiece + 1, from, kPiece, 0, 1, col, true, acc);
#pragma unroll
      for (int e = 0; e < VEC; ++e) acc[e] *= scale;
      Vec<T, VEC>::store(dw + (v0 + j) * c + col, acc);
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
  int64_t order, ids, offsets, pieces, blocks, sort, end;
};
Layout layout_of(int64_t n, int64_t rows, int c) {
  Layout l;
  l.order = 0;
  l.ids = align8(n);
  l.offsets = l.ids + align8(n);
  l.pieces = l.offsets + align8(rows + 1);
  l.blocks = l.pieces + align8(2 * ((n + kPiece - 1) / kPiece) * c);
  l.sort = l.blocks + (n > kBlock ? align8(2 * ((n + kBlock - 1) / kBlock) * c) : 0);
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
  float *pieces = (float*)(ws + l.pieces), *blocks = (float*)(ws + l.blocks);
  auto blocks_of = [&](int64_t units) { return blocks_for((units * lanes + 63) / 64); };
  if (n > 0)
    hipLaunchKernelGGL((pieces_kernel<T, VEC>), dim3(blocks_of((n + kPiece - 1) / kPiece * slabs)), dim3(kThreads), 0,
                       s, (const E*)dy, ldy, c, order, ids, (int)n, (int)rows, lanes, slabs, scale, pieces, (E*)dw);
  if (n > kBlock)
    hipLaunchKernelGGL((blocks_kernel<VEC>), dim3(blocks_for((n + kBlock - 1) / kBlock * slabs)), dim3(kThreads), 0, s,
                       c, ids, offsets, (int)n, (int)rows, lanes, slabs, (const float*)pieces, blocks);
  // eight rows in turn, so that their offsets are loaded together, where that leaves enough waves (both passes of 65536 rows
  // of 1024: 127 us against 132, with 256 tokens 44 against 62; of 8192 rows 87 against 77 one by one, of 65536 rows of 64
  // 75 against 63)
  if (rows * slabs * lanes < 64 * 65536)
    hipLaunchKernelGGL((rows_kernel<T, VEC, 1>), dim3(blocks_of(rows * slabs)), dim3(kThreads), 0, s, c, offsets, rows,
                       lanes, slabs, pieces, blocks, scale, (E*)dw);
  else
    hipLaunchKernelGGL((rows_kernel<T, VEC, 8>), dim3(blocks_of((rows + 7) / 8 * slabs)), dim3(kThreads), 0, s, c,
                       offsets, rows, lanes, slabs, pieces, blocks, scale, (E*)dw);
  return pv2::check_launch("embedding_backward");
}

}  // namespace

extern "C" {

int pv2_embedding_forward(const void* index, int index_is_64, int64_t n, const void* weight, int dtype, int64_t rows,
                          int c, int64_t row_stride, float scale, void* out, pv2_stream_t stream) {
  PV2_REQUIRE(index && weight && out, "embedding_forward: null pointer");
  PV2_REQUIRE(n > 0 && rows > 0 && c > 0 && c < kMaxWidth && row_stride >= 0, "embedding_forward: bad shape");
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
  PV2_REQUIRE(n >= 0 && rows > 0 && c > 0 && c < kMaxWidth && grad_row_stride >= 0, "embedding_backward: bad shape");
  PV2_REQUIRE((uintptr_t)workspace % 32 == 0, "embedding_backward: workspace not aligned to 32 bytes");
  PV2_REQUIRE(dtype == PV2_F32 || dtype == PV2_BF16 || dtype == PV2_F16, "embedding_backward: bad element type");
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
  return PV2_E_BADARG;
}

}  // extern "C"
