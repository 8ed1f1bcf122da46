// Distillation from a teacher's top logits.  A row has V student logits s and a list of k classes c_e with teacher
// logits t_e; with temperature tau
//     p_e = softmax_e(t_e / tau) over the row's listed classes,   q_j = softmax_j(s_j / tau) over all V,
//     loss = tau^2 sum_e p_e (log p_e - log q_{c_e}),             d loss / d s_j = tau (q_j - sum_{e: c_e = j} p_e).
// An entry counts if 0 <= c_e < V and t_e > -inf; a row without one has loss 0 and gradient 0 and its logits are not
// read.  Classes may repeat within a row: their p add.
//
// Bound by memory: the forward pass reads T V logits once - every thread keeps a running maximum and a sum of
// exponentials relative to it, joined at the end - and the backward pass reads them once more and writes T V gradients.
// Statistics, probabilities and sums are fp32, exponents relative to the row's maximum (see exponent() below: nothing is
// lost for large logits); gradients are rounded once, to the logits' type.
//   V <= 512       a row per 4 .. 64 lanes of a wave, held in registers;
//   larger V       a workgroup per row, or - few rows - several per row and a second launch that joins their statistics.
// Sums over rows are formed from per-workgroup sums in a fixed order: no atomics.
// Measured on MI355X: 4096 x 65 537 bf16, k = 32: forward 135 - 144 us, backward 206 - 210 us - 1.61 GB at 4.6 TB/s, where a copy
// reaches 5.1; without the exponentials the forward pass takes 142 us, without its lists 140.  92 001 x 25 fp32: 9 + 3 and
// 13 us; one row of 131 072: 11 and 7 us.
#include <type_traits>

#include "common.h"

namespace {

constexpr int kThreads = 256;
// (20000 rows of 512 classes: both passes 58 us this way, 140 by workgroups; 92001 rows of 25: 25 us, 638)
constexpr int kSmallV = 512;
constexpr int kPerLane = 8;          // elements of a row that a lane holds (V <= 512)
constexpr int kMaxTop = 1024;
constexpr int kSmallLds = 32 * 1024; // teacher entries of a workgroup's rows (V <= 512)
constexpr float kMinTau = 0.99e-4f, kMaxTau = 1.01e4f;   // (1e-4 .. 1e4, rounded either way)
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }  // results below 2^-126: 0
__device__ __forceinline__ float log2_of(float x) { return log2f(x); }

struct F32 {
  typedef float type;
  static constexpr int kVec = 4;
};
struct B16 {
  typedef __bf16 type;
  static constexpr int kVec = 8;
};
struct H16 {
  typedef _Float16 type;
  static constexpr int kVec = 8;
};

// (x - m) c, the exponent (base 2) of x relative to the maximum m.  One fused multiply-add relative to the rounded m c:
// every use of the same m has the same error in m c, so it leaves softmax and logarithms alone, and the result has one
// rounding of its own size.  That error is at most 1/2 where |m c| < 2^24; larger ones would carry the exponentials past the
// range of their type (at 2^32 by 2^128), masks of the type's lowest value overflow m c, infinities have no difference: for
// those the difference first, m - m being 0 for a finite m.
__device__ __forceinline__ bool plain(float mc) { return fabsf(mc) < 16777216.f; }
__device__ __forceinline__ float exponent_far(float x, float m, float c) {
  return x == m && fabsf(m) < __builtin_huge_valf() ? 0.f : (x - m) * c;
}
__device__ __forceinline__ float exponent(float x, float m, float c) {
#pragma clang fp contract(off)   // (the rounded product)
  const float mc = m * c;
  return plain(mc) ? fmaf(x, c, -mc) : exponent_far(x, m, c);
}

struct Stat {   // running maximum m and sum of exp2(exponent(x, m, c))
  float m, s;
};
constexpr float kNegInf = -__builtin_huge_valf();

// the factor of sums relative to `m` when the maximum becomes `to` >= m; relative to m means the rounded m c where that is
// plain, m c itself elsewhere, as in exponent()
__device__ __forceinline__ float rescale(float m, float to, float c) {
#pragma clang fp contract(off)   // the difference of the rounded products, as exponent() uses them
  if (m == to) return 1.f;
  const float mc = m * c, toc = to * c;
  const float d = plain(mc) ? (plain(toc) ? mc - toc : fmaf(-to, c, mc)) : plain(toc) ? fmaf(m, c, -toc) : (m - to) * c;
  return exp2_fast(d);
}
__device__ __forceinline__ Stat join(Stat a, Stat b, float c) {
  Stat r;
  r.m = fmaxf(a.m, b.m);
  // a side that saw nothing above -inf has sum 0 (or NaN, which has to stay)
  r.s = a.s * rescale(a.m, r.m, c) + b.s * rescale(b.m, r.m, c);
  return r;
}

__device__ __forceinline__ Stat join_wave(Stat a, float c, int width) {
  for (int d = 1; d < width; d <<= 1) {
    Stat b;
    b.m = __shfl_xor(a.m, d);
    b.s = __shfl_xor(a.s, d);
    a = join(a, b, c);
  }
  return a;
}

template <int N>
__device__ __forceinline__ void take(Stat& a, const float* x, float c) {
  float m = a.m;
#pragma unroll
  for (int j = 0; j < N; ++j) m = fmaxf(m, x[j]);
  float s = a.s;
  if (a.m != m) s *= rescale(a.m, m, c);
  const float mc = m * c;
  if (plain(mc)) {
    float part[4] = {s, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < N; ++j) part[j & 3] += exp2_fast(fmaf(x[j], c, -mc));
    s = (part[0] + part[1]) + (part[2] + part[3]);
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j)   // (only -inf so far: nothing to add)
      s += m == kNegInf && x[j] == m ? 0.f : exp2_fast(exponent_far(x[j], m, c));
  }
  a.m = m;
  a.s = s;
}

struct Teacher {   // lists of all rows
  const void* index;
  int is64;
  const void* logits;
  int dtype;       // PV2_F32 / BF16 / F16
  int k;
  int64_t ld_index, ld_logits;
  __device__ __forceinline__ int64_t id(int64_t row, int e) const {
    return is64 ? ((const int64_t*)index)[row * ld_index + e] : (int64_t)((const int32_t*)index)[row * ld_index + e];
  }
  __device__ __forceinline__ float logit(int64_t row, int e) const {
    const int64_t at = row * ld_logits + e;
    return dtype == PV2_F32    ? ((const float*)logits)[at]
           : dtype == PV2_BF16 ? (float)((const __bf16*)logits)[at]
                               : (float)((const _Float16*)logits)[at];
  }
};

// The list of `row`, by `width` lanes (a power of two, aligned): ids[e] (-1: does not count), p[e]; returns whether any
// entry counts, *log2_sum = log2 of sum exp2(exponent(t, *top, c)).
__device__ __forceinline__ bool read_list(const Teacher& t, int64_t row, int classes, float c, int lane, int width,
                                          int* ids, float* p, float* top, float* log2_sum) {
  float m = kNegInf;
  int any = 0;
  for (int e = lane; e < t.k; e += width) {
    const int64_t id = t.id(row, e);
    const float v = t.logit(row, e);
    const bool ok = id >= 0 && id < classes && !(v == kNegInf);
    ids[e] = ok ? (int)id : -1;
    p[e] = v;
    if (ok) {
      any = 1;
      m = fmaxf(m, v);
    }
  }
  for (int d = 1; d < width; d <<= 1) {
    m = fmaxf(m, __shfl_xor(m, d));
    any |= __shfl_xor(any, d);
  }
  float s = 0.f;
  for (int e = lane; e < t.k; e += width) {
    const float x = ids[e] >= 0 ? exp2_fast(exponent(p[e], m, c)) : 0.f;
    s += x;
  }
  for (int d = 1; d < width; d <<= 1) s += __shfl_xor(s, d);
  *top = m;
  *log2_sum = log2_of(s);
  return any != 0;
}

// sum over the list of p_e (log p_e - log q_e), by `width` lanes
template <typename E>
__device__ __forceinline__ float list_loss(const E* __restrict__ x, int k, int lane, int width, const int* ids,
                                           const float* t, float t_top, float t_log2, Stat st, float c) {
  const float s_log2 = log2_of(st.s);
  float sum = 0.f;
  for (int e = lane; e < k; e += width) {
    if (ids[e] < 0) continue;
    const float log_p = exponent(t[e], t_top, c) - t_log2;
    const float p = exp2_fast(log_p);
    const float xv = (float)x[ids[e]];
    const float log_q = exponent(xv, st.m, c) - s_log2;
    if (!(p == 0.f)) sum += p * (log_p - log_q);   // 0 log 0 = 0, also where q = 0
  }
  for (int d = 1; d < width; d <<= 1) sum += __shfl_xor(sum, d);
  return sum * kLn2;
}

struct Totals {   // of all rows: the sum of the losses (mean: over their rows) and the number of rows that count
  float *loss, *count;
  int mean;
  __device__ __forceinline__ void set(float sum, float rows) const {
    *loss = mean ? sum / fmaxf(rows, 1.f) : sum;
    *count = rows;
  }
};

// the workgroup's rows' losses and their number -> partial[2 blockIdx.x ..], or the totals if there is no other workgroup
__device__ __forceinline__ void block_sums(float loss, float rows, float* __restrict__ partial, const Totals& all) {
  __shared__ float s_l[kThreads / 64], s_n[kThreads / 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    loss += __shfl_xor(loss, d);
    rows += __shfl_xor(rows, d);
  }
  if (lane == 0) {
    s_l[wave] = loss;
    s_n[wave] = rows;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kThreads / 64; ++w) {
      loss += s_l[w];
      rows += s_n[w];
    }
    if (gridDim.x == 1) {
      all.set(loss, rows);
    } else {
      partial[2 * (int64_t)blockIdx.x] = loss;
      partial[2 * (int64_t)blockIdx.x + 1] = rows;
    }
  }
}

// ------------------------------------------------------------------------------------------ V <= 512
template <typename T>
__global__ __launch_bounds__(kThreads) void small_forward_kernel(const typename T::type* __restrict__ x, int64_t ld,
                                                                 int64_t rows, int V, Teacher t, float c, float scale,
                                                                 int width, float* __restrict__ stats,
                                                                 float* __restrict__ row_loss,
                                                                 float* __restrict__ partial, Totals all) {
  extern __shared__ float s_list[];   // [rows of the block][k] ids, then logits
  const int per_block = kThreads / width;
  const int lane = threadIdx.x & (width - 1), slot = threadIdx.x / width;
  int* ids = reinterpret_cast<int*>(s_list) + slot * t.k;
  float* tl = s_list + per_block * t.k + slot * t.k;
  float loss_sum = 0.f, row_sum = 0.f;
  for (int64_t row = (int64_t)blockIdx.x * per_block + slot; row < rows; row += (int64_t)gridDim.x * per_block) {
    float top, t_log2;
    const bool any = read_list(t, row, V, c, lane, width, ids, tl, &top, &t_log2);
    Stat st = {kNegInf, 0.f};
    float loss = 0.f;
    if (any) {
      const typename T::type* xr = x + row * ld;
      float v[kPerLane];
#pragma unroll
      for (int j = 0; j < kPerLane; ++j) {
        const int col = lane + j * width;
        v[j] = col < V ? (float)xr[col] : kNegInf;
      }
      take<kPerLane>(st, v, c);
      st = join_wave(st, c, width);
      loss = list_loss(xr, t.k, lane, width, ids, tl, top, t_log2, st, c) * scale;
    }
    if (lane == 0) {
      stats[2 * row] = st.m;
      stats[2 * row + 1] = st.s;
      if (row_loss) row_loss[row] = loss;
      loss_sum += loss;
      row_sum += any ? 1.f : 0.f;
    }
  }
  block_sums(loss_sum, row_sum, partial, all);
}

// what every row's gradient is multiplied by: upstream, tau and the mean's 1 / number of rows
struct Scale {
  const float* upstream;   // one value, or one for each row
  int per_row;
  const float* count;      // rows that count (mean), or null
  float tau;
  __device__ __forceinline__ float operator()(int64_t row) const {
    const float g = upstream[per_row ? row : 0] * tau;
    return count ? g / fmaxf(*count, 1.f) : g;
  }
};

// entry e's class's whole probability, or -1 if an earlier entry has the same class
__device__ __forceinline__ float class_share(const int* ids, const float* p, int k, int e) {
  const int id = ids[e];
  float sum = 0.f;
  for (int f = 0; f < k; ++f) {
    if (ids[f] != id) continue;
    if (f < e) return -1.f;
    sum += p[f];
  }
  return sum;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void small_backward_kernel(const typename T::type* __restrict__ x, int64_t ld,
                                                                  int64_t rows, int V, Teacher t, float c, Scale scale,
                                                                  int width, const float* __restrict__ stats,
                                                                  typename T::type* __restrict__ dx) {
  typedef typename T::type E;
  extern __shared__ float s_list[];
  const int per_block = kThreads / width;
  const int lane = threadIdx.x & (width - 1), slot = threadIdx.x / width;
  int* ids = reinterpret_cast<int*>(s_list) + slot * t.k;
  float* p = s_list + per_block * t.k + slot * t.k;
  for (int64_t row0 = (int64_t)blockIdx.x * per_block; row0 < rows; row0 += (int64_t)gridDim.x * per_block) {
    const int64_t row = row0 + slot;
    const bool mine = row < rows;
    bool any = false;
    float m = 0.f, s_log2 = 0.f, g = 0.f;
    if (mine) {
      float top, t_log2;
      any = read_list(t, row, V, c, lane, width, ids, p, &top, &t_log2);
      for (int e = lane; e < t.k; e += width) p[e] = ids[e] >= 0 ? exp2_fast(exponent(p[e], top, c) - t_log2) : 0.f;
      m = stats[2 * row];
      s_log2 = log2_of(stats[2 * row + 1]);
      g = any ? scale(row) : 0.f;
#pragma unroll
      for (int j = 0; j < kPerLane; ++j) {
        const int col = lane + j * width;
        if (col < V) {
          float d = 0.f;
          if (any) {
            const float v = (float)x[row * ld + col];
            d = g * exp2_fast(exponent(v, m, c) - s_log2);
          }
          dx[row * V + col] = (E)d;
        }
      }
    }
    __syncthreads();   // the lists are whole, and the dense values are written before the listed ones replace them
    if (mine && any)
      for (int e = lane; e < t.k; e += width) {
        if (ids[e] < 0) continue;
        const float share = class_share(ids, p, t.k, e);
        if (share < 0.f) continue;
        const float q = exp2_fast(exponent((float)x[row * ld + ids[e]], m, c) - s_log2);
        dx[row * V + ids[e]] = (E)(g * (q - share));
      }
    __syncthreads();
  }
}

// ------------------------------------------------------------------------------------------ larger V
// f(x, first column, count) over columns a .. b of a row: single elements up to a 16-byte boundary, vectors, the rest
template <typename T, int UNROLL, typename Body1, typename BodyN>
__device__ __forceinline__ void walk(const typename T::type* __restrict__ row, int64_t a, int64_t b, Body1 one,
                                     BodyN many) {
  typedef typename T::type E;
  constexpr int V = T::kVec;
  typedef E VecT __attribute__((ext_vector_type(V)));
  const int off = (int)(((uintptr_t)(row + a) / sizeof(E)) % V);
  int64_t body = a + (off ? V - off : 0);
  if (body > b) body = b;
  if ((int64_t)threadIdx.x < body - a) one(a + threadIdx.x, (float)row[a + threadIdx.x]);
  const int64_t vecs = (b - body) / V;
  int64_t i = threadIdx.x;
  const VecT* vec = reinterpret_cast<const VecT*>(row + body);
  VecT t[UNROLL];
  if (i + (UNROLL - 1) * kThreads < vecs) {
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) t[u] = vec[i + u * kThreads];
  }
  for (; i + (UNROLL - 1) * kThreads < vecs; i += UNROLL * kThreads) {
    float v[UNROLL * V];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
#pragma unroll
      for (int j = 0; j < V; ++j) v[u * V + j] = (float)t[u][j];
    if (i + (2 * UNROLL - 1) * kThreads < vecs) {   // the next vectors are on their way while these are worked on
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) t[u] = vec[i + (UNROLL + u) * kThreads];
    }
    many(body + i * V, v, std::integral_constant<int, UNROLL>());
  }
  for (; i < vecs; i += kThreads) {
    const VecT t = *reinterpret_cast<const VecT*>(row + body + i * V);
    float v[V];
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = (float)t[j];
    many(body + i * V, v, std::integral_constant<int, 1>());
  }
  const int64_t tail = body + vecs * V;
  if ((int64_t)threadIdx.x < b - tail) one(tail + threadIdx.x, (float)row[tail + threadIdx.x]);
}

__device__ __forceinline__ Stat join_block(Stat a, float c) {
  __shared__ Stat s_w[kThreads / 64];
  a = join_wave(a, c, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s_w[threadIdx.x >> 6] = a;
  __syncthreads();
  a = s_w[0];
#pragma unroll
  for (int w = 1; w < kThreads / 64; ++w) a = join(a, s_w[w], c);
  return a;
}

template <typename T>
__device__ __forceinline__ Stat row_stat(const typename T::type* __restrict__ row, int64_t a, int64_t b, float c) {
  constexpr int V = T::kVec;
  Stat st = {kNegInf, 0.f};
  walk<T, 2>(
      row, a, b, [&](int64_t, float v) { take<1>(st, &v, c); },
      [&](int64_t, const float* v, auto n) { take<decltype(n)::value * V>(st, v, c); });
  return join_block(st, c);
}

// whether any entry of the row's list counts (by the whole workgroup; nothing is kept)
__device__ __forceinline__ bool has_list(const Teacher& t, int64_t row, int V) {
  int any = 0;
  for (int e = threadIdx.x; e < t.k; e += kThreads) {
    const int64_t id = t.id(row, e);
    any |= id >= 0 && id < V && !(t.logit(row, e) == kNegInf);
  }
  return __syncthreads_or(any) != 0;
}

// blockIdx.x walks (row, split): the statistics of the split's columns
template <typename T>
__global__ __launch_bounds__(kThreads) void split_stats_kernel(const typename T::type* __restrict__ x, int64_t ld,
                                                               int64_t rows, int V, Teacher t, float c, int splits,
                                                               int64_t per_split, float* __restrict__ part) {
  for (int64_t unit = blockIdx.x; unit < rows * splits; unit += gridDim.x) {
    const int64_t row = unit / splits, a = (unit % splits) * per_split;
    Stat st = {kNegInf, 0.f};
    if (has_list(t, row, V)) st = row_stat<T>(x + row * ld, a, min((int64_t)V, a + per_split), c);
    if (threadIdx.x == 0) {
      part[2 * unit] = st.m;
      part[2 * unit + 1] = st.s;
    }
  }
}

// part == nullptr: the statistics here; else they are joined from the splits'
template <typename T>
__global__ __launch_bounds__(kThreads) void row_forward_kernel(const typename T::type* __restrict__ x, int64_t ld,
                                                               int64_t rows, int V, Teacher t, float c, float scale,
                                                               const float* __restrict__ part, int splits,
                                                               float* __restrict__ stats, float* __restrict__ row_loss,
                                                               float* __restrict__ partial, Totals all) {
  __shared__ int s_ids[kMaxTop];
  __shared__ float s_t[kMaxTop];
  float loss_sum = 0.f, row_sum = 0.f;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const typename T::type* xr = x + row * ld;
    const bool any = has_list(t, row, V);
    Stat st = {kNegInf, 0.f};
    if (any) {
      if (part == nullptr) {
        st = row_stat<T>(xr, 0, V, c);
      } else {
        for (int i = threadIdx.x; i < splits; i += kThreads) {
          const Stat o = {part[2 * (row * splits + i)], part[2 * (row * splits + i) + 1]};
          st = join(st, o, c);
        }
        st = join_block(st, c);
      }
    }
    if (threadIdx.x < 64) {
      float loss = 0.f;
      if (any) {
        float top, t_log2;
        read_list(t, row, V, c, threadIdx.x, 64, s_ids, s_t, &top, &t_log2);
        loss = list_loss(xr, t.k, threadIdx.x, 64, s_ids, s_t, top, t_log2, st, c) * scale;
      }
      if (threadIdx.x == 0) {
        stats[2 * row] = st.m;
        stats[2 * row + 1] = st.s;
        if (row_loss) row_loss[row] = loss;
        loss_sum += loss;
        row_sum += any ? 1.f : 0.f;
      }
    }
  }
  block_sums(loss_sum, row_sum, partial, all);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void row_backward_kernel(const typename T::type* __restrict__ x, int64_t ld,
                                                                int64_t rows, int V, Teacher t, float c, Scale scale,
                                                                int splits, int64_t per_split,
                                                                const float* __restrict__ stats,
                                                                typename T::type* __restrict__ dx) {
  typedef typename T::type E;
  constexpr int VN = T::kVec;
  __shared__ int s_ids[kMaxTop];
  __shared__ float s_p[kMaxTop];
  __shared__ int s_any;
  // last rows first: the forward pass read them last, and what it read last is still in the 256 MB cache
  for (int64_t unit = rows * splits - 1 - blockIdx.x; unit >= 0; unit -= gridDim.x) {
    const int64_t row = unit / splits, a = (unit % splits) * per_split, b = min((int64_t)V, a + per_split);
    if (threadIdx.x < 64) {
      float top, t_log2;
      const bool any = read_list(t, row, V, c, threadIdx.x, 64, s_ids, s_p, &top, &t_log2);
      for (int e = threadIdx.x; e < t.k; e += 64)
        s_p[e] = s_ids[e] >= 0 ? exp2_fast(exponent(s_p[e], top, c) - t_log2) : 0.f;
      if (threadIdx.x == 0) s_any = any;
    }
    __syncthreads();
    const bool any = s_any != 0;
    const float m = stats[2 * row], s_log2 = log2_of(stats[2 * row + 1]);
    const float g = any ? scale(row) : 0.f;
    const E* xr = x + row * ld;
    E* dr = dx + row * V;
    if (!any) {
      for (int64_t j = a + threadIdx.x; j < b; j += kThreads) dr[j] = (E)0.f;
    } else {
      // x and dx rows share their alignment when both begin alike; else every element is stored by itself
      const bool same = ((uintptr_t)xr % 16) == ((uintptr_t)dr % 16);
      auto dense = [&](auto q) {   // q(x): its probability
        walk<T, 2>(
            xr, a, b, [&](int64_t j, float v) { dr[j] = (E)(g * q(v)); },
            [&](int64_t j, const float* v, auto n) {
              typedef E VecT __attribute__((ext_vector_type(VN)));
#pragma unroll
              for (int u = 0; u < decltype(n)::value; ++u) {
                VecT o;
#pragma unroll
                for (int i = 0; i < VN; ++i) o[i] = (E)(g * q(v[u * VN + i]));
                E* at = dr + j + (int64_t)u * kThreads * VN;
                if (same) {
                  *reinterpret_cast<VecT*>(at) = o;
                } else {
#pragma unroll
                  for (int i = 0; i < VN; ++i) at[i] = o[i];
                }
              }
            });
      };
      const float mc = m * c;
      if (plain(mc)) dense([&](float v) { return exp2_fast(fmaf(v, c, -mc) - s_log2); });
      else dense([&](float v) { return exp2_fast(exponent_far(v, m, c) - s_log2); });
    }
    __syncthreads();   // the dense values are written before the listed ones replace them
    if (any)
      for (int e = threadIdx.x; e < t.k; e += kThreads) {
        const int id = s_ids[e];
        if (id < a || id >= b) continue;
        const float share = class_share(s_ids, s_p, t.k, e);
        if (share < 0.f) continue;
        const float q = exp2_fast(exponent((float)xr[id], m, c) - s_log2);
        dr[id] = (E)(g * (q - share));
      }
    __syncthreads();
  }
}

__global__ __launch_bounds__(1024) void totals_kernel(const float* __restrict__ partial, int n, Totals all) {
  __shared__ float s_l[16], s_n[16];
  float loss = 0.f, rows = 0.f;
  for (int i = threadIdx.x; i < n; i += 1024) {
    loss += partial[2 * i];
    rows += partial[2 * i + 1];
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    loss += __shfl_xor(loss, d);
    rows += __shfl_xor(rows, d);
  }
  if ((threadIdx.x & 63) == 0) {
    s_l[threadIdx.x >> 6] = loss;
    s_n[threadIdx.x >> 6] = rows;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 16; ++w) {
      loss += s_l[w];
      rows += s_n[w];
    }
    all.set(loss, rows);
  }
}

struct Plan {
  int width;        // lanes per row (V <= kSmallV), else 0
  int splits;       // workgroups per row otherwise
  int64_t per_split;
  int blocks;       // of the kernel that ends in block_sums
};

constexpr int kMaxBlocks = 4096;

Plan plan_of(int64_t rows, int V, int k) {
  Plan p = {0, 1, V, 1};
  if (V <= kSmallV) {
    p.width = 4;
    while (p.width * kPerLane < V || (kThreads / p.width) * k * 8 > kSmallLds) p.width <<= 1;
    const int per_block = kThreads / p.width;
    const int64_t b = (rows + per_block - 1) / per_block;
    p.blocks = (int)(b < kMaxBlocks ? b : kMaxBlocks);
    return p;
  }
  // at least 512 workgroups, each with 4096 columns or more (one row of 131072: both passes 17 us, 47 with one workgroup; 64
  // rows: 36 and 65; two workgroups for each of 512 rows of 32768 would be 50 against 45)
  int64_t splits = (512 + rows - 1) / rows;
  const int64_t most = (V + 4095) / 4096;
  if (splits > most) splits = most;
  p.per_split = ((V + splits - 1) / splits + 15) / 16 * 16;
  p.splits = (int)((V + p.per_split - 1) / p.per_split);
  p.blocks = (int)(rows < kMaxBlocks ? rows : kMaxBlocks);
  return p;
}

unsigned units_of(int64_t rows, int splits) {
  const int64_t u = rows * splits;
  return (unsigned)(u < (1 << 20) ? u : (1 << 20));
}

template <typename T>
int forward(const void* x, int64_t ld, int64_t rows, int V, const Teacher& t, float tau, int mean, float* stats,
            float* row_loss, float* loss, float* count, float* ws, hipStream_t s) {
  typedef typename T::type E;
  const Plan p = plan_of(rows, V, t.k);
  const float c = kLog2e / tau, scale = tau * tau;
  float* partial = ws;
  const Totals all = {loss, count, mean};
  if (p.width) {
    hipLaunchKernelGGL((small_forward_kernel<T>), dim3(p.blocks), dim3(kThreads),
                       (size_t)(kThreads / p.width) * t.k * 8, s, (const E*)x, ld, rows, V, t, c, scale, p.width,
                       stats, row_loss, partial, all);
  } else {
    float* part = nullptr;
    if (p.splits > 1) {
      part = ws + 2 * p.blocks;
      hipLaunchKernelGGL((split_stats_kernel<T>), dim3(units_of(rows, p.splits)), dim3(kThreads), 0, s, (const E*)x,
                         ld, rows, V, t, c, p.splits, p.per_split, part);
    }
    hipLaunchKernelGGL((row_forward_kernel<T>), dim3(p.blocks), dim3(kThreads), 0, s, (const E*)x, ld, rows, V, t, c,
                       scale, part, p.splits, stats, row_loss, partial, all);
  }
  if (p.blocks > 1) hipLaunchKernelGGL(totals_kernel, dim3(1), dim3(1024), 0, s, partial, p.blocks, all);
  return pv2::check_launch("topk_distill_forward");
}

template <typename T>
int backward(const void* x, int64_t ld, int64_t rows, int V, const Teacher& t, float tau, const Scale& scale,
             const float* stats, void* dx, hipStream_t s) {
  typedef typename T::type E;
  const Plan p = plan_of(rows, V, t.k);
  const float c = kLog2e / tau;
  if (p.width)
    hipLaunchKernelGGL((small_backward_kernel<T>), dim3(p.blocks), dim3(kThreads),
                       (size_t)(kThreads / p.width) * t.k * 8, s, (const E*)x, ld, rows, V, t, c, scale, p.width,
                       stats, (E*)dx);
  else
    hipLaunchKernelGGL((row_backward_kernel<T>), dim3(units_of(rows, p.splits)), dim3(kThreads), 0, s, (const E*)x, ld,
                       rows, V, t, c, scale, p.splits, p.per_split, stats, (E*)dx);
  return pv2::check_launch("topk_distill_backward");
}

int check_shapes(int64_t rows, int V, int64_t ld, int teacher_dtype, int k, float tau) {
  PV2_REQUIRE(rows > 0 && V > 0 && ld >= 0, "topk_distill: bad shape");
  PV2_REQUIRE(k >= 1 && k <= kMaxTop, "topk_distill: 1 to 1024 listed classes");
  PV2_REQUIRE(teacher_dtype >= PV2_F32 && teacher_dtype <= PV2_F16, "topk_distill: bad element type");
  PV2_REQUIRE(tau >= kMinTau && tau <= kMaxTau, "topk_distill: temperature out of range");
  return PV2_OK;
}

}  // namespace

extern "C" {

int64_t pv2_topk_distill_workspace_floats(int64_t rows, int classes, int k) {
  if (rows <= 0 || classes <= 0 || k < 1 || k > kMaxTop) return 1;
  const Plan p = plan_of(rows, classes, k);
  return 2 * (int64_t)p.blocks + (p.splits > 1 ? 2 * rows * p.splits : 0);
}

int pv2_topk_distill_forward(const void* logits, int dtype, int64_t rows, int classes, int64_t row_stride,
                             const void* teacher_index, int index_is_64, int64_t index_stride,
                             const void* teacher_logits, int teacher_dtype, int64_t teacher_stride, int k,
                             float temperature, int mean, float* workspace, float* stats, float* row_loss_or_null,
                             float* loss, float* count, pv2_stream_t stream) {
  PV2_REQUIRE(logits && teacher_index && teacher_logits && workspace && stats && loss && count,
              "topk_distill_forward: null pointer");
  const int st = check_shapes(rows, classes, row_stride, teacher_dtype, k, temperature);
  if (st != PV2_OK) return st;
  const Teacher t = {teacher_index, index_is_64, teacher_logits, teacher_dtype, k, index_stride, teacher_stride};
  hipStream_t s = (hipStream_t)stream;
  switch (dtype) {
    case PV2_F32:
      return forward<F32>(logits, row_stride, rows, classes, t, temperature, mean, stats, row_loss_or_null, loss, count,
                          workspace, s);
    case PV2_BF16:
      return forward<B16>(logits, row_stride, rows, classes, t, temperature, mean, stats, row_loss_or_null, loss, count,
                          workspace, s);
    case PV2_F16:
      return forward<H16>(logits, row_stride, rows, classes, t, temperature, mean, stats, row_loss_or_null, loss, count,
                          workspace, s);
  }
  PV2_REQUIRE(false, "topk_distill_forward: bad element type");
}

int pv2_topk_distill_backward(const void* logits, int dtype, int64_t rows, int classes, int64_t row_stride,
                              const void* teacher_index, int index_is_64, int64_t index_stride,
                              const void* teacher_logits, int teacher_dtype, int64_t teacher_stride, int k,
                              float temperature, const float* stats, const float* upstream, int upstream_per_row,
                              const float* count_or_null, void* grad_logits, pv2_stream_t stream) {
  PV2_REQUIRE(logits && teacher_index && teacher_logits && stats && upstream && grad_logits,
              "topk_distill_backward: null pointer");
  const int st = check_shapes(rows, classes, row_stride, teacher_dtype, k, temperature);
  if (st != PV2_OK) return st;
  const Teacher t = {teacher_index, index_is_64, teacher_logits, teacher_dtype, k, index_stride, teacher_stride};
  const Scale scale = {upstream, upstream_per_row, count_or_null, temperature};
  hipStream_t s = (hipStream_t)stream;
  switch (dtype) {
    case PV2_F32: return backward<F32>(logits, row_stride, rows, classes, t, temperature, scale, stats, grad_logits, s);
    case PV2_BF16: return backward<B16>(logits, row_stride, rows, classes, t, temperature, scale, stats, grad_logits, s);
    case PV2_F16: return backward<H16>(logits, row_stride, rows, classes, t, temperature, scale, stats, grad_logits, s);
  }
  PV2_REQUIRE(false, "topk_distill_backward: bad element type");
}

}  // extern "C"
