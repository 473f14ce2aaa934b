// rebel_amd/csrc/layer_norm_kernel.h -- kernels of layer normalisation, forward and backward, with an optional GELU behind it.
//
// Row x of n values, weight w, bias b, eps e:
//     m = sum x / n     v = sum (x - m)^2 / n     r = 1 / sqrt(v + e)     h = (x - m) r     z = h w + b
//     y = z,  or  y = z Phi(z) with the normal distribution Phi (GELU)
// and, with g = dy (GELU: g = dy (Phi(z) + z phi(z)), phi the density):
//     db = sum_rows g     dw = sum_rows g h     dx = r (g w - sum(g w) / n - h sum(g w h) / n)
//
// h is computed again from x and the two statistics of the row, so nothing else is kept between the passes.
//
// Large tensors are bound by memory, but for 16-bit rows with GELU.  Counted in the loops over the rows (bf16, branches and
// all), an element takes 14 to 20 issue slots forward and 16 to 28 backward; with GELU, whose exponential and reciprocal count fourfold,
// 38 to 44 and 47 to 66.  At 39 T lane slots a second (256 CUs, 64 lanes, 2.4 GHz) f32 + GELU hides behind the memory.  16-bit rows
// + GELU do not.  bf16, us, with GELU / the time of its slots / without GELU:
//     forward     8192 x 4096 39 / 36 / 27    8192 x 12000 122 / 110 / 80    65536 x 1280 125 / 92 / 62
//     backward    8192 x 4096 49 / 48 / 38    8192 x 12000 202 / 122 / 142    65536 x 1280 187 / 128 / 115
// What goes beyond the slots in the two widths that are no power of two: threads past the row's end (27 and 37 % of them) take part in
// the statistics, and backward two wavefronts to a SIMD have to cover the chains through exponential and reciprocal.
//
// So a row is read once and stays in registers, and a thread has as many of its elements as fit there: what is done once per row
// and thread (two sums over the group, the statistics) is then done least often.
//
// Times here and in layer_norm.h: rocprofv3's durations of the kernels, median of 30 passes over three sets of inputs in turn; "back to
// back": 200 calls of the C entry with nothing between them.
//
// The element types are compiled apart (layer_norm_f32.hip, layer_norm_f16.hip, layer_norm_bf16.hip); layer_norm.hip holds the C
// entries.
#pragma once
#include <algorithm>

#include "layer_norm.h"

namespace rbl {
namespace {

// Phi(z) and exp(-z^2 / 2).  For x = |z|: Phi(-x) = exp(-x^2 / 2) P(x) with P(x) = exp(x^2 / 2) erfc(x / sqrt 2) / 2, which
// falls smoothly from 1/2 like 1 / (x sqrt(2 pi)): a polynomial of degree 8 in u = 1 / (1 + 0.3 x) without a constant term
// (the form of Abramowitz and Stegun 7.1.26; coefficients from scripts/fit_normal_cdf.py, least relative error on [0, 14]:
// 1.5e-7 exactly, 4.3e-7 in f32).  The error is RELATIVE on the negative side too, where 1 + erf would cancel, and the exponential is
// the one that the derivative needs.  NaN stays NaN; +-inf give 1 and 0.
__device__ __forceinline__ float normal_cdf(float z, float* density_exp) {
  const float x = __builtin_fabsf(z);
  const float e = __builtin_amdgcn_exp2f(-0.72134752f * z * z);  // log2(e) / 2
  const float u = __builtin_amdgcn_rcpf(__builtin_fmaf(0.3f, x, 1.0f));
  float p = 3.567482242e-02f;
  p = __builtin_fmaf(p, u, -1.572032768e-01f);
  p = __builtin_fmaf(p, u, 2.063538244e-01f);
  p = __builtin_fmaf(p, u, -5.368391779e-02f);
  p = __builtin_fmaf(p, u, 1.285617593e-01f);
  p = __builtin_fmaf(p, u, 9.991345601e-02f);
  p = __builtin_fmaf(p, u, 1.207539611e-01f);
  p = __builtin_fmaf(p, u, 1.196292985e-01f);
  const float tail = p * u * e;
  *density_exp = e;
  return z > 0 ? 1.0f - tail : tail;
}

template <int ACT>
__device__ __forceinline__ float activate(float z) {
  if (ACT == RBL_ACT_NONE) return z;
  float e;
  const float phi = normal_cdf(z, &e);
  return z * phi;
}

// d activate / d z
template <int ACT>
__device__ __forceinline__ float activate_slope(float z) {
  if (ACT == RBL_ACT_NONE) return 1.0f;
  float e;
  const float phi = normal_cdf(z, &e);
  return __builtin_fmaf(z * 0.39894228f, e, phi);  // 1 / sqrt(2 pi)
}

template <class T>
__device__ __forceinline__ void put_param(const NormArgs& a, void* p, int col, float v) {
  if (a.param_f32)
    ((float*)p)[col] = v;
  else
    ((T*)p)[col] = (T)v;
}

// V consecutive elements in one access: 16 bytes, at the alignment of an element (the memory pipe takes any).
template <class T, int V>
struct Pack {
  typedef T type __attribute__((ext_vector_type(V), aligned(sizeof(T))));
};

// Which columns a thread of a row's group owns.  Vector v covers [v V, v V + V); the one that would reach past the row is moved
// back to end with it and leaves out (`skip`) what the vector before it owns already, so every load is a whole one and none needs
// a branch.  A vector that lies wholly past the row skips everything.
// The kernels for 8 threads and more are called for rows of more than half their capacity: the first half of a thread's vectors
// needs no such care.
template <int V, int TPR, int K, bool EVEN>
struct Place {
  int col, skip;
  bool busy;  // some lane of the wavefront owns something: the others leave its arithmetic out
  static __device__ __forceinline__ constexpr bool whole(int k) { return EVEN || (TPR >= 8 && 2 * k + 2 <= K); }
  Place() = default;
  __device__ __forceinline__ Place(int t, int k, int cols) {
    const int at = (t + k * TPR) * V;
    col = whole(k) || at + V <= cols ? at : cols - V;
    skip = whole(k) ? 0 : at - col;
    busy = whole(k) || __builtin_amdgcn_readfirstlane(at) < cols;
  }
  __device__ __forceinline__ bool owns(int k, int i) const { return whole(k) || i >= skip; }
};

// Stores the elements that a thread owns.  A moved-back vector stores its own alone: what it has computed for its neighbour's
// may differ in the last bit, since the compiler need not round the same way at another place of the vector.
template <class T, int V, bool EVEN, bool STREAM>
__device__ __forceinline__ void put_row(T* out, typename Pack<T, V>::type v, int skip) {
  typedef typename Pack<T, V>::type vec;
  if (EVEN || skip == 0) {
    if (STREAM)
      __builtin_nontemporal_store(v, (vec*)out);
    else
      *(vec*)out = v;
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i >= skip) out[i] = v[i];
  }
}

// A row's vectors.  STREAM: without a claim to the caches, for tensors that they cannot hold anyway.
template <class T, int V, bool STREAM, class PLACE, int K>
__device__ __forceinline__ void load_row(typename Pack<T, V>::type (&v)[K], const void* base, int64_t offset, const PLACE (&at)[K]) {
  typedef typename Pack<T, V>::type vec;
  const T* row = (const T*)base + offset;
#pragma unroll
  for (int k = 0; k < K; ++k)
    v[k] = STREAM ? __builtin_nontemporal_load((const vec*)(row + at[k].col)) : *(const vec*)(row + at[k].col);
}

template <class T, int V>
__device__ __forceinline__ void load_params(const NormArgs& a, const void* p, int col, float missing, float (&out)[V]) {
  if (!p) {
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = missing;
  } else if (a.param_f32) {
    const auto v = *(const typename Pack<float, V>::type*)((const float*)p + col);
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = v[i];
  } else {
    const auto v = *(const typename Pack<T, V>::type*)((const T*)p + col);
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = (float)v[i];
  }
}

// Sums of N numbers over the TPR threads that share a row, the same bits in each of them.  Groups of up to 64 stay in their
// wavefront; larger ones (whole workgroups) exchange one number per wavefront through LDS.  Two buffers in turn make one barrier
// per call enough: a wavefront can be at most one call ahead of another.
template <int TPR, int N>
__device__ __forceinline__ void sum_group(float (&v)[N], float* slots, int& turn) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if constexpr (TPR < 64) v[i] = sum_lanes<TPR>(v[i]);
    else v[i] = sum64(v[i]);
  }
  if constexpr (TPR > 64) {
    constexpr int W = TPR / 64;
    float* s = slots + turn * 2 * W;
    turn ^= 1;
    if (threadIdx.x % 64 == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) s[i * W + threadIdx.x / 64] = v[i];
    }
    lds_barrier();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float t = s[i * W];
#pragma unroll
      for (int w = 1; w < W; ++w) t += s[i * W + w];
      v[i] = t;
    }
  }
}

// 1 / sqrt(variance + eps) to two units in the last place; the instruction takes no subnormal numbers, so small ones are scaled.
__device__ __forceinline__ float inverse_deviation(float variance, float eps) {
  const float v = (variance < 0 ? 0 : variance) + eps;  // NaN stays
  const bool small = v < 0x1p-96f;
  return __builtin_amdgcn_rsqf(small ? v * 0x1p64f : v) * (small ? 0x1p32f : 1.0f);
}

// Mean and 1 / sqrt(variance + eps) of the row whose elements the group's threads hold.  The variance is the mean square of
// the deviations from the rounded mean; their sum, which would be zero but for that rounding, corrects both.
template <int V, int TPR, int K, bool EVEN>
__device__ __forceinline__ void statistics(const float (&x)[K][V], const Place<V, TPR, K, EVEN> (&at)[K], float inv_n, float eps,
                                           float* slots, int& turn, float& mean, float& r) {
  float s[1] = {0};
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) s[0] += at[k].owns(k, i) ? x[k][i] : 0.0f;
  sum_group<TPR>(s, slots, turn);
  const float first = s[0] * inv_n;
  float d[2] = {0, 0};
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float e = at[k].owns(k, i) ? x[k][i] - first : 0.0f;
      d[0] += e;
      d[1] = __builtin_fmaf(e, e, d[1]);
    }
  sum_group<TPR>(d, slots, turn);
  const float off = d[0] * inv_n;
  mean = first + off;
  r = inverse_deviation(__builtin_fmaf(-off, d[0], d[1]) * inv_n, eps);
}

// Workgroup size: groups within a wavefront share workgroups of four, larger groups are workgroups.
template <int TPR>
constexpr int forward_threads() { return TPR <= 64 ? 256 : TPR; }

// Forward, a row in the registers of TPR threads (K vectors of V elements each): read once, written once.  As many workgroups as
// the chip holds, each with the same number of rows, the parameters in registers and the next row on its way.  Bound by memory:
// 270336 x 256 f32 + GELU 103 us (5.4 TB/s; with 4 elements to a thread instead of 16 it was 149), 8192 x 4096 bf16 23.4 us (5.7),
// 32768 x 8192 bf16 178 us (6.0).  One row of 256: 2.6 us, a load, two sums and a store one after the other.
template <class T, int V, int TPR, int K, bool EVEN, int ACT, bool STREAM>
__global__ __launch_bounds__(forward_threads<TPR>()) void layer_norm_forward_kernel(NormArgs a) {
  constexpr int NT = forward_threads<TPR>(), RPB = NT / TPR;
  typedef typename Pack<T, V>::type vec;
  __shared__ float slots[TPR > 64 ? 4 * TPR / 64 : 1];
  int turn = 0;
  const int t = threadIdx.x % TPR;
  Place<V, TPR, K, EVEN> at[K];
  const int64_t step = (int64_t)gridDim.x * RPB;
  int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR;
  if (row >= a.rows) return;  // whole groups; of a group of more than a wavefront there is one to a workgroup
  constexpr bool KEEP = K * V <= 16;  // the parameters stay in registers
  float w[K][V], b[K][V];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    at[k] = Place<V, TPR, K, EVEN>(t, k, a.cols);
    if (KEEP) {
      load_params<T, V>(a, a.w, at[k].col, 1.0f, w[k]);
      load_params<T, V>(a, a.b, at[k].col, 0.0f, b[k]);
    }
  }
  constexpr bool AHEAD = K * V <= 16;  // the next row is on its way while one is computed
  vec next[K];
  if (AHEAD) load_row<T, V, STREAM>(next, a.x, row * a.x_stride, at);
  for (; row < a.rows; row += step) {
    if (!AHEAD) load_row<T, V, STREAM>(next, a.x, row * a.x_stride, at);
    float x[K][V];
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        x[k][i] = (float)next[k][i];
        if (!AHEAD) asm("" : "+v"(x[k][i]));  // not both the packed and the unpacked row: there is no room
      }
    const int64_t ahead = row + step < a.rows ? row + step : row;
    if (AHEAD) load_row<T, V, STREAM>(next, a.x, ahead * a.x_stride, at);
    float mean, r;
    statistics<V, TPR, K, EVEN>(x, at, a.inv_cols, a.eps, slots, turn, mean, r);
    T* y = (T*)a.y + row * a.cols;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (!at[k].busy) continue;
      if (!KEEP) {
        __builtin_amdgcn_sched_barrier(0);  // not all of the parameters at once: they would spill
        load_params<T, V>(a, a.w, at[k].col, 1.0f, w[k]);
        load_params<T, V>(a, a.b, at[k].col, 0.0f, b[k]);
      }
      vec out;
#pragma unroll
      for (int i = 0; i < V; ++i) out[i] = (T)activate<ACT>(__builtin_fmaf((x[k][i] - mean) * r, w[k][i], b[k][i]));
      put_row<T, V, EVEN, STREAM>(y + at[k].col, out, at[k].skip);
    }
    if (a.stats && t == 0) *(float2*)(a.stats + 2 * row) = make_float2(mean, r);
  }
}

// Rows that are longer than a workgroup's registers: chunks of kChunkK vectors to a thread, each with its own mean and sum of
// squared deviations, which the second kernel joins (Chan's formula) before it normalises its chunk.  x is read twice: 2000 x 65537
// f32 109 + 192 us (5.2 TB/s of three passes), 24 x 65537 4.1 + 5.8 us.  Batches of rows small enough for the second reading to come
// from the 256 MB cache were not faster (4096 x 65537: 608 us in one, 626 in batches of 128 MB).
template <int V>
constexpr int chunk_cols() { return kThreads * kChunkK * V; }

template <class T, int V>
__global__ __launch_bounds__(kThreads) void layer_norm_chunk_statistics_kernel(NormArgs a) {
  typedef typename Pack<T, V>::type vec;
  __shared__ float slots[4 * kThreads / 64];
  int turn = 0;
  for (int64_t item = blockIdx.x; item < a.rows * a.chunks; item += gridDim.x) {
    const int64_t row = item / a.chunks;
    const int chunk = (int)(item - row * a.chunks), begin = chunk * chunk_cols<V>();
    const int cols = min(a.cols - begin, chunk_cols<V>());
    const T* x = (const T*)a.x + row * a.x_stride + begin;
    float s[1] = {0}, e[2] = {0, 0};
    float v[kChunkK][V];
    bool own[kChunkK][V];
#pragma unroll
    for (int k = 0; k < kChunkK; ++k) {
      // the last chunk may be shorter than a vector: it reads back into the one before
      const int at = (threadIdx.x + k * kThreads) * V, col = at + V <= cols ? at : cols - V;
      const vec p = *(const vec*)(x + col);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        own[k][i] = i >= at - col;
        v[k][i] = own[k][i] ? (float)p[i] : 0.0f;
        s[0] += v[k][i];
      }
    }
    sum_group<kThreads>(s, slots, turn);
    const float n = (float)cols, first = s[0] / n;
#pragma unroll
    for (int k = 0; k < kChunkK; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float d = own[k][i] ? v[k][i] - first : 0.0f;
        e[0] += d;
        e[1] = __builtin_fmaf(d, d, e[1]);
      }
    sum_group<kThreads>(e, slots, turn);
    if (threadIdx.x == 0) *(float2*)(a.partial + 2 * item) = make_float2(first + e[0] / n, e[1] - e[0] * e[0] / n);
  }
}

// Every wavefront joins the chunks' statistics for itself.
template <int V>
__device__ __forceinline__ void join_chunks(const NormArgs& a, int64_t row, float& mean, float& r) {
  const float2* p = (const float2*)a.partial + row * a.chunks;
  const int lane = threadIdx.x % 64;
  const float pivot = p[0].x, n = (float)a.cols;
  float s = 0, q = 0;
  for (int c = lane; c < a.chunks; c += 64) s += (p[c].x - pivot) * (float)min(a.cols - c * chunk_cols<V>(), chunk_cols<V>());
  mean = pivot + sum64(s) / n;
  for (int c = lane; c < a.chunks; c += 64) {
    const float d = p[c].x - mean;
    q += __builtin_fmaf(d * d, (float)min(a.cols - c * chunk_cols<V>(), chunk_cols<V>()), p[c].y);
  }
  r = inverse_deviation(sum64(q) / n, a.eps);
}

template <class T, int V, int ACT>
__global__ __launch_bounds__(kThreads) void layer_norm_chunk_forward_kernel(NormArgs a) {
  typedef typename Pack<T, V>::type vec;
  for (int64_t item = blockIdx.x; item < a.rows * a.chunks; item += gridDim.x) {
    const int64_t row = item / a.chunks;
    const int begin = (int)(item - row * a.chunks) * chunk_cols<V>();
    const int cols = min(a.cols - begin, chunk_cols<V>());
    const T* x = (const T*)a.x + row * a.x_stride + begin;
    T* y = (T*)a.y + row * a.cols + begin;
    vec p[kChunkK];
    int col[kChunkK];
#pragma unroll
    for (int k = 0; k < kChunkK; ++k) {
      const int at = (threadIdx.x + k * kThreads) * V;
      col[k] = at + V <= cols ? at : cols - V;
      p[k] = *(const vec*)(x + col[k]);
    }
    float mean, r;
    join_chunks<V>(a, row, mean, r);
#pragma unroll
    for (int k = 0; k < kChunkK; ++k) {
      float w[V], b[V];
      load_params<T, V>(a, a.w, begin + col[k], 1.0f, w);
      load_params<T, V>(a, a.b, begin + col[k], 0.0f, b);
      vec out;
#pragma unroll
      for (int i = 0; i < V; ++i) out[i] = (T)activate<ACT>(__builtin_fmaf(((float)p[k][i] - mean) * r, w[i], b[i]));
      put_row<T, V, false, false>(y + col[k], out, (threadIdx.x + k * kThreads) * V - col[k]);
    }
    if (a.stats && begin == 0 && threadIdx.x == 0) *(float2*)(a.stats + 2 * row) = make_float2(mean, r);
  }
}

// Writes what a thread has summed up over rows for its V columns: the owned ones alone.
template <int V, bool EVEN>
__device__ __forceinline__ void put_sums(float* out, const float (&v)[V], int skip) {
  if (EVEN || skip == 0) {
    typename Pack<float, V>::type p;
#pragma unroll
    for (int i = 0; i < V; ++i) p[i] = v[i];
    *(typename Pack<float, V>::type*)out = p;
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i >= skip) out[i] = v[i];
  }
}

// Backward, a row in the registers of TPR threads: x and dy are read once, dx is written, and (SUMS) g h and g are summed up over
// the rows of the workgroup, in registers (rows of 1024 threads: in LDS, each thread its own 16-byte cells); the workgroups' sums
// are joined by layer_norm_sums_kernel.  Bound by memory: 270336 x 256 f32 + GELU 160 to 170 us behind a forward pass and
// 148 back to back (4.9 to 5.6 TB/s), 32768 x 8192 bf16 264 us (6.1), 8192 x 16384 bf16 178 to 188 us (4.3 to 4.5).  Workgroup `group` of `groups`.
template <class T, int V, int TPR, int K, bool EVEN, int ACT, bool SUMS, bool STREAM>
__device__ __forceinline__ void backward_of_rows(const NormArgs& a, int group, int groups) {
  constexpr int NT = backward_threads(TPR), RPB = NT / TPR;
  typedef typename Pack<T, V>::type vec;
  __shared__ float slots[TPR > 64 ? 4 * TPR / 64 : 1];
  __shared__ float joined[SUMS && TPR <= 64 ? 2 * TPR * K * V : 1];
  constexpr bool CELLS = SUMS && TPR == 1024;
  typedef float cell __attribute__((ext_vector_type(4)));
  __shared__ cell cells[CELLS ? 2 * K * V / 4 * TPR : 1];
  int turn = 0;
  const int t = threadIdx.x % TPR;
  Place<V, TPR, K, EVEN> at[K];
  const int64_t step = (int64_t)groups * RPB;
  int64_t row = (int64_t)group * RPB + threadIdx.x / TPR;
  constexpr bool KEEP = K * V <= 16 && TPR < 1024;
  float w[K][V], b[K][V], dw[CELLS ? 1 : K][V], db[CELLS ? 1 : K][V];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    at[k] = Place<V, TPR, K, EVEN>(t, k, a.cols);
    if (KEEP) {
      load_params<T, V>(a, a.w, at[k].col, 1.0f, w[k]);
      if (ACT != RBL_ACT_NONE) load_params<T, V>(a, a.b, at[k].col, 0.0f, b[k]);
    }
    if constexpr (CELLS) {
#pragma unroll
      for (int i = 0; i < V / 4; ++i)
        cells[(k * V / 4 + i) * TPR + t] = cells[((K + k) * V / 4 + i) * TPR + t] = cell{0, 0, 0, 0};
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) dw[k][i] = db[k][i] = 0;
    }
  }
  if (row < a.rows) {
    vec next_x[K], next_dy[K];
    float2 next_s = *(const float2*)(a.stats + 2 * row);
    constexpr bool AHEAD = TPR < 1024;  // the next row is on its way while one is computed
    // with one vector to a thread the branch costs more than it leaves out; in the largest groups with GELU there is no register for it
    constexpr bool LEAVE = K > 1 && !(TPR == 1024 && V == 8 && ACT != RBL_ACT_NONE);
    if (AHEAD) {
      load_row<T, V, STREAM>(next_x, a.x, row * a.x_stride, at);
      load_row<T, V, STREAM>(next_dy, a.dy, row * a.dy_stride, at);
    }
    for (; row < a.rows; row += step) {
      if (!AHEAD) {
        load_row<T, V, STREAM>(next_x, a.x, row * a.x_stride, at);
        load_row<T, V, STREAM>(next_dy, a.dy, row * a.dy_stride, at);
      }
      const float mean = next_s.x, r = next_s.y;
      float h[K][V], g[K][V];
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          h[k][i] = ((float)next_x[k][i] - mean) * r;
          g[k][i] = at[k].owns(k, i) ? (float)next_dy[k][i] : 0.0f;
        }
      const int64_t ahead = row + step < a.rows ? row + step : row;
      next_s = *(const float2*)(a.stats + 2 * ahead);
      if (AHEAD) {
        load_row<T, V, STREAM>(next_x, a.x, ahead * a.x_stride, at);
        load_row<T, V, STREAM>(next_dy, a.dy, ahead * a.dy_stride, at);
      }
      float s[2] = {0, 0};
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (LEAVE && !at[k].busy) continue;
        if (!KEEP) {
          __builtin_amdgcn_sched_barrier(0);
          load_params<T, V>(a, a.w, at[k].col, 1.0f, w[k]);
          if (ACT != RBL_ACT_NONE) load_params<T, V>(a, a.b, at[k].col, 0.0f, b[k]);
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
          if (ACT != RBL_ACT_NONE) g[k][i] *= activate_slope<ACT>(__builtin_fmaf(h[k][i], w[k][i], b[k][i]));
          if (SUMS && !CELLS) {
            dw[k][i] = __builtin_fmaf(g[k][i], h[k][i], dw[k][i]);
            db[k][i] += g[k][i];
          }
        }
        if constexpr (CELLS) {
#pragma unroll
          for (int i = 0; i < V / 4; ++i) {
            cell &p = cells[(k * V / 4 + i) * TPR + t], &q = cells[((K + k) * V / 4 + i) * TPR + t];
            cell u = p, v = q;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              u[j] = __builtin_fmaf(g[k][i * 4 + j], h[k][i * 4 + j], u[j]);
              v[j] += g[k][i * 4 + j];
            }
            p = u;
            q = v;
          }
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
          g[k][i] *= w[k][i];
          s[0] += g[k][i];
          s[1] = __builtin_fmaf(g[k][i], h[k][i], s[1]);
        }
      }
      if (a.dx) {
        sum_group<TPR>(s, slots, turn);
        const float p = s[0] * a.inv_cols, q = s[1] * a.inv_cols;
        T* dx = (T*)a.dx + row * a.cols;
#pragma unroll
        for (int k = 0; k < K; ++k) {
          if (LEAVE && !at[k].busy) continue;
          vec out;
#pragma unroll
          for (int i = 0; i < V; ++i) out[i] = (T)(r * (g[k][i] - __builtin_fmaf(h[k][i], q, p)));
          put_row<T, V, EVEN, STREAM>(dx + at[k].col, out, at[k].skip);
        }
      }
    }
  }
  if constexpr (SUMS) {
    const int64_t width = (a.cols + 3) / 4 * 4;
    float* out = a.partial + group * 2 * width;
    if constexpr (CELLS) {
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int which = 0; which < 2; ++which) {
          float v[V];
#pragma unroll
          for (int i = 0; i < V; ++i) v[i] = cells[((which * K + k) * V / 4 + i / 4) * TPR + t][i % 4];
          put_sums<V, EVEN>(out + which * width + at[k].col, v, at[k].skip);
        }
    } else if constexpr (TPR > 64) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        put_sums<V, EVEN>(out + at[k].col, dw[k], at[k].skip);
        put_sums<V, EVEN>(out + width + at[k].col, db[k], at[k].skip);
      }
    } else {
      // the wavefronts add their sums up one after the other
      constexpr int GROUPS = NT / 64;
#pragma unroll
      for (int d = TPR; d < 64; d *= 2)
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int i = 0; i < V; ++i) {
            dw[k][i] += __shfl_xor(dw[k][i], d);
            db[k][i] += __shfl_xor(db[k][i], d);
          }
      for (int wave = 0; wave < GROUPS; ++wave) {
        if ((int)threadIdx.x / 64 == wave && threadIdx.x % 64 < TPR) {
#pragma unroll
          for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) {
              // element i of vector v at [i][v]: consecutive lanes in consecutive banks
              float* p = joined + (k * V + i) * TPR + t;
              if (wave == 0) {
                p[0] = dw[k][i];
                p[TPR * K * V] = db[k][i];
              } else {
                p[0] += dw[k][i];
                p[TPR * K * V] += db[k][i];
              }
            }
        }
        lds_barrier();
      }
      for (int j = threadIdx.x; j < 2 * TPR * K; j += NT) {
        const int which = j / (TPR * K), v = j % (TPR * K), k = v / TPR;
        const Place<V, TPR, K, EVEN> place(v % TPR, k, a.cols);
        float sum[V];
#pragma unroll
        for (int i = 0; i < V; ++i) sum[i] = joined[which * TPR * K * V + (k * V + i) * TPR + v % TPR];
        put_sums<V, EVEN>(out + which * width + place.col, sum, place.skip);
      }
    }
  }
}

template <class T, int V, int TPR, int K, bool EVEN, int ACT, bool SUMS, bool STREAM>
__global__ __launch_bounds__(backward_threads(TPR)) void layer_norm_backward_kernel(NormArgs a) {
  backward_of_rows<T, V, TPR, K, EVEN, ACT, SUMS, STREAM>(a, blockIdx.x, gridDim.x);
}

// The parameters' gradients of few rows, straight from x and dy: 4 V columns to a workgroup, NT / 4 threads down the rows.  No
// partial sums and no second launch for them, but x and dy are read a second time.
template <class T, int V, int ACT, int NT>
__device__ __forceinline__ void backward_of_columns(const NormArgs& a, int block) {
  constexpr int LANES = 4, SLICES = NT / LANES, AHEAD = 4;
  typedef typename Pack<T, V>::type vec;
  __shared__ float part[NT / 64][2][LANES * V];
  const int lane = threadIdx.x % LANES, slice = threadIdx.x / LANES;
  // as in Place: the last vector is moved back to end with the row
  const int begin = (block * LANES + lane) * V, col = begin + V <= a.cols ? begin : a.cols - V, skip = begin - col;
  float w[V], b[V], dw[V], db[V];
  if (ACT != RBL_ACT_NONE) {
    load_params<T, V>(a, a.w, col, 1.0f, w);
    load_params<T, V>(a, a.b, col, 0.0f, b);
  }
#pragma unroll
  for (int i = 0; i < V; ++i) dw[i] = db[i] = 0;
  for (int64_t row = slice; row < a.rows; row += SLICES * AHEAD) {
    vec x[AHEAD], dy[AHEAD];
    float2 st[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {  // behind the last row: row again, and its gradient is left out
      const int64_t r = row + k * SLICES < a.rows ? row + k * SLICES : row;
      x[k] = *(const vec*)((const T*)a.x + r * a.x_stride + col);
      dy[k] = *(const vec*)((const T*)a.dy + r * a.dy_stride + col);
      st[k] = *(const float2*)(a.stats + 2 * r);
    }
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      if (k > 0 && row + k * SLICES >= a.rows) break;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float h = ((float)x[k][i] - st[k].x) * st[k].y;
        float g = (float)dy[k][i];
        if (ACT != RBL_ACT_NONE) g *= activate_slope<ACT>(__builtin_fmaf(h, w[i], b[i]));
        dw[i] = __builtin_fmaf(g, h, dw[i]);
        db[i] += g;
      }
    }
  }
#pragma unroll
  for (int d = LANES; d < 64; d *= 2)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      dw[i] += __shfl_xor(dw[i], d);
      db[i] += __shfl_xor(db[i], d);
    }
  if (threadIdx.x % 64 < LANES) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      part[threadIdx.x / 64][0][lane * V + i] = dw[i];
      part[threadIdx.x / 64][1][lane * V + i] = db[i];
    }
  }
  lds_barrier();
  for (int j = threadIdx.x; j < 2 * LANES * V; j += NT) {
    const int which = j / (LANES * V), c = j % (LANES * V);
    float v = part[0][which][c];
#pragma unroll
    for (int wave = 1; wave < NT / 64; ++wave) v += part[wave][which][c];
    const int at = (block * LANES + c / V) * V, first = at + V <= a.cols ? at : a.cols - V;
    if (c % V >= at - first) {
      if (which == 0 && a.dw) put_param<T>(a, a.dw, first + c % V, v);
      if (which == 1 && a.db) put_param<T>(a, a.db, first + c % V, v);
    }
  }
}

// Few rows, in one launch: the first `row_groups` workgroups make dx, the others the parameters' gradients.
template <class T, int V, int TPR, int K, bool EVEN, int ACT>
__global__ __launch_bounds__(backward_threads(TPR)) void layer_norm_backward_few_kernel(NormArgs a, int row_groups) {
  if ((int)blockIdx.x < row_groups)
    backward_of_rows<T, V, TPR, K, EVEN, ACT, false, false>(a, blockIdx.x, row_groups);
  else
    backward_of_columns<T, V, ACT, backward_threads(TPR)>(a, blockIdx.x - row_groups);
}

// The parameters' gradients from `count` rows of partial sums, each [2][width]: COLS columns to a workgroup, the other threads
// down the rows, in an order that depends on the counts alone.  16 columns where there are few (64-byte accesses, but four times
// the workgroups), else 64.
constexpr int kSumsThreads = 1024;
template <class T, int COLS>
__global__ __launch_bounds__(kSumsThreads) void layer_norm_sums_kernel(NormArgs a, int count) {
  constexpr int LANES = COLS / 4, SLICES = kSumsThreads / LANES;
  __shared__ float part[kSumsThreads / 64][COLS];
  const int width = (a.cols + 3) / 4 * 4;
  const int quad = threadIdx.x % LANES, slice = threadIdx.x / LANES;
  typedef Pack<float, 4>::type vec;
  for (int64_t first = (int64_t)blockIdx.x * COLS; first < 2 * (int64_t)width; first += (int64_t)gridDim.x * COLS) {
    const int64_t col = first + quad * 4;
    float s[4] = {0, 0, 0, 0};
    if (col < 2 * (int64_t)width) {
#pragma unroll 4
      for (int g = slice; g < count; g += SLICES) {
        const vec v = *(const vec*)(a.partial + (int64_t)g * 2 * width + col);
#pragma unroll
        for (int i = 0; i < 4; ++i) s[i] += v[i];
      }
    }
#pragma unroll
    for (int d = LANES; d < 64; d *= 2)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[i] += __shfl_xor(s[i], d);
    if (threadIdx.x % 64 < LANES) {
#pragma unroll
      for (int i = 0; i < 4; ++i) part[threadIdx.x / 64][quad * 4 + i] = s[i];
    }
    lds_barrier();
    const int64_t mine = first + threadIdx.x;
    if (threadIdx.x < COLS && mine < 2 * (int64_t)width) {
      float v = part[0][threadIdx.x];
#pragma unroll
      for (int k = 1; k < kSumsThreads / 64; ++k) v += part[k][threadIdx.x];
      const bool second = mine >= width;
      const int c = (int)(mine - (second ? width : 0));
      if (c < a.cols) {
        if (second && a.db) put_param<T>(a, a.db, c, v);
        if (!second && a.dw) put_param<T>(a, a.dw, c, v);
      }
    }
    lds_barrier();  // part is written again
  }
}

// Longer rows, in chunks: first the chunks' shares of sum(g w) and sum(g w h) ...
template <class T, int V, int ACT>
__global__ __launch_bounds__(kThreads) void layer_norm_chunk_backward_sums_kernel(NormArgs a) {
  typedef typename Pack<T, V>::type vec;
  __shared__ float slots[4 * kThreads / 64];
  int turn = 0;
  for (int64_t item = blockIdx.x; item < a.rows * a.chunks; item += gridDim.x) {
    const int64_t row = item / a.chunks;
    const int begin = (int)(item - row * a.chunks) * chunk_cols<V>();
    const int cols = min(a.cols - begin, chunk_cols<V>());
    const T *x = (const T*)a.x + row * a.x_stride + begin, *dy = (const T*)a.dy + row * a.dy_stride + begin;
    const float2 st = *(const float2*)(a.stats + 2 * row);
    float s[2] = {0, 0};
#pragma unroll
    for (int k = 0; k < kChunkK; ++k) {
      const int at = (threadIdx.x + k * kThreads) * V, col = at + V <= cols ? at : cols - V;
      const vec xs = *(const vec*)(x + col), ds = *(const vec*)(dy + col);
      float w[V], b[V];
      load_params<T, V>(a, a.w, begin + col, 1.0f, w);
      if (ACT != RBL_ACT_NONE) load_params<T, V>(a, a.b, begin + col, 0.0f, b);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float h = ((float)xs[i] - st.x) * st.y;
        float g = i >= at - col ? (float)ds[i] : 0.0f;
        if (ACT != RBL_ACT_NONE) g *= activate_slope<ACT>(__builtin_fmaf(h, w[i], b[i]));
        g *= w[i];
        s[0] += g;
        s[1] = __builtin_fmaf(g, h, s[1]);
      }
    }
    sum_group<kThreads>(s, slots, turn);
    if (threadIdx.x == 0) *(float2*)(a.row_sums + 2 * item) = make_float2(s[0], s[1]);
  }
}

// ... then dx, and the parameters' gradients summed up over every `slices`-th row of a chunk.  x and dy are read twice: 2000 x 65537
// f32 562 us for both kernels (4.7 TB/s of five passes).
template <class T, int V, int ACT, bool SUMS>
__device__ __forceinline__ void backward_of_chunk(const NormArgs& a, int block, int slices) {
  typedef typename Pack<T, V>::type vec;
  const int chunk = block % a.chunks, slice = block / a.chunks;
  const int begin = chunk * chunk_cols<V>(), cols = min(a.cols - begin, chunk_cols<V>());
  int col[kChunkK], skip[kChunkK];
  float dw[kChunkK][V], db[kChunkK][V];
#pragma unroll
  for (int k = 0; k < kChunkK; ++k) {
    const int at = (threadIdx.x + k * kThreads) * V;
    col[k] = begin + (at + V <= cols ? at : cols - V);
    skip[k] = begin + at - col[k];
#pragma unroll
    for (int i = 0; i < V; ++i) dw[k][i] = db[k][i] = 0;
  }
  for (int64_t row = slice; row < a.rows; row += slices) {
    vec xs[kChunkK], ds[kChunkK];
#pragma unroll
    for (int k = 0; k < kChunkK; ++k) {
      xs[k] = *(const vec*)((const T*)a.x + row * a.x_stride + col[k]);
      ds[k] = *(const vec*)((const T*)a.dy + row * a.dy_stride + col[k]);
    }
    const float2 st = *(const float2*)(a.stats + 2 * row);
    float p = 0, q = 0;
    if (a.dx) {
      const float2* s = (const float2*)a.row_sums + row * a.chunks;
      for (int c = threadIdx.x % 64; c < a.chunks; c += 64) {
        p += s[c].x;
        q += s[c].y;
      }
      p = sum64(p) / (float)a.cols;
      q = sum64(q) / (float)a.cols;
    }
    T* dx = (T*)a.dx + row * a.cols;
#pragma unroll
    for (int k = 0; k < kChunkK; ++k) {
      float w[V], b[V];
      load_params<T, V>(a, a.w, col[k], 1.0f, w);
      if (ACT != RBL_ACT_NONE) load_params<T, V>(a, a.b, col[k], 0.0f, b);
      vec out;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float h = ((float)xs[k][i] - st.x) * st.y;
        float g = (float)ds[k][i];
        if (ACT != RBL_ACT_NONE) g *= activate_slope<ACT>(__builtin_fmaf(h, w[i], b[i]));
        if (SUMS) {
          dw[k][i] = __builtin_fmaf(g, h, dw[k][i]);
          db[k][i] += g;
        }
        out[i] = (T)(st.y * (g * w[i] - __builtin_fmaf(h, q, p)));
      }
      if (a.dx) put_row<T, V, false, false>(dx + col[k], out, skip[k]);
    }
  }
  if constexpr (SUMS) {
    const int64_t width = (a.cols + 3) / 4 * 4;
    float* out = a.partial + slice * 2 * width;
#pragma unroll
    for (int k = 0; k < kChunkK; ++k) {
      put_sums<V, false>(out + col[k], dw[k], skip[k]);
      put_sums<V, false>(out + width + col[k], db[k], skip[k]);
    }
  }
}

// A tensor of this size leaves little in the cache of 256 MB that its next reader could use.  bf16 rows of 4096, past the caches
// against through them, us, forward with an elementwise pass over the result behind it, and backward:
//     64 MB   52 / 49, 38 / 37       128 MB   96 / 94, 72 / 80      192 MB   145 / 145, 104 / 120
//    256 MB  202 / 202, 138 / 156    384 MB  297 / 308, 200 / 226    512 MB   400 / 408, 267 / 298
// (32768 x 8192, 512 MB: 397 / 398, 274 / 303.)  Forward, the reader pays for it up to 256 MB.  Backward it pays from 128 MB on by itself,
// which this one threshold leaves; what reads dx was not timed.
constexpr int64_t kStreamBytes = (int64_t)512 << 20;
template <class T>
bool beyond_caches(const NormArgs& a) { return a.rows * a.cols * (int64_t)sizeof(T) >= kStreamBytes; }

template <class T, int V, int ACT, bool SUMS>
__global__ __launch_bounds__(kThreads) void layer_norm_chunk_backward_kernel(NormArgs a, int slices) {
  backward_of_chunk<T, V, ACT, SUMS>(a, blockIdx.x, slices);
}
// As layer_norm_backward_few_kernel; `slices` rows at a time.
template <class T, int V, int ACT>
__global__ __launch_bounds__(kThreads) void layer_norm_chunk_backward_few_kernel(NormArgs a, int slices) {
  const int row_groups = slices * a.chunks;
  if ((int)blockIdx.x < row_groups)
    backward_of_chunk<T, V, ACT, false>(a, blockIdx.x, slices);
  else
    backward_of_columns<T, V, ACT, kThreads>(a, blockIdx.x - row_groups);
}

int resident_groups(const void* kernel, int threads) {
  int n = 0;
  if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads, 0) != hipSuccess || n < 1)
    throw std::runtime_error("HIP error: occupancy of a kernel");
  return n * kCus;
}

template <class T, int V, int TPR, int K, bool EVEN, int ACT, bool STREAM>
void forward_launch(NormArgs a, hipStream_t st) {
  constexpr int NT = forward_threads<TPR>(), RPB = NT / TPR;
  const void* kernel = (const void*)layer_norm_forward_kernel<T, V, TPR, K, EVEN, ACT, STREAM>;
  static const int resident = resident_groups(kernel, NT);
  void* args[] = {&a};
  launch(kernel, even_grid((a.rows + RPB - 1) / RPB, resident), NT, args, st);
}
template <class T, int V, int TPR, int K, int ACT>
void forward_rows(const NormArgs& a, hipStream_t st) {
  const bool even = a.cols == TPR * K * V;
  if constexpr (TPR >= 16) {
    if (beyond_caches<T>(a))
      return even ? forward_launch<T, V, TPR, K, true, ACT, true>(a, st) : forward_launch<T, V, TPR, K, false, ACT, true>(a, st);
  }
  even ? forward_launch<T, V, TPR, K, true, ACT, false>(a, st) : forward_launch<T, V, TPR, K, false, ACT, false>(a, st);
}

template <class T, int ACT>
void run_forward(NormArgs a, hipStream_t st) {
  constexpr int V = 16 / sizeof(T);
  if (a.rows == 0) return;
  // 16 elements to a thread: fewer leave too much of the work on a row's two sums, more spill out of the registers
  constexpr int K = 16 / V;
  if (a.cols < V) return forward_launch<T, 1, 4, 2, false, ACT, false>(a, st);
  if (a.cols <= 64) return forward_rows<T, V, 4, K, ACT>(a, st);
  if (a.cols <= 128) return forward_rows<T, V, 8, K, ACT>(a, st);
  if (a.cols <= 256) return forward_rows<T, V, 16, K, ACT>(a, st);
  if (a.cols <= 512) return forward_rows<T, V, 32, K, ACT>(a, st);
  if (a.cols <= 1024) return forward_rows<T, V, 64, K, ACT>(a, st);
  if (a.cols <= 2048) return forward_rows<T, V, 128, K, ACT>(a, st);
  if (a.cols <= 4096) return forward_rows<T, V, 256, K, ACT>(a, st);
  if (a.cols <= 8192) return forward_rows<T, V, 512, K, ACT>(a, st);
  if (a.cols <= 16384) return forward_rows<T, V, 1024, K, ACT>(a, st);
  if (a.cols <= kForwardCols) return forward_rows<T, V, 1024, 2 * K, ACT>(a, st);
  a.chunks = chunks_of_row(a.cols, V);
  const int64_t items = a.rows * a.chunks;
  const unsigned grid = (unsigned)(items < 1 << 20 ? items : 1 << 20);
  void* args[] = {&a};
  launch((const void*)layer_norm_chunk_statistics_kernel<T, V>, grid, kThreads, args, st);
  launch((const void*)layer_norm_chunk_forward_kernel<T, V, ACT>, grid, kThreads, args, st);
}

template <class T, int V, int TPR, int K, int ACT>
void backward_rows(NormArgs a, const BackwardPlan& p, bool sums, hipStream_t st) {
  const bool even = V > 1 && a.cols == TPR * K * V;  // V = 1: rows of fewer elements than a vector has
  if (sums && p.few) {
    int row_groups = a.dx ? (int)p.groups : 0;
    void* args[] = {&a, &row_groups};
    launch(even ? (const void*)layer_norm_backward_few_kernel<T, V, TPR, K, (V > 1), ACT>
                : (const void*)layer_norm_backward_few_kernel<T, V, TPR, K, false, ACT>,
           (unsigned)(row_groups + (a.cols + 4 * V - 1) / (4 * V)), backward_threads(TPR), args, st);
    return;
  }
  const void* kernel = sums ? even ? (const void*)layer_norm_backward_kernel<T, V, TPR, K, (V > 1), ACT, true, false>
                                   : (const void*)layer_norm_backward_kernel<T, V, TPR, K, false, ACT, true, false>
                       : even ? (const void*)layer_norm_backward_kernel<T, V, TPR, K, (V > 1), ACT, false, false>
                              : (const void*)layer_norm_backward_kernel<T, V, TPR, K, false, ACT, false, false>;
  if constexpr (TPR >= 16) {
    if (sums && beyond_caches<T>(a))
      kernel = even ? (const void*)layer_norm_backward_kernel<T, V, TPR, K, true, ACT, true, true>
                    : (const void*)layer_norm_backward_kernel<T, V, TPR, K, false, ACT, true, true>;
  }
  void* args[] = {&a};
  launch(kernel, (unsigned)p.groups, backward_threads(TPR), args, st);
}

template <class T, int ACT>
void run_backward(NormArgs a, const BackwardPlan& p, hipStream_t st) {
  // 8 elements to a thread, 16 in the widest rows: x, dy, the parameters and both sums have to fit into its registers
  constexpr int V = 16 / sizeof(T), K = 8 / V;
  const bool sums = a.dw || a.db;
  if (a.rows > 0 && (a.dx || sums)) {
    if (a.cols < V) backward_rows<T, 1, 4, 2, ACT>(a, p, sums, st);
    else if (p.tpr == 4) backward_rows<T, V, 4, K, ACT>(a, p, sums, st);
    else if (p.tpr == 8) backward_rows<T, V, 8, K, ACT>(a, p, sums, st);
    else if (p.tpr == 16) backward_rows<T, V, 16, K, ACT>(a, p, sums, st);
    else if (p.tpr == 32) backward_rows<T, V, 32, K, ACT>(a, p, sums, st);
    else if (p.tpr == 64) backward_rows<T, V, 64, K, ACT>(a, p, sums, st);
    else if (p.tpr == 128) backward_rows<T, V, 128, K, ACT>(a, p, sums, st);
    else if (p.tpr == 256) backward_rows<T, V, 256, K, ACT>(a, p, sums, st);
    else if (p.tpr == 512 && a.cols <= 4096) backward_rows<T, V, 512, K, ACT>(a, p, sums, st);
    else if (p.tpr == 512) backward_rows<T, V, 512, 2 * K, ACT>(a, p, sums, st);
    else if (p.tpr == 1024) backward_rows<T, V, 1024, 2 * K, ACT>(a, p, sums, st);
    else {
      a.chunks = p.chunks;
      const int64_t items = a.rows * a.chunks;
      int slices = p.few && !a.dx ? 0 : (int)p.groups;
      void *one[] = {&a}, *two[] = {&a, &slices};
      if (a.dx)
        launch((const void*)layer_norm_chunk_backward_sums_kernel<T, V, ACT>, (unsigned)(items < 1 << 20 ? items : 1 << 20),
               kThreads, one, st);
      if (sums && p.few)
        launch((const void*)layer_norm_chunk_backward_few_kernel<T, V, ACT>,
               (unsigned)(slices * p.chunks + (a.cols + 4 * V - 1) / (4 * V)), kThreads, two, st);
      else
        launch(sums ? (const void*)layer_norm_chunk_backward_kernel<T, V, ACT, true>
                    : (const void*)layer_norm_chunk_backward_kernel<T, V, ACT, false>,
               (unsigned)(p.groups * p.chunks), kThreads, two, st);
    }
  }
  if (sums && !(p.few && a.rows > 0)) {
    int count = (int)p.groups;
    void* args[] = {&a, &count};
    const int64_t width = (a.cols + 3) / 4 * 4;
    const bool few = 2 * width < 64 * kCus / 2;
    launch(few ? (const void*)layer_norm_sums_kernel<T, 16> : (const void*)layer_norm_sums_kernel<T, 64>,
           (unsigned)std::min((2 * width + (few ? 15 : 63)) / (few ? 16 : 64), (int64_t)1 << 20), kSumsThreads, args, st);
  }
}

}  // namespace

template <class T>
void layer_norm_forward(const NormArgs& a, int activation, hipStream_t st) {
  activation == RBL_ACT_GELU ? run_forward<T, RBL_ACT_GELU>(a, st) : run_forward<T, RBL_ACT_NONE>(a, st);
}
template <class T>
void layer_norm_backward(const NormArgs& a, const BackwardPlan& p, int activation, hipStream_t st) {
  activation == RBL_ACT_GELU ? run_backward<T, RBL_ACT_GELU>(a, p, st) : run_backward<T, RBL_ACT_NONE>(a, p, st);
}

}  // namespace rbl
