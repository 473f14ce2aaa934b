// rebel_amd/csrc/layer_norm_kernel.hip -- layer normalisation, forward and backward, with an optional GELU behind it.
//
// Row x of n values, weight w, bias b, eps e:
//     m = sum x / n     v = sum (x - m)^2 / n     r = 1 / sqrt(v + e)     h = (x - m) r     z = h w + b
//     y = z,  or  y = z Phi(z) with the normal distribution Phi (GELU)
// and, with g = dy (GELU: g = dy (Phi(z) + z phi(z)), phi the density):
//     db = sum_rows g     dw = sum_rows g h     dx = r (g w - sum(g w) / n - h sum(g w h) / n)
//
// Simple form: a workgroup to a row, which it walks three times (the row stays in the caches); the parameters' gradients by a
// second kernel that walks columns.  h is computed again from x and the two statistics of the row, so nothing else is kept
// between the passes.
#include "train_kernels.h"

namespace rbl {
namespace {

constexpr int kThreads = 256;

// Phi(z) and exp(-z^2 / 2).  For x = |z|: Phi(-x) = exp(-x^2 / 2) P(x) with P(x) = exp(x^2 / 2) erfc(x / sqrt 2) / 2, which
// falls smoothly from 1/2 like 1 / (x sqrt(2 pi)): a polynomial of degree 8 in u = 1 / (1 + 0.3 x) without a constant term
// (the form of Abramowitz and Stegun 7.1.26; coefficients fitted here to the least relative error on [0, 14], 1.5e-7 exactly
// and 4.3e-7 in f32).  The error is RELATIVE on the negative side too, where 1 + erf would cancel, and the exponential is
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

struct NormArgs {
  const void *x, *dy, *w, *b;
  void *y, *dx, *dw, *db;
  float* stats;    // [rows][2]: mean, 1 / sqrt(variance + eps)
  int64_t rows, x_stride, dy_stride;
  int cols;
  int param_f32;  // the parameters' type: f32, or the rows' type
  float eps;
};

template <class T>
__device__ __forceinline__ float param(const NormArgs& a, const void* p, int col, float missing) {
  if (!p) return missing;
  return a.param_f32 ? ((const float*)p)[col] : (float)((const T*)p)[col];
}
template <class T>
__device__ __forceinline__ void put_param(const NormArgs& a, void* p, int col, float v) {
  if (a.param_f32)
    ((float*)p)[col] = v;
  else
    ((T*)p)[col] = (T)v;
}

// Sums of two numbers over the workgroup, the same bits in every thread.
__device__ __forceinline__ void sum_block(float& p, float& q, float (*slots)[2]) {
  const int wave = threadIdx.x / 64;
  p = sum64(p);
  q = sum64(q);
  __syncthreads();
  if (threadIdx.x % 64 == 0) {
    slots[wave][0] = p;
    slots[wave][1] = q;
  }
  __syncthreads();
  p = (slots[0][0] + slots[1][0]) + (slots[2][0] + slots[3][0]);
  q = (slots[0][1] + slots[1][1]) + (slots[2][1] + slots[3][1]);
}

template <class T, int ACT>
__global__ __launch_bounds__(kThreads) void layer_norm_forward_kernel(NormArgs a) {
  __shared__ float slots[kThreads / 64][2];
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = (const T*)a.x + row * a.x_stride;
    T* y = (T*)a.y + row * a.cols;
    float s = 0, zero = 0;
    for (int c = threadIdx.x; c < a.cols; c += kThreads) s += (float)x[c];
    sum_block(s, zero, slots);
    // the deviations from the rounded mean: their sum corrects it
    const float first = s / a.cols;
    float off = 0, square = 0;
    for (int c = threadIdx.x; c < a.cols; c += kThreads) {
      const float d = (float)x[c] - first;
      off += d;
      square = __builtin_fmaf(d, d, square);
    }
    sum_block(off, square, slots);
    const float mean = first + off / a.cols;
    float variance = (square - off * off / a.cols) / a.cols;
    variance = variance < 0 ? 0 : variance;  // NaN stays
    const float r = 1.0f / __builtin_sqrtf(variance + a.eps);
    for (int c = threadIdx.x; c < a.cols; c += kThreads) {
      const float h = ((float)x[c] - mean) * r;
      y[c] = (T)activate<ACT>(__builtin_fmaf(h, param<T>(a, a.w, c, 1.0f), param<T>(a, a.b, c, 0.0f)));
    }
    if (a.stats && threadIdx.x == 0) {
      a.stats[2 * row] = mean;
      a.stats[2 * row + 1] = r;
    }
  }
}

template <class T, int ACT>
__global__ __launch_bounds__(kThreads) void layer_norm_dx_kernel(NormArgs a) {
  __shared__ float slots[kThreads / 64][2];
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = (const T*)a.x + row * a.x_stride;
    const T* dy = (const T*)a.dy + row * a.dy_stride;
    T* dx = (T*)a.dx + row * a.cols;
    const float mean = a.stats[2 * row], r = a.stats[2 * row + 1];
    float p = 0, q = 0;
    for (int c = threadIdx.x; c < a.cols; c += kThreads) {
      const float h = ((float)x[c] - mean) * r, w = param<T>(a, a.w, c, 1.0f);
      const float gw = (float)dy[c] * activate_slope<ACT>(__builtin_fmaf(h, w, param<T>(a, a.b, c, 0.0f))) * w;
      p += gw;
      q = __builtin_fmaf(gw, h, q);
    }
    sum_block(p, q, slots);
    p /= a.cols;
    q /= a.cols;
    for (int c = threadIdx.x; c < a.cols; c += kThreads) {
      const float h = ((float)x[c] - mean) * r, w = param<T>(a, a.w, c, 1.0f);
      const float gw = (float)dy[c] * activate_slope<ACT>(__builtin_fmaf(h, w, param<T>(a, a.b, c, 0.0f))) * w;
      dx[c] = (T)(r * (gw - p - h * q));
    }
  }
}

// 64 columns x 4 row threads to a workgroup, over all rows.
template <class T, int ACT>
__global__ __launch_bounds__(kThreads) void layer_norm_dparam_kernel(NormArgs a) {
  __shared__ float part[2][4][64];
  const int lane = threadIdx.x % 64, slice = threadIdx.x / 64;
  const int c = blockIdx.x * 64 + lane;
  float dw = 0, db = 0;
  if (c < a.cols) {
    const float w = param<T>(a, a.w, c, 1.0f), b = param<T>(a, a.b, c, 0.0f);
    for (int64_t row = slice; row < a.rows; row += 4) {
      const float h = ((float)((const T*)a.x)[row * a.x_stride + c] - a.stats[2 * row]) * a.stats[2 * row + 1];
      const float g = (float)((const T*)a.dy)[row * a.dy_stride + c] * activate_slope<ACT>(__builtin_fmaf(h, w, b));
      dw = __builtin_fmaf(g, h, dw);
      db += g;
    }
  }
  part[0][slice][lane] = dw;
  part[1][slice][lane] = db;
  __syncthreads();
  if (slice == 0 && c < a.cols) {
    if (a.dw) put_param<T>(a, a.dw, c, (part[0][0][lane] + part[0][1][lane]) + (part[0][2][lane] + part[0][3][lane]));
    if (a.db) put_param<T>(a, a.db, c, (part[1][0][lane] + part[1][1][lane]) + (part[1][2][lane] + part[1][3][lane]));
  }
}

unsigned row_grid(int64_t rows) { return (unsigned)(rows < 16384 ? rows : 16384); }

template <class T, int ACT>
void run_forward(NormArgs a, hipStream_t st) {
  if (a.rows == 0) return;
  void* args[] = {&a};
  launch((const void*)layer_norm_forward_kernel<T, ACT>, row_grid(a.rows), kThreads, args, st);
}
template <class T, int ACT>
void run_backward(NormArgs a, hipStream_t st) {
  void* args[] = {&a};
  if (a.dx && a.rows > 0) launch((const void*)layer_norm_dx_kernel<T, ACT>, row_grid(a.rows), kThreads, args, st);
  if (a.dw || a.db)
    launch((const void*)layer_norm_dparam_kernel<T, ACT>, (unsigned)((a.cols + 63) / 64), kThreads, args, st);
}

void check(const rbl_layer_norm_shape* s) {
  if (!s) throw std::runtime_error("layer norm: shape is null");
  if (s->rows < 0) throw std::runtime_error("layer norm: rows is negative");
  if (s->cols < 1 || s->cols > (int64_t)1 << 30) throw std::runtime_error("layer norm: cols must be in [1, 2^30]");
  if (s->dtype != RBL_F32 && s->dtype != RBL_F16 && s->dtype != RBL_BF16) throw std::runtime_error("layer norm: unknown dtype");
  if (s->param_dtype != RBL_F32 && s->param_dtype != s->dtype)
    throw std::runtime_error("layer norm: param_dtype must be f32 or dtype");
  if (s->activation != RBL_ACT_NONE && s->activation != RBL_ACT_GELU)
    throw std::runtime_error("layer norm: unknown activation");
  if (s->x_stride < 0 || s->dy_stride < 0) throw std::runtime_error("layer norm: strides must not be negative");
  if (s->rows > 0 && s->rows > ((int64_t)1 << 60) / s->cols) throw std::runtime_error("layer norm: rows x cols is too large");
}

NormArgs args_of(const rbl_layer_norm_shape& s) {
  NormArgs a{};
  a.rows = s.rows;
  a.x_stride = s.x_stride;
  a.dy_stride = s.dy_stride;
  a.cols = (int)s.cols;
  a.param_f32 = s.param_dtype == RBL_F32;
  a.eps = s.eps;
  return a;
}

template <int ACT>
void forward_by_type(int dtype, const NormArgs& a, hipStream_t st) {
  if (dtype == RBL_F32) run_forward<float, ACT>(a, st);
  if (dtype == RBL_F16) run_forward<_Float16, ACT>(a, st);
  if (dtype == RBL_BF16) run_forward<__bf16, ACT>(a, st);
}
template <int ACT>
void backward_by_type(int dtype, const NormArgs& a, hipStream_t st) {
  if (dtype == RBL_F32) run_backward<float, ACT>(a, st);
  if (dtype == RBL_F16) run_backward<_Float16, ACT>(a, st);
  if (dtype == RBL_BF16) run_backward<__bf16, ACT>(a, st);
}

}  // namespace
}  // namespace rbl

extern "C" {

int64_t rbl_layer_norm_workspace(const rbl_layer_norm_shape* s, int backward) {
  int64_t bytes = -1;
  rbl::train_entry([&] {
    rbl::check(s);
    bytes = 0;
  });
  return bytes;
}

int rbl_layer_norm_forward(int device, const rbl_layer_norm_shape* s, const void* x_dev, const void* weight_dev,
                           const void* bias_dev, void* y_dev, float* stats_dev, void* workspace_dev, int64_t workspace_bytes,
                           void* stream) {
  return rbl::train_entry([&] {
    rbl::check(s);
    if (s->rows > 0 && (!x_dev || !y_dev)) throw std::runtime_error("layer norm: x or y is null");
    rbl::NormArgs a = rbl::args_of(*s);
    a.x = x_dev;
    a.w = weight_dev;
    a.b = bias_dev;
    a.y = y_dev;
    a.stats = stats_dev;
    rbl::DeviceScope scope(device);
    s->activation == RBL_ACT_GELU ? rbl::forward_by_type<RBL_ACT_GELU>(s->dtype, a, (hipStream_t)stream)
                                  : rbl::forward_by_type<RBL_ACT_NONE>(s->dtype, a, (hipStream_t)stream);
  });
}

int rbl_layer_norm_backward(int device, const rbl_layer_norm_shape* s, const void* dy_dev, const void* x_dev,
                            const void* weight_dev, const void* bias_dev, const float* stats_dev, void* dx_dev,
                            void* dweight_dev, void* dbias_dev, void* workspace_dev, int64_t workspace_bytes, void* stream) {
  return rbl::train_entry([&] {
    rbl::check(s);
    if (s->rows > 0 && (!x_dev || !dy_dev || !stats_dev)) throw std::runtime_error("layer norm: x, dy or stats is null");
    rbl::NormArgs a = rbl::args_of(*s);
    a.x = x_dev;
    a.dy = dy_dev;
    a.w = weight_dev;
    a.b = bias_dev;
    a.stats = const_cast<float*>(stats_dev);
    a.dx = dx_dev;
    a.dw = dweight_dev;
    a.db = dbias_dev;
    rbl::DeviceScope scope(device);
    s->activation == RBL_ACT_GELU ? rbl::backward_by_type<RBL_ACT_GELU>(s->dtype, a, (hipStream_t)stream)
                                  : rbl::backward_by_type<RBL_ACT_NONE>(s->dtype, a, (hipStream_t)stream);
  });
}

}  // extern "C"
