// rebel_amd/csrc/grad_norm_kernel.hip -- the norm of many gradients taken as one vector, and their clipping to a bound.
//
//     N = (sum |g|^p)^(1/p), p = 1, 2 or infinity     c = min(1, max_norm / (N + 1e-6))     g <- c g
//
// Every tensor is cut into chunks, a workgroup to a chunk.  The first kernel leaves one f64 sum per chunk; the second adds
// all of them up in every workgroup, in the same order, and scales its chunk.  Squares are formed and summed in f64: no
// gradient that is finite in f32 overflows or vanishes on the way, and the order of the sum does not show in an f32 result.
// The table of tensors travels in the kernel's arguments, as many as fit in 4 KB to a launch: nothing is copied to the device
// beforehand, so a captured call replays with the pointers it was captured with and needs no memory of the host's.
#include <vector>

#include "train_kernels.h"

namespace rbl {
namespace {

constexpr int kThreads = 256;
constexpr int kTableSize = 128;      // tensors per launch
constexpr int64_t kChunkMin = 2048;  // elements
constexpr int kChunksAim = 2048;     // workgroups that fill the chip: 8 to a CU

struct GradTable {
  void* data[kTableSize];
  int64_t numel[kTableSize];
  int first_chunk[kTableSize + 1];
  int8_t dtype[kTableSize];
};

struct ClipArgs {
  double* sums;          // one per chunk
  const float* norm_in;  // the norm, where it is known already
  float* norm_out;
  double max_norm;
  int64_t chunk;
  int count;       // tensors in the table
  int first;       // chunks before the table's first
  int total;       // chunks of all tables
  int norm;
};

__device__ __forceinline__ double magnitude(float v, int norm) {
  const double d = v;
  return norm == RBL_NORM_2 ? d * d : __builtin_fabs(d);
}
// Sum, or the maximum that keeps a NaN
__device__ __forceinline__ double join(double a, double b, int norm) {
  if (norm != RBL_NORM_INF) return a + b;
  return (b > a || b != b) ? b : a;
}

__device__ __forceinline__ double join_block(double v, int norm, double* slots) {
  for (int d = 1; d < 64; d *= 2) v = join(v, __shfl_xor(v, d), norm);
  if (threadIdx.x % 64 == 0) slots[threadIdx.x / 64] = v;
  __syncthreads();
  return join(join(slots[0], slots[1], norm), join(slots[2], slots[3], norm), norm);
}

// The chunk of this workgroup: which tensor, from where to where
struct Chunk {
  int tensor;
  int64_t begin, end;
};
__device__ __forceinline__ Chunk chunk_of(const GradTable& t, const ClipArgs& a, int index) {
  int lo = 0, hi = a.count;  // first_chunk[lo] <= index < first_chunk[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (t.first_chunk[mid] <= index)
      lo = mid;
    else
      hi = mid;
  }
  const int64_t begin = (index - t.first_chunk[lo]) * a.chunk, end = begin + a.chunk;
  return {lo, begin, end < t.numel[lo] ? end : t.numel[lo]};
}

template <class T>
__device__ __forceinline__ double sum_chunk(const T* g, int64_t begin, int64_t end, int norm) {
  double v = 0;
  for (int64_t i = begin + threadIdx.x; i < end; i += kThreads) v = join(v, magnitude((float)g[i], norm), norm);
  return v;
}

__global__ __launch_bounds__(kThreads) void grad_sums_kernel(GradTable t, ClipArgs a) {
  __shared__ double slots[kThreads / 64];
  const Chunk k = chunk_of(t, a, blockIdx.x);
  const void* p = t.data[k.tensor];
  const int dtype = t.dtype[k.tensor];
  double v = dtype == RBL_F32   ? sum_chunk((const float*)p, k.begin, k.end, a.norm)
             : dtype == RBL_F16 ? sum_chunk((const _Float16*)p, k.begin, k.end, a.norm)
                                : sum_chunk((const __bf16*)p, k.begin, k.end, a.norm);
  v = join_block(v, a.norm, slots);
  if (threadIdx.x == 0) a.sums[a.first + blockIdx.x] = v;
}

__device__ __forceinline__ double whole_norm(const ClipArgs& a, double* slots) {
  double v = 0;
  for (int i = threadIdx.x; i < a.total; i += kThreads) v = join(v, a.sums[i], a.norm);
  v = join_block(v, a.norm, slots);
  return a.norm == RBL_NORM_2 ? __builtin_sqrt(v) : v;
}

template <class T>
__device__ __forceinline__ void scale_chunk(T* g, int64_t begin, int64_t end, float c) {
  for (int64_t i = begin + threadIdx.x; i < end; i += kThreads) g[i] = (T)((float)g[i] * c);
}

__global__ __launch_bounds__(kThreads) void grad_scale_kernel(GradTable t, ClipArgs a) {
  __shared__ double slots[kThreads / 64];
  const double norm = a.norm_in ? (double)*a.norm_in : whole_norm(a, slots);
  if (a.norm_out && a.first == 0 && blockIdx.x == 0 && threadIdx.x == 0) *a.norm_out = (float)norm;
  const double c = a.max_norm / (norm + 1e-6);
  if (c >= 1.0) return;  // times 1: nothing changes
  const Chunk k = chunk_of(t, a, blockIdx.x);
  void* p = t.data[k.tensor];
  const int dtype = t.dtype[k.tensor];
  if (dtype == RBL_F32)
    scale_chunk((float*)p, k.begin, k.end, (float)c);
  else if (dtype == RBL_F16)
    scale_chunk((_Float16*)p, k.begin, k.end, (float)c);
  else
    scale_chunk((__bf16*)p, k.begin, k.end, (float)c);
}

__global__ __launch_bounds__(kThreads) void grad_norm_kernel(ClipArgs a) {
  __shared__ double slots[kThreads / 64];
  const double norm = whole_norm(a, slots);
  if (threadIdx.x == 0) *a.norm_out = (float)norm;
}

int64_t chunk_size(const rbl_grad* grads, int n) {
  int64_t all = 0;
  for (int i = 0; i < n; ++i) all += grads[i].numel;
  const int64_t even = (all + kChunksAim - 1) / kChunksAim;
  return (even + kChunkMin - 1) / kChunkMin * kChunkMin + (all == 0 ? kChunkMin : 0);
}

int64_t chunk_count(const rbl_grad* grads, int n, int64_t chunk) {
  int64_t all = 0;
  for (int i = 0; i < n; ++i) all += (grads[i].numel + chunk - 1) / chunk;
  return all;
}

void check(const rbl_grad* grads, int n) {
  if (n < 0) throw std::runtime_error("gradients: n is negative");
  if (n > 0 && !grads) throw std::runtime_error("gradients: the list is null");
  int64_t room = (int64_t)1 << 60;
  for (int i = 0; i < n; ++i) {
    if (grads[i].numel < 0 || grads[i].numel > room) throw std::runtime_error("gradients: numel is negative or too large");
    room -= grads[i].numel;
    if (grads[i].numel > 0 && !grads[i].data_dev) throw std::runtime_error("gradients: a tensor's data is null");
    if (grads[i].dtype != RBL_F32 && grads[i].dtype != RBL_F16 && grads[i].dtype != RBL_BF16)
      throw std::runtime_error("gradients: unknown dtype");
  }
}
void check_norm(int norm) {
  if (norm != RBL_NORM_1 && norm != RBL_NORM_2 && norm != RBL_NORM_INF)
    throw std::runtime_error("gradients: the norm must be 1, 2 or infinity");
}
void check_workspace(const rbl_grad* grads, int n, const void* workspace, int64_t bytes) {
  const int64_t need = 8 * chunk_count(grads, n, chunk_size(grads, n));
  if (bytes < need || (need > 0 && !workspace))
    throw std::runtime_error("gradients: the workspace must hold " + std::to_string(need) + " bytes");
}
void check_bound(double max_norm) {
  if (!(max_norm >= 0)) throw std::runtime_error("gradients: max_norm must be a number >= 0");
}

// One launch of `kernel` for every table of tensors
void for_tables(const void* kernel, const rbl_grad* grads, int n, ClipArgs a, hipStream_t st) {
  GradTable t;
  a.chunk = chunk_size(grads, n);
  a.total = (int)chunk_count(grads, n, a.chunk);
  a.first = 0;
  for (int i = 0; i < n;) {
    int count = 0, chunks = 0;
    for (; i < n && count < kTableSize; ++i) {
      if (grads[i].numel == 0) continue;
      t.data[count] = grads[i].data_dev;
      t.numel[count] = grads[i].numel;
      t.dtype[count] = (int8_t)grads[i].dtype;
      t.first_chunk[count] = chunks;
      chunks += (int)((grads[i].numel + a.chunk - 1) / a.chunk);
      ++count;
    }
    if (count == 0) break;
    t.first_chunk[count] = chunks;
    a.count = count;
    void* args[] = {&t, &a};
    launch(kernel, (unsigned)chunks, kThreads, args, st);
    a.first += chunks;
  }
}

}  // namespace
}  // namespace rbl

extern "C" {

int64_t rbl_grad_workspace(const rbl_grad* grads, int n) {
  int64_t bytes = -1;
  rbl::train_entry([&] {
    rbl::check(grads, n);
    bytes = 8 * rbl::chunk_count(grads, n, rbl::chunk_size(grads, n));
  });
  return bytes;
}

int rbl_grad_norm(int device, const rbl_grad* grads, int n, int norm, float* norm_dev, void* workspace_dev,
                  int64_t workspace_bytes, void* stream) {
  return rbl::train_entry([&] {
    rbl::check(grads, n);
    rbl::check_norm(norm);
    rbl::check_workspace(grads, n, workspace_dev, workspace_bytes);
    if (!norm_dev) throw std::runtime_error("gradients: norm_dev is null");
    rbl::DeviceScope scope(device);
    rbl::ClipArgs a{};
    a.sums = (double*)workspace_dev;
    a.norm_out = norm_dev;
    a.norm = norm;
    rbl::for_tables((const void*)rbl::grad_sums_kernel, grads, n, a, (hipStream_t)stream);
    a.total = (int)rbl::chunk_count(grads, n, rbl::chunk_size(grads, n));
    void* args[] = {&a};
    rbl::launch((const void*)rbl::grad_norm_kernel, 1, rbl::kThreads, args, (hipStream_t)stream);
  });
}

int rbl_grad_clip(int device, const rbl_grad* grads, int n, int norm, double max_norm, float* norm_dev, void* workspace_dev,
                  int64_t workspace_bytes, void* stream) {
  return rbl::train_entry([&] {
    rbl::check(grads, n);
    rbl::check_norm(norm);
    rbl::check_bound(max_norm);
    rbl::check_workspace(grads, n, workspace_dev, workspace_bytes);
    if (!norm_dev) throw std::runtime_error("gradients: norm_dev is null");
    rbl::DeviceScope scope(device);
    rbl::ClipArgs a{};
    a.sums = (double*)workspace_dev;
    a.norm_out = norm_dev;
    a.norm = norm;
    a.max_norm = max_norm;
    rbl::for_tables((const void*)rbl::grad_sums_kernel, grads, n, a, (hipStream_t)stream);
    if (rbl::chunk_count(grads, n, rbl::chunk_size(grads, n)) == 0) {  // nothing to scale: the norm of nothing
      void* args[] = {&a};
      rbl::launch((const void*)rbl::grad_norm_kernel, 1, rbl::kThreads, args, (hipStream_t)stream);
    }
    rbl::for_tables((const void*)rbl::grad_scale_kernel, grads, n, a, (hipStream_t)stream);
  });
}

int rbl_grad_scale(int device, const rbl_grad* grads, int n, double max_norm, const float* norm_dev, void* stream) {
  return rbl::train_entry([&] {
    rbl::check(grads, n);
    rbl::check_bound(max_norm);
    if (!norm_dev) throw std::runtime_error("gradients: norm_dev is null");
    rbl::DeviceScope scope(device);
    rbl::ClipArgs a{};
    a.norm_in = norm_dev;
    a.max_norm = max_norm;
    rbl::for_tables((const void*)rbl::grad_scale_kernel, grads, n, a, (hipStream_t)stream);
  });
}

}  // extern "C"
