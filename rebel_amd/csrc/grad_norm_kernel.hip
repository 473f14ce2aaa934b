// rebel_amd/csrc/grad_norm_kernel.hip -- the norm of many gradients taken as one vector, and their clipping to a bound.
//
//     N = (sum |g|^p)^(1/p), p = 1, 2 or infinity     c = min(1, max_norm / (N + 1e-6))     g <- c g
//
// Every tensor is cut into chunks of as many bytes, a workgroup to a chunk.  The first kernel leaves one f64 sum per chunk; the
// second adds all of them up in every workgroup, in the same order, and scales its chunk (where they are many, a kernel between
// the two has added them up).  Squares are formed and summed in f64: no gradient that is finite in f32 overflows or vanishes on
// the way, and the order of the sum does not show in an f32 result.
// Bound by memory, one reading for the sums and one reading and one writing for the scaling: 400 M f32 in 200 tensors 236 us (6.8
// TB/s) and 634 us (5.0 TB/s), 200 M bf16 in 200 tensors 65 us (6.1) and 163 us (4.9), 60 M f16 in 100 tensors 25 us (4.8) and 50 us
// (4.8).  A step whose norm stays under the bound ends after the sums.  Small sets are bound by latency, one load after the other:
// 3.0 and 3.8 us for the 76 thousand values of a net of two hidden layers of 256, with the chunks themselves in the arguments (3.8
// and 4.0 with a search for the tensor).  One workgroup that keeps such a set in its registers took 10.5 us, most of it for its 300 KB
// through one CU.
//
// The table of tensors travels in the kernel's arguments, as many as fit in 4 KB to a launch: nothing is copied to the device
// beforehand, so a captured call replays with the pointers it was captured with and needs no memory of the host's.
#include <algorithm>

#include "train_kernels.h"

namespace rbl {
namespace {

constexpr int kThreads = 256;
constexpr int kTableSize = 240;      // tensors per launch
// Chunks: 8 KB in small sets; then as many as the chip holds workgroups (8 to a CU), until they reach 128 KB; then four rounds of
// workgroups, so that none ends long after the others (1.6 GB scaled in 662 us by one round, 625 by four); then larger again.
constexpr int64_t kChunkMin = 8 << 10, kChunkFull = 128 << 10;
constexpr int kChunksResident = 2048, kChunksMost = 8192;
constexpr int kSumsMost = 4096;  // sums that every workgroup of the scaling adds up for itself

struct GradTable {
  void* data[kTableSize];
  int first_chunk[kTableSize + 1];
  unsigned last[kTableSize];  // elements of the tensor's last chunk; its type in the upper two bits
};
constexpr int kTypeShift = 30;

// Sets of few chunks: the chunks themselves, found without a search.
constexpr int kFewChunks = 320;
struct ChunkTable {
  void* data[kFewChunks];
  unsigned count[kFewChunks];  // elements; their type in the upper two bits
};

struct ClipArgs {
  double* sums;          // one per chunk, then their sum
  const float* norm_in;  // the norm, where it is known already
  float* norm_out;
  double max_norm;
  int chunk;  // bytes
  int count;  // tensors in the table
  int first;  // chunks before the table's first
  int total;  // chunks of all tables
};
static_assert(sizeof(GradTable) + sizeof(ClipArgs) <= 4096 && sizeof(ChunkTable) + sizeof(ClipArgs) <= 4096, "kernel arguments");

// One element's share of the norm, and how shares are joined: the sum, or the maximum that keeps a NaN.
template <int NORM>
__device__ __forceinline__ void take(double& s, float v) {
  const double d = v;
  if (NORM == RBL_NORM_2) s = __builtin_fma(d, d, s);
  if (NORM == RBL_NORM_1) s += __builtin_fabs(d);
  if (NORM == RBL_NORM_INF) s = (__builtin_fabs(d) > s || d != d) ? __builtin_fabs(d) : s;
}
template <int NORM>
__device__ __forceinline__ double join(double a, double b) {
  if (NORM != RBL_NORM_INF) return a + b;
  return (b > a || b != b) ? b : a;
}

template <int NORM, int WAVES = kThreads / 64>
__device__ __forceinline__ double join_block(double v, double* slots) {
  for (int d = 1; d < 64; d *= 2) v = join<NORM>(v, __shfl_xor(v, d));
  if (threadIdx.x % 64 == 0) slots[threadIdx.x / 64] = v;
  __syncthreads();
  v = slots[0];
#pragma unroll
  for (int w = 1; w < WAVES; ++w) v = join<NORM>(v, slots[w]);
  return v;
}

// A workgroup's chunk: its first element, how many, and their type
struct Chunk {
  void* data;
  int64_t begin;
  int count, type;
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
  const unsigned last = t.last[lo];
  const int type = (int)(last >> kTypeShift), whole = a.chunk / (type == RBL_F32 ? 4 : 2);
  const bool is_last = index + 1 == t.first_chunk[lo + 1];
  return {t.data[lo], (int64_t)(index - t.first_chunk[lo]) * whole, is_last ? (int)(last & ((1u << kTypeShift) - 1)) : whole, type};
}

__device__ __forceinline__ Chunk chunk_of(const ChunkTable& t, const ClipArgs&, int index) {
  return {t.data[index], 0, (int)(t.count[index] & ((1u << kTypeShift) - 1)), (int)(t.count[index] >> kTypeShift)};
}

// 16 bytes in one access, at the alignment of an element
template <class T>
struct Pack {
  static constexpr int V = 16 / sizeof(T);
  typedef T type __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
};

constexpr int kAhead = 4;  // loads in flight per thread
// The sums read without a claim to the caches: 1.6 GB at 6.7 TB/s instead of 5.8, and clipping 100 to 240 MB, which the cache of
// 256 MB could hold between the two kernels, is no slower for it (53 / 114 us).

template <class T, int NORM>
__device__ __forceinline__ double sum_chunk(const T* g, int count) {
  constexpr int V = Pack<T>::V, STEP = kThreads * V;
  typedef typename Pack<T>::type vec;
  double s[2] = {0, 0};
  int i = threadIdx.x * V;
  for (; i + (kAhead - 1) * STEP + V <= count; i += kAhead * STEP) {
    vec v[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) v[k] = __builtin_nontemporal_load((const vec*)(g + i + k * STEP));
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) take<NORM>(s[j % 2], (float)v[k][j]);
  }
  for (; i + V <= count; i += STEP) {
    const vec v = *(const vec*)(g + i);
#pragma unroll
    for (int j = 0; j < V; ++j) take<NORM>(s[j % 2], (float)v[j]);
  }
  const int rest = count / V * V + (int)threadIdx.x;  // fewer than V elements behind the last whole vector
  if (rest < count) take<NORM>(s[0], (float)g[rest]);
  return join<NORM>(s[0], s[1]);
}

template <int NORM, class TABLE>
__global__ __launch_bounds__(kThreads) void grad_sums_kernel(TABLE t, ClipArgs a) {
  __shared__ double slots[kThreads / 64];
  const Chunk k = chunk_of(t, a, blockIdx.x);
  double v = k.type == RBL_F32   ? sum_chunk<float, NORM>((const float*)k.data + k.begin, k.count)
             : k.type == RBL_F16 ? sum_chunk<_Float16, NORM>((const _Float16*)k.data + k.begin, k.count)
                                 : sum_chunk<__bf16, NORM>((const __bf16*)k.data + k.begin, k.count);
  v = join_block<NORM>(v, slots);
  if (threadIdx.x == 0) a.sums[a.first + blockIdx.x] = v;
}

template <int NORM>
__device__ __forceinline__ double whole_norm(const ClipArgs& a, double* slots) {
  if (a.total > kSumsMost) return a.sums[a.total];  // grad_norm_kernel has been there
  double v = 0;
#pragma unroll 4
  for (int i = threadIdx.x; i < a.total; i += kThreads) v = join<NORM>(v, a.sums[i]);
  v = join_block<NORM>(v, slots);
  return NORM == RBL_NORM_2 ? __builtin_sqrt(v) : v;
}

template <class T>
__device__ __forceinline__ void scale_chunk(T* g, int count, float c) {
  constexpr int V = Pack<T>::V, STEP = kThreads * V;
  typedef typename Pack<T>::type vec;
  int i = threadIdx.x * V;
  for (; i + (kAhead - 1) * STEP + V <= count; i += kAhead * STEP) {
    vec v[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) v[k] = *(const vec*)(g + i + k * STEP);
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
#pragma unroll
      for (int j = 0; j < V; ++j) v[k][j] = (T)((float)v[k][j] * c);
      *(vec*)(g + i + k * STEP) = v[k];
    }
  }
  for (; i + V <= count; i += STEP) {
    vec v = *(const vec*)(g + i);
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = (T)((float)v[j] * c);
    *(vec*)(g + i) = v;
  }
  const int rest = count / V * V + (int)threadIdx.x;
  if (rest < count) g[rest] = (T)((float)g[rest] * c);
}

// A factor that has no normal number in f32 (gradients near the type's end): products in f64
constexpr double kFactorLeast = 0x1p-126;
template <class T>
__device__ __forceinline__ void scale_chunk_wide(T* g, int count, double c) {
  for (int i = threadIdx.x; i < count; i += kThreads) g[i] = (T)(float)((double)(float)g[i] * c);
}

// NORM 0: the norm is there already
template <int NORM, class TABLE>
__global__ __launch_bounds__(kThreads) void grad_scale_kernel(TABLE t, ClipArgs a) {
  __shared__ double slots[kThreads / 64];
  double norm;
  if constexpr (NORM == 0) {
    norm = (double)*a.norm_in;
  } else {
    norm = whole_norm<NORM>(a, slots);
    if (a.first == 0 && blockIdx.x == 0 && threadIdx.x == 0) *a.norm_out = (float)norm;
  }
  const double c = a.max_norm / (norm + 1e-6);
  if (c >= 1.0) return;  // times 1: nothing changes
  // from the last chunk to the first: what the sums read last is what the cache still has
  const Chunk k = chunk_of(t, a, gridDim.x - 1 - blockIdx.x);
  const auto scale = [&](auto* g) { c > 0 && c < kFactorLeast ? scale_chunk_wide(g, k.count, c) : scale_chunk(g, k.count, (float)c); };
  if (k.type == RBL_F32)
    scale((float*)k.data + k.begin);
  else if (k.type == RBL_F16)
    scale((_Float16*)k.data + k.begin);
  else
    scale((__bf16*)k.data + k.begin);
}

// The norm from the chunks' sums, for those who ask for it and for a scaling that finds it behind the sums.
constexpr int kNormThreads = 1024;
template <int NORM>
__global__ __launch_bounds__(kNormThreads) void grad_norm_kernel(ClipArgs a) {
  __shared__ double slots[kNormThreads / 64];
  double v = 0;
#pragma unroll 8
  for (int i = threadIdx.x; i < a.total; i += kNormThreads) v = join<NORM>(v, a.sums[i]);
  v = join_block<NORM, kNormThreads / 64>(v, slots);
  if (threadIdx.x == 0) {
    const double norm = NORM == RBL_NORM_2 ? __builtin_sqrt(v) : v;
    *a.norm_out = (float)norm;
    if (a.total > kSumsMost) a.sums[a.total] = norm;
  }
}

// The kernels of a norm (0: it is known), for many chunks and for few
struct Kernels {
  const void *sums, *sums_few, *scale, *scale_few, *norm;
};
template <int NORM>
Kernels kernels() {
  return {(const void*)grad_sums_kernel<NORM, GradTable>, (const void*)grad_sums_kernel<NORM, ChunkTable>,
          (const void*)grad_scale_kernel<NORM, GradTable>, (const void*)grad_scale_kernel<NORM, ChunkTable>,
          (const void*)grad_norm_kernel<NORM>};
}
Kernels kernels_of(int norm) {
  return norm == RBL_NORM_1 ? kernels<RBL_NORM_1>() : norm == RBL_NORM_2 ? kernels<RBL_NORM_2>() : kernels<RBL_NORM_INF>();
}

int64_t size_of(const rbl_grad& g) { return g.dtype == RBL_F32 ? 4 : 2; }

struct Plan {
  int shift;  // a chunk has 2^shift bytes
  int total;  // chunks
};
int64_t chunks_of(const rbl_grad& g, int shift) { return (g.numel * size_of(g) + ((int64_t)1 << shift) - 1) >> shift; }

Plan plan_of(const rbl_grad* grads, int n) {
  int64_t all = 0, chunks = 0;
  for (int i = 0; i < n; ++i) all += grads[i].numel * size_of(grads[i]);
  const int64_t chunk = std::max({std::min(all / kChunksResident, kChunkFull), all / kChunksMost, kChunkMin});
  Plan p{0, 0};
  while ((int64_t)1 << p.shift < chunk) ++p.shift;
  for (int i = 0; i < n; ++i) chunks += chunks_of(grads[i], p.shift);
  p.total = (int)chunks;
  return p;
}
int64_t workspace_size(const Plan& p) { return p.total ? 8 * ((int64_t)p.total + 1) : 0; }

void check(const rbl_grad* grads, int n) {
  if (n < 0) throw std::runtime_error("gradients: n is negative");
  if (n > 0 && !grads) throw std::runtime_error("gradients: the list is null");
  int64_t room = (int64_t)1 << 40;  // 2^40 elements: a chunk's length fits into 30 bits
  for (int i = 0; i < n; ++i) {
    if (grads[i].numel < 0 || grads[i].numel > room) throw std::runtime_error("gradients: numel is negative or too large");
    room -= grads[i].numel;
    if (grads[i].numel > 0 && !grads[i].data_dev) throw std::runtime_error("gradients: a tensor's data is null");
    if (grads[i].dtype != RBL_F32 && grads[i].dtype != RBL_F16 && grads[i].dtype != RBL_BF16)
      throw std::runtime_error("gradients: unknown dtype");
    check_aligned(grads[i].data_dev, size_of(grads[i]), "gradients: a tensor's data");
  }
}
void check_norm(int norm) {
  if (norm != RBL_NORM_1 && norm != RBL_NORM_2 && norm != RBL_NORM_INF)
    throw std::runtime_error("gradients: the norm must be 1, 2 or infinity");
}
void check_workspace(const Plan& p, const void* workspace, int64_t bytes) {
  const int64_t need = workspace_size(p);
  if (bytes < need || (need > 0 && !workspace))
    throw std::runtime_error("gradients: the workspace must hold " + std::to_string(need) + " bytes");
  check_aligned(workspace, 8, "gradients: the workspace");
}
void check_bound(double max_norm) {
  if (!(max_norm >= 0)) throw std::runtime_error("gradients: max_norm must be a number >= 0");
}

// One launch of `kernel` for every table of tensors, or of `few` for all of few chunks; `backwards`: the last table first
void for_tables(const void* kernel, const void* few, const rbl_grad* grads, int n, ClipArgs a, const Plan& p, bool backwards,
                hipStream_t st) {
  a.chunk = 1 << p.shift;
  a.total = p.total;
  if (p.total == 0) return;
  if (p.total <= kFewChunks) {
    ChunkTable c;
    int count = 0;
    for (int i = 0; i < n; ++i) {
      const int64_t bytes = grads[i].numel * size_of(grads[i]);
      for (int64_t at = 0; at < bytes; at += a.chunk) {
        c.data[count] = (char*)grads[i].data_dev + at;
        c.count[count++] = (unsigned)(std::min(bytes - at, (int64_t)a.chunk) / size_of(grads[i])) | (unsigned)grads[i].dtype << kTypeShift;
      }
    }
    a.count = count;
    a.first = 0;
    void* args[] = {&c, &a};
    launch(few, (unsigned)count, kThreads, args, st);
    return;
  }
  GradTable t;
  int from = 0, to = n, first = backwards ? a.total : 0;
  while (from < to) {
    // the next table: tensors [from, end), or backwards [end, to)
    int end = backwards ? to : from, count = 0;
    while (backwards ? end > from : end < to) {
      if (count == kTableSize) break;
      if (grads[backwards ? end - 1 : end].numel > 0) ++count;
      end += backwards ? -1 : 1;
    }
    const int lo = backwards ? end : from, hi = backwards ? to : end;
    int chunks = 0;
    count = 0;
    for (int i = lo; i < hi; ++i) {
      if (grads[i].numel == 0) continue;
      const int64_t whole = chunks_of(grads[i], p.shift);
      t.data[count] = grads[i].data_dev;
      t.first_chunk[count] = chunks;
      t.last[count] = (unsigned)(grads[i].numel - (whole - 1) * (a.chunk / size_of(grads[i]))) | (unsigned)grads[i].dtype << kTypeShift;
      chunks += (int)whole;
      ++count;
    }
    if (count > 0) {
      t.first_chunk[count] = chunks;
      a.count = count;
      a.first = backwards ? first - chunks : first;
      void* args[] = {&t, &a};
      launch(kernel, (unsigned)chunks, kThreads, args, st);
      first += backwards ? -chunks : chunks;
    }
    (backwards ? to : from) = end;
  }
}

}  // namespace
}  // namespace rbl

extern "C" {

int64_t rbl_grad_workspace(const rbl_grad* grads, int n) {
  int64_t bytes = -1;
  rbl::train_entry([&] {
    rbl::check(grads, n);
    bytes = rbl::workspace_size(rbl::plan_of(grads, n));
  });
  return bytes;
}

int rbl_grad_norm(int device, const rbl_grad* grads, int n, int norm, float* norm_dev, void* workspace_dev,
                  int64_t workspace_bytes, void* stream) {
  return rbl::train_entry([&] {
    rbl::check(grads, n);
    rbl::check_norm(norm);
    const rbl::Plan p = rbl::plan_of(grads, n);
    rbl::check_workspace(p, workspace_dev, workspace_bytes);
    if (!norm_dev) throw std::runtime_error("gradients: norm_dev is null");
    rbl::DeviceScope scope(device);
    const rbl::Kernels k = rbl::kernels_of(norm);
    rbl::ClipArgs a{};
    a.sums = (double*)workspace_dev;
    a.norm_out = norm_dev;
    rbl::for_tables(k.sums, k.sums_few, grads, n, a, p, false, (hipStream_t)stream);
    a.total = p.total;
    void* args[] = {&a};
    rbl::launch(k.norm, 1, rbl::kNormThreads, args, (hipStream_t)stream);
  });
}

int rbl_grad_clip(int device, const rbl_grad* grads, int n, int norm, double max_norm, float* norm_dev, void* workspace_dev,
                  int64_t workspace_bytes, void* stream) {
  return rbl::train_entry([&] {
    rbl::check(grads, n);
    rbl::check_norm(norm);
    rbl::check_bound(max_norm);
    const rbl::Plan p = rbl::plan_of(grads, n);
    rbl::check_workspace(p, workspace_dev, workspace_bytes);
    if (!norm_dev) throw std::runtime_error("gradients: norm_dev is null");
    rbl::DeviceScope scope(device);
    const rbl::Kernels k = rbl::kernels_of(norm);
    rbl::ClipArgs a{};
    a.sums = (double*)workspace_dev;
    a.norm_out = norm_dev;
    a.max_norm = max_norm;
    rbl::for_tables(k.sums, k.sums_few, grads, n, a, p, false, (hipStream_t)stream);
    a.total = p.total;
    if (a.total == 0 || a.total > rbl::kSumsMost) {  // nothing to scale: the norm of nothing
      void* args[] = {&a};
      rbl::launch(k.norm, 1, rbl::kNormThreads, args, (hipStream_t)stream);
    }
    rbl::for_tables(k.scale, k.scale_few, grads, n, a, p, true, (hipStream_t)stream);
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
    rbl::for_tables((const void*)rbl::grad_scale_kernel<0, rbl::GradTable>, (const void*)rbl::grad_scale_kernel<0, rbl::ChunkTable>,
                    grads, n, a, rbl::plan_of(grads, n), true, (hipStream_t)stream);
  });
}

}  // extern "C"
