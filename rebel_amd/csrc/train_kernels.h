// rebel_amd/csrc/train_kernels.h -- what the training operators' files share: element types, the C entries' error guard and
// the reductions of a wavefront.
//
// The kernels themselves: layer_norm_kernel.h (forward and backward, compiled by layer_norm_{f32,f16,bf16}.hip) and
// grad_norm_kernel.hip (norm and clipping).
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>
#include <stdexcept>
#include <string>

#include "../../include/rebel_hip.h"

namespace rbl {

void set_last_error(const char* what);  // engine.hip: the message rbl_last_error() returns on this thread

// Every C entry of the training operators: no exception leaves it.
template <class F>
int train_entry(F&& f) {
  try {
    f();
    return 0;
  } catch (const std::exception& ex) {
    set_last_error(ex.what());
  } catch (...) {
    set_last_error("unknown error");
  }
  return 1;
}

inline void check_aligned(const void* p, uintptr_t bytes, const char* what) {
  if ((uintptr_t)p % bytes) throw std::runtime_error(std::string(what) + " must be aligned to " + std::to_string(bytes) + " bytes");
}

// Selects the device for the launches of one call; the one that was current is current again afterwards.  Made after the
// arguments have been checked, so that a refusal needs no GPU.
class DeviceScope {
 public:
  explicit DeviceScope(int device) {
    if (device < 0) throw std::runtime_error("device index is negative");
    if (hipGetDevice(&before_) != hipSuccess) throw std::runtime_error("HIP error: no device is available");
    if (before_ == device) return;
    if (hipSetDevice(device) != hipSuccess) throw std::runtime_error("HIP error: cannot select device " + std::to_string(device));
    changed_ = true;
  }
  ~DeviceScope() {
    if (changed_) (void)hipSetDevice(before_);
  }
  DeviceScope(const DeviceScope&) = delete;
  DeviceScope& operator=(const DeviceScope&) = delete;

 private:
  int before_ = -1;
  bool changed_ = false;
};

// One launch with its own status: hipGetLastError() would also report what an earlier call of the process left behind.
inline void launch(const void* kernel, unsigned grid, unsigned block, void** args, hipStream_t stream) {
  const hipError_t e = hipLaunchKernel(kernel, dim3(grid), dim3(block), args, 0, stream);
  if (e != hipSuccess) throw std::runtime_error(std::string("HIP error: kernel launch: ") + hipGetErrorString(e));
}

// Waits for this thread's LDS traffic and joins the workgroup.  __syncthreads() waits for outstanding global loads and stores
// too, i.e. for the rows that are being prefetched.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, true));
}

// Sum over the 2^k neighbouring lanes that share a row (4, 8, 16 or 32); every lane gets the same bits, since each step adds the
// same two numbers on both sides.
template <int LANES>
__device__ __forceinline__ float sum_lanes(float v) {
  static_assert(LANES == 4 || LANES == 8 || LANES == 16 || LANES == 32);
  v += dpp<0xB1>(v);                     // quad_perm [1,0,3,2]
  v += dpp<0x4E>(v);                     // quad_perm [2,3,0,1]
  if (LANES >= 8) v += dpp<0x141>(v);    // row_half_mirror
  if (LANES >= 16) v += dpp<0x140>(v);   // row_mirror
  if (LANES >= 32) {
    // v_permlane16_swap exchanges the odd rows of 16 lanes of one register with the even ones of another: copy, swap, add
    float c;
    asm("v_mov_b32 %1, %0\n\ts_nop 1\n\tv_permlane16_swap_b32 %0, %1\n\ts_nop 1" : "+v"(v), "=&v"(c));
    v += c;
  }
  return v;
}

// Sum over the wavefront, the same bits in every lane: four DPP rows, whose sums go through scalar registers.
__device__ __forceinline__ float sum64(float v) {
  v = sum_lanes<16>(v);
  const int i = __builtin_bit_cast(int, v);
  const float a = __builtin_bit_cast(float, __builtin_amdgcn_readlane(i, 0)),
              b = __builtin_bit_cast(float, __builtin_amdgcn_readlane(i, 16)),
              c = __builtin_bit_cast(float, __builtin_amdgcn_readlane(i, 32)),
              d = __builtin_bit_cast(float, __builtin_amdgcn_readlane(i, 48));
  return (a + b) + (c + d);
}

}  // namespace rbl
