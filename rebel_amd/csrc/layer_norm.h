// rebel_amd/csrc/layer_norm.h -- layer normalisation, host side: what the entries (layer_norm.hip) and the kernels' launchers
// (layer_norm_kernel.h, compiled once for each element type) share.
#pragma once
#include <algorithm>

#include "train_kernels.h"

namespace rbl {

constexpr int kCus = 256;

struct NormArgs {
  const void *x, *dy, *w, *b;
  void *y, *dx, *dw, *db;
  float* stats;    // [rows][2]: mean, 1 / sqrt(variance + eps)
  int64_t rows, x_stride, dy_stride;
  float* partial;   // workspace: statistics of chunks (forward), sums of the parameters' gradients (backward)
  float* row_sums;  // workspace: chunks' sums of g w and g w h
  int cols;
  int chunks;     // of a row that is longer than a workgroup's registers
  int param_f32;  // the parameters' type: f32, or the rows' type
  float eps, inv_cols;
};

// The widest rows that a workgroup holds: forward in its registers (32 elements to each of 1024 threads; 4096 x 32768 bf16 134 us
// against 189 in chunks), backward with both sums in 128 KB of LDS (8192 x 12000 f32 223 us against 460 in chunks).
constexpr int kForwardCols = 32768, kBackwardCols = 16384;

// Longer ones go in chunks of kChunkK vectors to each of kThreads threads.
constexpr int kThreads = 256, kChunkK = 4;
inline int chunks_of_row(int64_t cols, int elements_of_vector) {
  const int64_t chunk = kThreads * kChunkK * elements_of_vector;
  return (int)((cols + chunk - 1) / chunk);
}

// Workgroups for `need` shares of work: what the chip holds at once of this kernel, or fewer, so that all have the same
// number of shares but for one.
inline unsigned even_grid(int64_t need, int64_t resident) {
  const int64_t rounds = (need + resident - 1) / resident;
  return (unsigned)((need + rounds - 1) / rounds);
}

// Workgroup size of the backward kernel, as forward.  Eight wavefronts to a CU are the best number for rows that are bound by memory
// (more slow the three streams down and leave more partial sums: back to back, 270336 x 256 f32 + GELU 150 us with 8, 167 with 16, 178
// with 32; 8192 x 4096 bf16 44 / 48 / 56 us).  16-bit rows with GELU, which are bound by issue, were not measured with more.
constexpr int backward_threads(int tpr) { return tpr <= 64 ? 256 : tpr; }
constexpr int kBackwardWaves = 8;

// Workgroups of the backward kernels, i.e. rows of partial sums
struct BackwardPlan {
  int tpr;     // threads to a row; 0: rows in chunks
  int chunks;  // of a row
  int64_t groups;
  bool few;  // so few rows that the parameters' gradients are taken from x and dy in the same launch
};

// Few rows, f32, in one launch against two (the sum of both kernels; the second launch's gap comes on top), us, behind a forward pass:
//     512 x 256 + GELU 6.7 / 7.6    640 x 256 7.5 / 7.9    768 x 256 8.6 / 7.6    1024 x 256 10.6 / 7.7
//     512 x 4096 10.0 / 12.9    512 x 8192 19.6 / 15.4    256 x 16384 22.2 / 22.6    24 x 65537 9.8 / 18.5 (the second of two kernels)
// Back to back 512 x 256 takes 5.4 / 7.6, 768 x 256 6.7 / 7.4, 1024 x 256 8.0 / 7.6.  With more rows the second reading costs more than
// it saves.
constexpr int64_t kFewRows = 512, kFewElements = 1 << 21;

inline BackwardPlan backward_plan(const rbl_layer_norm_shape& s) {
  BackwardPlan p{};
  p.few = s.rows <= kFewRows && s.rows * s.cols <= kFewElements;
  if (s.cols <= kBackwardCols) {
    p.tpr = s.cols <= 32 ? 4 : 8;
    while (p.tpr < 512 && p.tpr * 8 < s.cols) p.tpr *= 2;
    if (s.cols > 8192) p.tpr = 1024;
    const int nt = backward_threads(p.tpr);
    const int64_t need = (s.rows * p.tpr + nt - 1) / nt;
    // Threads past the row's end have nothing to load.  16-bit rows have one vector to a thread, and make up for them with more
    // workgroups (65536 x 1280 bf16 without GELU 113 us instead of 131, 32768 x 2560 106 instead of 126); f32 rows have two, and are slower for it.
    const int64_t threads = kBackwardWaves * 64;
    int64_t per_cu = threads / nt;
    if (s.dtype != RBL_F32 && s.cols <= 4096) per_cu = (threads * p.tpr * 8 + nt * s.cols / 2) / (nt * s.cols);
    p.groups = p.few || need == 0 ? need : even_grid(need, kCus * std::clamp<int64_t>(per_cu, 1, 16));
  } else {
    p.chunks = chunks_of_row(s.cols, s.dtype == RBL_F32 ? 4 : 8);
    const int64_t most = (2 * kCus + p.chunks - 1) / p.chunks;  // eight wavefronts to a CU here too
    p.groups = p.few || s.rows < most ? s.rows : most;
  }
  return p;
}

// Enqueue the passes; T: float, _Float16 or __bf16.
template <class T>
void layer_norm_forward(const NormArgs& a, int activation, hipStream_t st);
template <class T>
void layer_norm_backward(const NormArgs& a, const BackwardPlan& p, int activation, hipStream_t st);

}  // namespace rbl
