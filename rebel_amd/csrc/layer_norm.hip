// rebel_amd/csrc/layer_norm.hip -- the C entries of layer normalisation: checks, workspaces, the choice of the element type.
#include <initializer_list>

#include "layer_norm.h"

namespace rbl {
namespace {

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

int64_t forward_workspace(const rbl_layer_norm_shape& s) {
  if (s.cols <= kForwardCols) return 0;
  return s.rows * chunks_of_row(s.cols, s.dtype == RBL_F32 ? 4 : 8) * 2 * (int64_t)sizeof(float);
}

// row_sums of the chunks, then the partial sums
int64_t backward_row_sums(const rbl_layer_norm_shape& s, const BackwardPlan& p) {
  return p.tpr ? 0 : s.rows * p.chunks * 2 * (int64_t)sizeof(float);
}
int64_t backward_workspace(const rbl_layer_norm_shape& s) {
  const BackwardPlan p = backward_plan(s);
  return (backward_row_sums(s, p) + 15) / 16 * 16 + (p.few ? 0 : p.groups) * 2 * ((s.cols + 3) / 4 * 4) * (int64_t)sizeof(float);
}

void check_workspace(int64_t need, const void* workspace, int64_t bytes) {
  if (bytes < need || (need > 0 && !workspace))
    throw std::runtime_error("layer norm: the workspace must hold " + std::to_string(need) + " bytes");
}

void check_pointers(const rbl_layer_norm_shape& s, const void* workspace, const void* stats, std::initializer_list<const void*> rows,
                    std::initializer_list<const void*> params) {
  check_aligned(workspace, 16, "layer norm: the workspace");
  check_aligned(stats, 8, "layer norm: stats");
  for (const void* p : rows) check_aligned(p, s.dtype == RBL_F32 ? 4 : 2, "layer norm: x, y, dy and dx");
  for (const void* p : params) check_aligned(p, s.param_dtype == RBL_F32 ? 4 : 2, "layer norm: weight, bias and their gradients");
}

NormArgs args_of(const rbl_layer_norm_shape& s) {
  NormArgs a{};
  a.rows = s.rows;
  a.x_stride = s.x_stride;
  a.dy_stride = s.dy_stride;
  a.cols = (int)s.cols;
  a.inv_cols = 1.0f / (float)s.cols;
  a.param_f32 = s.param_dtype == RBL_F32;
  a.eps = s.eps;
  return a;
}

}  // namespace
}  // namespace rbl

extern "C" {

int64_t rbl_layer_norm_workspace(const rbl_layer_norm_shape* s, int backward) {
  int64_t bytes = -1;
  rbl::train_entry([&] {
    rbl::check(s);
    bytes = backward ? rbl::backward_workspace(*s) : rbl::forward_workspace(*s);
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
    a.partial = (float*)workspace_dev;
    rbl::check_workspace(rbl::forward_workspace(*s), workspace_dev, workspace_bytes);
    rbl::check_pointers(*s, workspace_dev, stats_dev, {x_dev, y_dev}, {weight_dev, bias_dev});
    rbl::DeviceScope scope(device);
    const auto run = s->dtype == RBL_F32   ? rbl::layer_norm_forward<float>
                     : s->dtype == RBL_F16 ? rbl::layer_norm_forward<_Float16>
                                           : rbl::layer_norm_forward<__bf16>;
    run(a, s->activation, (hipStream_t)stream);
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
    rbl::check_workspace(rbl::backward_workspace(*s), workspace_dev, workspace_bytes);
    rbl::check_pointers(*s, workspace_dev, stats_dev, {x_dev, dy_dev, dx_dev}, {weight_dev, bias_dev, dweight_dev, dbias_dev});
    const rbl::BackwardPlan p = rbl::backward_plan(*s);
    a.row_sums = (float*)workspace_dev;
    a.partial = a.row_sums + (rbl::backward_row_sums(*s, p) + 15) / 16 * 4;
    rbl::DeviceScope scope(device);
    const auto run = s->dtype == RBL_F32   ? rbl::layer_norm_backward<float>
                     : s->dtype == RBL_F16 ? rbl::layer_norm_backward<_Float16>
                                           : rbl::layer_norm_backward<__bf16>;
    run(a, p, s->activation, (hipStream_t)stream);
  });
}

}  // extern "C"
