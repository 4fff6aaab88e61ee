// C ABI of the distillation operators: checks of arguments, then one launcher each.  Nothing in here
// throws.
#include <atomic>
#include <cstdio>

#include "../../include/b2fil.h"
#include "distill.hpp"

using namespace b2fil;
using namespace b2fil::distill;

namespace {

int invalid(const char* text) { return report_error(B2FIL_ERR_INVALID_ARG, text); }

int cuda_failed(const char* what, cudaError_t e)
{
  char text[256];
  std::snprintf(text, sizeof text, "%s: %s", what, cudaGetErrorString(e));
  return report_error(B2FIL_ERR_CUDA, text);
}

constexpr int kDevices = 64;
std::atomic<int> g_sms[kDevices];

// Streaming multiprocessors of a device, or a negative error code.
int sms_of(int device)
{
  if (device < 0 || device >= kDevices) return invalid("device_id out of range");
  int n = g_sms[device].load(std::memory_order_relaxed);
  if (n > 0) return n;
  const cudaError_t e = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return cuda_failed("device_id", e);
  }
  g_sms[device].store(n, std::memory_order_relaxed);
  return n;
}

// Makes a device current and puts the previous one back.  Also where it is current already: only this call
// gives a thread that has not used the device yet (autograd's, in a process's first backward pass) the
// context that encoding a tensor map needs.
struct OnDevice {
  int prev = -1;
  bool ok  = true;
  explicit OnDevice(int device)
  {
    if (cudaGetDevice(&prev) != cudaSuccess || prev == device) prev = -1;
    ok = cudaSetDevice(device) == cudaSuccess;
  }
  ~OnDevice()
  {
    if (prev >= 0) cudaSetDevice(prev);
  }
};

size_t type_bytes(int dtype)
{
  return dtype == B2FIL_TYPE_F64 ? 8 : dtype == B2FIL_TYPE_F32 ? 4 : dtype == B2FIL_TYPE_BF16 || dtype == B2FIL_TYPE_F16 ? 2 : 0;
}
bool aligned(const void* p, size_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

int check_workspace(const void* workspace, int64_t has, int64_t needs)
{
  if (needs < 0) return static_cast<int>(needs);
  if (needs > 0 && (!workspace || !aligned(workspace, 256))) return invalid("workspace is NULL or not 256-byte aligned");
  if (has < needs) return invalid("workspace is too small");
  return B2FIL_OK;
}

int check_teacher(const b2fil_teacher* t, int64_t n_rows, Teacher& out)
{
  if (!t) return invalid("teacher is NULL");
  if (t->k < 1 || t->k > B2FIL_MOST_TOP) return invalid("the teacher's k must be 1 to 256");
  if ((!t->index && n_rows > 0) || !aligned(t->index, t->index64 ? 8 : 4) || !aligned(t->values, 4) || !aligned(t->logsumexp, 4))
    return invalid("the teacher's index is NULL, or one of its arrays is not aligned to its elements");
  out = Teacher{t->values, t->index, t->logsumexp, t->values_stride, t->index_stride, t->k, t->index64 != 0, t->ignore};
  return B2FIL_OK;
}

int check_temperature(double t)
{
  // (1 / T and T^2 stay ordinary 32-bit numbers)
  return t >= 1e-6 && t <= 1e6 ? B2FIL_OK : invalid("temperature must be between 1e-6 and 1e6");
}

int check_top(int dtype, int64_t n_rows, int64_t n_cols, int k)
{
  if (!type_bytes(dtype)) return invalid("unknown element type");
  if (n_rows < 0 || n_cols < 1 || n_cols > INT32_MAX) return invalid("n_rows is negative, or n_cols is not in 1 to 2^31 - 1");
  if (k < 1 || k > n_cols || k > B2FIL_MOST_TOP) return invalid("k must be 1 to min(n_cols, 256)");
  return B2FIL_OK;
}

int check_loss(int dtype, int64_t n_rows, int64_t n_cols, int k)
{
  if (dtype == B2FIL_TYPE_F64 || !type_bytes(dtype)) return invalid("logits must be fp32, bf16 or fp16");
  if (n_rows < 0 || n_cols < 1 || n_cols > INT32_MAX) return invalid("n_rows is negative, or n_cols is not in 1 to 2^31 - 1");
  if (k < 1 || k > B2FIL_MOST_TOP) return invalid("the teacher's k must be 1 to 256");
  return B2FIL_OK;
}

int check_linear(int dtype, int64_t n_rows, int64_t n_cols, int64_t width, int k)
{
  if (dtype != B2FIL_TYPE_BF16 && dtype != B2FIL_TYPE_F16) return invalid("a linear layer must be bf16 or fp16");
  if (n_rows < 0 || n_rows >= INT32_MAX - 256 || n_cols < 1 || n_cols >= INT32_MAX - 256)
    return invalid("n_rows is not in 0 to 2^31 - 257, or n_cols not in 1 to 2^31 - 257");
  if (width < 1 || width > (1 << 20)) return invalid("width must be 1 to 2^20");
  if (k < 1 || k > B2FIL_MOST_TOP) return invalid("the teacher's k must be 1 to 256");
  return B2FIL_OK;
}

int check_layer(const void* hidden, int64_t hidden_stride, const void* weight, int64_t weight_stride, int64_t n_rows, int64_t width)
{
  if ((!hidden && n_rows > 0) || !weight) return invalid("NULL buffer");
  if (!aligned(hidden, 2) || !aligned(weight, 2)) return invalid("hidden or weight is not aligned to its elements");
  if (hidden_stride < width || weight_stride < width || hidden_stride > (1ll << 32) || weight_stride > (1ll << 32))
    return invalid("a row stride is smaller than width, or above 2^32");
  return B2FIL_OK;
}

int64_t rounded(size_t bytes) { return static_cast<int64_t>((bytes + 255) / 256 * 256); }

int finish(const char* what, cudaError_t e) { return e == cudaSuccess ? B2FIL_OK : cuda_failed(what, e); }

}  // namespace

extern "C" {

int64_t b2fil_top_scores_workspace(int dtype, int64_t n_rows, int64_t n_cols, int k, int device_id)
{
  int rc = check_top(dtype, n_rows, n_cols, k);
  if (rc != B2FIL_OK) return rc;
  const int sms = sms_of(device_id);
  if (sms < 0) return sms;
  TopArgs a{};
  a.n_rows = n_rows;
  a.n_cols = n_cols;
  a.k      = k;
  return rounded(n_rows ? top_workspace(dtype, a, sms) : 0);
}

int b2fil_top_scores(int dtype, const void* scores, int64_t n_rows, int64_t n_cols, int64_t row_stride, int k,
                     int probabilities, double temperature, void* values, int32_t* index, void* logsumexp, void* workspace,
                     int64_t workspace_bytes, int device_id, void* cuda_stream)
{
  int rc = check_top(dtype, n_rows, n_cols, k);
  if (rc == B2FIL_OK) rc = check_temperature(temperature);
  if (rc != B2FIL_OK) return rc;
  if (n_rows == 0) return B2FIL_OK;
  if (!scores || !values || !index) return invalid("NULL buffer");
  const size_t e = type_bytes(dtype);
  if (!aligned(scores, e) || !aligned(values, e) || !aligned(index, 4) || !aligned(logsumexp, e == 8 ? 8 : 4))
    return invalid("a buffer is not aligned to its elements");
  if (row_stride < n_cols && n_rows > 1) return invalid("row_stride is smaller than n_cols");
  rc = check_workspace(workspace, workspace_bytes, b2fil_top_scores_workspace(dtype, n_rows, n_cols, k, device_id));
  if (rc != B2FIL_OK) return rc;
  OnDevice on(device_id);
  if (!on.ok) return invalid("device_id cannot be made current");
  const TopArgs a{scores, n_rows, n_cols, row_stride, k, probabilities != 0, 1.0 / temperature, values, index, logsumexp};
  return finish("b2fil_top_scores",
                launch_top(dtype, a, workspace, sms_of(device_id), static_cast<cudaStream_t>(cuda_stream)));
}

int64_t b2fil_distill_loss_workspace(int dtype, int64_t n_rows, int64_t n_cols, int k, int device_id)
{
  int rc = check_loss(dtype, n_rows, n_cols, k);
  if (rc != B2FIL_OK) return rc;
  const int sms = sms_of(device_id);
  if (sms < 0) return sms;
  LossArgs a{};
  a.n_rows    = n_rows;
  a.n_cols    = n_cols;
  a.teacher.k = k;
  return rounded(loss_workspace(a, sms));
}

int b2fil_distill_loss(int dtype, const void* logits, int64_t n_rows, int64_t n_cols, int64_t row_stride,
                       const b2fil_teacher* teacher, double temperature, int reduction, float* row_loss, float* row_stats,
                       float* named_p, int32_t* named_at, float* loss, float* factor, void* workspace,
                       int64_t workspace_bytes, int device_id, void* cuda_stream)
{
  LossArgs a{};
  int rc = check_teacher(teacher, n_rows, a.teacher);
  if (rc == B2FIL_OK) rc = check_loss(dtype, n_rows, n_cols, a.teacher.k);
  if (rc == B2FIL_OK) rc = check_temperature(temperature);
  if (rc != B2FIL_OK) return rc;
  if (reduction < B2FIL_REDUCE_NONE || reduction > B2FIL_REDUCE_MEAN) return invalid("unknown reduction");
  if (reduction != B2FIL_REDUCE_NONE && (!loss || !factor || !aligned(loss, 4) || !aligned(factor, 4)))
    return invalid("a reduced loss needs loss and factor, aligned to their elements");
  if (n_rows > 0 && (!logits || !row_loss || !row_stats || !named_p || !named_at)) return invalid("NULL buffer");
  if (!aligned(logits, type_bytes(dtype)) || !aligned(row_stats, 16) || !aligned(row_loss, 4) || !aligned(named_p, 4) ||
      !aligned(named_at, 4))
    return invalid("a buffer is not aligned");
  if (row_stride < n_cols && n_rows > 1) return invalid("row_stride is smaller than n_cols");
  if (a.teacher.logsumexp && n_cols > (1 << 20)) return invalid("the teacher's logsumexp needs n_cols <= 2^20");
  rc = check_workspace(workspace, workspace_bytes, b2fil_distill_loss_workspace(dtype, n_rows, n_cols, a.teacher.k, device_id));
  if (rc != B2FIL_OK) return rc;
  OnDevice on(device_id);
  if (!on.ok) return invalid("device_id cannot be made current");
  a.logits      = logits;
  a.n_rows      = n_rows;
  a.n_cols      = n_cols;
  a.row_stride  = row_stride;
  a.temperature = Temperature(temperature);
  a.row_loss    = row_loss;
  a.row_stats   = reinterpret_cast<float4*>(row_stats);
  a.named       = Named{nullptr, named_p, named_at};
  return finish("b2fil_distill_loss", launch_loss(dtype, a, Reduced{reduction, loss, factor}, workspace,
                                                  sms_of(device_id), static_cast<cudaStream_t>(cuda_stream)));
}

int b2fil_distill_loss_grad(int dtype, const void* logits, int64_t n_rows, int64_t n_cols, int64_t row_stride,
                            int k, double temperature, const float* row_stats, const float* named_p,
                            const int32_t* named_at, const float* upstream, int64_t upstream_stride, const float* factor,
                            void* grad, int64_t grad_stride, int device_id, void* cuda_stream)
{
  LossGradArgs g{};
  LossArgs& a = g.fwd;
  int rc      = check_loss(dtype, n_rows, n_cols, k);
  if (rc == B2FIL_OK) rc = check_temperature(temperature);
  if (rc != B2FIL_OK) return rc;
  if (n_rows == 0) return B2FIL_OK;
  if (!logits || !row_stats || !named_p || !named_at || !upstream || !grad) return invalid("NULL buffer");
  if (!aligned(logits, type_bytes(dtype)) || !aligned(grad, type_bytes(dtype)) || !aligned(row_stats, 16) ||
      !aligned(named_p, 4) || !aligned(named_at, 4) || !aligned(upstream, 4) || !aligned(factor, 4))
    return invalid("a buffer is not aligned");
  if ((row_stride < n_cols || grad_stride < n_cols) && n_rows > 1) return invalid("a row stride is smaller than n_cols");
  const int sms = sms_of(device_id);
  if (sms < 0) return sms;
  OnDevice on(device_id);
  if (!on.ok) return invalid("device_id cannot be made current");
  a.logits          = logits;
  a.n_rows          = n_rows;
  a.n_cols          = n_cols;
  a.row_stride      = row_stride;
  a.temperature     = Temperature(temperature);
  a.row_stats       = const_cast<float4*>(reinterpret_cast<const float4*>(row_stats));
  a.teacher.k       = k;
  a.named           = Named{nullptr, const_cast<float*>(named_p), const_cast<int32_t*>(named_at)};
  g.upstream        = upstream;
  g.upstream_stride = upstream_stride;
  g.factor          = factor;
  g.grad            = grad;
  g.grad_stride     = grad_stride;
  return finish("b2fil_distill_loss_grad", launch_loss_grad(dtype, g, sms, static_cast<cudaStream_t>(cuda_stream)));
}

int64_t b2fil_linear_loss_workspace(int dtype, const void* hidden, int64_t hidden_stride, const void* weight,
                                    int64_t weight_stride, int64_t n_rows, int64_t n_cols, int64_t width, int k, int device_id)
{
  int rc = check_linear(dtype, n_rows, n_cols, width, k);
  if (rc == B2FIL_OK) rc = check_layer(hidden, hidden_stride, weight, weight_stride, n_rows, width);
  if (rc != B2FIL_OK) return rc;
  const int sms = sms_of(device_id);
  if (sms < 0) return sms;
  LinearArgs a{};
  a.hidden        = hidden;
  a.weight        = weight;
  a.hidden_stride = hidden_stride;
  a.weight_stride = weight_stride;
  a.n_rows        = n_rows;
  a.n_cols        = n_cols;
  a.width         = width;
  a.teacher.k     = k;
  return rounded(linear_workspace(a, sms));
}

int b2fil_linear_loss(int dtype, const void* hidden, int64_t hidden_stride, const void* weight, int64_t weight_stride,
                      int64_t n_rows, int64_t n_cols, int64_t width, const b2fil_teacher* teacher, double temperature,
                      int reduction, float* row_loss, float* row_stats, float* named_logit, float* named_p, int32_t* named_at,
                      float* loss, float* factor, void* workspace, int64_t workspace_bytes, int device_id, void* cuda_stream)
{
  LinearArgs a{};
  int rc = check_teacher(teacher, n_rows, a.teacher);
  if (rc == B2FIL_OK) rc = check_linear(dtype, n_rows, n_cols, width, a.teacher.k);
  if (rc == B2FIL_OK) rc = check_temperature(temperature);
  if (rc == B2FIL_OK) rc = check_layer(hidden, hidden_stride, weight, weight_stride, n_rows, width);
  if (rc != B2FIL_OK) return rc;
  if (a.teacher.logsumexp) return invalid("the loss of a linear layer takes no logsumexp of the teacher");
  if (reduction < B2FIL_REDUCE_NONE || reduction > B2FIL_REDUCE_MEAN) return invalid("unknown reduction");
  if (reduction != B2FIL_REDUCE_NONE && (!loss || !factor || !aligned(loss, 4) || !aligned(factor, 4)))
    return invalid("a reduced loss needs loss and factor, aligned to their elements");
  if (n_rows > 0 && (!row_loss || !row_stats || !named_logit || !named_p || !named_at)) return invalid("NULL buffer");
  if (!aligned(row_stats, 16) || !aligned(row_loss, 4) || !aligned(named_logit, 4) || !aligned(named_p, 4) || !aligned(named_at, 4))
    return invalid("a buffer is not aligned");
  rc = check_workspace(workspace, workspace_bytes, b2fil_linear_loss_workspace(dtype, hidden, hidden_stride, weight, weight_stride, n_rows, n_cols,
                                                                             width, a.teacher.k, device_id));
  if (rc != B2FIL_OK) return rc;
  OnDevice on(device_id);
  if (!on.ok) return invalid("device_id cannot be made current");
  a.hidden        = hidden;
  a.weight        = weight;
  a.n_rows        = n_rows;
  a.n_cols        = n_cols;
  a.width         = width;
  a.hidden_stride = hidden_stride;
  a.weight_stride = weight_stride;
  a.temperature   = Temperature(temperature);
  a.row_loss      = row_loss;
  a.row_stats     = reinterpret_cast<float4*>(row_stats);
  a.named         = Named{named_logit, named_p, named_at};
  return finish("b2fil_linear_loss", launch_linear(dtype, a, Reduced{reduction, loss, factor}, workspace,
                                                   sms_of(device_id), static_cast<cudaStream_t>(cuda_stream)));
}

int64_t b2fil_linear_loss_grad_workspace(int dtype, const void* hidden, int64_t hidden_stride, const void* weight,
                                         int64_t weight_stride, int64_t n_rows, int64_t n_cols, int64_t width, int k,
                                         int wants_hidden, int wants_weight, int device_id)
{
  int rc = check_linear(dtype, n_rows, n_cols, width, k);
  if (rc == B2FIL_OK) rc = check_layer(hidden, hidden_stride, weight, weight_stride, n_rows, width);
  if (rc != B2FIL_OK) return rc;
  const int sms = sms_of(device_id);
  if (sms < 0) return sms;
  LinearGradArgs g{};
  g.fwd.hidden        = hidden;
  g.fwd.weight        = weight;
  g.fwd.hidden_stride = hidden_stride;
  g.fwd.weight_stride = weight_stride;
  g.fwd.n_rows        = n_rows;
  g.fwd.n_cols        = n_cols;
  g.fwd.width         = width;
  g.fwd.teacher.k     = k;
  char some;
  g.grad_hidden = wants_hidden ? &some : nullptr;
  g.grad_weight = wants_weight ? &some : nullptr;
  return n_rows && (wants_hidden || wants_weight) ? rounded(linear_grad_workspace(g, sms)) : 0;
}

int b2fil_linear_loss_grad(int dtype, const void* hidden, int64_t hidden_stride, const void* weight, int64_t weight_stride,
                           int64_t n_rows, int64_t n_cols, int64_t width, int k, double temperature, const float* row_stats,
                           const float* named_logit, const float* named_p, const int32_t* named_at, const float* upstream,
                           int64_t upstream_stride, const float* factor, void* grad_hidden, void* grad_weight,
                           void* workspace, int64_t workspace_bytes, int device_id, void* cuda_stream)
{
  LinearGradArgs g{};
  LinearArgs& a = g.fwd;
  int rc        = check_linear(dtype, n_rows, n_cols, width, k);
  if (rc == B2FIL_OK) rc = check_temperature(temperature);
  if (rc == B2FIL_OK) rc = check_layer(hidden, hidden_stride, weight, weight_stride, n_rows, width);
  if (rc != B2FIL_OK) return rc;
  if (!grad_hidden && !grad_weight) return B2FIL_OK;
  if (n_rows > 0 && (!row_stats || !named_logit || !named_p || !named_at || !upstream)) return invalid("NULL buffer");
  if (!aligned(row_stats, 16) || !aligned(named_logit, 4) || !aligned(named_p, 4) || !aligned(named_at, 4) ||
      !aligned(upstream, 4) || !aligned(factor, 4) || !aligned(grad_hidden, 16) || !aligned(grad_weight, 16))
    return invalid("a buffer is not aligned");
  rc = check_workspace(workspace, workspace_bytes,
                       b2fil_linear_loss_grad_workspace(dtype, hidden, hidden_stride, weight, weight_stride, n_rows, n_cols,
                                                        width, k, grad_hidden != nullptr, grad_weight != nullptr, device_id));
  if (rc != B2FIL_OK) return rc;
  const int sms = sms_of(device_id);
  if (sms < 0) return sms;
  OnDevice on(device_id);
  if (!on.ok) return invalid("device_id cannot be made current");
  const cudaStream_t s = static_cast<cudaStream_t>(cuda_stream);
  if (n_rows == 0)
    return finish("b2fil_linear_loss_grad", grad_weight ? cudaMemsetAsync(grad_weight, 0, n_cols * width * 2, s) : cudaSuccess);
  a.hidden          = hidden;
  a.weight          = weight;
  a.n_rows          = n_rows;
  a.n_cols          = n_cols;
  a.width           = width;
  a.hidden_stride   = hidden_stride;
  a.weight_stride   = weight_stride;
  a.teacher.k       = k;
  a.temperature     = Temperature(temperature);
  a.row_stats       = const_cast<float4*>(reinterpret_cast<const float4*>(row_stats));
  a.named           = Named{const_cast<float*>(named_logit), const_cast<float*>(named_p), const_cast<int32_t*>(named_at)};
  g.upstream        = upstream;
  g.upstream_stride = upstream_stride;
  g.factor          = factor;
  g.grad_hidden     = grad_hidden;
  g.grad_weight     = grad_weight;
  return finish("b2fil_linear_loss_grad", launch_linear_grad(dtype, g, workspace, sms, s));
}

int b2fil_distill_status(int device_id, int32_t* status)
{
  if (!status) return invalid("status is NULL");
  *status       = 0;
  const int sms = sms_of(device_id);
  if (sms < 0) return sms;
  OnDevice on(device_id);
  if (!on.ok) return invalid("device_id cannot be made current");
  int word            = 0;
  const cudaError_t e = linear_status(&word);
  if (e != cudaSuccess) return cuda_failed("b2fil_distill_status", e);
  *status = word;
  return word ? report_error(B2FIL_ERR_TIMEOUT, "a bounded wait inside a kernel of the linear loss ran out") : B2FIL_OK;
}

int b2fil_distill_selftest_timeout(int device_id, void* cuda_stream)
{
  const int sms = sms_of(device_id);
  if (sms < 0) return sms;
  OnDevice on(device_id);
  if (!on.ok) return invalid("device_id cannot be made current");
  return finish("b2fil_distill_selftest_timeout", launch_linear_timeout(static_cast<cudaStream_t>(cuda_stream)));
}

}  // extern "C"
