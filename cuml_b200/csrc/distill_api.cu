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

// Makes a device current and puts the previous one back.
struct OnDevice {
  int prev = -1;
  bool ok  = true;
  explicit OnDevice(int device)
  {
    if (cudaGetDevice(&prev) != cudaSuccess) prev = -1;
    if (prev == device)
      prev = -1;
    else
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
                       float* loss, float* factor, void* workspace, int64_t workspace_bytes, int device_id,
                       void* cuda_stream)
{
  LossArgs a{};
  int rc = check_teacher(teacher, n_rows, a.teacher);
  if (rc == B2FIL_OK) rc = check_loss(dtype, n_rows, n_cols, a.teacher.k);
  if (rc == B2FIL_OK) rc = check_temperature(temperature);
  if (rc != B2FIL_OK) return rc;
  if (reduction < B2FIL_REDUCE_NONE || reduction > B2FIL_REDUCE_MEAN) return invalid("unknown reduction");
  if (reduction != B2FIL_REDUCE_NONE && (!loss || !factor)) return invalid("a reduced loss needs loss and factor");
  if (n_rows > 0 && (!logits || !row_loss || !row_stats)) return invalid("NULL buffer");
  if (!aligned(logits, type_bytes(dtype)) || !aligned(row_stats, 16) || !aligned(row_loss, 4))
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
  a.temperature = static_cast<float>(temperature);
  a.row_loss    = row_loss;
  a.row_stats   = reinterpret_cast<float4*>(row_stats);
  return finish("b2fil_distill_loss", launch_loss(dtype, a, Reduced{reduction, loss, factor}, workspace,
                                                  sms_of(device_id), static_cast<cudaStream_t>(cuda_stream)));
}

int b2fil_distill_loss_grad(int dtype, const void* logits, int64_t n_rows, int64_t n_cols, int64_t row_stride,
                            const b2fil_teacher* teacher, double temperature, const float* row_stats, const float* upstream,
                            int64_t upstream_stride, const float* factor, void* grad, int64_t grad_stride, int device_id,
                            void* cuda_stream)
{
  LossGradArgs g{};
  LossArgs& a = g.fwd;
  int rc      = check_teacher(teacher, n_rows, a.teacher);
  if (rc == B2FIL_OK) rc = check_loss(dtype, n_rows, n_cols, a.teacher.k);
  if (rc == B2FIL_OK) rc = check_temperature(temperature);
  if (rc != B2FIL_OK) return rc;
  if (n_rows == 0) return B2FIL_OK;
  if (!logits || !row_stats || !upstream || !grad) return invalid("NULL buffer");
  if (!aligned(logits, type_bytes(dtype)) || !aligned(grad, type_bytes(dtype)) || !aligned(row_stats, 16))
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
  a.temperature     = static_cast<float>(temperature);
  a.row_stats       = const_cast<float4*>(reinterpret_cast<const float4*>(row_stats));
  g.upstream        = upstream;
  g.upstream_stride = upstream_stride;
  g.factor          = factor;
  g.grad            = grad;
  g.grad_stride     = grad_stride;
  return finish("b2fil_distill_loss_grad", launch_loss_grad(dtype, g, sms, static_cast<cudaStream_t>(cuda_stream)));
}

}  // extern "C"
