// C ABI of the distillation operators: checks of arguments, then one launcher each.  Nothing in here
// throws.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdio>
#include <exception>
#include <vector>

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

int check_target(const b2fil_target* t, int64_t n_rows, const float* log_prob, Target& out)
{
  if (!t) return invalid("target is NULL");
  if (!aligned(t->index, t->index64 ? 8 : 4)) return invalid("the target's index is not aligned to its elements");
  if (n_rows > 0 && t->index && !log_prob) return invalid("a target needs log_prob");
  out = Target{t->index, t->stride, t->ignore, t->index64 != 0};
  return B2FIL_OK;
}

int check_scores(const float* log_prob, const float* entropy, const float* kept, int64_t n_rows)
{
  if (n_rows > 0 && (!entropy || !kept)) return invalid("NULL buffer");
  if (!aligned(log_prob, 4) || !aligned(entropy, 4) || !aligned(kept, 16)) return invalid("a buffer is not aligned");
  return B2FIL_OK;
}

int check_upstream(const float* of_log_prob, const float* of_entropy)
{
  return aligned(of_log_prob, 4) && aligned(of_entropy, 4) ? B2FIL_OK : invalid("a buffer is not aligned");
}

int check_gradients(const b2fil_gradient* g, int64_t n, bool scales)
{
  if (n < 0 || n > (1 << 24) || (n > 0 && !g)) return invalid("n is not in 0 to 2^24, or gradients is NULL");
  for (int64_t i = 0; i < n; ++i) {
    const b2fil_gradient& x = g[i];
    const size_t e = type_bytes(x.from_type), o = type_bytes(x.to_type);
    if (e == 0 || e == 8) return invalid("gradients must be fp32, bf16 or fp16");
    if (x.rows < 0 || x.cols < 0 || x.rows > (1ll << 40) || x.cols > (1ll << 40) || (x.rows && x.cols > (1ll << 40) / x.rows))
      return invalid("a gradient's sizes are negative, or it has more than 2^40 elements");
    if (x.rows == 0 || x.cols == 0) continue;
    if (x.from_row < 0 || x.from_col < 0 || x.to_row < 0 || x.to_col < 0) return invalid("a gradient's stride is negative");
    if (!x.from || !aligned(x.from, e)) return invalid("a gradient is NULL or not aligned to its elements");
    if (!scales) continue;
    if (o == 0 || o == 8) return invalid("gradients must be fp32, bf16 or fp16");
    if (!x.to || !aligned(x.to, o)) return invalid("a scaled gradient is NULL or not aligned to its elements");
    if (x.to == x.from && (x.from_type != x.to_type || (x.cols > 1 && x.from_col != x.to_col) || (x.rows > 1 && x.from_row != x.to_row)))
      return invalid("a gradient that is scaled in place has one type and layout");
  }
  return B2FIL_OK;
}

// An address range that is written, or read and not written in place.
struct Region {
  uintptr_t low, high;
  const b2fil_gradient* of;
  bool written;
  int64_t row, row_bytes;  // bytes from one row to the next, and of a row
};
Region region_of(const b2fil_gradient& g, bool written)
{
  const int64_t e = type_bytes(written ? g.to_type : g.from_type), row = (written ? g.to_row : g.from_row) * e,
                col = (written ? g.to_col : g.from_col) * e;
  const uintptr_t low = reinterpret_cast<uintptr_t>(written ? g.to : g.from);
  const int64_t rows_span = (g.rows - 1) * row, cols_span = (g.cols - 1) * col;
  const bool by_rows = rows_span >= cols_span;  // the longer step between what is then a row
  return Region{low, low + rows_span + cols_span + e, &g, written, by_rows ? row : col, (by_rows ? cols_span : rows_span) + e};
}
// Rows of one stride that lie side by side.
bool side_by_side(const Region& a, const Region& b)
{
  if (a.row != b.row || a.row <= 0) return false;
  const int64_t apart = static_cast<int64_t>((b.low - a.low) % static_cast<uintptr_t>(a.row));  // (b begins behind a)
  return apart >= a.row_bytes && apart + b.row_bytes <= a.row;
}

int check_overlap(const b2fil_gradient* g, int64_t n)
{
  std::vector<Region> regions;
  try {
    regions.reserve(2 * n);
  } catch (const std::exception&) {
    return report_error(B2FIL_ERR_NO_MEMORY, "no memory for the list of gradients");
  }
  for (int64_t i = 0; i < n; ++i) {
    if (g[i].rows == 0 || g[i].cols == 0) continue;
    const Region to = region_of(g[i], true);
    if ((g[i].rows > 1 && g[i].to_row == 0) || (g[i].cols > 1 && g[i].to_col == 0) || (to.row < to.row_bytes && g[i].rows > 1 && g[i].cols > 1))
      return invalid("the elements of a scaled gradient overlap in memory");
    regions.push_back(to);
    if (g[i].to != g[i].from) regions.push_back(region_of(g[i], false));
  }
  auto before = [](const Region& a, const Region& b) { return a.low < b.low; };
  if (!std::is_sorted(regions.begin(), regions.end(), before)) std::sort(regions.begin(), regions.end(), before);
  std::vector<const Region*> open;  // those that a later one may begin in
  try {
    open.reserve(regions.size());
  } catch (const std::exception&) {
    return report_error(B2FIL_ERR_NO_MEMORY, "no memory for the list of gradients");
  }
  for (const Region& r : regions) {
    size_t kept = 0;
    for (const Region* o : open) {
      if (o->high <= r.low) continue;
      open[kept++] = o;
      if (!(o->written || r.written) || (o->of->tensor == r.of->tensor && o->written == r.written) || side_by_side(*o, r)) continue;
      return invalid("gradients overlap in memory");
    }
    open.resize(kept);
    open.push_back(&r);
  }
  return B2FIL_OK;
}

ClipArgs clip_args(const std::vector<Gradient>& g, int kind, bool scales, double most, float* norm)
{
  return ClipArgs{g.data(), static_cast<int64_t>(g.size()), kind, scales, most, norm};
}

// False: no memory.
bool give_gradients(const b2fil_gradient* from, int64_t n, std::vector<Gradient>& to)
{
  try {
    to.reserve(n);
  } catch (const std::exception&) {
    return false;
  }
  for (int64_t i = 0; i < n; ++i) {
    const b2fil_gradient& x = from[i];
    to.push_back(Gradient{x.from, x.to, x.rows, x.cols, x.from_row, x.from_col, x.to_row, x.to_col, x.from_type, x.to_type});
  }
  return true;
}

int64_t rounded(size_t bytes) { return static_cast<int64_t>((bytes + 255) / 256 * 256); }

LinearArgs layer_args(const void* hidden, int64_t hidden_stride, const void* weight, int64_t weight_stride, int64_t n_rows,
                      int64_t n_cols, int64_t width)
{
  LinearArgs a{};
  a.hidden        = hidden;
  a.weight        = weight;
  a.n_rows        = n_rows;
  a.n_cols        = n_cols;
  a.width         = width;
  a.hidden_stride = hidden_stride;
  a.weight_stride = weight_stride;
  return a;
}

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

int64_t b2fil_log_probs_workspace(int dtype, int64_t n_rows, int64_t n_cols, int k, int device_id)
{
  int rc = check_loss(dtype, n_rows, n_cols, 1);
  if (rc != B2FIL_OK) return rc;
  if (k < 0 || k > n_cols || k > B2FIL_MOST_TOP) return invalid("k must be 0 to min(n_cols, 256)");
  const int sms = sms_of(device_id);
  if (sms < 0) return sms;
  ScoreArgs a{};
  a.n_rows = n_rows;
  a.n_cols = n_cols;
  a.k      = k;
  return n_rows ? rounded(score_workspace(dtype, a, sms)) : 0;
}

int b2fil_log_probs(int dtype, const void* logits, int64_t n_rows, int64_t n_cols, int64_t row_stride,
                    const b2fil_target* target, double temperature, int k, float* log_prob, float* entropy, float* kept,
                    float* top, int32_t* top_index, void* workspace, int64_t workspace_bytes, int device_id,
                    void* cuda_stream)
{
  ScoreArgs a{};
  int rc = check_target(target, n_rows, log_prob, a.target);
  if (rc == B2FIL_OK) rc = check_loss(dtype, n_rows, n_cols, 1);
  if (rc == B2FIL_OK) rc = check_temperature(temperature);
  if (rc == B2FIL_OK) rc = check_scores(log_prob, entropy, kept, n_rows);
  if (rc != B2FIL_OK) return rc;
  if (k < 0 || k > n_cols || k > B2FIL_MOST_TOP) return invalid("k must be 0 to min(n_cols, 256)");
  if (n_rows == 0) return B2FIL_OK;
  if (!logits || (k > 0 && (!top || !top_index))) return invalid("NULL buffer");
  if (!aligned(logits, type_bytes(dtype)) || !aligned(top, 4) || !aligned(top_index, 4)) return invalid("a buffer is not aligned");
  if (row_stride < n_cols && n_rows > 1) return invalid("row_stride is smaller than n_cols");
  rc = check_workspace(workspace, workspace_bytes, b2fil_log_probs_workspace(dtype, n_rows, n_cols, k, device_id));
  if (rc != B2FIL_OK) return rc;
  OnDevice on(device_id);
  if (!on.ok) return invalid("device_id cannot be made current");
  a.logits      = logits;
  a.n_rows      = n_rows;
  a.n_cols      = n_cols;
  a.row_stride  = row_stride;
  a.temperature = Temperature(temperature);
  a.out         = Scores{a.target.index ? log_prob : nullptr, entropy, reinterpret_cast<float4*>(kept)};
  a.k           = k;
  a.top         = top;
  a.top_index   = top_index;
  return finish("b2fil_log_probs", launch_score(dtype, a, workspace, sms_of(device_id), static_cast<cudaStream_t>(cuda_stream)));
}

int b2fil_log_probs_grad(int dtype, const void* logits, int64_t n_rows, int64_t n_cols, int64_t row_stride,
                         double temperature, const float* kept, const float* of_log_prob, int64_t of_log_prob_stride,
                         const float* of_entropy, int64_t of_entropy_stride, void* grad, int64_t grad_stride,
                         int device_id, void* cuda_stream)
{
  int rc = check_loss(dtype, n_rows, n_cols, 1);
  if (rc == B2FIL_OK) rc = check_temperature(temperature);
  if (rc == B2FIL_OK) rc = check_upstream(of_log_prob, of_entropy);
  if (rc != B2FIL_OK) return rc;
  if (n_rows == 0) return B2FIL_OK;
  if (!logits || !kept || !grad) return invalid("NULL buffer");
  if (!aligned(logits, type_bytes(dtype)) || !aligned(grad, type_bytes(dtype)) || !aligned(kept, 16))
    return invalid("a buffer is not aligned");
  if ((row_stride < n_cols || grad_stride < n_cols) && n_rows > 1) return invalid("a row stride is smaller than n_cols");
  const int sms = sms_of(device_id);
  if (sms < 0) return sms;
  OnDevice on(device_id);
  if (!on.ok) return invalid("device_id cannot be made current");
  ScoreGradArgs g{};
  g.fwd.logits      = logits;
  g.fwd.n_rows      = n_rows;
  g.fwd.n_cols      = n_cols;
  g.fwd.row_stride  = row_stride;
  g.fwd.temperature = Temperature(temperature);
  g.fwd.out.kept    = const_cast<float4*>(reinterpret_cast<const float4*>(kept));
  g.upstream        = ScoreUpstream{of_log_prob, of_entropy, of_log_prob_stride, of_entropy_stride};
  g.grad            = grad;
  g.grad_stride     = grad_stride;
  return finish("b2fil_log_probs_grad", launch_score_grad(dtype, g, sms, static_cast<cudaStream_t>(cuda_stream)));
}

int64_t b2fil_linear_log_probs_workspace(int dtype, const void* hidden, int64_t hidden_stride, const void* weight,
                                         int64_t weight_stride, int64_t n_rows, int64_t n_cols, int64_t width,
                                         int device_id)
{
  int rc = check_linear(dtype, n_rows, n_cols, width, 1);
  if (rc == B2FIL_OK) rc = check_layer(hidden, hidden_stride, weight, weight_stride, n_rows, width);
  if (rc != B2FIL_OK) return rc;
  const int sms = sms_of(device_id);
  if (sms < 0) return sms;
  LinearScoreArgs a{};
  a.layer = layer_args(hidden, hidden_stride, weight, weight_stride, n_rows, n_cols, width);
  return n_rows ? rounded(linear_score_workspace(a, sms)) : 0;
}

int b2fil_linear_log_probs(int dtype, const void* hidden, int64_t hidden_stride, const void* weight,
                           int64_t weight_stride, int64_t n_rows, int64_t n_cols, int64_t width,
                           const b2fil_target* target, double temperature, float* log_prob, float* entropy, float* kept,
                           void* workspace, int64_t workspace_bytes, int device_id, void* cuda_stream)
{
  LinearScoreArgs a{};
  int rc = check_target(target, n_rows, log_prob, a.target);
  if (rc == B2FIL_OK) rc = check_linear(dtype, n_rows, n_cols, width, 1);
  if (rc == B2FIL_OK) rc = check_temperature(temperature);
  if (rc == B2FIL_OK) rc = check_layer(hidden, hidden_stride, weight, weight_stride, n_rows, width);
  if (rc == B2FIL_OK) rc = check_scores(log_prob, entropy, kept, n_rows);
  if (rc != B2FIL_OK) return rc;
  if (n_rows == 0) return B2FIL_OK;
  rc = check_workspace(workspace, workspace_bytes, b2fil_linear_log_probs_workspace(dtype, hidden, hidden_stride, weight, weight_stride,
                                                                                   n_rows, n_cols, width, device_id));
  if (rc != B2FIL_OK) return rc;
  OnDevice on(device_id);
  if (!on.ok) return invalid("device_id cannot be made current");
  a.layer             = layer_args(hidden, hidden_stride, weight, weight_stride, n_rows, n_cols, width);
  a.layer.temperature = Temperature(temperature);
  a.out               = Scores{a.target.index ? log_prob : nullptr, entropy, reinterpret_cast<float4*>(kept)};
  return finish("b2fil_linear_log_probs",
                launch_linear_score(dtype, a, workspace, sms_of(device_id), static_cast<cudaStream_t>(cuda_stream)));
}

int64_t b2fil_linear_log_probs_grad_workspace(int dtype, const void* hidden, int64_t hidden_stride, const void* weight,
                                              int64_t weight_stride, int64_t n_rows, int64_t n_cols, int64_t width,
                                              int wants_hidden, int wants_weight, int device_id)
{
  int rc = check_linear(dtype, n_rows, n_cols, width, 1);
  if (rc == B2FIL_OK) rc = check_layer(hidden, hidden_stride, weight, weight_stride, n_rows, width);
  if (rc != B2FIL_OK) return rc;
  const int sms = sms_of(device_id);
  if (sms < 0) return sms;
  LinearScoreGradArgs g{};
  char some;
  g.fwd.layer   = layer_args(hidden, hidden_stride, weight, weight_stride, n_rows, n_cols, width);
  g.grad_hidden = wants_hidden ? &some : nullptr;
  g.grad_weight = wants_weight ? &some : nullptr;
  return n_rows && (wants_hidden || wants_weight) ? rounded(linear_score_grad_workspace(g, sms)) : 0;
}

int b2fil_linear_log_probs_grad(int dtype, const void* hidden, int64_t hidden_stride, const void* weight,
                                int64_t weight_stride, int64_t n_rows, int64_t n_cols, int64_t width,
                                double temperature, const float* kept, const float* of_log_prob,
                                int64_t of_log_prob_stride, const float* of_entropy, int64_t of_entropy_stride,
                                void* grad_hidden, void* grad_weight, void* workspace, int64_t workspace_bytes,
                                int device_id, void* cuda_stream)
{
  int rc = check_linear(dtype, n_rows, n_cols, width, 1);
  if (rc == B2FIL_OK) rc = check_temperature(temperature);
  if (rc == B2FIL_OK) rc = check_layer(hidden, hidden_stride, weight, weight_stride, n_rows, width);
  if (rc == B2FIL_OK) rc = check_upstream(of_log_prob, of_entropy);
  if (rc != B2FIL_OK) return rc;
  if (!grad_hidden && !grad_weight) return B2FIL_OK;
  if (n_rows > 0 && !kept) return invalid("NULL buffer");
  if (!aligned(kept, 16) || !aligned(grad_hidden, 16) || !aligned(grad_weight, 16)) return invalid("a buffer is not aligned");
  rc = check_workspace(workspace, workspace_bytes,
                       b2fil_linear_log_probs_grad_workspace(dtype, hidden, hidden_stride, weight, weight_stride, n_rows, n_cols,
                                                             width, grad_hidden != nullptr, grad_weight != nullptr, device_id));
  if (rc != B2FIL_OK) return rc;
  const int sms = sms_of(device_id);
  if (sms < 0) return sms;
  OnDevice on(device_id);
  if (!on.ok) return invalid("device_id cannot be made current");
  const cudaStream_t s = static_cast<cudaStream_t>(cuda_stream);
  if (n_rows == 0)
    return finish("b2fil_linear_log_probs_grad", grad_weight ? cudaMemsetAsync(grad_weight, 0, n_cols * width * 2, s) : cudaSuccess);
  LinearScoreGradArgs g{};
  g.fwd.layer             = layer_args(hidden, hidden_stride, weight, weight_stride, n_rows, n_cols, width);
  g.fwd.layer.temperature = Temperature(temperature);
  g.fwd.out.kept          = const_cast<float4*>(reinterpret_cast<const float4*>(kept));
  g.upstream              = ScoreUpstream{of_log_prob, of_entropy, of_log_prob_stride, of_entropy_stride};
  g.grad_hidden           = grad_hidden;
  g.grad_weight           = grad_weight;
  return finish("b2fil_linear_log_probs_grad", launch_linear_score_grad(dtype, g, workspace, sms, s));
}

int64_t b2fil_clip_gradients_workspace(const b2fil_gradient* gradients, int64_t n, int device_id)
{
  int rc = check_gradients(gradients, n, false);
  if (rc != B2FIL_OK) return rc;
  const int sms = sms_of(device_id);
  if (sms < 0) return sms;
  std::vector<Gradient> g;
  if (!give_gradients(gradients, n, g)) return report_error(B2FIL_ERR_NO_MEMORY, "no memory for the list of gradients");
  return rounded(clip_workspace(clip_args(g, 0, false, 0.0, nullptr), sms));
}

int b2fil_clip_gradients(const b2fil_gradient* gradients, int64_t n, int norm_kind, int scales, double most, float* norm,
                         void* workspace, int64_t workspace_bytes, int device_id, void* cuda_stream)
{
  int rc = check_gradients(gradients, n, scales != 0);
  if (rc != B2FIL_OK) return rc;
  if (norm_kind < B2FIL_NORM_LARGEST || norm_kind > B2FIL_NORM_SQUARES) return invalid("unknown kind of norm");
  if (scales && !(most >= 0)) return invalid("the largest norm must be 0 or more");
  if (scales && (rc = check_overlap(gradients, n)) != B2FIL_OK) return rc;
  if (!norm || !aligned(norm, 4)) return invalid("norm is NULL or not aligned");
  const int sms = sms_of(device_id);
  if (sms < 0) return sms;
  std::vector<Gradient> g;
  if (!give_gradients(gradients, n, g)) return report_error(B2FIL_ERR_NO_MEMORY, "no memory for the list of gradients");
  const ClipArgs a = clip_args(g, norm_kind, scales != 0, most, norm);
  rc = check_workspace(workspace, workspace_bytes, rounded(clip_workspace(a, sms)));
  if (rc != B2FIL_OK) return rc;
  OnDevice on(device_id);
  if (!on.ok) return invalid("device_id cannot be made current");
  return finish("b2fil_clip_gradients", launch_clip(a, workspace, sms, static_cast<cudaStream_t>(cuda_stream)));
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
