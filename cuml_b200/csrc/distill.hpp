// Launchers of the distillation kernels (best scores of a row, losses on logits and on a linear
// layer).  All of them enqueue on the given stream of the current device and return the CUDA error
// of the launch.
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace b2fil {

// Sets the calling thread's error text and returns `code` (api.cu).
int report_error(int code, const char* text);
// Adds to the process-wide count of kernel launches (api.cu).
void count_launches(int n);

namespace distill {

constexpr int kMostTop = 256;  // largest k

// ---- best scores of each row (distill_top.cu) ------------------------------------------------
struct TopArgs {
  const void* scores;  // (n_rows, n_cols), row_stride elements between rows
  int64_t n_rows, n_cols, row_stride;
  int k;
  bool probabilities;    // values are the logarithms of the scores
  double inv_temperature;
  void* values;        // (n_rows, k), type of the scores
  int32_t* index;      // (n_rows, k)
  void* logsumexp;     // (n_rows) double for double scores, else float; or null
};
size_t top_workspace(int dtype, const TopArgs& a, int n_sms);
cudaError_t launch_top(int dtype, const TopArgs& a, void* workspace, int n_sms, cudaStream_t s);

// ---- what a teacher says of each row ---------------------------------------------------------
struct Teacher {
  const float* values;     // (n_rows, k), stride values_stride; null: every entry weighs the same
  const void* index;       // (n_rows, k) int32 or int64, stride index_stride
  const float* logsumexp;  // (n_rows) of all the teacher's scores / T: the rest is one more class; null: no rest
  int64_t values_stride, index_stride;
  int k;
  bool index64;
  int64_t ignore;          // an index that does not count (besides those outside the classes)
};

// In 64 bits: rounded to 32, 0.1 is off by 2^-26 of itself, and what is left of 1 by that part of a score.
struct Temperature {
  double t = 1.0, inverse = 1.0;
  float c = 0.f;  // log2(e) / T
  Temperature() = default;
  explicit Temperature(double t) : t(t), inverse(1.0 / t), c(static_cast<float>(1.4426950408889634 / t)) {}
};

// What the teacher names in each row, kept for the gradient: (n_rows, k) each.
struct Named {
  float* logit;  // of the class; not used by the loss on logits
  float* p;      // the teacher's probability
  int32_t* at;   // the class, below 0: none
};

// ---- loss on logits (distill_loss.cu) --------------------------------------------------------
struct LossArgs {
  const void* logits;
  int64_t n_rows, n_cols, row_stride;
  Teacher teacher;
  Temperature temperature;
  float* row_loss;   // (n_rows)
  // (n_rows), for the gradient.  q of a class times the sum of all of p is 2^((z - x) c) y, the gradient over T by a class
  // that is not named 2^((z - z_o) c) w (z_o: the third component); all 0 where the row does not count.
  float4* row_stats;
  Named named;
};
// reduction: 0 none, 1 sum, 2 mean over the rows that count.
struct Reduced {
  int reduction;
  float* loss;    // the reduced loss
  float* factor;  // of the rows' losses in it
};
size_t loss_workspace(const LossArgs& a, int n_sms);
cudaError_t launch_loss(int dtype, const LossArgs& a, const Reduced& out, void* workspace, int n_sms, cudaStream_t s);

struct LossGradArgs {
  LossArgs fwd;            // row_loss is not used
  const float* upstream;   // one value (reduced) or one per row
  int64_t upstream_stride;
  const float* factor;     // device scalar that multiplies upstream, or null
  void* grad;              // (n_rows, n_cols), grad_stride elements between rows
  int64_t grad_stride;
};
cudaError_t launch_loss_grad(int dtype, const LossGradArgs& a, int n_sms, cudaStream_t s);

// ---- loss on a linear layer's output (distill_linear.cu) -------------------------------------
struct LinearArgs {
  const void* hidden;  // (n_rows, width)
  const void* weight;  // (n_cols, width)
  int64_t n_rows, n_cols, width, hidden_stride, weight_stride;
  Teacher teacher;     // no logsumexp
  Temperature temperature;
  float* row_loss;
  float4* row_stats;   // (n_rows) max, 1 / sum, 1, 1: the row counts
  Named named;
};
size_t linear_workspace(const LinearArgs& a, int n_sms);
cudaError_t launch_linear(int dtype, const LinearArgs& a, const Reduced& out, void* workspace, int n_sms, cudaStream_t s);

struct LinearGradArgs {
  LinearArgs fwd;
  const float* upstream;
  int64_t upstream_stride;
  const float* factor;  // null: upstream has one value per row
  void* grad_hidden;    // (n_rows, width) contiguous, or null
  void* grad_weight;    // (n_cols, width) contiguous, or null
};
size_t linear_grad_workspace(const LinearGradArgs& g, int n_sms);
cudaError_t launch_linear_grad(int dtype, const LinearGradArgs& g, void* workspace, int n_sms, cudaStream_t s);

// Waits for the current device, reads its status word and clears it: not 0 where a bounded wait ran out.
cudaError_t linear_status(int* status);
// A kernel whose only work is such a wait, which nothing ends and which gives up after a millisecond.
cudaError_t launch_linear_timeout(cudaStream_t s);

}  // namespace distill
}  // namespace b2fil
