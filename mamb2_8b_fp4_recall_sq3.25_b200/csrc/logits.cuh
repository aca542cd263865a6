// Operators on rows of logits: launch interfaces (logits.cu: drawing a token, the largest
// logits; distill.cu: the distillation loss and its gradient).
#pragma once
#include "common.cuh"

namespace sq {

enum LogitsType : int { kLogitsF16 = 0, kLogitsBf16 = 1, kLogitsF32 = 2 };

constexpr int kMaxRows = 1 << 24;         // rows times CTAs of a row stay within a grid
constexpr int kMaxVocab = 1 << 18;        // columns of a row
constexpr int kMaxRecord = 1024;          // entries of one row's record of largest logits

struct LogitsRows {
  const void* data;
  long long stride;                       // elements between rows
  int rows, vocab, type;
};

// 16-byte units of a row, one more where it may start inside a unit.
inline int row_units(const LogitsRows& x) { return (x.vocab * (x.type == kLogitsF32 ? 4 : 2) + 15) / 16 + 1; }

// Per-row settings of a draw; a null pointer means the one value for every row.
struct SampleParams {
  LogitsRows x;
  const float* uniform;
  const float *temperature, *top_p, *min_p;
  const int* top_k;
  float temperature_all, top_p_all, min_p_all;
  int top_k_all;
  long long* tokens;
};
int launch_sample(const SampleParams& P, cudaStream_t st);

struct TopParams {
  LogitsRows x;
  int k;
  void* values;                           // [rows][k], the logits' type
  int* indices;                           // [rows][k]
};
int launch_top_logits(const TopParams& P, cudaStream_t st);

struct DistillParams {
  LogitsRows x;                           // student
  const void* values;                     // teacher's record [rows][k]
  const int* indices;
  int k, values_type;
  float temperature;
  const float* weight;                    // factor of each row's gradient; null: 1
  long long weight_stride;                // 0: one factor for every row
  float* loss;                            // [rows]
  float4* stats;                          // [rows] {largest logit, 1 / S, v_max, 1 / Q (0: no record)}
  void* grad; long long grad_stride;      // the logits' type
};
int launch_distill_forward(const DistillParams& P, cudaStream_t st);   // loss, stats (optional)
int launch_distill_backward(const DistillParams& P, cudaStream_t st);  // grad from stats
int launch_distill_loss_grad(const DistillParams& P, cudaStream_t st); // loss, grad

}  // namespace sq
