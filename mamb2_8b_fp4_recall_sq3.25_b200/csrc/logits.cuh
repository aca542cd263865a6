// Operators on rows of logits: launch interfaces (logits.cu: drawing a token, the largest
// logits; distill.cu: the distillation loss and its gradient).
#pragma once
#include <atomic>
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

// Allows `kernel` up to `bytes` of dynamic shared memory, once per device (`done`: one flag a device).
template <typename K>
cudaError_t allow_shared(K kernel, int bytes, std::atomic<uint64_t>& done) {
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  const uint64_t flag = 1ull << (device & 63);
  if (device < 64 && (done.load(std::memory_order_acquire) & flag)) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && device < 64) done.fetch_or(flag, std::memory_order_release);
  return e;
}

// Launches `kernel(params)` with a cluster of `size` CTAs a row, or, if the kernel steps through the rows, with no
// more clusters than run at once (fewer than SMs allow: a cluster lies within a GPC).  Up to `room` CTAs
// this is not asked for.
template <typename K, typename P>
int launch_clusters(K kernel, const P& params, int size, int threads, size_t smem, cudaStream_t st, bool steps = false,
                    int room = 0) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = size; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  unsigned clusters = (unsigned)params.x.rows;
  cfg.gridDim = dim3(clusters * size);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (steps && params.x.rows * size > room) {
    int fit = 0;
    if (cudaOccupancyMaxActiveClusters(&fit, kernel, &cfg) != cudaSuccess) return launch_status();
    if (fit > 0 && (unsigned)fit < clusters) cfg.gridDim = dim3((unsigned)fit * size);
  }
  cudaLaunchKernelEx(&cfg, kernel, params);
  return launch_status();
}

constexpr int kSms = 148;                 // of a B200

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
