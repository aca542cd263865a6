// Distillation from a teacher's record of its largest logits, and its gradient.
//
// Student logits s over the whole vocabulary, teacher entries (v_k, j_k), temperature T,
// c = log2(e) / T, everything in powers of two:
//   q_k = 2^((v_k - v_max) c) / Q,  Q their sum      p_j = 2^((s_j - m) c) / S,  S the sum
//   loss = T^2 ln 2 sum_k q_k [ ((v_k - v_max) c - log2 Q) - ((s_jk - m) c - log2 S) ]
//   d loss / d s_j = T (p_j - sum over k with j_k = j of q_k)
// An entry whose index lies outside the vocabulary, or whose logit is -inf or NaN, is unused;
// a row without used entries has loss 0 and gradient 0.  Sums are fp32.
//
// One CTA per row.
#include "logits.cuh"
#include "logits_util.cuh"

namespace sq {
namespace {

constexpr int NT = 512, NW = NT / 32;

struct MaxSum { float m, s; };                   // largest value and sum of 2^((x - m) c)

__device__ __forceinline__ MaxSum merge(MaxSum a, MaxSum b, float c) {
  const float m = fmaxf(a.m, b.m);
  if (m == -INFINITY) return MaxSum{m, a.s + b.s};
  const float sa = a.m == m ? a.s : (a.m == -INFINITY ? a.s : a.s * ex2((a.m - m) * c));
  const float sb = b.m == m ? b.s : (b.m == -INFINITY ? b.s : b.s * ex2((b.m - m) * c));
  return MaxSum{m, sa + sb};
}
__device__ __forceinline__ MaxSum warp_merge(MaxSum v, float c) {
#pragma unroll
  for (int o = 16; o; o >>= 1)
    v = merge(v, MaxSum{__shfl_xor_sync(0xffffffffu, v.m, o), __shfl_xor_sync(0xffffffffu, v.s, o)}, c);
  return v;
}
__device__ MaxSum block_merge(MaxSum v, float c, MaxSum* part) {
  v = warp_merge(v, c);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  MaxSum t = part[0];
  for (int i = 1; i < NW; ++i) t = merge(t, part[i], c);
  return t;
}

__device__ __forceinline__ float record_value(const DistillParams& P, long long i) {
  switch (P.values_type) {
    case kLogitsF16: return __half2float(reinterpret_cast<const __half*>(P.values)[i]);
    case kLogitsBf16: return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(P.values)[i]);
  }
  return reinterpret_cast<const float*>(P.values)[i];
}

// The row's record in shared memory: index (-1: unused) and (v - v_max) c; returns Q (0: none).
__device__ float load_record(const DistillParams& P, int row, float c, int* at, float* e, MaxSum* part) {
  const long long base = (long long)row * P.k;
  float m = -INFINITY;
  for (int k = threadIdx.x; k < P.k; k += NT) {
    const int j = P.indices[base + k];
    const float v = record_value(P, base + k);
    const bool used = j >= 0 && j < P.x.vocab && v > -INFINITY;
    at[k] = used ? j : -1;
    e[k] = v;
    if (used) m = fmaxf(m, v);
  }
  m = block_merge(MaxSum{m, 0.f}, c, part).m;
  float sum = 0.f;
  for (int k = threadIdx.x; k < P.k; k += NT) {
    e[k] = at[k] < 0 ? -INFINITY : e[k] == m ? 0.f : (e[k] - m) * c;
    sum += ex2(e[k]);
  }
  return block_merge(MaxSum{0.f, sum}, c, part).s;
}

template <typename T, bool LOSS, bool GRAD>
__global__ void __launch_bounds__(NT) distill_kernel(const DistillParams P) {
  __shared__ MaxSum part[NW];
  __shared__ int at[kMaxRecord];
  __shared__ float e[kMaxRecord];
  const int row = blockIdx.x, tid = threadIdx.x;
  const float c = kLog2e / P.temperature;
  const T* s = reinterpret_cast<const T*>(P.x.data) + (long long)row * P.x.stride;
  const float Q = load_record(P, row, c, at, e, part);
  float m, inv;
  if (LOSS) {
    MaxSum v{-INFINITY, 0.f};
    for (int j = tid; j < P.x.vocab; j += NT) {
      const float x = to_f32(s[j]);
      const float nm = fmaxf(v.m, x);
      if (!(x == -INFINITY && v.m == -INFINITY)) {          // a NaN goes into the sum and stays there
        v.s = (v.m == -INFINITY ? v.s : v.s * ex2((v.m - nm) * c)) + ex2((x - nm) * c);
        v.m = nm;
      }
    }
    v = block_merge(v, c, part);
    m = v.m;
    inv = 1.0f / v.s;
    float l = 0.f;
    if (Q > 0.f)
      for (int k = tid; k < P.k; k += NT) {
        const float q = ex2(e[k]);
        if (at[k] >= 0 && q > 0.f)
          l += q * ((e[k] - log2f(Q)) - ((to_f32(s[at[k]]) - m) * c - log2f(v.s)));
      }
    l = block_merge(MaxSum{0.f, l}, c, part).s;
    if (tid == 0) {
      P.loss[row] = Q > 0.f ? P.temperature * P.temperature * kLn2 * (l / Q) : 0.f;
      if (P.stats) P.stats[row] = make_float2(m, inv);
    }
  } else {
    const float2 st = P.stats[row];
    m = st.x;
    inv = st.y;
  }
  if (GRAD) {
    T* g = reinterpret_cast<T*>(P.grad) + (long long)row * P.grad_stride;
    if (!(Q > 0.f)) {
      for (int j = tid; j < P.x.vocab; j += NT) g[j] = from_f32<T>(0.f);
      return;
    }
    const float f = P.temperature * (P.weight ? P.weight[row * P.weight_stride] : 1.0f);
    for (int j = tid; j < P.x.vocab; j += NT) g[j] = from_f32<T>(f * (ex2((to_f32(s[j]) - m) * c) * inv));
    __syncthreads();
    // the record's tokens once more, each by its first entry: repeated indices add up
    for (int k = tid; k < P.k; k += NT) {
      const int j = at[k];
      if (j < 0) continue;
      float q = 0.f;
      bool first = true;
      for (int i = 0; i < P.k; ++i)
        if (at[i] == j) {
          if (i < k) { first = false; break; }
          q += ex2(e[i]);
        }
      if (first) g[j] = from_f32<T>(f * (ex2((to_f32(s[j]) - m) * c) * inv - q / Q));
    }
  }
}

template <bool LOSS, bool GRAD>
int launch(const DistillParams& P, cudaStream_t st) {
  switch (P.x.type) {
    case kLogitsF16: distill_kernel<__half, LOSS, GRAD><<<P.x.rows, NT, 0, st>>>(P); return launch_status();
    case kLogitsBf16: distill_kernel<__nv_bfloat16, LOSS, GRAD><<<P.x.rows, NT, 0, st>>>(P); return launch_status();
    case kLogitsF32: distill_kernel<float, LOSS, GRAD><<<P.x.rows, NT, 0, st>>>(P); return launch_status();
  }
  return kEInval;
}

}  // namespace

int launch_distill_forward(const DistillParams& P, cudaStream_t st) { return launch<true, false>(P, st); }
int launch_distill_backward(const DistillParams& P, cudaStream_t st) { return launch<false, true>(P, st); }
int launch_distill_loss_grad(const DistillParams& P, cudaStream_t st) { return launch<true, true>(P, st); }

}  // namespace sq
