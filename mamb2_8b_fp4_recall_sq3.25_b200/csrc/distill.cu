// Distillation from a teacher's record of its largest logits, and its gradient.
//
// Student logits s over the whole vocabulary, teacher entries (v_k, j_k), temperature T,
// c = log2(e) / T, everything in powers of two:
//   q_k = 2^((v_k - v_max) c) / Q,  Q their sum      p_j = 2^((s_j - m) c) / S,  S the sum
//   loss = T^2 ln 2 sum_k q_k [ ((v_k - v_max) c - log2 Q) - ((s_jk - m) c - log2 S) ]
//   d loss / d s_j = T (p_j - sum over k with j_k = j of q_k)
// An entry whose index lies outside the vocabulary, or whose logit is -inf or NaN, is unused;
// a row without used entries has loss 0 and gradient 0.  Sums are fp32; p and the difference
// p - q are fp32 and rounded once to the logits' type.
//
// row_kernel: one cluster of 1..8 CTAs per row, the row in registers.  Every thread loads its
// units of 16 bytes at once, the record is read while they travel, and the CTAs exchange one
// (max, sum) pair through distributed shared memory.  With GRAD the gradient is written from
// the registers, so loss and gradient read the logits once.
// grad_kernel: the backward of a forward whose statistics were kept, one pass.
#include "logits.cuh"
#include "logits_util.cuh"

namespace sq {
namespace {

template <int NT>
struct Scratch {
  float part[2][NT / 32];
  float2 pair[8];                                // (max, sum) of each CTA of the cluster
  alignas(16) int at[kMaxRecord];
  float e[kMaxRecord];
};

template <int NT>
__device__ float block_max(float v, float* part) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  v = part[threadIdx.x & (NT / 32 - 1)];
#pragma unroll
  for (int o = NT / 64; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
template <int NT>
__device__ float block_sum(float v, float* part) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  v = part[threadIdx.x & (NT / 32 - 1)];
#pragma unroll
  for (int o = NT / 64; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Largest value of a unit; NaN is passed over (it shows up in the sum).
__device__ __forceinline__ float unit_max(const Unit<__half>& u) {
  const __half2* h = reinterpret_cast<const __half2*>(&u.q);
  const __half2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
  return fmaxf(__low2float(m), __high2float(m));
}
__device__ __forceinline__ float unit_max(const Unit<__nv_bfloat16>& u) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&u.q);
  const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
  return fmaxf(__low2float(m), __high2float(m));
}
__device__ __forceinline__ float unit_max(const Unit<float>& u) {
  return fmaxf(fmaxf(u.v[0], u.v[1]), fmaxf(u.v[2], u.v[3]));
}

__device__ __forceinline__ float record_value(const DistillParams& P, long long i) {
  switch (P.values_type) {
    case kLogitsF16: return __half2float(reinterpret_cast<const __half*>(P.values)[i]);
    case kLogitsBf16: return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(P.values)[i]);
  }
  return reinterpret_cast<const float*>(P.values)[i];
}
__device__ __forceinline__ bool used_entry(const DistillParams& P, int j, float v) {
  return j >= 0 && j < P.x.vocab && v > -INFINITY;
}
// (v - v_max) c; the largest entry is 0 even where it is infinite.
__device__ __forceinline__ float record_power(float v, float vmax, float c) { return v == vmax ? 0.0f : (v - vmax) * c; }

// Gradient at the record's tokens that lie in columns [j0, j1), over what the dense pass wrote
// there (a barrier before this call orders the two): every token by its first entry, repeated
// indices added up.  at: the row's indices (-1: unused) in shared memory, padded with -1 to a multiple of four.
template <typename T, int NT, typename Q>
__device__ void record_gradient(const T* s, T* g, const int* at, int k, int j0, int j1, float m, float c, float scale,
                                float f, Q q) {
  for (int i = threadIdx.x; i < k; i += NT) {
    const int j = at[i];
    if (j < j0 || j >= j1) continue;
    float sum = 0.f;
    bool first = true;
    for (int b = 0; b < k; b += 4) {
      const int4 a = *reinterpret_cast<const int4*>(at + b);
      const int same[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int o = 0; o < 4; ++o)
        if (same[o] == j) {
          if (b + o < i) first = false;
          sum += q(b + o);
        }
      if (!first) break;
    }
    if (first) g[j] = from_f32<T>(ex2((to_f32(s[j]) - m) * c) * scale - f * sum);
  }
}

template <typename T, int NT, int NV, bool GRAD>
__global__ void __launch_bounds__(NT) row_kernel(const DistillParams P) {
  __shared__ Scratch<NT> sh;
  const uint32_t rank = cluster_rank(), size = cluster_size();
  const int row = blockIdx.x / size, tid = threadIdx.x;
  const float c = kLog2e / P.temperature;
  const T* s = reinterpret_cast<const T*>(P.x.data) + (long long)row * P.x.stride;
  const RowSpan<T> span(s, P.x.vocab);
  const int per = (span.units + (int)size - 1) / (int)size;
  const int u0 = (int)rank * per, u1 = min(span.units, u0 + per);
  cluster_arrive();                              // waited for before the first remote store

  Unit<T> x[NV];
  const uint4* body = reinterpret_cast<const uint4*>(s + span.head);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int u = u0 + i * NT + tid;
    if (u < u1) x[i].q = load_unit(body + u);
  }
  const bool has_edge = rank == 0 && tid < span.edges();
  const int edge = has_edge ? span.edge(tid) : 0;
  const float xe = has_edge ? to_f32(s[edge]) : -INFINITY;

  // the record, while the units travel: Q everywhere, the student's logits at its tokens on rank 0
  const long long base = (long long)row * P.k;
  float vmax = -INFINITY, taken[kMaxRecord / NT];
#pragma unroll
  for (int i = 0; i < kMaxRecord / NT; ++i) {
    const int k = tid + i * NT;
    taken[i] = 0.f;
    if (k < P.k) {
      const int j = P.indices[base + k];
      const float v = record_value(P, base + k);
      const bool used = used_entry(P, j, v);
      sh.at[k] = used ? j : -1;
      sh.e[k] = v;
      if (used) {
        vmax = fmaxf(vmax, v);
        if (rank == 0) taken[i] = to_f32(s[j]);
      }
    } else {
      sh.at[k] = -1;
    }
  }
  vmax = block_max<NT>(vmax, sh.part[0]);
  float q = 0.f;
#pragma unroll
  for (int i = 0; i < kMaxRecord / NT; ++i) {
    const int k = tid + i * NT;
    if (k < P.k) {
      const float e = sh.at[k] < 0 ? -INFINITY : record_power(sh.e[k], vmax, c);
      sh.e[k] = e;
      q += ex2(e);
    }
  }
  const float Q = block_sum<NT>(q, sh.part[1]);

  // this CTA's max and sum
  float m = xe;
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (u0 + i * NT + tid < u1) m = fmaxf(m, unit_max(x[i]));
  m = block_max<NT>(m, sh.part[0]);
  const float ref = m == -INFINITY ? 0.f : m;    // nothing above -inf: powers of -inf are 0, NaN stays
  float sum = has_edge ? ex2((xe - ref) * c) : 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (u0 + i * NT + tid < u1) {
#pragma unroll
      for (int v = 0; v < kUnit<T>; ++v) sum += ex2((to_f32(x[i].v[v]) - ref) * c);
    }
  sum = block_sum<NT>(sum, sh.part[1]);
  cluster_wait();
  if (tid < (int)size) remote_store(remote_smem(&sh.pair[rank], tid), m, sum);
  cluster_arrive();
  cluster_wait();
  m = -INFINITY;
  for (int i = 0; i < (int)size; ++i) m = fmaxf(m, sh.pair[i].x);
  sum = 0.f;
  for (int i = 0; i < (int)size; ++i)
    sum += sh.pair[i].x == m ? sh.pair[i].y : sh.pair[i].y * ex2((sh.pair[i].x - m) * c);
  const float inv = 1.0f / sum;

  if (rank == 0) {
    float l = 0.f;
    if (Q > 0.f) {
      const float rest = log2f(sum) - log2f(Q);
#pragma unroll
      for (int i = 0; i < kMaxRecord / NT; ++i) {
        const int k = tid + i * NT;
        if (k < P.k && sh.at[k] >= 0) {
          const float w = ex2(sh.e[k]);
          if (w > 0.f) l += w * (sh.e[k] - (taken[i] - m) * c + rest);
        }
      }
    }
    l = block_sum<NT>(l, sh.part[0]);
    if (tid == 0) {
      P.loss[row] = Q > 0.f ? P.temperature * P.temperature * kLn2 * (l / Q) : 0.f;
      if (P.stats) P.stats[row] = make_float4(m, inv, vmax, Q > 0.f ? 1.0f / Q : 0.f);
    }
  }
  if (GRAD) {
    T* g = reinterpret_cast<T*>(P.grad) + (long long)row * P.grad_stride;
    const bool any = Q > 0.f;
    const float f = P.temperature * (P.weight ? P.weight[row * P.weight_stride] : 1.0f), scale = f * inv;
    if (has_edge) g[edge] = from_f32<T>(any ? ex2((xe - m) * c) * scale : 0.f);
    T* gb = g + span.head;
    const bool vec = ((uintptr_t)gb & 15) == 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int u = u0 + i * NT + tid;
      if (u < u1) {
        Unit<T> o;
#pragma unroll
        for (int v = 0; v < kUnit<T>; ++v) o.v[v] = from_f32<T>(any ? ex2((to_f32(x[i].v[v]) - m) * c) * scale : 0.f);
        if (vec) {
          reinterpret_cast<uint4*>(gb)[u] = o.q;
        } else {
#pragma unroll
          for (int v = 0; v < kUnit<T>; ++v) gb[u * kUnit<T> + v] = o.v[v];
        }
      }
    }
    if (any) {
      __syncthreads();
      // the edges belong to rank 0, at both ends of the row
      const float iq = 1.0f / Q;
      const auto qk = [&](int k) { return ex2(sh.e[k]) * iq; };
      const int b = span.head;
      record_gradient<T, NT>(s, g, sh.at, P.k, b + u0 * kUnit<T>, b + u1 * kUnit<T>, m, c, scale, f, qk);
      if (rank == 0) {
        record_gradient<T, NT>(s, g, sh.at, P.k, 0, b, m, c, scale, f, qk);
        record_gradient<T, NT>(s, g, sh.at, P.k, b + span.units * kUnit<T>, P.x.vocab, m, c, scale, f, qk);
      }
    }
  }
}

constexpr int kGradThreads = 256, kGradUnits = 4;    // a CTA of the backward writes 16 KB of a row

template <typename T>
__global__ void __launch_bounds__(kGradThreads) grad_kernel(const DistillParams P, int parts) {
  constexpr int NT = kGradThreads, NV = kGradUnits;
  __shared__ __align__(16) int at[kMaxRecord];
  const int row = blockIdx.x / parts, part = blockIdx.x - row * parts, tid = threadIdx.x;
  const float c = kLog2e / P.temperature;
  const T* s = reinterpret_cast<const T*>(P.x.data) + (long long)row * P.x.stride;
  T* g = reinterpret_cast<T*>(P.grad) + (long long)row * P.grad_stride;
  const RowSpan<T> span(s, P.x.vocab);
  const int u0 = part * NT * NV, u1 = min(span.units, u0 + NT * NV);
  const uint4* body = reinterpret_cast<const uint4*>(s + span.head);
  Unit<T> x[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (u0 + i * NT + tid < u1) x[i].q = load_unit(body + u0 + i * NT + tid);
  const float4 st = P.stats[row];
  const float m = st.x, f = P.temperature * (P.weight ? P.weight[row * P.weight_stride] : 1.0f), scale = f * st.y;
  const bool any = st.w > 0.f;
  const long long base = (long long)row * P.k;
  for (int k = tid; k < ((P.k + 3) & ~3); k += NT) {
    const int j = k < P.k ? P.indices[base + k] : -1;
    at[k] = k < P.k && used_entry(P, j, record_value(P, base + k)) ? j : -1;
  }
  if (part == 0 && tid < span.edges()) {
    const int e = span.edge(tid);
    g[e] = from_f32<T>(any ? ex2((to_f32(s[e]) - m) * c) * scale : 0.f);
  }
  T* gb = g + span.head;
  const bool vec = ((uintptr_t)gb & 15) == 0;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int u = u0 + i * NT + tid;
    if (u < u1) {
      Unit<T> o;
#pragma unroll
      for (int v = 0; v < kUnit<T>; ++v) o.v[v] = from_f32<T>(any ? ex2((to_f32(x[i].v[v]) - m) * c) * scale : 0.f);
      if (vec) {
        reinterpret_cast<uint4*>(gb)[u] = o.q;
      } else {
#pragma unroll
        for (int v = 0; v < kUnit<T>; ++v) gb[u * kUnit<T> + v] = o.v[v];
      }
    }
  }
  __syncthreads();
  if (!any) return;
  const auto qk = [&](int k) { return ex2(record_power(record_value(P, base + k), st.z, c)) * st.w; };
  const int b = span.head;
  record_gradient<T, NT>(s, g, at, P.k, b + u0 * kUnit<T>, b + u1 * kUnit<T>, m, c, scale, f, qk);
  if (part == 0) {
    record_gradient<T, NT>(s, g, at, P.k, 0, b, m, c, scale, f, qk);
    record_gradient<T, NT>(s, g, at, P.k, b + span.units * kUnit<T>, P.x.vocab, m, c, scale, f, qk);
  }
}

template <typename T, int NT, int NV, bool GRAD>
int launch_rows(const DistillParams& P, int size, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = size; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3(P.x.rows * size);
  cfg.blockDim = dim3(NT);
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, row_kernel<T, NT, NV, GRAD>, P) != cudaSuccess) return launch_status();
  return launch_status();
}

template <typename T, bool GRAD>
int launch_by_size(const DistillParams& P, cudaStream_t st) {
  const int units = (P.x.vocab + kUnit<T> - 1) / kUnit<T>;
  // CTAs of 512 threads hold 8 units a thread (64 KB of the row), as many as the row needs; few
  // rows take more CTAs each until the GPU is full.  Rows over 512 KB need 1024 threads.
  int size = 1;
  while (size < 8 && size * 512 * 8 < units) size *= 2;
  while (size < 8 && P.x.rows * size < 2 * 148 && size * 512 < units) size *= 2;
  const int per = (units + size * 512 - 1) / (size * 512);
  if (per <= 1) return launch_rows<T, 512, 1, GRAD>(P, size, st);
  if (per <= 2) return launch_rows<T, 512, 2, GRAD>(P, size, st);
  if (per <= 4) return launch_rows<T, 512, 4, GRAD>(P, size, st);
  if (per <= 8) return launch_rows<T, 512, 8, GRAD>(P, size, st);
  return launch_rows<T, 1024, 8, GRAD>(P, size, st);
}

template <typename F>
int by_type(int type, F f) {
  switch (type) {
    case kLogitsF16: return f(__half());
    case kLogitsBf16: return f(__nv_bfloat16());
    case kLogitsF32: return f(float());
  }
  return kEInval;
}

}  // namespace

int launch_distill_forward(const DistillParams& P, cudaStream_t st) {
  return by_type(P.x.type, [&](auto t) { return launch_by_size<decltype(t), false>(P, st); });
}
int launch_distill_loss_grad(const DistillParams& P, cudaStream_t st) {
  return by_type(P.x.type, [&](auto t) { return launch_by_size<decltype(t), true>(P, st); });
}
int launch_distill_backward(const DistillParams& P, cudaStream_t st) {
  return by_type(P.x.type, [&](auto t) {
    using T = decltype(t);
    const int units = P.x.vocab / kUnit<T>, per = kGradThreads * kGradUnits;
    const int parts = units > per ? (units + per - 1) / per : 1;
    grad_kernel<T><<<(unsigned)P.x.rows * parts, kGradThreads, 0, st>>>(P, parts);
    return launch_status();
  });
}

}  // namespace sq
