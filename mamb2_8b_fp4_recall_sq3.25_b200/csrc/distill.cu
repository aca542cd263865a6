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
// loss_kernel: the forward.  The CTAs of a cluster stream their parts of the row with a running
// maximum and sum per thread.
// row_kernel: loss and gradient in one pass.  The CTAs of a cluster hold the row in registers:
// every thread loads its units of 16 bytes at once, the record is worked through while they
// travel, and the gradient is written from the registers.
// In both each warp sends its (max, sum) to every CTA of the cluster through distributed shared
// memory, so a row costs one cluster barrier.
// grad_kernel: the backward of a forward whose statistics were kept, streaming.
#include "logits.cuh"
#include "logits_util.cuh"
#include <type_traits>

namespace sq {
namespace {

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


// Sum of 2^((x - ref) c) over a unit.
template <typename T>
__device__ __forceinline__ float unit_power_sum(const Unit<T>& u, float ref, float c) {
  float s = 0.f;
#pragma unroll
  for (int v = 0; v < kUnit<T>; ++v) s += ex2((to_f32(u.v[v]) - ref) * c);
  return s;
}
// scale 2^((x - m) c) for a unit, written at column-unit u of `g`.
template <typename T>
__device__ __forceinline__ void store_gradient(T* g, int u, bool vec, const Unit<T>& x, float m, float c, float scale) {
  Unit<T> o;
#pragma unroll
  for (int v = 0; v < kUnit<T>; ++v) o.v[v] = from_f32<T>(ex2((to_f32(x.v[v]) - m) * c) * scale);
  if (vec) {
    reinterpret_cast<uint4*>(g)[u] = o.q;
  } else {
#pragma unroll
    for (int v = 0; v < kUnit<T>; ++v) g[u * kUnit<T> + v] = o.v[v];
  }
}
template <typename T>
__device__ __forceinline__ void zero_gradient(T* g, int u, bool vec) {
  if (vec) {
    reinterpret_cast<uint4*>(g)[u] = make_uint4(0, 0, 0, 0);
  } else {
#pragma unroll
    for (int v = 0; v < kUnit<T>; ++v) g[u * kUnit<T> + v] = from_f32<T>(0.f);
  }
}

// (max, sum) of every warp of the cluster.
template <int NW> struct Pairs { float2 p[8 * NW]; };

// Each warp hands its pair to all CTAs; afterwards every thread has the row's.  `m` is the warp's
// maximum and `sum` this thread's share relative to it (to 0 where m is -inf: powers of -inf
// are 0 and a NaN stays one).  The caller has arrived at the cluster barrier once before.
template <int NW>
__device__ void cluster_merge(float& m, float& sum, float c, Pairs<NW>& pairs, uint32_t rank, uint32_t size) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  cluster_wait();                                // every CTA of the cluster runs
  if (lane < (int)size) remote_store(remote_smem(&pairs.p[rank * NW + warp], lane), m, sum);
  cluster_arrive();
  cluster_wait();
  const int n = (int)size * NW;
  m = -INFINITY;
  for (int i = lane; i < n; i += 32) m = fmaxf(m, pairs.p[i].x);
#pragma unroll
  for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  sum = 0.f;
  for (int i = lane; i < n; i += 32) {
    const float2 p = pairs.p[i];
    sum += p.x == m ? p.y : p.y * ex2((p.x - m) * c);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// One row's record: each thread holds entries tid, tid + NT, ...
template <typename T, int NT>
struct Record {
  static constexpr int N = kMaxRecord / NT;
  int at[N];                                     // -1: unused
  float e[N];                                    // (v - v_max) c
  float taken[N];                                // student's logit there
  float vmax, Q;
  // Reads it all and, for entries with `wants(index)`, the student's logit.
  template <typename W>
  __device__ void load(const DistillParams& P, const T* s, long long base, float c, float (*part)[NT / 32], W wants) {
    vmax = -INFINITY;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int k = threadIdx.x + i * NT;
      at[i] = -1;
      if (k < P.k) {
        const int j = P.indices[base + k];
        e[i] = record_value(P, base + k);
        if (used_entry(P, j, e[i])) {
          at[i] = j;
          vmax = fmaxf(vmax, e[i]);
          if (wants(j)) taken[i] = to_f32(s[j]);
        }
      }
    }
    vmax = block_max<NT>(vmax, part[0]);
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      e[i] = at[i] < 0 ? -INFINITY : record_power(e[i], vmax, c);
      q += ex2(e[i]);
    }
    Q = block_sum<NT>(q, part[1]);
  }
  // Loss of the row, known to thread 0 (every thread of the CTA calls, `taken` was wanted everywhere).
  __device__ float loss(float m, float sum, float c, float temperature, float (*part)[NT / 32]) const {
    float l = 0.f;
    const float rest = Q > 0.f ? log2f(sum) - log2f(Q) : 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float w = ex2(e[i]);
      if (at[i] >= 0 && w > 0.f) l += w * (e[i] - (taken[i] - m) * c + rest);
    }
    l = block_sum<NT>(l, part[0]);
    return Q > 0.f ? temperature * temperature * kLn2 * (l / Q) : 0.f;
  }
};

constexpr int kLossThreads = 256, kLossUnits = 4;

template <typename T>
__global__ void __launch_bounds__(kLossThreads, 4) loss_kernel(const DistillParams P) {
  constexpr int NT = kLossThreads, NV = kLossUnits, NW = NT / 32;
  __shared__ Pairs<NW> pairs;
  __shared__ float part[2][NW];
  const uint32_t rank = cluster_rank(), size = cluster_size();
  const int row = blockIdx.x / size, tid = threadIdx.x;
  const float c = kLog2e / P.temperature;
  const T* s = reinterpret_cast<const T*>(P.x.data) + (long long)row * P.x.stride;
  const RowSpan<T> span(s, P.x.vocab);
  const int per = (span.units + (int)size - 1) / (int)size;
  const int u0 = (int)rank * per, u1 = min(span.units, u0 + per);
  cluster_arrive();
  const uint4* body = reinterpret_cast<const uint4*>(s + span.head);
  const auto load = [&](Unit<T> (&x)[NV], int at) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int u = at + i * NT + tid;
      x[i].q = u < u1 ? load_unit(body + u) : neg_inf_unit<T>();
    }
  };
  Unit<T> x[NV];
  load(x, u0);
  float m = rank == 0 && tid < span.edges() ? to_f32(s[span.edge(tid)]) : -INFINITY;
  float sum = m == -INFINITY ? 0.f : 1.f;
  if (m != m) { sum = m; m = -INFINITY; }
  Record<T, NT> rec;
  if (rank == 0) rec.load(P, s, (long long)row * P.k, c, part, [](int) { return true; });
  for (int at = u0; at < u1; at += NT * NV) {
    Unit<T> next[NV];
    load(next, at + NT * NV);
    float top = unit_max(x[0]);
#pragma unroll
    for (int i = 1; i < NV; ++i) top = fmaxf(top, unit_max(x[i]));
    if (top > m) {
      sum *= ex2((m - top) * c);
      m = top;
    }
    const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int i = 0; i < NV; ++i) sum += unit_power_sum(x[i], ref, c);
#pragma unroll
    for (int i = 0; i < NV; ++i) x[i] = next[i];
  }
  const float wm = warp_max(m);
  if (m != wm) sum *= ex2((m - wm) * c);
  m = wm;
  cluster_merge<NW>(m, sum, c, pairs, rank, size);
  if (rank != 0) return;
  const float l = rec.loss(m, sum, c, P.temperature, part);
  if (tid == 0) {
    P.loss[row] = l;
    if (P.stats) P.stats[row] = make_float4(m, 1.0f / sum, rec.vmax, rec.Q > 0.f ? 1.0f / rec.Q : 0.f);
  }
}

// The record's tokens in the gradient: each by its first entry, repeated indices added up.
// at, w: the row's indices (-1: unused, and up to a multiple of four) and 2^e in shared memory.
// Returns the sum of 2^e over the entries of index j if entry k is the first of them, else -1.
__device__ __forceinline__ float sum_of_index(const int* at, const float* w, int n, int k, int j) {
  float sum = 0.f;
  for (int b = 0; b < n; b += 4) {
    const int4 a = *reinterpret_cast<const int4*>(at + b);
    const int same[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int o = 0; o < 4; ++o)
      if (same[o] == j) {
        if (b + o < k) return -1.f;
        sum += w[b + o];
      }
  }
  return sum;
}

template <typename T, int NT, int NV>
__global__ void __launch_bounds__(NT, 1024 / NT) row_kernel(const DistillParams P) {
  constexpr int NW = NT / 32;
  __shared__ Pairs<NW> pairs;
  __shared__ float part[2][NW];
  __shared__ __align__(16) int at[kMaxRecord];
  __shared__ float w[kMaxRecord];
  const uint32_t rank = cluster_rank(), size = cluster_size();
  const int row = blockIdx.x / size, tid = threadIdx.x;
  const float c = kLog2e / P.temperature;
  const T* s = reinterpret_cast<const T*>(P.x.data) + (long long)row * P.x.stride;
  const RowSpan<T> span(s, P.x.vocab);
  const int per = (span.units + (int)size - 1) / (int)size;
  const int u0 = (int)rank * per, u1 = min(span.units, u0 + per);
  cluster_arrive();

  Unit<T> x[NV];
  const uint4* body = reinterpret_cast<const uint4*>(s + span.head);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int u = u0 + i * NT + tid;
    x[i].q = u < u1 ? load_unit(body + u) : neg_inf_unit<T>();
  }
  const bool has_edge = rank == 0 && tid < span.edges();
  const int edge = has_edge ? span.edge(tid) : 0;
  const float xe = has_edge ? to_f32(s[edge]) : -INFINITY;

  // the record: this CTA corrects the tokens in its own columns, rank 0 those of the edges too
  const auto mine = [&](int j) {
    const int u = (j - span.head) / kUnit<T>;
    return j < span.head || u >= span.units ? rank == 0 : u >= u0 && u < u1;
  };
  Record<T, NT> rec;
  rec.load(P, s, (long long)row * P.k, c, part, [&](int j) { return rank == 0 || mine(j); });
#pragma unroll
  for (int i = 0; i < rec.N; ++i) {
    at[tid + i * NT] = rec.at[i];
    w[tid + i * NT] = ex2(rec.e[i]);
  }
  __syncthreads();
  float token[rec.N];                            // sum of the token's q, or < 0: not for this thread
#pragma unroll
  for (int i = 0; i < rec.N; ++i)
    token[i] = rec.at[i] >= 0 && mine(rec.at[i]) ? sum_of_index(at, w, P.k, tid + i * NT, rec.at[i]) : -1.f;

  float m = xe;
#pragma unroll
  for (int i = 0; i < NV; ++i) m = fmaxf(m, unit_max(x[i]));
  m = warp_max(m);
  const float ref = m == -INFINITY ? 0.f : m;
  float sum = has_edge ? ex2((xe - ref) * c) : 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) sum += unit_power_sum(x[i], ref, c);
  cluster_merge<NW>(m, sum, c, pairs, rank, size);

  T* g = reinterpret_cast<T*>(P.grad) + (long long)row * P.grad_stride;
  T* gb = g + span.head;
  const bool vec = ((uintptr_t)gb & 15) == 0;
  const bool any = rec.Q > 0.f;
  const float f = P.temperature * (P.weight ? P.weight[row * P.weight_stride] : 1.0f), scale = f / sum;
  if (has_edge) g[edge] = from_f32<T>(any ? ex2((xe - m) * c) * scale : 0.f);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int u = u0 + i * NT + tid;
    if (u < u1) {
      if (any) store_gradient(gb, u, vec, x[i], m, c, scale);
      else zero_gradient(gb, u, vec);
    }
  }
  if (rank == 0) {
    const float l = rec.loss(m, sum, c, P.temperature, part);
    if (tid == 0) P.loss[row] = l;
  }
  if (!any) return;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < rec.N; ++i)
    if (token[i] >= 0.f) g[rec.at[i]] = from_f32<T>(ex2((rec.taken[i] - m) * c) * scale - f * (token[i] / rec.Q));
}

constexpr int kGradThreads = 256, kGradUnits = 4, kGradRounds = 4;   // a CTA of the backward writes 64 KB of a row

template <typename T>
__global__ void __launch_bounds__(kGradThreads) grad_kernel(const DistillParams P, int parts) {
  constexpr int NT = kGradThreads, NV = kGradUnits;
  __shared__ __align__(16) int at[kMaxRecord];
  __shared__ float w[kMaxRecord];
  const int row = blockIdx.x / parts, part = blockIdx.x - row * parts, tid = threadIdx.x;
  const float c = kLog2e / P.temperature;
  const T* s = reinterpret_cast<const T*>(P.x.data) + (long long)row * P.x.stride;
  T* g = reinterpret_cast<T*>(P.grad) + (long long)row * P.grad_stride;
  const RowSpan<T> span(s, P.x.vocab);
  const int u0 = part * NT * NV * kGradRounds, u1 = min(span.units, u0 + NT * NV * kGradRounds);
  const uint4* body = reinterpret_cast<const uint4*>(s + span.head);
  const auto load = [&](Unit<T> (&x)[NV], int from) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int u = from + i * NT + tid;
      if (u < u1) x[i].q = load_unit(body + u);
    }
  };
  Unit<T> x[NV];
  load(x, u0);
  const float4 st = P.stats[row];
  const float m = st.x, f = P.temperature * (P.weight ? P.weight[row * P.weight_stride] : 1.0f), scale = f * st.y;
  const bool any = st.w > 0.f;
  const long long base = (long long)row * P.k;
  for (int k = tid; k < ((P.k + 3) & ~3); k += NT) {
    const int j = k < P.k ? P.indices[base + k] : -1;
    const float v = k < P.k ? record_value(P, base + k) : 0.f;
    const bool used = used_entry(P, j, v);
    at[k] = used ? j : -1;
    w[k] = used ? ex2(record_power(v, st.z, c)) : 0.f;
  }
  if (part == 0 && tid < span.edges()) {
    const int e = span.edge(tid);
    g[e] = from_f32<T>(any ? ex2((to_f32(s[e]) - m) * c) * scale : 0.f);
  }
  T* gb = g + span.head;
  const bool vec = ((uintptr_t)gb & 15) == 0;
  for (int from = u0; from < u1; from += NT * NV) {
    Unit<T> next[NV];
    load(next, from + NT * NV);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int u = from + i * NT + tid;
      if (u < u1) {
        if (any) store_gradient(gb, u, vec, x[i], m, c, scale);
        else zero_gradient(gb, u, vec);
      }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) x[i] = next[i];
  }
  __syncthreads();
  if (!any) return;
  for (int k = tid; k < P.k; k += NT) {
    const int j = at[k];
    if (j < 0) continue;
    const int u = (j - span.head) / kUnit<T>;
    if (j < span.head || u >= span.units ? part != 0 : u < u0 || u >= u1) continue;
    const float q = sum_of_index(at, w, P.k, k, j);
    if (q >= 0.f) g[j] = from_f32<T>(ex2((to_f32(s[j]) - m) * c) * scale - f * (q * st.w));
  }
}

template <typename K>
int launch_clusters(K kernel, const DistillParams& P, int size, int threads, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = size; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3((unsigned)P.x.rows * size);
  cfg.blockDim = dim3(threads);
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, kernel, P);
  return launch_status();
}

template <typename T>
int launch_loss(const DistillParams& P, cudaStream_t st) {
  const int units = (P.x.vocab + kUnit<T> - 1) / kUnit<T>;
  // more CTAs a row while the GPU is not many times full and each keeps some rounds of loads
  int size = 1;
  while (size < 8 && P.x.rows * size < 16 * 148 && units > size * 2 * kLossThreads * kLossUnits) size *= 2;
  return launch_clusters(loss_kernel<T>, P, size, kLossThreads, st);
}

template <typename T>
int launch_rows(const DistillParams& P, cudaStream_t st) {
  const int units = (P.x.vocab + kUnit<T> - 1) / kUnit<T>;
  // CTAs of 512 threads hold 8 units a thread (64 KB of the row), as many as the row needs; few
  // rows take more CTAs each until the GPU is full.  Rows over 512 KB
  // (fp32 only) need 1024 threads.
  int size = 1;
  while (size < 8 && size * 512 * 8 < units) size *= 2;
  while (size < 8 && P.x.rows * size < 2 * 148 && size * 512 < units) size *= 2;
  const int per = (units + size * 512 - 1) / (size * 512);
  if (per <= 1) return launch_clusters(row_kernel<T, 512, 1>, P, size, 512, st);
  if (per <= 2) return launch_clusters(row_kernel<T, 512, 2>, P, size, 512, st);
  if (per <= 4) return launch_clusters(row_kernel<T, 512, 4>, P, size, 512, st);
  if constexpr (sizeof(T) == 4)
    if (per > 8) return launch_clusters(row_kernel<T, 1024, 8>, P, size, 1024, st);
  return launch_clusters(row_kernel<T, 512, 8>, P, size, 512, st);
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
  return by_type(P.x.type, [&](auto t) { return launch_loss<decltype(t)>(P, st); });
}
int launch_distill_loss_grad(const DistillParams& P, cudaStream_t st) {
  return by_type(P.x.type, [&](auto t) { return launch_rows<decltype(t)>(P, st); });
}
int launch_distill_backward(const DistillParams& P, cudaStream_t st) {
  return by_type(P.x.type, [&](auto t) {
    using T = decltype(t);
    const int units = P.x.vocab / kUnit<T>, per = kGradThreads * kGradUnits * kGradRounds;
    const int parts = units > per ? (units + per - 1) / per : 1;
    grad_kernel<T><<<(unsigned)P.x.rows * parts, kGradThreads, 0, st>>>(P, parts);
    return launch_status();
  });
}

}  // namespace sq
