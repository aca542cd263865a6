// Distillation from a teacher's record of its largest logits, and its gradient.
//
// Student logits s over the whole vocabulary, teacher entries (v_k, j_k), temperature T,
// c = log2(e) / T, everything in powers of two:
//   q_k = 2^((v_k - v_max) c) / Q,  Q their sum      p_j = 2^((s_j - m) c) / S,  S the sum
//   loss = T sum_k q_k [ T ln 2 ((v_k - v_max) c + log2 S - log2 Q) - (s_jk - m) ]
//   d loss / d s_j = T (p_j - sum over k with j_k = j of q_k)
// An entry whose index lies outside the vocabulary, or whose logit is -inf or NaN, is unused;
// a row without used entries has loss 0 and gradient 0.  Sums are fp32; p and the difference
// p - q are fp32 and rounded once to the logits' type.
//
// loss_kernel: the forward.  The CTAs of a cluster stream their parts of the row with a running
// maximum and sum per thread, eight loads of 16 bytes in flight each.  Bound by HBM: 512 rows of 256,000 fp16
// logits (262 MB) take 56 us, 4.7 TB/s; 2,048 rows of bf16 182 us, 5.8 TB/s; 1,024 rows of fp32 164 us, 6.4 TB/s.  At 512
// rows 1,024 CTAs meet 592 places (64 registers, four CTAs an SM): the second wave is three quarters full.  In 16 bits the
// power unit is half busy.
// row_kernel: loss and gradient in one pass.  The CTAs of a cluster hold the row in shared memory:
// asynchronous copies bring it while the record is worked through, and the gradient is computed from
// there, so the logits are read from HBM once.  Eight data warps and a record warp a CTA, three CTAs on an
// SM, stepping through the rows: a thread refills the place of a unit as soon as it has written its gradient, and
// nothing but one cluster barrier a row stands between a row's two passes.  2,048 rows of 256,000 bf16 logits
// (1.05 GB in, 1.05 GB out) take 0.49 ms, 4.3 TB/s; what is left is the wait at that barrier and the issue of
// 17 instructions a logit (two powers among them).  That is with records of 64: equal indices are looked for by a scan of
// the record for each entry, and records of 256 take 0.97 ms, of 1,024 7.0 ms.  Reading the logits a second time from L2 instead of keeping them
// (no shared memory, four CTAs on an SM) took 0.62 ms.
// In both each warp sends its (maximum, sum) to every CTA of the cluster through distributed shared
// memory.  The sums are formed in a fixed order: the same call gives the same bits.
// grad_kernel: the backward of a forward whose statistics were kept, streaming; p is computed again from
// them.  1,024 rows of 256,000 bf16 logits take 0.18 ms, 5.8 TB/s.
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
// c: finite for every T, so that 0 c stays 0 (infinite below T = 4e-39 otherwise).
__device__ __forceinline__ float slope(float temperature) { return fminf(kLog2e / temperature, 3.4028234e38f); }
// (v - v_max) c; the largest entry is 0 even where it is infinite.
__device__ __forceinline__ float record_power(float v, float vmax, float c) { return v == vmax ? 0.0f : (v - vmax) * c; }
// The loss over T of a row whose record's powers sum to Q, entry by entry: the student's gap is taken as it is and T enters
// once, since c and T^2 leave fp32's range long before T does.
struct LossTerm {
  float scale, rest;                             // T ln 2, T ln 2 (log2 S - log2 Q)
  __device__ LossTerm(float temperature, float sum, float Q)
      : scale(temperature * kLn2), rest(scale * (log2f(sum) - log2f(Q))) {}
  // e: the entry's exponent; gap: the student's logit less its reference
  __device__ float operator()(float e, float gap) const { return fmaf(e, scale, rest) - gap; }
};

// (x - r) c for two: r is the largest logit, or 0 where there is none above -inf (powers of -inf are 0
// then, and a NaN stays one).
__device__ __forceinline__ float2 exponent2(float2 x, float c, float r) {
  return __fmul2_rn(__fadd2_rn(x, make_float2(-r, -r)), make_float2(c, c));
}
template <typename T>
__device__ __forceinline__ float2 pair_of(const Unit<T>& u, int v) { return make_float2(to_f32(u.v[v]), to_f32(u.v[v + 1])); }

// Adds the powers of a unit to two running sums.
template <typename T>
__device__ __forceinline__ void add_powers(float2& sum, const Unit<T>& u, float c, float r) {
#pragma unroll
  for (int v = 0; v < kUnit<T>; v += 2) {
    const float2 t = exponent2(pair_of(u, v), c, r);
    sum = __fadd2_rn(sum, make_float2(ex2(t.x), ex2(t.y)));
  }
}
__device__ __forceinline__ void store_pair(Unit<__half>& o, int v, float2 p) {
  reinterpret_cast<__half2*>(&o.q)[v / 2] = __float22half2_rn(p);
}
__device__ __forceinline__ void store_pair(Unit<__nv_bfloat16>& o, int v, float2 p) {
  reinterpret_cast<__nv_bfloat162*>(&o.q)[v / 2] = __float22bfloat162_rn(p);
}
__device__ __forceinline__ void store_pair(Unit<float>& o, int v, float2 p) { o.v[v] = p.x; o.v[v + 1] = p.y; }
// Stores the units of a warp's first n lanes one behind the other from `to` on.  The gradient's rows may lie
// otherwise in their 16 bytes than the logits' rows: then (`vec` false) the units pass through `buf` (512
// bytes of shared memory a warp) and leave it in whole units of the destination, whose ends go element by element.
template <typename T>
__device__ __forceinline__ void store_units(T* to, const Unit<T>& o, int n, bool vec, uint4* buf) {
  const int lane = threadIdx.x & 31;
  if (vec) {
    if (lane < n) reinterpret_cast<uint4*>(to)[lane] = o.q;
    return;
  }
  __syncwarp();
  buf[lane] = o.q;
  __syncwarp();
  const int head = (16 - (int)((uintptr_t)to & 15)) / (int)sizeof(T);        // elements up to the first whole unit
  if (lane < n - 1) {
    const uint32_t a = (uint32_t)__cvta_generic_to_shared(buf) + 16u * lane + head * (uint32_t)sizeof(T), word = a & ~3u;
    uint32_t w[5];
#pragma unroll
    for (int b = 0; b < 5; ++b) asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[b]) : "r"(word + 4u * b));
    if (sizeof(T) == 2 && (a & 2)) {
#pragma unroll
      for (int b = 0; b < 4; ++b) w[b] = __funnelshift_r(w[b], w[b + 1], 16);
    }
    *reinterpret_cast<uint4*>(to + head + lane * kUnit<T>) = make_uint4(w[0], w[1], w[2], w[3]);
  }
  if (lane < kUnit<T> && n > 0) {
    const int e = lane < head ? lane : (n - 1) * kUnit<T> + lane;
    to[e] = reinterpret_cast<const T*>(buf)[e];
  }
}
// Copies n elements from shared memory to `to` in whole 16-byte units of the destination, its ends element
// by element.
template <typename T, int NT>
__device__ void copy_out(T* to, int n, const T* from) {
  const int head = min(n, (int)((16 - ((uintptr_t)to & 15)) & 15) / (int)sizeof(T)), units = (n - head) / kUnit<T>;
  const uint32_t src = (uint32_t)__cvta_generic_to_shared(from + head);
  for (int i = threadIdx.x; i < units; i += NT) {
    const uint32_t a = src + 16u * i, word = a & ~3u;
    uint32_t w[5];
#pragma unroll
    for (int b = 0; b < 4; ++b) asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[b]) : "r"(word + 4u * b));
    if (sizeof(T) == 2 && (a & 2)) {
      asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[4]) : "r"(word + 16u));
#pragma unroll
      for (int b = 0; b < 4; ++b) w[b] = __funnelshift_r(w[b], w[b + 1], 16);
    }
    reinterpret_cast<uint4*>(to + head)[i] = make_uint4(w[0], w[1], w[2], w[3]);
  }
  const int tail = head + units * kUnit<T>;
  for (int i = threadIdx.x; i < head + n - tail; i += NT) {
    const int j = i < head ? i : tail + (i - head);
    to[j] = from[j];
  }
}
__device__ __forceinline__ float reference(float m) { return m == -INFINITY ? 0.f : m; }
// scale 2^((x - r) c) for a unit; zeros where `any` is not set.
template <typename T>
__device__ __forceinline__ Unit<T> gradient(const Unit<T>& x, float c, float r, float scale, bool any) {
  Unit<T> o;
  o.q = make_uint4(0, 0, 0, 0);
  if (any) {
#pragma unroll
    for (int v = 0; v < kUnit<T>; v += 2) {
      const float2 t = exponent2(pair_of(x, v), c, r);
      const float2 p = __fmul2_rn(make_float2(ex2(t.x), ex2(t.y)), make_float2(scale, scale));
      store_pair(o, v, p);
    }
  }
  return o;
}

__device__ __forceinline__ float warp_total(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// Barrier of the warps that work on the row.
template <int NT> __device__ __forceinline__ void data_barrier() { asm volatile("bar.sync 1, %0;" :: "n"(NT) : "memory"); }

// (maximum, sum relative to its reference) of every warp of the cluster.
template <int NW>
struct Pairs {
  float2 p[8 * NW];
  // Hands a warp's maximum and the threads' shares of its sum to all CTAs of the cluster, which run; a
  // cluster barrier has to follow.
  __device__ void send(float m, float sum, uint32_t rank, uint32_t size) {
    sum = warp_total(sum);
    const int lane = threadIdx.x & 31;
    if (lane < (int)size)
      remote_store(remote_smem(&p[rank * NW + (threadIdx.x >> 5)], lane), m, sum);
  }
  // The row's reference and sum.
  __device__ void merge(uint32_t size, float c, float& r, float& sum) const {
    const int n = (int)size * NW;
    float top = -INFINITY;
    for (int i = threadIdx.x & 31; i < n; i += 32) top = fmaxf(top, p[i].x);
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    sum = 0.f;
    for (int i = threadIdx.x & 31; i < n; i += 32) sum += p[i].x == top ? p[i].y : p[i].y * ex2((p[i].x - top) * c);
    sum = warp_total(sum);
    r = reference(top);
  }
};
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// One row's record of at most N NT entries: each thread holds entries tid, tid + NT, ...
template <typename T, int NT, int N>
struct Record {
  int at[N];                                     // -1: unused
  float e[N];                                    // (v - v_max) c
  float taken[N];                                // student's logit there
  float vmax, Q;
  __device__ void read(const DistillParams& P, int row, const T* s, float c, float (*part)[NT / 32]) {
    const long long base = (long long)row * P.k;
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
          taken[i] = to_f32(s[j]);
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
  // Loss of the row, to thread 0; every thread of the CTA calls.
  __device__ float loss(float r, float sum, float temperature, float (*part)[NT / 32]) const {
    float l = 0.f;
    const LossTerm term(temperature, sum, Q);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float w = ex2(e[i]);
      if (at[i] >= 0 && w > 0.f) l += w * term(e[i], taken[i] - r);
    }
    l = block_sum<NT>(l, part[0]);
    return Q > 0.f ? temperature * (l / Q) : 0.f;
  }
};

constexpr int kLossUnits = 8;

template <typename T, int NT, int N>
__global__ void __launch_bounds__(NT, 1024 / NT) loss_kernel(const DistillParams P) {
  constexpr int NV = kLossUnits, NW = NT / 32;
  __shared__ Pairs<NW> pairs;
  __shared__ float part[2][NW];
  const uint32_t rank = cluster_rank(), size = cluster_size();
  const int row = blockIdx.x / size, tid = threadIdx.x;
  const float c = slope(P.temperature);
  const Span<T> span(P.x, row, rank, size);
  cluster_arrive_relaxed();
  const uint4* body = reinterpret_cast<const uint4*>(span.p + span.col(0, 0));
  const auto load = [&](Unit<T> (&x)[NV], int from) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int u = from + i * NT + tid;
      x[i].q = neg_inf_unit<T>();
      if (u < span.hi) x[i].q = load_unit(body + u);
    }
  };
  float m = -INFINITY, ref = 0.f;
  float2 sum = make_float2(0.f, 0.f);
  const auto raise = [&](float top) {
    if (top > m) {
      const float f = m == -INFINITY ? 1.0f : ex2((m - top) * c);
      sum = __fmul2_rn(sum, make_float2(f, f));
      m = ref = top;
    }
  };
  Unit<T> x[NV];
  load(x, span.lo);
  Record<T, NT, N> rec;
  if (rank == 0) rec.read(P, row, span.p, c, part);
#pragma unroll 1
  for (int from = span.lo; from < span.hi; from += NT * NV) {
    if (from != span.lo) load(x, from);
    float top = unit_max(x[0]);
#pragma unroll
    for (int i = 1; i < NV; ++i) top = fmaxf(top, unit_max(x[i]));
    raise(top);
#pragma unroll
    for (int i = 0; i < NV; ++i) add_powers(sum, x[i], c, ref);
  }
  if (tid < 2) {                                 // the row's ragged ends
    const int at = tid == 0 ? (span.lo > 0 ? 0 : -1) : (span.hi < span.n ? span.hi : -1);
    if (at >= 0) {
      const Unit<T> end = span.ragged(at);
      raise(unit_max(end));
      add_powers(sum, end, c, ref);
    }
  }
  const float wm = warp_max(m);
  float own = sum.x + sum.y, r;
  if (m != -INFINITY && m != wm) own *= ex2((m - wm) * c);
  cluster_wait();                                // every CTA of the cluster runs
  pairs.send(wm, own, rank, size);
  cluster_arrive();
  cluster_wait();
  pairs.merge(size, c, r, own);
  if (rank != 0) return;
  const float l = rec.loss(r, own, P.temperature, part);
  if (tid == 0) {
    P.loss[row] = l;
    if (P.stats) P.stats[row] = make_float4(r, 1.0f / own, rec.vmax, rec.Q > 0.f ? 1.0f / rec.Q : 0.f);
  }
}

// The record's tokens in the gradient: each by its first entry, repeated indices added up.
// at: the row's indices (-1: unused, and up to a multiple of four) in shared memory; q(i): entry i's 2^e.
// Returns the sum of q over the entries of index j if entry k is the first of them, else -1.
template <typename F>
__device__ __forceinline__ float sum_of_index(const int* at, int n, int k, int j, F q) {
  float sum = 0.f;
  for (int b = 0; b < n; b += 4) {
    const int4 a = *reinterpret_cast<const int4*>(at + b);
    if (a.x != j && a.y != j && a.z != j && a.w != j) continue;
    const int same[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int o = 0; o < 4; ++o)
      if (same[o] == j) {
        if (b + o < k) return -1.f;
        sum += q(b + o);
      }
  }
  return sum;
}

// The record warp's side of row_kernel: one row's record in shared memory, lane l works on entries l, l + 32, ...
template <typename T>
struct RowRecord {
  int* at;                                       // index (-1: unused, and up to a multiple of four)
  float *e, *taken, *token;                      // (v - v_max) c; student's logit; sum of 2^e over the index, or < 0
  float Q;
  static __device__ __host__ size_t bytes(int k4) { return (size_t)k4 * 16; }
  __device__ RowRecord(unsigned char* p, int k4) {
    at = reinterpret_cast<int*>(p);
    e = reinterpret_cast<float*>(at + k4);
    taken = e + k4;
    token = taken + k4;
  }
  // Columns [col0, col1) are this CTA's to correct; CTA 0 needs the student's logit everywhere.
  __device__ void prepare(const DistillParams& P, int row, const T* s, float c, bool all, int col0, int col1) {
    const int lane = threadIdx.x & 31, k4 = (P.k + 3) & ~3;
    const long long base = (long long)row * P.k;
    float vmax = -INFINITY, q = 0.f;
    for (int k = lane; k < k4; k += 32) {
      int j = -1;
      float v = -INFINITY;
      if (k < P.k) {
        j = P.indices[base + k];
        v = record_value(P, base + k);
        if (!used_entry(P, j, v)) j = -1;
        else vmax = fmaxf(vmax, v);
      }
      at[k] = j;
      e[k] = v;
      const bool mine = j >= col0 && j < col1;
      token[k] = mine ? 0.f : -1.f;
      if (j >= 0 && (all || mine)) taken[k] = to_f32(s[j]);
    }
    vmax = warp_max(vmax);
    for (int k = lane; k < k4; k += 32) {
      const float p = at[k] < 0 ? -INFINITY : record_power(e[k], vmax, c);
      e[k] = p;
      q += ex2(p);
    }
    Q = warp_total(q);
    __syncwarp();
    for (int k = lane; k < P.k; k += 32)
      if (token[k] == 0.f) token[k] = sum_of_index(at, P.k, k, at[k], [&](int i) { return ex2(e[i]); });
    __syncwarp();
  }
  __device__ float loss(int n, float r, float sum, float temperature) const {
    float l = 0.f;
    if (!(Q > 0.f)) return 0.f;
    const LossTerm term(temperature, sum, Q);
    for (int k = threadIdx.x & 31; k < n; k += 32) {
      const float w = ex2(e[k]);
      if (at[k] >= 0 && w > 0.f) l += w * term(e[k], taken[k] - r);
    }
    return temperature * (warp_total(l) / Q);
  }
  // The gradient at the record's tokens, over what the data warps wrote there.
  __device__ void correct(int n, T* g, float r, float c, float scale, float f) const {
    if (!(Q > 0.f)) return;
    const float fq = f / Q;
    for (int k = threadIdx.x & 31; k < n; k += 32)
      if (token[k] >= 0.f) g[at[k]] = from_f32<T>(ex2((taken[k] - r) * c) * scale - fq * token[k]);
  }
};

// DW warps work on the row, one more on the record: it prepares the next row's while they compute this
// one's gradient, and corrects the gradient of a row after the next row's barrier.
template <typename T, int DW>
__global__ void __launch_bounds__(DW * 32 + 32, 24 / DW) row_kernel(const DistillParams P) {
  constexpr int NT = DW * 32;
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ Pairs<DW> pairs[2];                 // of this row and, from CTAs ahead, of the next
  __shared__ int has_record[2];
  const uint32_t rank = cluster_rank(), size = cluster_size();
  const int tid = threadIdx.x, step = gridDim.x / size, k4 = (P.k + 3) & ~3;
  const float c = slope(P.temperature);
  cluster_arrive_relaxed();
  int row = blockIdx.x / size;
  Span<T> span(P.x, row, rank, size);
  const auto first_col = [](const Span<T>& s) { return max(0, s.col(0, 0)); };
  const auto last_col = [](const Span<T>& s) { return min(s.vocab, s.col(s.n, 0)); };
  const auto weight = [&](int row) { return P.temperature * (P.weight ? P.weight[row * P.weight_stride] : 1.0f); };

  if (tid >= NT) {
    RowRecord<T> now(dyn, k4), before(dyn + RowRecord<T>::bytes(k4), k4);
    T* g_before = nullptr;
    float r_before = 0.f, scale_before = 0.f, f_before = 0.f;
    now.prepare(P, row, span.p, c, rank == 0, first_col(span), last_col(span));
    if (tid == NT) has_record[0] = now.Q > 0.f;
    cluster_wait();                              // every CTA of the cluster runs
    for (int turn = 0; row < P.x.rows; row += step) {
      float r, sum;
      const float f = weight(row);
      cluster_arrive();
      cluster_wait();
      pairs[turn].merge(size, c, r, sum);
      turn ^= 1;
      if (g_before) before.correct(P.k, g_before, r_before, c, scale_before, f_before);
      if (rank == 0) {
        const float l = now.loss(P.k, r, sum, P.temperature);
        if (tid == NT) P.loss[row] = l;
      }
      g_before = reinterpret_cast<T*>(P.grad) + (long long)row * P.grad_stride;
      r_before = r; scale_before = f / sum; f_before = f;
      const RowRecord<T> swap = before;
      before = now;
      now = swap;
      if (row + step < P.x.rows) {
        const Span<T> next(P.x, row + step, rank, size);
        __syncwarp();
        now.prepare(P, row + step, next.p, c, rank == 0, first_col(next), last_col(next));
        if (tid == NT) has_record[turn] = now.Q > 0.f;
      }
    }
    __syncthreads();
    before.correct(P.k, g_before, r_before, c, scale_before, f_before);
    return;
  }

  // whole units, from that of column span.col(span.lo, 0); a thread brings and uses tid, tid + NT, ...
  Unit<T>* unit = reinterpret_cast<Unit<T>*>(dyn + 2 * RowRecord<T>::bytes(k4));
  for (int i = tid; i < span.hi - span.lo; i += NT) cp_async16(unit + i, span.p + span.col(span.lo + i, 0));
  // a ragged end of the row, held by one of two threads
  const auto end_of = [&](const Span<T>& s) { return tid == 0 && s.lo > 0 ? 0 : tid == 1 && s.hi < s.n ? s.hi : -1; };
  int end_unit = end_of(span);
  Unit<T> end;
  end.q = neg_inf_unit<T>();
  if (end_unit >= 0) end = span.ragged(end_unit);
  cluster_wait();                                // every CTA of the cluster runs

  for (int turn = 0; row < P.x.rows; row += step, turn ^= 1) {
    const int units = span.hi - span.lo;
    const float f = weight(row);
    cp_async_wait_all();
    float m = unit_max(end), ref = reference(m);
    float2 sums = make_float2(0.f, 0.f);
    add_powers(sums, end, c, ref);
    const auto raise = [&](float top) {
      if (top > m) {
        const float f = m == -INFINITY ? 1.0f : ex2((m - top) * c);
        sums = __fmul2_rn(sums, make_float2(f, f));
        m = ref = top;
      }
    };
    int i = tid;
    for (; i + 3 * NT < units; i += 4 * NT) {
      Unit<T> x[4];
#pragma unroll
      for (int a = 0; a < 4; ++a) x[a].q = unit[i + a * NT].q;
      raise(fmaxf(fmaxf(unit_max(x[0]), unit_max(x[1])), fmaxf(unit_max(x[2]), unit_max(x[3]))));
#pragma unroll
      for (int a = 0; a < 4; ++a) add_powers(sums, x[a], c, ref);
    }
    for (; i < units; i += NT) {
      Unit<T> x;
      x.q = unit[i].q;
      raise(unit_max(x));
      add_powers(sums, x, c, ref);
    }
    float sum = sums.x + sums.y, r;
    const float wm = warp_max(m);
    if (m != -INFINITY && m != wm) sum *= ex2((m - wm) * c);
    pairs[turn].send(wm, sum, rank, size);
    cluster_arrive();
    cluster_wait();
    pairs[turn].merge(size, c, r, sum);

    T* g = reinterpret_cast<T*>(P.grad) + (long long)row * P.grad_stride;
    const bool any = has_record[turn];
    const float scale = f / sum;
    // the units of the next row follow into the places of this one's as these are done
    const bool more = row + step < P.x.rows;
    const Span<T> next(P.x, more ? row + step : row, rank, size);
    const int fetched = more ? next.hi - next.lo : 0;
    const T* from = next.p + next.col(next.lo, 0);
    T* to = g + span.col(span.lo, 0);
    i = tid;
    if (((uintptr_t)to & 15) == 0) {
#pragma unroll 2
      for (; i < units; i += NT) {
        Unit<T> x;
        x.q = unit[i].q;
        reinterpret_cast<uint4*>(to)[i] = gradient(x, c, r, scale, any).q;
        if (i < fetched) cp_async16(unit + i, from + i * kUnit<T>);
      }
    } else {
      // The gradient's rows lie otherwise in their 16 bytes than the logits' rows: it takes the logits'
      // place in shared memory and is copied out from there in whole units of its own.
      for (; i < units; i += NT) {
        Unit<T> x;
        x.q = unit[i].q;
        unit[i].q = gradient(x, c, r, scale, any).q;
      }
      data_barrier<NT>();
      copy_out<T, NT>(to, units * kUnit<T>, reinterpret_cast<const T*>(unit));
      data_barrier<NT>();
      i = tid;
    }
    for (; i < fetched; i += NT) cp_async16(unit + i, from + i * kUnit<T>);
    if (end_unit >= 0) {
      const Unit<T> o = gradient(end, c, r, scale, any);
      for (int v = 0; v < kUnit<T>; ++v) {
        const int j = span.col(end_unit, v);
        if (j >= 0 && j < span.vocab) g[j] = o.v[v];
      }
    }
    span = next;
    end_unit = end_of(span);
    end.q = neg_inf_unit<T>();
    if (more && end_unit >= 0) end = span.ragged(end_unit);
  }
  __syncthreads();
}

constexpr int kGradUnits = 8;

template <typename T, int NT>
__global__ void __launch_bounds__(NT, 1024 / NT) grad_kernel(const DistillParams P, int parts) {
  constexpr int NV = kGradUnits;
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ uint4 bounce[NT / 32][32];
  int* at = reinterpret_cast<int*>(dyn);         // the record's indices (-1: unused) and 2^e
  float* w = reinterpret_cast<float*>(at + ((P.k + 3) & ~3));
  const int row = blockIdx.x / parts, part = blockIdx.x - row * parts, tid = threadIdx.x;
  const float c = slope(P.temperature);
  const Span<T> span(P.x, row, part, parts);
  const T* s = span.p;
  T* g = reinterpret_cast<T*>(P.grad) + (long long)row * P.grad_stride;
  const uint4* body = reinterpret_cast<const uint4*>(s + span.col(span.lo, 0));
  T* to = g + span.col(span.lo, 0);
  const int units = span.hi - span.lo;
  const auto load = [&](Unit<T> (&x)[NV], int from) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int u = from + i * NT + tid;
      if (u < units) x[i].q = load_unit(body + u);
    }
  };
  Unit<T> x[NV];
  load(x, 0);
  const float4 st = P.stats[row];
  const float r = st.x, f = P.temperature * (P.weight ? P.weight[row * P.weight_stride] : 1.0f), scale = f * st.y;
  const bool any = st.w > 0.f;
  const long long base = (long long)row * P.k;
  for (int k = tid; k < ((P.k + 3) & ~3); k += NT) {
    const int j = k < P.k ? P.indices[base + k] : -1;
    const float v = k < P.k ? record_value(P, base + k) : 0.f;
    const bool used = used_entry(P, j, v);
    at[k] = used ? j : -1;
    w[k] = used ? ex2(record_power(v, st.z, c)) : 0.f;
  }
  const bool vec = ((uintptr_t)to & 15) == 0;
#pragma unroll 1
  for (int from = 0; from < units; from += NT * NV) {
    if (from) load(x, from);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int first = from + i * NT + tid - (tid & 31);
      store_units(to + first * kUnit<T>, gradient(x[i], c, r, scale, any), max(0, min(32, units - first)), vec, bounce[tid >> 5]);
    }
  }
  const int col0 = max(0, span.col(0, 0)), col1 = min(span.vocab, span.col(span.n, 0));
  if (tid < 2) {                                 // the row's ragged ends
    const int u = tid == 0 ? (span.lo > 0 ? 0 : -1) : (span.hi < span.n ? span.hi : -1);
    if (u >= 0) {
      const Unit<T> o = gradient(span.ragged(u), c, r, scale, any);
      for (int v = 0; v < kUnit<T>; ++v) {
        const int j = span.col(u, v);
        if (j >= col0 && j < col1) g[j] = o.v[v];
      }
    }
  }
  __syncthreads();
  if (!any) return;
  for (int k = tid; k < P.k; k += NT) {
    const int j = at[k];
    if (j < col0 || j >= col1) continue;         // unused, or another CTA's
    const float q = sum_of_index(at, P.k, k, j, [&](int i) { return w[i]; });
    if (q >= 0.f) g[j] = from_f32<T>(ex2((to_f32(s[j]) - r) * c) * scale - f * (q * st.w));
  }
}

template <typename T>
int launch_loss(const DistillParams& P, cudaStream_t st) {
  // long parts stream best: more CTAs a row only until there are six for each SM (512 rows of 256,000 fp16: 56 us;
  // until three 60, until twelve 61); short rows, many at once, take CTAs of two warps
  // (16,384 rows of 8,191 bf16 logits: 98 us, with eight 181)
  const int units = row_units(P.x);
  if (units <= 1280 && P.x.rows > 4 * kSms && P.k <= 128) return launch_clusters(loss_kernel<T, 64, 2>, P, 1, 64, 0, st);
  int size = 1;
  while (size < 8 && P.x.rows * size < 6 * kSms && units > size * 256 * kLossUnits) size *= 2;
  return launch_clusters(loss_kernel<T, 256, 4>, P, size, 256, 0, st);
}

template <typename T, int DW>
int launch_rows(const DistillParams& P, int size, cudaStream_t st) {
  const size_t smem = 2 * RowRecord<T>::bytes((P.k + 3) & ~3) + (size_t)((row_units(P.x) + size - 1) / size) * 16;
  const auto kernel = row_kernel<T, DW>;
  static std::atomic<uint64_t> done{0};
  if (allow_shared(kernel, 200 * 1024, done) != cudaSuccess) return launch_status();
  // up to two CTAs an SM one row is a cluster's work; beyond, clusters step through the rows
  return launch_clusters(kernel, P, size, DW * 32 + 32, smem, st, true, 2 * kSms);
}

template <typename T>
int launch_loss_grad(const DistillParams& P, cudaStream_t st) {
  // As many CTAs a row as keep its part within 64 KB, three of eight data warps on an SM; few rows take
  // more, down to a unit a thread.  Short rows, many at once, are better served by CTAs of two data warps
  // (16,384 rows of 8,191 bf16 logits: 225 us, with eight 428).  fp32 rows of 512 to 768 KB leave parts of 64 to 96 KB,
  // two or three of them on an SM; longer ones parts of which one fits an SM, with 16 warps.
  const int units = row_units(P.x);
  int size = 1;
  while (size < 8 && (units + size - 1) / size > 4096) size *= 2;
  while (size < 8 && P.x.rows * size < 2 * kSms && units > size * 256) size *= 2;
  if constexpr (sizeof(T) == 4)
    if ((units + size - 1) / size > 6144) return launch_rows<T, 16>(P, size, st);
  if (size == 1 && units <= 1280 && P.x.rows > 4 * kSms) return launch_rows<T, 2>(P, size, st);
  return launch_rows<T, 8>(P, size, st);
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
  return by_type(P.x.type, [&](auto t) { return launch_loss_grad<decltype(t)>(P, st); });
}
int launch_distill_backward(const DistillParams& P, cudaStream_t st) {
  return by_type(P.x.type, [&](auto t) {
    using T = decltype(t);
    // a CTA of eight warps writes 64 KB of a row; short rows, many at once, take two warps each (16,384 rows of
    // 8,191 bf16 logits: 106 us, with eight 213)
    const int units = row_units(P.x), smem = ((P.k + 3) & ~3) * 8;
    if (units <= 1280 && P.x.rows > 4 * kSms) {
      grad_kernel<T, 64><<<(unsigned)P.x.rows, 64, smem, st>>>(P, 1);
    } else {
      const int parts = (units + 4095) / 4096;
      grad_kernel<T, 256><<<(unsigned)P.x.rows * parts, 256, smem, st>>>(P, parts);
    }
    return launch_status();
  });
}

}  // namespace sq
