// Drawing a token from a row of logits, and the k largest logits of a row.
//
// Draw.  With m the largest logit and c = log2(e) / T, token j has y_j = 2^((x_j - m) c)
// and the whole weight w_j = rint(y_j 2^31).  Tokens are ordered by logit, equal ones by
// index.  Top-k keeps the first k; top-p those whose predecessors hold less than p of the
// kept weight; min-p those with y_j >= min_p.  The token drawn is the first in index order
// at which the running weight passes floor(u W), W the weight that is left.  Weights are
// integers and their sums 64-bit, so no sum depends on the order it is formed in, and the
// token is a function of the inputs alone.  A token 2^-32 times less likely than the most
// likely one has weight 0; rounding moves at most 2^-32 of the largest weight a token.
//
// One CTA per row.  What top-k and top-p keep is a prefix of the order, described by the key
// of its last logit and the last index kept among equal logits (struct Cut); it is found by
// four passes over 8-bit digits of the key with a histogram of counts or weights.
#include "logits.cuh"
#include "logits_util.cuh"
#include <type_traits>

namespace sq {
namespace {

constexpr int NT = 512, NW = NT / 32;
typedef unsigned long long u64;

struct Cut { uint32_t key; int last; };          // kept: key above, or equal and index <= last

template <typename T>
struct Row {
  const T* p; int n;
  __device__ float at(int j) const { return plain_logit(to_f32(p[j])); }
};

struct Shared {
  u64 hist[256];
  u64 part[NW];
  float fpart[NW];
  uint32_t pick_key; u64 pick_above; int pick_index;
};

__device__ __forceinline__ u64 warp_sum_u64(u64 v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ u64 block_sum(u64 v, Shared& s) {
  v = warp_sum_u64(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s.part[threadIdx.x >> 5] = v;
  __syncthreads();
  u64 t = 0;
  for (int i = 0; i < NW; ++i) t += s.part[i];
  return t;
}
__device__ float block_max(float v, Shared& s) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s.fpart[threadIdx.x >> 5] = v;
  __syncthreads();
  float t = -INFINITY;
  for (int i = 0; i < NW; ++i) t = fmaxf(t, s.fpart[i]);
  return t;
}

// First index in index order at which the running sum of w(j, x) passes `target`
// (target < the total).  Each warp sums a contiguous stretch; the one that holds the
// crossing walks its stretch again.
template <typename T, typename W>
__device__ int locate(const Row<T>& r, W w, u64 target, Shared& s) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int len = (r.n + NW - 1) / NW, j0 = warp * len, j1 = min(r.n, j0 + len);
  u64 sum = 0;
  for (int j = j0 + lane; j < j1; j += 32) sum += w(j, r.at(j));
  sum = warp_sum_u64(sum);
  __syncthreads();
  if (lane == 0) s.part[warp] = sum;
  __syncthreads();
  u64 before = 0;
  for (int i = 0; i < warp; ++i) before += s.part[i];
  if (target >= before && target < before + sum) {
    for (int j = j0; j < j1; j += 32) {
      const int jj = j + lane;
      u64 v = jj < j1 ? w(jj, r.at(jj)) : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const u64 u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, before + v > target);
      if (hit) {
        if (lane == 0) s.pick_index = j + __ffs(hit) - 1;
        break;
      }
      before += __shfl_sync(0xffffffffu, v, 31);
    }
  }
  __syncthreads();
  const int at = s.pick_index;
  __syncthreads();
  return at;
}

// The cut after the first tokens of the order whose weights reach `need` (0 < need <= total):
// the last one kept is the first at which the running weight is >= need.
template <typename T, typename W>
__device__ Cut select(const Row<T>& r, W w, u64 need, Shared& s) {
  uint32_t prefix = 0;
  u64 above = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    __syncthreads();
    for (int i = threadIdx.x; i < 256; i += NT) s.hist[i] = 0;
    __syncthreads();
    for (int j = threadIdx.x; j < r.n; j += NT) {
      const float x = r.at(j);
      const uint32_t key = order_key(x);
      if (shift == 24 || (key >> (shift + 8)) == prefix) {
        const u64 v = w(j, x);
        if (v) atomicAdd(&s.hist[(key >> shift) & 255], v);
      }
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      u64 sum = above;
      int b = 255;
      while (b > 0 && sum + s.hist[b] < need) sum += s.hist[b--];
      s.pick_key = (prefix << 8) | b;
      s.pick_above = sum;
    }
    __syncthreads();
    prefix = s.pick_key;
    above = s.pick_above;
  }
  // equal logits have equal weights: the last kept is the one at which `above` reaches `need`
  const int last = locate(r, [&](int j, float x) -> u64 { return order_key(x) == prefix ? w(j, x) : 0; },
                          need - above - 1, s);
  return Cut{prefix, last};
}

template <typename T>
__global__ void __launch_bounds__(NT) sample_kernel(const SampleParams P) {
  __shared__ Shared s;
  const int row = blockIdx.x;
  const Row<T> r{reinterpret_cast<const T*>(P.x.data) + (long long)row * P.x.stride, P.x.vocab};
  const float temperature = P.temperature ? P.temperature[row] : P.temperature_all;
  const int top_k = P.top_k ? P.top_k[row] : P.top_k_all;
  const float top_p = P.top_p ? P.top_p[row] : P.top_p_all;
  const float min_p = fminf(P.min_p ? P.min_p[row] : P.min_p_all, 1.0f);
  float m = -INFINITY;
  for (int j = threadIdx.x; j < r.n; j += NT) m = fmaxf(m, r.at(j));
  m = block_max(m, s);
  if (m == -INFINITY) {
    if (threadIdx.x == 0) P.tokens[row] = -1;
    return;
  }
  if (!(temperature > 0.0f)) {
    const int at = locate(r, [&](int, float x) -> u64 { return x == m; }, 0, s);
    if (threadIdx.x == 0) P.tokens[row] = at;
    return;
  }
  const float c = __fdiv_rn(kLog2e, temperature);
  const auto power = [&](float x) { return x == m ? 1.0f : ex2(__fmul_rn(x - m, c)); };
  const auto weight = [&](float x) -> u64 { return __float2uint_rn(power(x) * 2147483648.0f); };
  Cut cut{0u, 0x7fffffff};
  const auto kept = [&](int j, float x) { const uint32_t k = order_key(x); return k > cut.key || (k == cut.key && j <= cut.last); };
  if (top_k > 0 && top_k < r.n) cut = select(r, [](int, float) -> u64 { return 1; }, (u64)top_k, s);
  if (!(top_p >= 1.0f)) {
    u64 z = 0;
    for (int j = threadIdx.x; j < r.n; j += NT) { const float x = r.at(j); if (kept(j, x)) z += weight(x); }
    z = block_sum(z, s);
    // kept: weight before it < top_p z; the first always
    const double limit = (double)top_p * (double)z;
    u64 need = limit > 1.0 ? (u64)ceil(limit) : 1;
    if (need > z) need = z;
    cut = select(r, [&](int j, float x) -> u64 { return kept(j, x) ? weight(x) : 0; }, need, s);
  }
  const auto left = [&](int j, float x) -> u64 { return kept(j, x) && power(x) >= min_p ? weight(x) : 0; };
  u64 total = 0;
  for (int j = threadIdx.x; j < r.n; j += NT) total += left(j, r.at(j));
  total = block_sum(total, s);
  const long long t = (long long)((double)P.uniform[row] * (double)total);
  const u64 target = t < 0 ? 0 : ((u64)t >= total ? total - 1 : (u64)t);
  const int at = locate(r, left, target, s);
  if (threadIdx.x == 0) P.tokens[row] = at;
}

template <typename T>
__global__ void __launch_bounds__(NT) top_kernel(const TopParams P) {
  __shared__ Shared s;
  __shared__ u64 list[kMaxRecord];
  __shared__ int count;
  const int row = blockIdx.x;
  const Row<T> r{reinterpret_cast<const T*>(P.x.data) + (long long)row * P.x.stride, P.x.vocab};
  u64 n = 0;
  for (int j = threadIdx.x; j < r.n; j += NT) n += r.at(j) > -INFINITY;
  n = block_sum(n, s);
  const int k = (int)min((u64)P.k, n);
  Cut cut{0u, -1};
  if (k > 0) cut = select(r, [](int, float x) -> u64 { return x > -INFINITY; }, (u64)k, s);
  int size = 32;
  while (size < P.k) size <<= 1;
  if (threadIdx.x == 0) count = 0;
  for (int i = threadIdx.x; i < size; i += NT) list[i] = 0;
  __syncthreads();
  if (k > 0)
    for (int j = threadIdx.x; j < r.n; j += NT) {
      const uint32_t key = order_key(r.at(j));
      if (key > cut.key || (key == cut.key && j <= cut.last))
        list[atomicAdd(&count, 1)] = ((u64)key << 32) | (uint32_t)~j;
    }
  __syncthreads();
  for (int len = 2; len <= size; len <<= 1)                    // bitonic, falling
    for (int d = len >> 1; d; d >>= 1) {
      for (int i = threadIdx.x; i < size; i += NT) {
        const int o = i ^ d;
        if (o > i) {
          const u64 a = list[i], b = list[o];
          if ((a < b) == ((i & len) == 0)) { list[i] = b; list[o] = a; }
        }
      }
      __syncthreads();
    }
  T* values = reinterpret_cast<T*>(P.values) + (long long)row * P.k;
  int* indices = P.indices + (long long)row * P.k;
  for (int i = threadIdx.x; i < P.k; i += NT) {
    const int j = i < k ? (int)~(uint32_t)list[i] : -1;
    values[i] = j >= 0 ? r.p[j] : from_f32<T>(-INFINITY);
    indices[i] = j;
  }
}

template <typename F>
int by_type(int type, F f) {
  switch (type) {
    case kLogitsF16: f((__half*)nullptr); return launch_status();
    case kLogitsBf16: f((__nv_bfloat16*)nullptr); return launch_status();
    case kLogitsF32: f((float*)nullptr); return launch_status();
  }
  return kEInval;
}

}  // namespace

int launch_sample(const SampleParams& P, cudaStream_t st) {
  return by_type(P.x.type, [&](auto* t) {
    sample_kernel<std::remove_pointer_t<decltype(t)>><<<P.x.rows, NT, 0, st>>>(P);
  });
}

int launch_top_logits(const TopParams& P, cudaStream_t st) {
  return by_type(P.x.type, [&](auto* t) {
    top_kernel<std::remove_pointer_t<decltype(t)>><<<P.x.rows, NT, 0, st>>>(P);
  });
}

}  // namespace sq
