// Short causal convolution of a mixer's channels, its gradients and its one-token form, and activations kept in 8 bits
// (sm_100a).
//
//   z[t,c] = bias[c] + sum_k w[c,k] x[t - (taps-1) + k, c],   y = z sigmoid(z) or z
//
// Tokens before the first are the carried state's, or zero.  Everything is fp32 inside and rounded once.  All of it is
// bound by memory: a thread owns four channels and a strip of tokens, with the last taps' inputs in registers, so that
// each input is read once but for the strips' edges.  The backward pass computes z again from the input (or from its
// 8-bit codes); sums for weights and bias are kept a strip and added in order by a second kernel, the same in every run.
//
// 8 bits: 128 neighbouring channels of a token share the scale max|x| (1 / 127), an fp32 product; a code is the fp32 quotient
// x / scale rounded to even, at most 127.
#include "conv.cuh"
#include "selective.cuh"
#include "device_util.cuh"
#include "logits_util.cuh"
#include "pairs.cuh"

namespace sq {
namespace {

constexpr int kThreads = 128;
constexpr int kTaps = 4;                            // most taps; fewer use the last ones
// Channels of a thread of the convolutions.  Four: eight of 16 bits would take 235 registers in the gradients, with too few
// warps on an SM to have the loads in flight that memory needs.
constexpr int kWide = 4;

// V neighbouring values as memory has them; `n` of them are there.  vec: all are, and lie at a multiple of their size.
template <int BYTES> struct Word;
template <> struct Word<16> { using type = uint4; };
template <> struct Word<8> { using type = uint2; };
template <> struct Word<4> { using type = uint32_t; };
template <typename T, int V> union Values {
  typename Word<V * (int)sizeof(T)>::type q;
  T v[V];
};
template <typename T, int V> __device__ __forceinline__ Values<T, V> no_values() {
  Values<T, V> u;
  u.q = decltype(u.q){};
  return u;
}
template <typename T, int V> __device__ __forceinline__ Values<T, V> raw_values(const T* p, bool vec, int n) {
  Values<T, V> u;
  if (vec) {
    u.q = *reinterpret_cast<const decltype(u.q)*>(p);
  } else {
    u.q = decltype(u.q){};
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < n) u.v[i] = p[i];
  }
  return u;
}
template <typename T, int V> __device__ __forceinline__ void load_values(const T* p, bool vec, int n, float (&f)[V]) {
  const Values<T, V> u = raw_values<T, V>(p, vec, n);
#pragma unroll
  for (int i = 0; i < V; ++i) f[i] = to_f32(u.v[i]);
}
// Neighbours 2i and 2i + 1.
template <typename T, int V> __device__ __forceinline__ float2 two(const Values<T, V>& u, int i) {
  if constexpr (sizeof(T) == 4) return make_float2(u.v[2 * i], u.v[2 * i + 1]);
  else return unpack2<T>(reinterpret_cast<const uint32_t*>(&u)[i]);
}
template <typename T, int V> __device__ __forceinline__ void load_pairs(const T* p, bool vec, int n, float2 (&f)[V / 2]) {
  const Values<T, V> u = raw_values<T, V>(p, vec, n);
#pragma unroll
  for (int i = 0; i < V / 2; ++i) f[i] = two<T, V>(u, i);
}
template <typename T, int V> __device__ __forceinline__ void store_pairs(T* p, bool vec, int n, const float2* f) {
  Values<T, V> u;
#pragma unroll
  for (int i = 0; i < V / 2; ++i) {
    if constexpr (sizeof(T) == 4) { u.v[2 * i] = f[i].x; u.v[2 * i + 1] = f[i].y; }
    else reinterpret_cast<uint32_t*>(&u)[i] = pack2<T>(f[i].x, f[i].y);
  }
  if (vec) {
    *reinterpret_cast<decltype(u.q)*>(p) = u.q;
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < n) p[i] = u.v[i];
  }
}

// ---------------------------------------------------------------- 8 bits
constexpr float kWhole = 12582912.0f;               // 1.5 * 2^23: added to a small number it leaves the rounded one in the low bits

template <int V> __device__ __forceinline__ void store_codes(int8_t* p, bool vec, int n, const Values<int8_t, V>& u) {
  if (vec) {
    *reinterpret_cast<decltype(u.q)*>(p) = u.q;
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < n) p[i] = u.v[i];
  }
}
// A code as the low byte of 2^23 + 128 + code: no conversion, which has a sixteenth of the adds' rate.
template <int V> __device__ __forceinline__ void decode(const Values<int8_t, V>& u, float scale, float2 (&f)[V / 2]) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(&u);
#pragma unroll
  for (int i = 0; i < V / 2; ++i) {
    const uint32_t four = w[i >> 1] ^ 0x80808080u;
    const float2 v = words2(__byte_perm(four, 0x4b000000u, 0x7540 + 2 * (i & 1)), __byte_perm(four, 0x4b000000u, 0x7541 + 2 * (i & 1)));
    f[i] = mul2(add2(v, pair(-8388736.0f)), pair(scale));
  }
}
// The largest magnitude of some values, as its fp32 bits; a NaN is larger than any number.
template <int V> __device__ __forceinline__ uint32_t top_bits(const Values<float, V>& u) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < V; ++i) m = max(m, __float_as_uint(u.v[i]) & 0x7fffffffu);
  return m;
}
template <typename T, int V> __device__ __forceinline__ uint32_t top_bits(const Values<T, V>& u) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(&u);
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < V / 2; ++i) m = __vmaxu2(m, w[i] & 0x7fff7fffu);
  return __float_as_uint(to_f32(from_bits<T>(max(m & 0xffffu, m >> 16))));
}
// Scale and codes of the 128 values of which this thread has V; the others are its neighbours'.  A NaN or an infinity
// makes the block's scale one, and its values NaN.
template <typename T, int V> __device__ __forceinline__ float encode(const Values<T, V>& x, const float2 (&f)[V / 2], Values<int8_t, V>& u) {
  uint32_t m = top_bits(x);
#pragma unroll
  for (int o = kPackBlock / V / 2; o; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  const float top = __uint_as_float(m);
  const float scale = top * (1.0f / 127.0f);
  uint32_t q[V];
  if (top >= 1e-20f && top <= 3.0e38f) {
    // Quotients by the reciprocal: product, remainder, and the remainder's share give the quotient's rounding where
    // nothing underflows (Markstein).
    const float2 inverse = pair(__frcp_rn(scale)), minus = pair(-scale);
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      const float2 t = mul2(f[i], inverse), v = add2(fma2(fma2(t, minus, f[i]), inverse, t), pair(kWhole));
      q[2 * i] = __float_as_uint(v.x);
      q[2 * i + 1] = __float_as_uint(v.y);
    }
  } else {                                          // tiny ones by division; none of zeros, infinities and NaN
#pragma unroll
    for (int i = 0; i < V; ++i)
      q[i] = scale > 0.f && scale <= 3.0e38f ? (uint32_t)__float2int_rn(fmaxf(-127.f, fminf(127.f, __fdiv_rn(i & 1 ? f[i / 2].y : f[i / 2].x, scale)))) : 0;
  }
  uint32_t* w = reinterpret_cast<uint32_t*>(&u);
#pragma unroll
  for (int i = 0; i < V; i += 4)
    w[i >> 2] = __byte_perm(__byte_perm(q[i], q[i + 1], 0x0040), __byte_perm(q[i + 2], q[i + 3], 0x0040), 0x5410);
  return scale;
}

__device__ __forceinline__ float reciprocal(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <typename T> __device__ __forceinline__ float2 sigmoid(float2 z) {
  if constexpr (sizeof(T) == 4) {
    return make_float2(1.0f / (1.0f + expf(-z.x)), 1.0f / (1.0f + expf(-z.y)));
  } else {                                          // a few ulp of fp32, far below a 16-bit result's half step
    float2 e = mul2(z, pair(-kLog2e));
    e = add2(make_float2(ex2(e.x), ex2(e.y)), pair(1.0f));
    return make_float2(reciprocal(e.x), reciprocal(e.y));
  }
}

// A thread's V channels: weights and bias.
template <typename WT, int V>
struct Taps {
  float2 w[kTaps][V / 2], b[V / 2];
  __device__ Taps(const void* weights, const void* biases, int taps, int c, int n) {
    const WT* weight = reinterpret_cast<const WT*>(weights) + (long long)c * taps;
    if (taps == kTaps && n == V && ((uintptr_t)weight & (4 * sizeof(WT) - 1)) == 0) {
#pragma unroll
      for (int i = 0; i < V; i += 2) {
        float f[2][kTaps];
        load_values<WT, kTaps>(weight + i * kTaps, true, kTaps, f[0]);
        load_values<WT, kTaps>(weight + (i + 1) * kTaps, true, kTaps, f[1]);
#pragma unroll
        for (int k = 0; k < kTaps; ++k) w[k][i / 2] = make_float2(f[0][k], f[1][k]);
      }
    } else {
      auto at = [&](int i, int j) { return i < n && j >= 0 ? to_f32(weight[i * taps + j]) : 0.f; };
#pragma unroll
      for (int i = 0; i < V; i += 2)
#pragma unroll
        for (int k = 0; k < kTaps; ++k) {
          const int j = k - (kTaps - taps);
          w[k][i / 2] = make_float2(at(i, j), at(i + 1, j));
        }
    }
    const WT* bias = reinterpret_cast<const WT*>(biases) + c;
    if (biases) {
      load_pairs<WT, V>(bias, n == V && ((uintptr_t)bias & (V * sizeof(WT) - 1)) == 0, n, b);
    } else {
#pragma unroll
      for (int i = 0; i < V / 2; ++i) b[i] = pair(0.f);
    }
  }
};

__device__ __forceinline__ int tokens_of(const ConvParams& P, int b) {
  return P.lengths ? max(0, min(P.length, P.lengths[b])) : P.length;
}

// A thread's inputs along the tokens, as memory has them: of x, or of codes and scales.  VEC: its channels are all there
// and lie at multiples of their size.  Loads come in two steps, so that those of later tokens are under way while
// earlier ones are worked on.
template <typename T, bool CODES, bool VEC, int V> struct Inputs {
  using Raw = Values<typename std::conditional<CODES, int8_t, T>::type, V>;
  const T* x;
  const int8_t* codes;
  const float* scales;
  long long step, scale_step;
  int n;
  __device__ Inputs(const ConvParams& P, int b, int c, int n_) : x(nullptr), codes(nullptr), scales(nullptr), n(n_) {
    if constexpr (CODES) {
      step = P.channels;
      scale_step = (P.channels + kPackBlock - 1) / kPackBlock;
      codes = P.codes + (long long)b * P.length * step + c;
      scales = P.scales + (long long)b * P.length * scale_step + c / kPackBlock;
    } else {
      step = P.x_st;
      scale_step = 0;
      x = reinterpret_cast<const T*>(P.x) + b * P.x_sb + c;
    }
  }
  __device__ __forceinline__ Raw load(int t, bool take, float& scale) const {
    Raw u;
    if constexpr (CODES) {
      scale = take ? scales[t * scale_step] : 0.f;
      if (take) u = raw_values<int8_t, V>(codes + t * step, VEC, n);
      else u = Raw{};
    } else {
      if (take) u = raw_values<T, V>(x + t * step, VEC, n);
      else u = no_values<T, V>();
    }
    return u;
  }
  // U tokens from t on, those from `end` on as zero.
  template <int U> __device__ __forceinline__ void load_batch(int t, int end, bool take, Raw (&u)[U], float (&scale)[U]) const {
    if constexpr (CODES) {
      const int8_t* p = codes + t * step;
      const float* s = scales + t * scale_step;
      if (take && t + U <= end) {
#pragma unroll
        for (int j = 0; j < U; ++j, p += step, s += scale_step) { u[j] = raw_values<int8_t, V>(p, VEC, n); scale[j] = *s; }
      } else {
#pragma unroll
        for (int j = 0; j < U; ++j, p += step, s += scale_step) {
          const bool in = take && t + j < end;
          if (in) u[j] = raw_values<int8_t, V>(p, VEC, n);
          else u[j] = Raw{};
          scale[j] = in ? *s : 0.f;
        }
      }
    } else {
      const T* p = x + t * step;
      if (take && t + U <= end) {
#pragma unroll
        for (int j = 0; j < U; ++j, p += step) { u[j] = raw_values<T, V>(p, VEC, n); scale[j] = 0.f; }
      } else {
#pragma unroll
        for (int j = 0; j < U; ++j, p += step) {
          scale[j] = 0.f;
          if (take && t + j < end) u[j] = raw_values<T, V>(p, VEC, n);
          else u[j] = no_values<T, V>();
        }
      }
    }
  }
  static __device__ __forceinline__ void get(const Raw& u, float scale, float2 (&f)[V / 2]) {
    if constexpr (CODES) {
      decode<V>(u, scale, f);
    } else {
#pragma unroll
      for (int i = 0; i < V / 2; ++i) f[i] = two<T, V>(u, i);
    }
  }
  // The input at any token, the state's before the first.
  __device__ void at(const ConvParams& P, int b, int t, int c, float2 (&f)[V / 2]) const {
    if (t >= 0) {
      float scale = 0.f;
      const Raw u = load(t, true, scale);
      get(u, scale, f);
    } else if (P.state_in && t >= 1 - P.taps) {
      const long long at = ((long long)b * (P.taps - 1) + t + P.taps - 1) * P.channels + c;
      load_pairs<T, V>(reinterpret_cast<const T*>(P.state_in) + at, false, n, f);
    } else {
#pragma unroll
      for (int i = 0; i < V / 2; ++i) f[i] = pair(0.f);
    }
  }
};

// z of a token's channels 2i and 2i + 1, whose last four inputs are x0..x3, oldest first.  Taps that are not there are
// passed over, not multiplied by zero: their inputs may be infinite.
template <typename WT, int V>
__device__ __forceinline__ float2 conv_at(const Taps<WT, V>& W, const int taps, int i, float2 x0, float2 x1, float2 x2, float2 x3) {
  float2 z = W.b[i];
  if (taps > 3) z = fma2(W.w[0][i], x0, z);
  if (taps > 2) z = fma2(W.w[1][i], x1, z);
  return fma2(W.w[3][i], x3, fma2(W.w[2][i], x2, z));
}

// KEEP: the input is kept in 8 bits besides.  FAST: four taps, silu and whole aligned pieces, as mixers have them; without
// them a third of the instructions would be the questions.  Bound by the latency of loads: the next four tokens' are under
// way while four are worked on, 32 KB an SM.  4 x 2,048 tokens of 10,240 channels in bf16: 68 us, 4.9 TB/s of input and
// output (fp32 120 us, 5.6 TB/s); keeping the input in 8 bits besides 105 us, 4.0 TB/s, for the rows' maxima.
template <typename T, typename WT, bool KEEP, bool FAST>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 4 || KEEP ? 5 : 8) conv_kernel(const ConvParams P, int strip) {
  constexpr int V = kWide, U = 4;                                      // U: tokens whose loads are in flight together
  constexpr bool VEC = FAST;
  using In = Inputs<T, false, VEC, V>;
  const int taps = FAST ? kTaps : P.taps;
  const bool silu = FAST || P.silu;
  const int c = (blockIdx.y * kThreads + threadIdx.x) * V, b = blockIdx.z;
  const int n = min(V, P.channels - c);                                // may be negative: shuffles need every lane
  if (!KEEP && n <= 0) return;
  const int len = tokens_of(P, b), t0 = blockIdx.x * strip, t1 = min(P.length, t0 + strip), end = min(t1, len);
  const In in(P, b, n > 0 ? c : 0, n);
  T* y = reinterpret_cast<T*>(P.y) + b * P.y_sb + (long long)t0 * P.y_st + c;
  const int blocks = (P.channels + kPackBlock - 1) / kPackBlock;
  int8_t* codes = KEEP ? P.codes + ((long long)b * P.length + t0) * P.channels + c : nullptr;
  float* scales = KEEP ? P.scales + ((long long)b * P.length + t0) * blocks + c / kPackBlock : nullptr;
  if (n > 0 && blockIdx.x == 0 && P.state_out) {                       // the last inputs
    for (int j = 0; j < taps - 1; ++j) {
      float2 f[V / 2];
      in.at(P, b, len - (taps - 1) + j, c, f);
      store_pairs<T, V>(reinterpret_cast<T*>(P.state_out) + ((long long)b * (taps - 1) + j) * P.channels + c, false, n, f);
    }
  }
  if (t0 < end) {
    float2 x[kTaps - 1][V / 2];
    float scale[U];
    typename In::Raw now[U];
    in.template load_batch<U>(t0, end, n > 0, now, scale);
    const Taps<WT, V> W(P.weight, P.bias, taps, n > 0 ? c : 0, n);
#pragma unroll
    for (int k = 0; k < kTaps - 1; ++k)
      if (n > 0) in.at(P, b, t0 - (kTaps - 1) + k, c, x[k]);
    auto token = [&](const typename In::Raw& raw, float s, bool there) {
      float2 out[V / 2], f[V / 2];
      In::get(raw, s, f);
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        const float2 z = conv_at<WT, V>(W, taps, i, x[0][i], x[1][i], x[2][i], f[i]);
        out[i] = silu ? mul2(z, sigmoid<T>(z)) : z;
        x[0][i] = x[1][i]; x[1][i] = x[2][i]; x[2][i] = f[i];
      }
      if (there) store_pairs<T, V>(y, VEC, n, out);
      y += P.y_st;
      if constexpr (KEEP) {
        Values<int8_t, V> q;
        const float top = encode<T, V>(raw, f, q);
        if (there) {
          store_codes<V>(codes, VEC, n, q);
          if ((threadIdx.x & 31) == 0) *scales = top;
        }
        codes += P.channels;
        scales += blocks;
      }
    };
    for (int t = t0; t < end; t += U) {
      typename In::Raw next[U];
      float later[U];
      in.template load_batch<U>(t + U, end, n > 0, next, later);
      if (t + U <= end) {                                              // the same for the whole CTA: codes take shuffles
#pragma unroll
        for (int j = 0; j < U; ++j) token(now[j], scale[j], n > 0);
      } else {
#pragma unroll
        for (int j = 0; j < U; ++j) token(now[j], scale[j], n > 0 && t + j < end);
      }
#pragma unroll
      for (int j = 0; j < U; ++j) {
        now[j] = next[j];
        scale[j] = later[j];
      }
    }
  }
  if (n <= 0) return;
  const float2 zero[V / 2] = {};
  y = reinterpret_cast<T*>(P.y) + b * P.y_sb + c;
  for (int t = max(t0, len); t < t1; ++t) {
    store_pairs<T, V>(y + t * P.y_st, VEC, n, zero);
    if constexpr (KEEP) {
      const long long row = (long long)b * P.length + t;
      store_codes<V>(P.codes + row * P.channels + c, VEC, n, Values<int8_t, V>{});
      if ((threadIdx.x & 31) == 0) P.scales[row * blocks + c / kPackBlock] = 0.f;
    }
  }
}

// Copies to shared memory that a thread makes for itself: it alone waits for them and reads them.  `take`: else zeros.
template <int BYTES> __device__ __forceinline__ void copy_async(uint32_t dst, const void* src, bool take) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" :: "r"(dst), "l"(src), "n"(BYTES), "r"(take ? BYTES : 0) : "memory");
}
__device__ __forceinline__ void read_own(uint32_t a, uint2& v) {
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory");
}
__device__ __forceinline__ void read_own(uint32_t a, uint4& v) {
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
}

// A strip's gradients: dz_t = dy_t y'(z_t), dx_t = sum_k w_k dz_{t + taps-1 - k}, and the strip's sums of dz_t x_{t - (taps-1) + k}
// and dz_t.  The walk goes three tokens past the strip, whose dz its last inputs need.  Bound by registers (sums, taps and what
// is under way) and with them by the loads in flight.  RING: those of 16-bit tensors go to shared memory, twelve tokens of
// a thread, which leaves 96 registers and five CTAs an SM; 4 x 2,048 tokens of 10,240 channels in bf16 take 105 us, 4.8 TB/s, and
// conv_weights_kernel 6 us more.  In registers (odd forms, codes) eight tokens and four CTAs: 119 us, from codes too; codes in the ring, by
// copies of four bytes, take 167.  An fp32 dy, a scan's, goes through the ring also beside codes: 2 x 2,048 tokens 69 us, with a bf16 dy 64.  fp32 has three CTAs (188 us; four spill, 215).  Two channels a thread have twice the warps, but in loads of four bytes, and are slower by
// a third.
constexpr int kStages = 3, kRingCtas = 5;
template <typename T, typename WT, typename DY, bool CODES, bool FAST>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 4 ? 3 : FAST && !CODES ? kRingCtas : 4) conv_grad_kernel(const ConvParams P, int strip) {
  constexpr int V = kWide, U = 4;
  // what goes through the ring: x of 16 bits, and with it dy; an fp32 dy also beside codes
  constexpr bool VEC = FAST, RING_X = FAST && !CODES && sizeof(T) == 2, RING = RING_X || (FAST && sizeof(DY) > sizeof(T));
  constexpr uint32_t kXBytes = RING_X ? kThreads * 8 : 0, kToken = kXBytes + kThreads * V * (uint32_t)sizeof(DY), kRing = RING ? kStages * U * kToken : 16;
  __shared__ __align__(16) unsigned char ring[kRing];
  using In = Inputs<T, CODES, VEC, V>;
  const int taps = FAST ? kTaps : P.taps;
  const bool silu = FAST || P.silu;
  const int c = (blockIdx.y * kThreads + threadIdx.x) * V, b = blockIdx.z;
  const int n = min(V, P.channels - c);
  if (n <= 0) return;
  const int len = tokens_of(P, b), t0 = blockIdx.x * strip, t1 = min(P.length, t0 + strip), back = taps - 1;
  const In in(P, b, c, n);
  const DY* dy = reinterpret_cast<const DY*>(P.dy) + b * P.dy_sb + c;
  T* dx = reinterpret_cast<T*>(P.dx) + (long long)b * P.length * P.channels + c;
  float2 dw[kTaps][V / 2] = {}, db[V / 2] = {};
  if (t0 < len || t0 == 0) {
    const int stop = t1 + kTaps - 1, end = min(stop, len), own = min(t1, len), lowest = t0 == 0 ? -back : t0;
    float2 x[kTaps - 1][V / 2], dz[kTaps - 1][V / 2] = {};
    float scale[RING_X ? 1 : U];
    typename In::Raw now[RING_X ? 1 : U];
    Values<DY, V> up[RING ? 1 : U];
    auto load_up = [&](int t, Values<DY, V>(&u)[U]) {
      const DY* p = dy + t * P.dy_st;
      if (t + U <= end) {
#pragma unroll
        for (int j = 0; j < U; ++j, p += P.dy_st) u[j] = raw_values<DY, V>(p, VEC, n);
      } else {
#pragma unroll
        for (int j = 0; j < U; ++j, p += P.dy_st) {
          if (t + j < end) u[j] = raw_values<DY, V>(p, VEC, n);
          else u[j] = no_values<DY, V>();
        }
      }
    };
    // RING: the next stages of U tokens each, a token's x before its dy
    const uint32_t slots = (uint32_t)__cvta_generic_to_shared(ring), x_slot = slots + threadIdx.x * 8,
                   dy_slot = slots + kXBytes + threadIdx.x * (V * (uint32_t)sizeof(DY));
    uint32_t put_at = 0, get_at = 0;
    const T* x_next = in.x + t0 * in.step;
    const DY* dy_next = dy + t0 * P.dy_st;
    auto stage = [&](int t) {
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const uint32_t at = put_at + j * kToken;
        const bool there = t + j < end;
        if constexpr (RING_X) {
          copy_async<8>(x_slot + at, there ? x_next : in.x, there);
          x_next += in.step;
        }
        copy_async<V * (int)sizeof(DY)>(dy_slot + at, there ? dy_next : dy, there);
        dy_next += P.dy_st;
      }
      put_at = (put_at + U * kToken) % (kStages * U * kToken);
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    if constexpr (RING) {
#pragma unroll
      for (int k = 0; k < kStages - 1; ++k) stage(t0 + k * U);
    } else {
      load_up(t0, up);
    }
    if constexpr (!RING_X) in.template load_batch<U>(t0, end, true, now, scale);
    const Taps<WT, V> W(P.weight, P.bias, taps, c, n);
#pragma unroll
    for (int k = 0; k < kTaps - 1; ++k) in.at(P, b, t0 - (kTaps - 1) + k, c, x[k]);
    T* put = dx + (long long)(t0 - (kTaps - 1)) * P.channels;          // of the token whose input's gradient is whole next
    // inner: the token and the one whose gradient becomes whole are both this strip's
    auto token = [&](const typename In::Raw& raw, float s_in, const Values<DY, V>& raw_up, int at, auto inner) {
      constexpr bool INNER = decltype(inner)::value;
      const int to = at - (kTaps - 1);
      const bool mine = INNER || at < own;
      float2 f[V / 2], out[V / 2];
      In::get(raw, s_in, f);
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        float2 d = two<DY, V>(raw_up, i);
        if (silu) {
          const float2 z = conv_at<WT, V>(W, taps, i, x[0][i], x[1][i], x[2][i], f[i]);
          const float2 s = sigmoid<T>(z);
          d = mul2(d, fma2(s, mul2(z, fma2(s, pair(-1.0f), pair(1.0f))), s));
        }
        if (!INNER && at >= end) d = pair(0.f);                        // z of what is not there may be anything
        if (mine) {
          db[i] = add2(db[i], d);
          if (taps > 3) dw[0][i] = fma2(d, x[0][i], dw[0][i]);
          if (taps > 2) dw[1][i] = fma2(d, x[1][i], dw[1][i]);
          dw[2][i] = fma2(d, x[2][i], dw[2][i]);
          dw[3][i] = fma2(d, f[i], dw[3][i]);
        }
        x[0][i] = x[1][i]; x[1][i] = x[2][i]; x[2][i] = f[i];
        // dz[0..2] and d are those of `to` .. `to` + 3
        float2 g = fma2(W.w[2][i], dz[1][i], mul2(W.w[3][i], dz[0][i]));
        if (taps > 2) g = fma2(W.w[1][i], dz[2][i], g);
        if (taps > 3) g = fma2(W.w[0][i], d, g);
        dz[0][i] = dz[1][i]; dz[1][i] = dz[2][i]; dz[2][i] = d;
        out[i] = g;
      }
      T* here = put;
      put += P.channels;
      if (INNER) {
        store_pairs<T, V>(here, VEC, n, out);
        return;
      }
      if (to >= t1 || to < lowest) return;
      if (P.dstate_out && to >= len - back && to < len) {
        float2 late[V / 2];
        const long long at_state = ((long long)b * back + to - (len - back)) * P.channels + c;
        load_pairs<T, V>(reinterpret_cast<const T*>(P.dstate_out) + at_state, false, n, late);
#pragma unroll
        for (int i = 0; i < V / 2; ++i) out[i] = add2(out[i], late[i]);
      }
      if (to >= 0) {
        if (to < len) store_pairs<T, V>(here, VEC, n, out);
      } else if (P.dstate_in) {
        store_pairs<T, V>(reinterpret_cast<T*>(P.dstate_in) + ((long long)b * back + to + back) * P.channels + c, false, n, out);
      }
    };
    const int calm = P.dstate_out ? min(own, len - back) : own;        // below it no gradient of the last inputs comes in
    auto tokens = [&](int t, auto inner) {
#pragma unroll
      for (int j = 0; j < U; ++j) {
        if constexpr (RING) {
          const uint32_t at = get_at + j * kToken;
          Values<DY, V> raw_up;
          read_own(dy_slot + at, raw_up.q);
          if constexpr (RING_X) {
            typename In::Raw raw;
            read_own(x_slot + at, raw.q);
            token(raw, 0.f, raw_up, t + j, inner);
          } else {
            token(now[j], scale[j], raw_up, t + j, inner);
          }
        } else {
          token(now[j], scale[j], up[j], t + j, inner);
        }
      }
    };
    for (int t = t0; t < stop; t += U) {
      typename In::Raw next[RING_X ? 1 : U];
      Values<DY, V> up_next[RING ? 1 : U];
      float later[RING_X ? 1 : U];
      if constexpr (RING) stage(t + (kStages - 1) * U);                // its place was read a turn ago
      if constexpr (!RING_X) in.template load_batch<U>(t + U, end, true, next, later);
      if constexpr (RING) asm volatile("cp.async.wait_group %0;" :: "n"(kStages - 1) : "memory");
      else load_up(t + U, up_next);
      if (t >= t0 + U && t + U <= calm) tokens(t, std::true_type{});
      else tokens(t, std::false_type{});
      if constexpr (RING) get_at = (get_at + U * kToken) % (kStages * U * kToken);
#pragma unroll
      for (int j = 0; j < U; ++j) {
        if constexpr (!RING_X) {
          now[j] = next[j];
          scale[j] = later[j];
        }
        if constexpr (!RING) up[j] = up_next[j];
      }
    }
    if constexpr (RING) asm volatile("cp.async.wait_group 0;" ::: "memory");
  }
  const float2 zero[V / 2] = {};
  for (int t = max(t0, len); t < t1; ++t) store_pairs<T, V>(dx + (long long)t * P.channels, VEC, n, zero);
  if (P.dweight || P.dbias) {
    float* part = P.workspace + ((long long)b * gridDim.x + blockIdx.x) * (kTaps + 1) * P.channels + c;
#pragma unroll
    for (int k = 0; k <= kTaps; ++k) store_pairs<float, V>(part + (long long)k * P.channels, VEC, n, k < kTaps ? dw[k] : db);
  }
}

// ---------------------------------------------------------------- tiles for a scan
// Four channels c .. c + 3 of a token, `n` of them there; codes may lie on both sides of a block's border.
template <typename T, bool CODES>
__device__ __forceinline__ void four_channels(const ConvParams& P, int b, int t, int c, int n, float2 (&f)[2]) {
  if (t < 0) {
    if (P.state_in && t >= 1 - P.taps) {
      const long long at = ((long long)b * (P.taps - 1) + t + P.taps - 1) * P.channels + c;
      load_pairs<T, 4>(reinterpret_cast<const T*>(P.state_in) + at, false, n, f);
    } else {
      f[0] = f[1] = pair(0.f);
    }
  } else if constexpr (CODES) {
    const long long row = (long long)b * P.length + t;
    const int8_t* q = P.codes + row * P.channels + c;
    const float* s = P.scales + row * ((P.channels + kPackBlock - 1) / kPackBlock);
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < n ? (float)q[i] * s[(c + i) / kPackBlock] : 0.f;
    f[0] = make_float2(v[0], v[1]);
    f[1] = make_float2(v[2], v[3]);
  } else {
    load_pairs<T, 4>(reinterpret_cast<const T*>(P.x) + b * P.x_sb + t * P.x_st + c, false, n, f);
  }
}

// One CTA: a chunk's tile of B or C (128 channels of a group), or two of x (64 channels of a head each).  A thread has four
// channels of eight neighbouring tokens in registers, all loads before the first use; a tile's largest value gives its
// scale.  VEC: four taps, and four channels are one aligned load.  Bound by the two exponential-unit instructions of a
// sigmoid and by the loads' latency before a CTA's first use: 2 x 2,048 tokens of 10,240 channels 54 us, from codes 60 us.
constexpr int kTileThreads = 512;
template <typename T, typename WT, bool CODES, bool VEC>
__global__ void __launch_bounds__(kTileThreads, 2) conv_tiles_kernel(const ConvParams P, const ConvTiles A) {
  constexpr int TOKENS = 8;
  using In = Inputs<T, CODES, true, 4>;
  __shared__ uint32_t tops[kTileThreads / 32];
  const int chunk = blockIdx.x, b = blockIdx.z;
  const int rows = min(kScanChunk, tokens_of(P, b) - chunk * kScanChunk);
  if (rows <= 0) return;                                               // not read
  const long long bc = (long long)b * A.chunks + chunk;
  const bool group = (int)blockIdx.y < 2 * A.groups;
  const int half = threadIdx.x >> 8;
  int at, r0, c0, cols;
  uint16_t* out = nullptr;
  float* back = nullptr;
  if (group) {
    const int g = blockIdx.y >> 1, second = blockIdx.y & 1;
    at = threadIdx.x & 31;
    r0 = threadIdx.x / 32 * TOKENS;
    c0 = A.heads * A.dim + (second ? A.groups * 128 : 0) + g * 128;
    cols = 128;
    out = (second ? A.c : A.b) + (bc * A.groups + g) * (kScanChunk * 128);
    back = (second ? A.cback : A.bback) + bc * A.groups + g;
  } else {
    const int ptiles = A.units / A.heads, u = 2 * (blockIdx.y - 2 * A.groups) + half, p0 = (u % ptiles) * kScanTile;
    at = threadIdx.x & 15;
    r0 = (threadIdx.x & 255) / 16 * TOKENS;
    c0 = u / ptiles * A.dim + p0;
    cols = u < A.units ? min(kScanTile, A.dim - p0) : 0;
    if (u < A.units) {
      out = A.x + (bc * A.units + u) * (kScanChunk * kScanTile);
      back = A.xback + bc * A.units + u;
    }
  }
  const int n = max(0, min(4, cols - at * 4)), c = n > 0 ? c0 + at * 4 : 0;
  const int t0 = chunk * kScanChunk + r0, end = n > 0 ? chunk * kScanChunk + rows : 0;
  float2 z[TOKENS][2], x[3][2];
  typename In::Raw raw[VEC ? TOKENS + 3 : 1];
  float scale[VEC ? TOKENS + 3 : 1];
  const In in(P, b, c, 4);
  if constexpr (VEC) {
    if (t0 > 0) {
      in.template load_batch<TOKENS + 3>(t0 - 3, end, n > 0, raw, scale);
    } else {
#pragma unroll
      for (int j = 0; j < TOKENS + 3; ++j) raw[j] = in.load(j - 3, j >= 3 && j - 3 < end, scale[j]);
    }
  }
  const int taps = VEC ? kTaps : P.taps;
  const Taps<WT, 4> W(P.weight, P.bias, taps, c, n);
  if (VEC && t0 > 0) {
#pragma unroll
    for (int k = 0; k < 3; ++k) In::get(raw[k], scale[k], x[k]);
  } else {
#pragma unroll
    for (int k = 0; k < 3; ++k) four_channels<T, CODES>(P, b, t0 < end ? t0 - 3 + k : -kTaps, c, n, x[k]);
  }
#pragma unroll
  for (int j = 0; j < TOKENS; ++j) {
    float2 f[2];
    if constexpr (VEC) In::get(raw[j + 3], scale[j + 3], f);
    else four_channels<T, CODES>(P, b, t0 + j < end ? t0 + j : -kTaps, c, n, f);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float2 v = conv_at<WT, 4>(W, taps, i, x[0][i], x[1][i], x[2][i], f[i]);
      z[j][i] = mul2(v, sigmoid<T>(v));
      x[0][i] = x[1][i]; x[1][i] = x[2][i]; x[2][i] = f[i];
    }
  }
  if (t0 + TOKENS > end || n < 4) {
#pragma unroll
    for (int j = 0; j < TOKENS; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (t0 + j >= end || 2 * i >= n) z[j][i].x = 0.f;
        if (t0 + j >= end || 2 * i + 1 >= n) z[j][i].y = 0.f;
      }
  }
  float top = 0.f;
#pragma unroll
  for (int j = 0; j < TOKENS; ++j)
    top = fmaxf(top, fmaxf(fmaxf(fabsf(z[j][0].x), fabsf(z[j][0].y)), fmaxf(fabsf(z[j][1].x), fabsf(z[j][1].y))));
  uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(top));
  if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = bits;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 8; ++k) bits = max(bits, group ? max(tops[k], tops[8 + k]) : tops[half * 8 + k]);
  if (!out) return;
  int e = (int)(bits >> 23) - 140;                                     // to [2^13, 2^14)
  e = bits ? max(-110, e) : 0;
  const float there = __uint_as_float((uint32_t)(127 - e) << 23);
  // an infinity leaves a tile's other numbers no scale: all that is made of them is NaN
  if (r0 + at == 0) *back = __uint_as_float(bits >= 0x7f800000u ? 0x7fffffffu : (uint32_t)(127 + e) << 23);
  const int piece = at / 2;
  char* p = reinterpret_cast<char*>(out) + (piece >> 3) * 16384 + r0 * 128 + (at & 1) * 8;
#pragma unroll
  for (int j = 0; j < TOKENS; ++j) {                                   // r0 is a multiple of eight
    const float2 lo = mul2(z[j][0], pair(there)), hi = mul2(z[j][1], pair(there));
    *reinterpret_cast<uint2*>(p + j * 128 + (((piece & 7) ^ (j & 7)) << 4)) = make_uint2(pack2<__half>(lo.x, lo.y), pack2<__half>(hi.x, hi.y));
  }
}
template <typename T, typename WT, bool CODES, bool VEC> void conv_tiles(const ConvParams& P, const ConvTiles& A, cudaStream_t st) {
  conv_tiles_kernel<T, WT, CODES, VEC><<<dim3(A.chunks, 2 * A.groups + (A.units + 1) / 2, P.batch), kTileThreads, 0, st>>>(P, A);
}
// The last inputs of a sequence.
template <typename T, bool CODES>
__global__ void __launch_bounds__(kThreads) conv_last_kernel(const ConvParams P) {
  const int c = (blockIdx.x * kThreads + threadIdx.x) * 4, b = blockIdx.y, n = min(4, P.channels - c), back = P.taps - 1;
  if (n <= 0) return;
  const int len = tokens_of(P, b);
  for (int j = 0; j < back; ++j) {
    float2 f[2];
    four_channels<T, CODES>(P, b, len - back + j, c, n, f);
    store_pairs<T, 4>(reinterpret_cast<T*>(P.state_out) + ((long long)b * back + j) * P.channels + c, false, n, f);
  }
}

// The strips' sums for a channel's tap or bias, in order: eight threads share a channel's strips.  6 us for 64 strips of
// 10,240 channels.
template <typename WT>
__global__ void __launch_bounds__(256) conv_weights_kernel(const ConvParams P, int strips) {
  __shared__ float sums[8][33];
  const int lane = threadIdx.x & 31, sub = threadIdx.x >> 5, k = blockIdx.y;
  const int c = blockIdx.x * 32 + lane;
  if (k < kTaps - P.taps) return;
  float v = 0.f;
  if (c < P.channels)
    for (int s = sub; s < strips; s += 8) v += P.workspace[((long long)s * (kTaps + 1) + k) * P.channels + c];
  sums[sub][lane] = v;
  __syncthreads();
  if (sub || c >= P.channels) return;
#pragma unroll
  for (int i = 1; i < 8; ++i) v += sums[i][lane];
  if (k == kTaps) {
    if (P.dbias) reinterpret_cast<WT*>(P.dbias)[c] = from_f32<WT>(v);
  } else if (P.dweight) {
    reinterpret_cast<WT*>(P.dweight)[(long long)c * P.taps + k - (kTaps - P.taps)] = from_f32<WT>(v);
  }
}

// One token: a thread owns four channels, shifts their state and puts the token at its end.  64 rows of 10,240 channels: 6 us.
template <typename T, typename WT, typename YT>
__global__ void __launch_bounds__(kThreads) conv_step_kernel(const ConvStepParams P, int vec) {
  constexpr int V = kWide;
  const int c = (blockIdx.x * kThreads + threadIdx.x) * V, b = blockIdx.y;
  const int n = min(V, P.channels - c);
  launch_dependents();
  if (n <= 0) return;
  const bool v = vec && n == V;
  T* state = reinterpret_cast<T*>(P.state) + (long long)b * (P.taps - 1) * P.channels + c;
  float2 x[kTaps][V / 2] = {};
  load_pairs<T, V>(reinterpret_cast<const T*>(P.x) + b * P.x_sb + c, v, n, x[3]);
#pragma unroll
  for (int k = 0; k < kTaps - 1; ++k) {
    const int j = k - (kTaps - P.taps);
    if (j >= 0) load_pairs<T, V>(state + (long long)j * P.channels, v, n, x[k]);
  }
  const Taps<WT, V> W(P.weight, P.bias, P.taps, c, n);
  float2 out[V / 2];
#pragma unroll
  for (int i = 0; i < V / 2; ++i) {
    const float2 z = conv_at<WT, V>(W, P.taps, i, x[0][i], x[1][i], x[2][i], x[3][i]);
    out[i] = P.silu ? mul2(z, sigmoid<T>(z)) : z;
  }
  YT* y = reinterpret_cast<YT*>(P.y) + (long long)b * P.channels + c;
  store_pairs<YT, V>(y, v, n, out);
#pragma unroll
  for (int k = 0; k < kTaps - 1; ++k) {
    const int j = k - (kTaps - P.taps);
    if (j >= 0) store_pairs<T, V>(state + (long long)j * P.channels, v, n, x[k + 1]);
  }
}

// Rows in 8 bits: a thread has 16 bytes of the input, kRows rows at a time.  Bound by instructions (15 a value: conversion,
// maximum, quotient, code).  8,192 x 10,240 in bf16: 53 us, 4.8 TB/s.
constexpr int kRows = 4;
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads, 10) pack_kernel(const PackParams P) {
  constexpr int V = kUnit<T>;
  const int c = (blockIdx.x * kThreads + threadIdx.x) * V;
  const int n = min(V, P.width - c), blocks = (P.width + kPackBlock - 1) / kPackBlock;
  for (long long r0 = (long long)blockIdx.y * kRows; r0 < P.rows; r0 += (long long)gridDim.y * kRows) {
    Values<T, V> x[kRows];
#pragma unroll
    for (int j = 0; j < kRows; ++j)
      x[j] = n > 0 && r0 + j < P.rows ? raw_values<T, V>(reinterpret_cast<const T*>(P.x) + (r0 + j) * P.x_stride + c, VEC, n)
                                      : no_values<T, V>();
#pragma unroll
    for (int j = 0; j < kRows; ++j) {
      float2 f[V / 2];
#pragma unroll
      for (int i = 0; i < V / 2; ++i) f[i] = two<T, V>(x[j], i);
      Values<int8_t, V> q;
      const float scale = encode<T, V>(x[j], f, q);
      if (n > 0 && r0 + j < P.rows) {
        store_codes<V>(P.codes + (r0 + j) * P.width + c, VEC, n, q);
        if ((c & (kPackBlock - 1)) == 0) P.scales[(r0 + j) * blocks + c / kPackBlock] = scale;
      }
    }
  }
}
// Back: a thread has sixteen codes.  8,192 x 10,240 to bf16: 50 us, 5.1 TB/s.
constexpr int kCodes = 16;
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads, 10) unpack_kernel(const PackParams P) {
  constexpr int V = kUnit<T>;
  const int c = (blockIdx.x * kThreads + threadIdx.x) * kCodes;
  const int n = min(kCodes, P.width - c), blocks = (P.width + kPackBlock - 1) / kPackBlock;
  if (n <= 0) return;
  for (long long r0 = (long long)blockIdx.y * kRows; r0 < P.rows; r0 += (long long)gridDim.y * kRows) {
    float scale[kRows];
    Values<int8_t, kCodes> q[kRows];
#pragma unroll
    for (int j = 0; j < kRows; ++j) {
      const bool in = r0 + j < P.rows;
      scale[j] = in ? P.scales[(r0 + j) * blocks + c / kPackBlock] : 0.f;
      if (in) q[j] = raw_values<int8_t, kCodes>(P.codes + (r0 + j) * P.width + c, VEC, n);
    }
#pragma unroll
    for (int j = 0; j < kRows; ++j)
      if (r0 + j < P.rows) {
        float2 f[kCodes / 2];
        decode<kCodes>(q[j], scale[j], f);
        T* out = reinterpret_cast<T*>(P.y) + (r0 + j) * P.width + c;
#pragma unroll
        for (int i = 0; i < kCodes; i += V) store_pairs<T, V>(out + i, VEC, n - i, f + i / 2);
      }
  }
}

int unit_of(int type) { return type == 2 ? 4 : 8; }
// Whether `wide` neighbours starting at multiples of `wide` can be moved at once.
bool whole(const void* p, int type, int wide, long long a, long long b = 0) {
  return ((uintptr_t)p & (wide * (type == 2 ? 4 : 2) - 1)) == 0 && (a | b) % wide == 0;
}

// Tokens of a strip: long ones read fewer edges twice, short ones make more CTAs.
int strip_of(int batch, int length, int channels, int least, int most) {
  const long long wide = (long long)batch * ((channels + kWide - 1) / kWide);
  int s = most;
  while (s > least && wide * ((length + s - 1) / s) < 148 * 1024) s /= 2;
  return s;
}
constexpr int kLeast = 16, kMost = 128;

template <typename F> int by_type(int type, int weight_type, F f) {
  if (type == 2) return f(float{}, float{});
  if (type == 1) return weight_type == 2 ? f(__nv_bfloat16{}, float{}) : f(__nv_bfloat16{}, __nv_bfloat16{});
  return weight_type == 2 ? f(__half{}, float{}) : f(__half{}, __half{});
}

}  // namespace

int launch_conv_tiles(const ConvParams& P, const ConvTiles& A, cudaStream_t st) {
  return by_type(P.type, P.weight_type, [&](auto t, auto w) {
    using T = decltype(t);
    using WT = decltype(w);
    if constexpr (sizeof(T) == 2) {
      // every head's channels begin at a multiple of four, and so do the rows
      const bool vec = P.taps == kTaps && A.dim % 4 == 0 && (P.codes ? P.channels % 4 == 0 && ((uintptr_t)P.codes & 3) == 0 : whole(P.x, P.type, 4, P.x_sb, P.x_st));
      if (P.codes) vec ? conv_tiles<T, WT, true, true>(P, A, st) : conv_tiles<T, WT, true, false>(P, A, st);
      else vec ? conv_tiles<T, WT, false, true>(P, A, st) : conv_tiles<T, WT, false, false>(P, A, st);
      return launch_status();
    }
    return (int)kEInval;
  });
}
int launch_conv_last(const ConvParams& P, cudaStream_t st) {
  const dim3 grid((P.channels + 4 * kThreads - 1) / (4 * kThreads), P.batch);
  return by_type(P.type, P.weight_type, [&](auto t, auto) {
    using T = decltype(t);
    if constexpr (sizeof(T) == 2) {                 // before a scan, which takes no fp32
      if (P.codes) conv_last_kernel<T, true><<<grid, kThreads, 0, st>>>(P);
      else conv_last_kernel<T, false><<<grid, kThreads, 0, st>>>(P);
      return launch_status();
    }
    return (int)kEInval;
  });
}

long long conv_workspace(int batch, int length, int channels) {
  const int strip = strip_of(batch, length, channels, kLeast, kMost);
  return (long long)batch * ((length + strip - 1) / strip) * (kTaps + 1) * channels * 4;
}

int launch_conv_forward(const ConvParams& P, cudaStream_t st) {
  const int strip = strip_of(P.batch, P.length, P.channels, 16, 64), per = kThreads * kWide;
  const dim3 grid((P.length + strip - 1) / strip, (P.channels + per - 1) / per, P.batch);
  const bool fast = P.taps == kTaps && P.silu && whole(P.x, P.type, kWide, P.x_sb, P.x_st) &&
                   whole(P.y, P.type, kWide, P.y_sb, P.y_st) && P.channels % kWide == 0 && ((uintptr_t)P.codes & (kWide - 1)) == 0;
  return by_type(P.type, P.weight_type, [&](auto t, auto w) {
    using T = decltype(t);
    using WT = decltype(w);
    if (P.codes) fast ? conv_kernel<T, WT, true, true><<<grid, kThreads, 0, st>>>(P, strip) : conv_kernel<T, WT, true, false><<<grid, kThreads, 0, st>>>(P, strip);
    else fast ? conv_kernel<T, WT, false, true><<<grid, kThreads, 0, st>>>(P, strip) : conv_kernel<T, WT, false, false><<<grid, kThreads, 0, st>>>(P, strip);
    return launch_status();
  });
}

int launch_conv_backward(const ConvParams& P, cudaStream_t st) {
  const int strip = strip_of(P.batch, P.length, P.channels, kLeast, kMost), per = kThreads * kWide;
  const dim3 grid((P.length + strip - 1) / strip, (P.channels + per - 1) / per, P.batch);
  const bool fast = P.taps == kTaps && P.silu && (!P.x || whole(P.x, P.type, kWide, P.x_sb, P.x_st)) &&
                   whole(P.dy, P.dy_f32 ? 2 : P.type, kWide, P.dy_sb, P.dy_st) && whole(P.dx, P.type, kWide, P.channels) && whole(P.workspace, 2, kWide, 0) && ((uintptr_t)P.codes & (kWide - 1)) == 0;
  return by_type(P.type, P.weight_type, [&](auto t, auto w) {
    using T = decltype(t);
    using WT = decltype(w);
    const auto launch = [&](auto d) {
      using DY = decltype(d);
      if (P.codes) fast ? conv_grad_kernel<T, WT, DY, true, true><<<grid, kThreads, 0, st>>>(P, strip) : conv_grad_kernel<T, WT, DY, true, false><<<grid, kThreads, 0, st>>>(P, strip);
      else fast ? conv_grad_kernel<T, WT, DY, false, true><<<grid, kThreads, 0, st>>>(P, strip) : conv_grad_kernel<T, WT, DY, false, false><<<grid, kThreads, 0, st>>>(P, strip);
    };
    if (P.dy_f32) launch(float{});
    else launch(T{});
    if (int s = launch_status()) return s;
    if (P.dweight || P.dbias) {
      conv_weights_kernel<WT><<<dim3((P.channels + 31) / 32, kTaps + 1), 256, 0, st>>>(P, (int)grid.x * P.batch);
      return launch_status();
    }
    return (int)kOk;
  });
}

int launch_conv_step(const ConvStepParams& P, cudaStream_t st) {
  const int per = kThreads * kWide;
  const dim3 grid((P.channels + per - 1) / per, P.batch);
  const int vec = whole(P.x, P.type, kWide, P.x_sb, P.channels) && whole(P.state, P.type, kWide, 0) && whole(P.y, P.y_f32 ? 2 : P.type, kWide, 0);
  return by_type(P.type, P.weight_type, [&](auto t, auto w) {
    using T = decltype(t);
    using WT = decltype(w);
    if (P.y_f32) conv_step_kernel<T, WT, float><<<grid, kThreads, 0, st>>>(P, vec);
    else conv_step_kernel<T, WT, T><<<grid, kThreads, 0, st>>>(P, vec);
    return launch_status();
  });
}

namespace {
dim3 pack_grid(const PackParams& P, int of_a_thread) {
  const int per = kThreads * of_a_thread, wide = (P.width + per - 1) / per;
  long long rows = (P.rows + kRows - 1) / kRows, most = 148 * 16 / wide;      // CTAs that an SM's threads hold
  most = most < 1 ? 1 : most > 65535 ? 65535 : most;
  return dim3(wide, (unsigned)(rows < most ? rows : most));
}
}  // namespace

// VEC: whole aligned pieces.
int launch_pack(const PackParams& P, cudaStream_t st) {
  const int unit = unit_of(P.type);
  const bool vec = whole(P.x, P.type, unit, P.x_stride, P.width) && ((uintptr_t)P.codes & 7) == 0;
  const dim3 grid = pack_grid(P, unit);
  return by_type(P.type, P.type, [&](auto t, auto) {
    using T = decltype(t);
    vec ? pack_kernel<T, true><<<grid, kThreads, 0, st>>>(P) : pack_kernel<T, false><<<grid, kThreads, 0, st>>>(P);
    return launch_status();
  });
}
int launch_unpack(const PackParams& P, cudaStream_t st) {
  const bool vec = whole(P.y, P.type, unit_of(P.type), P.width) && P.width % kCodes == 0 && ((uintptr_t)P.codes & 15) == 0;
  const dim3 grid = pack_grid(P, kCodes);
  return by_type(P.type, P.type, [&](auto t, auto) {
    using T = decltype(t);
    vec ? unpack_kernel<T, true><<<grid, kThreads, 0, st>>>(P) : unpack_kernel<T, false><<<grid, kThreads, 0, st>>>(P);
    return launch_status();
  });
}

}  // namespace sq
