// Device helpers shared by the kernels on rows of logits (logits.cu, distill.cu).
#pragma once
#include <cuda_bf16.h>
#include <type_traits>
#include "common.cuh"
#include "logits.cuh"

namespace sq {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;

// 2^x by the hardware instruction; exp2f gives the same bits for x in [-64, 0] (compared over
// 2^30 arguments), so the integer weights of a draw can be computed outside this library.
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(float v) { return v; }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
// The bits of a 16-bit number, of the largest one not above v.
template <typename T> __device__ __forceinline__ uint32_t bits_below(float v) {
  if constexpr (std::is_same<T, __half>::value) return __half_as_ushort(__float2half_rd(v));
  else return __bfloat16_as_ushort(__float2bfloat16_rd(v));
}
template <typename T> __device__ __forceinline__ T from_bits(uint32_t bits) {
  if constexpr (std::is_same<T, __half>::value) return __ushort_as_half((unsigned short)bits);
  else return __ushort_as_bfloat16((unsigned short)bits);
}

// Order-preserving key of a logit that is no NaN; callers add 0 first, so that -0 and +0 share one.
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t b = __float_as_uint(v);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_logit(uint32_t key) {       // inverse, for keys of numbers
  return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}
constexpr uint32_t kKeyLowest = 0x00800000u;     // order_key of the lowest finite number, one above -inf

// 16 bytes of a row.
template <typename T> constexpr int kUnit = 16 / (int)sizeof(T);
template <typename T> union Unit {
  uint4 q;
  T v[kUnit<T>];
};
__device__ __forceinline__ uint4 load_unit(const void* p) { return __ldg(reinterpret_cast<const uint4*>(p)); }

template <typename T> __device__ __forceinline__ uint4 neg_inf_unit() {
  const uint32_t w = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
  return make_uint4(w, w, w, w);
}
// Largest value of a unit, NaN passed over: -inf where there is nothing else.
__device__ __forceinline__ float unit_max(const Unit<__half>& u) {
  const __half2* h = reinterpret_cast<const __half2*>(&u.q);
  const __half2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
  return fmaxf(fmaxf(__low2float(m), __high2float(m)), -INFINITY);
}
__device__ __forceinline__ float unit_max(const Unit<__nv_bfloat16>& u) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&u.q);
  const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
  return fmaxf(fmaxf(__low2float(m), __high2float(m)), -INFINITY);
}
__device__ __forceinline__ float unit_max(const Unit<float>& u) {
  return fmaxf(fmaxf(fmaxf(u.v[0], u.v[1]), fmaxf(u.v[2], u.v[3])), -INFINITY);
}

// Running maximum of units, element by element or two by two; NaN is passed over.
__device__ __forceinline__ void fold_max(Unit<__half>& top, const Unit<__half>& u) {
  __half2* t = reinterpret_cast<__half2*>(&top.q);
  const __half2* h = reinterpret_cast<const __half2*>(&u.q);
  t[0] = __hmax2(t[0], __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
}
__device__ __forceinline__ void fold_max(Unit<__nv_bfloat16>& top, const Unit<__nv_bfloat16>& u) {
  __nv_bfloat162* t = reinterpret_cast<__nv_bfloat162*>(&top.q);
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&u.q);
  t[0] = __hmax2(t[0], __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
}
__device__ __forceinline__ void fold_max(Unit<float>& top, const Unit<float>& u) {
  top.v[0] = fmaxf(top.v[0], fmaxf(fmaxf(u.v[0], u.v[1]), fmaxf(u.v[2], u.v[3])));
}

// Where the part of a row that CTA `rank` of `size` works on lies: units of 16 bytes at 16-byte
// addresses.  Rows start where their stride puts them: the first and the last unit of a row may be
// ragged, and are filled up with -inf.
template <typename T>
struct Span {
  const T* p;
  int vocab, off, u0, n;                         // the part's first unit of the row and its units
  int lo, hi;                                    // whole units of the part: [lo, hi)
  __device__ Span(const LogitsRows& x, int row, uint32_t rank, uint32_t size) {
    p = reinterpret_cast<const T*>(x.data) + (long long)row * x.stride;
    vocab = x.vocab;
    off = (int)((uintptr_t)p & 15) / (int)sizeof(T);
    const int units = (off + vocab + kUnit<T> - 1) / kUnit<T>, per = (units + (int)size - 1) / (int)size;
    u0 = (int)rank * per;
    n = max(0, min(units, u0 + per) - u0);
    lo = n > 0 && col(0, 0) < 0 ? 1 : 0;
    hi = n > lo && col(n, 0) > vocab ? n - 1 : n;
  }
  __device__ int col(int i, int v) const { return (u0 + i) * kUnit<T> - off + v; }
  __device__ Unit<T> ragged(int i) const {
    Unit<T> u;
#pragma unroll
    for (int v = 0; v < kUnit<T>; ++v) {
      const int c = col(i, v);
      u.v[v] = c >= 0 && c < vocab ? p[c] : from_f32<T>(-INFINITY);
    }
    return u;
  }
};

// Cluster of the CTAs that share a row.
__device__ __forceinline__ uint32_t cluster_rank() { uint32_t r; asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ uint32_t cluster_size() { uint32_t r; asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.aligned;" ::: "memory"); }
// Says that this CTA runs, without ordering memory.
__device__ __forceinline__ void cluster_arrive_relaxed() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }
// Address of `p` (shared memory of this CTA) in the CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t remote_smem(const void* p, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ void remote_store(uint32_t addr, float a, float b) {
  asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" :: "r"(addr), "f"(a), "f"(b) : "memory");
}
__device__ __forceinline__ void remote_store(uint32_t addr, unsigned long long v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" :: "r"(addr), "l"(v) : "memory");
}
__device__ __forceinline__ unsigned long long remote_load(uint32_t addr) {
  unsigned long long v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
  return v;
}

}  // namespace sq
