// Selective scan in unquantised states (sm_100a): prompts, gradients, single tokens.
//
//   s_t = softplus(dt_t + bias),  H_t = exp(A s_t) H_{t-1} + s_t x_t B_t^T,  y_t = H_t C_t + D x_t
//
// per head, H fp32 [dim, 128], B and C shared by the heads of a group.  Work goes by chunks of 128 tokens.  With
// l_t the sum of A s over the chunk up to t,
//
//   y_t   = sum_{s<=t} exp(l_t - l_s) s_s (C_t . B_s) x_s + exp(l_t) H_in C_t + D x_t
//   H_out = exp(l_end) H_in + sum_s exp(l_end - l_s) s_s x_s B_s^T
//
// so that all but the chunks' order is matrix products: state_pass_kernel walks a head's chunks and leaves the state
// that enters each one, out_kernel then does every (chunk, group) on its own, and grad_kernel does the same for the
// gradients, with the states' own gradients from state_pass_kernel walking backwards (G_in = exp(l_end) G_out +
// sum_t exp(l_t) dy_t C_t^T).  All products run on tcgen05 with fp32 accumulators in TMEM.
//
// Operands are 16 bits.  B and C are brought to scaled fp16 once (prepare_kernel), so that states and weighted tokens can
// be fp16 beside them, value and remainder (22 bits) wherever a 32-bit result hangs on them.  Rounded to one number are:
//   * the pairs' weights exp(l_t - l_s) s_s (C_t . B_s) beside x and dy, in their type;
//   * the states in y, and the operands of dB and dC beside the states and of the pairs' part, in fp16.
// Their results are 16-bit tensors, whose own rounding is as large.  fp16 operands are scaled by powers of two per row,
// tile, chunk or CTA, whatever the range of bf16; tokens and states of up to 2^118 have sums that are fp32 numbers.  A bf16 number of B or
// C below 2^-28 of its tile's largest loses bits that no sum can hold; so do a head's products for dB and dC below 2^-28 of the
// largest among the heads of its CTA.
// Sums of A s are doubles, kept as two floats: neighbours' differences keep 24 bits wherever in the chunk they lie.
#include "selective.cuh"
#include <type_traits>
#include "device_util.cuh"
#include "logits_util.cuh"
#include "pairs.cuh"
#include "tc_util.cuh"

namespace sq {
namespace {

using namespace tc;

constexpr int Q = kScanChunk;
constexpr int TP = kScanTile;
constexpr int kN = 128;
constexpr int kThreads = 256;
constexpr int kRecord = 7;                                 // numbers that a token of a head has
constexpr uint32_t kTile128 = 32768, kTile64 = 16384;      // bytes of a [128][128] and a [128][64] 16-bit tile

// ---------------------------------------------------------------- operands in shared memory
// Tiles are rows of 128 bytes (64 numbers) with the 128-byte swizzle: 16-byte piece j of row r lies at
// r * 128 + ((j ^ (r & 7)) << 4).  A [128][128] tile is two such tiles, columns 0..63 and 64..127.
__device__ __forceinline__ uint32_t piece(int row, int j) { return (uint32_t)(row * 128 + ((j ^ (row & 7)) << 4)); }
__device__ __forceinline__ uint32_t piece2(int row, int j) { return (uint32_t)((j >> 3) * kTile64) + piece(row, j & 7); }

__device__ __forceinline__ uint4 lds16(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void sts16(uint32_t a, uint4 v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" :: "r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool take) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" :: "r"(dst), "l"(src), "r"(take ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int K> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" :: "n"(K) : "memory"); }
// What the threads wrote to shared memory becomes visible to the tensor cores (after the next CTA barrier).
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Matrix descriptors of operands in such tiles.  K-major: a row is an index of M or N, its columns are K
// (16 of K: 32 bytes on).  MN-major: a row is an index of K, its columns are M or N (16 of K: 2,048 bytes on; the
// second 64 columns of M or N 16,384 bytes on).
__device__ __forceinline__ uint64_t desc_k(uint32_t a) { return sw128_desc(a); }
__device__ __forceinline__ uint64_t desc_mn(uint32_t a) {
  return (uint64_t)((a & 0x3FFFFu) >> 4) | (uint64_t)(kTile64 >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
template <typename T> __device__ __forceinline__ constexpr uint32_t idesc(int n, bool a_mn, bool b_mn) {
  const uint32_t f = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  return (1u << 4) | (f << 7) | (f << 10) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | (8u << 24);
}
// A state's plane: 16-byte pieces (eight rows p) [8][128 columns n], without swizzle.  As N = p, K = n: 16 of K are
// 256 bytes on; as N = n, K = p: 4,096 bytes on.
__device__ __forceinline__ uint64_t desc_plain(uint32_t a, uint32_t lbo, uint32_t sbo) {
  return (uint64_t)((a & 0x3FFFFu) >> 4) | (uint64_t)(lbo >> 4) << 16 | (uint64_t)(sbo >> 4) << 32 | (uint64_t)1 << 46;
}
enum Form { kK, kMn, kPlaneP, kPlaneN };            // K-major tile, MN-major tile, plane with N = p, plane with N = n
template <Form F> __device__ __forceinline__ uint64_t desc_at(uint32_t a, int k) {
  if constexpr (F == kK) return desc_k(a + (uint32_t)((k >> 2) * kTile64 + (k & 3) * 32));
  else if constexpr (F == kMn) return desc_mn(a + (uint32_t)k * 2048);
  else if constexpr (F == kPlaneP) return desc_plain(a + (uint32_t)k * 256, 128, 2048);
  else return desc_plain(a + (uint32_t)k * 4096, 2048, 128);
}
// D[128][n] (+)= A . B over K = 16 * steps; a / b: addresses of the tiles.  K-major tiles of 128 columns go on in
// their second half after four steps.
template <Form FA, Form FB>
__device__ __forceinline__ void mma(uint32_t d, uint32_t a, uint32_t b, uint32_t id, int steps, bool accumulate) {
#pragma unroll
  for (int k = 0; k < steps; ++k) umma_f16(d, desc_at<FA>(a, k), desc_at<FB>(b, k), id, accumulate || k);
}
// `bytes` (a multiple of 16) from global to shared memory, counted by the barrier.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               :: "r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
// Brings what a later load reads to the L2 cache.
__device__ __forceinline__ void prefetch(const void* src) { asm volatile("prefetch.global.L2 [%0];" :: "l"(src)); }
__device__ __forceinline__ void tmem_ld32_nowait(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}

__device__ __forceinline__ void tmem_ld16_nowait(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  tmem_ld16_nowait(taddr, r);
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

// Keeps uses of a tcgen05.ld's registers behind the wait that precedes this call.
template <int N> __device__ __forceinline__ void settle(uint32_t (&r)[N]) {
#pragma unroll
  for (int i = 0; i < N; i += 8)
    asm volatile("" : "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3]), "+r"(r[i + 4]), "+r"(r[i + 5]), "+r"(r[i + 6]), "+r"(r[i + 7]));
}

// Eight numbers are worked on as four pairs: the adders and multipliers take two fp32 numbers an instruction.
struct Eight { float2 v[4]; };
template <typename T> __device__ __forceinline__ Eight unpack8(uint4 u) {
  return {{unpack2<T>(u.x), unpack2<T>(u.y), unpack2<T>(u.z), unpack2<T>(u.w)}};
}
template <typename T> __device__ __forceinline__ uint4 pack8(const Eight& f) {
  return make_uint4(pack2<T>(f.v[0].x, f.v[0].y), pack2<T>(f.v[1].x, f.v[1].y), pack2<T>(f.v[2].x, f.v[2].y), pack2<T>(f.v[3].x, f.v[3].y));
}
__device__ __forceinline__ Eight mul8(const Eight& a, float f) {
  return {{mul2(a.v[0], pair(f)), mul2(a.v[1], pair(f)), mul2(a.v[2], pair(f)), mul2(a.v[3], pair(f))}};
}
// Value and remainder of eight numbers.
template <typename T> __device__ __forceinline__ void split8(const Eight& f, uint4& hi, uint4& lo) {
  hi = pack8<T>(f);
  const Eight r = unpack8<T>(hi);
  lo = pack8<T>({{sub2(f.v[0], r.v[0]), sub2(f.v[1], r.v[1]), sub2(f.v[2], r.v[2]), sub2(f.v[3], r.v[3])}});
}
// The largest magnitude of two by two 16-bit numbers; NaN is passed over.
__device__ __forceinline__ __half2 fold(__half2 m, uint32_t v) { return __hmax2(m, __habs2(*reinterpret_cast<const __half2*>(&v))); }
__device__ __forceinline__ __nv_bfloat162 fold(__nv_bfloat162 m, uint32_t v) { return __hmax2(m, __habs2(*reinterpret_cast<const __nv_bfloat162*>(&v))); }
template <typename T> struct Two;
template <> struct Two<__half> { using type = __half2; };
template <> struct Two<__nv_bfloat16> { using type = __nv_bfloat162; };
// Pairs' weights in bf16, a product of two scaled rows (2^35 at most) each: the sums that they make with tokens of up to 2^118 are fp32
// numbers.
constexpr float kWeightThere = 0x1p-32f, kWeightBack = 0x1p32f;

// The power of two that brings `bits` (a maximum's, sign cleared) to [2^13, 2^14) and its inverse: {there, back}.  NaN where the
// maximum is an infinity or NaN, which leaves the other numbers no scale: what is made of them is then NaN, and not zero.
// Zeros come back by 0, so that they weigh nothing where scales are compared.
// Maxima below 2^-97 are brought less far, so that a scale is a normal number.
__device__ __forceinline__ float2 scale_of(uint32_t bits) {
  if (bits >= 0x7f800000u) return make_float2(__uint_as_float(0x7fffffffu), __uint_as_float(0x7fffffffu));
  int e = (int)(bits >> 23) - 140;
  e = bits ? max(-110, e) : 0;
  return make_float2(__uint_as_float((uint32_t)(127 - e) << 23), bits ? __uint_as_float((uint32_t)(127 + e) << 23) : 0.f);
}

__device__ __forceinline__ float number(const void* p, int type, int i) {
  if (!p) return 0.f;
  return type == SQ_TYPE_F32 ? reinterpret_cast<const float*>(p)[i]
         : type == SQ_TYPE_BF16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i])
                                : __half2float(reinterpret_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void put_number(void* p, int type, int i, float v) {
  if (type == SQ_TYPE_F32) reinterpret_cast<float*>(p)[i] = v;
  else if (type == SQ_TYPE_BF16) reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else reinterpret_cast<__half*>(p)[i] = __float2half_rn(v);
}

__device__ __forceinline__ int tokens_of(const SelectiveParams& P, int b) {
  return P.lengths ? max(0, min(P.length, P.lengths[b])) : P.length;
}

// ---------------------------------------------------------------- workspace
struct Space {
  int nc, ptiles, units;              // chunks of the longest sequence, tiles of a head's rows, heads * ptiles
  long long lp;
  float* rec;                         // [B][H][nc][kRecord][Q], see prepare_kernel
  float* smax;                        // [B][H][nc]: the largest s of a chunk
  uint16_t *bt, *ct;                  // [B][nc][G][128][128]: B and C as shared memory holds them
  float *bback, *cback;               // [B][nc][G]: what brings them back
  uint16_t *xt, *yt;                  // [B][nc][units][128][64]: x and dy in the same form, behind a convolution
  float *xback, *yback;               // [B][nc][units]
  uint16_t *h, *g;                    // [B][nc][units][2][8][128][8]: states entering a chunk, gradients of those leaving it
  float2 *hs, *gs;                    // [B][nc][units]: scale of the state, scale of the chunk's weighted tokens; 0 of zeros
  float2* parts;                      // [B][units][lp]: gradient of A s, gradient of s through the tokens
  float2* unit_sums;                  // [B][nc][units]: gradients of D and of A by chunk
  float* bias_sums;                   // [B][nc][H][4]: gradient of the bias by 32 tokens
  float *pb, *pc;                     // [splits][B][nc * Q][G][128]: dB and dC by split
  int splits;
  long long bytes;
};

constexpr int kSms = 148;

// CTAs that share a group's units.  A CTA's time is that of its units and of what it does once; all CTAs' time is that of
// the rounds in which the SMs' places take them.  2 x 2,048 tokens at 128 heads, gradients: 16 units a CTA (2 rounds).
int splits_of(long long tiles, int units, int places, double once) {
  int best = 1;
  double least = 1e30;
  for (int s = 1; s <= units; ++s) {
    const int per = (units + s - 1) / s, used = (units + per - 1) / per;
    if (used != s) continue;
    const double time = (double)((tiles * s + places - 1) / places) * (per + once * (s > 1 ? 1.5 : 1.0));
    if (time < 0.999 * least) { least = time; best = s; }
  }
  return best;
}

Space space_of(const SelectiveParams& P, bool backward, bool tiled) {
  Space w{};
  w.nc = (P.length + Q - 1) / Q;
  w.lp = (long long)w.nc * Q;
  w.ptiles = (P.dim + TP - 1) / TP;
  w.units = P.heads * w.ptiles;
  const long long bc = (long long)P.batch * w.nc, bcu = bc * w.units, bh = (long long)P.batch * P.heads;
  char* base = reinterpret_cast<char*>(P.workspace);
  long long at = 0;
  auto take = [&](long long bytes) { char* p = base + at; at += (bytes + 255) / 256 * 256; return p; };
  w.rec = reinterpret_cast<float*>(take(bh * w.lp * kRecord * 4));
  w.bt = reinterpret_cast<uint16_t*>(take(bc * P.groups * kTile128));
  w.ct = reinterpret_cast<uint16_t*>(take(bc * P.groups * kTile128));
  w.bback = reinterpret_cast<float*>(take(bc * P.groups * 4));
  w.cback = reinterpret_cast<float*>(take(bc * P.groups * 4));
  w.smax = reinterpret_cast<float*>(take(bh * w.nc * 4));
  if (tiled) {
    w.xt = reinterpret_cast<uint16_t*>(take(bcu * kTile64));
    w.xback = reinterpret_cast<float*>(take(bcu * 4));
    if (backward) {
      w.yt = reinterpret_cast<uint16_t*>(take(bcu * kTile64));
      w.yback = reinterpret_cast<float*>(take(bcu * 4));
    }
  }
  const long long plane = (long long)kN * TP * 2 * 2;
  w.h = reinterpret_cast<uint16_t*>(take(bcu * plane));
  w.hs = reinterpret_cast<float2*>(take(bcu * 8));
  w.splits = splits_of(bc * P.groups, w.units / P.groups, backward ? kSms : 2 * kSms, backward ? 1.0 : 0.5);
  if (backward) {
    w.g = reinterpret_cast<uint16_t*>(take(bcu * plane));
    w.gs = reinterpret_cast<float2*>(take(bcu * 8));
    w.parts = reinterpret_cast<float2*>(take((long long)P.batch * w.units * w.lp * 8));
    w.unit_sums = reinterpret_cast<float2*>(take(bcu * 8));
    w.bias_sums = reinterpret_cast<float*>(take(bc * P.heads * 16));
    if (w.splits > 1) {
      const long long part = bc * Q * P.groups * kN * 4 * w.splits;
      w.pb = reinterpret_cast<float*>(take(part));
      w.pc = reinterpret_cast<float*>(take(part));
    }
  }
  w.bytes = at;
  return w;
}

// ---------------------------------------------------------------- tiles from global memory
// A tile [128][64]: row t at src + t * stride, rows from `rows` on and columns from `cols` on are zero.  vec: 16-byte
// pieces are whole and aligned.
template <typename T>
__device__ __forceinline__ uint4 ragged_piece(const T* p, int n) {
  uint32_t u[4] = {0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (e < n) u[e >> 1] |= (uint32_t)reinterpret_cast<const uint16_t*>(p)[e] << (16 * (e & 1));
  return make_uint4(u[0], u[1], u[2], u[3]);
}
template <typename T, int THREADS = kThreads>
__device__ __forceinline__ void load_tile(uint32_t dst, const T* src, long long stride, int rows, int cols, bool vec) {
  const int j = threadIdx.x & 7;
  const T* p = src + (long long)(threadIdx.x >> 3) * stride + j * 8;
#pragma unroll
  for (int i = 0; i < Q * 8 / THREADS; ++i, p += (THREADS / 8) * stride) {
    const int r = (threadIdx.x >> 3) + i * (THREADS / 8);
    const uint32_t a = dst + piece(r, j);
    const bool in = r < rows && j * 8 < cols;
    if (vec) cp16(a, in ? p : src, in);
    else sts16(a, in ? ragged_piece(p, cols - j * 8) : make_uint4(0, 0, 0, 0));
  }
}
// The first `rows` rows and `cols` columns of a tile [128][64] to global memory.
template <typename T, int THREADS = kThreads>
__device__ __forceinline__ void store_tile(T* dst, long long stride, uint32_t src, int rows, int cols, bool vec) {
  for (int i = threadIdx.x; i < Q * 8; i += THREADS) {
    const int r = i >> 3, j = i & 7;
    if (r >= rows || j * 8 >= cols) continue;
    const uint4 v = lds16(src + piece(r, j));
    T* p = dst + (long long)r * stride + j * 8;
    if (vec) {
      *reinterpret_cast<uint4*>(p) = v;
    } else {
      const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (j * 8 + e < cols) reinterpret_cast<uint16_t*>(p)[e] = (uint16_t)(u[e >> 1] >> (16 * (e & 1)));
    }
  }
}
// The same of a tile [128][64] of fp32: rows of 256 bytes, 16-byte piece j of row r at r * 256 + ((j ^ (r & 7)) << 4).
__device__ __forceinline__ uint32_t piece_f32(int row, int j) { return (uint32_t)(row * 256 + ((j ^ (row & 7)) << 4)); }
template <int THREADS>
__device__ __forceinline__ void store_tile(float* dst, long long stride, uint32_t src, int rows, int cols, bool) {
  const bool vec = ((uintptr_t)dst & 15) == 0 && ((stride | cols) & 3) == 0;
  for (int i = threadIdx.x; i < Q * 16; i += THREADS) {
    const int r = i >> 4, j = i & 15;
    if (r >= rows || j * 4 >= cols) continue;
    const uint4 v = lds16(src + piece_f32(r, j));
    float* p = dst + (long long)r * stride + j * 4;
    if (vec) {
      *reinterpret_cast<uint4*>(p) = v;
    } else {
      const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (j * 4 + e < cols) p[e] = __uint_as_float(u[e]);
    }
  }
}
__device__ __forceinline__ bool vector_ok(const void* p, long long s0, long long s1, int cols) {
  return ((uintptr_t)p & 15) == 0 && ((s0 | s1 | cols) & 7) == 0;
}

// A barrier that a CTA's threads wait on: for the tensor cores' work, or for bulk copies.  A wait that expires is
// recorded, and no further one is begun (`ok` is the thread's own).
struct Gate {
  uint32_t bar, parity;
  __device__ void wait(bool& ok, int* err) {
    if (ok && !mbar_wait(bar, parity)) {
      ok = false;
      atomicOr(err, (int)kDevTimeoutMma);
    }
    parity ^= 1;
  }
};
// Barriers [count] at `bars` and COLS columns of TMEM; `slot` holds their address.
template <int COLS>
__device__ __forceinline__ uint32_t tensor_begin(uint64_t* bars, int count, uint32_t* slot) {
  if (threadIdx.x == 0) {
    for (int i = 0; i < count; ++i) mbar_init(smem_u32(bars + i), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_async();
  }
  if (threadIdx.x < 32) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(smem_u32(slot)), "n"(COLS));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  return *slot;
}
// A CTA whose wait expired (`ok` false) gives what it has in flight, bulk copies and products, two milliseconds before its shared
// memory and TMEM are another's: a thousand times what they take.
template <int COLS> __device__ __forceinline__ void tensor_end(uint32_t tmem, bool ok) {
  if (!ok) {
    const uint64_t since = gtime();
    for (int i = 0; i < 4000 && gtime() - since < 2000000; ++i) __nanosleep(1000);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (threadIdx.x < 32) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(tmem), "n"(COLS));
}

// ---------------------------------------------------------------- steps and decays
// A in base 2.  An A of zero becomes one that decays nothing either, so that time can be told from l.
__device__ __forceinline__ double decay_rate(float A) {
  return fabsf(A) < 1e-20f ? -1e-20 : (double)A * 1.4426950408889634;
}
__device__ __forceinline__ float decay_rate_f32(float A) { return fabsf(A) < 1e-20f ? -1e-20f : A * kLog2e; }
// One CTA: a chunk of eight heads (a warp a head, four tokens a lane), or a chunk's tile of B or C (behind a convolution, of
// dy).  Eight heads: their steps of a token are 16 neighbouring bytes.  2 x 2,048 tokens of 128 heads: 11 us, most of it a
// launch's latency and the sums' chain in double; with the tiles of dy 28 us.
constexpr int kPrepHeads = 8;
template <typename T>
__global__ void __launch_bounds__(kThreads) prepare_kernel(const SelectiveParams P, const Space W, int head_blocks) {
  __shared__ float step[kPrepHeads][Q + 4], slope[kPrepHeads][Q + 4];
  __shared__ uint32_t tops[kThreads / 32];
  launch_dependents();
  const int c = blockIdx.x, b = blockIdx.z, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int len = tokens_of(P, b), rows = min(Q, len - c * Q);
  if ((int)blockIdx.y >= head_blocks) {
    const int i = blockIdx.y - head_blocks;
    if (rows <= 0) return;                               // not read
    // a tile of B or C [128][128], or behind a convolution one of dy [128][64]
    const bool narrow = P.tiled;
    const int g = i >> 1, u = i, pieces = narrow ? 8 : 16, j = threadIdx.x & (pieces - 1), step = kThreads / pieces;
    const long long st = narrow ? P.dy_st : i & 1 ? P.c_st : P.b_st;
    const T* src;
    int cols = kN;
    if (narrow) {
      const int p0 = (u % W.ptiles) * TP;
      cols = min(TP, P.dim - p0);
      src = reinterpret_cast<const T*>(P.dy) + (long long)b * P.dy_sb + (long long)c * Q * st + (long long)(u / W.ptiles) * P.dim + p0;
    } else {
      src = reinterpret_cast<const T*>(i & 1 ? P.C : P.B) + (long long)b * (i & 1 ? P.c_sb : P.b_sb) + (long long)c * Q * st + g * kN;
    }
    const bool vec = vector_ok(src, st, 0, cols);
    const int count = pieces / 2;
    uint4 u4[8];
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      u4[k] = make_uint4(0, 0, 0, 0);
      const int r = threadIdx.x / pieces + k * step;
      const T* p = src + (long long)r * st + j * 8;
      if (k < count && r < rows && j * 8 < cols) u4[k] = vec ? *reinterpret_cast<const uint4*>(p) : ragged_piece(p, cols - j * 8);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t w[4] = {u4[k].x, u4[k].y, u4[k].z, u4[k].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) m = __vmaxu2(m, w[e] & 0x7fff7fffu);
    }
    m = __reduce_max_sync(0xffffffffu, max(m & 0xffff, m >> 16));
    if (lane == 0) tops[warp] = m;
    __syncthreads();
    m = 0;
#pragma unroll
    for (int k = 0; k < kThreads / 32; ++k) m = max(m, tops[k]);
    const float2 sc = scale_of(__float_as_uint(to_f32(from_bits<T>(m))));
    const long long bc = (long long)b * W.nc + c, at = narrow ? bc * W.units + u : bc * P.groups + g;
    char* out = reinterpret_cast<char*>(narrow ? W.yt + at * (Q * TP) : (i & 1 ? W.ct : W.bt) + at * (Q * kN));
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < count) *reinterpret_cast<uint4*>(out + piece2(threadIdx.x / pieces + k * step, j)) = pack8<__half>(mul8(unpack8<T>(u4[k]), sc.x));
    if (threadIdx.x == 0) (narrow ? W.yback : i & 1 ? W.cback : W.bback)[at] = sc.y;
    return;
  }
  const int h0 = blockIdx.y * kPrepHeads, hl = threadIdx.x & 7;
  const T* dt = reinterpret_cast<const T*>(P.dt) + (long long)b * P.dt_sb;
  const float bias = h0 + hl < P.heads ? number(P.dt_bias, P.bias_type, h0 + hl) : 0.f;
#pragma unroll
  for (int k = 0; k < Q / 32; ++k) {
    const int t = (threadIdx.x >> 3) + k * 32;
    float s = 0.f, d = 0.f;
    if (t < rows && h0 + hl < P.heads) {
      const float v = to_f32(dt[(long long)(c * Q + t) * P.dt_st + h0 + hl]) + bias;
      s = v <= 20.0f ? log1pf(expf(v)) : v;
      d = 1.0f / (1.0f + expf(-v));
    }
    step[hl][t] = s;
    slope[hl][t] = d;
  }
  __syncthreads();
  const int h = h0 + warp;
  if (h >= P.heads) return;
  const double rate = decay_rate(P.A[h]);
  const float4 s4 = *reinterpret_cast<const float4*>(&step[warp][4 * lane]);
  const float s[4] = {s4.x, s4.y, s4.z, s4.w};
  double l[4], sum = 0.0;
#pragma unroll
  for (int i = 0; i < 4; ++i) l[i] = sum += rate * (double)s[i];
  double before = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double v = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= o) before += v;
  }
  before -= sum;
  float hi[4], lo[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    hi[i] = (float)(before + l[i]);
    lo[i] = (float)(before + l[i] - (double)hi[i]);
  }
  // The chunk in blocks of 32 tokens: l from the block's beginning (the l before its first token) and to its end
  const double begin = __shfl_sync(0xffffffffu, before, lane & 24), finish = __shfl_sync(0xffffffffu, before + l[3], lane | 7);
  float in_block[4], since[4], until[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    in_block[i] = (float)(before + l[i] - begin);
    since[i] = exp2f(in_block[i]);
    until[i] = s[i] * exp2f((float)(finish - (before + l[i])));
  }
  const long long row = ((long long)b * P.heads + h) * W.nc + c;
  float4* out = reinterpret_cast<float4*>(W.rec + row * (kRecord * Q)) + lane;
  out[0] = s4;                                                               // s
  out[Q / 4] = make_float4(hi[0], hi[1], hi[2], hi[3]);                      // l in base 2, value
  out[2 * Q / 4] = make_float4(lo[0], lo[1], lo[2], lo[3]);                  // and remainder
  out[3 * Q / 4] = make_float4(until[0], until[1], until[2], until[3]);      // s 2^(l at the block's end - l)
  out[4 * Q / 4] = make_float4(since[0], since[1], since[2], since[3]);      // 2^(l - l before the block)
  out[5 * Q / 4] = make_float4(in_block[0], in_block[1], in_block[2], in_block[3]);
  out[6 * Q / 4] = *reinterpret_cast<const float4*>(&slope[warp][4 * lane]); // sigmoid(dt + bias)
  const uint32_t m = __reduce_max_sync(0xffffffffu, __float_as_uint(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]))));
  if (lane == 0) W.smax[row] = __uint_as_float(m);
}

// ---------------------------------------------------------------- states by chunk
// One CTA walks the chunks of one unit (64 rows of a head's state), forwards or backwards.  The state is fp32 in
// registers: thread (n, half) holds state[n][32 half .. +32].  A chunk's addition is B^T (w x), with w x as value and
// remainder.  Written before each chunk: the state that enters it, value and (LO) remainder.  Bound by the chain from chunk
// to chunk (tokens, their largest value, the product, the new state: 2.6 to 3 us), not by bytes or products: 64 rows a CTA
// let two walk side by side on an SM, 256 of them at once.  2 x 2,048 tokens of 128 heads: 48 us; both ways of a
// backward pass, 512 walks on 296 places, 101 us.
constexpr uint32_t kPassX = 2 * kTile128, kPassW = kPassX + kTile64, kPassBytes = kPassW + 2 * kTile64, kPassSmem = kPassBytes + 64;

template <typename T, bool REV, bool LO, bool TILED>
__device__ __forceinline__ void state_pass(const SelectiveParams& P, const Space& W, float* state_out) {
  extern __shared__ __align__(1024) unsigned char smem[];
  const uint32_t base = smem_u32(smem);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kPassBytes);           // tensor cores, tile 0, tile 1, tokens (TILED)
  uint32_t* slot = reinterpret_cast<uint32_t*>(smem + kPassBytes + 48);
  uint32_t* tops = reinterpret_cast<uint32_t*>(smem + kPassBytes + 32);      // [2][2]: of the tokens, of the state
  const int u = blockIdx.x, b = blockIdx.y;
  const int h = u / W.ptiles, p0 = (u % W.ptiles) * TP, g = h / (P.heads / P.groups);
  const int cols = min(TP, P.dim - p0);
  const int len = tokens_of(P, b), nc = (len + Q - 1) / Q;
  const int n = threadIdx.x & 127, half = threadIdx.x >> 7, quad = threadIdx.x >> 5 & 3;
  const float* first = REV ? P.dstate_out : P.state_in;
  float* last = REV ? P.dstate_in : state_out;
  uint16_t* planes = REV ? W.g : W.h;
  float2* scales = REV ? W.gs : W.hs;
  const T* tok = reinterpret_cast<const T*>(REV ? P.dy : P.x) + (long long)b * (REV ? P.dy_sb : P.x_sb) + (long long)h * P.dim + p0;
  const long long tok_st = REV ? P.dy_st : P.x_st;
  const bool tok_vec = vector_ok(tok, tok_st, 0, cols);
  const uint16_t* tiles = (REV ? W.ct : W.bt) + ((long long)b * W.nc * P.groups + g) * (Q * kN);
  const float* tile_back = (REV ? W.cback : W.bback) + (long long)b * W.nc * P.groups + g;
  const float* recs = W.rec + ((long long)b * P.heads + h) * W.nc * (kRecord * Q);
  const long long state_at = (((long long)b * P.heads + h) * P.dim + p0) * kN + n;
  if (threadIdx.x < 4) tops[threadIdx.x] = 0;
  launch_dependents();
  const uint32_t tmem = tensor_begin<128>(bars, 4, slot);
  wait_for_launch();
  Gate done{smem_u32(bars), 0}, tokens{smem_u32(bars + 3), 0};
  using X = typename std::conditional<TILED, __half, T>::type;
  const uint16_t* xt = TILED ? (REV ? W.yt : W.xt) + ((long long)b * W.nc * W.units + u) * (Q * TP) : nullptr;
  const float* xback = TILED ? (REV ? W.yback : W.xback) + (long long)b * W.nc * W.units + u : nullptr;
  bool ok = true;
  const uint32_t mine = tmem + ((uint32_t)quad << 21) + (uint32_t)half * 32;

  auto load = [&](int i) {
    const int c = REV ? nc - 1 - i : i;
    if (threadIdx.x == 0 && (i + 1 < nc || last)) {
      mbar_expect_tx(smem_u32(bars + 1 + (i & 1)), kTile128);
      bulk_load(base + (i & 1) * kTile128, tiles + (long long)c * P.groups * (Q * kN), kTile128, smem_u32(bars + 1 + (i & 1)));
    }
    if constexpr (TILED) {
      if (threadIdx.x == 0) {
        mbar_expect_tx(tokens.bar, kTile64);
        bulk_load(base + kPassX, xt + (long long)c * W.units * (Q * TP), kTile64, tokens.bar);
      }
    } else {
      load_tile<T>(base + kPassX, tok + (long long)c * Q * tok_st, tok_st, len - c * Q, cols, tok_vec);
      cp_commit();
    }
    // The chunk after it, where tokens come from memory and one walk does not hide that: 4 prompts of up to 4,096 tokens 96 ->
    // 83 us.  Tiles behind a convolution are in the cache, and two ways at once wait for each other instead: nothing gained.
    if constexpr (!TILED && !LO) {
      const int t = (c + 1) * Q + n;
      if (half && t < len) prefetch(tok + (long long)t * tok_st);
    }
  };
  float s, lh, ll, eh, el, back, xb = 1.f;                         // of the next chunk: my token's, the chunk's end's, the tile's
  auto load_record = [&](int i) {
    const int c = REV ? nc - 1 - i : i;
    const float* r = recs + (long long)c * (kRecord * Q);
    s = r[n]; lh = r[Q + n]; ll = r[2 * Q + n]; eh = r[2 * Q - 1]; el = r[3 * Q - 1];
    back = tile_back[(long long)c * P.groups];
    if (TILED) xb = xback[(long long)c * W.units];
  };
  if (nc > 0) { load(0); load_record(0); }
  float2 S[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int p = half * 32 + 2 * i;
    S[i].x = first && p < cols ? first[state_at + (long long)p * kN] : 0.f;
    S[i].y = first && p + 1 < cols ? first[state_at + (long long)(p + 1) * kN] : 0.f;
  }
  using Pair = typename Two<X>::type;
  uint32_t parity = 0;                                   // of the tiles' barriers, a bit each
  for (int i = 0; i < nc; ++i) {
    const int c = REV ? nc - 1 - i : i;
    const long long at = ((long long)b * W.nc + c) * W.units + u;
    const bool update = i + 1 < nc || last, write = i > 0 || first;
    if (write) {
      float m = 0.f;
#pragma unroll
      for (int k = 0; k < 16; ++k) m = fmaxf(m, fmaxf(fabsf(S[k].x), fabsf(S[k].y)));
      const uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(m));
      if ((threadIdx.x & 31) == 0) atomicMax(&tops[2 * (i & 1) + 1], bits);
    }
    const float w = (REV ? exp2f(lh + ll) : s * exp2f((eh - lh) + (el - ll))) * xb, decay = exp2f(eh + el), tback = back;
    if constexpr (TILED) tokens.wait(ok, P.err);
    else cp_wait<0>();
    __syncthreads();
    uint4 v[4];
    const uint32_t none = 0;
    Pair m2 = *reinterpret_cast<const Pair*>(&none);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[j] = lds16(base + kPassX + piece(n, half * 4 + j));
      m2 = fold(fold(fold(fold(m2, v[j].x), v[j].y), v[j].z), v[j].w);
    }
    {
      const uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(fmaxf(to_f32(m2.x), to_f32(m2.y)) * w));
      if ((threadIdx.x & 31) == 0) atomicMax(&tops[2 * (i & 1)], bits);
    }
    __syncthreads();
    if (i + 1 < nc) load(i + 1);                         // all have their tokens, and the other tile was used two chunks ago
    const float2 wsc = scale_of(tops[2 * (i & 1)]), ssc = scale_of(tops[2 * (i & 1) + 1]);
    if (update) {
      const float ws = w * wsc.x;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint4 hi, lo;
        split8<__half>(mul8(unpack8<X>(v[j]), ws), hi, lo);
        sts16(base + kPassW + piece(n, half * 4 + j), hi);
        sts16(base + kPassW + kTile64 + piece(n, half * 4 + j), lo);
      }
      fence_async();
    }
    __syncthreads();
    if (threadIdx.x < 2) tops[2 * (i & 1) + threadIdx.x] = 0;                // read by all, used again in two chunks
    if (update && threadIdx.x == 0) {
      Gate tile{smem_u32(bars + 1 + (i & 1)), parity >> (i & 1) & 1};
      tile.wait(ok, P.err);
      parity ^= 1u << (i & 1);
      if (ok) {
        tc_fence_after();
        // values and remainders side by side: a product of 128 columns takes little longer than one of 64
        mma<kMn, kMn>(tmem, base + (i & 1) * kTile128, base + kPassW, idesc<__half>(2 * TP, true, true), 8, false);
        umma_commit(done.bar);
      }
    }
    if (i + 1 < nc) load_record(i + 1);
    if (write) {
      uint16_t* out = planes + at * (2 * kN * TP) + ((half * 4) * kN + n) * 8;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const Eight f = mul8({{S[4 * j], S[4 * j + 1], S[4 * j + 2], S[4 * j + 3]}}, ssc.x);
        uint4 hi, lo;
        if (LO) split8<__half>(f, hi, lo);
        else hi = pack8<__half>(f);
        *reinterpret_cast<uint4*>(out + j * (kN * 8)) = hi;
        if (LO) *reinterpret_cast<uint4*>(out + kN * TP + j * (kN * 8)) = lo;
      }
    }
    if (threadIdx.x == 0) scales[at] = make_float2(ssc.y, wsc.y);
    if (update) {
      done.wait(ok, P.err);
      tc_fence_after();
      const float f = wsc.y * tback;
#pragma unroll
      for (int j = 0; j < 32; j += 16) {
        uint32_t r[16], q[16];
        tmem_ld16_nowait(mine + j, r);
        tmem_ld16(mine + TP + j, q);
        settle(r);
#pragma unroll
        for (int k = 0; k < 8; ++k)
          S[j / 2 + k] = fma2(S[j / 2 + k], pair(decay), mul2(add2(words2(r[2 * k], r[2 * k + 1]), words2(q[2 * k], q[2 * k + 1])), pair(f)));
      }
      tc_fence_before();
    }
  }
  if (last)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int p = half * 32 + 2 * i;
      if (p < cols) last[state_at + (long long)p * kN] = S[i].x;
      if (p + 1 < cols) last[state_at + (long long)(p + 1) * kN] = S[i].y;
    }
  tensor_end<128>(tmem, ok);
}
template <typename T, bool TILED>
__global__ void __launch_bounds__(kThreads, 2) state_pass_kernel(const SelectiveParams P, const Space W) {
  state_pass<T, false, false, TILED>(P, W, P.state_out);
}
// A backward's: the states again, with remainders, and their gradients, whose walks do not need one another.
template <typename T, bool TILED>
__global__ void __launch_bounds__(kThreads, 2) state_passes_kernel(const SelectiveParams P, const Space W) {
  if (blockIdx.z == 0) state_pass<T, false, true, TILED>(P, W, nullptr);
  else state_pass<T, true, true, TILED>(P, W, nullptr);
}

// ---------------------------------------------------------------- outputs by chunk and group
// One CTA: a chunk and some units of a group.  C B^T once (128 columns of TMEM), then a unit at a time: the pairs'
// weights go to shared memory as the operand M, C H_in and M x to 64 columns each.  What a unit needs of the next is
// on its way as soon as its products are done.  Bound by a unit's chain (loads, weights, product, output: 5 us, three
// CTA barriers) with two CTAs an SM, half of the issue slots in use: shared memory and TMEM have no room for a third.
// 2 x 2,048 tokens of 128 heads: 74 us.  Exponentials a block in place of a pair on the diagonal, and L2 prefetches of
// the next unit, change nothing.
constexpr uint32_t kOutM = kTile128, kOutX = 2 * kTile128, kOutH = kOutX + kTile64, kOutRec = kOutH + kTile64, kRecBytes = 4 * Q * 4,
                   kOutTop = kOutRec + 2 * kRecBytes, kOutBar = kOutTop + 2 * Q * 4, kOutSmem = kOutBar + 32;

template <typename T, bool TILED>
__global__ void __launch_bounds__(kThreads, 2) out_kernel(const SelectiveParams P, const Space W, int per) {
  using X = typename std::conditional<TILED, __half, T>::type;
  constexpr bool kScaled = std::is_same<X, __half>::value;
  extern __shared__ __align__(1024) unsigned char smem[];
  const uint32_t base = smem_u32(smem);
  float* tops = reinterpret_cast<float*>(smem + kOutTop);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kOutBar);              // tensor cores, tiles, units
  const int c = blockIdx.x, b = blockIdx.z;
  const int gunits = W.units / P.groups, g = blockIdx.y / W.splits;
  const int u0 = g * gunits + (blockIdx.y % W.splits) * per, u1 = min(u0 + per, (g + 1) * gunits);
  const int len = tokens_of(P, b), rows = min(Q, len - c * Q), out_rows = min(Q, P.length - c * Q);
  const int row = threadIdx.x & 127, half = threadIdx.x >> 7, quad = threadIdx.x >> 5 & 3;
  T* y = reinterpret_cast<T*>(P.y) + (long long)b * P.y_sb + (long long)c * Q * P.y_st;
  launch_dependents();
  if (rows <= 0) {                                       // behind the sequence's end
    for (int u = u0; u < u1; ++u) {
      const int h = u / W.ptiles, p0 = (u % W.ptiles) * TP, cols = min(TP, P.dim - p0);
      for (int i = threadIdx.x; i < out_rows * cols; i += kThreads)
        y[(long long)(i / cols) * P.y_st + (long long)h * P.dim + p0 + i % cols] = from_f32<T>(0.f);
    }
    wait_for_launch();
    return;
  }
  const bool has_state = c > 0 || P.state_in;
  const long long bc = (long long)b * W.nc + c, tile_at = bc * P.groups + g;
  const T* xc = reinterpret_cast<const T*>(P.x) + (long long)b * P.x_sb + (long long)c * Q * P.x_st;
  const uint32_t tmem = tensor_begin<256>(bars, 3, reinterpret_cast<uint32_t*>(smem + kOutBar + 24));
  wait_for_launch();
  Gate done{smem_u32(bars), 0}, tiles{smem_u32(bars + 1), 0}, unit{smem_u32(bars + 2), 0};
  bool ok = true;
  auto load_unit = [&](int u) {                          // state and record (one thread), tokens (all)
    const int h = u / W.ptiles, p0 = (u % W.ptiles) * TP, cols = min(TP, P.dim - p0);
    if (threadIdx.x == 0) {
      mbar_expect_tx(unit.bar, kRecBytes + (has_state ? kTile64 : 0) + (TILED ? kTile64 : 0));
      bulk_load(base + kOutRec + ((u - u0) & 1) * kRecBytes, W.rec + (((long long)b * P.heads + h) * W.nc + c) * (kRecord * Q), kRecBytes, unit.bar);
      if (has_state) bulk_load(base + kOutH, W.h + (bc * W.units + u) * (2 * kN * TP), kTile64, unit.bar);
    }
    if constexpr (TILED) {
      if (threadIdx.x == 0) bulk_load(base + kOutX, W.xt + (bc * W.units + u) * (Q * TP), kTile64, unit.bar);
    } else {
      const T* p = xc + (long long)h * P.dim + p0;
      load_tile<T>(base + kOutX, p, P.x_st, rows, cols, vector_ok(p, P.x_st, 0, cols));
      cp_commit();
    }
  };
  if (threadIdx.x == 0) {
    mbar_expect_tx(tiles.bar, 2 * kTile128);
    bulk_load(base, W.ct + tile_at * (Q * kN), kTile128, tiles.bar);
    bulk_load(base + kOutM, W.bt + tile_at * (Q * kN), kTile128, tiles.bar);
  }
  load_unit(u0);
  const float cback = W.cback[tile_at], both_back = cback * W.bback[tile_at];
  const uint32_t lanes = tmem + ((uint32_t)quad << 21);
  if (threadIdx.x == 0) {
    tiles.wait(ok, P.err);
    tc_fence_after();
    if (ok) {
      mma<kK, kK>(tmem, base, base + kOutM, idesc<__half>(Q, false, false), 8, false);
      umma_commit(done.bar);
    }
  }
  done.wait(ok, P.err);
  tc_fence_after();
  float top = 0.f;
  if (kScaled) {                                         // the largest |C_t . B_s| of my row's pairs
    uint32_t m = 0;
    for (int cb = half; cb <= quad; cb += 2) {
      uint32_t r[32];
      tmem_ld32(lanes + cb * 32, r);
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (cb * 32 + i <= row) m = max(m, r[i] & 0x7fffffffu);
    }
    tops[half * Q + row] = __uint_as_float(m);
    __syncthreads();
    top = fmaxf(tops[row], tops[Q + row]);
  }
  for (int cb = half; cb < 4; cb += 2)                   // pairs above the diagonal weigh nothing, for every unit
    if (cb > quad)
      for (int k = 0; k < 4; ++k) sts16(base + kOutM + piece2(row, cb * 4 + k), make_uint4(0, 0, 0, 0));

  for (int u = u0; u < u1; ++u) {
    const int h = u / W.ptiles, p0 = (u % W.ptiles) * TP, cols = min(TP, P.dim - p0);
    const float* rec = reinterpret_cast<const float*>(smem + kOutRec + ((u - u0) & 1) * kRecBytes);
    if constexpr (!TILED) {
      cp_wait<0>();
      fence_async();
    }
    unit.wait(ok, P.err);
    __syncthreads();
    if (threadIdx.x == 0 && has_state && ok) {
      tc_fence_after();
      mma<kK, kPlaneP>(tmem + 128, base, base + kOutH, idesc<__half>(TP, false, true), 8, false);
    }
    const float lh = rec[Q + row], ll = rec[2 * Q + row];
    uint4 x[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = lds16(base + kOutX + piece(row, half * 4 + j));
    float2 sc = make_float2(kWeightThere, kWeightBack);
    if (kScaled) sc = scale_of(__float_as_uint(top * W.smax[((long long)b * P.heads + h) * W.nc + c]) & 0x7fffffffu);
    for (int cb = half; cb <= quad; cb += 2) {
      uint32_t r[32];
      tmem_ld32(lanes + cb * 32, r);
      if (cb < quad) {
        // a block of earlier tokens: the decay to the block's end and from there on are both at most 1
        const float from = ex2((lh - rec[Q + cb * 32 + 31]) + (ll - rec[2 * Q + cb * 32 + 31])) * sc.x;
        const float4* until = reinterpret_cast<const float4*>(rec + 3 * Q) + cb * 8;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          Eight f;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float4 v = until[k * 2 + e];
            f.v[2 * e] = mul2(mul2(words2(r[k * 8 + 4 * e], r[k * 8 + 4 * e + 1]), pair(from)), make_float2(v.x, v.y));
            f.v[2 * e + 1] = mul2(mul2(words2(r[k * 8 + 4 * e + 2], r[k * 8 + 4 * e + 3]), pair(from)), make_float2(v.z, v.w));
          }
          sts16(base + kOutM + piece2(row, cb * 4 + k), pack8<X>(f));
        }
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          Eight f;
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            const int col = cb * 32 + k * 8 + e;
            const float2 sv = *reinterpret_cast<const float2*>(rec + col), hv = *reinterpret_cast<const float2*>(rec + Q + col),
                         lv = *reinterpret_cast<const float2*>(rec + 2 * Q + col);
            const float2 gap = add2(sub2(pair(lh), hv), sub2(pair(ll), lv));
            float2 v = mul2(mul2(make_float2(ex2(gap.x), ex2(gap.y)), sv), words2(r[k * 8 + e], r[k * 8 + e + 1]));
            v = mul2(v, pair(sc.x));
            f.v[e >> 1] = make_float2(col <= row ? v.x : 0.f, col + 1 <= row ? v.y : 0.f);
          }
          sts16(base + kOutM + piece2(row, cb * 4 + k), pack8<X>(f));
        }
      }
    }
    if (quad == 0 && half == 1)                          // where the output of the unit before was laid out
      for (int k = 0; k < 4; ++k) sts16(base + kOutM + piece2(row, 4 + k), make_uint4(0, 0, 0, 0));
    tc_fence_before();
    fence_async();
    __syncthreads();
    if (threadIdx.x == 0 && ok) {
      tc_fence_after();
      mma<kK, kMn>(tmem + 192, base + kOutM, base + kOutX, idesc<X>(TP, false, true), 8, false);
      umma_commit(done.bar);
    }
    const float xb = TILED ? W.xback[bc * W.units + u] : 1.f, d = number(P.D, P.d_type, h) * xb;
    const float carry = has_state ? ex2(lh + ll) * W.hs[bc * W.units + u].x * cback : 0.f, mixed = sc.y * both_back * xb;
    done.wait(ok, P.err);
    tc_fence_after();
    if (u + 1 < u1) load_unit(u + 1);
    uint32_t y0[32], y1[32];
    if (has_state) tmem_ld32_nowait(lanes + 128 + half * 32, y0);
    tmem_ld32(lanes + 192 + half * 32, y1);
    if (has_state) settle(y0);
    tc_fence_before();
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      Eight f = mul8(unpack8<X>(x[j]), d);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        f.v[e] = fma2(words2(y1[j * 8 + 2 * e], y1[j * 8 + 2 * e + 1]), pair(mixed), f.v[e]);
        if (has_state) f.v[e] = fma2(words2(y0[j * 8 + 2 * e], y0[j * 8 + 2 * e + 1]), pair(carry), f.v[e]);
      }
      sts16(base + kOutM + piece(row, half * 4 + j), row < rows ? pack8<T>(f) : make_uint4(0, 0, 0, 0));
    }
    __syncthreads();
    T* out = y + (long long)h * P.dim + p0;
    store_tile<T>(out, P.y_st, base + kOutM, out_rows, cols, vector_ok(out, P.y_st, 0, cols));
  }
  tensor_end<256>(tmem, ok);
}

// ---------------------------------------------------------------- gradients by chunk and group
// One CTA: a chunk and some units of a group, tokens s as rows.  TMEM: B C^T (128 columns), a work area (128), and the
// sums over the units of what reaches C and B through the states (128 each).  A unit takes three steps:
//   1. G B_s and H C_t (64 columns each): the states' part of x's gradient, and q_t = exp(l_t) dy_t . H C_t and
//      r_s = exp(l_end - l_s) x_s . G B_s, from states with their remainders: the gradients of A, dt and the bias, which
//      are 32-bit sums, hang on them.
//   2. x_s . dy_t (128 columns), and the units' sums for C and B on the tensor cores.  The pairs' weights give the
//      operand of step 3, the group's sum of s_s exp(l_t - l_s) (dy_t . x_s), and its products with C_t . B_s summed
//      by row and by column.
//   3. the pairs' part of x's gradient; prefix and suffix sums over the tokens give the gradient of A s.
// After the last unit the group's sum gives the pairs' part of dB and dC in two products.
// Bound by a unit's chain of three products and the barriers between them (four; they are the first stall), with one CTA an
// SM: its shared memory and its 512 columns are full.  35% of the issue slots, 18% of memory.  2 x 2,048 tokens of 128
// heads: 325 us (32 chunks x 8 groups, 16 units each).  Value and remainder side by side in
// one product of 128 columns, as in state_pass_kernel, cost the overlap of a unit with the one before (345 us).
constexpr uint32_t kGRecBytes = kRecord * Q * 4;
constexpr uint32_t kGB = 0, kGC = kTile128, kGX = 2 * kTile128, kGY = kGX + kTile64, kGHigh = kGY + 2 * kTile64,
                   kGLow = kGHigh + 2 * kTile64, kGM = kGLow + 2 * kTile64, kGRec = kGM + kTile128, kGRow = kGRec + 2 * kGRecBytes,
                   kGCol = kGRow + 13 * Q * 4, kGRed = kGCol + 4 * Q * 4, kGBar = kGRed + 64 * 4, kGradSmem = kGBar + 48;
constexpr int kGradThreads = 512;                  // four threads a token: sixteen warps hide each other's waits

// Sums over a warp's lanes of e[column], for column = lane / 2.
__device__ __forceinline__ float column_sums(float (&e)[16], int lane) {
#pragma unroll
  for (int o = 8; o; o >>= 1) {
    const bool up = lane & (2 * o);
#pragma unroll
    for (int i = 0; i < o; ++i) {
      const float send = up ? e[i] : e[i + o], keep = up ? e[i + o] : e[i];
      e[i] = keep + __shfl_xor_sync(0xffffffffu, send, 2 * o);
    }
  }
  return e[0] + __shfl_xor_sync(0xffffffffu, e[0], 1);
}

template <typename T, bool TILED>
__global__ void __launch_bounds__(kGradThreads, 1) grad_kernel(const SelectiveParams P, const Space W, int per) {
  using X = typename std::conditional<TILED, __half, T>::type;
  using G = typename std::conditional<TILED, float, T>::type;    // of dx, dB and dC
  constexpr bool kScaled = std::is_same<X, __half>::value;
  extern __shared__ __align__(1024) unsigned char smem[];
  const uint32_t base = smem_u32(smem);
  float* rpairs = reinterpret_cast<float*>(smem + kGRow);        // [4][Q] each: r by pairs, r by states, q by states; [Q]: r by the token itself
  float *rstate = rpairs + 4 * Q, *qstate = rpairs + 8 * Q, *rself = rpairs + 12 * Q;
  float* qpairs = reinterpret_cast<float*>(smem + kGCol);        // [4][Q]
  float* red = reinterpret_cast<float*>(smem + kGRed);           // [16] each: <G, H>, x . dy, pairs' time, maxima
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kGBar);    // tensor cores, tiles, values, remainders
  const int c = blockIdx.x, b = blockIdx.z;
  const int gunits = W.units / P.groups, g = blockIdx.y / W.splits, split = blockIdx.y % W.splits;
  const int u0 = g * gunits + split * per, u1 = min(u0 + per, (g + 1) * gunits);
  const int len = tokens_of(P, b), rows = min(Q, len - c * Q), out_rows = min(Q, P.length - c * Q);
  const int row = threadIdx.x & 127, part = threadIdx.x >> 7, warp = threadIdx.x >> 5, quad = warp & 3, lane = threadIdx.x & 31;
  const long long bc = (long long)b * W.nc + c, tile_at = bc * P.groups + g;
  // Pointers are made where they are used: registers are what this kernel is short of.
  auto dx_at = [&](int h, int p0) { return reinterpret_cast<G*>(P.dx) + b * P.dx_sb + (long long)c * Q * P.dx_st + (long long)h * P.dim + p0; };
  auto group_at = [&](void* p) { return reinterpret_cast<G*>(p) + b * P.dg_sb + (long long)c * Q * P.dg_st + g * kN; };
  launch_dependents();
  if (rows <= 0) {                                       // behind the sequence's end
    for (int u = u0; u < u1; ++u) {
      const int h = u / W.ptiles, p0 = (u % W.ptiles) * TP, cols = min(TP, P.dim - p0);
      for (int i = threadIdx.x; i < out_rows * cols; i += kGradThreads)
        dx_at(h, p0)[(long long)(i / cols) * P.dx_st + i % cols] = from_f32<G>(0.f);
      if (threadIdx.x == 0) W.unit_sums[bc * W.units + u] = make_float2(0.f, 0.f);
      if (W.ptiles == 1) {
        if (threadIdx.x < 4) W.bias_sums[(bc * P.heads + h) * 4 + threadIdx.x] = 0.f;
        T* ddt = reinterpret_cast<T*>(P.ddt) + ((long long)b * P.length + (long long)c * Q) * P.heads + h;
        for (int i = threadIdx.x; i < out_rows; i += kGradThreads) ddt[(long long)i * P.heads] = from_f32<T>(0.f);
      }
    }
    if (W.splits == 1)
      for (int i = threadIdx.x; i < out_rows * kN; i += kGradThreads)
        group_at(P.dB)[(long long)(i / kN) * P.dg_st + i % kN] = group_at(P.dC)[(long long)(i / kN) * P.dg_st + i % kN] = from_f32<G>(0.f);
    wait_for_launch();
    return;
  }
  const bool has_h = c > 0 || P.state_in, has_g = (c + 1) * Q < len || P.dstate_out;
  const uint32_t tmem = tensor_begin<512>(bars, 4, reinterpret_cast<uint32_t*>(smem + kGBar + 32));
  const uint32_t lanes = tmem + ((uint32_t)quad << 21), work = tmem + 128, sum_c = tmem + 256, sum_b = tmem + 384;
  wait_for_launch();
  Gate done{smem_u32(bars), 0}, tiles{smem_u32(bars + 1), 0}, high{smem_u32(bars + 2), 0}, low{smem_u32(bars + 3), 0};
  bool ok = true;
  // One thread: the record and the states' values of a unit, and their remainders.  H lies at 0, G 16,384 bytes on.
  auto load_high = [&](int u) {
    const long long at = (bc * W.units + u) * (2 * kN * TP);
    mbar_expect_tx(high.bar, kGRecBytes + ((int)has_h + (int)has_g + (TILED ? 2 : 0)) * kTile64);
    bulk_load(base + kGRec + ((u - u0) & 1) * kGRecBytes, W.rec + (((long long)b * P.heads + u / W.ptiles) * W.nc + c) * (kRecord * Q), kGRecBytes,
              high.bar);
    if (TILED) {
      bulk_load(base + kGX, W.xt + (bc * W.units + u) * (Q * TP), kTile64, high.bar);
      bulk_load(base + kGY + ((u - u0) & 1) * kTile64, W.yt + (bc * W.units + u) * (Q * TP), kTile64, high.bar);
    }
    if (has_h) bulk_load(base + kGHigh, W.h + at, kTile64, high.bar);
    if (has_g) bulk_load(base + kGHigh + kTile64, W.g + at, kTile64, high.bar);
  };
  auto load_low = [&](int u) {
    if (!has_h && !has_g) return;
    const long long at = (bc * W.units + u) * (2 * kN * TP) + kN * TP;
    mbar_expect_tx(low.bar, ((int)has_h + (int)has_g) * kTile64);
    if (has_h) bulk_load(base + kGLow, W.h + at, kTile64, low.bar);
    if (has_g) bulk_load(base + kGLow + kTile64, W.g + at, kTile64, low.bar);
  };
  auto load_x = [&](int u) {
    if constexpr (TILED) return;
    const int h = u / W.ptiles, p0 = (u % W.ptiles) * TP, cols = min(TP, P.dim - p0);
    const T* p = reinterpret_cast<const T*>(P.x) + b * P.x_sb + (long long)c * Q * P.x_st + (long long)h * P.dim + p0;
    load_tile<T, kGradThreads>(base + kGX, p, P.x_st, rows, cols, vector_ok(p, P.x_st, 0, cols));
  };
  auto load_y = [&](int u) {
    if constexpr (TILED) return;
    const int h = u / W.ptiles, p0 = (u % W.ptiles) * TP, cols = min(TP, P.dim - p0);
    const T* p = reinterpret_cast<const T*>(P.dy) + b * P.dy_sb + (long long)c * Q * P.dy_st + (long long)h * P.dim + p0;
    load_tile<T, kGradThreads>(base + kGY + ((u - u0) & 1) * kTile64, p, P.dy_st, rows, cols, vector_ok(p, P.dy_st, 0, cols));
  };
  if (threadIdx.x == 0) {
    mbar_expect_tx(tiles.bar, 2 * kTile128);
    bulk_load(base + kGB, W.bt + tile_at * (Q * kN), kTile128, tiles.bar);
    bulk_load(base + kGC, W.ct + tile_at * (Q * kN), kTile128, tiles.bar);
    load_high(u0);
    load_low(u0);
  }
  load_x(u0);
  load_y(u0);
  cp_commit();
  // units' sums for C and B share a scale: that of the largest product of a state's and its tokens' scales.  A head whose
  // state or tokens are zero has none: it would take the bits of heads with small gradients.
  float cscale = 0.f, bscale = 0.f;
  if (has_h || has_g)
    for (int u = u0; u < u1; ++u) {
      const float2 hs = W.hs[bc * W.units + u], gs = W.gs[bc * W.units + u];
      cscale = fmaxf(cscale, hs.x * gs.y);
      bscale = fmaxf(bscale, gs.x * hs.y);
    }
  if (cscale == 0.f) cscale = 1.f;                       // zeros, or products that no number here can hold
  if (bscale == 0.f) bscale = 1.f;
  const float bback = W.bback[tile_at], cback = W.cback[tile_at], both_back = bback * cback;
  if (threadIdx.x == 0) {
    tiles.wait(ok, P.err);
    tc_fence_after();
    if (ok) {
      mma<kK, kK>(tmem, base + kGB, base + kGC, idesc<__half>(Q, false, false), 8, false);
      umma_commit(done.bar);
    }
  }
  done.wait(ok, P.err);
  tc_fence_after();
  float2 sc = make_float2(kWeightThere, kWeightBack);
  if (kScaled) {                                         // by the largest |B_s . C_t| of my row's pairs
    uint32_t m = 0;
    if (part >= quad) {
      uint32_t r[32];
      tmem_ld32(lanes + part * 32, r);
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (part * 32 + i >= row) m = max(m, r[i] & 0x7fffffffu);
    }
    rpairs[part * Q + row] = __uint_as_float(m);
    __syncthreads();
    sc = scale_of(__float_as_uint(fmaxf(fmaxf(rpairs[row], rpairs[Q + row]), fmaxf(rpairs[2 * Q + row], rpairs[3 * Q + row]))));
  }
  float2 ds[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) ds[i] = make_float2(0.f, 0.f);

  for (int u = u0; u < u1; ++u) {
    const int h = u / W.ptiles, p0 = (u % W.ptiles) * TP, cols = min(TP, P.dim - p0);
    const float* rec = reinterpret_cast<const float*>(smem + kGRec + ((u - u0) & 1) * kGRecBytes);
    const uint32_t ytile = base + kGY + ((u - u0) & 1) * kTile64;
    cp_wait<0>();
    fence_async();
    high.wait(ok, P.err);
    if (has_h || has_g) low.wait(ok, P.err);
    __syncthreads();
    // step 1
    if (threadIdx.x == 0 && (has_h || has_g) && ok) {
      tc_fence_after();
      if (has_g) {
        mma<kK, kPlaneP>(work, base + kGB, base + kGHigh + kTile64, idesc<__half>(TP, false, true), 8, false);
        mma<kK, kPlaneP>(work, base + kGB, base + kGLow + kTile64, idesc<__half>(TP, false, true), 8, true);
      }
      if (has_h) {
        mma<kK, kPlaneP>(work + 64, base + kGC, base + kGHigh, idesc<__half>(TP, false, true), 8, false);
        mma<kK, kPlaneP>(work + 64, base + kGC, base + kGLow, idesc<__half>(TP, false, true), 8, true);
      }
      umma_commit(done.bar);
    }
    const float xb = TILED ? W.xback[bc * W.units + u] : 1.f, yb = TILED ? W.yback[bc * W.units + u] : 1.f, xy = xb * yb;
    const float s = rec[row], lh = rec[Q + row], ll = rec[2 * Q + row], eh = rec[2 * Q - 1], el = rec[3 * Q - 1];
    float2 hs = make_float2(1.f, 1.f), gs = make_float2(1.f, 1.f);
    if (has_h || has_g) { hs = W.hs[bc * W.units + u]; gs = W.gs[bc * W.units + u]; }
    const float from_in = ex2(lh + ll), to_end = ex2((eh - lh) + (el - ll));
    const float wy = has_h && gs.y != 0.f ? from_in * (hs.x / cscale) * yb : 0.f, wx = has_g && hs.y != 0.f ? s * to_end * (gs.x / bscale) * xb : 0.f;
    float2 gh2 = make_float2(0.f, 0.f);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint32_t at = piece(row, part * 2 + j), plane = (uint32_t)((part * 2 + j) * kN + row) * 16;
      if (has_h) sts16(base + kGM + at, pack8<__half>(mul8(unpack8<X>(lds16(ytile + at)), wy)));
      if (has_g) sts16(base + kGM + kTile64 + at, pack8<__half>(mul8(unpack8<X>(lds16(base + kGX + at)), wx)));
      if (has_h && has_g) {                              // my row of the states: <G, H>
        const Eight h1 = unpack8<__half>(lds16(base + kGHigh + plane)), h2 = unpack8<__half>(lds16(base + kGLow + plane));
        const Eight g1 = unpack8<__half>(lds16(base + kGHigh + kTile64 + plane)), g2 = unpack8<__half>(lds16(base + kGLow + kTile64 + plane));
#pragma unroll
        for (int e = 0; e < 4; ++e) gh2 = fma2(add2(h1.v[e], h2.v[e]), add2(g1.v[e], g2.v[e]), gh2);
      }
    }
    float gh = gh2.x + gh2.y;
    gh = warp_sum(gh);
    if (lane == 0) red[warp] = gh;
    fence_async();
    float2 dxi[8];
    float r_part = 0.f, q_part = 0.f;
    if (has_h || has_g) {
      done.wait(ok, P.err);
      tc_fence_after();
      uint32_t r[16];
      if (has_g) {
        tmem_ld16(lanes + 128 + part * 16, r);
        const float f = to_end * gs.x * bback;
        float2 sum = make_float2(0.f, 0.f);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const Eight x = unpack8<X>(lds16(base + kGX + piece(row, part * 2 + j)));
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            dxi[j * 4 + e] = mul2(words2(r[j * 8 + 2 * e], r[j * 8 + 2 * e + 1]), pair(f));
            sum = fma2(dxi[j * 4 + e], x.v[e], sum);
          }
        }
        r_part = (sum.x + sum.y) * xb;
      }
      if (has_h) {
        tmem_ld16(lanes + 192 + part * 16, r);
        const float f = from_in * hs.x * cback;
        float2 sum = make_float2(0.f, 0.f);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const Eight y = unpack8<X>(lds16(ytile + piece(row, part * 2 + j)));
#pragma unroll
          for (int e = 0; e < 4; ++e) sum = fma2(mul2(words2(r[j * 8 + 2 * e], r[j * 8 + 2 * e + 1]), pair(f)), y.v[e], sum);
        }
        q_part = (sum.x + sum.y) * yb;
      }
      tc_fence_before();
    }
    rstate[part * Q + row] = r_part;
    qstate[part * Q + row] = q_part;
    if (!has_g)
#pragma unroll
      for (int i = 0; i < 8; ++i) dxi[i] = make_float2(0.f, 0.f);
    __syncthreads();
    // step 2
    if (threadIdx.x == 0) {
      if (u + 1 < u1) load_low(u + 1);
      if (ok) {
        tc_fence_after();
        mma<kK, kK>(work, base + kGX, ytile, idesc<X>(Q, false, false), 4, false);
        if (has_h) mma<kK, kPlaneN>(sum_c, base + kGM, base + kGHigh, idesc<__half>(kN, false, false), 4, u > u0);
        if (has_g) mma<kK, kPlaneN>(sum_b, base + kGM + kTile64, base + kGHigh + kTile64, idesc<__half>(kN, false, false), 4, u > u0);
        umma_commit(done.bar);
      }
    }
    if (u + 1 < u1) { load_y(u + 1); cp_commit(); }
    done.wait(ok, P.err);
    tc_fence_after();
    if (u + 1 < u1) {
      if (threadIdx.x == 0) load_high(u + 1);
      load_x(u + 1);
      cp_commit();
    }
    float r_sum = 0.f, diag = 0.f, pair_time = 0.f;
    const float one_back = sc.y * both_back * xy, sb = s * one_back, sxy = s * xy;   // of a pair's weight, and of a pair without C . B
    const int cb = part;
    if (cb >= quad) {
      float2 rs2 = make_float2(0.f, 0.f), time2 = make_float2(0.f, 0.f);
      const bool later = cb > quad;
      // a block of later tokens: the decay to its beginning and from there on are both at most 1
      const float th = later ? rec[Q + cb * 32 - 1] - lh : 0.f, tl = later ? rec[2 * Q + cb * 32 - 1] - ll : 0.f, to_block = ex2(th + tl);
      const float ds_in = sxy * to_block, mine = to_block * sc.x;
#pragma unroll
      for (int part16 = 0; part16 < 2; ++part16) {       // sixteen columns in registers at a time
        uint32_t r[16], d[16];
        tmem_ld16_nowait(lanes + cb * 32 + part16 * 16, r);
        tmem_ld16(lanes + 128 + cb * 32 + part16 * 16, d);
        settle(r);
        float e[16];
        if (later) {
          const float4 *since = reinterpret_cast<const float4*>(rec + 4 * Q) + cb * 8 + part16 * 4;
          const float4 *in_block = reinterpret_cast<const float4*>(rec + 5 * Q) + cb * 8 + part16 * 4;
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            Eight f;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const float4 w4 = since[j * 2 + i], l4 = in_block[j * 2 + i];
#pragma unroll
              for (int o = 0; o < 2; ++o) {
                const int q = j * 8 + i * 4 + o * 2, at = part16 * 16 + q;
                const float2 w = o ? make_float2(w4.z, w4.w) : make_float2(w4.x, w4.y), l = o ? make_float2(l4.z, l4.w) : make_float2(l4.x, l4.y);
                const float2 dm = words2(d[q], d[q + 1]), m = mul2(words2(r[q], r[q + 1]), w);
                ds[at >> 1] = fma2(mul2(dm, w), pair(ds_in), ds[at >> 1]);
                f.v[i * 2 + o] = mul2(m, pair(mine));
                const float2 both = mul2(mul2(f.v[i * 2 + o], dm), pair(sb));
                rs2 = add2(rs2, both);
                time2 = fma2(both, l, time2);
                e[q] = both.x;
                e[q + 1] = both.y;
              }
            }
            sts16(base + kGM + piece2(row, cb * 4 + part16 * 2 + j), pack8<X>(f));
          }
        } else {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            Eight f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int q = j * 8 + i * 2, at = part16 * 16 + q, t = cb * 32 + at;
              const float2 hv = *reinterpret_cast<const float2*>(rec + Q + t), lv = *reinterpret_cast<const float2*>(rec + 2 * Q + t);
              float2 gap = add2(sub2(hv, pair(lh)), sub2(lv, pair(ll)));
              if (t < row) gap.x = 0.f;
              if (t + 1 < row) gap.y = 0.f;
              float2 w = make_float2(ex2(gap.x), ex2(gap.y));
              if (t < row) w.x = 0.f;                    // pairs under the diagonal weigh nothing
              if (t + 1 < row) w.y = 0.f;
              const float2 dm = words2(d[q], d[q + 1]), m = mul2(words2(r[q], r[q + 1]), w);
              ds[at >> 1] = fma2(pair(sxy), mul2(dm, w), ds[at >> 1]);
              f.v[i] = mul2(m, pair(sc.x));
              float2 both = mul2(f.v[i], dm);
              if (t == row) { diag = dm.x; rself[row] = both.x * one_back; both.x = 0.f; }
              if (t + 1 == row) { diag = dm.y; rself[row] = both.y * one_back; both.y = 0.f; }
              both = mul2(both, pair(sb));               // no decay between a token and itself: kept out of the sums
              rs2 = add2(rs2, both);
              time2 = fma2(both, gap, time2);
              e[q] = both.x;
              e[q + 1] = both.y;
            }
            sts16(base + kGM + piece2(row, cb * 4 + part16 * 2 + j), pack8<X>(f));
          }
        }
        const float column = column_sums(e, lane);
        if (!(lane & 1)) qpairs[quad * Q + cb * 32 + part16 * 16 + (lane >> 1)] = column;
      }
      r_sum = rs2.x + rs2.y;                             // by s: the row's own factor
      pair_time = (time2.x + time2.y) + r_sum * (th + tl);
    } else {
      for (int j = 0; j < 4; ++j) sts16(base + kGM + piece2(row, cb * 4 + j), make_uint4(0, 0, 0, 0));
      qpairs[quad * Q + cb * 32 + lane] = 0.f;
    }
    rpairs[part * Q + row] = r_sum;
    diag = warp_sum(diag * xy);
    pair_time = warp_sum(pair_time);
    if (lane == 0) { red[16 + warp] = diag; red[32 + warp] = pair_time; }
    tc_fence_before();
    fence_async();
    __syncthreads();
    // step 3
    if (threadIdx.x == 0 && ok) {
      tc_fence_after();
      mma<kK, kMn>(work, base + kGM, ytile, idesc<X>(TP, false, true), 8, false);
      umma_commit(done.bar);
    }
    if (warp >= 12) {                                    // four warps, a token a lane
      const int t = quad * 32 + lane;
      const float rate = P.A[h];
      const auto four = [&](const float* v) { return (v[t] + v[Q + t]) + (v[2 * Q + t] + v[3 * Q + t]); };
      const float st = rec[t], rp = four(rpairs), rs = four(rstate), qs = four(qstate), lt = rec[Q + t], lt2 = rec[2 * Q + t];
      const float r = (st > 0.f ? __fdividef(rp, st) : 0.f) + rs + rself[t];   // rp is by s, as the columns' sums are
      const float a = four(qpairs) + qs - rp, bs = st * rs;
      float after = a, before = bs;                      // sums from this token on, and up to it
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const float va = __shfl_down_sync(0xffffffffu, after, o), vb = __shfl_up_sync(0xffffffffu, before, o);
        if (lane + o < 32) after += va;
        if (lane >= o) before += vb;
      }
      const float time = warp_sum(qs * (lt + lt2) + bs * ((eh - lt) + (el - lt2)));
      if (lane == 0) { red[48 + quad] = after; red[56 + quad] = time; }
      if (lane == 31) red[52 + quad] = before;
      const float through = warp_sum(lane < 16 ? red[lane] : 0.f) * ex2(eh + el) * (hs.x * gs.x);
      asm volatile("bar.sync 1, 128;" ::: "memory");
      before -= bs;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (k > quad) after += red[48 + k];
        if (k < quad) before += red[52 + k];
      }
      const float all = after + before + through;        // gradient of A s
      if (W.ptiles == 1) {
        const float v = t < rows ? (rate * all + r) * rec[6 * Q + t] : 0.f;
        if (t < out_rows) reinterpret_cast<T*>(P.ddt)[((long long)b * P.length + (long long)c * Q + t) * P.heads + h] = from_f32<T>(v);
        const float sum_bias = warp_sum(v);
        if (lane == 0) W.bias_sums[(bc * P.heads + h) * 4 + quad] = sum_bias;
      } else {
        W.parts[((long long)b * W.units + u) * W.lp + (long long)c * Q + t] = make_float2(all, r);
      }
      if (warp == 15) {
        // A's gradient: each contribution by the time that A works on it, which l tells; no differences of large sums
        const float dd = warp_sum(lane < 16 ? red[16 + lane] : 0.f);
        float da = warp_sum(lane < 16 ? red[32 + lane] : 0.f);
        da += ((red[56] + red[57]) + (red[58] + red[59])) + through * (eh + el);
        if (lane == 0) W.unit_sums[bc * W.units + u] = make_float2(dd, __fdividef(da, decay_rate_f32(rate)));
      }
    }
    const float dskip = number(P.D, P.d_type, h) * yb, mixed = sc.y * both_back * yb;
    done.wait(ok, P.err);
    tc_fence_after();
    {
      uint32_t r[16];
      tmem_ld16(lanes + 128 + part * 16, r);
      tc_fence_before();
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint32_t at = piece(row, part * 2 + j);
        Eight f = mul8(unpack8<X>(lds16(ytile + at)), dskip);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          f.v[e] = fma2(fma2(words2(r[j * 8 + 2 * e], r[j * 8 + 2 * e + 1]), pair(mixed), dxi[j * 4 + e]), pair(s), f.v[e]);
        if (row >= rows) f = {};
        if constexpr (TILED) {
#pragma unroll
          for (int e = 0; e < 2; ++e)
            sts16(base + kGM + piece_f32(row, part * 4 + j * 2 + e), make_uint4(__float_as_uint(f.v[2 * e].x), __float_as_uint(f.v[2 * e].y),
                                                                                __float_as_uint(f.v[2 * e + 1].x), __float_as_uint(f.v[2 * e + 1].y)));
        } else {
          sts16(base + kGM + at, pack8<T>(f));
        }
      }
    }
    __syncthreads();
    G* out = dx_at(h, p0);
    if constexpr (TILED) store_tile<kGradThreads>(out, P.dx_st, base + kGM, out_rows, cols, true);
    else store_tile<T, kGradThreads>(out, P.dx_st, base + kGM, out_rows, cols, vector_ok(out, P.dx_st, 0, cols));
  }
  __syncthreads();

  // the pairs' part of dB and dC
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) top = max(top, max(__float_as_uint(ds[i].x) & 0x7fffffffu, __float_as_uint(ds[i].y) & 0x7fffffffu));
  top = __reduce_max_sync(0xffffffffu, top);
  if (lane == 0) red[48 + warp] = __uint_as_float(top);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 16; ++i) top = max(top, __float_as_uint(red[48 + i]));
  const float2 all = scale_of(top);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    sts16(base + kGM + piece2(row, part * 4 + j), pack8<__half>(mul8({{ds[4 * j], ds[4 * j + 1], ds[4 * j + 2], ds[4 * j + 3]}}, all.x)));
  }
  tc_fence_before();
  fence_async();
  __syncthreads();
  if (threadIdx.x == 0 && ok) {
    tc_fence_after();
    mma<kK, kMn>(work, base + kGM, base + kGC, idesc<__half>(kN, false, true), 8, false);
    mma<kMn, kMn>(tmem, base + kGM, base + kGB, idesc<__half>(kN, true, true), 8, false);
    umma_commit(done.bar);
  }
  done.wait(ok, P.err);
  tc_fence_after();
#pragma unroll
  for (int which = 0; which < 2; ++which) {              // dB, dC
    const uint32_t pairs = lanes + (which ? 0 : 128), states = lanes + (which ? 256 : 384);
    const bool has = which ? has_h : has_g;
    const float back = which ? cscale : bscale, pairs_back = all.y * (which ? bback : cback);
    float* sums = which ? W.pc : W.pb;
    {
      uint32_t r[32], d[32];
      if (has) tmem_ld32_nowait(states + part * 32, d);
      tmem_ld32(pairs + part * 32, r);
      if (has) settle(d);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        Eight f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          f.v[e] = mul2(words2(r[j * 8 + 2 * e], r[j * 8 + 2 * e + 1]), pair(pairs_back));
          if (has) f.v[e] = fma2(words2(d[j * 8 + 2 * e], d[j * 8 + 2 * e + 1]), pair(back), f.v[e]);
          if (row >= rows) f.v[e] = make_float2(0.f, 0.f);
        }
        if (TILED && W.splits == 1) {
          // whole lines a thread, once a CTA: through shared memory they would need twice its room
          if (row < out_rows) {
            float* p = reinterpret_cast<float*>(group_at(which ? P.dC : P.dB)) + (long long)row * P.dg_st + part * 32 + j * 8;
            if (((uintptr_t)p & 15) == 0) {
              *reinterpret_cast<float4*>(p) = make_float4(f.v[0].x, f.v[0].y, f.v[1].x, f.v[1].y);
              *reinterpret_cast<float4*>(p + 4) = make_float4(f.v[2].x, f.v[2].y, f.v[3].x, f.v[3].y);
            } else {
#pragma unroll
              for (int e = 0; e < 4; ++e) { p[2 * e] = f.v[e].x; p[2 * e + 1] = f.v[e].y; }
            }
          }
        } else if (W.splits > 1) {
          float* p = sums + ((((long long)split * P.batch + b) * W.lp + (long long)c * Q + row) * P.groups + g) * kN + part * 32 + j * 8;
          *reinterpret_cast<float4*>(p) = make_float4(f.v[0].x, f.v[0].y, f.v[1].x, f.v[1].y);
          *reinterpret_cast<float4*>(p + 4) = make_float4(f.v[2].x, f.v[2].y, f.v[3].x, f.v[3].y);
        } else {
          sts16(base + (which ? kGHigh : kGM) + piece2(row, part * 4 + j), pack8<T>(f));
        }
      }
    }
  }
  if constexpr (!TILED) {
    if (W.splits == 1) {
      __syncthreads();
      for (int hf = 0; hf < 2; ++hf) {
        T *dB = group_at(P.dB) + hf * 64, *dC = group_at(P.dC) + hf * 64;
        store_tile<T, kGradThreads>(dB, P.dg_st, base + kGM + hf * kTile64, out_rows, 64, vector_ok(dB, P.dg_st, 0, 64));
        store_tile<T, kGradThreads>(dC, P.dg_st, base + kGHigh + hf * kTile64, out_rows, 64, vector_ok(dC, P.dg_st, 0, 64));
      }
    }
  }
  tensor_end<512>(tmem, ok);
}

// ---------------------------------------------------------------- sums behind the gradients
// For heads of more than one unit (grad_kernel does the others itself): one CTA a chunk of eight heads, a warp a head, four
// tokens a lane.  The gradient of dt, and the chunk's sum for the bias.
template <typename T>
__global__ void __launch_bounds__(kThreads) finish_dt_kernel(const SelectiveParams P, const Space W) {
  __shared__ float grad[kPrepHeads][Q + 4];
  launch_dependents();
  wait_for_launch();
  const int c = blockIdx.x, h0 = blockIdx.y * kPrepHeads, b = blockIdx.z, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int h = h0 + warp, rows = min(Q, tokens_of(P, b) - c * Q);
  if (h < P.heads) {
    const long long row = (long long)b * P.heads + h;
    const float rate = P.A[h];
    const float4 slope = *(reinterpret_cast<const float4*>(W.rec + (row * W.nc + c) * (kRecord * Q) + 6 * Q) + lane);
    float out[4] = {0.f, 0.f, 0.f, 0.f};
    if (4 * lane < rows) {
      float4 ga = make_float4(0.f, 0.f, 0.f, 0.f), gs = ga;
      for (int p = 0; p < W.ptiles; ++p) {
        const float4* v = reinterpret_cast<const float4*>(W.parts + ((long long)b * W.units + h * W.ptiles + p) * W.lp + (long long)c * Q + 4 * lane);
        const float4 u = v[0], w = v[1];
        ga.x += u.x; gs.x += u.y; ga.y += u.z; gs.y += u.w;
        ga.z += w.x; gs.z += w.y; ga.w += w.z; gs.w += w.w;
      }
      out[0] = (rate * ga.x + gs.x) * slope.x;
      out[1] = (rate * ga.y + gs.y) * slope.y;
      out[2] = (rate * ga.z + gs.z) * slope.z;
      out[3] = (rate * ga.w + gs.w) * slope.w;
#pragma unroll
      for (int i = 1; i < 4; ++i)
        if (4 * lane + i >= rows) out[i] = 0.f;
    }
    const float db = warp_sum((out[0] + out[1]) + (out[2] + out[3]));
    if (lane < 4) W.bias_sums[(((long long)b * W.nc + c) * P.heads + h) * 4 + lane] = lane ? 0.f : db;
    *reinterpret_cast<float4*>(&grad[warp][4 * lane]) = make_float4(out[0], out[1], out[2], out[3]);
  }
  __syncthreads();
  T* ddt = reinterpret_cast<T*>(P.ddt) + ((long long)b * P.length + (long long)c * Q) * P.heads + h0;
  const int hl = threadIdx.x & 7;
  for (int t = threadIdx.x >> 3; t < Q && c * Q + t < P.length; t += 32)
    if (h0 + hl < P.heads) ddt[(long long)t * P.heads + hl] = from_f32<T>(grad[hl][t]);
}

// The first `head_blocks` CTAs: gradients of A, the bias and D, a warp a head.  The others, where CTAs shared a group's
// units: dB and dC from the splits' sums, four columns a thread.  4 us.
template <typename G>
__global__ void __launch_bounds__(kThreads) finish_kernel(const SelectiveParams P, const Space W, int head_blocks) {
  launch_dependents();
  wait_for_launch();
  if ((int)blockIdx.x < head_blocks) {
    const int h = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (h >= P.heads) return;
    float da = 0.f, db = 0.f, dd = 0.f;
    for (int i = lane; i < P.batch * W.nc; i += 32) {
      const float4 v4 = *reinterpret_cast<const float4*>(W.bias_sums + ((long long)i * P.heads + h) * 4);
      db += (v4.x + v4.y) + (v4.z + v4.w);
      for (int p = 0; p < W.ptiles; ++p) {
        const float2 v = W.unit_sums[(long long)i * W.units + h * W.ptiles + p];
        dd += v.x;
        da += v.y;
      }
    }
    da = warp_sum(da);
    db = warp_sum(db);
    dd = warp_sum(dd);
    if (lane == 0) {
      if (P.dA) P.dA[h] = da;
      if (P.dbias) put_number(P.dbias, P.bias_type, h, db);
      if (P.dD) put_number(P.dD, P.d_type, h, dd);
    }
    return;
  }
  const long long i = (long long)(blockIdx.x - head_blocks) * kThreads + threadIdx.x, width = (long long)P.groups * kN;
  const long long all = (long long)P.batch * P.length * width;
  if (i * 4 >= all) return;
  const long long token = i * 4 / width, b = token / P.length, t = token % P.length;
  const bool in = t < tokens_of(P, (int)b);
  const long long at = (b * W.lp + t) * width + i * 4 % width, step = (long long)P.batch * W.lp * width;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const float* p = which ? W.pc : W.pb;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (in)
      for (int s = 0; s < W.splits; ++s) {
        const float4 a = *reinterpret_cast<const float4*>(p + s * step + at);
        v.x += a.x; v.y += a.y; v.z += a.z; v.w += a.w;
      }
    G* out = reinterpret_cast<G*>(which ? P.dC : P.dB) + b * P.dg_sb + t * P.dg_st + i * 4 % width;
    if constexpr (std::is_same<G, float>::value) {
      if (((uintptr_t)out & 15) == 0) {
        *reinterpret_cast<float4*>(out) = v;
      } else {
        out[0] = v.x; out[1] = v.y; out[2] = v.z; out[3] = v.w;
      }
    } else {
      const uint32_t lo = pack2<G>(v.x, v.y), hi = pack2<G>(v.z, v.w);
      if (((uintptr_t)out & 7) == 0) {
        *reinterpret_cast<uint2*>(out) = make_uint2(lo, hi);
      } else {
        uint16_t* o = reinterpret_cast<uint16_t*>(out);
        o[0] = (uint16_t)lo; o[1] = (uint16_t)(lo >> 16); o[2] = (uint16_t)hi; o[3] = (uint16_t)(hi >> 16);
      }
    }
  }
}

// ---------------------------------------------------------------- one token
// Four neighbouring numbers.
template <typename T> __device__ __forceinline__ float4 four(const T* p, bool vec) {
  if constexpr (std::is_same<T, float>::value) {
    if (vec) return *reinterpret_cast<const float4*>(p);
  } else if (vec) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    const float2 a = unpack2<T>(u.x), b = unpack2<T>(u.y);
    return make_float4(a.x, a.y, b.x, b.y);
  }
  return make_float4(to_f32(p[0]), to_f32(p[1]), to_f32(p[2]), to_f32(p[3]));
}

// A warp takes eight rows of a head's state, four at a time: eight lanes a row, four 16-byte loads a lane.  The state
// does not wait for the kernel before, which may still be writing x, B and C.  Bound by memory: a state is read and written
// once.  64 rows of 128 heads x 64 x 128: 537 MB in 80 us, 6.7 TB/s.
template <typename T, typename X>
__global__ void __launch_bounds__(128) step_kernel(const SelectiveStepParams P) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, h = blockIdx.y, b = blockIdx.z, g = h / (P.heads / P.groups);
  const int l8 = lane & 7, sub = lane >> 3;
  float4* state = reinterpret_cast<float4*>(P.state) + ((long long)b * P.heads + h) * P.dim * 32 + l8;
  float4 now[2][4];
  int row[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    row[k] = blockIdx.x * 32 + warp * 8 + k * 4 + sub;
    if (row[k] < P.dim)
#pragma unroll
      for (int j = 0; j < 4; ++j) now[k][j] = state[(long long)row[k] * 32 + j * 8];
  }
  const float v = to_f32((reinterpret_cast<const T*>(P.dt) + b * P.dt_sb)[h]) + number(P.dt_bias, P.bias_type, h);
  const float s = v <= 20.0f ? log1pf(expf(v)) : v, decay = expf(s * P.A[h]), skip = number(P.D, P.d_type, h);
  const X* Bp = reinterpret_cast<const X*>(P.B) + b * P.b_sb + g * kN + l8 * 4;
  const X* Cp = reinterpret_cast<const X*>(P.C) + b * P.c_sb + g * kN + l8 * 4;
  const X* xp = reinterpret_cast<const X*>(P.x) + b * P.x_sb + (long long)h * P.dim;
  const bool bvec = ((uintptr_t)Bp & (4 * sizeof(X) - 1)) == 0, cvec = ((uintptr_t)Cp & (4 * sizeof(X) - 1)) == 0;
  T* yp = reinterpret_cast<T*>(P.y) + ((long long)b * P.heads + h) * P.dim;
  wait_for_launch();
  float x[2];
  float4 Bv[4], Cv[4];
#pragma unroll
  for (int k = 0; k < 2; ++k) x[k] = row[k] < P.dim ? to_f32(xp[row[k]]) : 0.f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    Bv[j] = four(Bp + j * 32, bvec);
    Cv[j] = four(Cp + j * 32, cvec);
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    float y = 0.f;
    if (row[k] < P.dim) {
      const float u = s * x[k];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float4 n = now[k][j];
        n.x = n.x * decay + u * Bv[j].x; n.y = n.y * decay + u * Bv[j].y;
        n.z = n.z * decay + u * Bv[j].z; n.w = n.w * decay + u * Bv[j].w;
        y += (n.x * Cv[j].x + n.y * Cv[j].y) + (n.z * Cv[j].z + n.w * Cv[j].w);
        state[(long long)row[k] * 32 + j * 8] = n;
      }
    }
    y += __shfl_xor_sync(0xffffffffu, y, 4);
    y += __shfl_xor_sync(0xffffffffu, y, 2);
    y += __shfl_xor_sync(0xffffffffu, y, 1);
    if (l8 == 0 && row[k] < P.dim) yp[row[k]] = from_f32<T>(y + skip * x[k]);
  }
}

// ---------------------------------------------------------------- launches
// Dynamic shared memory of a kernel beyond 48 KB, asked for once a thread and device.
template <auto K> int allow(uint32_t bytes) {
  static thread_local bool done[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return kECuda;
  if (!done[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(K, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e != cudaSuccess) { last_launch_error() = e; return kECuda; }
    done[dev] = true;
  }
  return kOk;
}

// Launches a kernel that begins while the one before it ends: every kernel here waits (wait_for_launch) before it reads
// what earlier ones wrote or ends, so that each of a call's kernels comes after all before it.  The first is launched
// plainly, behind whatever the stream holds.
template <typename... A> int behind(void (*kernel)(A...), dim3 grid, int threads, uint32_t bytes, cudaStream_t st, A... args) {
  cudaLaunchAttribute early{};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t at{};
  at.gridDim = grid;
  at.blockDim = dim3(threads);
  at.dynamicSmemBytes = bytes;
  at.stream = st;
  at.attrs = &early;
  at.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&at, kernel, args...);
  if (e != cudaSuccess) { cudaGetLastError(); last_launch_error() = e; return kECuda; }
  return launch_status();
}

template <typename T> int prepare(const SelectiveParams& P, const Space& W, bool backward, cudaStream_t st) {
  const int head_blocks = (P.heads + kPrepHeads - 1) / kPrepHeads, tiles = !P.tiled ? 2 * P.groups : backward ? W.units : 0;
  prepare_kernel<T><<<dim3(W.nc, head_blocks + tiles, P.batch), kThreads, 0, st>>>(P, W, head_blocks);
  return launch_status();
}

template <typename T, bool TILED> int forward(const SelectiveParams& P, cudaStream_t st) {
  const Space W = space_of(P, false, TILED);
  if (int s = allow<out_kernel<T, TILED>>(kOutSmem)) return s;
  if (int s = allow<state_pass_kernel<T, TILED>>(kPassSmem)) return s;
  if (int s = prepare<T>(P, W, false, st)) return s;
  if (W.nc > 1 || P.state_in || P.state_out)
    if (int s = behind(state_pass_kernel<T, TILED>, dim3(W.units, P.batch), kThreads, kPassSmem, st, P, W)) return s;
  const int gunits = W.units / P.groups, per = (gunits + W.splits - 1) / W.splits;
  return behind(out_kernel<T, TILED>, dim3(W.nc, P.groups * W.splits, P.batch), kThreads, kOutSmem, st, P, W, per);
}

template <typename T, bool TILED> int backward(const SelectiveParams& P, cudaStream_t st) {
  const Space W = space_of(P, true, TILED);
  if (int s = allow<grad_kernel<T, TILED>>(kGradSmem)) return s;
  if (int s = allow<state_passes_kernel<T, TILED>>(kPassSmem)) return s;
  if (int s = prepare<T>(P, W, true, st)) return s;
  if (W.nc > 1 || P.state_in || P.dstate_out || P.dstate_in)
    if (int s = behind(state_passes_kernel<T, TILED>, dim3(W.units, P.batch, 2), kThreads, kPassSmem, st, P, W)) return s;
  const int gunits = W.units / P.groups, per = (gunits + W.splits - 1) / W.splits;
  if (int s = behind(grad_kernel<T, TILED>, dim3(W.nc, P.groups * W.splits, P.batch), kGradThreads, kGradSmem, st, P, W, per)) return s;
  if (W.ptiles > 1)
    if (int s = behind(finish_dt_kernel<T>, dim3(W.nc, (P.heads + kPrepHeads - 1) / kPrepHeads, P.batch), kThreads, 0, st, P, W)) return s;
  const int head_blocks = P.dA || P.dD || P.dbias ? (P.heads + kThreads / 32 - 1) / (kThreads / 32) : 0;
  const long long all = W.splits > 1 ? (long long)P.batch * P.length * P.groups * (kN / 4) : 0;
  const long long blocks = head_blocks + (all + kThreads - 1) / kThreads;
  return blocks ? behind(finish_kernel<typename std::conditional<TILED, float, T>::type>, dim3((unsigned)blocks), kThreads, 0, st, P, W, head_blocks) : (int)kOk;
}

}  // namespace

long long selective_workspace(int batch, int length, int heads, int dim, int groups, bool backward, bool tiled) {
  SelectiveParams P{};
  P.batch = batch; P.length = length; P.heads = heads; P.dim = dim; P.groups = groups;
  return space_of(P, backward, tiled).bytes;
}
ConvTiles selective_tiles(const SelectiveParams& P, bool backward) {
  const Space W = space_of(P, backward, true);
  return {P.heads, P.dim, P.groups, W.nc, W.units, W.xt, W.bt, W.ct, W.xback, W.bback, W.cback};
}
int launch_selective_forward(const SelectiveParams& P, cudaStream_t st) {
  if (P.tiled) return P.type == SQ_TYPE_F16 ? forward<__half, true>(P, st) : forward<__nv_bfloat16, true>(P, st);
  return P.type == SQ_TYPE_F16 ? forward<__half, false>(P, st) : forward<__nv_bfloat16, false>(P, st);
}
int launch_selective_backward(const SelectiveParams& P, cudaStream_t st) {
  if (P.tiled) return P.type == SQ_TYPE_F16 ? backward<__half, true>(P, st) : backward<__nv_bfloat16, true>(P, st);
  return P.type == SQ_TYPE_F16 ? backward<__half, false>(P, st) : backward<__nv_bfloat16, false>(P, st);
}
int launch_selective_step(const SelectiveStepParams& P, cudaStream_t st) {
  cudaLaunchAttribute early{};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t at{};
  at.gridDim = dim3((P.dim + 31) / 32, P.heads, P.batch);
  at.blockDim = dim3(128);
  at.stream = st;
  at.attrs = &early;
  at.numAttrs = P.behind ? 1 : 0;
  const cudaError_t e = P.type == SQ_TYPE_F16 ? (P.x_f32 ? cudaLaunchKernelEx(&at, step_kernel<__half, float>, P)
                                                         : cudaLaunchKernelEx(&at, step_kernel<__half, __half>, P))
                                              : (P.x_f32 ? cudaLaunchKernelEx(&at, step_kernel<__nv_bfloat16, float>, P)
                                                         : cudaLaunchKernelEx(&at, step_kernel<__nv_bfloat16, __nv_bfloat16>, P));
  if (e != cudaSuccess) { cudaGetLastError(); last_launch_error() = e; return kECuda; }
  return launch_status();
}

}  // namespace sq
