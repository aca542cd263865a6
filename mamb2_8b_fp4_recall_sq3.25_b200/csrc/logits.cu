// Drawing a token from a row of logits, and the k largest logits of a row.
//
// Draw.  With m the largest logit and c = log2(e) / T, token j has y_j = 2^((x_j - m) c)
// and the whole weight w_j = rint(y_j 2^31).  Tokens are ordered by logit, equal ones by
// index.  Top-k keeps the first k; top-p those whose predecessors hold less than p of the
// kept weight; min-p those with y_j >= min_p.  The token drawn is the first in index order
// at which the running weight passes floor(u W), W the weight that is left.  Weights are
// integers and their sums 64-bit, so no sum depends on the order it is formed in, and the
// token is a function of the inputs alone.  A token 2^-32 times less likely than the most
// likely one has weight 0; rounding moves at most 2^-32 of the largest weight a token.  Products with u and with p are
// 64-bit floating point.  u is an fp32 number: on a grid of 2^-24 a token with a smaller share of the weight than that is
// drawn only where a grid point falls on it.
//
// A cluster of 1..8 CTAs shares a row; CTAs exchange single numbers, lists and histograms through
// distributed shared memory.
//
// Few tokens wanted (top_logits, top-k up to 256, greedy): every thread streams its units of 16 bytes and
// keeps eight maxima, of every eighth unit each.  The r-th largest of a CTA's maxima, r = k / CTAs, to
// 16 bits of its key, is reached by r logits at least; the least of the CTAs' bounds by k logits of the
// row, and by few more.  Only the units under a maximum that reaches it are read again (from L2), and
// CTA 0 sorts what is not below it.  Rows where that is too much (thousands of equal logits at the
// bound) are listed in column order instead, with a bound that is raised on the way.  Bound by HBM where there are
// many rows: the 64 largest of 2,048 rows of 256,000 fp16 logits (1.05 GB) take 200 us, 5.2 TB/s.  One row of 256,000
// takes 8 to 11 us on the device: a read of 62 KB a CTA, eight rounds of counting, three cluster barriers.
//
// Otherwise (top-p, large k, none) the row stays on chip, each CTA with its part in shared memory: it is read
// from HBM once.  A histogram over 256 steps of 1/8 octave of y, with exact weights, finds the
// step in which the running weight reaches what is wanted; the members of that step are
// narrowed by histograms over their keys until one key is left (16-bit types mostly by counting their values, in one
// pass).  What is kept is then "logit above the cut, or equal and index not above the last one kept".  Elements that need
// more than an addition to one word (weights of 2^18 and more, members of the step) are noted by position and worked on
// with all lanes busy.
// Bound by instructions (43 a logit) and by the waits of eight CTAs for one another: top-p of 512 rows of
// 256,000 bf16 logits takes 0.34 ms, eight times the time to read them; of that the read and the maximum are 17%, the
// histogram 35%, the step it crosses in 23%, the cut and the draw 25%.
#include "logits.cuh"
#include "logits_util.cuh"
#include <type_traits>

namespace sq {
namespace {

constexpr int kTopThreads = 256;
typedef unsigned long long u64;

// Histogram over rint(-7.96875 log2 y): 256 steps hold every weight but 0 (y > 2^-32).  Four copies
// of it, by lane, so that fewer lanes meet in one word: a word sums the low 18 bits of at most a quarter of
// the threads times the elements of one, < 2^14 (a part has at most 32776 elements).
// The upper 13 bits are not 0 for y >= 2^-13 only, the first 105 steps.
constexpr int kSteps = 256, kCols = 4, kLowBits = 18, kHighSteps = 106;
constexpr float kPerOctave = 7.96875f;
constexpr int kFine = 128;                       // entries of the narrowing histograms, laid out alike
constexpr int kWorkBytes = (kSteps + kHighSteps) * kCols * 4;
constexpr int kMembers = kHighSteps * kCols * 4 / 2;           // members of a step held as 16-bit positions
constexpr int kList = 2048;                      // listed logits of a CTA
constexpr int kMaxima = 8;                       // of a thread
template <int NT> constexpr int kListBytes = kList * 8 + kMaxima * NT * 2;
constexpr int kMaxListed = kList / 8;            // top-k up to this many goes by the list

// Kept: above x, or equal and column <= last.  ties: if not 0, `last` is the column of the CTA's equal token of that number,
// which is not located yet.
struct Cut { float x; int last, ties; };

struct Shared {
  u64 slot[2][8];
  u64 part[16];                                  // a warp's each
  float fpart[16];
  u64 sums[2][kSteps];                           // this CTA's histogram, and the one before
  u64 found_above, found_mine, found_need;
  int found, count, pick;
  uint2 counts[2][16];
  int groups;
};

__device__ __forceinline__ u64 warp_sum(u64 v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The CTAs of a cluster, NT threads each, and what they exchange.
template <int NT>
struct Team {
  static constexpr int NW = NT / 32;
  static_assert(NW <= 16, "Shared has room for 16 warps");
  Shared& s;
  uint32_t rank, size;
  int tid, phase;
  __device__ explicit Team(Shared& s)
      : s(s), rank(cluster_rank()), size(cluster_size()), tid(threadIdx.x), phase(0) { cluster_arrive_relaxed(); }
  // before the first remote access: every CTA runs
  __device__ void ready() const { cluster_wait(); }
  __device__ void barrier() const { cluster_arrive(); cluster_wait(); }
  // Hands `v` (the same in every thread) to all CTAs; afterwards got(r) is CTA r's.
  __device__ void exchange(u64 v) {
    phase ^= 1;
    if (tid < (int)size) remote_store(remote_smem(&s.slot[phase][rank], tid), v);
    barrier();
  }
  __device__ u64 got(int r) const { return s.slot[phase][r]; }
  __device__ float row_max(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    if ((tid & 31) == 0) s.fpart[tid >> 5] = v;
    __syncthreads();
    v = s.fpart[0];
    for (int i = 1; i < NW; ++i) v = fmaxf(v, s.fpart[i]);
    exchange(__float_as_uint(v));
    for (int r = 0; r < (int)size; ++r) v = fmaxf(v, __uint_as_float((uint32_t)got(r)));
    return v;
  }
  // Exclusive running sum of v over the threads; `total` the whole.
  __device__ u64 block_scan(u64 v, u64& total) {
    u64 run = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 a = __shfl_up_sync(0xffffffffu, run, o);
      if ((tid & 31) >= o) run += a;
    }
    __syncthreads();
    if ((tid & 31) == 31) s.part[tid >> 5] = run;
    __syncthreads();
    u64 before = 0;
    total = 0;
    for (int i = 0; i < NW; ++i) {
      if (i < (tid >> 5)) before += s.part[i];
      total += s.part[i];
    }
    return before + run - v;
  }
  // The largest number t of `bits` bits (`bits` is even) for which count(t) summed over the block is at
  // least r (0 where there is none); count falls with t and is at most 31 a thread.  Two bits a round.
  template <typename C>
  __device__ u64 search(int bits, int r, C count) {
    u64 t = 0;
#pragma unroll 1
    for (int b = bits - 2; b >= 0; b -= 2) {
      uint32_t c[3];
#pragma unroll
      for (int i = 0; i < 3; ++i) c[i] = count(t | (u64)(i + 1) << b);
      const uint32_t c01 = __reduce_add_sync(0xffffffffu, c[0] | c[1] << 16), c2 = __reduce_add_sync(0xffffffffu, c[2]);
      uint2* out = s.counts[b >> 1 & 1];         // the other half is being read by slower warps
      if ((tid & 31) == 0) out[tid >> 5] = make_uint2(c01, c2);
      __syncthreads();
      uint2 sum = out[0];
      for (int i = 1; i < NW; ++i) { sum.x += out[i].x; sum.y += out[i].y; }
      const int at = (int)sum.y >= r ? 3 : (int)(sum.x >> 16) >= r ? 2 : (int)(sum.x & 0xffffu) >= r ? 1 : 0;
      t |= (u64)at << b;
    }
    return t;
  }
};

// The k largest logits of a row.  Items are key << 32 | ~column: distinct, and larger
// ones come first in the order.
template <typename T, int NT>
struct Listing {
  static constexpr int NV = 4, G = kMaxima;                 // units of a batch in column order; maxima of a thread
  Team<NT>& t;
  Span<T> span;
  u64* list;                                     // [kList], with room for [kMaxima NT] 16-bit numbers behind it
  int k;
  float bound;
  u64 least;                                     // items not above it are no longer wanted

  // Raises the bound to the k-th largest of the n >= k items listed, to 16 bits.
  __device__ void raise(int n) {
    const uint32_t key = (uint32_t)t.search(16, k, [&](u64 q) {
      uint32_t c = 0;
      for (int i = t.tid; i < n; i += NT) c += (uint32_t)(list[i] >> 48) >= (uint32_t)q;
      return c;
    });
    bound = fmaxf(bound, key_logit(max(key << 16, kKeyLowest)));
  }
  // Leaves the k largest of n > k items.
  __device__ void compress(int n) {
    constexpr int N = kList / NT;
    u64 item[N];
#pragma unroll
    for (int a = 0; a < N; ++a) item[a] = t.tid + a * NT < n ? list[t.tid + a * NT] : 0;
    least = t.search(64, k, [&](u64 q) {
      uint32_t c = 0;
#pragma unroll
      for (int a = 0; a < N; ++a) c += item[a] >= q;
      return c;
    });
    if (t.tid == 0) t.s.count = 0;
    __syncthreads();
#pragma unroll
    for (int a = 0; a < N; ++a)
      if (item[a] >= least) list[atomicAdd(&t.s.count, 1)] = item[a];
    bound = fmaxf(bound, key_logit((uint32_t)(least >> 32)));
    __syncthreads();
  }
  // Whole units only, so that the loads of a batch are in flight together; -inf past the end.
  __device__ void load(Unit<T> (&x)[NV], int from) const {
    const uint4* body = reinterpret_cast<const uint4*>(span.p + span.col(0, 0));
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int u = from + i * NT + t.tid;
      x[i].q = neg_inf_unit<T>();
      if (u < span.hi) x[i].q = load_unit(body + u);
    }
  }
  // Lists what is wanted of a batch whose unit i starts at column col(i).
  template <int N, typename C>
  __device__ void add(const Unit<T> (&x)[N], C col, int& mark) {
    uint32_t done = 0;                           // elements of this thread that are listed
    bool again;
    do {
      int top = -1;
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (unit_max(x[i]) >= bound) {
#pragma unroll
          for (int v = 0; v < kUnit<T>; ++v) {
            const float f = to_f32(x[i].v[v]);
            if (f >= bound && !(done >> (i * kUnit<T> + v) & 1)) {
              const u64 item = (u64)order_key(f + 0.0f) << 32 | (uint32_t)~(col(i) + v);
              if (item > least) {
                const int at = atomicAdd(&t.s.count, 1);
                if (at < kList) {
                  list[at] = item;
                  done |= 1u << (i * kUnit<T> + v);
                }
                top = at;
              }
            }
          }
        }
      again = false;
      if (__syncthreads_or(top >= min(mark, kList))) {
        const int n = t.s.count;
        __syncthreads();
        if (n > kList) {                         // some found no place: room for them, and again
          compress(kList);
          again = true;
          mark = 2 * k;
        } else {
          raise(n);
          mark = n + k;
        }
      }
    } while (again);
  }
  // Column order.  Lists at least the k largest of this CTA's part, or all that are not masked; returns
  // their number.
  __device__ int collect() {
    Unit<T> x[NV];
    load(x, span.lo);
    uint32_t high[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) high[i] = order_key(unit_max(x[i]) + 0.0f) >> 16;
    const uint32_t key = (uint32_t)t.search(16, k, [&](u64 q) {
      uint32_t c = 0;
#pragma unroll
      for (int i = 0; i < NV; ++i) c += high[i] >= (uint32_t)q;
      return c;
    });
    bound = key_logit(max(key << 16, kKeyLowest));
    least = 0;
    int mark = 2 * k;                            // raise the bound when this many are listed
    if (t.tid == 0) t.s.count = 0;
    __syncthreads();
    for (int from = span.lo; from < span.hi; from += NT * NV) {
      Unit<T> next[NV];
      load(next, from + NT * NV);
      add(x, [&](int i) { return span.col(from + i * NT + t.tid, 0); }, mark);
#pragma unroll
      for (int i = 0; i < NV; ++i) x[i] = next[i];
    }
    if (span.lo > 0 || span.hi < span.n) {       // the row's ragged ends
      Unit<T> end[1];
      end[0].q = neg_inf_unit<T>();
      const int at = t.tid == 0 && span.lo > 0 ? 0 : t.tid == 1 && span.hi < span.n ? span.hi : -1;
      if (at >= 0) end[0] = span.ragged(at);
      add(end, [&](int) { return span.col(at, 0); }, mark);
    }
    __syncthreads();
    return t.s.count;
  }
  // Lists logits that are not below `bound` from unit i of the part (the list's length is not bounded by
  // kList, what it holds is).
  __device__ void pick(const Unit<T>& x, int i) {
    if (!(unit_max(x) >= bound)) return;
#pragma unroll
    for (int v = 0; v < kUnit<T>; ++v) {
      const float f = to_f32(x.v[v]);
      if (f >= bound) {
        const int at = atomicAdd(&t.s.count, 1);
        if (at < kList) list[at] = (u64)order_key(f + 0.0f) << 32 | (uint32_t)~span.col(i, v);
      }
    }
  }
  // As collect, for the row's k largest, by the maxima of groups of units; the list may not hold them all.
  __device__ int pick_groups() {
    const uint4* body = reinterpret_cast<const uint4*>(span.p + span.col(0, 0));
    Unit<T> top[G];
#pragma unroll
    for (int a = 0; a < G; ++a) top[a].q = neg_inf_unit<T>();
#pragma unroll 1
    for (int from = span.lo + t.tid; from < span.hi; from += NT * G) {
      Unit<T> x[G];
#pragma unroll
      for (int a = 0; a < G; ++a) {
        const int u = from + a * NT;
        x[a].q = neg_inf_unit<T>();
        if (u < span.hi) x[a].q = load_unit(body + u);
      }
#pragma unroll
      for (int a = 0; a < G; ++a) fold_max(top[a], x[a]);
    }
    t.ready();
    float high[G];
    uint32_t key[G];
#pragma unroll
    for (int a = 0; a < G; ++a) {
      high[a] = unit_max(top[a]);
      key[a] = order_key(high[a] + 0.0f) >> 16;
    }
    if (t.tid == 0) { t.s.count = 0; t.s.groups = 0; }
    const u64 mine = t.search(16, (k + (int)t.size - 1) / (int)t.size, [&](u64 q) {
      uint32_t c = 0;
#pragma unroll
      for (int a = 0; a < G; ++a) c += key[a] >= (uint32_t)q;
      return c;
    });
    uint32_t least_key = (uint32_t)mine;
    if (t.size > 1) {
      t.exchange(mine);
      for (int r = 0; r < (int)t.size; ++r) least_key = min(least_key, (uint32_t)t.got(r));
    }
    bound = key_logit(max(least_key << 16, kKeyLowest));
    // groups to be read again, half a warp each
    uint16_t* groups = reinterpret_cast<uint16_t*>(list + kList);
#pragma unroll
    for (int a = 0; a < G; ++a)
      if (high[a] >= bound) groups[atomicAdd(&t.s.groups, 1)] = (uint16_t)(t.tid * G + a);
    __syncthreads();
    const int n = t.s.groups, lane = t.tid & 15;
    for (int i = t.tid >> 4; i < n; i += NT / 16) {
      const int g = groups[i];
      for (int u = span.lo + g / G + (g % G) * NT + lane * NT * G; u < span.hi; u += 16 * NT * G) {
        Unit<T> x;
        x.q = load_unit(body + u);
        pick(x, u);
      }
    }
    if (t.tid == 0 && span.lo > 0) pick(span.ragged(0), 0);
    if (t.tid == 32 && span.hi < span.n) pick(span.ragged(span.hi), span.hi);
    __syncthreads();
    return t.s.count;
  }
  // The row's k largest (or more) in the list of CTA 0, largest first; returns their number, to CTA 0 alone.
  __device__ int gather() {
    int n = pick_groups(), total = n, at = 0;
    const auto count = [&] {
      if (t.size == 1) { total = n; return; }
      t.exchange((u64)n);
      total = at = 0;
      for (int r = 0; r < (int)t.size; ++r) {
        if (r < (int)t.rank) at += (int)t.got(r);
        total += (int)t.got(r);
      }
    };
    count();
    if (total > kList) {
      n = collect();
      const int share = kList / (int)t.size;     // >= k
      if (n > share) {
        compress(n);
        n = t.s.count;
      }
      count();
    }
    if (t.size > 1) {
      if (t.rank != 0) {
        const uint32_t to = remote_smem(list, 0);
        for (int i = t.tid; i < n; i += NT) remote_store(to + 8u * (at + i), list[i]);
      }
      t.barrier();
      if (t.rank != 0) return 0;
    }
    sort(total);
    return total;
  }
  // list[0 .. n) by falling value.  Few items are placed by counting the larger ones, which takes two
  // barriers; more by a bitonic network.
  __device__ void sort(int n) {
    if (n <= 512) {
      __syncthreads();
      u64 item[2];
      int place[2] = {0, 0};
#pragma unroll
      for (int a = 0; a < 2; ++a) item[a] = t.tid + a * NT < n ? list[t.tid + a * NT] : 0;
      const bool both = n > NT;
#pragma unroll 4
      for (int j = 0; j < n; ++j) {
        const u64 other = list[j];
        place[0] += other > item[0];
        if (both) place[1] += other > item[1];
      }
      __syncthreads();
#pragma unroll
      for (int a = 0; a < 2; ++a)
        if (t.tid + a * NT < n) list[place[a]] = item[a];
      __syncthreads();
      return;
    }
    int size = 1;
    while (size < n) size <<= 1;
    for (int i = n + t.tid; i < size; i += NT) list[i] = 0;
    for (int len = 2; len <= size; len <<= 1)
      for (int d = len >> 1; d; d >>= 1) {
        __syncthreads();
        for (int i = t.tid; i < size / 2; i += NT) {
          const int a = 2 * i - (i & (d - 1)), b = a + d;
          const u64 x = list[a], y = list[b];
          if ((x < y) == ((a & len) == 0)) { list[a] = y; list[b] = x; }
        }
      }
    __syncthreads();
  }
};

// t = (x - m) c of a token, m the largest logit: its weight is rint(2^t 2^31).
struct Exponent {
  float m, c;
  __device__ float operator()(float x) const { return __fmul_rn(x - m, c); }
  __device__ float2 operator()(float2 x) const { return __fmul2_rn(__fadd2_rn(x, make_float2(-m, -m)), make_float2(c, c)); }
};
__device__ __forceinline__ uint32_t weight_of(float t) {
  const float y = ex2(t);
  // below 2^-8 the sum y + 2^-8 rounds y to a multiple of 2^-31, as rint does, and holds it in its low bits
  if (t < -8.01f) return __float_as_uint(y + 0.00390625f) & 0x7fffffu;
  return __float2uint_rn(y * 2147483648.0f);
}

// Adds `w` to the histogram word at `address` if the weight is light, -32.01 < t < kLight; sets `bit` of `rest` if t is not
// below kLight (without branches: most are light).
constexpr float kLight = -13.02f;
__device__ __forceinline__ void add_light(uint32_t address, uint32_t w, float t, uint32_t& rest, uint32_t bit) {
  asm volatile("{\n.reg .pred p;\nsetp.lt.f32 p, %3, %4;\n@!p or.b32 %0, %0, %6;\nsetp.gt.and.f32 p, %3, %5, p;\n"
               "@p red.shared.add.u32 [%1], %2;\n}\n"
               : "+r"(rest) : "r"(address), "r"(w), "f"(t), "f"(kLight), "f"(-32.01f), "r"(bit) : "memory");
}

// Counts one at the shared word at `address` if d < width (without a branch).
__device__ __forceinline__ void count_if(uint32_t address, uint32_t d, uint32_t width) {
  asm volatile("{\n.reg .pred p;\nsetp.lt.u32 p, %1, %2;\n@p red.shared.add.u32 [%0], 1;\n}\n"
               :: "r"(address), "r"(d), "r"(width) : "memory");
}

// One CTA's part of a row in shared memory.
template <typename T, int NT>
struct Row : Team<NT> {
  using Base = Team<NT>;
  Span<T> d;
  unsigned char* work;                           // histogram and members
  Unit<T>* unit;
  int turn = 0;                                  // of s.sums
  using Base::s; using Base::tid; using Base::rank; using Base::size; using Base::barrier; using Base::exchange; using Base::got;
  static constexpr int NW = NT / 32;

  __device__ Row(const Base& t, const Span<T>& d, unsigned char* dyn)
      : Base(t), d(d), work(dyn), unit(reinterpret_cast<Unit<T>*>(dyn + kWorkBytes)) {
    for (int i = tid; i < d.n; i += NT) {
      if (i >= d.lo && i < d.hi) cp_async16(unit + i, d.p + d.col(i, 0));
      else unit[i] = d.ragged(i);
    }
    cp_async_wait_all();                         // each thread's own units
    this->ready();
  }

  // f(unit, exponents) over this thread's units.
  template <typename F>
  __device__ void each_unit(Exponent e, F f) const {
    for (int i = tid; i < d.n; i += NT) {
      Unit<T> u;
      u.q = unit[i].q;
      float2 t[kUnit<T> / 2];
#pragma unroll
      for (int v = 0; v < kUnit<T>; v += 2) t[v / 2] = e(make_float2(to_f32(u.v[v]), to_f32(u.v[v + 1])));
      f(i, t);
    }
  }
  // f(position) for the elements of unit i whose bits are set in `which`.
  template <typename F>
  __device__ void each_bit(uint32_t which, int i, F f) const {
    while (which) {
      f(i * kUnit<T> + __ffs(which) - 1);
      which &= which - 1;
    }
  }
  __device__ float at(int position) const { return to_f32(reinterpret_cast<const T*>(unit)[position]); }
  // Positions are noted in list[0 .. most) for a second pass with all lanes busy; returns whether there was room.
  __device__ bool note(uint16_t* list, int most, int position) {
    const int k = atomicAdd(&s.count, 1);
    if (k < most) list[k] = (uint16_t)position;
    return k < most;
  }
  __device__ float own_max() const {
    float m = -INFINITY;
#pragma unroll 4
    for (int i = tid; i < d.n; i += NT) {
      Unit<T> u;
      u.q = unit[i].q;
      m = fmaxf(m, unit_max(u));
    }
    return m;
  }
  __device__ u64 part_sums(u64 sum) {
    sum = warp_sum(sum);
    __syncthreads();
    if ((tid & 31) == 0) s.part[tid >> 5] = sum;
    __syncthreads();
    u64 t = 0;
    for (int i = 0; i < NW; ++i) t += s.part[i];
    return t;
  }
  // Sums of w(x, col) over contiguous stretches, one a warp, in s.part; returns this CTA's total.
  // w is 0 below `least`.
  template <typename W>
  __device__ u64 stretch_sums(W w, float least) {
    const int len = (d.n + NW - 1) / NW, i0 = (tid >> 5) * len, i1 = min(d.n, i0 + len);
    u64 sum = 0;
    for (int i = i0 + (tid & 31); i < i1; i += 32) {
      Unit<T> u;
      u.q = unit[i].q;
      if (!(unit_max(u) >= least)) continue;
#pragma unroll
      for (int v = 0; v < kUnit<T>; ++v) sum += w(to_f32(u.v[v]), d.col(i, v));
    }
    return part_sums(sum);
  }
  // stretch_sums of the weights of what `cut` and min-p leave; nothing is left below `least`.
  __device__ u64 left_sums(Exponent e, Cut cut, float min_p, float least) {
    const int len = (d.n + NW - 1) / NW, i0 = (tid >> 5) * len, i1 = min(d.n, i0 + len);
    min_p = fmaxf(min_p, 1e-10f);                // below 2^-33 the weight is 0: masked logits are no ties
    u64 sum = 0;
    for (int i = i0 + (tid & 31); i < i1; i += 32) {
      Unit<T> u;
      u.q = unit[i].q;
      if (!(unit_max(u) >= least)) continue;
      uint32_t ties = 0;
#pragma unroll
      for (int v = 0; v < kUnit<T>; v += 2) {
        const float2 x = make_float2(to_f32(u.v[v]), to_f32(u.v[v + 1])), t = e(x);
        const float2 y = make_float2(ex2(t.x), ex2(t.y));
        if (x.x > cut.x && y.x >= min_p) sum += __float2uint_rn(y.x * 2147483648.0f);
        if (x.y > cut.x && y.y >= min_p) sum += __float2uint_rn(y.y * 2147483648.0f);
        if (x.x == cut.x && y.x >= min_p) ties |= 1u << v;
        if (x.y == cut.x && y.y >= min_p) ties |= 2u << v;
      }
      each_bit(ties, i, [&](int p) { if (d.col(0, p) <= cut.last) sum += weight_of(e(at(p))); });
    }
    return part_sums(sum);
  }
  // After stretch_sums: the first column of this CTA, in order, at which the running sum passes
  // `target` (below the total).
  template <typename W>
  __device__ int locate(W w, u64 target) {
    const int warp = tid >> 5, lane = tid & 31;
    const int len = (d.n + NW - 1) / NW, i0 = warp * len, i1 = min(d.n, i0 + len);
    u64 before = 0;
    for (int i = 0; i < warp; ++i) before += s.part[i];
    if (target >= before && target < before + s.part[warp]) {
      for (int i = i0; i < i1; i += 32) {
        Unit<T> u;
        u64 own = 0;
        if (i + lane < i1) {
          u.q = unit[i + lane].q;
#pragma unroll
          for (int v = 0; v < kUnit<T>; ++v) own += w(to_f32(u.v[v]), d.col(i + lane, v));
        }
        u64 run = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const u64 a = __shfl_up_sync(0xffffffffu, run, o);
          if (lane >= o) run += a;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, before + run > target);
        if (hit) {
          if (lane == __ffs(hit) - 1) {
            u64 at = before + run - own;
            int found = -1;
#pragma unroll
            for (int v = 0; v < kUnit<T>; ++v) {
              at += w(to_f32(u.v[v]), d.col(i + lane, v));
              if (found < 0 && at > target) found = d.col(i + lane, v);
            }
            s.pick = found;
          }
          break;
        }
        before += __shfl_sync(0xffffffffu, run, 31);
      }
    }
    __syncthreads();
    return s.pick;
  }

  // `mine`: entry tid of this CTA's histogram.  The first entry of the row's histogram, the sum over the CTAs,
  // at which the running weight, from `above` on, reaches need(whole weight); adds the entries before
  // it to `above`, and of this CTA's histogram to `mine_above`.  Returns -1 if it is not reached.  s.sums
  // alternates, so that CTAs ahead do not overwrite what others still read.
  template <typename N>
  __device__ int crossing(u64 mine, N need_of, u64& above, u64& mine_above) {
    constexpr int E = kSteps / 32;
    turn ^= 1;
    const u64* sums = s.sums[turn];
    u64* total = reinterpret_cast<u64*>(work);   // the histogram's words have been read
    if (tid < kSteps) s.sums[turn][tid] = mine;
    barrier();
    if (tid < kSteps) {
      u64 all = 0;
      for (int r = 0; r < (int)size; ++r) all += remote_load(remote_smem(&sums[tid], r));
      total[tid] = all;
    }
    __syncthreads();
    if (tid < 32) {                              // eight entries a lane
      u64 sum = 0, own = 0;
      for (int i = 0; i < E; ++i) { sum += total[tid * E + i]; own += sums[tid * E + i]; }
      u64 run = sum, own_run = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const u64 a = __shfl_up_sync(0xffffffffu, run, o), b = __shfl_up_sync(0xffffffffu, own_run, o);
        if (tid >= o) { run += a; own_run += b; }
      }
      const u64 need = need_of(__shfl_sync(0xffffffffu, run, 31));
      u64 before = above + run - sum, own_before = mine_above + own_run - own;
      const bool here = before < need && before + sum >= need;
      if (here) {
        int i = tid * E;
        for (; before + total[i] < need; ++i) { before += total[i]; own_before += sums[i]; }
        s.found = i;
        s.found_above = before;
        s.found_mine = own_before;
        s.found_need = need;
      }
      if (!__any_sync(0xffffffffu, here) && tid == 0) s.found = -1;
    }
    __syncthreads();
    const int at = s.found;
    if (at >= 0) { above = s.found_above; mine_above = s.found_mine; }
    return at;
  }

  // The cut after the first tokens of the order whose weights w(t) reach need(whole weight), among
  // elements with kept(x, col).  t = (x - m) c is the exponent of y; w depends on it alone, is 0 where the
  // token's weight is, and below 2^31 + 1.  False: the whole weight does not reach it.
  // kept_here: this CTA's share of the weight that is kept.  PLAIN: every element is kept and w is weight_of.
  // A cluster barrier has to follow before the CTA ends (others read its sums).
  template <bool PLAIN, typename K, typename W, typename N>
  __device__ bool select(K kept, W w, Exponent e, N need_of, Cut& cut, u64& kept_here) {
    static_assert(kSteps <= NT, "a thread per step");
    constexpr int SH = std::is_same<T, __half>::value ? 13 : std::is_same<T, __nv_bfloat16>::value ? 16 : 0;
    constexpr uint32_t kLow = (1u << kLowBits) - 1;
    uint32_t* low = reinterpret_cast<uint32_t*>(work);
    uint32_t* high = low + kSteps * kCols;
    uint16_t* members = reinterpret_cast<uint16_t*>(high);
    const int lane = tid & (kCols - 1);
    // 2^23 + the step, as a float: its bits are in order and end in the step
    const auto step = [&](float2 t) { return __ffma2_rn(t, make_float2(-kPerOctave, -kPerOctave), make_float2(8388608.0f, 8388608.0f)); };
    constexpr uint32_t kStep0 = 0x4b000000u;
    const auto count = [&](int p) {
      const float x = at(p), t = e(x);
      const uint32_t q = w(t), b = (__float_as_uint(fmaf(t, -kPerOctave, 8388608.0f)) - kStep0) * kCols + lane;
      if (!q || !(PLAIN || kept(x, d.col(0, p)))) return;
      atomicAdd(low + b, q & kLow);
      if (q >> kLowBits) atomicAdd(high + b, q >> kLowBits);
    };
    __syncthreads();
    for (int i = tid; i < (kSteps + kHighSteps) * kCols; i += NT) low[i] = 0;
    if (tid == 0) s.count = 0;
    __syncthreads();
    // no CTA reads sums of the other turn any more, and this one writes them after the next barrier of its own
    uint16_t* noted = reinterpret_cast<uint16_t*>(s.sums[turn ^ 1]);
    constexpr int kNoted = sizeof(s.sums[0]) / sizeof(uint16_t);
    const uint32_t words = (uint32_t)__cvta_generic_to_shared(low + lane) - kStep0 * kCols * 4;
    each_unit(e, [&](int i, const float2 (&t)[kUnit<T> / 2]) {
      uint32_t rest = 0;                         // elements that are not simply added
#pragma unroll
      for (int a = 0; a < kUnit<T> / 2; ++a) {
        if (PLAIN) {
          // weight_of for y < 2^-13, which fits the low word
          const float2 y = __fadd2_rn(make_float2(ex2(t[a].x), ex2(t[a].y)), make_float2(0.00390625f, 0.00390625f)), b = step(t[a]);
          add_light(words + __float_as_uint(b.x) * (kCols * 4), __float_as_uint(y.x) & 0x7fffffu, t[a].x, rest, 1u << (2 * a));
          add_light(words + __float_as_uint(b.y) * (kCols * 4), __float_as_uint(y.y) & 0x7fffffu, t[a].y, rest, 2u << (2 * a));
        } else {
          if (t[a].x > -32.01f) rest |= 1u << (2 * a);
          if (t[a].y > -32.01f) rest |= 2u << (2 * a);
        }
      }
      if (__popc(rest) <= 2) {
        each_bit(rest, i, [&](int p) { if (!note(noted, kNoted, p)) count(p); });
      } else {                                   // a flat stretch: element by element, without the detour
#pragma unroll
        for (int v = 0; v < kUnit<T>; ++v)
          if (rest >> v & 1) count(i * kUnit<T> + v);
      }
    });
    __syncthreads();
    for (int k = tid; k < min(s.count, kNoted); k += NT) count(noted[k]);
    __syncthreads();
    u64 mine = 0;
    for (int i = 0; i < kCols; ++i) {
      if (tid < kSteps) mine += low[tid * kCols + i];
      if (tid < kHighSteps) mine += (u64)high[tid * kCols + i] << kLowBits;
    }
    u64 above = 0, mine_above = 0;
    const int found = crossing(mine, need_of, above, mine_above);
    if (found < 0) return false;
    const u64 need = s.found_need;
    const uint32_t wanted_step = kStep0 + found;
    // the step's edges in x, widened by far more than the rounding of t and of this (NaN, from infinities, widens
    // to everything)
    const float first = e.m - (found - 0.5f) / kPerOctave / e.c, last = e.m - (found + 0.5f) / kPerOctave / e.c;
    const float most = fminf(e.m, first + 4e-6f * (fabsf(e.m) + fabsf(first - e.m)));
    const float least = fmaxf(-3.4028235e38f, last - 4e-6f * (fabsf(e.m) + fabsf(last - e.m)));
    int entry;
    if constexpr (PLAIN && SH != 0) {
      // 16-bit logits of one sign take few values in a step: each value's tokens are counted, and a thread a value weighs
      // them (top-p of 512 rows of 256,000 bf16 logits 388 us; by listing the step's members, as below, 420).
      const uint32_t a = bits_below<T>(most), b = bits_below<T>(least), base = min(a, b), width = max(a, b) - base + 1;
      if ((least > 0.0f || most < 0.0f) && width <= kSteps) {
        for (int i = tid; i < kSteps * kCols; i += NT) low[i] = 0;
        __syncthreads();
        const uint32_t counts = (uint32_t)__cvta_generic_to_shared(low + lane);
        for (int i = tid; i < d.n; i += NT) {
          const uint4 q = unit[i].q;
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            const uint32_t two = v == 0 ? q.x : v == 1 ? q.y : v == 2 ? q.z : q.w;
            const uint32_t d0 = (two & 0xffffu) - base, d1 = (two >> 16) - base;
            count_if(counts + d0 * (kCols * 4), d0, width);
            count_if(counts + d1 * (kCols * 4), d1, width);
          }
        }
        __syncthreads();
        const auto value = [&](int i) { return to_f32(from_bits<T>(base + (least > 0.0f ? width - 1 - i : i))); };
        mine = 0;
        if (tid < (int)width) {
          const float t = e(value(tid));
          const int i = least > 0.0f ? width - 1 - tid : tid;
          uint32_t n = 0;
          for (int c = 0; c < kCols; ++c) n += low[i * kCols + c];
          // the values beside the step are in the widened window only
          if (__float_as_uint(fmaf(t, -kPerOctave, 8388608.0f)) == wanted_step) mine = (u64)n * w(t);
        }
        entry = crossing(mine, [&](u64) { return need; }, above, mine_above);
        return finish(value(entry), entry, w, e, need - above, cut, kept_here, mine_above);
      }
    }
    uint32_t hi = order_key(most + 0.0f) >> SH, lo = order_key(least) >> SH;
    // narrowing: histograms of the step's members over their keys; the members' positions are listed first
    // (if they are too many, every round goes through the part)
    uint32_t* upper = low + kFine * kCols;
    int shift;
    const auto begin = [&] {
      for (shift = 0; ((hi - lo) >> shift) >= (uint32_t)kFine; ++shift) {}
      for (int i = tid; i < 2 * kFine * kCols; i += NT) low[i] = 0;
      __syncthreads();                           // and the members are listed
    };
    const auto add = [&](int p) {
      const float x = at(p);
      const uint32_t k = order_key(x + 0.0f) >> SH;
      if (k < lo || k > hi) return;              // decided by an earlier round
      const uint32_t b = ((hi - k) >> shift) * kCols + lane, q = w(e(x));
      if (!PLAIN && !kept(x, d.col(0, p))) return;
      atomicAdd(low + b, q & kLow);
      if (q >> kLowBits) atomicAdd(upper + b, q >> kLowBits);
    };
    const auto each_in_step = [&](auto f) {
      each_unit(e, [&](int i, const float2 (&t)[kUnit<T> / 2]) {
        uint32_t which = 0;
#pragma unroll
        for (int a = 0; a < kUnit<T> / 2; ++a) {
          const float2 b = step(t[a]);
          if (__float_as_uint(b.x) == wanted_step) which |= 1u << (2 * a);
          if (__float_as_uint(b.y) == wanted_step) which |= 2u << (2 * a);
        }
        each_bit(which, i, f);
      });
    };
    if (tid == 0) s.count = 0;
    __syncthreads();
    each_in_step([&](int p) { note(members, kMembers, p); });
    for (;;) {
      begin();
      if (s.count <= kMembers) {
        for (int k = tid; k < s.count; k += NT) add(members[k]);
      } else {
        each_in_step(add);
      }
      __syncthreads();
      mine = 0;
      if (tid < kFine)
        for (int i = 0; i < kCols; ++i)
          mine += low[tid * kCols + i] + ((u64)upper[tid * kCols + i] << kLowBits);
      entry = crossing(mine, [&](u64) { return need; }, above, mine_above);
      if (shift == 0) break;
      hi = hi - ((uint32_t)entry << shift);
      const uint32_t width = (1u << shift) - 1;
      if (hi - lo > width) lo = hi - width;
    }
    const uint32_t key = hi - entry;
    // the key of 16-bit types stands for one logit: its low bits are those of an exact value
    const float x = key_logit(SH == 0 ? key : (key << SH) | ((key << SH) & 0x80000000u ? 0u : (1u << SH) - 1u));
    return finish(x, entry, w, e, need - above, cut, kept_here, mine_above);
  }

  // The cut at logit x, entry `entry` of the histogram last crossed: of its tokens the first that reach `need` are kept.
  template <typename W>
  __device__ bool finish(float x, int entry, W w, Exponent e, u64 need, Cut& cut, u64& kept_here, u64 mine_above) {
    u64 key_before = 0;                          // weight of that logit in the CTAs before this one
    for (int r = 0; r < (int)rank; ++r) key_before += remote_load(remote_smem(&s.sums[turn][entry], r));
    const u64 here = s.sums[turn][entry];
    // quotients of numbers below 2^50 by one below 2^32: a double holds them closely enough for floor()
    const u64 each_w = w(e(x));
    const double by = (double)each_w;
    const u64 wanted = (u64)floor((double)(need + each_w - 1) / by), earlier = (u64)floor((double)key_before / by);
    const u64 ties = (u64)floor((double)here / by);
    cut.x = x;
    cut.ties = 0;
    u64 taken = ties;
    if (wanted >= earlier + ties) {
      cut.last = 0x7fffffff;
    } else if (wanted <= earlier) {
      cut.last = -1;
      taken = 0;
    } else {
      taken = wanted - earlier;
      cut.ties = (int)taken;
    }
    kept_here = mine_above + taken * each_w;
    return true;
  }
  // Locates the last equal token that a selection among `kept` took.  Left to the CTA that draws where only that one needs
  // it: a pass over the part in one CTA holds up the seven others (512 rows of 256,000: 340 us, before the exchange 388).
  template <typename K>
  __device__ void settle(K kept, Cut& cut) {
    if (!cut.ties) return;
    const float x = cut.x;
    const auto tie = [&](float v, int col) -> u64 { return v == x && kept(v, col) ? 1 : 0; };
    stretch_sums(tie, x);
    cut.last = locate(tie, cut.ties - 1);
    cut.ties = 0;
  }
};

__device__ __forceinline__ u64 draw(double u, u64 total) {
  const long long t = (long long)(u * (double)total);
  return t < 0 ? 0 : ((u64)t >= total ? total - 1 : (u64)t);
}

template <typename T, int NT>
__global__ void __launch_bounds__(NT, 768 / NT + (NT > 256)) sample_kernel(const SampleParams P) {
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ Shared s;
  Team<NT> team(s);
  const Span<T> span(P.x, blockIdx.x / team.size, team.rank, team.size);
  const int row = blockIdx.x / team.size, tid = threadIdx.x;
  const float temperature = P.temperature ? P.temperature[row] : P.temperature_all;
  const bool greedy = !(temperature > 0.0f);
  const int top_k = greedy ? 1 : P.top_k ? P.top_k[row] : P.top_k_all;
  const float top_p = P.top_p ? P.top_p[row] : P.top_p_all;
  const float min_p = fminf(P.min_p ? P.min_p[row] : P.min_p_all, 1.0f);
  const double u = P.uniform[row];
  Exponent e;
  e.c = fminf(__fdiv_rn(kLog2e, temperature), 3.4028234e38f);  // finite: 0 c stays 0
  // weight that top-p leaves of the whole: tokens with less than p z before them, the first always
  const auto wanted = [&](u64 z) {
    const double limit = (double)top_p * (double)z;
    const u64 need = limit > 1.0 ? (u64)ceil(limit) : 1;
    return top_p >= 1.0f || need > z ? z : need;
  };

  if (top_k > 0 && top_k <= kMaxListed) {
    u64* list = reinterpret_cast<u64*>(dyn);
    Listing<T, NT> l{team, span, list, top_k};
    const int n = min(top_k, l.gather());
    if (team.rank != 0) return;
    if (n <= 1 || greedy) {
      if (tid == 0) P.tokens[row] = n ? (long long)~(uint32_t)list[0] : -1;
      return;
    }
    static_assert(kMaxListed <= NT, "a thread per listed token");
    const u64 item = tid < n ? list[tid] : 0;
    const float x = key_logit((uint32_t)(item >> 32));
    e.m = key_logit((uint32_t)(list[0] >> 32));
    const float t = x == e.m ? 0.0f : e(x);      // equal to m: also where that is infinite
    const uint32_t w = tid < n ? weight_of(t) : 0;
    u64 whole;
    const u64 before = team.block_scan(w, whole);
    const bool in = w && (tid == 0 || (before < wanted(whole) && ex2(t) >= min_p));
    // the first in index order whose running weight passes the target: each sums what stands before it
    u64* left = list + NT;
    left[tid] = in ? item << 32 | w : 0;         // ~column above the weight
    __syncthreads();
    if (!in) return;
    u64 from = 0;
    whole = 0;
#pragma unroll 4
    for (int j = 0; j < n; ++j) {
      const u64 other = left[j];
      if (other >> 32 > (item & 0xffffffffu)) from += (uint32_t)other;
      whole += (uint32_t)other;
    }
    const u64 target = draw(u, whole);
    if (target >= from && target < from + w) P.tokens[row] = (long long)~(uint32_t)item;
    return;
  }

  Row<T, NT> r(team, span, dyn);
  e.m = r.row_max(r.own_max());
  if (e.m == -INFINITY) {
    if (r.rank == 0 && tid == 0) P.tokens[row] = -1;
    return;
  }
  if (e.m == INFINITY) {                         // infinite logits share all the weight
    for (int i = tid; i < span.n; i += NT)
#pragma unroll
      for (int v = 0; v < kUnit<T>; ++v)
        r.unit[i].v[v] = from_f32<T>(to_f32(r.unit[i].v[v]) == INFINITY ? 1.0f : -INFINITY);
    __syncthreads();
    e.m = 1.0f;
  }
  Cut cut{-INFINITY, 0x7fffffff, 0};
  const auto kept = [&](float x, int col) { return x > cut.x || (x == cut.x && col <= cut.last); };
  const auto all = [](float, int) { return true; };
  bool known = false;                            // `mine` is this CTA's kept weight
  u64 mine = 0;
  const bool by_rank = top_k > 0 && top_k < P.x.vocab;
  if (by_rank) {
    r.select<false>(all, [](float t) { return weight_of(t) ? 1u : 0u; }, e, [&](u64) { return (u64)top_k; }, cut, mine);
    r.settle(all, cut);
  }
  if (!(top_p >= 1.0f)) {
    Cut inner = cut;
    if (by_rank) {
      r.select<false>(kept, weight_of, e, wanted, inner, mine);
      r.settle(kept, inner);
      if (inner.x != cut.x || inner.last < cut.last) cut = inner;
    } else {
      r.select<true>(all, weight_of, e, wanted, cut, mine);
    }
    known = !(min_p > 0.0f);
  }
  const auto left = [&](float x, int col) -> u64 {
    const float t = e(x);
    return kept(x, col) && ex2(t) >= min_p ? weight_of(t) : 0;
  };
  // nothing below this passes min-p: a hundredth of an octave is far more than the rounding of t
  const float least = fmaxf(cut.x, e.m + (log2f(min_p) - 0.01f) / e.c);
  if (!known) {
    r.settle(all, cut);
    mine = r.left_sums(e, cut, min_p, least);
  }
  __syncthreads();
  r.exchange(mine);
  u64 total = 0, before = 0;
  for (int i = 0; i < (int)r.size; ++i) {
    if (i < (int)r.rank) before += r.got(i);
    total += r.got(i);
  }
  const u64 target = draw(u, total);
  if (target < before || target >= before + mine) return;      // the token is another CTA's
  if (known) {
    r.settle(all, cut);
    r.left_sums(e, cut, min_p, least);
  }
  const int at = r.locate(left, target - before);
  if (tid == 0) P.tokens[row] = at;
}

template <typename T>
__global__ void __launch_bounds__(kTopThreads, 4) top_kernel(const TopParams P) {
  constexpr int NT = kTopThreads;
  __shared__ Shared s;
  __shared__ u64 list[kListBytes<NT> / 8];
  Team<NT> team(s);
  const Span<T> span(P.x, blockIdx.x / team.size, team.rank, team.size);
  Listing<T, NT> l{team, span, list, P.k};
  const int n = l.gather(), row = blockIdx.x / team.size;
  if (team.rank != 0) return;
  T* values = reinterpret_cast<T*>(P.values) + (long long)row * P.k;
  int* indices = P.indices + (long long)row * P.k;
  for (int i = threadIdx.x; i < P.k; i += NT) {
    const int col = i < n ? (int)~(uint32_t)list[i] : -1;
    values[i] = col >= 0 ? span.p[col] : from_f32<T>(-INFINITY);
    indices[i] = col;
  }
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

template <typename T, int NT>
int launch_sample_threads(const SampleParams& P, int size, bool listed, cudaStream_t st) {
  size_t smem = listed ? 0 : (size_t)kWorkBytes + (size_t)((row_units(P.x) + size - 1) / size) * 16;
  if (smem < kListBytes<NT>) smem = kListBytes<NT>;
  const auto kernel = sample_kernel<T, NT>;
  static std::atomic<uint64_t> done{0};
  if (allow_shared(kernel, 160 * 1024, done) != cudaSuccess) return launch_status();
  return launch_clusters(kernel, P, size, NT, smem, st);
}
// CTAs a row for listing k: one lists the fewest logits; more as long as they all run at once (a second wave of a
// few costs more: 333 rows of 50,001 fp32 logits by one CTA each 28 us, by two 39) and their lists fit that of the first.
int listing_size(const LogitsRows& x, int k) {
  const int units = row_units(x);
  int size = 1;
  while (size < 8 && x.rows * size * 2 <= 4 * kSms && units > size * 2 * kTopThreads && 2 * size * k <= kList) size *= 2;
  return size;
}

}  // namespace

int launch_sample(const SampleParams& P, cudaStream_t st) {
  // Where every row is known to be listed (one top-k for all), nothing but the lists is on chip.  Otherwise as many
  // CTAs a row as keep its part within 64 KB; few rows take more, down to a unit a thread.
  const bool listed = !P.top_k && P.top_k_all > 0 && P.top_k_all <= kMaxListed;
  const int units = row_units(P.x);
  int size = 1;
  if (listed) {
    size = listing_size(P.x, P.top_k_all);
  } else {
    while (size < 8 && (units + size - 1) / size > 4096) size *= 2;
    while (size < 8 && P.x.rows * size < 2 * kSms && units > size * 256) size *= 2;
  }
  // Rows that are all on the GPU at once and are not just listed want threads: 512 (one row of 256,000 fp16
  // logits, top-p: 26 us, with 256 threads 38).  Many rows want three CTAs on an SM: 256 (512 rows of bf16, top-p:
  // 340 us, with 512 threads 390); so do lists (top-k 50 of one row: 9.5 us, with 512 threads 11.5).
  // Parts of which one fits an SM (fp32 rows over 768 KB) want 512 as well.
  const bool wide = !listed && ((P.x.rows * size <= 2 * kSms && units > size * 256) || units > size * 6144);
  return by_type(P.x.type, [&](auto t) {
    using T = decltype(t);
    return wide ? launch_sample_threads<T, 512>(P, size, listed, st) : launch_sample_threads<T, 256>(P, size, listed, st);
  });
}

int launch_top_logits(const TopParams& P, cudaStream_t st) {
  const int size = listing_size(P.x, P.k);
  return by_type(P.x.type, [&](auto t) { return launch_clusters(top_kernel<decltype(t)>, P, size, kTopThreads, 0, st); });
}

}  // namespace sq
