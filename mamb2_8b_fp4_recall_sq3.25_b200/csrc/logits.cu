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
// A cluster of 1..8 CTAs shares a row, each with its part of it in shared memory: the row is
// read from HBM once, every later pass runs on chip.  The CTAs exchange single numbers and
// histograms through distributed shared memory.
//
// Record (few tokens wanted: top_logits, top-k).  Every thread knows the largest of its logits.
// Each CTA finds the r-th largest of those, r = ceil(k / CTAs), to 16 bits of the key by
// counting; at least k logits are not below the least of these bounds, and few more
// (in rows that are not adversarial 1.1 k to 2 k).  Only threads whose largest passes look at their
// logits again.  The candidates go to the first CTA, which ranks them by comparing all with all.
//
// Cut (top-p, large k).  A histogram over 256 steps of 1/8 octave of y, with exact weights, finds
// the step in which the running weight reaches what is wanted; the members of that step are
// narrowed by histograms over their keys until one key is left.  What is kept is then "logit
// above the cut, or equal and index not above the last one kept".
#include "logits.cuh"
#include "logits_util.cuh"
#include <type_traits>

namespace sq {
namespace {

constexpr int NT = 512, NW = NT / 32;
typedef unsigned long long u64;

constexpr int kSteps = 256;                      // histogram over -8 log2 y
constexpr int kCols = 8;                         // copies of it, by lane: fewer lanes meet in one word
// A word of the histogram sums the low 19 bits of at most NT / 8 threads x 72 elements: < 2^32.
// The upper 12 bits are not 0 for y >= 2^-12 only, the first 97 steps.
constexpr int kLowBits = 19, kHighSteps = 98;
constexpr int kFine = 256, kFineCols = 4, kFineLowBits = 18;   // narrowing: 128 threads x 72 x 2^18 < 2^32
constexpr int kListBytes = kSteps * kCols * 4;   // candidates: 1024 of 8 bytes, or 2048 where k > 256
constexpr int kMembers = kHighSteps * kCols * 4 / 2;           // members of a step held as 16-bit positions

struct Cut { float x; int last; };               // kept: above x, or equal and column <= last

struct Shared {
  u64 slot[2][8];
  u64 part[NW];
  float fpart[NW];
  u64 sums[kSteps];                              // this CTA's histogram
  u64 scan[NW];
  u64 found_above, found_mine;
  int found, count, pick;
  uint32_t key_low, key_high;
  uint32_t weight[1024];
};

__device__ __forceinline__ u64 warp_sum(u64 v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// One CTA's part of a row in shared memory.
template <typename T>
struct Part {
  Unit<T>* unit;
  int n, col0;                                   // units; column of the first element (may be < 0)
  __device__ int col(int i, int v) const { return col0 + i * kUnit<T> + v; }
};

template <typename T>
struct Row {
  Shared& s;
  Part<T> d;
  unsigned char* work;                           // histogram / candidates / members
  uint32_t rank, size;
  int tid, phase;

  __device__ Row(Shared& s, unsigned char* dyn, const LogitsRows& x, int work_bytes)
      : s(s), work(dyn), rank(cluster_rank()), size(cluster_size()), tid(threadIdx.x), phase(0) {
    cluster_arrive();
    const T* p = reinterpret_cast<const T*>(x.data) + (long long)(blockIdx.x / size) * x.stride;
    const int off = (int)((uintptr_t)p & 15) / (int)sizeof(T);
    const int units = (off + x.vocab + kUnit<T> - 1) / kUnit<T>;
    const int per = (units + (int)size - 1) / (int)size, u0 = (int)rank * per;
    d.unit = reinterpret_cast<Unit<T>*>(dyn + work_bytes);
    d.n = max(0, min(units, u0 + per) - u0);
    d.col0 = u0 * kUnit<T> - off;
    for (int i = tid; i < d.n; i += NT) {
      const int c = d.col(i, 0);
      if (c >= 0 && c + kUnit<T> <= x.vocab) {
        cp_async16(d.unit + i, p + c);
      } else {                                   // the row's ragged ends
        Unit<T> u;
#pragma unroll
        for (int v = 0; v < kUnit<T>; ++v)
          u.v[v] = c + v >= 0 && c + v < x.vocab ? p[c + v] : from_f32<T>(-INFINITY);
        d.unit[i].q = u.q;
      }
    }
    cp_async_wait_all();                         // each thread's own units
    cluster_wait();
  }

  // f(x, column) over this thread's elements.
  template <typename F>
  __device__ void each(F f) const {
    for (int i = tid; i < d.n; i += NT) {
      Unit<T> u;
      u.q = d.unit[i].q;
#pragma unroll
      for (int v = 0; v < kUnit<T>; ++v) f(to_f32(u.v[v]), i, v);
    }
  }
  __device__ float own_max() const {
    float m = -INFINITY;
    for (int i = tid; i < d.n; i += NT) {
      Unit<T> u;
      u.q = d.unit[i].q;
      m = fmaxf(m, unit_max(u));
    }
    return m;
  }
  __device__ void barrier() { cluster_arrive(); cluster_wait(); }
  // Hands `v` (the same in every thread that stores) to all CTAs; afterwards got(r) is CTA r's.
  __device__ void exchange(u64 v) {
    phase ^= 1;
    if (tid < (int)size) remote_store(remote_smem(&s.slot[phase][rank], tid), v);
    barrier();
  }
  __device__ u64 got(int r) const { return s.slot[phase][r]; }
  __device__ u64 block_sum(u64 v) {
    v = warp_sum(v);
    __syncthreads();
    if ((tid & 31) == 0) s.part[tid >> 5] = v;
    __syncthreads();
    u64 t = 0;
    for (int i = 0; i < NW; ++i) t += s.part[i];
    return t;
  }
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

  // Sums of w(x, col) over contiguous stretches, one a warp, in s.part; returns this CTA's total.
  template <typename W>
  __device__ u64 stretch_sums(W w) {
    const int len = (d.n + NW - 1) / NW, i0 = (tid >> 5) * len, i1 = min(d.n, i0 + len);
    u64 sum = 0;
    for (int i = i0 + (tid & 31); i < i1; i += 32) {
      Unit<T> u;
      u.q = d.unit[i].q;
#pragma unroll
      for (int v = 0; v < kUnit<T>; ++v) sum += w(to_f32(u.v[v]), d.col(i, v));
    }
    sum = warp_sum(sum);
    __syncthreads();
    if ((tid & 31) == 0) s.part[tid >> 5] = sum;
    __syncthreads();
    u64 t = 0;
    for (int i = 0; i < NW; ++i) t += s.part[i];
    return t;
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
          u.q = d.unit[i + lane].q;
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

  // Lower bound of the k-th largest logit of the row (finite): at least k logits, or all that are
  // not -inf, are not below it.
  __device__ float bound(float own, int k) {
    const uint32_t key = order_key(own + 0.0f) >> 16;
    const int r = (k + (int)size - 1) / (int)size;
    uint32_t t = 0;
#pragma unroll 1
    for (int bit = 15; bit >= 0; --bit)
      if (__syncthreads_count(key >= (t | (1u << bit))) >= r) t |= 1u << bit;
    exchange(t);
    for (int i = 0; i < (int)size; ++i) t = min(t, (uint32_t)got(i));
    return key_logit(max(t << 16, kKeyLowest));
  }
  // Logits from `least` up, as key << 32 | ~column, in the work area of CTA 0 (nothing is written if
  // there are more than `most`); returns their number.
  __device__ int gather(float own, float least, int most) {
    if (tid == 0) s.count = 0;
    __syncthreads();
    int mine = 0, at = 0;
    if (own >= least) {
      each([&](float x, int, int) { mine += x >= least; });
      at = atomicAdd(&s.count, mine);
    }
    __syncthreads();
    exchange((u64)s.count);
    int n = 0;
    for (int r = 0; r < (int)size; ++r) {
      if (r < (int)rank) at += (int)got(r);
      n += (int)got(r);
    }
    if (n > most) return n;
    if (own >= least) {
      const uint32_t list = remote_smem(work, 0);
      each([&](float x, int i, int v) {
        if (x >= least) {
          remote_store(list + 8u * at, (u64)order_key(x + 0.0f) << 32 | (uint32_t)~d.col(i, v));
          ++at;
        }
      });
    }
    barrier();
    return n;
  }

  // Scan of `total` (thread i < 256: weight of histogram entry i over the row, `mine` this CTA's) for the
  // first entry at which the running weight reaches need(whole weight), starting from `above`; adds the
  // entries before it to `above` and `mine_above`.  Returns -1 if it is not reached.
  template <typename N>
  __device__ int crossing(u64 total, u64 mine, N need_of, u64& above, u64& mine_above) {
    const int warp = tid >> 5, lane = tid & 31;
    u64 run = total, own = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 a = __shfl_up_sync(0xffffffffu, run, o), b = __shfl_up_sync(0xffffffffu, own, o);
      if (lane >= o) { run += a; own += b; }
    }
    __syncthreads();
    if (lane == 31 && warp < kSteps / 32) { s.scan[warp] = run; s.part[warp] = own; }
    if (tid == 0) s.found = -1;
    __syncthreads();
    u64 whole = 0;
    for (int i = 0; i < kSteps / 32; ++i) whole += s.scan[i];
    const u64 need = need_of(whole);
    if (tid < kSteps) {
      u64 before = above, mb = mine_above;
      for (int i = 0; i < warp; ++i) { before += s.scan[i]; mb += s.part[i]; }
      if (before + run >= need && before + run - total < need) {
        s.found = tid;
        s.found_above = before + run - total;
        s.found_mine = mb + own - mine;
      }
    }
    __syncthreads();
    if (s.found >= 0) { above = s.found_above; mine_above = s.found_mine; }
    return s.found;
  }

  // The cut after the first tokens of the order whose weights w(x) reach need(whole weight), among
  // elements with kept(x, col).  w depends on x alone and is below 2^31 + 1; m is the largest logit, c the
  // scale of the steps.  False: the whole weight does not reach it.
  // kept_here: this CTA's share of the weight that is kept.
  template <typename K, typename W, typename N>
  __device__ bool select(K kept, W w, float m, float c, N need_of, Cut& cut, u64& kept_here) {
    constexpr int SH = std::is_same<T, __half>::value ? 13 : std::is_same<T, __nv_bfloat16>::value ? 16 : 0;
    uint32_t* low = reinterpret_cast<uint32_t*>(work);
    uint32_t* high = low + kSteps * kCols;
    uint16_t* members = reinterpret_cast<uint16_t*>(high);
    const auto step = [&](float x) {             // rint(-8 t), capped; NaN and -inf fall in the last
      return min((uint32_t)(__float_as_uint(fmaf(fmaxf(__fmul_rn(x - m, c), -32.0f), -8.0f, 8388608.0f)) & 0x7fffffu),
                 (uint32_t)(kSteps - 1));
    };
    __syncthreads();
    for (int i = tid; i < (kSteps + kHighSteps) * kCols; i += NT) low[i] = 0;
    __syncthreads();
    each([&](float x, int i, int v) {
      const uint32_t q = w(x);
      if (q && kept(x, d.col(i, v))) {
        const uint32_t b = step(x) * kCols + (tid & (kCols - 1));
        atomicAdd(low + b, q & ((1u << kLowBits) - 1));
        if (q >> kLowBits) atomicAdd(high + b, q >> kLowBits);
      }
    });
    __syncthreads();
    u64 mine = 0, total = 0;
    if (tid < kSteps) {
      for (int i = 0; i < kCols; ++i) {
        mine += low[tid * kCols + i];
        if (tid < kHighSteps) mine += (u64)high[tid * kCols + i] << kLowBits;
      }
      s.sums[tid] = mine;
    }
    barrier();
    if (tid < kSteps)
      for (int r = 0; r < (int)size; ++r) total += remote_load(remote_smem(&s.sums[tid], r));
    u64 above = 0, mine_above = 0, need = 0;
    const int at = crossing(total, mine, [&](u64 whole) { return need = need_of(whole); }, above, mine_above);
    if (at < 0) { barrier(); return false; }
    // the step's members, a list of positions (the whole part again where they are too many), and
    // the range of their keys
    if (tid == 0) { s.count = 0; s.key_low = 0xffffffffu; s.key_high = 0; }
    __syncthreads();
    const auto member = [&](float x, int i, int v) { return step(x) == (uint32_t)at && w(x) && kept(x, d.col(i, v)); };
    uint32_t lo = 0xffffffffu, hi = 0;
    each([&](float x, int i, int v) {
      if (member(x, i, v)) {
        const int k = atomicAdd(&s.count, 1);
        if (k < kMembers) members[k] = (uint16_t)(i * kUnit<T> + v);
        const uint32_t key = order_key(x + 0.0f) >> SH;
        lo = min(lo, key);
        hi = max(hi, key);
      }
    });
    lo = __reduce_min_sync(0xffffffffu, lo);
    hi = __reduce_max_sync(0xffffffffu, hi);
    if ((tid & 31) == 0 && lo <= hi) { atomicMin(&s.key_low, lo); atomicMax(&s.key_high, hi); }
    __syncthreads();
    const int listed = s.count;
    exchange((u64)s.key_high << 32 | s.key_low);
    for (int r = 0; r < (int)size; ++r) {
      lo = min(r ? lo : 0xffffffffu, (uint32_t)got(r));
      hi = max(r ? hi : 0u, (uint32_t)(got(r) >> 32));
    }
    const auto each_member = [&](auto f) {
      if (listed <= kMembers) {
        for (int k = tid; k < listed; k += NT) f(to_f32(d.unit[members[k] / kUnit<T>].v[members[k] % kUnit<T>]));
      } else {
        each([&](float x, int i, int v) { if (member(x, i, v)) f(x); });
      }
    };
    uint32_t key;
    int entry;
    u64 key_before = 0;                          // weight of that key in the CTAs before this one
    for (;;) {
      int shift = 0;
      while (((hi - lo) >> shift) >= (uint32_t)kFine) ++shift;
      uint32_t* flow = low;
      uint32_t* fhigh = low + kFine * kFineCols;
      __syncthreads();
      for (int i = tid; i < 2 * kFine * kFineCols; i += NT) low[i] = 0;
      barrier();                                 // and every CTA has read the sums of the round before
      each_member([&](float x) {
        const uint32_t k = order_key(x + 0.0f) >> SH;
        if (k < lo || k > hi) return;            // decided by an earlier round
        const uint32_t b = ((hi - k) >> shift) * kFineCols + (tid & (kFineCols - 1)), q = w(x);
        atomicAdd(flow + b, q & ((1u << kFineLowBits) - 1));
        if (q >> kFineLowBits) atomicAdd(fhigh + b, q >> kFineLowBits);
      });
      __syncthreads();
      mine = total = 0;
      if (tid < kFine) {
        for (int i = 0; i < kFineCols; ++i)
          mine += flow[tid * kFineCols + i] + ((u64)fhigh[tid * kFineCols + i] << kFineLowBits);
        s.sums[tid] = mine;
      }
      barrier();
      if (tid < kFine)
        for (int r = 0; r < (int)size; ++r) total += remote_load(remote_smem(&s.sums[tid], r));
      entry = crossing(total, mine, [&](u64) { return need; }, above, mine_above);
      if (shift == 0) {
        key = hi - entry;
        for (int r = 0; r < (int)rank; ++r) key_before += remote_load(remote_smem(&s.sums[entry], r));
        break;
      }
      hi = hi - ((uint32_t)entry << shift);
      const uint32_t width = (1u << shift) - 1;
      if (hi - lo > width) lo = hi - width;
    }
    const u64 here = s.sums[entry];
    // the key of 16-bit types stands for one logit: its low bits are those of an exact value
    const float x = key_logit(SH == 0 ? key : (key << SH) | ((key << SH) & 0x80000000u ? 0u : (1u << SH) - 1u));
    const u64 each_w = w(x), wanted = (need - above + each_w - 1) / each_w, earlier = key_before / each_w;
    const u64 ties = here / each_w;
    cut.x = x;
    u64 taken = ties;
    if (wanted >= earlier + ties) {
      cut.last = 0x7fffffff;
    } else if (wanted <= earlier) {
      cut.last = -1;
      taken = 0;
    } else {
      taken = wanted - earlier;
      const auto tie = [&](float v, int col) -> u64 { return v == x && kept(v, col) ? 1 : 0; };
      stretch_sums(tie);
      cut.last = locate(tie, taken - 1);
    }
    kept_here = mine_above + taken * each_w;
    barrier();                                   // sums are read before anybody goes on
    return true;
  }
};

template <typename T>
__global__ void __launch_bounds__(NT, 2) sample_kernel(const SampleParams P) {
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ Shared s;
  constexpr int kWork = (kSteps + kHighSteps) * kCols * 4;
  Row<T> r(s, dyn, P.x, kWork);
  const int row = blockIdx.x / r.size, tid = threadIdx.x;
  const float temperature = P.temperature ? P.temperature[row] : P.temperature_all;
  const int top_k = P.top_k ? P.top_k[row] : P.top_k_all;
  const float top_p = P.top_p ? P.top_p[row] : P.top_p_all;
  const float min_p = fminf(P.min_p ? P.min_p[row] : P.min_p_all, 1.0f);
  const double u = P.uniform[row];
  float own = r.own_max();
  float m = r.row_max(own);
  if (m == -INFINITY) {
    if (r.rank == 0 && tid == 0) P.tokens[row] = -1;
    return;
  }
  if (m == INFINITY) {                           // infinite logits share all the weight
    __syncthreads();
    for (int i = tid; i < r.d.n; i += NT)
#pragma unroll
      for (int v = 0; v < kUnit<T>; ++v)
        r.d.unit[i].v[v] = from_f32<T>(to_f32(r.d.unit[i].v[v]) == INFINITY ? 1.0f : -INFINITY);
    __syncthreads();
    m = 1.0f;
    own = own == INFINITY ? 1.0f : -INFINITY;
  }
  const auto draw = [&](u64 total) {
    const long long t = (long long)(u * (double)total);
    return t < 0 ? 0 : ((u64)t >= total ? total - 1 : (u64)t);
  };
  // finds the CTA that holds `target` and the token in it; `mine`: this CTA's weight, in s.part if `summed`
  const auto finish = [&](auto w, u64 mine, bool summed, bool greedy) {
    __syncthreads();
    r.exchange(mine);
    u64 total = 0, before = 0;
    for (int i = 0; i < (int)r.size; ++i) {
      if (i < (int)r.rank) before += r.got(i);
      total += r.got(i);
    }
    const u64 target = greedy ? 0 : draw(total);
    if (target < before || target >= before + mine) return;
    if (!summed) r.stretch_sums(w);
    const int at = r.locate(w, target - before);
    if (tid == 0) P.tokens[row] = at;
  };
  if (!(temperature > 0.0f)) {
    const auto largest = [&](float x, int) -> u64 { return x == m; };
    const u64 mine = r.stretch_sums(largest);
    finish(largest, mine, true, true);
    return;
  }
  const float c = fminf(__fdiv_rn(kLog2e, temperature), 3.4028234e38f);      // finite: 0 c stays 0
  const auto power = [&](float x) { return x == m ? 1.0f : ex2(__fmul_rn(x - m, c)); };
  const auto weight = [&](float x) { return __float2uint_rn(power(x) * 2147483648.0f); };
  Cut cut{-INFINITY, 0x7fffffff};
  const auto kept = [&](float x, int col) { return x > cut.x || (x == cut.x && col <= cut.last); };
  bool known = false;                            // `mine` is this CTA's kept weight
  u64 mine = 0;
  if (top_k > 0 && top_k < P.x.vocab) {
    const int most = kListBytes / 8;
    if (top_k <= most / 2) {
      const float least = r.bound(own, top_k);
      const int n = r.gather(own, least, most);
      if (n <= most) {                           // all that is left is on CTA 0's list
        if (r.rank != 0) return;
        const u64* list = reinterpret_cast<const u64*>(r.work);
        for (int i = tid; i < n; i += NT) s.weight[i] = weight(key_logit((uint32_t)(list[i] >> 32)));
        __syncthreads();
        constexpr int N = kListBytes / 8 / NT;
        u64 item[N] = {}, before[N];
        uint32_t w[N];
        int place[N];
        u64 z = 0;
#pragma unroll
        for (int a = 0; a < N; ++a) {
          const int i = tid + a * NT;
          before[a] = 0;
          place[a] = top_k;
          w[a] = 0;
          if (i < n) {
            item[a] = list[i];
            int rank = 0;
            u64 sum = 0;
            for (int j = 0; j < n; ++j)
              if (list[j] > item[a]) { ++rank; sum += s.weight[j]; }
            place[a] = rank;
            before[a] = sum;
            w[a] = rank < top_k ? s.weight[i] : 0;
            z += w[a];
          }
        }
        z = r.block_sum(z);
        const double limit = (double)top_p * (double)z;
        u64 left = 0;
#pragma unroll
        for (int a = 0; a < N; ++a) {
          const bool in = place[a] == 0 || ((top_p >= 1.0f || (double)before[a] < limit) &&
                                            power(key_logit((uint32_t)(item[a] >> 32))) >= min_p);
          if (!in) w[a] = 0;
          if (tid + a * NT < n) s.weight[tid + a * NT] = w[a];
          left += w[a];
        }
        left = r.block_sum(left);
        const u64 target = draw(left);
#pragma unroll
        for (int a = 0; a < N; ++a)
          if (w[a]) {
            const uint32_t col = ~(uint32_t)item[a];
            u64 sum = 0;
            for (int j = 0; j < n; ++j)
              if (~(uint32_t)list[j] < col) sum += s.weight[j];
            if (target >= sum && target < sum + w[a]) P.tokens[row] = (long long)col;
          }
        return;
      }
    }
    u64 ignored;
    r.select([](float, int) { return true; }, [&](float x) { return weight(x) ? 1u : 0u; }, m, c,
             [&](u64) { return (u64)top_k; }, cut, ignored);
  }
  if (!(top_p >= 1.0f)) {
    Cut inner;
    r.select(kept, weight, m, c, [&](u64 z) {
      const double limit = (double)top_p * (double)z;          // kept: weight before it below this, the first always
      const u64 need = limit > 1.0 ? (u64)ceil(limit) : 1;
      return need > z ? z : need;
    }, inner, mine);
    if (inner.x != cut.x || inner.last < cut.last) cut = inner;
    known = true;
  }
  const auto left = [&](float x, int col) -> u64 { return kept(x, col) && power(x) >= min_p ? weight(x) : 0; };
  if (!known || min_p > 0.0f) mine = r.stretch_sums(left);
  finish(left, mine, !known || min_p > 0.0f, false);
}

template <typename T>
__global__ void __launch_bounds__(NT, 2) top_kernel(const TopParams P, int most) {
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ Shared s;
  Row<T> r(s, dyn, P.x, most * 8);
  const int row = blockIdx.x / r.size, tid = threadIdx.x;
  const T* p = reinterpret_cast<const T*>(P.x.data) + (long long)row * P.x.stride;
  const float own = r.own_max();
  int n = r.gather(own, r.bound(own, P.k), most);
  if (n > most) {
    // many equal logits, or k near the width: the k-th key by halving, counted over the cluster
    u64 all = 0;
    r.each([&](float x, int, int) { all += x > -INFINITY; });
    all = r.block_sum(all);
    __syncthreads();
    r.exchange(all);
    all = 0;
    for (int i = 0; i < (int)r.size; ++i) all += r.got(i);
    const int k = (int)min((u64)P.k, all);
    uint32_t key = 0;
    u64 above = 0;
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t t = key | (1u << bit);
      u64 c = 0;
      r.each([&](float x, int, int) { c += x > -INFINITY && order_key(x + 0.0f) >= t; });
      c = r.block_sum(c);
      __syncthreads();
      r.exchange(c);
      c = 0;
      for (int i = 0; i < (int)r.size; ++i) c += r.got(i);
      if (c >= (u64)k) key = t;
      else above = c;                            // logits above the final key
    }
    const float x0 = key_logit(key);
    const auto tie = [&](float x, int) -> u64 { return x == x0; };
    const u64 ties = r.stretch_sums(tie);
    __syncthreads();
    r.exchange(ties);
    u64 earlier = 0;
    for (int i = 0; i < (int)r.rank; ++i) earlier += r.got(i);
    const u64 wanted = k - above;
    Cut cut{x0, 0x7fffffff};
    if (wanted <= earlier) cut.last = -1;
    else if (wanted < earlier + ties) cut.last = r.locate(tie, wanted - earlier - 1);
    // as gather(), for what the cut keeps
    const auto kept = [&](float x, int col) { return x > cut.x || (x == cut.x && col <= cut.last); };
    if (tid == 0) s.count = 0;
    __syncthreads();
    int mine = 0, at;
    r.each([&](float x, int i, int v) { mine += kept(x, r.d.col(i, v)); });
    at = atomicAdd(&s.count, mine);
    __syncthreads();
    r.exchange((u64)s.count);
    for (int i = 0; i < (int)r.rank; ++i) at += (int)r.got(i);
    const uint32_t list = remote_smem(r.work, 0);
    r.each([&](float x, int i, int v) {
      if (kept(x, r.d.col(i, v))) {
        remote_store(list + 8u * at, (u64)order_key(x + 0.0f) << 32 | (uint32_t)~r.d.col(i, v));
        ++at;
      }
    });
    r.barrier();
    n = k;
  }
  if (r.rank != 0) return;
  const u64* list = reinterpret_cast<const u64*>(r.work);
  T* values = reinterpret_cast<T*>(P.values) + (long long)row * P.k;
  int* indices = P.indices + (long long)row * P.k;
  for (int i = tid; i < n; i += NT) {
    const u64 item = list[i];
    int place = 0;
    for (int j = 0; j < n; ++j) place += list[j] > item;
    if (place < P.k) {
      const int col = (int)~(uint32_t)item;
      values[place] = p[col];
      indices[place] = col;
    }
  }
  for (int i = n + tid; i < P.k; i += NT) {
    values[i] = from_f32<T>(-INFINITY);
    indices[i] = -1;
  }
}

template <typename K, typename... A>
int launch_clusters(K kernel, const LogitsRows& x, int work_bytes, cudaStream_t st, A... args) {
  const int bytes = x.type == kLogitsF32 ? 4 : 2;
  const int units = (x.vocab * bytes + 15) / 16 + 1;             // one more where the row starts inside a unit
  // As many CTAs a row as keep its part within 64 KB; few rows take more, down to a unit a thread.
  int size = 1;
  while (size < 8 && (units + size - 1) / size > 4096) size *= 2;
  while (size < 8 && x.rows * size < 2 * 148 && units > size * NT) size *= 2;
  const size_t smem = (size_t)work_bytes + (size_t)((units + size - 1) / size) * 16;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024) != cudaSuccess) return launch_status();
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = size; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3((unsigned)x.rows * size);
  cfg.blockDim = dim3(NT);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, kernel, args...);
  return launch_status();
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

int launch_sample(const SampleParams& P, cudaStream_t st) {
  return by_type(P.x.type, [&](auto t) {
    return launch_clusters(sample_kernel<decltype(t)>, P.x, (kSteps + kHighSteps) * kCols * 4, st, P);
  });
}

int launch_top_logits(const TopParams& P, cudaStream_t st) {
  const int most = P.k <= 256 ? 1024 : 2048;
  return by_type(P.x.type, [&](auto t) {
    return launch_clusters(top_kernel<decltype(t)>, P.x, most * 8, st, P, most);
  });
}

}  // namespace sq
