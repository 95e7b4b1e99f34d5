// One token per row of logits under temperature, top-k, top-p and min-p, each
// row with its own settings, from given uniform numbers.  The filters of the
// reference's sampler (aceflow-core/src/cpu/sampler.rs:83-180) and min-p
// (Nguyen et al. 2024), which the reference lacks.
//
// Order a row's tokens by logit, largest first, equal ones by lowest index;
// w_i = exp((l_i - max) / temperature), F the running sum of w in that order.
// Every filter keeps a prefix of that order:
//   top-k  the first k;  Z = F at its end
//   top-p  through the first place where F > top_p Z
//   min-p  while w >= min_p (the largest w is 1)
// and the draw is the first place where F >= u M, M = F at the shortest
// prefix's end.  So the row is never sorted.  A cluster of CTAs holds it in
// shared memory, one slice each (one read of the logits from HBM), and
//   1. finds the maximum;
//   2. with top-k: counts the tokens in bins of 1/16 octave of w and takes the
//      bins through the one that holds the k-th; else: sums w, which bounds
//      from below the w of any token that can still matter (a token below
//      (1 - top_p) Z / V lies behind the crossing: all such tokens together
//      weigh less than (1 - top_p) Z);
//   3. if at most kList tokens are left, the first CTA sorts them, sums along
//      them and reads every place off; this is the usual case;
//   4. else (a broad nucleus) the masses go into the same bins, a place's bin
//      follows from their running sum, and only that bin's tokens are sorted;
//   5. else (a bin of more than kList tokens: great numbers of equal or nearly
//      equal logits, or a top_k above kList) every place is found by
//      descending the digits of its key over histograms.
//
// Masses are whole numbers in units of 2^-44, w to 31 significant bits (less
// than 2^-29 of itself off), in 64 bits: their sums do not depend on any
// order, so a row's token is the same in every run and in every launch shape.
//
// Bound: a long row by instructions (about 35 per token for the mass; two
// histogram additions where step 4 runs), a short one by the chain of cluster
// barriers.
#include "common.cuh"
#include "sm100.cuh"

namespace {

using u64 = unsigned long long;
using sm100::cluster_ctarank;
constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCtas = 8;              // CTAs of a row's cluster
constexpr int kList = 2048;              // tokens that are sorted at once
constexpr int kBins = 46 * 16;           // w down to 2^-46 in sixteenths of an octave
constexpr int kBinRoom = (kBins + kThreads) / kThreads * kThreads;
constexpr u64 kOne = 1ull << 44;         // the mass of the largest logit

// A logit as it is kept: NaN counts as -inf (it is never drawn), -0 is +0.
__device__ __forceinline__ float kept(float x) { return x == x ? x + 0.0f : -INFINITY; }
// Logit to key: larger key, larger logit.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

struct SampleParams {
  const void *logits;
  int b16;
  int64_t ld;
  int V, slice;  // tokens of a CTA: slice (a multiple of 8), the last ones fewer
  int vec;       // rows allow 16-byte loads
  const int32_t *ctx;
  int64_t ctx_stride;
  int ctx_len;
  const float *temperature, *top_p, *min_p, *penalty;  // per row, or NULL: the value for all
  const int32_t *top_k;
  float temperature_all, top_p_all, min_p_all, penalty_all;
  int top_k_all;
  const float *uniforms;
  int32_t *token;
  float *logprob;
};

// Shared memory of a CTA, byte offsets: this with the slice's logits, then the
// bits of the context's tokens.  It is addressed by 32-bit shared addresses throughout, the
// same for this CTA's memory and (after mapa) another's.
struct Layout {
  static constexpr uint32_t list = 0;                      // u64 [kList]: (~key, index), ascending is the order
  static constexpr uint32_t run = list + 8 * kList;        // u64 [kList]: running mass along the list; step 5's sums
  static constexpr uint32_t lo = run;                      // u32 [kBinRoom], hi alike: this CTA's bins, done with
  static constexpr uint32_t hi = lo + 4 * kBinRoom;        //   before a list is ordered
  static constexpr uint32_t bins = run + 8 * kList;        // u64 [kBinRoom]: running masses (counts) of the row's bins
  static constexpr uint32_t power = bins + 8 * kBinRoom;   // double [16]: 2^(44 - j / 16)
  static constexpr uint32_t slot = power + 8 * 16;           // u64 [2][kMaxCtas]
  static constexpr uint32_t warp = slot + 8 * 2 * kMaxCtas;  // u64 [kWarps]
  static constexpr uint32_t before = warp + 8 * kWarps;      // u64 [2]
  static constexpr uint32_t listed = before + 16;            // u32, then found
  static constexpr uint32_t found = listed + 4;
  static constexpr uint32_t logits = found + 12;  // float [slice]
};
static_assert(Layout::logits % 16 == 0, "logits are read sixteen bytes at a time");
static_assert(8 * kList >= 8 * kBinRoom, "the bins lie where the running masses come");

__device__ __forceinline__ u64 lds64(uint32_t a) {
  u64 v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void sts64(uint32_t a, u64 v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(a), "l"(v) : "memory");
}
__device__ __forceinline__ void sts32(uint32_t a, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(a), "r"(v) : "memory");
}
__device__ __forceinline__ uint32_t add32(uint32_t a, uint32_t v) {
  uint32_t old;
  asm volatile("atom.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(old) : "r"(a), "r"(v) : "memory");
  return old;
}
// This CTA's memory alone: the additions whose old value nobody needs, and vectors.
__device__ __forceinline__ void red32(uint32_t a, uint32_t v) {
  asm volatile("red.shared.add.u32 [%0], %1;" ::"r"(a), "r"(v) : "memory");
}
__device__ __forceinline__ void red64(uint32_t a, u64 v) {
  asm volatile("red.shared.add.u64 [%0], %1;" ::"r"(a), "l"(v) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void sts128(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
// The same address in the cluster's CTA `rank`.
__device__ __forceinline__ uint32_t in_cta(uint32_t a, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
  return r;
}
__device__ __forceinline__ uint32_t cluster_ctas() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
// All threads of the cluster, whether or not their warps have reconverged.
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive;\n\tbarrier.cluster.wait;" ::: "memory");
}

// The mass of a token: w = 2^-t, t = (max - l) log2(e) / T, in 64 bits.  With k
// the whole number next to 16 t and f = t - k / 16, 2^-f is the Taylor series of
// exp(-f ln 2) to its fourth power (|f| <= 1/32: 2^-34 off), 2^(-(k mod 16) / 16)
// comes from a table whose 16 doubles lie in 32 different banks, and the octave
// k / 16 goes into the exponent.  The 64-bit pipe has half the fp32 rate and
// nothing else to do here.
struct Weigher {
  float top, ch;
  double dtop, c;
  uint32_t power;
  // t in fp32: never smaller for a smaller logit.
  __device__ __forceinline__ float lead(float x) const { return __fmul_rn(top - x, ch); }
  __device__ __forceinline__ static bool some(float t) { return t < 46.0f; }
  // k, and 31 bits of w with the shift that makes them the mass, one shift for
  // all tokens of a k.  Only for some(lead(x)).
  __device__ __forceinline__ uint32_t bits(float x, int &k, int &shift) const {
    const double t = (dtop - (double)x) * c;
    const double r = t + 422212465065984.0;  // 1.5 * 2^48: sixteenths stand in the low bits
    k = __double2loint(r);
    const double f = t - (r - 422212465065984.0);
    double q = fma(f, 0.009618129107628477, -0.05550410866482158);  // (-ln 2)^n / n!, n = 4 .. 1
    q = fma(f, q, 0.24022650695910072);
    q = fma(f, q, -0.6931471805599453);
    const int octave = k >> 4;
    shift = max(13 - octave, 0);
    u64 table;  // not volatile: nothing writes it any more, so loads of several tokens may overlap
    asm("ld.shared.u64 %0, [%1];" : "=l"(table) : "r"(power + 8 * (k & 15)));
    const double w = __hiloint2double((int)(table >> 32) - (octave << 20), (int)(uint32_t)table);
    // w 2^-f, behind 2^(52 + shift): the bits above the shift stand in the low word
    return (uint32_t)__double2loint(fma(w, f * q, w + __hiloint2double(0x43300000 + (shift << 20), 0)));
  }
  __device__ __forceinline__ u64 operator()(float x) const {
    if (!some(lead(x))) return 0;
    int k, shift;
    const uint32_t q = bits(x, k, shift);
    return (u64)__funnelshift_l(q, 0u, shift) << 32 | (q << shift);
  }
  // log(w / mass): w's logarithm needs none.
  __device__ __forceinline__ float log_share(float x, u64 mass) const {
    return (float)(((double)x - dtop) * c * 0.6931471805599453 - log((double)mass * (1.0 / (double)kOne)));
  }
  // The sixteenth of an octave by t's fp32 form, for counts.
  __device__ __forceinline__ int bin(float x) const {
    const float t = lead(x);
    return some(t) ? __float_as_int(__fadd_rd(t * 16.0f, 12582912.0f)) - 0x4b400000 : kBins;
  }
  // Bounds on the logits of all tokens with t below (above) the given one.
  __device__ __forceinline__ float logit_below(double t) const {
    return fmaxf(__double2float_rd(dtop - (t + 1.0 / 64) / c), -3.4028235e38f);
  }
  __device__ __forceinline__ float logit_above(double t) const {
    return __double2float_ru(dtop - (t - 1.0 / 64) / c);
  }
};

// A place in the order: the first `rank` (from 1) of the tokens with that key,
// and the mass of all keys above it.
struct Place {
  uint32_t key;
  unsigned rank;
  u64 above;
};
__device__ __forceinline__ Place shorter(const Place &a, const Place &b) {
  return a.key > b.key || (a.key == b.key && a.rank <= b.rank) ? a : b;
}

struct Row {
  uint32_t sm;  // this CTA's shared memory
  int n, base, ctas, rank;  // tokens of this CTA, their first index, CTAs of the row, this one's place
  int flip = 0;

  // This CTA's value to every CTA of the row, from warp 0; then a cluster
  // barrier.  The slots alternate, so the next exchange cannot overtake a reader.
  __device__ __forceinline__ uint32_t exchange(u64 v) {
    const uint32_t slot = sm + Layout::slot + 8 * kMaxCtas * flip;
    flip ^= 1;
    if (threadIdx.x < (unsigned)ctas) sts64(in_cta(slot + 8 * rank, threadIdx.x), v);
    cluster_barrier();
    return slot;
  }
  // The sum over all threads of the row.
  __device__ u64 total(u64 v) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (lane == 0) sts64(sm + Layout::warp + 8 * (threadIdx.x >> 5), v);
    __syncthreads();
    if (threadIdx.x < 32) {
      v = lane < kWarps ? lds64(sm + Layout::warp + 8 * lane) : 0;
#pragma unroll
      for (int o = kWarps / 2; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
      v = __shfl_sync(0xffffffffu, v, 0);
    }
    const uint32_t slot = exchange(v);
    v = 0;
    for (int c = 0; c < ctas; ++c) v += lds64(slot + 8 * c);
    return v;
  }
  // The largest key over all threads of the row.
  __device__ uint32_t largest(uint32_t v) {
    const int lane = threadIdx.x & 31;
    v = __reduce_max_sync(0xffffffffu, v);
    if (lane == 0) sts32(sm + Layout::warp + 8 * (threadIdx.x >> 5), v);
    __syncthreads();
    if (threadIdx.x < 32) v = __reduce_max_sync(0xffffffffu, lane < kWarps ? lds32(sm + Layout::warp + 8 * lane) : 0);
    const uint32_t slot = exchange(v);
    v = 0;
    for (int c = 0; c < ctas; ++c) v = max(v, lds32(slot + 8 * c));
    return v;
  }

  template <typename F>
  __device__ __forceinline__ void each(F &&f) const {  // f(logit, index in the slice), four a load
    const int n4 = (n + 3) / 4;  // logits behind n are -inf: no candidates
    for (int i = threadIdx.x; i < n4; i += kThreads) {
      const uint4 v = lds128(sm + Layout::logits + 16 * i);
      f(__uint_as_float(v.x), 4 * i), f(__uint_as_float(v.y), 4 * i + 1);
      f(__uint_as_float(v.z), 4 * i + 2), f(__uint_as_float(v.w), 4 * i + 3);
    }
  }

  // Brings the tokens of the row whose logits lie in [lo, hi] and that `take`
  // accepts onto the first CTA's list; returns their number.  More than kList
  // are only counted.  Each CTA lists its own, then moves them behind those of
  // the CTAs before it.  Ends with a cluster barrier.
  template <typename F>
  __device__ unsigned collect(float lo, float hi, F &&take) {
    const uint32_t listed = sm + Layout::listed, list = sm + Layout::list;
    if (threadIdx.x == 0) sts32(listed, 0);
    __syncthreads();
    each([&](float x, int i) {
      if (x >= lo && x <= hi && take(x)) {
        const unsigned group = __activemask(), lane = threadIdx.x & 31;  // one addition for the lanes that are here
        uint32_t at = 0;
        if (lane == __ffs(group) - 1) at = add32(listed, __popc(group));
        at = __shfl_sync(group, at, __ffs(group) - 1) + __popc(group & ((1u << lane) - 1));
        if (at < kList) sts64(list + 8 * at, (u64)~key_of(x) << 32 | (unsigned)(base + i));
      }
    });
    __syncthreads();
    const unsigned own = lds32(listed);
    const uint32_t slot = exchange(own);
    unsigned all = 0, before = 0;
    for (int c = 0; c < ctas; ++c) {
      const unsigned have = (unsigned)lds64(slot + 8 * c);
      all += have;
      before += c < rank ? have : 0;
    }
    if (rank && all <= kList) {
      const uint32_t to = in_cta(list, 0) + 8 * before;
      for (unsigned i = threadIdx.x; i < own; i += kThreads) sts64(to + 8 * i, lds64(list + 8 * i));
    }
    cluster_barrier();
    return all;
  }

  __device__ __forceinline__ u64 listed_at(int i) const { return lds64(sm + Layout::list + 8 * i); }
  __device__ __forceinline__ float logit_at(int i) const { return value_of((uint32_t)~(listed_at(i) >> 32)); }
  __device__ __forceinline__ u64 run_at(int i) const { return lds64(sm + Layout::run + 8 * i); }
  // Bitonic sort of the list, E neighbours per thread in registers: partners in
  // the same thread or warp trade without shared memory.
  template <int E>
  __device__ void sort_list(int m, int size) {
    const uint32_t list = sm + Layout::list + 8 * E * threadIdx.x;
    const int first = E * threadIdx.x;
    u64 v[E];
#pragma unroll
    for (int r = 0; r < E; ++r) v[r] = first + r < m ? lds64(list + 8 * r) : ~0ull;
    for (int k = 2; k <= size; k <<= 1) {
      int j = k >> 1;
      for (; j >= 32 * E; j >>= 1) {  // partners in other warps
        __syncthreads();
#pragma unroll
        for (int r = 0; r < E; ++r) sts64(list + 8 * r, v[r]);
        __syncthreads();
        const bool small = ((first & j) == 0) == ((first & k) == 0);
        const uint32_t other = sm + Layout::list + 8 * (first ^ j);
#pragma unroll
        for (int r = 0; r < E; ++r) {
          const u64 o = lds64(other + 8 * r);
          v[r] = (o < v[r]) == small ? o : v[r];
        }
      }
      for (; j >= E; j >>= 1) {
        const bool small = ((first & j) == 0) == ((first & k) == 0);
#pragma unroll
        for (int r = 0; r < E; ++r) {
          const u64 o = __shfl_xor_sync(0xffffffffu, v[r], j / E);
          v[r] = (o < v[r]) == small ? o : v[r];
        }
      }
#pragma unroll
      for (int jj = E / 2; jj; jj >>= 1)
        if (jj <= j) {
#pragma unroll
          for (int r = 0; r < E; ++r)
            if (!(r & jj)) {
              const bool up = ((first + r) & k) == 0;
              const u64 x = v[r], y = v[r | jj];
              v[r] = (x < y) == up ? x : y;
              v[r | jj] = (x < y) == up ? y : x;
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < E; ++r) sts64(list + 8 * r, v[r]);
    __syncthreads();
  }
  // Sorts the list's m tokens and sums their masses along it (one CTA).
  template <typename W>
  __device__ void order_list(int m, const W &weigh) {
    int size = 2;
    while (size < m) size <<= 1;
    if (size <= kThreads)
      sort_list<1>(m, size);
    else
      sort_list<kList / kThreads>(m, size);
    u64 before = 0;
    for (int i = 0; i < m; i += kThreads) {
      const int at = i + (int)threadIdx.x;
      before = scan(at < m ? weigh(logit_at(at)) : 0, before, sm + Layout::run + 8 * at);
    }
    __syncthreads();
  }

  // Running sum over the CTA's threads behind `before`, into `to`; returns the total.
  __device__ u64 scan(u64 v, u64 before, uint32_t to) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 u = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += u;
    }
    __syncthreads();  // the last call's sums have been read
    if (lane == 31) sts64(sm + Layout::warp + 8 * (threadIdx.x >> 5), v);
    __syncthreads();
    u64 w = lane < kWarps ? lds64(sm + Layout::warp + 8 * lane) : 0;
#pragma unroll
    for (int o = 1; o < kWarps; o <<= 1) {
      const u64 u = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += u;
    }
    const int mine = threadIdx.x >> 5;
    const u64 prior = __shfl_sync(0xffffffffu, w, mine ? mine - 1 : 0);
    sts64(to, before + (mine ? prior : 0) + v);
    return before + __shfl_sync(0xffffffffu, w, kWarps - 1);
  }

  // How many of the first m places satisfy `is` (one CTA; every thread gets it).
  template <typename F>
  __device__ int count_places(int m, F &&is) {
    int c = 0;
    for (int i = 0; i < m; i += kThreads) c += __syncthreads_count(i + (int)threadIdx.x < m && is(i + threadIdx.x));
    return c;
  }

  __device__ void clear_bins() {
    for (int b = threadIdx.x; b < 2 * kBinRoom; b += kThreads) sts32(sm + Layout::lo + 4 * b, 0);  // lo and hi
    __syncthreads();
  }
  // Sums the bins of all CTAs into running masses (counts) over the bins: every CTA
  // does it for itself.  Call between two cluster barriers.
  __device__ void run_bins(bool counts) {
    u64 before = 0;
    for (int i = 0; i <= kBins; i += kThreads) {
      const int b = i + (int)threadIdx.x;
      u64 lo = 0, hi = 0;
      if (b <= kBins)
        for (int c = 0; c < ctas; ++c) {
          lo += lds32(in_cta(sm + Layout::lo + 4 * b, c));
          if (!counts) hi += lds32(in_cta(sm + Layout::hi + 4 * b, c));
        }
      before = scan(counts ? lo : ((hi << 16) + lo) << max(13 - (b >> 4), 0), before, sm + Layout::bins + 8 * b);
    }
    __syncthreads();
  }
  __device__ __forceinline__ u64 through_bin(int b) const { return lds64(sm + Layout::bins + 8 * b); }
  // The first bin whose running sum reaches target (<= the last one).
  __device__ int bin_of(u64 target) {
    int c = 0;
    for (int b = 0; b <= kBins; b += kThreads)
      c += __syncthreads_count(b + (int)threadIdx.x <= kBins && through_bin(b + (int)threadIdx.x) < target);
    return min(c, kBins);
  }

  // Step 5: the first place where the running count (or mass) reaches `target`,
  // by digits of the key.  All CTAs take part and know the answer.
  template <typename W>
  __device__ Place descend(bool by_mass, u64 target, const W &weigh) {
    const uint32_t mass = sm + Layout::run, count = mass + 8 * 256, sum_m = count + 8 * 256, sum_n = sum_m + 8 * 256;
    Place at{0u, 1u, 0};
    u64 before_n = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
      cluster_barrier();
      for (int i = threadIdx.x; i < 512; i += kThreads) sts64(mass + 8 * i, 0);
      __syncthreads();
      each([&](float x, int) {
        const uint32_t k = key_of(x);
        if (x > -INFINITY && (shift == 24 || (k >> (shift + 8)) == (at.key >> (shift + 8)))) {
          red64(count + 8 * (k >> shift & 255), 1ull);
          red64(mass + 8 * (k >> shift & 255), weigh(x));
        }
      });
      cluster_barrier();
      for (int i = threadIdx.x; i < 256; i += kThreads) {
        u64 m = 0, c = 0;
        for (int r = 0; r < ctas; ++r) m += lds64(in_cta(mass + 8 * i, r)), c += lds64(in_cta(count + 8 * i, r));
        sts64(sum_m + 8 * i, m);
        sts64(sum_n + 8 * i, c);
      }
      __syncthreads();
      if (threadIdx.x == 0) {
        u64 m = at.above, c = before_n;
        int d = 255;  // the target is at most what the histogram holds
        for (; d > 0; --d) {
          const u64 dm = m + lds64(sum_m + 8 * d), dc = c + lds64(sum_n + 8 * d);
          if ((by_mass ? dm : dc) >= target) break;
          m = dm, c = dc;
        }
        sts32(sm + Layout::found, d);
        sts64(sm + Layout::before, m);
        sts64(sm + Layout::before + 8, c);
      }
      __syncthreads();
      at.key |= lds32(sm + Layout::found) << shift;
      at.above = lds64(sm + Layout::before), before_n = lds64(sm + Layout::before + 8);
    }
    cluster_barrier();
    if (by_mass) {
      const u64 w = weigh(value_of(at.key)), need = target - at.above;
      at.rank = w ? (unsigned)((need + w - 1) / w) : 1u;
    } else {
      at.rank = (unsigned)(target - before_n);
    }
    return at;
  }

  // The index of a place's token, on every thread of the CTA that holds it; -1 elsewhere.
  __device__ int token_at(float logit, unsigned place) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int per = (n + kWarps * 32 - 1) / (kWarps * 32) * 32, i0 = min(warp * per, n), i1 = min(i0 + per, n);
    const uint32_t logits = sm + Layout::logits, found = sm + Layout::found;
    auto is = [&](int i) { return i < i1 && __uint_as_float(lds32(logits + 4 * i)) == logit; };
    unsigned have = 0;  // in this warp's stretch of the slice
    for (int i = i0; i < i1; i += 32)
      have += __popc(__ballot_sync(0xffffffffu, is(i + lane)));
    if (threadIdx.x == 0) sts32(found, ~0u);
    const u64 own = scan(lane ? 0 : have, 0, sm + Layout::run + 8 * threadIdx.x);  // of this CTA
    __syncthreads();
    const uint32_t slot = exchange(own);
    u64 before = run_at(32 * warp) - have;
    for (int c = 0; c < rank; ++c) before += lds64(slot + 8 * c);
    if (before < place && place <= before + have)
      for (int i = i0; i < i1; i += 32) {
        const bool hit = is(i + lane);
        const unsigned hits = __ballot_sync(0xffffffffu, hit);
        if (hit && before + __popc(hits & ((2u << lane) - 1)) == place) sts32(found, base + i + lane);
        before += __popc(hits);
      }
    __syncthreads();
    return (int)lds32(found);
  }
};

__global__ void __launch_bounds__(kThreads) sample_tokens_kernel(SampleParams p) {
  extern __shared__ __align__(16) unsigned char smem[];
  const uint32_t sm = sm100::smem_u32(smem), logits = sm + Layout::logits;
  const uint32_t seen = logits + 4 * p.slice;  // a bit for each token of the context in this slice
  const int tid = threadIdx.x, ctas = (int)cluster_ctas(), rank = (int)cluster_ctarank();
  const int r = blockIdx.x / ctas;
  const int base = rank * p.slice, n = max(0, min(p.slice, p.V - base));
  Row row{sm, n, base, ctas, rank};

  const float temp = p.temperature ? p.temperature[r] : p.temperature_all;
  const float top_p = p.top_p ? p.top_p[r] : p.top_p_all;
  const float min_p = p.min_p ? p.min_p[r] : p.min_p_all;
  const float pen = p.penalty ? p.penalty[r] : p.penalty_all;
  const int top_k = p.top_k ? p.top_k[r] : p.top_k_all;
  const float u = fminf(fmaxf(p.uniforms[r], 0.0f), 0.99999994f);

  // the slice
  const bool penalise = p.ctx_len > 0 && pen != 1.0f;
  if (penalise) {
    for (int i = tid; i < (n + 31) / 32; i += kThreads) sts32(seen + 4 * i, 0);
    __syncthreads();
    for (int i = tid; i < p.ctx_len; i += kThreads) {
      const int t = p.ctx[(int64_t)r * p.ctx_stride + i] - base;
      if (t >= 0 && t < n)
        asm volatile("red.shared.or.b32 [%0], %1;" ::"r"(seen + 4 * (t >> 5)), "r"(1u << (t & 31)) : "memory");
    }
    __syncthreads();
  }
  float top = -INFINITY;
  auto keep = [&](float x, int i) {
    if (penalise && (lds32(seen + 4 * (i >> 5)) >> (i & 31) & 1)) x = x > 0.f ? x / pen : x * pen;
    x = kept(x);
    top = fmaxf(top, x);
    return __float_as_uint(x);
  };
  const int64_t at0 = (int64_t)r * p.ld + base;
  constexpr int kBatch = 8;  // loads a thread has in flight
  auto scalar = [&](int from, auto &&load) {
    for (int i0 = from + tid; i0 < n; i0 += kBatch * kThreads) {
      float v[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        if (i0 + j * kThreads < n) v[j] = load(i0 + j * kThreads);
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        if (i0 + j * kThreads < n) sts32(logits + 4 * (i0 + j * kThreads), keep(v[j], i0 + j * kThreads));
    }
  };
  if (p.b16) {
    const __nv_bfloat16 *l = static_cast<const __nv_bfloat16 *>(p.logits) + at0;
    const int nv = p.vec ? n / 8 : 0;
    for (int i0 = tid; i0 < nv; i0 += kBatch * kThreads) {
      uint4 v[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        if (i0 + j * kThreads < nv) v[j] = __ldcs(reinterpret_cast<const uint4 *>(l) + i0 + j * kThreads);
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const int i = i0 + j * kThreads;
        if (i < nv) {
          const uint32_t w[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
          uint32_t k[8];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            k[2 * c] = keep(__uint_as_float(w[c] << 16), 8 * i + 2 * c);
            k[2 * c + 1] = keep(__uint_as_float(w[c] & 0xffff0000u), 8 * i + 2 * c + 1);
          }
          sts128(logits + 32 * i, k[0], k[1], k[2], k[3]);
          sts128(logits + 32 * i + 16, k[4], k[5], k[6], k[7]);
        }
      }
    }
    scalar(8 * nv, [&](int i) { return __bfloat162float(l[i]); });
  } else {
    const float *l = static_cast<const float *>(p.logits) + at0;
    const int nv = p.vec ? n / 4 : 0;
    for (int i0 = tid; i0 < nv; i0 += kBatch * kThreads) {
      float4 v[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        if (i0 + j * kThreads < nv) v[j] = __ldcs(reinterpret_cast<const float4 *>(l) + i0 + j * kThreads);
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const int i = i0 + j * kThreads;
        if (i < nv) {
          const uint32_t a = keep(v[j].x, 4 * i), b = keep(v[j].y, 4 * i + 1), c = keep(v[j].z, 4 * i + 2),
                         d = keep(v[j].w, 4 * i + 3);
          sts128(logits + 16 * i, a, b, c, d);
        }
      }
    }
    scalar(4 * nv, [&](int i) { return l[i]; });
  }
  for (int i = n + tid; i < min(p.slice, (n + 3) & ~3); i += kThreads) sts32(logits + 4 * i, 0xff800000u);  // -inf
  if (tid < 16) sts64(sm + Layout::power + 8 * tid, (u64)__double_as_longlong(exp2(44.0 - tid / 16.0)));
  __syncthreads();

  // 1. the maximum
  top = value_of(row.largest(key_of(top)));
  auto write = [&](int token, float logp) {
    p.token[r] = token;
    if (p.logprob) p.logprob[r] = logp;
  };
  if (!(top > -INFINITY)) {
    if (rank == 0 && tid == 0) write(-1, -INFINITY);
    return;
  }
  if (!(temp > 1e-4f)) {
    const int t = row.token_at(top, 1);
    if (t >= 0 && tid == 0) write(t, 0.f);
    return;
  }
  const double c = 1.4426950408889634 / (double)fminf(temp, 1e36f);  // octaves of w per unit of a logit
  const Weigher weigh{top, (float)c, (double)top, c, sm + Layout::power};

  const bool cut_p = !(top_p >= 1.0f), cut_k = top_k > 0 && top_k < p.V, cut_m = min_p > 0.0f;
  const double share = cut_p ? (top_p > 0.f ? (double)top_p : 0.0) : 1.0;
  const u64 floor_m = cut_m ? (u64)ceil(fmin((double)min_p, 1.0) * (double)kOne) : 1;
  u64 z = 0;
  if (top < INFINITY) {
    int end = 0, m = 0;
    if (cut_k) {
      // 2. counts: the tokens through the bin that holds the k-th
      row.clear_bins();
      row.each([&](float x, int) {
        if (x > -INFINITY) red32(sm + Layout::lo + 4 * weigh.bin(x), 1u);
      });
      cluster_barrier();
      row.run_bins(true);
      const int last = row.bin_of((u64)top_k);
      m = (int)min(row.through_bin(last), (u64)(kList + 1));
      if (m <= kList) {
        m = (int)row.collect(last < kBins ? weigh.logit_below((last + 1) / 16.0) : -3.4028235e38f, INFINITY,
                             [&](float x) { return weigh.bin(x) <= last; });
        if (rank) return;
        row.order_list(m, weigh);
        end = min(top_k, m);
        z = row.run_at(end - 1);
      }
    } else {
      // 2. the sum of all masses, then the tokens that can still matter
      u64 least = floor_m;
      if (cut_p || !cut_m) {
        row.each([&](float x, int) { z += weigh(x); });
        z = row.total(z);
        const double behind = (cut_p ? 1.0 - share : 1.0 - (double)u) * (double)z / (double)p.V;
        const u64 t = behind > 2.0 ? (u64)behind - 1 : 1;
        least = t > least ? t : least;
      }
      const float lowest = weigh.logit_below(44.0 - log2((double)least));
      m = (int)row.collect(lowest, INFINITY, [&](float x) { return weigh(x) >= least; });
      if (m <= kList) {
        if (rank) return;
        row.order_list(m, weigh);
        end = m;
        if (!cut_p && cut_m) z = row.run_at(m - 1);
      } else {
        // 4. masses by bins; the crossing of top_p and the draw each in one bin
        row.clear_bins();
        row.each([&](float x, int) {
          if (x >= lowest && weigh.some(weigh.lead(x))) {
            int k, shift;
            const uint32_t q = weigh.bits(x, k, shift);
            if (((u64)q << shift) >= least) {
              red32(sm + Layout::lo + 4 * k, q & 0xffffu);
              red32(sm + Layout::hi + 4 * k, q >> 16);
            }
          }
        });
        cluster_barrier();
        row.run_bins(false);
        const u64 held = row.through_bin(kBins);
        u64 mass = cut_m ? held : z;  // of the kept tokens, unless top_p crosses before
        const u64 over = (u64)floor(share * (double)z) + 1;
        bool fits = true;
        for (int pass = cut_p && over <= held ? 0 : 1; pass < 2 && fits; ++pass) {
          u64 target = over;
          if (pass) {
            target = (u64)ceil((double)u * (double)mass);
            target = target < 1 ? 1 : (target > mass ? mass : target);
            target = target > held ? held : target;
          }
          const int b = row.bin_of(target);
          const u64 before = b ? row.through_bin(b - 1) : 0;
          const unsigned in_bin =
              row.collect(weigh.logit_below((b + 0.5) / 16.0), weigh.logit_above((b - 0.5) / 16.0), [&](float x) {
                int k = -1, shift;
                const uint32_t q = weigh.some(weigh.lead(x)) ? weigh.bits(x, k, shift) : 0;
                return k == b && ((u64)q << shift) >= least;
              });
          fits = in_bin <= kList;
          if (fits && rank == 0) {
            row.order_list((int)in_bin, weigh);
            const int i = min(row.count_places((int)in_bin, [&](int j) { return before + row.run_at(j) < target; }),
                              (int)in_bin - 1);
            if (tid == 0) {
              sts64(sm + Layout::before, before + row.run_at(i));
              if (pass) write((int)(uint32_t)row.listed_at(i), weigh.log_share(row.logit_at(i), mass));
            }
          }
          if (fits && pass) return;
          cluster_barrier();
          if (fits) mass = lds64(in_cta(sm + Layout::before, 0));
        }
      }
    }
    if (end) {
      // 3. every place along the sorted list
      if (cut_p) {
        const u64 over = (u64)floor(share * (double)z) + 1;
        end = min(end, 1 + row.count_places(end, [&](int i) { return row.run_at(i) < over; }));
      }
      if (cut_m)
        end = min(end, max(1, row.count_places(end, [&](int i) {
                return weigh(row.logit_at(i)) >= floor_m;
              })));
      // without a cut the list is the head of a longer row: the whole row's mass counts
      const u64 mass = cut_k || cut_p || cut_m ? row.run_at(end - 1) : z;
      u64 target = (u64)ceil((double)u * (double)mass);
      target = target < 1 ? 1 : target;
      const int i = min(row.count_places(end, [&](int j) { return row.run_at(j) < target; }), end - 1);
      if (tid == 0) write((int)(uint32_t)row.listed_at(i), weigh.log_share(row.logit_at(i), mass));
      return;
    }
  }

  // 5. places by digits of the key
  const bool inf = top == INFINITY;  // only its equals have mass
  auto mass_of = [&](float x) { return inf ? (x == top ? kOne : 0ull) : weigh(x); };
  z = 0;
  u64 live = 0;
  row.each([&](float x, int) { z += mass_of(x), live += x > -INFINITY; });
  z = row.total(z);
  live = row.total(live);
  Place stop{0u, 1u, z};
  auto through = [&](const Place &a) { return a.key ? a.above + (u64)a.rank * mass_of(value_of(a.key)) : a.above; };
  if (cut_k && (u64)top_k < live) {
    stop = row.descend(false, (u64)top_k, mass_of);
    z = through(stop);
  }
  if (cut_p) {
    const u64 over = (u64)floor(share * (double)z) + 1;
    if (over <= z) stop = shorter(row.descend(true, over, mass_of), stop);
  }
  if (cut_m) {
    u64 kept_m = 0;
    row.each([&](float x, int) {
      const u64 w = mass_of(x);
      kept_m += w >= floor_m ? w : 0;
    });
    stop = shorter(row.descend(true, row.total(kept_m), mass_of), stop);
  }
  const u64 mass = through(stop);
  u64 target = (u64)ceil((double)u * (double)mass);
  target = target < 1 ? 1 : (target > mass ? mass : target);
  const Place at = shorter(row.descend(true, target, mass_of), stop);
  const int t = row.token_at(value_of(at.key), at.rank);
  if (t >= 0 && tid == 0) write(t, inf ? -logf((float)(mass >> 44)) : weigh.log_share(value_of(at.key), mass));
}

}  // namespace

extern "C" int af_sample_tokens(af_ctx *ctx, const void *logits, int logits_bf16, int64_t row_stride, int rows,
                                int vocab, const int32_t *context_tokens, int64_t context_stride, int context_len,
                                const float *temperature, float temperature_all, const int32_t *top_k, int top_k_all,
                                const float *top_p, float top_p_all, const float *min_p, float min_p_all,
                                const float *penalty, float penalty_all, const float *uniforms, int32_t *token,
                                float *logprob, af_stream_t stream) {
  const char *fn = "af_sample_tokens";
  af::DeviceScope scope;
  AF_ENTER(ctx, fn);
  AF_REQUIRE(rows >= 0 && vocab > 0, "af_sample_tokens", "bad sizes");
  AF_REQUIRE(rows <= (1 << 24), "af_sample_tokens", "%d rows: at most 2^24 are supported", rows);
  AF_REQUIRE(vocab <= AF_SAMPLE_TOKENS_MAX_VOCAB, "af_sample_tokens", "vocab %d exceeds the maximum %d", vocab,
             AF_SAMPLE_TOKENS_MAX_VOCAB);
  AF_REQUIRE(context_len >= 0 && (context_len == 0 || context_tokens), "af_sample_tokens", "bad context");
  AF_REQUIRE(penalty || penalty_all > 0.f, "af_sample_tokens", "the repetition penalty must be positive");
  if (rows == 0) return AF_OK;
  AF_REQUIRE(logits && uniforms && token, "af_sample_tokens", "null argument");
  // CTAs per row: slices of at most 16384 tokens (two CTAs share an SM), more
  // of them while the rows do not fill the SMs and a slice keeps 2048 tokens.
  int ctas = 1;
  while (ctas < kMaxCtas && (vocab > 16384 * ctas || (rows * ctas <= ctx->num_sms && vocab >= 4096 * ctas))) ctas *= 2;
  const int slice = ((vocab + ctas - 1) / ctas + 7) & ~7;
  const int per16 = logits_bf16 ? 8 : 4;
  const int vec = af::aligned16(logits) && (rows == 1 || row_stride % per16 == 0);
  SampleParams p{logits, logits_bf16 != 0, row_stride, vocab, slice, vec, context_tokens, context_stride, context_len,
                 temperature, top_p, min_p, penalty, top_k, temperature_all, top_p_all, min_p_all, penalty_all,
                 top_k_all, uniforms, token, logprob};
  auto bytes = [](int s) { return (size_t)Layout::logits + (size_t)s * 4 + (size_t)((s + 31) / 32) * 4; };
  static std::atomic<unsigned long long> attr_devices{0};
  if (int rc = af::smem_attr(ctx, reinterpret_cast<const void *>(sample_tokens_kernel),
                             bytes((AF_SAMPLE_TOKENS_MAX_VOCAB / kMaxCtas + 7) & ~7), attr_devices, fn))
    return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)rows * ctas);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = bytes(slice);
  cfg.stream = af::stream_of(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  AF_CUDA(cudaLaunchKernelEx(&cfg, sample_tokens_kernel, p), fn);
  return af::launched(ctx, fn);
}
