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
// Bound: a long row by instructions (about 30 per token for the mass, from
// 256 tabulated powers and a cubic; two histogram additions where step 4
// runs), a short one by the chain of cluster barriers.
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
constexpr float kSteps = 256.0f;         // table steps per octave
constexpr u64 kOne = 1ull << 44;         // the mass of the largest logit
constexpr uint32_t kNothing = 0x007fffffu;  // key of -inf: keys above it are candidates

// Logit to key: larger key, larger logit; -0 and +0 are one key.  NaN counts
// as -inf: it is never drawn.
__device__ __forceinline__ uint32_t key_of(float x) {
  x = x == x ? x + 0.0f : -INFINITY;
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

// Shared memory of a CTA, byte offsets: this, the keys, then the bits of the
// context's tokens.  It is addressed by 32-bit shared addresses throughout, the
// same for this CTA's memory and (after mapa) another's.
struct Layout {
  static constexpr uint32_t list = 0;                      // u64 [kList]: (~key, index), ascending is the order
  static constexpr uint32_t run = list + 8 * kList;        // u64 [kList]: running mass along the list; step 5's sums
  static constexpr uint32_t bins = run + 8 * kList;        // u64 [kBinRoom]: running masses (counts) of the row's bins
  static constexpr uint32_t lo = bins + 8 * kBinRoom;      // u32 [kBinRoom], hi alike: this CTA's bins
  static constexpr uint32_t hi = lo + 4 * kBinRoom;
  static constexpr uint32_t power = hi + 4 * kBinRoom;     // u32 pairs [256]: 2^(31 - j / 256) rounded, and as fp32
  static constexpr uint32_t slot = power + 8 * 256;        // u64 [2][2][kMaxCtas]
  static constexpr uint32_t warp = slot + 8 * 4 * kMaxCtas;  // u64 [2][kWarps]
  static constexpr uint32_t before = warp + 8 * 2 * kWarps;  // u64 [2]
  static constexpr uint32_t listed = before + 16;            // u32, then found
  static constexpr uint32_t found = listed + 4;
  static constexpr uint32_t keys = found + 12;  // u32 [slice]
};
static_assert(Layout::keys % 16 == 0, "keys are read sixteen bytes at a time");

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

// The mass of a token: w = 2^(-t / 256), t = (max - l) 256 log2(e) / T formed
// in two fp32 parts; w = 2^(-i / 256) 2^(-f / 256), i = rint(t), the first
// factor from the table, the second 1 + (g + g^2/2 + g^3/6) with |g| < 0.00136.
struct Weigher {
  float top, ch, cl;
  uint32_t power;  // Layout::power's address
  // The place of t's whole steps, or -1 where w < 2^-46.
  __device__ __forceinline__ int step(float x, float &f) const {
    const float d = top - x, bb = d - top, e = (top - (d - bb)) - (x + bb);  // d + e = top - x
    const float t = __fmul_rn(d, ch);
    if (!(t < 46.0f * kSteps)) return -1;
    const float tl = fmaf(d, ch, -t) + fmaf(e, ch, d * cl);
    const float r = __fadd_rn(t, 12582912.0f);  // 1.5 * 2^23: rounds to a whole number
    f = (t - (r - 12582912.0f)) + tl;
    return __float_as_int(r) - 0x4b400000;
  }
  // 31 bits of w and their shift: the mass is q << shift.
  __device__ __forceinline__ uint32_t bits(int i, float f, int &shift) const {
    const uint32_t at = power + 8 * (i & 255);
    const float g = f * -0.0027076061740622863f;  // ln 2 / 256
    const float ex = fmaf(g * g, fmaf(g, 0.16666667f, 0.5f), g);
    const uint32_t q = lds32(at) + (uint32_t)(__float_as_int(fmaf(__uint_as_float(lds32(at + 4)), ex, 12582912.0f)) - 0x4b400000);
    const int o = i >> 8;
    shift = max(13 - o, 0);
    return o > 13 ? q >> min(o - 13, 31) : q;
  }
  __device__ __forceinline__ u64 operator()(uint32_t key) const {
    float f;
    const int i = step(value_of(key), f);
    if (i < 0) return 0;
    int sh;
    const uint32_t q = bits(i, f, sh);
    return (u64)q << sh;
  }
  // The bin by the leading part of t alone: never smaller for a smaller logit.
  __device__ __forceinline__ int bin(uint32_t key) const {
    const float t = __fmul_rn(top - value_of(key), ch);
    return t < 46.0f * kSteps ? (__float_as_int(__fadd_rn(t, 12582912.0f)) - 0x4b400000) >> 4 : kBins;
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

  // Totals of a and b over the row (max: the larger a).  One cluster barrier;
  // the slots alternate, so the next exchange cannot overtake a reader.
  __device__ void totals(u64 &a, u64 &b, bool max_a = false) {
    const int lane = threadIdx.x & 31;
    auto reduce = [&](int width) {
      for (int o = width / 2; o; o >>= 1) {
        const u64 v = __shfl_xor_sync(0xffffffffu, a, o);
        a = max_a ? (v > a ? v : a) : a + v;
        b += __shfl_xor_sync(0xffffffffu, b, o);
      }
    };
    reduce(32);
    const uint32_t warp = sm + Layout::warp, slot = sm + Layout::slot + 16 * kMaxCtas * flip;
    if (lane == 0) {
      sts64(warp + 8 * (threadIdx.x >> 5), a);
      sts64(warp + 8 * (kWarps + (threadIdx.x >> 5)), b);
    }
    __syncthreads();
    if (threadIdx.x < 32) {
      a = b = 0;
      if (lane < kWarps) a = lds64(warp + 8 * lane), b = lds64(warp + 8 * (kWarps + lane));
      reduce(32);
      if (lane < ctas) {
        sts64(in_cta(slot + 8 * rank, lane), a);
        sts64(in_cta(slot + 8 * (kMaxCtas + rank), lane), b);
      }
    }
    cluster_barrier();
    a = b = 0;
    if (lane < ctas) a = lds64(slot + 8 * lane), b = lds64(slot + 8 * (kMaxCtas + lane));
    reduce(32);
    flip ^= 1;
  }

  template <typename F>
  __device__ __forceinline__ void each(F &&f) const {  // f(key, index in the slice), four keys a load
    const int n4 = (n + 3) / 4;  // keys behind n are 0: no candidates
    for (int i = threadIdx.x; i < n4; i += kThreads) {
      const uint4 k = lds128(sm + Layout::keys + 16 * i);
      f(k.x, 4 * i), f(k.y, 4 * i + 1), f(k.z, 4 * i + 2), f(k.w, 4 * i + 3);
    }
  }

  // Puts the tokens that `take` accepts on the first CTA's list (those that do
  // not fit are only counted).
  template <typename F>
  __device__ void gather(F &&take) {
    const uint32_t listed = in_cta(sm + Layout::listed, 0), list = in_cta(sm + Layout::list, 0);
    each([&](uint32_t k, int i) {
      if (k > kNothing && take(k)) {
        const uint32_t at = add32(listed, 1u);
        if (at < kList) sts64(list + 8 * at, (u64)~k << 32 | (unsigned)(base + i));
      }
    });
  }

  // Sorts the list's m tokens and sums their masses along it (one CTA).
  __device__ __forceinline__ u64 listed_at(int i) const { return lds64(sm + Layout::list + 8 * i); }
  __device__ __forceinline__ uint32_t key_at(int i) const { return (uint32_t)~(listed_at(i) >> 32); }
  __device__ __forceinline__ u64 run_at(int i) const { return lds64(sm + Layout::run + 8 * i); }
  template <typename W>
  __device__ void order_list(int m, const W &weigh) {
    const uint32_t list = sm + Layout::list;
    int size = 2;
    while (size < m) size <<= 1;
    for (int i = m + (int)threadIdx.x; i < size; i += kThreads) sts64(list + 8 * i, ~0ull);
    for (int k = 2; k <= size; k <<= 1)
      for (int j = k >> 1; j; j >>= 1) {
        __syncthreads();
        for (int i = threadIdx.x; i < size / 2; i += kThreads) {
          const int a = ((i & ~(j - 1)) << 1) | (i & (j - 1)), b = a | j;
          const u64 x = lds64(list + 8 * a), y = lds64(list + 8 * b);
          if ((x > y) == ((a & k) == 0)) {
            sts64(list + 8 * a, y);
            sts64(list + 8 * b, x);
          }
        }
      }
    __syncthreads();
    u64 before = 0;
    for (int i = 0; i < m; i += kThreads) {
      const int at = i + (int)threadIdx.x;
      before = scan(at < m ? weigh(key_at(at)) : 0, before, sm + Layout::run + 8 * at);
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
      each([&](uint32_t k, int) {
        if (k > kNothing && (shift == 24 || (k >> (shift + 8)) == (at.key >> (shift + 8)))) {
          red64(count + 8 * (k >> shift & 255), 1ull);
          red64(mass + 8 * (k >> shift & 255), weigh(k));
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
      const u64 w = weigh(at.key), need = target - at.above;
      at.rank = w ? (unsigned)((need + w - 1) / w) : 1u;
    } else {
      at.rank = (unsigned)(target - before_n);
    }
    return at;
  }

  // The index of a place's token, on every thread of the CTA that holds it; -1 elsewhere.
  __device__ int token_at(uint32_t key, unsigned place) {
    const int per = (n + kThreads - 1) / kThreads, i0 = min((int)threadIdx.x * per, n), i1 = min(i0 + per, n);
    const uint32_t keys = sm + Layout::keys, found = sm + Layout::found;
    unsigned have = 0;
    for (int i = i0; i < i1; ++i) have += lds32(keys + 4 * i) == key;
    if (threadIdx.x == 0) sts32(found, ~0u);
    const u64 through = scan(have, 0, sm + Layout::run + 8 * threadIdx.x);  // of this CTA
    const uint32_t slot = sm + Layout::slot + 16 * kMaxCtas * flip;
    u64 mine = threadIdx.x ? 0 : through, none = 0;
    __syncthreads();
    totals(mine, none);
    u64 before = run_at(threadIdx.x) - have;
    for (int c = 0; c < rank; ++c) before += lds64(slot + 8 * c);
    if (before < place && place <= before + have)
      for (int i = i0; i < i1; ++i)
        if (lds32(keys + 4 * i) == key && ++before == place) sts32(found, base + i);
    __syncthreads();
    return (int)lds32(found);
  }
};

__device__ __forceinline__ float log_share(u64 w, u64 mass) { return (float)(log((double)w) - log((double)mass)); }

__global__ void __launch_bounds__(kThreads) sample_tokens_kernel(SampleParams p) {
  extern __shared__ __align__(16) unsigned char smem[];
  const uint32_t sm = sm100::smem_u32(smem), keys = sm + Layout::keys;
  const uint32_t seen = keys + 4 * p.slice;  // a bit for each token of the context in this slice
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

  // the slice as keys
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
  uint32_t kmax = 0;
  auto keep = [&](float x, int i) {
    if (penalise && (lds32(seen + 4 * (i >> 5)) >> (i & 31) & 1)) x = x > 0.f ? x / pen : x * pen;
    const uint32_t k = key_of(x);
    kmax = max(kmax, k);
    return k;
  };
  const int64_t at0 = (int64_t)r * p.ld + base;
  if (p.b16) {
    const __nv_bfloat16 *l = static_cast<const __nv_bfloat16 *>(p.logits) + at0;
    const int nv = p.vec ? n / 8 : 0;
    for (int i = tid; i < nv; i += kThreads) {
      const uint4 v = __ldcs(reinterpret_cast<const uint4 *>(l) + i);
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
      uint32_t k[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        k[2 * j] = keep(__uint_as_float(w[j] << 16), 8 * i + 2 * j);
        k[2 * j + 1] = keep(__uint_as_float(w[j] & 0xffff0000u), 8 * i + 2 * j + 1);
      }
      sts128(keys + 32 * i, k[0], k[1], k[2], k[3]);
      sts128(keys + 32 * i + 16, k[4], k[5], k[6], k[7]);
    }
    for (int i = 8 * nv + tid; i < n; i += kThreads) sts32(keys + 4 * i, keep(__bfloat162float(l[i]), i));
  } else {
    const float *l = static_cast<const float *>(p.logits) + at0;
    const int nv = p.vec ? n / 4 : 0;
    for (int i = tid; i < nv; i += kThreads) {
      const float4 v = __ldcs(reinterpret_cast<const float4 *>(l) + i);
      const uint32_t a = keep(v.x, 4 * i), b = keep(v.y, 4 * i + 1), c = keep(v.z, 4 * i + 2), d = keep(v.w, 4 * i + 3);
      sts128(keys + 16 * i, a, b, c, d);
    }
    for (int i = 4 * nv + tid; i < n; i += kThreads) sts32(keys + 4 * i, keep(__ldcs(l + i), i));
  }
  for (int i = n + tid; i < min(p.slice, (n + 3) & ~3); i += kThreads) sts32(keys + 4 * i, 0);  // behind the slice: no candidates
  if (tid < 256) {
    const double v = exp2(31.0 - tid / 256.0);
    sts32(sm + Layout::power + 8 * tid, (uint32_t)__double2ull_rn(v));
    sts32(sm + Layout::power + 8 * tid + 4, __float_as_uint((float)v));
  }
  for (int b = tid; b < 2 * kBinRoom; b += kThreads) sts32(sm + Layout::lo + 4 * b, 0);  // lo and hi
  if (tid == 0) sts32(sm + Layout::listed, 0);
  __syncthreads();

  // 1. the maximum
  u64 best = kmax, live = 0;
  row.totals(best, live, true);
  kmax = (uint32_t)best;
  const float top = value_of(kmax);
  auto write = [&](int token, float logp) {
    p.token[r] = token;
    if (p.logprob) p.logprob[r] = logp;
  };
  if (kmax <= kNothing) {
    if (rank == 0 && tid == 0) write(-1, -INFINITY);
    return;
  }
  if (!(temp > 1e-4f)) {
    const int t = row.token_at(kmax, 1);
    if (t >= 0 && tid == 0) write(t, 0.f);
    return;
  }
  const double c = 256.0 * 1.4426950408889634 / (double)temp;
  Weigher weigh{top, (float)c, (float)(c - (double)(float)c), sm + Layout::power};

  const bool cut_p = !(top_p >= 1.0f), cut_k = top_k > 0 && top_k < p.V, cut_m = min_p > 0.0f;
  const double share = cut_p ? (top_p > 0.f ? (double)top_p : 0.0) : 1.0;
  const u64 floor_m = cut_m ? (u64)ceil(fmin((double)min_p, 1.0) * (double)kOne) : 1;
  u64 z = 0, none = 0;
  if (top < INFINITY) {
    int end = 0, m = 0;
    if (cut_k) {
      // 2. counts: the tokens through the bin that holds the k-th
      row.each([&](uint32_t k, int) {
        if (k > kNothing) red32(sm + Layout::lo + 4 * weigh.bin(k), 1u);
      });
      cluster_barrier();
      row.run_bins(true);
      const int last = row.bin_of((u64)top_k);
      m = (int)min(row.through_bin(last), (u64)(kList + 1));
      if (m <= kList) row.gather([&](uint32_t k) { return weigh.bin(k) <= last; });
      cluster_barrier();
      if (m <= kList) {
        if (rank) return;
        row.order_list(m, weigh);
        end = min(top_k, m);
        z = row.run_at(end - 1);
      }
    } else {
      // 2. the sum of all masses, then the tokens that can still matter
      if (cut_p || !cut_m) {
        row.each([&](uint32_t k, int) { z += weigh(k); });
        row.totals(z, none);
      }
      u64 least = floor_m;
      if (cut_p || !cut_m) {
        const double behind = (cut_p ? 1.0 - share : 1.0 - (double)u) * (double)z / (double)p.V;
        const u64 t = behind > 2.0 ? (u64)behind - 1 : 1;
        least = t > least ? t : least;
      }
      row.gather([&](uint32_t k) { return weigh(k) >= least; });
      cluster_barrier();
      const unsigned left = lds32(in_cta(sm + Layout::listed, 0));
      if (left <= kList) {
        cluster_barrier();
        if (rank) return;
        m = (int)left;
        row.order_list(m, weigh);
        end = m;
        if (!cut_p && cut_m) z = row.run_at(m - 1);
      } else {
        // 4. masses by bins; the crossing of top_p and the draw each in one bin
        row.each([&](uint32_t k, int) {
          float f;
          const int i = weigh.step(value_of(k), f);
          if (i >= 0) {
            int s;
            const uint32_t q = weigh.bits(i, f, s);
            if (((u64)q << s) >= least) {
              red32(sm + Layout::lo + 4 * (i >> 4), q & 0xffffu);
              red32(sm + Layout::hi + 4 * (i >> 4), q >> 16);
            }
          }
        });
        cluster_barrier();
        row.run_bins(false);
        const u64 held = row.through_bin(kBins);
        u64 mass = cut_m ? held : z;  // of the kept tokens, unless top_p crosses before
        const u64 over = (u64)floor(share * (double)z) + 1;
        bool fits = true, done = false;
        for (int pass = cut_p && over <= held ? 0 : 1; pass < 2 && fits; ++pass) {
          u64 target = over;
          if (pass) {
            target = (u64)ceil((double)u * (double)mass);
            target = target < 1 ? 1 : (target > mass ? mass : target);
            target = target > held ? held : target;
          }
          const int b = row.bin_of(target);
          const u64 before = b ? row.through_bin(b - 1) : 0;
          if (rank == 0 && tid == 0) sts32(sm + Layout::listed, 0);
          cluster_barrier();
          row.gather([&](uint32_t k) {
            float f;
            const int i = weigh.step(value_of(k), f);
            return i >= 0 && (i >> 4) == b && weigh(k) >= least;
          });
          cluster_barrier();
          const unsigned in_bin = lds32(in_cta(sm + Layout::listed, 0));
          fits = in_bin <= kList;
          if (fits && rank == 0) {
            row.order_list((int)in_bin, weigh);
            const int i = min(row.count_places((int)in_bin, [&](int j) { return before + row.run_at(j) < target; }),
                              (int)in_bin - 1);
            if (tid == 0) {
              sts64(sm + Layout::before, before + row.run_at(i));
              if (pass) write((int)(uint32_t)row.listed_at(i), log_share(weigh(row.key_at(i)), mass));
            }
          }
          cluster_barrier();
          if (fits && !pass) mass = lds64(in_cta(sm + Layout::before, 0));
          done = fits && pass;
        }
        if (done) {
          cluster_barrier();
          return;
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
                return weigh(row.key_at(i)) >= floor_m;
              })));
      // without a cut the list is the head of a longer row: the whole row's mass counts
      const u64 mass = cut_k || cut_p || cut_m ? row.run_at(end - 1) : z;
      u64 target = (u64)ceil((double)u * (double)mass);
      target = target < 1 ? 1 : target;
      const int i = min(row.count_places(end, [&](int j) { return row.run_at(j) < target; }), end - 1);
      if (tid == 0) write((int)(uint32_t)row.listed_at(i), log_share(weigh(row.key_at(i)), mass));
      return;
    }
  }

  // 5. places by digits of the key
  const bool inf = top == INFINITY;  // only its equals have mass
  auto mass_of = [&](uint32_t k) { return inf ? (k == kmax ? kOne : 0ull) : weigh(k); };
  z = 0;
  live = 0;
  row.each([&](uint32_t k, int) { z += mass_of(k), live += k > kNothing; });
  row.totals(z, live);
  Place stop{kNothing, 1u, z};
  auto through = [&](const Place &a) { return a.above + (u64)a.rank * mass_of(a.key); };
  if (cut_k && (u64)top_k < live) {
    stop = row.descend(false, (u64)top_k, mass_of);
    z = through(stop);
  }
  if (cut_p) {
    const u64 over = (u64)floor(share * (double)z) + 1;
    if (over <= z) stop = shorter(row.descend(true, over, mass_of), stop);
  }
  if (cut_m) {
    u64 kept = 0;
    row.each([&](uint32_t k, int) {
      const u64 w = mass_of(k);
      kept += w >= floor_m ? w : 0;
    });
    row.totals(kept, none);
    stop = shorter(row.descend(true, kept, mass_of), stop);
  }
  const u64 mass = through(stop);
  u64 target = (u64)ceil((double)u * (double)mass);
  target = target < 1 ? 1 : (target > mass ? mass : target);
  const Place at = shorter(row.descend(true, target, mass_of), stop);
  const int t = row.token_at(at.key, at.rank);
  if (t >= 0 && tid == 0) write(t, log_share(mass_of(at.key), mass));
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
  auto bytes = [](int s) { return (size_t)Layout::keys + (size_t)s * 4 + (size_t)((s + 31) / 32) * 4; };
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
