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
// so the shortest prefix is the one with the least mass M, and the draw is the
// first place where F >= u M.  The row is never sorted.  A cluster of CTAs
// holds it in shared memory, one slice each (one read of the logits), and
//   1. finds the maximum;
//   2. with top-k: counts the tokens in bins of 1/16 octave of w and takes
//      those through the bin that holds the k-th; with min-p alone: takes what
//      it may keep;
//   3. if at most kList tokens were taken, the first CTA reads the places off
//      them: it sums their masses by bins, finds a place's bin from the running
//      sum and orders that bin's few tokens;
//   4. without top-k: the row's masses go into the bins.  Their running sums
//      give Z and the bin where top-p is crossed, and that bin's two ends the
//      few bins where the draw can end; the first CTA gets the tokens of all
//      these at once and finds both places, each by finer bins of one bin;
//   5. else (a bin of more than kList tokens: great numbers of equal or nearly
//      equal logits, or a top_k above kList) every place is found by
//      descending the digits of its key over histograms.
//
// Masses are whole numbers in units of 2^-44, in 64 bits: their sums do not
// depend on any order, so a row's token is the same in every run and in every
// launch shape.  A mass has at most 31 significant bits and is off by at most
// the larger of 2^-29 of itself and half a unit (a token below 2^-45 has none
// and is never drawn): together no more than 2^-29 + vocab 2^-45 of a row, 1.2e-8
// at the largest vocabulary.  What min-p keeps is decided on the logits in 64
// bits, not on these masses, so that it holds for small weights too.
//
// Bound: one read of the logits would take 20.5 us for 256 rows of 131072 in
// fp32; with top-p 0.95 over a broad row the call takes 184 us: in 7 waves of
// clusters, each a chain of about 48000 cycles (8300 to load, 9300 for the
// masses, the rest barriers, scans and the first CTA's search).  Summing Z in
// a pass of its own, with a second one for the bins and a collection for each
// place, took 365 us.  Few rows are bound by the chain alone: 12.4 us for one
// row of 32000 with top-k 40, 24 us for 64 such rows with mixed settings.
// Step 5 costs a row of 131072 0.3 ms (all logits equal) to 0.5 ms (all within a
// few bins).
#include "common.cuh"
#include "sm100.cuh"

#include <algorithm>

namespace {

using u64 = unsigned long long;
using sm100::cluster_ctarank;
constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCtas = 8;       // CTAs of a row's cluster
constexpr int kList = 2048;       // tokens the first CTA takes over at once
constexpr int kSome = 512;        // of them, those of one bin that are sorted at once
constexpr int kPairs = 128;       // tokens that are compared each with each
constexpr int kBins = 46 * 16;    // w down to 2^-46 in sixteenths of an octave; the rest behind them
constexpr int kBinRoom = 2 * kThreads;
constexpr int kWords = 3;         // words that hold a bit for each of a thread's tokens
static_assert(kWords * 32 * kThreads * kMaxCtas >= AF_SAMPLE_TOKENS_MAX_VOCAB + 8 * kMaxCtas, "every token has a bit");
constexpr u64 kOne = 1ull << 44;  // the mass of the largest logit
constexpr float kLowest = -3.4028235e38f;

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
// bits of the context's tokens.  It is addressed by 32-bit shared addresses
// throughout.
struct Layout {
  static constexpr uint32_t list = 0;                  // u64 [kList]: (~key, index), ascending is the order
  static constexpr uint32_t run = list + 8 * kList;    // u64 [kList]: running mass along a sorted list
  static constexpr uint32_t lo = run;                  // u32 [kBinRoom], hi alike: bins while they are filled
  static constexpr uint32_t hi = lo + 4 * kBinRoom;
  static constexpr uint32_t some = run;                // u64 [kSome]: the tokens of one bin of the list,
  static constexpr uint32_t some_run = some + 8 * kSome;  // u64 [kSome]: and their running mass
  static constexpr uint32_t bins = run + 8 * kList;    // u64 [kBinRoom]: running masses (counts) over the row's bins
  static constexpr uint32_t own_bins = hi + 4 * kBinRoom;  // alike, over the list's, until the whole list is sorted
  static constexpr uint32_t power = bins + 8 * kBinRoom;   // double [16]
  static constexpr uint32_t slot = power + 8 * 16;           // u64 [2][kMaxCtas]
  static constexpr uint32_t warp = slot + 8 * 2 * kMaxCtas;  // u64 [kWarps]
  static constexpr uint32_t before = warp + 8 * kWarps;      // u64 [2]
  static constexpr uint32_t listed = before + 16;            // u32
  static constexpr uint32_t found = listed + 4;              // u32
  static constexpr uint32_t settings = found + 4;             // u32 [5]
  static constexpr uint32_t logits = settings + 24;           // float [slice]
};
static_assert(Layout::logits % 16 == 0, "logits are read sixteen bytes at a time");
static_assert(16 * kBinRoom <= 8 * kList && 16 * kSome <= 8 * kBinRoom, "what shares the running masses' place fits");
static_assert(kBins < kBinRoom, "every bin has room");

__device__ __forceinline__ u64 lds64(uint32_t a) {
  u64 v;
  asm volatile("ld.shared.u64 %0, [%1];" : "=l"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void sts64(uint32_t a, u64 v) {
  asm volatile("st.shared.u64 [%0], %1;" ::"r"(a), "l"(v) : "memory");
}
__device__ __forceinline__ void sts32(uint32_t a, uint32_t v) {
  asm volatile("st.shared.u32 [%0], %1;" ::"r"(a), "r"(v) : "memory");
}
__device__ __forceinline__ uint32_t add32(uint32_t a, uint32_t v) {
  uint32_t old;
  asm volatile("atom.shared.add.u32 %0, [%1], %2;" : "=r"(old) : "r"(a), "r"(v) : "memory");
  return old;
}
// Additions whose old value nobody needs.
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
// Another CTA's memory, by an address from in_cta (slower, this CTA's own too:
// such an access leaves the SM).
__device__ __forceinline__ u64 far64(uint32_t a) {
  u64 v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t far32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void put_far64(uint32_t a, u64 v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(a), "l"(v) : "memory");
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
// Another CTA's memory may be touched only once that CTA runs: each says so as
// it starts and waits for the others in front of the first exchange, by when
// its slice is loaded.
__device__ __forceinline__ void cluster_started() { asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory"); }
__device__ __forceinline__ void cluster_all_started() { asm volatile("barrier.cluster.wait;" ::: "memory"); }
// All threads of the cluster, whether or not their warps have reconverged.
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive;\n\tbarrier.cluster.wait;" ::: "memory");
}

// 2^(44 - (j + 1/2) / 16): the middle of each sixteenth of the first octave.
__constant__ double kPower[16] = {17215221774114.625, 16485352848845.686, 15786427971528.205, 15117135216047.139,
                                  14476218277650.682, 13862474114786.947, 13274750690919.037, 12711944812079.727,
                                  12173000056106.76,  11656904789671.754, 11162690269380.588, 10689428823380.896,
                                  10236232110063.44,  9802249450588.832,  9386666232109.658,  8988702378690.727};

// The mass of a token: w = 2^-t, t = (max - l) log2(e) / T.  b = floor(16 t) by
// t's fp32 form (never smaller for a smaller logit) is its bin; in 64 bits, with
// f = t - (b + 1/2) / 16, 2^-f is the Taylor series of exp(-f ln 2) to its
// fourth power (|f| <= 1/32: 2^-34 off), 2^-((b mod 16 + 1/2) / 16) comes from a
// table whose 16 doubles lie in 32 different banks, and the octave b / 16 goes
// into the exponent.  The 64-bit pipe has half the fp32 rate and nothing else
// to do here.
struct Weigher {
  float top, ch;
  double dtop, c;
  uint32_t power;
  __device__ __forceinline__ float lead(float x) const { return __fmul_rn(top - x, ch); }
  __device__ __forceinline__ static bool some(float t) { return t < 46.0f; }
  // floor(16 t): behind 1.5 * 2^23 a sum holds no fraction.
  __device__ __forceinline__ static int sixteenths(float t) {
    return __float_as_int(__fmaf_rd(t, 16.0f, 12582912.0f)) - 0x4b400000;
  }
  __device__ __forceinline__ int bin(float x) const {
    const float t = lead(x);
    return some(t) ? sixteenths(t) : kBins;
  }
  // The mass in a bin is its 31 bits << shift.
  __device__ __forceinline__ static int shift(int b) { return max(13 - (b >> 4), 0); }
  __device__ __forceinline__ uint32_t bits(float x, int b) const {
    const double t = fma(dtop - (double)x, c, -0.03125);
    const double f = t - (__hiloint2double(0x42f80000, b) - 422212465065984.0);  // 1.5 * 2^48 + b / 16
    double q = fma(f, 0.009618129107628477, -0.05550410866482158);  // (-ln 2)^n / n!, n = 4 .. 1
    q = fma(f, q, 0.24022650695910072);
    q = fma(f, q, -0.6931471805599453);
    u64 table;  // not volatile: nothing writes it any more, so the loads of several tokens may overlap
    asm("ld.shared.u64 %0, [%1];" : "=l"(table) : "r"(power + 8 * (b & 15)));
    const double w = __hiloint2double((int)(table >> 32) - ((b >> 4) << 20), (int)(uint32_t)table);
    // behind 2^(52 + shift) the bits above the shift stand in the low word
    return (uint32_t)__double2loint(fma(w, f * q, w) + __hiloint2double(0x43300000 + (shift(b) << 20), 0));
  }
  __device__ __forceinline__ u64 operator()(float x) const {
    const float t = lead(x);
    const int b = sixteenths(fminf(t, 46.0f)), s = shift(b);
    const uint32_t q = bits(x, b);
    const u64 m = (u64)__funnelshift_l(q, 0u, s) << 32 | (q << s);
    return some(t) ? m : 0;
  }
  // log(w / mass): w's logarithm needs none.
  __device__ __forceinline__ float log_share(float x, u64 mass) const {
    return (float)(((double)x - dtop) * c * 0.6931471805599453 - log((double)mass * (1.0 / (double)kOne)));
  }
  // Bounds on the logits of all tokens with t below (above) the given one.
  __device__ __forceinline__ float logit_below(double t) const {
    return fmaxf(__double2float_rd(dtop - (t + 1.0 / 64) / c), kLowest);
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

// A place on the first CTA's list: the mass through it, and its token.
struct Pick {
  u64 through;
  uint32_t token;
  float logit;
};

struct Row {
  uint32_t sm;  // this CTA's shared memory
  int n, base, ctas, rank;  // tokens of this CTA, their first index, CTAs of the row, this one's place
  int flip = 0;

  // ---- over the row
  // The first CTA's value, on every CTA.
  __device__ __forceinline__ u64 from_first(u64 v) { return lds64(exchange(v)); }
  // This CTA's value to every CTA of the row, then a cluster barrier.  The slots
  // alternate, so the next exchange cannot overtake a reader.
  __device__ __forceinline__ uint32_t exchange(u64 v) {
    const uint32_t slot = sm + Layout::slot + 8 * kMaxCtas * flip;
    flip ^= 1;
    if (threadIdx.x < (unsigned)ctas) put_far64(in_cta(slot + 8 * rank, threadIdx.x), v);
    cluster_barrier();
    return slot;
  }
  // The sum over the CTA's threads, on every thread.
  __device__ u64 block_sum(u64 v) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if (lane == 0) sts64(sm + Layout::warp + 8 * (threadIdx.x >> 5), v);
    __syncthreads();
    v = lds64(sm + Layout::warp + 8 * (lane & (kWarps - 1)));
#pragma unroll
    for (int o = kWarps / 2; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  }
  __device__ u64 total(u64 v) {
    const uint32_t slot = exchange(block_sum(v));
    v = 0;
#pragma unroll
    for (int c = 0; c < kMaxCtas; ++c) v += c < ctas ? lds64(slot + 8 * c) : 0;
    return v;
  }
  // The largest key over all threads of the row.
  __device__ uint32_t largest(uint32_t v) {
    const int lane = threadIdx.x & 31;
    v = __reduce_max_sync(0xffffffffu, v);
    if (lane == 0) sts32(sm + Layout::warp + 8 * (threadIdx.x >> 5), v);
    __syncthreads();
    v = __reduce_max_sync(0xffffffffu, lds32(sm + Layout::warp + 8 * (lane & (kWarps - 1))));
    const uint32_t slot = exchange(v);
    v = 0;
#pragma unroll
    for (int c = 0; c < kMaxCtas; ++c) v = max(v, c < ctas ? lds32(slot + 8 * c) : 0);
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
  // Brings the tokens of the row that `take` accepts to the first CTA's memory
  // at `to`, in no order; returns their number, with nothing brought if it is
  // above kList.  Ends with a cluster barrier.
  template <typename F>
  __device__ unsigned bring(uint32_t to, F &&take) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n4 = (n + 3) / 4;
    const uint32_t mine = sm + Layout::run;  // this CTA's, before their place is known
    unsigned hits[kWords], through = 0;
#pragma unroll
    for (int w = 0; w < kWords; ++w) {
      hits[w] = 0;
      const int i0 = threadIdx.x + 8 * w * kThreads;
#pragma unroll 4
      for (int j = 0; j < 8; ++j)
        if (i0 + j * kThreads < n4) {
          const uint4 v = lds128(sm + Layout::logits + 16 * (i0 + j * kThreads));
          hits[w] |= ((unsigned)take(__uint_as_float(v.x)) | (unsigned)take(__uint_as_float(v.y)) << 1 |
                      (unsigned)take(__uint_as_float(v.z)) << 2 | (unsigned)take(__uint_as_float(v.w)) << 3)
                     << 4 * j;
        }
      through += __popc(hits[w]);
    }
    unsigned to_at = through;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned v = __shfl_up_sync(0xffffffffu, through, o);
      if (lane >= o) through += v;
    }
    to_at = through - to_at;
    __syncthreads();
    if (lane == 31) sts32(sm + Layout::warp + 8 * warp, through);
    __syncthreads();
    const unsigned of = lds32(sm + Layout::warp + 8 * (lane & (kWarps - 1)));
    to_at += __reduce_add_sync(0xffffffffu, lane < warp ? of : 0);
    const unsigned have = __reduce_add_sync(0xffffffffu, lane < kWarps ? of : 0);
#pragma unroll
    for (int w = 0; w < kWords; ++w)
      for (; hits[w]; hits[w] &= hits[w] - 1) {
        const int k = __ffs(hits[w]) - 1, i = 4 * (threadIdx.x + (8 * w + (k >> 2)) * kThreads) + (k & 3);
        const float x = __uint_as_float(lds32(sm + Layout::logits + 4 * i));
        if (to_at < kList) sts64(mine + 8 * to_at, (u64)~key_of(x) << 32 | (unsigned)(base + i));
        ++to_at;
      }
    const uint32_t slot = exchange(have);
    unsigned at = 0, all = 0;
#pragma unroll
    for (int c = 0; c < kMaxCtas; ++c) {
      const unsigned v = c < ctas ? (unsigned)lds64(slot + 8 * c) : 0;
      all += v;
      at += c < rank ? v : 0;
    }
    if (all <= kList) {
      const uint32_t there = in_cta(to, 0) + 8 * at;
      for (unsigned i = threadIdx.x; i < have; i += kThreads) put_far64(there + 8 * i, lds64(mine + 8 * i));
    }
    cluster_barrier();
    return all;
  }

  // ---- bins
  __device__ void clear_bins() {
    for (int b = threadIdx.x; b < 2 * kBinRoom; b += kThreads) sts32(sm + Layout::lo + 4 * b, 0);  // lo and hi
    __syncthreads();
  }
  __device__ __forceinline__ void add_to_bin(int b, uint32_t q) const {
    red32(sm + Layout::lo + 4 * b, q & 0xffffu);
    red32(sm + Layout::hi + 4 * b, q >> 16);
  }
  __device__ __forceinline__ static u64 in_bin(u64 lo, u64 hi, int s) { return s < 0 ? lo : ((hi << 16) + lo) << s; }
  // Running sums over kBinRoom bins, two neighbours a thread.
  __device__ void run_sums(u64 a, u64 b, uint32_t to) {
    to += 16 * threadIdx.x;
    scan(a + b, 0, to + 8);
    sts64(to, lds64(to + 8) - b);
    __syncthreads();
  }
  // Of this CTA's bins.
  template <typename S>
  __device__ void run_own_bins(S &&shift) {
    const int b = 2 * threadIdx.x;
    const uint32_t lo = sm + Layout::lo + 4 * b, hi = sm + Layout::hi + 4 * b;
    run_sums(in_bin(lds32(lo), lds32(hi), shift(b)), in_bin(lds32(lo + 4), lds32(hi + 4), shift(b + 1)),
             sm + Layout::own_bins);
  }
  // Of the whole row's, on every CTA: each CTA adds up its share of the bins
  // over all CTAs and gives the sums to all.  shift(b) < 0: counts.  Returns the
  // sum of `also` over the CTAs.
  template <typename S>
  __device__ u64 run_bins(u64 also, S &&shift) {
    const uint32_t slot = exchange(also), to = sm + Layout::bins;
    const int share = (kBins + ctas - 1) / ctas;
    for (int i = threadIdx.x; i < share; i += kThreads) {
      const int b = rank * share + i, s = shift(b);
      if (b >= kBins) break;
      uint32_t l[kMaxCtas], h[kMaxCtas];  // all loads under way before the first is used
#pragma unroll
      for (int c = 0; c < kMaxCtas; ++c) {
        l[c] = c < ctas ? far32(in_cta(sm + Layout::lo + 4 * b, c)) : 0;
        h[c] = c < ctas && s >= 0 ? far32(in_cta(sm + Layout::hi + 4 * b, c)) : 0;
      }
      u64 lo = 0, hi = 0;
#pragma unroll
      for (int c = 0; c < kMaxCtas; ++c) lo += l[c], hi += h[c];
      const u64 v = in_bin(lo, hi, s);
#pragma unroll
      for (int c = 0; c < kMaxCtas; ++c)
        if (c < ctas) put_far64(in_cta(to + 8 * b, c), v);
    }
    cluster_barrier();
    const int b = 2 * threadIdx.x;
    static_assert(kBins % 2 == 0, "a thread's two bins are both used or neither");
    const u64 v = b < kBins ? lds64(to + 8 * b) : 0, w = b < kBins ? lds64(to + 8 * b + 8) : 0;
    run_sums(v, w, to);
    u64 sum = 0;
#pragma unroll
    for (int c = 0; c < kMaxCtas; ++c) sum += c < ctas ? lds64(slot + 8 * c) : 0;
    return sum;
  }
  __device__ __forceinline__ u64 through_bin(int b, uint32_t of = Layout::bins) const {
    return b < 0 ? 0 : lds64(sm + of + 8 * b);
  }
  // The first bin whose running sum reaches target (<= the last one).
  __device__ int bin_of(u64 target, uint32_t of = Layout::bins) {
    int c = 0;
#pragma unroll
    for (int b = 0; b < kBinRoom; b += kThreads) c += __syncthreads_count(through_bin(b + (int)threadIdx.x, of) < target);
    return min(c, kBinRoom - 1);
  }

  // ---- in one CTA
  // Of m entries, those that `take` accepts onto this CTA's list; their number.
  template <typename F>
  __device__ int select(uint32_t from, int m, F &&take) {
    __syncthreads();  // what was on the list has been read
    if (threadIdx.x == 0) sts32(sm + Layout::listed, 0);
    __syncthreads();
    for (int i = threadIdx.x; i < m; i += kThreads) {
      const u64 e = lds64(from + 8 * i);
      if (take(logit_of(e))) sts64(sm + Layout::list + 8 * add32(sm + Layout::listed, 1), e);
    }
    __syncthreads();
    return (int)lds32(sm + Layout::listed);
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
    u64 w = lds64(sm + Layout::warp + 8 * (lane & (kWarps - 1)));
#pragma unroll
    for (int o = 1; o < kWarps; o <<= 1) {
      const u64 u = __shfl_up_sync(0xffffffffu, w, o, kWarps);
      if ((lane & (kWarps - 1)) >= o) w += u;
    }
    const int mine = threadIdx.x >> 5;
    const u64 prior = __shfl_sync(0xffffffffu, w, mine ? mine - 1 : 0);
    sts64(to, before + (mine ? prior : 0) + v);
    return before + __shfl_sync(0xffffffffu, w, kWarps - 1);
  }
  // Bitonic sort of m places of a list (padded to size), E neighbours per thread
  // in registers: partners in the same thread or warp trade without shared memory.
  template <int E>
  __device__ void sort_list(uint32_t list, int m, int size) {
    const int first = E * threadIdx.x;
    const uint32_t mine = list + 8 * first;
    const bool in = first < size;  // whole warps
    u64 v[E];
#pragma unroll
    for (int r = 0; r < E; ++r) v[r] = first + r < m ? lds64(mine + 8 * r) : ~0ull;
    for (int k = 2; k <= size; k <<= 1) {
      int j = k >> 1;
      for (; j >= 32 * E; j >>= 1) {  // partners in other warps
        __syncthreads();
        if (in) {
#pragma unroll
          for (int r = 0; r < E; ++r) sts64(mine + 8 * r, v[r]);
        }
        __syncthreads();
        if (in) {
          const bool small = ((first & j) == 0) == ((first & k) == 0);
          const uint32_t other = list + 8 * (first ^ j);
#pragma unroll
          for (int r = 0; r < E; ++r) {
            const u64 o = lds64(other + 8 * r);
            v[r] = (o < v[r]) == small ? o : v[r];
          }
        }
      }
      if (!in) continue;
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
    for (int r = 0; r < E; ++r)
      if (first + r < m) sts64(mine + 8 * r, v[r]);
    __syncthreads();
  }
  __device__ __forceinline__ static float logit_of(u64 entry) { return value_of((uint32_t)~(entry >> 32)); }
  // Sorts a list's m tokens and sums their masses along it.  All threads have
  // seen the list's entries; they see the results.
  template <typename W>
  __device__ void order(uint32_t list, uint32_t run, int m, const W &weigh) {
    const int tid = threadIdx.x;
    if (m <= kPairs) {  // few: every token against every other
      u64 e = 0, through = 0;
      int place = -1;
      if (tid < m) {
        e = lds64(list + 8 * tid);
        sts64(run + 8 * tid, weigh(logit_of(e)));
      }
      __syncthreads();
      if (tid < m) {
#pragma unroll 4
        for (int i = 0; i < m; ++i)
          if (lds64(list + 8 * i) <= e) through += lds64(run + 8 * i), ++place;
      }
      __syncthreads();
      if (tid < m) sts64(list + 8 * place, e), sts64(run + 8 * place, through);
      __syncthreads();
      return;
    }
    int size = 2 * kPairs;
    while (size < m) size <<= 1;
    if (size <= kThreads)
      sort_list<1>(list, m, size);
    else
      sort_list<kList / kThreads>(list, m, size);
    u64 before = 0;
    for (int i = 0; i < m; i += kThreads) {
      const int at = i + (int)threadIdx.x;
      before = scan(at < m ? weigh(logit_of(lds64(list + 8 * at))) : 0, before, run + 8 * at);
    }
    __syncthreads();
  }
};

// Finds places by mass among those of the m tokens at `from` that `take`
// accepts (the first CTA's list, or a part of what lies elsewhere): all tokens of
// the order between two places, `base` the mass in front of them.  bin(logit)
// puts them into at most kBinRoom bins in their order, a bin's masses have
// `shift`.
template <typename W, typename T, typename B, typename S>
struct Head {
  Row &row;
  const W &weigh;
  T take;
  B bin;
  S shift;
  uint32_t from;
  int m;
  u64 base;
  bool part;
  uint32_t list = 0, run = 0;  // what is sorted now: all of them, or the tokens of bin `at`
  int n = 0, at = -1;
  u64 before = 0;  // the mass in front of what is sorted

  __device__ __forceinline__ u64 entry(int i) const { return lds64(from + 8 * i); }
  __device__ void sort_all() {
    list = row.sm + Layout::list, run = row.sm + Layout::run;
    n = part ? row.select(from, m, take) : m;
    at = kBinRoom, before = base;
    row.order(list, run, n, weigh);
  }
  __device__ void begin() {
    if (!part && m <= kPairs) return sort_all();
    row.clear_bins();
    for (int i = threadIdx.x; i < m; i += kThreads) {
      const float x = Row::logit_of(entry(i));
      if (take(x)) {
        const int b = bin(x);
        row.add_to_bin(b, (uint32_t)(weigh(x) >> shift(b)));
      }
    }
    __syncthreads();
    row.run_own_bins(shift);
  }
  __device__ u64 mass() const { return at == kBinRoom ? lds64(run + 8 * (n - 1)) : row.through_bin(kBinRoom - 1, Layout::own_bins); }
  __device__ void focus(int b) {
    if (at == kBinRoom || at == b) return;
    if (threadIdx.x == 0) sts32(row.sm + Layout::listed, 0);
    __syncthreads();
    list = row.sm + Layout::some, run = row.sm + Layout::some_run;
    for (int i = threadIdx.x; i < m; i += kThreads) {
      const u64 e = entry(i);
      const float x = Row::logit_of(e);
      if (take(x) && bin(x) == b) {
        const uint32_t p = add32(row.sm + Layout::listed, 1);
        if (p < kSome) sts64(list + 8 * p, e);
      }
    }
    __syncthreads();
    n = (int)lds32(row.sm + Layout::listed);
    if (n > kSome) return sort_all();
    at = b, before = base + row.through_bin(b - 1, Layout::own_bins);
    row.order(list, run, n, weigh);
  }
  __device__ Pick pick(int i) const {
    const u64 e = lds64(list + 8 * i);
    return Pick{before + lds64(run + 8 * i), (uint32_t)e, Row::logit_of(e)};
  }
  // The first place where the mass reaches `target`.
  __device__ Pick by_mass(u64 target) {
    if (at != kBinRoom) focus(row.bin_of(target - base, Layout::own_bins));
    int c = 0;
    for (int i = 0; i < n; i += kThreads)
      c += __syncthreads_count(i + (int)threadIdx.x < n && before + lds64(run + 8 * (i + threadIdx.x)) < target);
    return pick(min(c, n - 1));
  }
  // The place of the given rank (from 1), `in_front` of the list's tokens lying in the bins in front of its bin b.
  __device__ Pick by_rank(int rank, int b, int in_front) {
    focus(b);
    return pick((at == kBinRoom ? rank : rank - in_front) - 1);
  }
};
template <typename W, typename T, typename B, typename S>
__device__ __forceinline__ Head<W, T, B, S> head_of(Row &row, const W &weigh, T take, B bin, S shift, uint32_t from,
                                                    int m, u64 base, bool part) {
  return Head<W, T, B, S>{row, weigh, take, bin, shift, from, m, base, part};
}

__device__ __forceinline__ u64 draw_target(float u, u64 mass) {
  const u64 t = (u64)ceil((double)u * (double)mass);
  return t < 1 ? 1 : (t > mass ? mass : t);
}

// Step 5, by digits of the key: all CTAs take part and know the answers.
struct Descent {
  Row row;
  Weigher weigh;
  bool inf;  // the largest logit is +inf: only its equals have mass

  __device__ __forceinline__ u64 mass(float x) const { return inf ? (x == INFINITY ? kOne : 0) : weigh(x); }
  __device__ __forceinline__ u64 through(const Place &a) const {
    return a.key ? a.above + (u64)a.rank * mass(value_of(a.key)) : a.above;
  }
  // The first place where the running count (or mass) reaches `target`.
  __device__ Place find(bool by_mass, u64 target) {
    const uint32_t masses = row.sm + Layout::run, counts = masses + 8 * 256, sum_m = counts + 8 * 256,
                   sum_n = sum_m + 8 * 256;
    Place at{0u, 1u, 0};
    u64 before_n = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
      cluster_barrier();
      for (int i = threadIdx.x; i < 512; i += kThreads) sts64(masses + 8 * i, 0);
      __syncthreads();
      const int lane = threadIdx.x & 31;
      for (int i0 = threadIdx.x - lane; i0 < row.n; i0 += kThreads) {  // whole warps
        const float x = i0 + lane < row.n ? __uint_as_float(lds32(row.sm + Layout::logits + 4 * (i0 + lane))) : -INFINITY;
        const uint32_t k = key_of(x), digit = k >> shift & 255;
        const bool in = x > -INFINITY && (shift == 24 || (k >> (shift + 8)) == (at.key >> (shift + 8)));
        const unsigned who = __ballot_sync(0xffffffffu, in);
        if (!who) continue;
        u64 m = in ? mass(x) : 0;
        // a warp that adds to one place adds once: equal logits would queue there token by token
        const uint32_t first = __shfl_sync(0xffffffffu, digit, __ffs(who) - 1);
        if (__all_sync(0xffffffffu, !in || digit == first)) {
#pragma unroll
          for (int o = 16; o; o >>= 1) m += __shfl_xor_sync(0xffffffffu, m, o);
          if (lane == 0) red64(counts + 8 * first, (u64)__popc(who)), red64(masses + 8 * first, m);
        } else if (in) {
          red64(counts + 8 * digit, 1ull);
          red64(masses + 8 * digit, m);
        }
      }
      cluster_barrier();
      for (int i = threadIdx.x; i < 256; i += kThreads) {
        u64 m = 0, c = 0;
        for (int r = 0; r < row.ctas; ++r) m += far64(in_cta(masses + 8 * i, r)), c += far64(in_cta(counts + 8 * i, r));
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
        sts32(row.sm + Layout::found, d);
        sts64(row.sm + Layout::before, m);
        sts64(row.sm + Layout::before + 8, c);
      }
      __syncthreads();
      at.key |= lds32(row.sm + Layout::found) << shift;
      at.above = lds64(row.sm + Layout::before), before_n = lds64(row.sm + Layout::before + 8);
    }
    cluster_barrier();
    if (by_mass) {
      const u64 w = mass(value_of(at.key)), need = target - at.above;
      at.rank = w ? (unsigned)((need + w - 1) / w) : 1u;
    } else {
      at.rank = (unsigned)(target - before_n);
    }
    return at;
  }
};

// The index of the place-th (from 1) token with that logit, on every thread of
// the CTA that holds it; -1 elsewhere.
__device__ int token_at(Row &row, float logit, unsigned place) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int per = (row.n + kWarps * 32 - 1) / (kWarps * 32) * 32;
  const int i0 = min(warp * per, row.n), i1 = min(i0 + per, row.n);  // this warp's stretch of the slice
  const uint32_t logits = row.sm + Layout::logits, found = row.sm + Layout::found;
  auto is = [&](int i) { return i < i1 && __uint_as_float(lds32(logits + 4 * i)) == logit; };
  unsigned have = 0;
  for (int i = i0; i < i1; i += 32) have += __popc(__ballot_sync(0xffffffffu, is(i + lane)));
  if (threadIdx.x == 0) sts32(found, ~0u);
  const u64 own = row.scan(lane ? 0 : have, 0, row.sm + Layout::run + 8 * threadIdx.x);  // of this CTA
  __syncthreads();
  const uint32_t slot = row.exchange(own);
  u64 before = lds64(row.sm + Layout::run + 8 * 32 * warp) - have;
  for (int c = 0; c < row.rank; ++c) before += lds64(slot + 8 * c);
  if (before < place && place <= before + have)
    for (int i = i0; i < i1; i += 32) {
      const bool hit = is(i + lane);
      const unsigned hits = __ballot_sync(0xffffffffu, hit);
      if (hit && before + __popc(hits & ((2u << lane) - 1)) == place) sts32(found, row.base + i + lane);
      before += __popc(hits);
    }
  __syncthreads();
  return (int)lds32(found);
}

struct Filters {
  bool cut_k, cut_p, cut_m;
  int top_k;
  double share;  // top_p
  float lowest;  // the lowest logit that min_p keeps
  float u;
  __device__ __forceinline__ u64 over(u64 z) const { return (u64)floor(share * (double)z) + 1; }  // F > top_p Z
};

// Step 5 (kept out of line: it hardly ever runs, and would cost the rest registers).
__device__ __noinline__ void descend(Row row, Weigher weigh, Filters f, int32_t *token, float *logprob) {
  Descent d{row, weigh, weigh.top == INFINITY};
  u64 z = 0, live = 0;
  d.row.each([&](float x, int) { z += d.mass(x), live += x > -INFINITY; });
  z = d.row.total(z);
  live = d.row.total(live);
  Place stop{0u, 1u, z};
  if (f.cut_k && (u64)f.top_k < live) {
    stop = d.find(false, (u64)f.top_k);
    z = d.through(stop);
  }
  if (f.cut_p && f.over(z) <= z) stop = shorter(d.find(true, f.over(z)), stop);
  if (f.cut_m) {
    u64 m = 0;
    d.row.each([&](float x, int) {
      const u64 w = d.mass(x);
      m += x >= f.lowest ? w : 0;
    });
    stop = shorter(d.find(true, d.row.total(m)), stop);
  }
  const u64 mass = d.through(stop);
  const Place at = shorter(d.find(true, draw_target(f.u, mass)), stop);
  const float x = value_of(at.key);
  const int t = token_at(d.row, x, at.rank);
  if (t >= 0 && threadIdx.x == 0) {
    *token = t;
    if (logprob) *logprob = d.inf ? -logf((float)(mass >> 44)) : weigh.log_share(x, mass);
  }
}

__global__ void __launch_bounds__(kThreads, 2) sample_tokens_kernel(SampleParams p) {
  cluster_started();
  extern __shared__ __align__(16) unsigned char smem[];
  const uint32_t sm = sm100::smem_u32(smem), logits = sm + Layout::logits;
  const uint32_t seen = logits + 4 * p.slice;  // a bit for each token of the context in this slice
  const int tid = threadIdx.x, ctas = (int)cluster_ctas(), rank = (int)cluster_ctarank();
  const int r = blockIdx.x / ctas;
  const int base = rank * p.slice, n = max(0, min(p.slice, p.V - base));
  Row row{sm, n, base, ctas, rank};

  const float pen = p.penalty ? p.penalty[r] : p.penalty_all;
  if (tid == 0) {  // the row's settings, until the slice is there
    sts32(sm + Layout::settings, __float_as_uint(p.temperature ? p.temperature[r] : p.temperature_all));
    sts32(sm + Layout::settings + 4, __float_as_uint(p.top_p ? p.top_p[r] : p.top_p_all));
    sts32(sm + Layout::settings + 8, __float_as_uint(p.min_p ? p.min_p[r] : p.min_p_all));
    sts32(sm + Layout::settings + 12, p.top_k ? p.top_k[r] : p.top_k_all);
    sts32(sm + Layout::settings + 16, __float_as_uint(p.uniforms[r]));
  }
  if (tid < 16) sts64(sm + Layout::power + 8 * tid, (u64)__double_as_longlong(kPower[tid]));

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
  constexpr int kBatch = 4;  // loads a thread has in flight
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
  __syncthreads();

  // 1. the maximum
  cluster_all_started();
  top = value_of(row.largest(key_of(top)));
  auto write = [&](int token, float logp) {
    p.token[r] = token;
    if (p.logprob) p.logprob[r] = logp;
  };
  if (!(top > -INFINITY)) {
    if (rank == 0 && tid == 0) write(-1, -INFINITY);
    return;
  }
  auto setting = [&](int i) { return lds32(sm + Layout::settings + 4 * i); };
  const float temp = __uint_as_float(setting(0));
  if (!(temp > 1e-4f)) {
    const int t = token_at(row, top, 1);
    if (t >= 0 && tid == 0) write(t, 0.f);
    return;
  }
  const double c = 1.4426950408889634 / (double)fminf(temp, 1e36f);  // octaves of w per unit of a logit
  const Weigher weigh{top, (float)c, (double)top, c, sm + Layout::power};
  const float top_p = __uint_as_float(setting(1)), min_p = __uint_as_float(setting(2));
  const int top_k = (int)setting(3);
  const float u = fminf(fmaxf(__uint_as_float(setting(4)), 0.0f), 0.99999994f);
  Filters f;
  f.cut_p = !(top_p >= 1.0f), f.cut_k = top_k > 0 && top_k < p.V, f.cut_m = min_p > 0.0f;
  f.top_k = top_k, f.u = u;
  f.share = f.cut_p ? (top_p > 0.f ? (double)top_p : 0.0) : 1.0;
  // w >= min_p where (l - max) c >= log2(min_p): the first fp32 value that is
  f.lowest = kLowest;
  if (f.cut_m) f.lowest = fmaxf(__double2float_ru(weigh.dtop + log2(fmin((double)min_p, 1.0)) / c), kLowest);

  unsigned m = kList + 1;
  int last = 0, in_front = 0;
  if (top == INFINITY) {
    // step 5 alone knows what to do
  } else if (f.cut_k) {
    // 2. counts: the tokens through the bin that holds the k-th (tokens behind all bins have no mass)
    row.clear_bins();
    row.each([&](float x, int) {
      const float t = weigh.lead(x);
      if (weigh.some(t)) red32(sm + Layout::lo + 4 * weigh.sixteenths(t), 1u);
    });
    row.run_bins(0, [](int) { return -1; });
    last = row.bin_of(min((u64)top_k, row.through_bin(kBinRoom - 1)));
    in_front = (int)row.through_bin(last - 1);
    const float end = (last + 1) / 16.0f;
    if (row.through_bin(last) <= kList)
      m = row.bring(sm + Layout::list, [&](float x) { return weigh.lead(x) < end; });
  } else if (!f.cut_p && f.cut_m) {
    // 2. the tokens that min-p may keep
    m = row.bring(sm + Layout::list, [&](float x) { return x >= f.lowest; });
  }

  if (m <= kList) {
    // 3. every place is on the first CTA's list
    if (rank) return;
    auto head = head_of(row, weigh, [](float) { return true; }, [&](float x) { return weigh.bin(x); },
                        [](int b) { return Weigher::shift(b); }, sm + Layout::list, (int)m, 0, false);
    head.begin();
    const u64 held = head.mass();
    const u64 z = f.cut_k && (int)m > top_k ? head.by_rank(top_k, last, in_front).through : held;
    u64 mass = z;
    if (f.cut_m) {
      u64 v = 0;
      for (int i = tid; i < (int)m; i += kThreads) {
        const float x = Row::logit_of(head.entry(i));
        v += x >= f.lowest ? weigh(x) : 0;
      }
      mass = min(mass, row.block_sum(v));
    }
    if (f.cut_p && f.over(z) <= held) mass = min(mass, head.by_mass(f.over(z)).through);
    const Pick t = head.by_mass(min(draw_target(u, mass), held));
    if (tid == 0) write((int)t.token, weigh.log_share(t.logit, mass));
    return;
  }

  if (!f.cut_k && top < INFINITY) {
    // 4. masses by bins, and in which of them the places lie
    row.clear_bins();
    u64 kept_m = 0;
    for (int i = tid; i < (n + 3) / 4; i += kThreads) {
      const uint4 v = lds128(logits + 16 * i);
      const float x[4] = {__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z), __uint_as_float(v.w)};
      float t[4];
      int b[4];
      uint32_t q[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        t[j] = weigh.lead(x[j]);
        b[j] = weigh.sixteenths(fminf(t[j], 46.0f));
        q[j] = weigh.bits(x[j], b[j]);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (weigh.some(t[j])) {
          row.add_to_bin(b[j], q[j]);
          if (f.cut_m) kept_m += x[j] >= f.lowest ? (u64)q[j] << weigh.shift(b[j]) : 0;
        }
    }
    if (f.cut_m) kept_m = row.block_sum(kept_m);
    kept_m = row.run_bins(kept_m, [](int b) { return Weigher::shift(b); });
    const u64 z = row.through_bin(kBinRoom - 1);
    u64 mass = f.cut_m ? min(z, kept_m) : z;
    // the crossing of top_p, unless it lies behind the mass that min-p keeps; the mass through it lies between
    // its bin's ends, and the draw in few bins
    const u64 over = f.cut_p ? f.over(z) : mass;
    const bool crossing = over < mass;
    const int b1 = crossing ? row.bin_of(over) : -1;
    const int b2 = row.bin_of(draw_target(u, min(mass, over)));
    const int b3 = crossing ? row.bin_of(draw_target(u, min(mass, row.through_bin(b1)))) : b2;
    const uint32_t stash = logits;  // nobody needs the first CTA's logits once its tokens are counted
    // t >= 0, so its bits have its order
    auto bits_at = [](int b) { return __float_as_uint(b / 16.0f); };
    auto in = [](float t, uint32_t from, uint32_t span) { return __float_as_uint(t) - from < span; };
    const uint32_t from1 = bits_at(b1), span1 = crossing ? bits_at(b1 + 1) - from1 : 0;
    const uint32_t from2 = bits_at(b2), span2 = bits_at(b3 + 1) - from2;
    m = row.bring(stash, [&](float x) {
      const float t = weigh.lead(x);
      return in(t, from1, span1) | in(t, from2, span2);
    });
    const bool all_there = m <= kList;  // else one bin after the other
    if (all_there && rank) return;
    for (bool draw = !crossing;; draw = true) {
      const u64 target = draw ? draw_target(u, mass) : over;
      const int b = row.bin_of(target);
      const uint32_t from = bits_at(b), span = bits_at(b + 1) - from;
      auto here = [&](float x) { return in(weigh.lead(x), from, span); };
      if (!all_there && (m = row.bring(sm + Layout::list, here)) > kList) break;
      if (rank == 0) {
        const uint32_t first = key_of(weigh.logit_above(b / 16.0)), span = first - key_of(weigh.logit_below((b + 1) / 16.0));
        const int s = max(0, 32 - __clz(span) - 10);  // span >> s < kBinRoom
        auto fine = [&](float x) { return (int)min((first - key_of(x)) >> s, kBinRoom - 1u); };
        auto head = head_of(row, weigh, here, fine, [&](int) { return Weigher::shift(b); },
                            all_there ? stash : sm + Layout::list, (int)m, row.through_bin(b - 1), all_there);
        head.begin();
        const Pick t = head.by_mass(target);
        if (draw && tid == 0) write((int)t.token, weigh.log_share(t.logit, mass));
        mass = min(mass, t.through);
      }
      if (draw) return;
      if (!all_there) mass = row.from_first(mass);
    }
  }
  descend(row, weigh, f, p.token + r, p.logprob ? p.logprob + r : nullptr);
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
  auto bytes = [](int s) {  // the slice with its context's bits; later the first CTA's tokens of a few bins
    return (size_t)Layout::logits + std::max((size_t)s * 4 + (size_t)((s + 31) / 32) * 4, (size_t)8 * kList);
  };
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
