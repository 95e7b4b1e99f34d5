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
// prefix's end.  So nothing is sorted: a place is a key (the logit as an
// order-preserving 32-bit number) and a rank among its equals, and each place
// is found by descending the key's digits over histograms of counts and
// masses.
//
// Masses are whole numbers, w in units of 2^-44 (2^19 tokens sum to less than
// 2^64): their sums do not depend on any order, so a row's token is the same
// in every run and every launch shape, and no border between two tokens moves
// by more than 2^-26 of the total even where 2^19 roundings all agree.
#include "common.cuh"

namespace {

using u64 = unsigned long long;
constexpr int kThreads = 512;
constexpr double kOne = 17592186044416.0;  // 2^44: the mass of the largest logit

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
constexpr uint32_t kNothing = 0x007fffffu;  // key of -inf: keys above it are candidates

struct SampleParams {
  const void *logits;
  int b16;
  int64_t ld;
  int V;
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

struct Weigher {
  double top, c;  // largest logit, log2(e) / temperature
  bool inf;       // the largest logit is +inf: only its equals have mass
  __device__ __forceinline__ u64 operator()(uint32_t key) const {
    if (key <= kNothing) return 0;
    const float x = value_of(key);
    if (inf) return x == INFINITY ? (u64)kOne : 0;
    const double a = ((double)x - top) * c;
    return a > -46.0 ? __double2ull_rn(exp2(a) * kOne) : 0;
  }
};

struct Shared {
  u64 mass[256];
  unsigned count[256];
  u64 red[32];
  unsigned digit, before_n;
  u64 before_m;
  unsigned scan[kThreads];
};

template <typename F>
__device__ u64 block_total(Shared &sh, F &&mine) {
  u64 v = mine();
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh.red[threadIdx.x >> 5] = v;
  __syncthreads();
  u64 t = 0;
  for (int w = 0; w < kThreads / 32; ++w) t += sh.red[w];
  return t;
}

// A place in the order: the first `rank` (from 1) of the tokens with that key,
// and the mass of all keys above it.
struct Place {
  uint32_t key;
  unsigned rank;
  u64 above;
};

__global__ void __launch_bounds__(kThreads) sample_tokens_kernel(SampleParams p) {
  extern __shared__ uint32_t seen[];  // a bit for each token of the row's context
  __shared__ Shared sh;
  const int r = blockIdx.x, tid = threadIdx.x, V = p.V;
  const float temp = p.temperature ? p.temperature[r] : p.temperature_all;
  const float top_p = p.top_p ? p.top_p[r] : p.top_p_all;
  const float min_p = p.min_p ? p.min_p[r] : p.min_p_all;
  const float pen = p.penalty ? p.penalty[r] : p.penalty_all;
  const int top_k = p.top_k ? p.top_k[r] : p.top_k_all;
  const bool penalise = p.ctx_len > 0 && pen != 1.0f;
  if (penalise) {
    for (int i = tid; i < (V + 31) / 32; i += kThreads) seen[i] = 0;
    __syncthreads();
    for (int i = tid; i < p.ctx_len; i += kThreads) {
      const int t = p.ctx[(int64_t)r * p.ctx_stride + i];
      if (t >= 0 && t < V) atomicOr(&seen[t >> 5], 1u << (t & 31));
    }
    __syncthreads();
  }
  auto key_at = [&](int i) {
    const int64_t at = (int64_t)r * p.ld + i;
    float x = p.b16 ? __bfloat162float(static_cast<const __nv_bfloat16 *>(p.logits)[at])
                    : static_cast<const float *>(p.logits)[at];
    if (penalise && (seen[i >> 5] >> (i & 31) & 1)) x = x > 0.f ? x / pen : x * pen;
    return key_of(x);
  };

  uint32_t kmax = 0;
  for (int i = tid; i < V; i += kThreads) kmax = max(kmax, key_at(i));
  kmax = __reduce_max_sync(0xffffffffu, kmax);
  if ((tid & 31) == 0) sh.red[tid >> 5] = kmax;
  __syncthreads();
  for (int w = 0; w < kThreads / 32; ++w) kmax = max(kmax, (uint32_t)sh.red[w]);
  if (kmax <= kNothing) {
    if (tid == 0) {
      p.token[r] = -1;
      if (p.logprob) p.logprob[r] = -INFINITY;
    }
    return;
  }

  // The index of the rank-th token (from 1) with that key.
  auto token_of = [&](uint32_t key, unsigned rank) {
    const int per = (V + kThreads - 1) / kThreads, i0 = min(tid * per, V), i1 = min(i0 + per, V);
    unsigned n = 0;
    for (int i = i0; i < i1; ++i) n += key_at(i) == key;
    sh.scan[tid] = n;
    __syncthreads();
    unsigned before = 0;
    for (int k = 0; k < tid; ++k) before += sh.scan[k];
    if (before < rank && rank <= before + n) {
      for (int i = i0; i < i1; ++i)
        if (key_at(i) == key && ++before == rank) sh.digit = i;
    }
    __syncthreads();
    return (int)sh.digit;
  };

  const bool greedy = !(temp > 1e-4f);
  if (greedy) {
    const int t = token_of(kmax, 1);
    if (tid == 0) {
      p.token[r] = t;
      if (p.logprob) p.logprob[r] = 0.f;
    }
    return;
  }
  Weigher weigh{(double)value_of(kmax), 1.4426950408889634 / (double)fmaxf(temp, 1e-5f), value_of(kmax) == INFINITY};

  // The first place where the running count (by_mass false) or mass reaches
  // `target` (>= 1).
  auto find = [&](bool by_mass, u64 target) {
    uint32_t prefix = 0;
    u64 bm = 0;
    unsigned bn = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
      __syncthreads();
      for (int i = tid; i < 256; i += kThreads) sh.mass[i] = 0, sh.count[i] = 0;
      __syncthreads();
      for (int i = tid; i < V; i += kThreads) {
        const uint32_t k = key_at(i);
        if (k > kNothing && (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8)))) {
          atomicAdd(&sh.count[k >> shift & 255], 1u);
          atomicAdd(&sh.mass[k >> shift & 255], weigh(k));
        }
      }
      __syncthreads();
      if (tid == 0) {
        u64 m = bm;
        unsigned n = bn;
        int d = 255;  // the target is at most what the histogram holds
        for (; d > 0 && (by_mass ? m + sh.mass[d] : (u64)(n + sh.count[d])) < target; --d)
          m += sh.mass[d], n += sh.count[d];
        sh.digit = d;
        sh.before_m = m, sh.before_n = n;
      }
      __syncthreads();
      prefix |= sh.digit << shift;
      bm = sh.before_m, bn = sh.before_n;
    }
    Place at;
    at.key = prefix, at.above = bm;
    if (by_mass) {
      const u64 w = weigh(prefix), need = target - bm;
      at.rank = w ? (unsigned)((need + w - 1) / w) : 1u;
    } else {
      at.rank = (unsigned)(target - bn);
    }
    return at;
  };
  auto mass_through = [&](const Place &a) { return a.above + (u64)a.rank * weigh(a.key); };
  auto shorter = [](const Place &a, const Place &b) {
    return a.key > b.key || (a.key == b.key && a.rank <= b.rank) ? a : b;
  };

  // candidates and their mass
  const u64 all = block_total(sh, [&] {
    u64 m = 0;
    for (int i = tid; i < V; i += kThreads) m += key_at(i) > kNothing;
    return m;
  });
  Place end{kNothing, 1u, 0};
  u64 z;
  if (top_k > 0 && (u64)top_k < all) {
    end = find(false, (u64)top_k);
    z = mass_through(end);
  } else {
    z = block_total(sh, [&] {
      u64 m = 0;
      for (int i = tid; i < V; i += kThreads) m += weigh(key_at(i));
      return m;
    });
    end.above = z;
  }
  if (top_p < 1.0f || top_p != top_p) {
    const u64 over = (u64)floor(fmax((double)top_p, 0.0) * (double)z) + 1;  // F > top_p z
    if (over <= z) end = shorter(find(true, over), end);
  }
  if (min_p > 0.0f) {
    const u64 floor_m = (u64)ceil(fmin((double)min_p, 1.0) * kOne);
    // the mass of w >= min_p, and the place of its last token
    const u64 m = block_total(sh, [&] {
      u64 s = 0;
      for (int i = tid; i < V; i += kThreads) {
        const u64 w = weigh(key_at(i));
        if (w >= floor_m) s += w;
      }
      return s;
    });
    end = shorter(find(true, m), end);
  }
  const u64 mass = mass_through(end);
  const float u = fminf(fmaxf(p.uniforms[r], 0.0f), 0.99999994f);
  u64 target = (u64)ceil((double)u * (double)mass);
  target = target < 1 ? 1 : (target > mass ? mass : target);
  const Place at = shorter(find(true, target), end);
  const int t = token_of(at.key, at.rank);
  if (tid == 0) {
    p.token[r] = t;
    if (p.logprob) p.logprob[r] = (float)(log((double)weigh(at.key)) - log((double)mass));
  }
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
  AF_REQUIRE(vocab <= AF_SAMPLE_TOKENS_MAX_VOCAB, "af_sample_tokens", "vocab %d exceeds the maximum %d", vocab,
             AF_SAMPLE_TOKENS_MAX_VOCAB);
  AF_REQUIRE(context_len >= 0 && (context_len == 0 || context_tokens), "af_sample_tokens", "bad context");
  AF_REQUIRE(penalty || penalty_all > 0.f, "af_sample_tokens", "the repetition penalty must be positive");
  if (rows == 0) return AF_OK;
  AF_REQUIRE(logits && uniforms && token, "af_sample_tokens", "null argument");
  SampleParams p{logits, logits_bf16 != 0, row_stride, vocab, context_tokens, context_stride, context_len, temperature,
                 top_p, min_p, penalty, top_k, temperature_all, top_p_all, min_p_all, penalty_all, top_k_all, uniforms,
                 token, logprob};
  const size_t smem = context_len ? (size_t)((vocab + 31) / 32) * 4 : 0;
  static std::atomic<unsigned long long> attr_devices{0};
  if (int rc = af::smem_attr(ctx, reinterpret_cast<const void *>(sample_tokens_kernel),
                             AF_SAMPLE_TOKENS_MAX_VOCAB / 8, attr_devices, fn))
    return rc;
  sample_tokens_kernel<<<rows, kThreads, smem, af::stream_of(stream)>>>(p);
  return af::launched(ctx, fn);
}
