// Rotary positions (Su et al. 2021): every pair (a, b) of a head's values is
// turned by an angle that grows with the token's position,
//     u = s (a cos th - b sin th),   v = s (a sin th + b cos th),
//     th = position * inv_freq[i],   i the pair's place in the head,
// so that q_t . k_s depends on t - s alone.  RetNet as published turns its
// queries and keys this way in front of the retention (Sun et al. 2023, eq. 5);
// the reference's layer has no positions (aceflow/nn/retention.py:44-66).
// The gradient is the same map with -th, so one kernel serves both directions.
//
// Angles.  position * inv_freq in fp32 is off by 2^-24 of the angle: 0.06 rad
// at position 10^6.  The product is therefore formed in 64 bits, in turns,
// reduced to [-1/2, 1/2] there, and only the remainder goes to sincospif
// (2^-26 turns off, 1e-7 rad).
//
// Bound: HBM, each value read once and written once.  An angle costs two
// 64-bit multiplies and a sincospif (about 40 instructions), so a thread keeps
// the angles of its few pairs in registers and uses them for several heads.
#include "common.cuh"

namespace {

struct RotaryParams {
  const void *x;
  void *out;
  int64_t xb, xt, xh, ob, ot, oh;  // strides in elements: stream, token, head
  int T, heads, dim, rot;
  unsigned tokens;   // streams * T
  unsigned cols;     // column groups per head
  unsigned items;    // (head slot, column group) pairs per token
  int per_thread;    // heads a thread turns
  unsigned slots;    // ceil(heads / per_thread)
  unsigned block_tokens;
  const float *inv_freq;
  const void *pos;  // int32 or int64, or NULL: start + t
  int pos64;
  int64_t pb, pt, start;
  float scale;
  int inverse;
};

template <typename T, int W>
struct alignas(sizeof(T) * W) Pack {
  T v[W];
};
__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) {
  return __float2bfloat16(v);
}

__device__ __forceinline__ double position_of(const RotaryParams &p, unsigned b, unsigned t) {
  if (!p.pos) return (double)(p.start + (int64_t)t);
  const int64_t i = (int64_t)b * p.pb + (int64_t)t * p.pt;
  return p.pos64 ? (double)static_cast<const int64_t *>(p.pos)[i] : (double)static_cast<const int32_t *>(p.pos)[i];
}

// cos and sin (times the scale) of pair i at this position.
__device__ __forceinline__ void angle(const RotaryParams &p, double pos, int i, float &c, float &s) {
  const double turns = pos * ((double)p.inv_freq[i] * 0.15915494309189535);
  const float r = (float)(turns - rint(turns));
  sincospif(2.0f * r, &s, &c);
  c *= p.scale;
  s *= p.inverse ? -p.scale : p.scale;
}

constexpr int kThreads = 256;
constexpr int kFlight = 4;  // heads whose loads a thread has in flight

// W: values per access.  HALF: pairs (i, i + rot/2), a column group is W
// pairs, then groups of W values behind the turned part; else pairs
// (2i, 2i + 1), a column group is max(W, 2) values of the head.
template <typename T, int W, bool HALF>
__global__ void __launch_bounds__(kThreads) rotary_kernel(RotaryParams p) {
  constexpr int G = HALF ? W : (W < 2 ? 2 : W);  // values of one access group
  constexpr int N = HALF ? W : G / 2;            // pairs a thread turns
  constexpr int A = G / W;                       // accesses per group (2 for scalar interleaved pairs)
  using V = Pack<T, W>;
  const unsigned token0 = blockIdx.x * p.block_tokens;
  const unsigned ntok = min(p.block_tokens, p.tokens - token0);
  const T *xin = static_cast<const T *>(p.x);
  T *out = static_cast<T *>(p.out);
  const int half = p.rot / 2;
  for (unsigned it = threadIdx.x; it < ntok * p.items; it += kThreads) {
    const unsigned tl = it / p.items, rem = it - tl * p.items;
    const unsigned slot = rem / p.cols, col = rem - slot * p.cols;
    const unsigned token = token0 + tl, b = token / (unsigned)p.T, t = token - b * (unsigned)p.T;
    const T *xr = xin + (int64_t)b * p.xb + (int64_t)t * p.xt;
    T *orow = out + (int64_t)b * p.ob + (int64_t)t * p.ot;
    // where the group lies in a head, and the angles of its pairs
    int first, second = 0, turned;
    if (HALF) {
      const int groups = half / W;
      turned = (int)col < groups ? N : 0;
      first = turned ? (int)col * W : p.rot + ((int)col - groups) * W;
      second = first + half;
    } else {
      first = (int)col * G;
      turned = min(max((p.rot - first) / 2, 0), N);
    }
    float c[N], s[N];
    if (turned) {
      const double pos = position_of(p, b, t);
      const int i0 = HALF ? first : first / 2;
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (i < turned) angle(p, pos, i0 + i, c[i], s[i]);
    }
    const int h_end = min((int)(slot + 1) * p.per_thread, p.heads);
    for (int h0 = (int)slot * p.per_thread; h0 < h_end; h0 += kFlight) {
      V va[kFlight][A], vb[kFlight];
#pragma unroll
      for (int j = 0; j < kFlight; ++j) {
        if (h0 + j < h_end) {
          const T *src = xr + (int64_t)(h0 + j) * p.xh;
#pragma unroll
          for (int a = 0; a < A; ++a)
            if (first + a * W < p.dim) va[j][a] = *reinterpret_cast<const V *>(src + first + a * W);
          if (HALF && turned) vb[j] = *reinterpret_cast<const V *>(src + second);
        }
      }
#pragma unroll
      for (int j = 0; j < kFlight; ++j) {
        if (h0 + j < h_end) {
          T *dst = orow + (int64_t)(h0 + j) * p.oh;
          if (HALF) {
            if (turned) {
#pragma unroll
              for (int i = 0; i < N; ++i) {
                const float a = to_f(va[j][0].v[i]), bb = to_f(vb[j].v[i]);
                va[j][0].v[i] = from_f<T>(a * c[i] - bb * s[i]);
                vb[j].v[i] = from_f<T>(a * s[i] + bb * c[i]);
              }
              *reinterpret_cast<V *>(dst + second) = vb[j];
            }
            *reinterpret_cast<V *>(dst + first) = va[j][0];
          } else {
#pragma unroll
            for (int i = 0; i < N; ++i) {
              T &ra = va[j][(2 * i) / W].v[(2 * i) % W];
              T &rb = va[j][(2 * i + 1) / W].v[(2 * i + 1) % W];
              if (i < turned) {
                const float a = to_f(ra), bb = to_f(rb);
                ra = from_f<T>(a * c[i] - bb * s[i]);
                rb = from_f<T>(a * s[i] + bb * c[i]);
              }
            }
#pragma unroll
            for (int a = 0; a < A; ++a)
              if (first + a * W < p.dim) *reinterpret_cast<V *>(dst + first + a * W) = va[j][a];
          }
        }
      }
    }
  }
}

template <typename T, int W>
cudaError_t launch(const RotaryParams &p, bool half, unsigned blocks, cudaStream_t st) {
  if (half)
    rotary_kernel<T, W, true><<<blocks, kThreads, 0, st>>>(p);
  else
    rotary_kernel<T, W, false><<<blocks, kThreads, 0, st>>>(p);
  return cudaSuccess;
}

}  // namespace

extern "C" int af_rotary(af_ctx *ctx, const void *x, void *out, int is_bf16, const int64_t *x_strides,
                         const int64_t *out_strides, int batch, int T, int heads, int head_dim, const float *inv_freq,
                         int rot_dim, const void *positions, int positions_i64, const int64_t *pos_strides,
                         int64_t start, int interleaved, float scale, int inverse, af_stream_t stream) {
  const char *fn = "af_rotary";
  af::DeviceScope scope;
  AF_ENTER(ctx, fn);
  AF_REQUIRE(batch >= 0 && T >= 0 && heads >= 0 && head_dim > 0, "af_rotary", "bad sizes");
  AF_REQUIRE(rot_dim >= 2 && rot_dim % 2 == 0 && rot_dim <= head_dim, "af_rotary",
             "rot_dim %d must be even, at least 2 and at most head_dim %d", rot_dim, head_dim);
  AF_REQUIRE((int64_t)batch * T < (1ll << 31), "af_rotary", "batch * T must be below 2^31");
  if ((int64_t)batch * T == 0 || heads == 0) return AF_OK;
  AF_REQUIRE(x && out && inv_freq && x_strides && out_strides && (!positions || pos_strides), "af_rotary",
             "null argument");
  const size_t es = is_bf16 ? 2 : 4;
  // widest access that base addresses, strides, the head and its turned part allow
  int W = is_bf16 ? 8 : 4;
  auto fits = [&](int w) {
    if (reinterpret_cast<uintptr_t>(x) % (w * es) || reinterpret_cast<uintptr_t>(out) % (w * es)) return false;
    const int64_t ext[3] = {batch, T, heads};  // the stride of a dimension of one is never used
    for (int i = 0; i < 3; ++i)
      if (ext[i] > 1 && (x_strides[i] % w || out_strides[i] % w)) return false;
    return head_dim % w == 0 && (interleaved || (rot_dim / 2) % w == 0);
  };
  while (W > 1 && !fits(W)) W /= 2;
  RotaryParams p;
  p.x = x, p.out = out;
  p.xb = x_strides[0], p.xt = x_strides[1], p.xh = x_strides[2];
  p.ob = out_strides[0], p.ot = out_strides[1], p.oh = out_strides[2];
  p.T = T, p.heads = heads, p.dim = head_dim, p.rot = rot_dim;
  p.tokens = (unsigned)((int64_t)batch * T);
  const int G = interleaved && W < 2 ? 2 : W;
  p.cols = interleaved ? (unsigned)((head_dim + G - 1) / G) : (unsigned)(rot_dim / 2 / W + (head_dim - rot_dim) / W);
  // Heads per thread: 8 share one thread's angles once that still leaves every
  // SM a full set of threads; a short call rather spreads over the SMs.
  const int64_t fill = (int64_t)ctx->num_sms * 2048;
  p.per_thread = 8;
  while (p.per_thread > 1 && (int64_t)p.tokens * p.cols * ((heads + p.per_thread - 1) / p.per_thread) < fill)
    p.per_thread /= 2;
  p.slots = (unsigned)((heads + p.per_thread - 1) / p.per_thread);
  AF_REQUIRE((int64_t)p.slots * p.cols < (1 << 24), "af_rotary", "heads * head_dim is too large");
  p.items = p.slots * p.cols;
  p.block_tokens = p.items >= kThreads ? 1 : kThreads / p.items;
  p.inv_freq = inv_freq, p.pos = positions, p.pos64 = positions_i64;
  p.pb = positions ? pos_strides[0] : 0, p.pt = positions ? pos_strides[1] : 0;
  p.start = start, p.scale = scale, p.inverse = inverse;
  const unsigned blocks = (p.tokens + p.block_tokens - 1) / p.block_tokens;
  cudaStream_t st = af::stream_of(stream);
  if (is_bf16) {
    using B16 = __nv_bfloat16;
    W == 8   ? launch<B16, 8>(p, !interleaved, blocks, st)
    : W == 4 ? launch<B16, 4>(p, !interleaved, blocks, st)
    : W == 2 ? launch<B16, 2>(p, !interleaved, blocks, st)
             : launch<B16, 1>(p, !interleaved, blocks, st);
  } else {
    W == 4   ? launch<float, 4>(p, !interleaved, blocks, st)
    : W == 2 ? launch<float, 2>(p, !interleaved, blocks, st)
             : launch<float, 1>(p, !interleaved, blocks, st);
  }
  return af::launched(ctx, fn);
}
