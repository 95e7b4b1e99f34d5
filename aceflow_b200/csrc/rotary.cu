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
// reduced to [-1/2, 1/2] there, and only the remainder goes to sincospif in
// fp32; what its rounding leaves (2^-26 turns, 1e-7 rad at most) turns the result
// on to first order, so that cos and sin are off by their own roundings alone.
//
// Bound: HBM, each value read once and written once: 84 us for q and k of 8 x
// 4096 tokens (16 heads of 256, bf16, 0.54 GB), 0.97 of the measured copy rate.
// An angle costs two 64-bit multiplies and a sincospif (about 45
// instructions), so a thread keeps the angles of its few pairs in registers
// for up to 16 heads, whose first loads are under way while they are formed.
// bf16 values are taken apart and put together two at a time: one by one the
// conversions alone made the same call 100 us.
#include "common.cuh"

#include <algorithm>

namespace {

// n / d for n < 2^31 by a multiplication (Granlund and Montgomery 1994): 2^s >= d,
// m = floor(2^32 (2^s - d) / d) + 1.
struct Div {
  uint32_t d, m, s;
  void set(uint32_t by) {
    d = by, s = 0;
    while ((1ull << s) < by) ++s;
    m = (uint32_t)(((1ull << 32) * ((1ull << s) - by)) / by + 1);
  }
  __device__ __forceinline__ uint32_t of(uint32_t n) const { return (__umulhi(n, m) + n) >> s; }
};

struct RotaryParams {
  const void *x;
  void *out;
  int64_t xb, xt, xh, ob, ot, oh;  // strides in elements: stream, token, head
  int heads, dim, rot;
  unsigned tokens;        // streams * T
  Div T, cols, items;     // tokens of a stream, column groups of a head, (heads' slot, column group) items of a token
  unsigned block_tokens;  // tokens of a block
  int slot_heads;         // heads of a slot
  const float *inv_freq;
  const void *pos;  // int32 or int64, or NULL: start + t
  int pos64;
  int64_t pb, pt, start;
  float scale;
  int inverse;
};

// W values of one access, and as fp32.
template <typename T, int W>
struct alignas(sizeof(T) * W) Pack {
  T v[W];
};
template <int W>
__device__ __forceinline__ void unpack(const Pack<float, W> &p, float (&f)[W]) {
#pragma unroll
  for (int i = 0; i < W; ++i) f[i] = p.v[i];
}
template <int W>
__device__ __forceinline__ void unpack(const Pack<__nv_bfloat16, W> &p, float (&f)[W]) {
  if constexpr (W == 1) {
    f[0] = __bfloat162float(p.v[0]);
  } else {
    const uint32_t *w = reinterpret_cast<const uint32_t *>(&p);
#pragma unroll
    for (int i = 0; i < W / 2; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
}
template <int W>
__device__ __forceinline__ Pack<float, W> packed(const float (&f)[W], float) {
  Pack<float, W> p;
#pragma unroll
  for (int i = 0; i < W; ++i) p.v[i] = f[i];
  return p;
}
template <int W>
__device__ __forceinline__ Pack<__nv_bfloat16, W> packed(const float (&f)[W], __nv_bfloat16) {
  Pack<__nv_bfloat16, W> p;
  if constexpr (W == 1) {
    p.v[0] = __float2bfloat16(f[0]);
  } else {
    __nv_bfloat162 *w = reinterpret_cast<__nv_bfloat162 *>(&p);
#pragma unroll
    for (int i = 0; i < W / 2; ++i) w[i] = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
  }
  return p;
}

__device__ __forceinline__ double position_of(const RotaryParams &p, unsigned b, unsigned t) {
  if (!p.pos) return (double)(p.start + (int64_t)t);
  const int64_t i = (int64_t)b * p.pb + (int64_t)t * p.pt;
  return p.pos64 ? (double)static_cast<const int64_t *>(p.pos)[i] : (double)static_cast<const int32_t *>(p.pos)[i];
}

// cos and sin (times the scale) of pair i at this position.
__device__ __forceinline__ float2 angle(const RotaryParams &p, double pos, int i) {
  const double turns = pos * ((double)p.inv_freq[i] * 0.15915494309189535);
  const double left = turns - rint(turns);
  const float r = (float)left, rest = (float)(left - (double)r) * 6.2831855f;
  float c, s;
  sincospif(2.0f * r, &s, &c);
  const float cr = fmaf(-s, rest, c), sr = fmaf(c, rest, s);
  return make_float2(cr * p.scale, sr * (p.inverse ? -p.scale : p.scale));
}

constexpr int kThreads = 256;
constexpr int kHeads = 16;  // heads that share one thread's angles at most

// W: values per access.  HALF: pairs (i, i + rot/2), a column group is W
// pairs, then groups of W values behind the turned part; else pairs
// (2i, 2i + 1), a column group is max(W, 2) values of the head.
template <typename T, int W, bool HALF>
__global__ void __launch_bounds__(kThreads, 3) rotary_kernel(RotaryParams p) {
  constexpr int G = HALF ? W : (W < 2 ? 2 : W);  // values of one access group
  constexpr int N = HALF ? W : G / 2;            // pairs a thread turns
  constexpr int A = G / W;                       // accesses per group (2 for scalar interleaved pairs)
  constexpr int kFlight = HALF ? 2 : 4;        // heads whose loads (two each with HALF) a thread has in flight
  using V = Pack<T, W>;
  const unsigned token0 = blockIdx.x * p.block_tokens;
  const unsigned ntok = min(p.block_tokens, p.tokens - token0);
  const T *x = static_cast<const T *>(p.x);
  T *out = static_cast<T *>(p.out);
  const int half = p.rot / 2;
  for (unsigned it = blockIdx.y * kThreads + threadIdx.x; it < ntok * p.items.d; it += gridDim.y * kThreads) {
    const unsigned tl = p.items.of(it), rem = it - tl * p.items.d, slot = p.cols.of(rem);
    const int col = (int)(rem - slot * p.cols.d);
    const unsigned token = token0 + tl, b = p.T.of(token), t = token - b * p.T.d;
    // where the group lies in a head, and how many of its pairs turn
    int first, turned;
    if (HALF) {
      const int groups = half / W;
      turned = col < groups ? N : 0;
      first = col < groups ? col * W : p.rot + (col - groups) * W;
    } else {
      first = col * G;
      turned = min(max((p.rot - first) / 2, 0), N);
    }
    int h = (int)slot * p.slot_heads;
    const int h_end = min(h + p.slot_heads, p.heads);
    const T *src = x + ((int64_t)b * p.xb + (int64_t)t * p.xt + (int64_t)h * p.xh + first);
    T *dst = out + ((int64_t)b * p.ob + (int64_t)t * p.ot + (int64_t)h * p.oh + first);
    V va[kFlight][A], vb[kFlight];
    auto fetch = [&]() {
#pragma unroll
      for (int j = 0; j < kFlight; ++j)
        if (h + j < h_end) {
          const T *s = src + (int64_t)j * p.xh;
#pragma unroll
          for (int a = 0; a < A; ++a)
            if (W > 1 || first + a < p.dim) va[j][a] = *reinterpret_cast<const V *>(s + a * W);
          if (HALF && turned) vb[j] = *reinterpret_cast<const V *>(s + half);
        }
    };
    fetch();  // under way while the angles are formed
    float2 cs[N];
#pragma unroll
    for (int i = 0; i < N; ++i) cs[i] = make_float2(1.f, 0.f);
    if (turned) {
      const double pos = position_of(p, b, t);
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (i < turned) cs[i] = angle(p, pos, (HALF ? first : first / 2) + i);
    }
    for (;;) {
#pragma unroll
      for (int j = 0; j < kFlight; ++j) {
        if (h + j < h_end) {
          T *d = dst + (int64_t)j * p.oh;
          if (HALF && turned) {
            float a[W], bb[W], u[W], v[W];
            unpack(va[j][0], a);
            unpack(vb[j], bb);
#pragma unroll
            for (int i = 0; i < W; ++i) {
              u[i] = a[i] * cs[i].x - bb[i] * cs[i].y;
              v[i] = a[i] * cs[i].y + bb[i] * cs[i].x;
            }
            va[j][0] = packed(u, T());
            *reinterpret_cast<V *>(d + half) = packed(v, T());
          } else if (!HALF && turned) {
            float f[A][W];
#pragma unroll
            for (int a = 0; a < A; ++a) unpack(va[j][a], f[a]);
#pragma unroll
            for (int i = 0; i < N; ++i) {
              float &ra = f[(2 * i) / W][(2 * i) % W], &rb = f[(2 * i + 1) / W][(2 * i + 1) % W];
              const float a = ra, bb = rb;
              if (N == 1 || i < turned) {  // behind the turned part values are copied
                ra = a * cs[i].x - bb * cs[i].y;
                rb = a * cs[i].y + bb * cs[i].x;
              }
            }
#pragma unroll
            for (int a = 0; a < A; ++a) va[j][a] = packed(f[a], T());
          }
#pragma unroll
          for (int a = 0; a < A; ++a)
            if (W > 1 || first + a < p.dim) *reinterpret_cast<V *>(d + a * W) = va[j][a];
        }
      }
      h += kFlight;
      if (h >= h_end) break;
      src += kFlight * p.xh;
      dst += kFlight * p.oh;
      fetch();
    }
  }
}

template <typename T, int W>
void launch(const RotaryParams &p, bool half, dim3 grid, cudaStream_t st) {
  if (half)
    rotary_kernel<T, W, true><<<grid, kThreads, 0, st>>>(p);
  else
    rotary_kernel<T, W, false><<<grid, kThreads, 0, st>>>(p);
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
  p.heads = heads, p.dim = head_dim, p.rot = rot_dim;
  p.tokens = (unsigned)((int64_t)batch * T);
  const int G = interleaved && W < 2 ? 2 : W;
  const int cols = interleaved ? (head_dim + G - 1) / G : rot_dim / 2 / W + (head_dim - rot_dim) / W;
  // Heads per thread: up to 16 share one thread's angles, fewer while that
  // leaves an SM less than a full set of threads (8 x 4096 tokens of 16 heads of
  // 256: 84 us with 16, 90 with 8); then evenly over the threads of a token.
  const int64_t fill = (int64_t)ctx->num_sms * 2048;
  int share = kHeads;
  while (share > 1 && (int64_t)p.tokens * cols * ((heads + share - 1) / share) < fill) share /= 2;
  const int slots = (heads + share - 1) / share;
  p.slot_heads = (heads + slots - 1) / slots;
  AF_REQUIRE((int64_t)slots * cols < (1 << 24), "af_rotary", "heads * head_dim is too large");
  p.block_tokens = slots * cols >= kThreads ? 1 : kThreads / (slots * cols);
  p.T.set((uint32_t)T), p.cols.set((uint32_t)cols), p.items.set((uint32_t)(slots * cols));
  p.inv_freq = inv_freq, p.pos = positions, p.pos64 = positions_i64;
  p.pb = positions ? pos_strides[0] : 0, p.pt = positions ? pos_strides[1] : 0;
  p.start = start, p.scale = scale, p.inverse = inverse;
  const dim3 grid((p.tokens + p.block_tokens - 1) / p.block_tokens,
                  std::min((slots * cols + kThreads - 1) / kThreads, 65535));
  const cudaStream_t st = af::stream_of(stream);
  const bool half = !interleaved;
  if (is_bf16) {
    using B16 = __nv_bfloat16;
    W == 8   ? launch<B16, 8>(p, half, grid, st)
    : W == 4 ? launch<B16, 4>(p, half, grid, st)
    : W == 2 ? launch<B16, 2>(p, half, grid, st)
             : launch<B16, 1>(p, half, grid, st);
  } else {
    W == 4   ? launch<float, 4>(p, half, grid, st)
    : W == 2 ? launch<float, 2>(p, half, grid, st)
             : launch<float, 1>(p, half, grid, st);
  }
  return af::launched(ctx, fn);
}
