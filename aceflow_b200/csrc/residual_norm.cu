// The seam between two blocks of a decoder layer in one pass: the norm behind
// a block, its gate and residual scale, the residual add, and the norm in
// front of the next block.  For a residual row x, a block's output h, gate
// logits g, weights w1, s, w2 and a factor alpha,
//     n = h r1 w1,  r1 = 1 / sqrt(mean(h^2) + eps)      (n = h without w1)
//     z = alpha x + s swish(g) n                        (s, swish(g): 1 without)
//     y = z r2 w2,  r2 = 1 / sqrt(mean(z^2) + eps)      (no y without w2)
// The reference runs the add and the norm of its pre-norm layer apart
// (aceflow-core/src/cpu/mod.rs:672-700, norm.rs:6-59) and has no norm behind a
// block; DeepNet's alpha (Wang et al. 2022) and a learnt scale per channel
// (Touvron et al. 2021) are the usual residual scales.
//
// Backward, from dz and dy: with zh = z r2, hh = h r1, t = dy w2,
//     Z  = dz + r2 (t - zh mean(t zh))                  dx = alpha Z
//     dw2 = sum dy zh,  ds = sum Z swish(g) n,  dg = Z s n swish'(g)
//     N  = Z s swish(g),  dw1 = sum N hh  (= s A,  ds = w1 A,  A = sum Z swish(g) hh)
//     dh = r1 (N w1 - hh mean(N w1 hh))
// mean(N w1 hh) needs Z, which needs the other mean.  Both come from one
// reduction of three sums: with q = s swish(g) w1 hh,
//     sum N w1 hh = sum (dz + r2 t) q - r2 mean(t zh) sum zh q.
// z is formed again in fp32 from x, h and g (reading x costs what reading z
// would), so the rounding of the stored z does not enter the gradients.
//
// Bound: HBM, every row of every tensor moved once.  A row is held in
// registers by one group of threads; sums, statistics and the row itself are
// fp32, and each output is rounded once.  The column sums of the weights'
// gradients stay in registers while a block walks its rows, go out as one
// partial row per block and are added in a fixed order by a second kernel: no
// atomics, the same bits every run.
#include "common.cuh"

#include <algorithm>
#include <initializer_list>

namespace {

struct SeamParams {
  const void *x, *h, *g;  // g NULL: no gate (its type is h's)
  int64_t ldx, ldh, ldg;
  int x16, h16, y16;  // bf16 flags
  const float *w1, *s, *w2;
  float alpha, eps, inv_d;
  int rows, d;
  void *z, *y;     // contiguous rows; y NULL without w2
  float *stats;    // [2][rows]: r1, r2 (written by the forward when not NULL, read by the backward)
  const void *dz, *dy;  // either may be NULL (zero)
  int64_t lddz, lddy;
  void *dx, *dh, *dg;
  float *part;  // [2][parts][d]: sum Z swish(g) hh, sum dy zh
  int parts;
};

// VEC consecutive values of a row as they lie in memory: loads are issued
// without waiting, whatever the type; the conversion comes with the first use.
template <int VEC>
struct Raw;
template <>
struct Raw<8> {
  uint4 a, b;
  __device__ __forceinline__ void load(const void *p, int64_t i, bool b16) {
    const char *q = static_cast<const char *>(p) + i * (b16 ? 2 : 4);
    a = __ldcs(reinterpret_cast<const uint4 *>(q));
    if (!b16) b = __ldcs(reinterpret_cast<const uint4 *>(q) + 1);
  }
  __device__ __forceinline__ void get(float (&v)[8], bool b16) const {
    if (b16) {
      const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    } else {
      const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(w[i]);
    }
  }
};
template <>
struct Raw<2> {
  uint32_t a, b;
  __device__ __forceinline__ void load(const void *p, int64_t i, bool b16) {
    if (b16) {
      a = __ldcs(reinterpret_cast<const unsigned int *>(static_cast<const char *>(p) + 2 * i));
    } else {
      const uint2 q = __ldcs(reinterpret_cast<const uint2 *>(static_cast<const char *>(p) + 4 * i));
      a = q.x, b = q.y;
    }
  }
  __device__ __forceinline__ void get(float (&v)[2], bool b16) const {
    v[0] = __uint_as_float(b16 ? a << 16 : a);
    v[1] = __uint_as_float(b16 ? a & 0xffff0000u : b);
  }
};
template <>
struct Raw<1> {
  uint32_t a;
  __device__ __forceinline__ void load(const void *p, int64_t i, bool b16) {
    if (b16)
      a = __ldcs(static_cast<const unsigned short *>(p) + i);
    else
      a = __ldcs(static_cast<const unsigned int *>(p) + i);
  }
  __device__ __forceinline__ void get(float (&v)[1], bool b16) const { v[0] = __uint_as_float(b16 ? a << 16 : a); }
};

template <int VEC>
__device__ __forceinline__ void put(void *p, int64_t i, const float (&v)[VEC], bool b16);
template <>
__device__ __forceinline__ void put<8>(void *p, int64_t i, const float (&v)[8], bool b16) {
  if (b16) {
    uint4 r;
    __nv_bfloat162 *e = reinterpret_cast<__nv_bfloat162 *>(&r);
#pragma unroll
    for (int k = 0; k < 4; ++k) e[k] = __floats2bfloat162_rn(v[2 * k], v[2 * k + 1]);
    *reinterpret_cast<uint4 *>(static_cast<__nv_bfloat16 *>(p) + i) = r;
  } else {
    float4 *q = reinterpret_cast<float4 *>(static_cast<float *>(p) + i);
    q[0] = make_float4(v[0], v[1], v[2], v[3]);
    q[1] = make_float4(v[4], v[5], v[6], v[7]);
  }
}
template <>
__device__ __forceinline__ void put<2>(void *p, int64_t i, const float (&v)[2], bool b16) {
  if (b16)
    *reinterpret_cast<__nv_bfloat162 *>(static_cast<__nv_bfloat16 *>(p) + i) = __floats2bfloat162_rn(v[0], v[1]);
  else
    *reinterpret_cast<float2 *>(static_cast<float *>(p) + i) = make_float2(v[0], v[1]);
}
template <>
__device__ __forceinline__ void put<1>(void *p, int64_t i, const float (&v)[1], bool b16) {
  if (b16)
    static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16(v[0]);
  else
    static_cast<float *>(p)[i] = v[0];
}

template <int VEC>
__device__ __forceinline__ void weights(const float *w, int col, float (&v)[VEC]) {
  if constexpr (VEC == 8) {
    const float4 a = __ldg(reinterpret_cast<const float4 *>(w + col)),
                 b = __ldg(reinterpret_cast<const float4 *>(w + col) + 1);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else if constexpr (VEC == 2) {
    const float2 a = __ldg(reinterpret_cast<const float2 *>(w + col));
    v[0] = a.x, v[1] = a.y;
  } else {
    v[0] = __ldg(w + col);
  }
}

// Arithmetic on VEC values: eight go two to an instruction (fma.rn.f32x2), which
// halves what the kernels, bound by issue before it, spend on sums and products.
__device__ __forceinline__ void mul_pair(float &ox, float &oy, float ax, float ay, float bx, float by) {
  asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmul.rn.f32x2 a, a, b;\n\t"
      "mov.b64 {%0, %1}, a;\n\t}"
      : "=f"(ox), "=f"(oy)
      : "f"(ax), "f"(ay), "f"(bx), "f"(by));
}
__device__ __forceinline__ void fma_pair(float &ox, float &oy, float ax, float ay, float bx, float by, float cx,
                                         float cy) {
  asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 a, a, b, c;\n\tmov.b64 {%0, %1}, a;\n\t}"
      : "=f"(ox), "=f"(oy)
      : "f"(ax), "f"(ay), "f"(bx), "f"(by), "f"(cx), "f"(cy));
}
// o = a b
template <int VEC>
__device__ __forceinline__ void mul(float (&o)[VEC], const float (&a)[VEC], const float (&b)[VEC]) {
  if constexpr (VEC == 1) {
    o[0] = a[0] * b[0];
  } else {
#pragma unroll
    for (int i = 0; i < VEC; i += 2) mul_pair(o[i], o[i + 1], a[i], a[i + 1], b[i], b[i + 1]);
  }
}
// o = a s
template <int VEC>
__device__ __forceinline__ void mul(float (&o)[VEC], const float (&a)[VEC], float s) {
  if constexpr (VEC == 1) {
    o[0] = a[0] * s;
  } else {
#pragma unroll
    for (int i = 0; i < VEC; i += 2) mul_pair(o[i], o[i + 1], a[i], a[i + 1], s, s);
  }
}
// o = a b + c
template <int VEC>
__device__ __forceinline__ void fma(float (&o)[VEC], const float (&a)[VEC], const float (&b)[VEC],
                                    const float (&c)[VEC]) {
  if constexpr (VEC == 1) {
    o[0] = fmaf(a[0], b[0], c[0]);
  } else {
#pragma unroll
    for (int i = 0; i < VEC; i += 2) fma_pair(o[i], o[i + 1], a[i], a[i + 1], b[i], b[i + 1], c[i], c[i + 1]);
  }
}
// o = a s + c
template <int VEC>
__device__ __forceinline__ void fma(float (&o)[VEC], const float (&a)[VEC], float s, const float (&c)[VEC]) {
  if constexpr (VEC == 1) {
    o[0] = fmaf(a[0], s, c[0]);
  } else {
#pragma unroll
    for (int i = 0; i < VEC; i += 2) fma_pair(o[i], o[i + 1], a[i], a[i + 1], s, s, c[i], c[i + 1]);
  }
}
template <int VEC>
__device__ __forceinline__ void fill(float (&o)[VEC], float s) {
#pragma unroll
  for (int i = 0; i < VEC; ++i) o[i] = s;
}
// A running sum of products, in two halves.
struct Dot {
  float x = 0.f, y = 0.f;
  template <int VEC>
  __device__ __forceinline__ void add(const float (&a)[VEC], const float (&b)[VEC]) {
    if constexpr (VEC == 1) {
      x = fmaf(a[0], b[0], x);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; i += 2) fma_pair(x, y, a[i], a[i + 1], b[i], b[i + 1], x, y);
    }
  }
  __device__ __forceinline__ float sum() const { return x + y; }
};

// The sigmoid with the hardware's exponential and reciprocal: 2^-21 of itself
// off (4 times that at |g| = 16), against 2^-9 of a bf16 result; with expf and
// an IEEE division the forward spent half its instructions here.
__device__ __forceinline__ float sigmoid(float g) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(g * -1.4426950408889634f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
  return r;
}
// sw = swish(g), sg = sigmoid(g), o = o sw
template <int VEC>
__device__ __forceinline__ void gate_by(float (&o)[VEC], const float (&g)[VEC], float (&sw)[VEC], float (&sg)[VEC]) {
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    sg[i] = sigmoid(g[i]);
    sw[i] = fmaxf(g[i], -3.0e38f);  // at -inf (where sg is 0) swish has the limit 0
  }
  mul(sw, sw, sg);
  mul(o, o, sw);
}
// o = o swish'(g) = o (sg + sw - sw sg)
template <int VEC>
__device__ __forceinline__ void slope_by(float (&o)[VEC], const float (&sw)[VEC], const float (&sg)[VEC]) {
  float v[VEC];
  const float one = 1.f;
  mul(v, sw, -one);
  fma(v, v, sg, sg);
  fma(v, sw, one, v);
  mul(o, o, v);
}

constexpr int kRed = 2 * 3 * 32;
// Sums of n values over the row's threads: a warp (one_warp) or the block.
// `red` holds 2 x 3 x 32 floats, those of absent warps 0; `flip` alternates its
// halves, so one barrier per sum is enough.
template <int NV>
__device__ __forceinline__ void row_sum(float (&v)[NV], bool one_warp, float *red, int &flip) {
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (one_warp || NV != 3) v[i] = warp_sum(v[i]);
  if (one_warp) return;
  float *r = red + flip * 96;
  flip ^= 1;
  if constexpr (NV == 3) {  // the lanes share the three sums: half the shuffles, an eighth of the reads
    const int lane = threadIdx.x & 31;
    float a = __shfl_xor_sync(0xffffffffu, lane & 16 ? v[0] : v[1], 16) + (lane & 16 ? v[1] : v[0]);
    const float b = v[2] + __shfl_xor_sync(0xffffffffu, v[2], 16);
    a = __shfl_xor_sync(0xffffffffu, lane & 8 ? a : b, 8) + (lane & 8 ? b : a);
#pragma unroll
    for (int o = 4; o; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
    // lanes 0 .. 7 have the first sum, 16 .. 23 the second, the rest the third
    const int which = lane & 8 ? 2 : lane >> 4;
    if ((lane & 7) == 0 && lane < 24) r[which * 32 + (threadIdx.x >> 5)] = a;
    __syncthreads();
    const float *q = r + which * 32 + (lane & 7);
    a = q[0];
    if ((int)blockDim.x > 256) a += q[8];  // 16 warps at most
#pragma unroll
    for (int o = 4; o; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
    v[0] = __shfl_sync(0xffffffffu, a, 0), v[1] = __shfl_sync(0xffffffffu, a, 16), v[2] = __shfl_sync(0xffffffffu, a, 8);
    return;
  }
  if ((threadIdx.x & 31) == 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i) r[i * 32 + (threadIdx.x >> 5)] = v[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const float4 *q = reinterpret_cast<const float4 *>(r + i * 32);
    float4 a = q[0], b = q[1];
#pragma unroll
    for (int k = 2; k < 8; k += 2)
      if ((int)blockDim.x > 128 * k) {  // more than 4 k warps
        const float4 c = q[k], d = q[k + 1];
        a.x += c.x, a.y += c.y, a.z += c.z, a.w += c.w;
        b.x += d.x, b.y += d.y, b.z += d.z, b.w += d.w;
      }
    v[i] = ((a.x + b.x) + (a.y + b.y)) + ((a.z + b.z) + (a.w + b.w));
  }
}
__device__ __forceinline__ void clear_red(float *red) {
  const int t = threadIdx.y * blockDim.x + threadIdx.x;
  for (int i = t; i < kRed; i += blockDim.x * blockDim.y) red[i] = 0.f;
  __syncthreads();
}

// post_w scale (what is not given counts as 1) of VEC columns.
template <int VEC>
__device__ __forceinline__ void both_weights(const SeamParams &p, int col, float (&v)[VEC]) {
  fill(v, 1.f);
  if (p.w1) weights<VEC>(p.w1, col, v);
  if (p.s) {
    float s[VEC];
    weights<VEC>(p.s, col, s);
    mul(v, v, s);
  }
}

// Those and pre_w of all of a thread's columns.
template <int VEC, int K>
__device__ __forceinline__ void keep_weights(const SeamParams &p, int n, float (&w1)[K][VEC], float (&w2)[K][VEC]) {
#pragma unroll
  for (int c = 0; c < K; ++c) {
    const int col = (c * n + (int)threadIdx.x) * VEC;
    fill(w1[c], 0.f), fill(w2[c], 0.f);
    if (col < p.d) {
      both_weights<VEC>(p, col, w1[c]);
      if (p.w2) weights<VEC>(p.w2, col, w2[c]);
    }
  }
}

// Threads of a row: a warp (blockDim.y rows per block) or the whole block
// (blockDim.y == 1).  Thread k of a row holds values (c * n + k) * VEC ..,
// c < K, n the row's threads.  Where those are few, the weights stay in
// registers while a block walks over rows, and a row's loads are under way
// while the row before it is summed.
template <int VEC, int K, int TX, int TH>
__global__ void __launch_bounds__(VEC == 8 && K == 1 ? 1024 : 512, VEC == 8 ? 1 : 2) seam_forward_kernel(SeamParams p) {
  constexpr bool kAhead = VEC * K <= 8 && K <= 4;
  __shared__ __align__(16) float red[kRed];
  int flip = 0;
  clear_red(red);
  const int n = blockDim.x;
  const bool one_warp = n == 32, x16 = TX == 1, h16 = TH == 1;
  const int step = gridDim.x * blockDim.y;
  Raw<VEC> hr[K], gr[K], xr[K];
  auto fetch = [&](int row) {
#pragma unroll
    for (int c = 0; c < K; ++c) {
      const int col = (c * n + (int)threadIdx.x) * VEC;
      if (col < p.d) {
        hr[c].load(p.h, row * p.ldh + col, h16);
        if (p.g) gr[c].load(p.g, row * p.ldg + col, h16);
        xr[c].load(p.x, row * p.ldx + col, x16);
      }
    }
  };
  float kept1[K][VEC], kept2[K][VEC];  // with kAhead: post_w scale, pre_w
  if (kAhead) keep_weights<VEC, K>(p, n, kept1, kept2);
  int row = blockIdx.x * blockDim.y + threadIdx.y;
  if (kAhead && row < p.rows) fetch(row);
  for (; row < p.rows; row += step) {  // a block's threads leave together where they share a row
    if (!kAhead) fetch(row);
    float z[K][VEC], x[K][VEC];
    Dot dot;
#pragma unroll
    for (int c = 0; c < K; ++c) {
      const int col = (c * n + (int)threadIdx.x) * VEC;
      if (col < p.d) {
        hr[c].get(z[c], h16);
        dot.add(z[c], z[c]);
        // all of n but r1
        if (p.g) {
          float v[VEC], sw[VEC], sg[VEC];
          gr[c].get(v, h16);
          gate_by(z[c], v, sw, sg);
        }
        if (kAhead) {
          mul(z[c], z[c], kept1[c]);
        } else {
          float v[VEC];
          both_weights<VEC>(p, col, v);
          mul(z[c], z[c], v);
        }
        xr[c].get(x[c], x16);
        mul(x[c], x[c], p.alpha);
      }
    }
    if (kAhead && row + step < p.rows) fetch(row + step);
    float r1 = 1.f;
    if (p.w1) {
      float sq[1] = {dot.sum()};
      row_sum(sq, one_warp, red, flip);
      r1 = rsqrtf(fmaf(sq[0], p.inv_d, p.eps));
    }
    Dot dz;
#pragma unroll
    for (int c = 0; c < K; ++c) {
      const int col = (c * n + (int)threadIdx.x) * VEC;
      if (col < p.d) {
        fma(z[c], z[c], r1, x[c]);
        dz.add(z[c], z[c]);
        put<VEC>(p.z, (int64_t)row * p.d + col, z[c], x16);
      }
    }
    float r2 = 1.f;
    if (p.w2) {
      float sz[1] = {dz.sum()};
      row_sum(sz, one_warp, red, flip);
      r2 = rsqrtf(fmaf(sz[0], p.inv_d, p.eps));
#pragma unroll
      for (int c = 0; c < K; ++c) {
        const int col = (c * n + (int)threadIdx.x) * VEC;
        if (col < p.d) {
          mul(z[c], z[c], r2);
          if (kAhead) {
            mul(z[c], z[c], kept2[c]);
          } else {
            float v[VEC];
            weights<VEC>(p.w2, col, v);
            mul(z[c], z[c], v);
          }
          put<VEC>(p.y, (int64_t)row * p.d + col, z[c], p.y16);
        }
      }
    }
    if (p.stats && threadIdx.x == 0) {
      p.stats[row] = r1;
      p.stats[p.rows + row] = r2;
    }
  }
}

template <int VEC, int K, int TX, int TH, bool one_warp>
__global__ void __launch_bounds__(512, 1) seam_backward_kernel(SeamParams p) {
  constexpr bool kAhead = VEC * K <= 8 && K <= 4;
  __shared__ __align__(16) float red[kRed];
  int flip = 0;
  clear_red(red);
  const int n = blockDim.x;
  const bool x16 = TX == 1, h16 = TH == 1;
  float a1[K][VEC], a2[K][VEC];  // this thread's columns of sum Z swish hh and of dw2
#pragma unroll
  for (int c = 0; c < K; ++c) fill(a1[c], 0.f), fill(a2[c], 0.f);
  float kept1[K][VEC], kept2[K][VEC];  // with kAhead: post_w scale, pre_w
  if (kAhead) keep_weights<VEC, K>(p, n, kept1, kept2);
  Raw<VEC> hr[K], gr[K], xr[K], dzr[K], dyr[K];
  auto fetch = [&](int row) {
#pragma unroll
    for (int c = 0; c < K; ++c) {
      const int col = (c * n + (int)threadIdx.x) * VEC;
      if (col < p.d) {
        hr[c].load(p.h, row * p.ldh + col, h16);
        if (p.g) gr[c].load(p.g, row * p.ldg + col, h16);
        if (p.dz) dzr[c].load(p.dz, row * p.lddz + col, x16);
        if (p.dy) {
          dyr[c].load(p.dy, row * p.lddy + col, p.y16);
          xr[c].load(p.x, row * p.ldx + col, x16);
        }
      }
    }
  };
  // also this row group's place among all; one for the whole block keeps a row's address in uniform registers
  const int part = one_warp ? blockIdx.x * blockDim.y + threadIdx.y : blockIdx.x;
  if (kAhead && part < p.rows) fetch(part);
  for (int row = part; row < p.rows; row += p.parts) {
    if (!kAhead) fetch(row);
    const float r1 = p.w1 ? p.stats[row] : 1.f, r2 = p.w2 ? p.stats[p.rows + row] : 1.f;
    Dot tz, eq, zq;  // t zh, e q, zh q
    // hh (h without post_w), the gate and its sigmoid, zh, e = dz + r2 t; q is what z has of n
    float hh[K][VEC], sw[K][VEC], sg[K][VEC], zh[K][VEC], e[K][VEC];
#pragma unroll
    for (int c = 0; c < K; ++c) {
      const int col = (c * n + (int)threadIdx.x) * VEC;
      if (col < p.d) {
        float q[VEC], v[VEC], w[VEC];
        hr[c].get(hh[c], h16);
        mul(hh[c], hh[c], r1);
        if (kAhead) {
          mul(q, hh[c], kept1[c]);
        } else {
          both_weights<VEC>(p, col, w);
          mul(q, hh[c], w);
        }
        if (p.g) {
          gr[c].get(v, h16);
          gate_by(q, v, sw[c], sg[c]);
        }
        if (p.dz)
          dzr[c].get(e[c], x16);
        else
          fill(e[c], 0.f);
        if (p.dy) {
          float dy[VEC];
          xr[c].get(v, x16);
          dyr[c].get(dy, p.y16);
          fma(zh[c], v, p.alpha, q);
          mul(zh[c], zh[c], r2);
          fma(a2[c], dy, zh[c], a2[c]);
          if (kAhead) {
            mul(dy, dy, kept2[c]);  // t
          } else {
            weights<VEC>(p.w2, col, w);
            mul(dy, dy, w);
          }
          tz.add(dy, zh[c]);
          fma(e[c], dy, r2, e[c]);
          zq.add(zh[c], q);
        }
        eq.add(e[c], q);
      }
    }
    if (kAhead && row + p.parts < p.rows) fetch(row + p.parts);
    float sum[3] = {tz.sum(), eq.sum(), zq.sum()};
    if (p.w1 || p.dy) row_sum(sum, one_warp, red, flip);
    const float m2 = p.dy ? r2 * (sum[0] * p.inv_d) : 0.f;  // r2 mean(t zh)
    const float m1 = (sum[1] - m2 * sum[2]) * p.inv_d;       // mean(N w1 hh)
#pragma unroll
    for (int c = 0; c < K; ++c) {
      const int col = (c * n + (int)threadIdx.x) * VEC;
      if (col < p.d) {
        const int64_t at = (int64_t)row * p.d + col;
        float o[VEC], v[VEC], w[VEC];
        if (p.dy) fma(e[c], zh[c], -m2, e[c]);  // Z
        mul(o, e[c], p.alpha);
        put<VEC>(p.dx, at, o, x16);
        if (!kAhead) both_weights<VEC>(p, col, w);
        mul(o, e[c], hh[c]);
        if (kAhead)
          mul(v, e[c], kept1[c]);
        else
          mul(v, e[c], w);
        if (p.g) {
          fma(a1[c], o, sw[c], a1[c]);
          mul(o, v, hh[c]);
          slope_by(o, sw[c], sg[c]);
          put<VEC>(p.dg, at, o, h16);
          mul(v, v, sw[c]);
        } else {
#pragma unroll
          for (int i = 0; i < VEC; ++i) a1[c][i] += o[i];
        }
        if (p.w1) {  // v = N w1
          fma(v, hh[c], -m1, v);
          mul(v, v, r1);
        }
        put<VEC>(p.dh, at, v, h16);
      }
    }
  }
  const int64_t plane = (int64_t)p.parts * p.d;
#pragma unroll
  for (int c = 0; c < K; ++c) {
    const int col = (c * n + (int)threadIdx.x) * VEC;
    if (col < p.d) {
      const int64_t at = (int64_t)part * p.d + col;
      if (p.w1 || p.s) put<VEC>(p.part, at, a1[c], false);
      if (p.w2) put<VEC>(p.part, plane + at, a2[c], false);
    }
  }
}

// The same for wide rows, in two passes that each form a row's values anew: what
// a thread has of a row as it lies in memory,
template <int VEC>
struct RawRow {
  Raw<VEC> h, g, x, dz, dy;
  __device__ __forceinline__ void load(const SeamParams &p, int row, int col, bool x16, bool h16) {
    h.load(p.h, row * p.ldh + col, h16);
    if (p.g) g.load(p.g, row * p.ldg + col, h16);
    if (p.dz) dz.load(p.dz, row * p.lddz + col, x16);
    if (p.dy) {
      dy.load(p.dy, row * p.lddy + col, p.y16);
      x.load(p.x, row * p.ldx + col, x16);
    }
  }
};
// and the values that follow from it (w: post_w scale; t = dy pre_w; e = dz + r2 t).
template <int VEC>
struct SeamValues {
  float hh[VEC], sw[VEC], sg[VEC], w[VEC], q[VEC], zh[VEC], e[VEC], dy[VEC], t[VEC];
  __device__ __forceinline__ void form(const SeamParams &p, const RawRow<VEC> &r, int col, float r1, float r2, bool x16,
                                       bool h16) {
    both_weights<VEC>(p, col, w);
    r.h.get(hh, h16);
    mul(hh, hh, r1);
    mul(q, hh, w);
    if (p.g) {
      float g[VEC];
      r.g.get(g, h16);
      gate_by(q, g, sw, sg);
    }
    fill(e, 0.f), fill(zh, 0.f), fill(t, 0.f), fill(dy, 0.f);
    if (p.dz) r.dz.get(e, x16);
    if (p.dy) {
      float v[VEC];
      r.x.get(v, x16);
      r.dy.get(dy, p.y16);
      fma(zh, v, p.alpha, q);
      mul(zh, zh, r2);
      weights<VEC>(p.w2, col, v);
      mul(t, dy, v);
      fma(e, t, r2, e);
    }
  }
  // The gradients; o1 and o2: what they add to the columns' sums.
  __device__ __forceinline__ void write(const SeamParams &p, int64_t at, float r1, float m1, float m2, bool x16, bool h16,
                                        float (&o1)[VEC], float (&o2)[VEC]) {
    float v[VEC];
    fma(e, zh, -m2, e);  // Z
    mul(v, e, p.alpha);
    put<VEC>(p.dx, at, v, x16);
    mul(o1, e, hh);
    mul(o2, dy, zh);
    mul(v, e, w);
    if (p.g) {
      float o[VEC];
      mul(o1, o1, sw);
      mul(o, v, hh);
      slope_by(o, sw, sg);
      put<VEC>(p.dg, at, o, h16);
      mul(v, v, sw);
    }
    if (p.w1) {
      fma(v, hh, -m1, v);
      mul(v, v, r1);
    }
    put<VEC>(p.dh, at, v, h16);
  }
};

__device__ __forceinline__ void ahead(const void *p, int64_t i, bool b16) {
  asm volatile("prefetch.global.L2 [%0];" ::"l"(static_cast<const char *>(p) + i * (b16 ? 2 : 4)));
}

// Rows of up to K 512 VEC values: the row as it lies in memory and the columns'
// sums stay in registers, the block's next row is on its way into L2.
template <int VEC, int K, int TX, int TH>
__global__ void __launch_bounds__(512, 1) seam_backward_held_kernel(SeamParams p) {
  __shared__ __align__(16) float red[kRed];
  int flip = 0;
  clear_red(red);
  const int n = blockDim.x;
  const bool x16 = TX == 1, h16 = TH == 1;
  float a1[K][VEC], a2[K][VEC];
#pragma unroll
  for (int c = 0; c < K; ++c) fill(a1[c], 0.f), fill(a2[c], 0.f);
  for (int row = blockIdx.x; row < p.rows; row += p.parts) {
    RawRow<VEC> raw[K];
#pragma unroll
    for (int c = 0; c < K; ++c) {
      const int col = (c * n + (int)threadIdx.x) * VEC;
      if (col < p.d) raw[c].load(p, row, col, x16, h16);
    }
    const int next = row + p.parts;
    if (next < p.rows && threadIdx.x % 4 == 0) {
#pragma unroll
      for (int c = 0; c < K; ++c) {
        const int col = (c * n + (int)threadIdx.x) * VEC;
        if (col < p.d) {
          ahead(p.h, next * p.ldh + col, h16);
          if (p.g) ahead(p.g, next * p.ldg + col, h16);
          if (p.dz) ahead(p.dz, next * p.lddz + col, x16);
          if (p.dy) ahead(p.dy, next * p.lddy + col, p.y16), ahead(p.x, next * p.ldx + col, x16);
        }
      }
    }
    const float r1 = p.w1 ? p.stats[row] : 1.f, r2 = p.w2 ? p.stats[p.rows + row] : 1.f;
    Dot tz, eq, zq;
#pragma unroll
    for (int c = 0; c < K; ++c) {
      const int col = (c * n + (int)threadIdx.x) * VEC;
      if (col < p.d) {
        SeamValues<VEC> s;
        s.form(p, raw[c], col, r1, r2, x16, h16);
        tz.add(s.t, s.zh);
        eq.add(s.e, s.q);
        zq.add(s.zh, s.q);
      }
    }
    float sum[3] = {tz.sum(), eq.sum(), zq.sum()};
    row_sum(sum, false, red, flip);
    const float m2 = r2 * (sum[0] * p.inv_d), m1 = (sum[1] - m2 * sum[2]) * p.inv_d;
#pragma unroll
    for (int c = 0; c < K; ++c) {
      const int col = (c * n + (int)threadIdx.x) * VEC;
      if (col < p.d) {
        SeamValues<VEC> s;
        float o1[VEC], o2[VEC];
        s.form(p, raw[c], col, r1, r2, x16, h16);
        s.write(p, (int64_t)row * p.d + col, r1, m1, m2, x16, h16, o1, o2);
#pragma unroll
        for (int i = 0; i < VEC; ++i) a1[c][i] += o1[i], a2[c][i] += o2[i];
      }
    }
  }
  const int64_t plane = (int64_t)p.parts * p.d;
#pragma unroll
  for (int c = 0; c < K; ++c) {
    const int col = (c * n + (int)threadIdx.x) * VEC;
    if (col < p.d) {
      const int64_t at = (int64_t)blockIdx.x * p.d + col;
      if (p.w1 || p.s) put<VEC>(p.part, at, a1[c], false);
      if (p.w2) put<VEC>(p.part, plane + at, a2[c], false);
    }
  }
}

// Wider ones: the second pass reads the row from the caches, the column sums
// lie in shared memory, [2][d], where every thread alone touches its columns.
template <int VEC, int TX, int TH>
__global__ void __launch_bounds__(512, 1) seam_backward_wide_kernel(SeamParams p) {
  extern __shared__ __align__(16) float acc[];
  __shared__ __align__(16) float red[kRed];
  int flip = 0;
  clear_red(red);
  const int n = blockDim.x;
  const bool x16 = TX == 1, h16 = TH == 1;
  float *a1 = acc, *a2 = acc + p.d;
  for (int col = threadIdx.x * VEC; col < p.d; col += n * VEC)
#pragma unroll
    for (int i = 0; i < VEC; ++i) a1[col + i] = a2[col + i] = 0.f;
  for (int row = blockIdx.x; row < p.rows; row += p.parts) {
    const float r1 = p.w1 ? p.stats[row] : 1.f, r2 = p.w2 ? p.stats[p.rows + row] : 1.f;
    Dot tz, eq, zq;
    for (int col = threadIdx.x * VEC; col < p.d; col += n * VEC) {
      RawRow<VEC> raw;
      SeamValues<VEC> s;
      raw.load(p, row, col, x16, h16);
      s.form(p, raw, col, r1, r2, x16, h16);
      tz.add(s.t, s.zh);
      eq.add(s.e, s.q);
      zq.add(s.zh, s.q);
    }
    float sum[3] = {tz.sum(), eq.sum(), zq.sum()};
    row_sum(sum, false, red, flip);
    const float m2 = r2 * (sum[0] * p.inv_d), m1 = (sum[1] - m2 * sum[2]) * p.inv_d;
    for (int col = threadIdx.x * VEC; col < p.d; col += n * VEC) {
      RawRow<VEC> raw;
      SeamValues<VEC> s;
      float o1[VEC], o2[VEC];
      raw.load(p, row, col, x16, h16);
      s.form(p, raw, col, r1, r2, x16, h16);
      s.write(p, (int64_t)row * p.d + col, r1, m1, m2, x16, h16, o1, o2);
#pragma unroll
      for (int i = 0; i < VEC; ++i) a1[col + i] += o1[i], a2[col + i] += o2[i];
    }
  }
  const int64_t plane = (int64_t)p.parts * p.d;
  for (int col = threadIdx.x * VEC; col < p.d; col += n * VEC) {
    const int64_t at = (int64_t)blockIdx.x * p.d + col;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      if (p.w1 || p.s) p.part[at + i] = a1[col + i];
      if (p.w2) p.part[plane + at + i] = a2[col + i];
    }
  }
}

// Column sums of the [parts][d] planes (blockIdx.y: which): 16 warps share a
// block of 32 columns, each adds every sixteenth part in order.  The first
// plane's sum times scale is dw1, times post_w it is ds.
__global__ void __launch_bounds__(512) seam_columns_kernel(const float *part, int parts, int d, const float *w1,
                                                           const float *s, float *dw1, float *ds, float *dw2) {
  __shared__ float red[16][32];
  if (blockIdx.y ? !dw2 : !(dw1 || ds)) return;
  const int col = blockIdx.x * 32 + threadIdx.x;
  const float *src = part + (int64_t)blockIdx.y * parts * d + col;
  float t = 0.f;
  if (col < d) {
#pragma unroll 4
    for (int k = threadIdx.y; k < parts; k += 16) t += src[(int64_t)k * d];
  }
  red[threadIdx.y][threadIdx.x] = t;
  __syncthreads();
  if (threadIdx.y == 0 && col < d) {
    for (int k = 1; k < 16; ++k) t += red[k][threadIdx.x];
    if (blockIdx.y) {
      dw2[col] = t;
    } else {
      if (dw1) dw1[col] = s ? t * s[col] : t;
      if (ds) ds[col] = w1 ? t * w1[col] : t;
    }
  }
}

constexpr int kMaxWidth = 16384;

// Threads of a row and values per thread for rows of d values.  A block's
// registers allow 512 threads (1024 in the vectorised forward); while they
// suffice, few values a thread, so that much is under way.
struct Shape {
  int vec, k, threads, rows_per_block;
};
Shape shape_of(int d, int vec, bool backward) {
  auto threads = [&](int per) { return (d + per * 32 - 1) / (per * 32) * 32; };  // whole warps that hold d values
  if (vec == 8) {
    if (d <= 256) return {8, 1, 32, 4};
    if (d <= (backward ? 4096 : 8192)) return {8, 1, threads(8), 1};
    if (backward && d <= 8192) return {8, 2, threads(16), 1};
    return {8, backward ? 0 : 4, 512, 1};
  }
  if (d <= 128) return {1, 4, 32, 4};
  if (vec == 2) {
    if (d <= 2048) return {2, 2, threads(4), 1};
    if (d <= 4096) return {2, 4, threads(8), 1};
    return backward ? Shape{2, 0, 512, 1} : Shape{2, 16, 512, 1};
  }
  if (d <= 2048) return {1, 4, threads(4), 1};
  if (d <= 4096) return {1, 8, threads(8), 1};
  if (backward) return {1, 0, 512, 1};
  return d <= 8192 ? Shape{1, 16, 512, 1} : Shape{1, 32, 512, 1};
}
bool walks(const Shape &s) { return s.vec * s.k <= 8 && s.k > 0 && s.k <= 4; }  // the kernels' kAhead

// The kernel of a shape (k 0: the two-pass backward).
using SeamKernel = void (*)(SeamParams);
template <int TX, int TH>
SeamKernel typed_kernel(const Shape &s, bool backward) {
  if (backward) {
    const bool warp = s.rows_per_block > 1;
    if (s.vec == 8)
      return s.k == 1   ? (warp ? seam_backward_kernel<8, 1, TX, TH, true> : seam_backward_kernel<8, 1, TX, TH, false>)
             : s.k == 2 ? seam_backward_held_kernel<8, 2, TX, TH>
                        : seam_backward_wide_kernel<8, TX, TH>;
    if (s.vec == 2)
      return s.k == 2   ? seam_backward_kernel<2, 2, TX, TH, false>
             : s.k == 4 ? seam_backward_kernel<2, 4, TX, TH, false>
                        : seam_backward_wide_kernel<2, TX, TH>;
    return s.k == 4   ? (warp ? seam_backward_kernel<1, 4, TX, TH, true> : seam_backward_kernel<1, 4, TX, TH, false>)
           : s.k == 8 ? seam_backward_kernel<1, 8, TX, TH, false>
                      : seam_backward_wide_kernel<1, TX, TH>;
  }
  if (s.vec == 8) return s.k == 1 ? seam_forward_kernel<8, 1, TX, TH> : seam_forward_kernel<8, 4, TX, TH>;
  if (s.vec == 2)
    return s.k == 2   ? seam_forward_kernel<2, 2, TX, TH>
           : s.k == 4 ? seam_forward_kernel<2, 4, TX, TH>
                      : seam_forward_kernel<2, 16, TX, TH>;
  return s.k == 4    ? seam_forward_kernel<1, 4, TX, TH>
         : s.k == 8  ? seam_forward_kernel<1, 8, TX, TH>
         : s.k == 16 ? seam_forward_kernel<1, 16, TX, TH>
                     : seam_forward_kernel<1, 32, TX, TH>;
}
SeamKernel kernel_of(const Shape &s, bool x16, bool h16, bool backward) {
  if (x16) return h16 ? typed_kernel<1, 1>(s, backward) : typed_kernel<1, 0>(s, backward);
  return h16 ? typed_kernel<0, 1>(s, backward) : typed_kernel<0, 0>(s, backward);
}

// Values an access may take where rows lie at p, ld elements apart: 8 need 16
// bytes (of fp32 rows, which are then aligned too, every half), 2 the pair's size.
int access_of(const void *p, int64_t ld, int is16) {
  if (!p) return 8;
  const uintptr_t a = reinterpret_cast<uintptr_t>(p);
  if (a % 16 == 0 && ld % (is16 ? 8 : 4) == 0) return 8;
  return a % (is16 ? 4 : 8) == 0 && ld % 2 == 0 ? 2 : 1;
}
int least_access(int d, std::initializer_list<int> all) {
  const int v = std::min(all);
  return d % v == 0 ? v : d % 2 == 0 && v >= 2 ? 2 : 1;
}

// Row groups that share the rows of a backward: about 512 threads an SM, as
// many as its registers hold; few enough that their partial rows stay small
// beside the data.
int parts_of(int num_sms, int rows, const Shape &s) {
  const int per_sm = 512 / (s.threads * s.rows_per_block), blocks = num_sms * (per_sm < 1 ? 1 : per_sm);
  const int need = (rows + s.rows_per_block - 1) / s.rows_per_block;
  return (need < blocks ? need : blocks) * s.rows_per_block;
}

}  // namespace

extern "C" {

int af_residual_norm(af_ctx *ctx, const void *x, int64_t ldx, int x_bf16, const void *h, int64_t ldh, int h_bf16,
                     const void *gate, int64_t ldg, const float *post_w, const float *scale, const float *pre_w,
                     float alpha, float eps, int64_t rows, int d, void *z, void *y, int y_bf16, float *stats,
                     af_stream_t stream) {
  const char *fn = "af_residual_norm";
  af::DeviceScope scope;
  AF_ENTER(ctx, fn);
  AF_REQUIRE(rows >= 0 && rows < (1ll << 31) && d > 0, "af_residual_norm", "bad sizes");
  AF_REQUIRE(d <= kMaxWidth, "af_residual_norm", "rows of %d values: at most %d are supported", d, kMaxWidth);
  if (rows == 0) return AF_OK;
  AF_REQUIRE(x && h && z && (!pre_w || y), "af_residual_norm", "null argument");
  SeamParams p = {};
  p.x = x, p.h = h, p.g = gate, p.ldx = ldx, p.ldh = ldh, p.ldg = ldg;
  p.x16 = x_bf16 != 0, p.h16 = h_bf16 != 0, p.y16 = y_bf16 != 0;
  p.w1 = post_w, p.s = scale, p.w2 = pre_w, p.alpha = alpha, p.eps = eps, p.inv_d = 1.0f / (float)d;
  p.rows = (int)rows, p.d = d, p.z = z, p.y = y, p.stats = stats;
  const int vec = least_access(
      d, {access_of(x, ldx, x_bf16), access_of(h, ldh, h_bf16), access_of(gate, ldg, h_bf16), access_of(post_w, 8, 0),
          access_of(scale, 8, 0), access_of(pre_w, 8, 0), access_of(z, d, x_bf16), access_of(y, d, y_bf16)});
  const Shape s = shape_of(d, vec, false);
  int64_t blocks = (rows + s.rows_per_block - 1) / s.rows_per_block;
  if (walks(s)) {  // blocks that walk: 1024 threads an SM, what its registers hold
    const int per_sm = 1024 / (s.threads * s.rows_per_block);
    blocks = std::min<int64_t>(blocks, (int64_t)ctx->num_sms * (per_sm < 1 ? 1 : per_sm));
  }
  kernel_of(s, p.x16, p.h16, false)<<<(unsigned)blocks, dim3(s.threads, s.rows_per_block), 0,
                                      af::stream_of(stream)>>>(p);
  return af::launched(ctx, fn);
}

int af_residual_norm_scratch(af_ctx *ctx, int64_t rows, int d, int64_t *floats) {
  const char *fn = "af_residual_norm_scratch";
  af::DeviceScope scope;
  AF_ENTER(ctx, fn);
  AF_REQUIRE(floats && rows >= 0 && rows < (1ll << 31) && d > 0 && d <= kMaxWidth, "af_residual_norm_scratch",
             "bad sizes");
  int most = 0;  // whatever accesses the call's tensors will allow
  for (int vec : {1, 2, 8})
    if (d % vec == 0) most = std::max(most, parts_of(ctx->num_sms, (int)rows, shape_of(d, vec, true)));
  *floats = 2ll * most * d;
  return AF_OK;
}

int af_residual_norm_backward(af_ctx *ctx, const void *dz, int64_t lddz, const void *dy, int64_t lddy, const void *x,
                              int64_t ldx, int x_bf16, const void *h, int64_t ldh, int h_bf16, const void *gate,
                              int64_t ldg, int y_bf16, const float *post_w, const float *scale, const float *pre_w,
                              float alpha, int64_t rows, int d, const float *stats, void *dx, void *dh, void *dgate,
                              float *dpost_w, float *dscale, float *dpre_w, float *scratch, int64_t scratch_floats,
                              af_stream_t stream) {
  const char *fn = "af_residual_norm_backward";
  af::DeviceScope scope;
  AF_ENTER(ctx, fn);
  AF_REQUIRE(rows >= 0 && rows < (1ll << 31) && d > 0, "af_residual_norm_backward", "bad sizes");
  AF_REQUIRE(d <= kMaxWidth, "af_residual_norm_backward", "rows of %d values: at most %d are supported", d, kMaxWidth);
  AF_REQUIRE(!dy || pre_w, "af_residual_norm_backward", "dy without the norm that made y");
  AF_REQUIRE((!post_w || dpost_w) && (!scale || dscale) && (!pre_w || dpre_w), "af_residual_norm_backward",
             "a weight without room for its gradient");
  cudaStream_t st = af::stream_of(stream);
  if (rows == 0) {
    float *w[3] = {post_w ? dpost_w : nullptr, scale ? dscale : nullptr, pre_w ? dpre_w : nullptr};
    for (float *q : w)
      if (q) AF_CUDA(cudaMemsetAsync(q, 0, (size_t)d * 4, st), fn);
    return AF_OK;
  }
  AF_REQUIRE(x && h && dx && dh && (!gate || dgate) && (!(post_w || pre_w) || stats), "af_residual_norm_backward",
             "null argument");
  SeamParams p = {};
  p.x = x, p.h = h, p.g = gate, p.ldx = ldx, p.ldh = ldh, p.ldg = ldg;
  p.x16 = x_bf16 != 0, p.h16 = h_bf16 != 0, p.y16 = y_bf16 != 0;
  p.w1 = post_w, p.s = scale, p.w2 = pre_w, p.alpha = alpha, p.inv_d = 1.0f / (float)d;
  p.rows = (int)rows, p.d = d, p.stats = const_cast<float *>(stats);
  p.dz = dz, p.dy = dy, p.lddz = lddz, p.lddy = lddy, p.dx = dx, p.dh = dh, p.dg = dgate, p.part = scratch;
  const int vec = least_access(
      d, {access_of(x, ldx, x_bf16), access_of(h, ldh, h_bf16), access_of(gate, ldg, h_bf16), access_of(post_w, 8, 0),
          access_of(scale, 8, 0), access_of(pre_w, 8, 0), access_of(dz, lddz, x_bf16), access_of(dy, lddy, y_bf16),
          access_of(dx, d, x_bf16), access_of(dh, d, h_bf16), access_of(dgate, d, h_bf16), access_of(scratch, 8, 0)});
  const Shape s = shape_of(d, vec, true);
  p.parts = parts_of(ctx->num_sms, (int)rows, s);
  const bool sums = post_w || scale || pre_w;
  AF_REQUIRE(!sums || (scratch && scratch_floats >= 2ll * p.parts * d), "af_residual_norm_backward",
             "scratch of %lld floats, %lld are needed", (long long)scratch_floats, 2ll * p.parts * d);
  const SeamKernel kernel = kernel_of(s, p.x16, p.h16, true);
  size_t smem = 0;
  if (s.k == 0) {
    smem = (size_t)2 * d * sizeof(float);
    static std::atomic<unsigned long long> attr_devices[3][4];
    if (int rc = af::smem_attr(ctx, reinterpret_cast<const void *>(kernel), (size_t)2 * kMaxWidth * sizeof(float),
                               attr_devices[s.vec == 8 ? 2 : s.vec - 1][p.x16 * 2 + p.h16], fn))
      return rc;
  }
  kernel<<<(unsigned)(p.parts / s.rows_per_block), dim3(s.threads, s.rows_per_block), smem, st>>>(p);
  if (int rc = af::launched(ctx, fn)) return rc;
  if (!sums) return AF_OK;
  seam_columns_kernel<<<dim3((unsigned)((d + 31) / 32), 2), dim3(32, 16), 0, st>>>(
      scratch, p.parts, d, post_w, scale, post_w ? dpost_w : nullptr, scale ? dscale : nullptr,
      pre_w ? dpre_w : nullptr);
  return af::launched(ctx, fn);
}

}  // extern "C"
