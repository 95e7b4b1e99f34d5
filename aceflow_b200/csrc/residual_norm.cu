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
// Bound: HBM, every row of every tensor moved once; wide and odd rows by the
// issue of instructions and their latency, at 16 warps an SM.  A row is
// held in registers by one group of threads; sums, statistics and the row itself
// are fp32, and each output is rounded once.  The column sums of the weights'
// gradients stay with the threads while a block walks its rows, go out as one
// partial row per group and are added in a fixed order by a second kernel: no
// atomics, the same bits every run.
// Measured with gate and all weights (floor: the tensors' bytes at 6547 GB/s):
//   32768 x 2048 bf16   forward 110 us (0.93 of it), backward 181 (0.91)
//   16384 x 2048 fp32            118 (0.87),                  190 (0.86)
//    4096 x 8192 bf16             64 (0.80),                  134 (0.61)
//   16384 x 1531 bf16             72 (0.53),                  135 (0.45)
//   16384 x 1531 fp32            115 (0.67),                  220 (0.56)
#include "common.cuh"

#include <algorithm>

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
  float *part;    // planes of [parts][d], `plane` apart: sum Z swish(g) hh, sum dy zh
  int64_t plane;
  int parts;      // row groups: group i has the rows i, i + parts, ..
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

// The sigmoid.  Where x and h are bf16 (`fast`) by the hardware's exponential and
// reciprocal: 2^-21 and |g| 2^-24 of itself off, against the 2^-8 of
// the tensors (y, if asked for in fp32, and the weights' gradients carry it
// too); expf and a division took 32768 x 2048 from 109 and 181 us (forward,
// backward) to 135 and 234.  Where either is fp32, expf and a division all the
// same: 16384 x 2048 fp32 122 and 185 us without, 118 and 190 with, 16384 x 1531 fp32
// 100 and 194, 115 and 220.
__device__ __forceinline__ float sigmoid(float g, bool fast) {
  if (!fast) return 1.0f / (1.0f + expf(-g));
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(g * -1.4426950408889634f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
  return r;
}
// sw = swish(g), sg = sigmoid(g), o = o sw
template <int VEC>
__device__ __forceinline__ void gate_by(float (&o)[VEC], const float (&g)[VEC], float (&sw)[VEC], float (&sg)[VEC],
                                        bool fast) {
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    sg[i] = sigmoid(g[i], fast);
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
    if (blockDim.x > 256) {
      v[i] = warp_sum(r[i * 32 + (threadIdx.x & 31)]);
    } else {  // 8 warps at most
      const float4 *q = reinterpret_cast<const float4 *>(r + i * 32);
      const float4 a = q[0], b = q[1];
      v[i] = ((a.x + b.x) + (a.y + b.y)) + ((a.z + b.z) + (a.w + b.w));
    }
  }
}
__device__ __forceinline__ void clear_red(float *red) {
  const int t = threadIdx.y * blockDim.x + threadIdx.x;
  for (int i = t; i < kRed; i += blockDim.x * blockDim.y) red[i] = 0.f;
  __syncthreads();
}

// The VEC columns of a thread's chunk c.  Rows whose width is no multiple of 8
// start anywhere in 16 bytes (SHIFT); a group's rows, 8 or a multiple of it
// apart, all at the same place, so its threads' chunks start `phase` values in
// front of the row, where every access is aligned.  The chunks at a row's ends
// are cut: their values outside [lo, hi) count as 0 and are not written.
template <int VEC, bool SHIFT>
struct Chunk {
  int col, lo, hi;
  bool in, cut;
  __device__ __forceinline__ Chunk(const SeamParams &p, int c, int phase) {
    col = (c * (int)blockDim.x + (int)threadIdx.x) * VEC - (SHIFT ? phase : 0);
    in = col < p.d, cut = false, lo = 0, hi = VEC;
    if (SHIFT) {
      lo = max(0, -col), hi = min(VEC, p.d - col);
      cut = in && hi - lo < VEC;
    }
  }
  // Loads of a row.  A cut chunk's values outside belong to the rows next to it,
  // or lie behind the tensor's last value: there, single loads.
  __device__ __forceinline__ void load(Raw<VEC> &r, const SeamParams &p, const void *from, int row, int64_t ld,
                                       bool b16) const {
    const int64_t at = row * ld + col;
    if constexpr (SHIFT) {
      if (hi < VEC && at + VEC > (p.rows - 1) * ld + p.d) {
        uint32_t w[8] = {};
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (i >= lo && i < hi) {
            if (b16)
              w[i / 2] |= (uint32_t) static_cast<const unsigned short *>(from)[at + i] << (16 * (i & 1));
            else
              w[i] = static_cast<const uint32_t *>(from)[at + i];
          }
        r.a = make_uint4(w[0], w[1], w[2], w[3]), r.b = make_uint4(w[4], w[5], w[6], w[7]);
        return;
      }
    }
    r.load(from, at, b16);
  }
  __device__ __forceinline__ void get(const Raw<VEC> &r, float (&v)[VEC], bool b16) const {
    r.get(v, b16);
    if (SHIFT && cut) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[i] = i >= lo && i < hi ? v[i] : 0.f;
    }
  }
  __device__ __forceinline__ void store(void *to, int64_t row_at, const float (&v)[VEC], bool b16) const {
    if (SHIFT && cut) {
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (i >= lo && i < hi) {
          const float one[1] = {v[i]};
          put<1>(to, row_at + col + i, one, b16);
        }
    } else {
      put<VEC>(to, row_at + col, v, b16);
    }
  }
  __device__ __forceinline__ void weight(const float *w, float (&v)[VEC]) const {
    if constexpr (SHIFT) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[i] = i >= lo && i < hi ? __ldg(w + col + i) : 0.f;
    } else {
      weights<VEC>(w, col, v);
    }
  }
  // post_w scale (what is not given counts as 1).
  __device__ __forceinline__ void both_weights(const SeamParams &p, float (&v)[VEC]) const {
    fill(v, 1.f);
    if (p.w1) weight(p.w1, v);
    if (p.s) {
      float s[VEC];
      weight(p.s, s);
      mul(v, v, s);
    }
  }
  // Those and pre_w.
  __device__ __forceinline__ void all_weights(const SeamParams &p, float (&v)[VEC], float (&w2)[VEC]) const {
    fill(v, 0.f), fill(w2, 0.f);
    if (in) {
      both_weights(p, v);
      if (p.w2) weight(p.w2, w2);
    }
  }
};
// Where the rows of a group start in 16 bytes, its first one given.
__device__ __forceinline__ int phase_of(int row, int d) { return (int)((int64_t)row * d & 7); }

// Threads of a row: a warp (blockDim.y rows per block) or the whole block
// (blockDim.y == 1).  Thread k of a row holds chunks c * n + k of VEC values,
// c < K, n the row's threads.  Where those are few, the weights stay in
// registers while a block walks over rows, and a row's loads are under way
// while the row before it is summed.
template <int VEC, int K, int TX, int TH, bool SHIFT>
__global__ void __launch_bounds__(VEC == 8 && K == 1 ? 1024 : 512, VEC == 8 ? 1 : 2) seam_forward_kernel(SeamParams p) {
  constexpr bool kAhead = VEC * K <= 8 && K <= 4;
  static_assert(kAhead || !SHIFT, "a group's rows share their phase");
  __shared__ __align__(16) float red[kRed];
  int flip = 0;
  clear_red(red);
  const int n = blockDim.x;
  const bool one_warp = n == 32, x16 = TX == 1, h16 = TH == 1;
  const int step = p.parts;  // row groups
  int row = blockIdx.x * blockDim.y + threadIdx.y;
  const int phase = SHIFT ? phase_of(row, p.d) : 0;
  Raw<VEC> hr[K], gr[K], xr[K];
  auto fetch = [&](int row) {
#pragma unroll
    for (int c = 0; c < K; ++c) {
      const Chunk<VEC, SHIFT> k(p, c, phase);
      if (k.in) {
        k.load(hr[c], p, p.h, row, p.ldh, h16);
        if (p.g) k.load(gr[c], p, p.g, row, p.ldg, h16);
        k.load(xr[c], p, p.x, row, p.ldx, x16);
      }
    }
  };
  float kept1[K][VEC], kept2[K][VEC];  // with kAhead: post_w scale, pre_w
  if (kAhead) {
#pragma unroll
    for (int c = 0; c < K; ++c) Chunk<VEC, SHIFT>(p, c, phase).all_weights(p, kept1[c], kept2[c]);
  }
  if (kAhead && row < p.rows) fetch(row);
  for (; row < p.rows; row += step) {  // a block's threads leave together where they share a row
    if (!kAhead) fetch(row);
    const int64_t at = (int64_t)row * p.d;
    float z[K][VEC], x[K][VEC];
    Dot dot;
#pragma unroll
    for (int c = 0; c < K; ++c) {
      const Chunk<VEC, SHIFT> k(p, c, phase);
      if (k.in) {
        k.get(hr[c], z[c], h16);
        dot.add(z[c], z[c]);
        // all of n but r1
        if (p.g) {
          float v[VEC], sw[VEC], sg[VEC];
          k.get(gr[c], v, h16);
          gate_by(z[c], v, sw, sg, x16 && h16);
        }
        if (kAhead) {
          mul(z[c], z[c], kept1[c]);
        } else {
          float v[VEC];
          k.both_weights(p, v);
          mul(z[c], z[c], v);
        }
        k.get(xr[c], x[c], x16);
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
      const Chunk<VEC, SHIFT> k(p, c, phase);
      if (k.in) {
        fma(z[c], z[c], r1, x[c]);
        dz.add(z[c], z[c]);
        k.store(p.z, at, z[c], x16);
      }
    }
    float r2 = 1.f;
    if (p.w2) {
      float sz[1] = {dz.sum()};
      row_sum(sz, one_warp, red, flip);
      r2 = rsqrtf(fmaf(sz[0], p.inv_d, p.eps));
#pragma unroll
      for (int c = 0; c < K; ++c) {
        const Chunk<VEC, SHIFT> k(p, c, phase);
        if (k.in) {
          mul(z[c], z[c], r2);
          if (kAhead) {
            mul(z[c], z[c], kept2[c]);
          } else {
            float v[VEC];
            k.weight(p.w2, v);
            mul(z[c], z[c], v);
          }
          k.store(p.y, at, z[c], p.y16);
        }
      }
    }
    if (p.stats && threadIdx.x == 0) {
      p.stats[row] = r1;
      p.stats[p.rows + row] = r2;
    }
  }
}

// What a thread has of a row in the backward, as it lies in memory.
template <int VEC>
struct RawRow {
  Raw<VEC> h, g, x, dz, dy;
  template <bool SHIFT>
  __device__ __forceinline__ void load(const SeamParams &p, const Chunk<VEC, SHIFT> &k, int row, bool x16, bool h16) {
    k.load(h, p, p.h, row, p.ldh, h16);
    if (p.g) k.load(g, p, p.g, row, p.ldg, h16);
    if (p.dz) k.load(dz, p, p.dz, row, p.lddz, x16);
    if (p.dy) {
      k.load(dy, p, p.dy, row, p.lddy, p.y16);
      k.load(x, p, p.x, row, p.ldx, x16);
    }
  }
};

// A row's statistics.
struct RowStats {
  float r1 = 1.f, r2 = 1.f;
  __device__ __forceinline__ void load(const SeamParams &p, int row) {
    if (row >= p.rows) return;
    if (p.w1) r1 = p.stats[row];
    if (p.w2) r2 = p.stats[p.rows + row];
  }
};

__device__ __forceinline__ void ahead(const void *p, int64_t i, bool b16) {
  asm volatile("prefetch.global.L2 [%0];" ::"l"(static_cast<const char *>(p) + i * (b16 ? 2 : 4)));
}

// Sends a chunk of a row that is not the first on its way into L2 (what is in
// front of it is there); one thread in four reaches every 128 bytes.
template <int VEC, bool SHIFT>
__device__ __forceinline__ void ahead(const SeamParams &p, const Chunk<VEC, SHIFT> &k, int row, bool x16, bool h16) {
  ahead(p.h, row * p.ldh + k.col, h16);
  if (p.g) ahead(p.g, row * p.ldg + k.col, h16);
  if (p.dz) ahead(p.dz, row * p.lddz + k.col, x16);
  if (p.dy) ahead(p.dy, row * p.lddy + k.col, p.y16), ahead(p.x, row * p.ldx + k.col, x16);
}

// A row group's column sums, each its part of the planes.
template <int VEC, int K, bool SHIFT>
__device__ __forceinline__ void write_part(const SeamParams &p, int part, int phase, const float (&a1)[K][VEC],
                                           const float (&a2)[K][VEC]) {
#pragma unroll
  for (int c = 0; c < K; ++c) {
    const Chunk<VEC, SHIFT> k(p, c, phase);
    if (k.in) {
      if (p.w1 || p.s) k.store(p.part, (int64_t)part * p.d, a1[c], false);
      if (p.w2) k.store(p.part + p.plane, (int64_t)part * p.d, a2[c], false);
    }
  }
}

template <int VEC, int K, int TX, int TH, bool one_warp, bool SHIFT>
__global__ void __launch_bounds__(512, 1) seam_backward_kernel(SeamParams p) {
  constexpr bool kAhead = VEC * K <= 8 && K <= 4;
  static_assert(kAhead || !SHIFT, "a group's rows share their phase");
  // A row's statistics are read with the row before it (else it waits for them:
  // 32768 x 2048 bf16 196 us against 224), and the row behind the next is sent on
  // its way into L2 (182 against 196; fp32 rows have bytes enough under way
  // without, 8192 x 4096 took 206 us against 194).  Where the threads at a row's
  // ends need registers for their masks, either spills: 16384 x 1531 bf16 146 us
  // against 132.
  constexpr bool kStats = !SHIFT, kToL2 = VEC == 8 && !SHIFT && (TX || TH);
  __shared__ __align__(16) float red[kRed];
  int flip = 0;
  clear_red(red);
  const bool x16 = TX == 1, h16 = TH == 1;
  // the row group's place among all; one for the whole block keeps a row's address in uniform registers
  const int part = one_warp ? blockIdx.x * blockDim.y + threadIdx.y : blockIdx.x;
  const int phase = SHIFT ? phase_of(part, p.d) : 0;
  float a1[K][VEC], a2[K][VEC];  // this thread's columns of sum Z swish hh and of dw2
#pragma unroll
  for (int c = 0; c < K; ++c) fill(a1[c], 0.f), fill(a2[c], 0.f);
  float kept1[K][VEC], kept2[K][VEC];  // with kAhead: post_w scale, pre_w
  if (kAhead) {
#pragma unroll
    for (int c = 0; c < K; ++c) Chunk<VEC, SHIFT>(p, c, phase).all_weights(p, kept1[c], kept2[c]);
  }
  RawRow<VEC> raw[K];
  auto fetch = [&](int row) {
#pragma unroll
    for (int c = 0; c < K; ++c) {
      const Chunk<VEC, SHIFT> k(p, c, phase);
      if (k.in) raw[c].load(p, k, row, x16, h16);
    }
  };
  RowStats stats;
  if (kStats) stats.load(p, part);
  if (kAhead && part < p.rows) fetch(part);
  for (int row = part; row < p.rows; row += p.parts) {
    if (!kAhead) fetch(row);
    if (!kStats) stats.load(p, row);
    const float r1 = stats.r1, r2 = stats.r2;
    Dot tz, eq, zq;  // t zh, e q, zh q
    // hh (h without post_w), swish and sigmoid of the gate, zh, e = dz + r2 t; q is what z has of n
    float hh[K][VEC], sw[K][VEC], sg[K][VEC], zh[K][VEC], e[K][VEC];
#pragma unroll
    for (int c = 0; c < K; ++c) {
      const Chunk<VEC, SHIFT> k(p, c, phase);
      if (k.in) {
        float q[VEC], v[VEC], w[VEC];
        k.get(raw[c].h, hh[c], h16);
        mul(hh[c], hh[c], r1);
        if (kAhead) {
          mul(q, hh[c], kept1[c]);
        } else {
          k.both_weights(p, w);
          mul(q, hh[c], w);
        }
        if (p.g) {
          k.get(raw[c].g, v, h16);
          gate_by(q, v, sw[c], sg[c], x16 && h16);
        }
        if (p.dz)
          k.get(raw[c].dz, e[c], x16);
        else
          fill(e[c], 0.f);
        if (p.dy) {
          float dy[VEC];
          k.get(raw[c].x, v, x16);
          k.get(raw[c].dy, dy, p.y16);
          fma(zh[c], v, p.alpha, q);
          mul(zh[c], zh[c], r2);
          fma(a2[c], dy, zh[c], a2[c]);
          if (kAhead) {
            mul(dy, dy, kept2[c]);  // t
          } else {
            k.weight(p.w2, w);
            mul(dy, dy, w);
          }
          tz.add(dy, zh[c]);
          fma(e[c], dy, r2, e[c]);
          zq.add(zh[c], q);
        }
        eq.add(e[c], q);
      }
    }
    if (kStats) stats.load(p, row + p.parts);
    if (kAhead && row + p.parts < p.rows) fetch(row + p.parts);
    if (kToL2 && row + 2 * p.parts < p.rows && threadIdx.x % 4 == 0) {
#pragma unroll
      for (int c = 0; c < K; ++c) {
        const Chunk<VEC, SHIFT> k(p, c, phase);
        if (k.in) ahead(p, k, row + 2 * p.parts, x16, h16);
      }
    }
    float sum[3] = {tz.sum(), eq.sum(), zq.sum()};
    if (p.w1 || p.dy) row_sum(sum, one_warp, red, flip);
    const float m2 = p.dy ? r2 * (sum[0] * p.inv_d) : 0.f;  // r2 mean(t zh)
    const float m1 = (sum[1] - m2 * sum[2]) * p.inv_d;       // mean(N w1 hh)
    const int64_t at = (int64_t)row * p.d;
#pragma unroll
    for (int c = 0; c < K; ++c) {
      const Chunk<VEC, SHIFT> k(p, c, phase);
      if (k.in) {
        float o[VEC], v[VEC], w[VEC];
        if (p.dy) fma(e[c], zh[c], -m2, e[c]);  // Z
        mul(o, e[c], p.alpha);
        k.store(p.dx, at, o, x16);
        if (!kAhead) k.both_weights(p, w);
        mul(o, e[c], hh[c]);
        if (kAhead)
          mul(v, e[c], kept1[c]);
        else
          mul(v, e[c], w);
        if (p.g) {
          fma(a1[c], o, sw[c], a1[c]);
          mul(o, v, hh[c]);
          slope_by(o, sw[c], sg[c]);
          k.store(p.dg, at, o, h16);
          mul(v, v, sw[c]);
        } else {
#pragma unroll
          for (int i = 0; i < VEC; ++i) a1[c][i] += o[i];
        }
        if (p.w1) {  // v = N w1
          fma(v, hh[c], -m1, v);
          mul(v, v, r1);
        }
        k.store(p.dh, at, v, h16);
      }
    }
  }
  write_part<VEC, K, SHIFT>(p, part, phase, a1, a2);
}

// For wide rows, in two passes that each form a row's values anew from those in
// memory (w: post_w scale; t = dy pre_w; e = dz + r2 t).
// `of` gives the weights where they are needed.
template <int VEC>
struct SeamValues {
  float hh[VEC], sw[VEC], sg[VEC], w[VEC], q[VEC], zh[VEC], e[VEC], dy[VEC], t[VEC];
  template <bool SHIFT, typename W>
  __device__ __forceinline__ void form(const SeamParams &p, const Chunk<VEC, SHIFT> &k, const RawRow<VEC> &r,
                                       const W &of, float r1, float r2, bool x16, bool h16) {
    of.both(w);
    k.get(r.h, hh, h16);
    mul(hh, hh, r1);
    mul(q, hh, w);
    if (p.g) {
      float g[VEC];
      k.get(r.g, g, h16);
      gate_by(q, g, sw, sg, x16 && h16);
    }
    fill(e, 0.f), fill(zh, 0.f), fill(t, 0.f), fill(dy, 0.f);
    if (p.dz) k.get(r.dz, e, x16);
    if (p.dy) {
      float v[VEC];
      k.get(r.x, v, x16);
      k.get(r.dy, dy, p.y16);
      fma(zh, v, p.alpha, q);
      mul(zh, zh, r2);
      of.pre(v);
      mul(t, dy, v);
      fma(e, t, r2, e);
    }
  }
  // The gradients; what they add to the columns' sums goes to a1 and a2.
  template <bool SHIFT>
  __device__ __forceinline__ void write(const SeamParams &p, const Chunk<VEC, SHIFT> &k, int64_t at, float r1, float m1, float m2, bool x16, bool h16,
                                        float (&a1)[VEC], float (&a2)[VEC]) {
    float v[VEC], o[VEC];
    fma(a2, dy, zh, a2);
    fma(e, zh, -m2, e);  // Z
    mul(v, e, p.alpha);
    k.store(p.dx, at, v, x16);
    mul(o, e, hh);
    mul(v, e, w);
    if (p.g) {
      fma(a1, o, sw, a1);
      mul(o, v, hh);
      slope_by(o, sw, sg);
      k.store(p.dg, at, o, h16);
      mul(v, v, sw);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) a1[i] += o[i];
    }
    if (p.w1) {
      fma(v, hh, -m1, v);
      mul(v, v, r1);
    }
    k.store(p.dh, at, v, h16);
  }
};

template <int VEC, bool SHIFT>
struct GivenWeights {
  const SeamParams &p;
  const Chunk<VEC, SHIFT> &k;
  __device__ __forceinline__ void both(float (&v)[VEC]) const { k.both_weights(p, v); }
  __device__ __forceinline__ void pre(float (&v)[VEC]) const { k.weight(p.w2, v); }
};
// A thread's own vectors in shared memory, each as two halves that lie `half`
// apart: those of its chunks, then as many of another kind.
struct Own {
  float4 *at;
  int half, kind;
  __device__ __forceinline__ void read(int i, float (&v)[8]) const {
    const float4 a = at[i], b = at[i + half];
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  }
  __device__ __forceinline__ void write(int i, const float (&v)[8]) const {
    at[i] = make_float4(v[0], v[1], v[2], v[3]), at[i + half] = make_float4(v[4], v[5], v[6], v[7]);
  }
  __device__ __forceinline__ void both(float (&v)[8]) const { read(0, v); }
  __device__ __forceinline__ void pre(float (&v)[8]) const { read(kind, v); }
};

// Rows of up to K 512 chunks: the row as it lies in memory stays in registers,
// the columns' sums in shared memory where each thread alone touches its own, the
// block's next row is on its way into L2.  So do weights of rows that start
// anywhere: no vector holds them elsewhere.
template <int K, int TX, int TH, bool SHIFT>
__global__ void __launch_bounds__(512, 1) seam_backward_held_kernel(SeamParams p) {
  constexpr int VEC = 8;
  extern __shared__ __align__(16) float4 own[];  // [sums, weights][2][K][2][threads]
  __shared__ __align__(16) float red[kRed];
  int flip = 0;
  clear_red(red);
  const int n = blockDim.x;
  const bool x16 = TX == 1, h16 = TH == 1;
  const int phase = SHIFT ? phase_of(blockIdx.x, p.d) : 0;
  auto sums = [&](int c) { return Own{own + c * 2 * n + threadIdx.x, n, 2 * K * n}; };
  auto own_weights = [&](int c) { return Own{own + (2 * K + c) * 2 * n + threadIdx.x, n, 2 * K * n}; };
#pragma unroll
  for (int c = 0; c < K; ++c) {
    float w[VEC], w2[VEC];
    fill(w, 0.f);
    sums(c).write(0, w), sums(c).write(sums(c).kind, w);
    if (SHIFT) {
      Chunk<VEC, SHIFT>(p, c, phase).all_weights(p, w, w2);
      own_weights(c).write(0, w), own_weights(c).write(own_weights(c).kind, w2);
    }
  }
  auto form = [&](SeamValues<VEC> &s, const Chunk<VEC, SHIFT> &k, int c, const RawRow<VEC> &r, float r1, float r2) {
    if constexpr (SHIFT)
      s.form(p, k, r, own_weights(c), r1, r2, x16, h16);
    else
      s.form(p, k, r, GivenWeights<VEC, SHIFT>{p, k}, r1, r2, x16, h16);
  };
  for (int row = blockIdx.x; row < p.rows; row += p.parts) {
    RawRow<VEC> raw[K];
#pragma unroll
    for (int c = 0; c < K; ++c) {
      const Chunk<VEC, SHIFT> k(p, c, phase);
      if (k.in) raw[c].load(p, k, row, x16, h16);
    }
    const int next = row + p.parts;
    if (next < p.rows && threadIdx.x % 4 == 0) {
#pragma unroll
      for (int c = 0; c < K; ++c) {
        const Chunk<VEC, SHIFT> k(p, c, phase);
        if (k.in) ahead(p, k, next, x16, h16);
      }
    }
    const float r1 = p.w1 ? p.stats[row] : 1.f, r2 = p.w2 ? p.stats[p.rows + row] : 1.f;
    Dot tz, eq, zq;
#pragma unroll
    for (int c = 0; c < K; ++c) {
      const Chunk<VEC, SHIFT> k(p, c, phase);
      if (k.in) {
        SeamValues<VEC> s;
        form(s, k, c, raw[c], r1, r2);
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
      const Chunk<VEC, SHIFT> k(p, c, phase);
      if (k.in) {
        SeamValues<VEC> s;
        form(s, k, c, raw[c], r1, r2);
        float a1[VEC], a2[VEC];
        sums(c).read(0, a1), sums(c).read(sums(c).kind, a2);
        s.write(p, k, (int64_t)row * p.d, r1, m1, m2, x16, h16, a1, a2);
        sums(c).write(0, a1), sums(c).write(sums(c).kind, a2);
      }
    }
  }
  float a1[K][VEC], a2[K][VEC];
#pragma unroll
  for (int c = 0; c < K; ++c) sums(c).read(0, a1[c]), sums(c).read(sums(c).kind, a2[c]);
  write_part<VEC, K, SHIFT>(p, blockIdx.x, phase, a1, a2);
}

// Wider ones: the second pass reads the row from the caches, the column sums
// lie in shared memory, [2][d], where every thread alone touches its columns.
template <int VEC, int TX, int TH>
__global__ void __launch_bounds__(512, 1) seam_backward_wide_kernel(SeamParams p) {
  extern __shared__ __align__(16) float acc[];
  __shared__ __align__(16) float red[kRed];
  int flip = 0;
  clear_red(red);
  const bool x16 = TX == 1, h16 = TH == 1;
  const int chunks = (p.d + VEC * (int)blockDim.x - 1) / (VEC * (int)blockDim.x);
  float *a1 = acc, *a2 = acc + p.d;
  for (int c = 0; c < chunks; ++c) {
    const Chunk<VEC, false> k(p, c, 0);
    if (k.in) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) a1[k.col + i] = a2[k.col + i] = 0.f;
    }
  }
  auto values = [&](const Chunk<VEC, false> &k, int row, float r1, float r2, SeamValues<VEC> &s) {
    RawRow<VEC> raw;
    raw.load(p, k, row, x16, h16);
    s.form(p, k, raw, GivenWeights<VEC, false>{p, k}, r1, r2, x16, h16);
  };
  for (int row = blockIdx.x; row < p.rows; row += p.parts) {
    const float r1 = p.w1 ? p.stats[row] : 1.f, r2 = p.w2 ? p.stats[p.rows + row] : 1.f;
    Dot tz, eq, zq;
    for (int c = 0; c < chunks; ++c) {
      const Chunk<VEC, false> k(p, c, 0);
      if (!k.in) continue;
      SeamValues<VEC> s;
      values(k, row, r1, r2, s);
      tz.add(s.t, s.zh);
      eq.add(s.e, s.q);
      zq.add(s.zh, s.q);
    }
    float sum[3] = {tz.sum(), eq.sum(), zq.sum()};
    row_sum(sum, false, red, flip);
    const float m2 = r2 * (sum[0] * p.inv_d), m1 = (sum[1] - m2 * sum[2]) * p.inv_d;
    for (int c = 0; c < chunks; ++c) {
      const Chunk<VEC, false> k(p, c, 0);
      if (!k.in) continue;
      SeamValues<VEC> s;
      float b1[VEC], b2[VEC];
      values(k, row, r1, r2, s);
#pragma unroll
      for (int i = 0; i < VEC; ++i) b1[i] = a1[k.col + i], b2[i] = a2[k.col + i];
      s.write(p, k, (int64_t)row * p.d, r1, m1, m2, x16, h16, b1, b2);
#pragma unroll
      for (int i = 0; i < VEC; ++i) a1[k.col + i] = b1[i], a2[k.col + i] = b2[i];
    }
  }
  for (int c = 0; c < chunks; ++c) {
    const Chunk<VEC, false> k(p, c, 0);
    if (!k.in) continue;
    const int64_t at = (int64_t)blockIdx.x * p.d + k.col;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      if (p.w1 || p.s) p.part[at + i] = a1[k.col + i];
      if (p.w2) p.part[p.plane + at + i] = a2[k.col + i];
    }
  }
}

// Column sums of the [parts][d] planes (blockIdx.y: which): 16 warps share a
// block of 32 columns, each adds every sixteenth part in order.  The first
// plane's sum times scale is dw1, times post_w it is ds.
__global__ void __launch_bounds__(512) seam_columns_kernel(const float *part, int64_t plane, int parts, int d,
                                                           const float *w1, const float *s, float *dw1, float *ds,
                                                           float *dw2) {
  __shared__ float red[16][32];
  if (blockIdx.y ? !dw2 : !(dw1 || ds)) return;
  const int col = blockIdx.x * 32 + threadIdx.x;
  const float *src = part + blockIdx.y * plane + col;
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
// suffice, few values a thread, so that much is under way.  Vectors where the
// rows' addresses allow them (vec 8): in rows of any width, `shift` then says
// that they start anywhere in 16 bytes and a thread's vectors may start 7 values
// in front of the row.  16384 x 1531 bf16: forward 72 us, backward 135, against
// 181 and 241 with single values.  Backward rows wider than 4096 (k 2; 4, where x
// and h are bf16, `narrow`) keep their raw values: 4096 x 8192 bf16 134 us,
// against 323 with a second reading of the row (k 0), which remains for what no
// thread can hold.
struct Shape {
  int vec, k, threads, rows_per_block;
  bool shift;
};
Shape shape_of(int d, int vec, bool backward, bool narrow) {
  const bool shift = vec == 8 && d % 8 != 0;
  const int span = shift ? d + 7 : d;
  auto threads = [&](int per) { return (span + per * 32 - 1) / (per * 32) * 32; };  // whole warps that hold a row
  if (vec == 8) {
    if (span <= 256) return {8, 1, 32, 4, shift};
    if (span <= (backward ? 4096 : 8192)) return {8, 1, threads(8), 1, shift};
    if (backward && span <= 8192) return {8, 2, threads(16), 1, shift};
    if (backward && narrow && !shift) return {8, 4, 512, 1, false};
    if (!shift) return {8, backward ? 0 : 4, 512, 1, false};
  }
  if (d <= 128) return {1, 4, 32, 4, false};
  if (d <= 2048) return {1, 4, threads(4), 1, false};
  if (d <= 4096) return {1, 8, threads(8), 1, false};
  if (backward) return {1, 0, 512, 1, false};
  return d <= 8192 ? Shape{1, 16, 512, 1, false} : Shape{1, 32, 512, 1, false};
}
bool walks(const Shape &s) { return s.vec * s.k <= 8 && s.k > 0 && s.k <= 4; }  // the kernels' kAhead

// The kernel of a shape (k 0: the two-pass backward).
using SeamKernel = void (*)(SeamParams);
template <int TX, int TH>
SeamKernel typed_kernel(const Shape &s, bool backward) {
  const bool warp = s.rows_per_block > 1;
  if (backward) {
    if (s.vec == 8) {
      if (s.k == 1 && s.shift)
        return warp ? seam_backward_kernel<8, 1, TX, TH, true, true> : seam_backward_kernel<8, 1, TX, TH, false, true>;
      if (s.k == 1)
        return warp ? seam_backward_kernel<8, 1, TX, TH, true, false> : seam_backward_kernel<8, 1, TX, TH, false, false>;
      if (s.k == 2) return s.shift ? seam_backward_held_kernel<2, TX, TH, true> : seam_backward_held_kernel<2, TX, TH, false>;
      if constexpr (TX && TH)
        return seam_backward_held_kernel<4, TX, TH, false>;
      else
        return seam_backward_wide_kernel<8, TX, TH>;
    }
    return s.k == 4   ? (warp ? seam_backward_kernel<1, 4, TX, TH, true, false>
                              : seam_backward_kernel<1, 4, TX, TH, false, false>)
           : s.k == 8 ? seam_backward_kernel<1, 8, TX, TH, false, false>
                      : seam_backward_wide_kernel<1, TX, TH>;
  }
  if (s.vec == 8)
    return s.k == 1 ? (s.shift ? seam_forward_kernel<8, 1, TX, TH, true> : seam_forward_kernel<8, 1, TX, TH, false>)
                    : seam_forward_kernel<8, 4, TX, TH, false>;
  return s.k == 4    ? seam_forward_kernel<1, 4, TX, TH, false>
         : s.k == 8  ? seam_forward_kernel<1, 8, TX, TH, false>
         : s.k == 16 ? seam_forward_kernel<1, 16, TX, TH, false>
                     : seam_forward_kernel<1, 32, TX, TH, false>;
}
SeamKernel kernel_of(const Shape &s, bool x16, bool h16, bool backward) {
  if (x16) return h16 ? typed_kernel<1, 1>(s, backward) : typed_kernel<1, 0>(s, backward);
  return h16 ? typed_kernel<0, 1>(s, backward) : typed_kernel<0, 0>(s, backward);
}

// Values an access may take where rows of d values lie at p, ld elements apart:
// 8 if the first row starts on 16 bytes and every row does (fp32 rows: half of
// the accesses then start between), or all rows start where contiguous ones
// would.
int access_of(const void *p, int64_t ld, int d, int is16) {
  if (!p) return 8;
  if (reinterpret_cast<uintptr_t>(p) % 16) return 1;
  return d % 8 == 0 ? (ld % (is16 ? 8 : 4) == 0 ? 8 : 1) : (ld >= d && (ld - d) % 8 == 0 ? 8 : 1);
}
// Weights: the shifted kernels read them one by one.
int access_of(const float *w, int d) { return d % 8 ? 8 : access_of(w, 8, 8, 0); }

// Row groups that share the rows: `threads` an SM, as many as its registers
// hold; few enough that the backward's partial rows stay small beside the data.
// Where a group has several rows they start alike: the groups are a multiple of 8.
int parts_of(int num_sms, int64_t rows, const Shape &s, int threads) {
  const int per_sm = threads / (s.threads * s.rows_per_block);
  const int64_t blocks = (int64_t)num_sms * (per_sm < 1 ? 1 : per_sm), need = (rows + s.rows_per_block - 1) / s.rows_per_block;
  if (need <= blocks) return (int)need * s.rows_per_block;
  return (int)(s.shift ? blocks / 8 * 8 : blocks) * s.rows_per_block;
}
// Of a plane of partial rows, so that the second starts on 16 bytes too.
int64_t plane_of(int parts, int d) { return ((int64_t)parts * d + 7) / 8 * 8; }
constexpr int64_t kMaxRows = 1 << 30;  // rows and row groups are counted in 31 bits

}  // namespace

extern "C" {

int af_residual_norm(af_ctx *ctx, const void *x, int64_t ldx, int x_bf16, const void *h, int64_t ldh, int h_bf16,
                     const void *gate, int64_t ldg, const float *post_w, const float *scale, const float *pre_w,
                     float alpha, float eps, int64_t rows, int d, void *z, void *y, int y_bf16, float *stats,
                     af_stream_t stream) {
  const char *fn = "af_residual_norm";
  af::DeviceScope scope;
  AF_ENTER(ctx, fn);
  AF_REQUIRE(rows >= 0 && rows <= kMaxRows && d > 0, "af_residual_norm", "bad sizes");
  AF_REQUIRE(d <= kMaxWidth, "af_residual_norm", "rows of %d values: at most %d are supported", d, kMaxWidth);
  if (rows == 0) return AF_OK;
  AF_REQUIRE(x && h && z && (!pre_w || y), "af_residual_norm", "null argument");
  SeamParams p = {};
  p.x = x, p.h = h, p.g = gate, p.ldx = ldx, p.ldh = ldh, p.ldg = ldg;
  p.x16 = x_bf16 != 0, p.h16 = h_bf16 != 0, p.y16 = y_bf16 != 0;
  p.w1 = post_w, p.s = scale, p.w2 = pre_w, p.alpha = alpha, p.eps = eps, p.inv_d = 1.0f / (float)d;
  p.rows = (int)rows, p.d = d, p.z = z, p.y = y, p.stats = stats;
  const int vec = std::min({access_of(x, ldx, d, x_bf16), access_of(h, ldh, d, h_bf16), access_of(gate, ldg, d, h_bf16),
                            access_of(post_w, d), access_of(scale, d), access_of(pre_w, d), access_of(z, d, d, x_bf16),
                            access_of(y, d, d, y_bf16)});
  const Shape s = shape_of(d, vec, false, p.x16 && p.h16);
  int64_t blocks = (rows + s.rows_per_block - 1) / s.rows_per_block;
  if (walks(s)) blocks = parts_of(ctx->num_sms, rows, s, 1024) / s.rows_per_block;
  p.parts = (int)blocks * s.rows_per_block;
  kernel_of(s, p.x16, p.h16, false)<<<(unsigned)blocks, dim3(s.threads, s.rows_per_block), 0,
                                      af::stream_of(stream)>>>(p);
  return af::launched(ctx, fn);
}

int af_residual_norm_scratch(af_ctx *ctx, int64_t rows, int d, int64_t *floats) {
  const char *fn = "af_residual_norm_scratch";
  af::DeviceScope scope;
  AF_ENTER(ctx, fn);
  AF_REQUIRE(floats && rows >= 0 && rows <= kMaxRows && d > 0 && d <= kMaxWidth, "af_residual_norm_scratch",
             "bad sizes");
  int most = 0;  // whatever accesses the call's tensors will allow
  for (int vec : {1, 8}) most = std::max(most, parts_of(ctx->num_sms, rows, shape_of(d, vec, true, false), 512));
  *floats = 2 * plane_of(most, d);
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
  AF_REQUIRE(rows >= 0 && rows <= kMaxRows && d > 0, "af_residual_norm_backward", "bad sizes");
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
  const int vec = std::min({access_of(x, ldx, d, x_bf16), access_of(h, ldh, d, h_bf16), access_of(gate, ldg, d, h_bf16),
                            access_of(post_w, d), access_of(scale, d), access_of(pre_w, d), access_of(dz, lddz, d, x_bf16),
                            access_of(dy, lddy, d, y_bf16), access_of(dx, d, d, x_bf16), access_of(dh, d, d, h_bf16),
                            access_of(dgate, d, d, h_bf16), access_of(scratch, d, d, 0)});
  const Shape s = shape_of(d, vec, true, p.x16 && p.h16);
  p.parts = parts_of(ctx->num_sms, rows, s, 512), p.plane = plane_of(p.parts, d);
  const bool sums = post_w || scale || pre_w;
  AF_REQUIRE(!sums || (scratch && scratch_floats >= 2 * p.plane), "af_residual_norm_backward",
             "scratch of %lld floats, %lld are needed", (long long)scratch_floats, 2ll * p.plane);
  const SeamKernel kernel = kernel_of(s, p.x16, p.h16, true);
  size_t smem = 0;
  if (s.k == 0 || (s.vec == 8 && s.k > 1)) {  // column sums, with weights
    smem = s.k == 0 ? (size_t)2 * d * sizeof(float) : (size_t)(s.shift ? 4 : 2) * 8 * s.k * s.threads * sizeof(float);
    static std::atomic<unsigned long long> attr_devices[5][4];
    const int which = s.k == 0 ? s.vec == 8 : s.k + s.shift;
    if (int rc = af::smem_attr(ctx, reinterpret_cast<const void *>(kernel), (size_t)2 * kMaxWidth * sizeof(float),
                               attr_devices[which][p.x16 * 2 + p.h16], fn))
      return rc;
  }
  kernel<<<(unsigned)(p.parts / s.rows_per_block), dim3(s.threads, s.rows_per_block), smem, st>>>(p);
  if (int rc = af::launched(ctx, fn)) return rc;
  if (!sums) return AF_OK;
  seam_columns_kernel<<<dim3((unsigned)((d + 31) / 32), 2), dim3(32, 16), 0, st>>>(
      scratch, p.plane, p.parts, d, post_w, scale, post_w ? dpost_w : nullptr, scale ? dscale : nullptr,
      pre_w ? dpre_w : nullptr);
  return af::launched(ctx, fn);
}

}  // extern "C"
