// The gated residual between two norms, forward and backward, one pass over the rows each:
//   m = post-norm(y) (none, rms or layer), u = post_w m
//   x' = x + alpha gate[item] u
//   n = pre-norm(x') (rms or layer), h = pre_w n (1 + scale[item]) + shift[item]
// with the normalised rows n = (t - mean) r (rms: mean = 0), r = 1 / sqrt(mean((t - mean)^2) + eps).
// Backward, from dh and the gradient dx' that reaches x' from behind:
//   g = dh (1 + scale) pre_w,  G = dx' + r (g - mean(g) - n mean(g n))     (rms: without mean(g))
//   dx = G,  du = alpha gate G,  g = du post_w,  dy = r_y (g - mean(g) - m mean(g m))
//   dgate = alpha sum_item G u,  dscale = sum_item dh n pre_w,  dshift = sum_item dh,
//   dpost_w = sum du m,  dpre_w = sum dh (1 + scale) n
// The statistics are computed again from y and x' (a row is in registers anyway), so the forward saves
// nothing.
//
// Both passes are bound by HBM in fp32 and at 2048 columns (forward 82%, backward 90% of the copy rate); a
// backward of 1024 columns in 16 bits with a post norm is not: 4593 rows take 22.7 us for 8.6, with 767
// instructions a warp and row, 60% of the issue slots and 19% of DRAM's rate. A row is held in registers by
// T = C / V threads (V = 8 columns a thread, or 1 where the columns or alignments are odd); the row's sums are
// warp shuffles and one exchange through shared memory a round. Where the threads hold 8 columns each (4096: 16)
// and none is idle (C = 256, 512, 1024, 2048, 4096), mean, squares about the mean and products with the gradient
// come from one round: the threads' own moments about their own means are merged pairwise, which loses no
// digits to a large mean. The other widths take two to four dependent rounds a row, with no row in flight ahead.
// The backward's column sums stay in registers over the rows
// of a block, each block writes one partial row of sums and a second kernel adds the partials in a
// fixed order: no atomics, the same inputs give the same bits.

#include "internal.h"
#include "sm100.cuh"

namespace anima {
namespace resnorm {

constexpr int kNone = 0, kRms = 1, kLayer = 2;
constexpr int kThreads = 256;
constexpr int kMaxCols = 4096;  // 16 columns a thread: the backward's five sums of each fit its registers
constexpr int kMaxSums = 5;

struct Params {
  const void* x;   // forward: x; backward: x'
  const void* y;
  const void* dh;  // backward
  const void* dx;  // backward: the gradient that reaches x' from behind, or NULL
  void* o0;        // forward: x'; backward: dx
  void* o1;        // forward: h;  backward: dy
  long long ldx, ldy, lddh, lddx, ldo0, ldo1;
  int dtx, dty, dth;  // x, x', dx share a type, so do y and dy, and h and dh
  int rows, C, L;     // L rows an item
  int post, pre;
  float alpha, eps;
  const float *gate, *scale, *shift, *post_w, *pre_w;
  long long ldgate, ldscale, ldshift;
  int layer_threads;  // T
  // backward: the partial sums [item][part][k][C] and which sum is where (-1: not asked for)
  float* part;
  int parts, part_rows, sums;
  int places;  // of the ring
  int s_gate, s_postw, s_prew, s_scale, s_shift;
};

__device__ __forceinline__ float lo16(uint32_t w, int dt) {
  return dt == ANIMA_BF16 ? __uint_as_float(w << 16) : __half2float(__ushort_as_half(static_cast<unsigned short>(w)));
}
__device__ __forceinline__ float hi16(uint32_t w, int dt) {
  return dt == ANIMA_BF16 ? __uint_as_float(w & 0xFFFF0000u)
                          : __half2float(__ushort_as_half(static_cast<unsigned short>(w >> 16)));
}

// V elements as they lie in memory: 8 of 32 bits take both vectors, 8 of 16 bits the first.
template <int V>
struct Raw {
  uint4 a, b;
};
template <>
struct Raw<1> {
  uint32_t a;
};

template <int V>
__device__ __forceinline__ void load_raw(Raw<V>& r, const void* p, int dt, size_t at) {
  if constexpr (V == 8) {
    if (dt == ANIMA_F32) {
      const uint4* q = reinterpret_cast<const uint4*>(static_cast<const float*>(p) + at);
      r.a = q[0];  // plain loads: an output may be its input
      r.b = q[1];
    } else {
      r.a = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + at);
    }
  } else {
    r.a = dt == ANIMA_F32 ? static_cast<const uint32_t*>(p)[at]
                          : static_cast<uint32_t>(static_cast<const uint16_t*>(p)[at]);
  }
}

template <int V>
__device__ __forceinline__ void unpack(const Raw<V>& r, int dt, float (&v)[V]) {
  if constexpr (V == 8) {
    const uint32_t a[4] = {r.a.x, r.a.y, r.a.z, r.a.w};
    if (dt == ANIMA_F32) {
      const uint32_t b[4] = {r.b.x, r.b.y, r.b.z, r.b.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[i] = __uint_as_float(a[i]);
        v[4 + i] = __uint_as_float(b[i]);
      }
    } else {
      // (one branch for all eight: a choice for each element would cost more than the row's sums)
      if (dt == ANIMA_BF16) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[2 * i] = lo16(a[i], ANIMA_BF16);
          v[2 * i + 1] = hi16(a[i], ANIMA_BF16);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&a[i]));
          v[2 * i] = f.x;
          v[2 * i + 1] = f.y;
        }
      }
    }
  } else {
    v[0] = dt == ANIMA_F32 ? __uint_as_float(r.a) : lo16(r.a, dt);
  }
}

__device__ __forceinline__ uint32_t pack16(float a, float b, int dt) {
  if (dt == ANIMA_BF16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <int V>
__device__ __forceinline__ void store(void* p, int dt, size_t at, const float (&v)[V]) {
  if constexpr (V == 8) {
    if (dt == ANIMA_F32) {
      float4* q = reinterpret_cast<float4*>(static_cast<float*>(p) + at);
      q[0] = make_float4(v[0], v[1], v[2], v[3]);
      q[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      uint4* q = reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + at);
      if (dt == ANIMA_BF16)
        *q = make_uint4(pack16(v[0], v[1], ANIMA_BF16), pack16(v[2], v[3], ANIMA_BF16), pack16(v[4], v[5], ANIMA_BF16),
                        pack16(v[6], v[7], ANIMA_BF16));
      else
        *q = make_uint4(pack16(v[0], v[1], ANIMA_F16), pack16(v[2], v[3], ANIMA_F16), pack16(v[4], v[5], ANIMA_F16),
                        pack16(v[6], v[7], ANIMA_F16));
    }
  } else {
    if (dt == ANIMA_F32)
      static_cast<float*>(p)[at] = v[0];
    else
      static_cast<uint16_t*>(p)[at] = static_cast<uint16_t>(pack16(v[0], 0.f, dt));
  }
}

// fp32 parameters of the row's columns (modulations, norm weights); `none` where there are none
template <int V>
__device__ __forceinline__ void param(const float* p, size_t at, float none, float (&v)[V]) {
  if (!p) {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = none;
  } else if constexpr (V == 8) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(p + at)), b = __ldg(reinterpret_cast<const float4*>(p + at) + 1);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
    v[0] = __ldg(p + at);
  }
}

// Sums of K values over the T threads of a row, to all of them. `buf` alternates between the calls on `red`,
// so one barrier a call is enough: a value is read before its thread can reach the barrier after next, behind
// which its place is written again. That needs all calls on one array to have places of one size, so
// row_moments has an array and a `buf` of its own.
template <int K>
__device__ __forceinline__ void row_sum(float (&v)[K], float* red, int& buf) {
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) v[k] += __shfl_xor_sync(0xffffffffu, v[k], s);
  const int W = blockDim.x >> 5;
  if (W == 1) return;
  float* slot = red + (buf * blockDim.y + threadIdx.y) * (W * 2);
  buf ^= 1;
  if ((threadIdx.x & 31) == 0) {
#pragma unroll
    for (int k = 0; k < K; ++k) slot[(threadIdx.x >> 5) * 2 + k] = v[k];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < K; ++k) {
    v[k] = 0.f;
    for (int w = 0; w < W; ++w) v[k] += slot[w * 2 + k];
  }
}
constexpr int kRedFloats = 2 * 2 * (kThreads / 32);  // [2 buffers][rows][warps][2 values]

// A thread's columns: NV vectors of V, T V apart.
template <int V, int NV>
struct Cols {
  int c0, step, C;
  __device__ __forceinline__ Cols(const Params& p) : c0(threadIdx.x * V), step(blockDim.x * V), C(p.C) {}
  __device__ __forceinline__ int at(int k) const { return c0 + k * step; }
  __device__ __forceinline__ bool in(int k) const { return at(k) < C; }  // V divides C
};

// In place: t -> its normalised row; returns r. Columns past C hold 0 and do not count.
template <int V, int NV>
__device__ __forceinline__ float normalise(float (&t)[NV][V], const Cols<V, NV>& cols, int kind, float inv_c, float eps,
                                           float* red, int& buf) {
  if (kind == kLayer) {
    float s[1] = {0.f};
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) s[0] += t[k][i];
    row_sum(s, red, buf);
    const float mean = s[0] * inv_c;
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (cols.in(k)) {
#pragma unroll
        for (int i = 0; i < V; ++i) t[k][i] -= mean;
      }
  }
  float q[1] = {0.f};
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) q[0] = fmaf(t[k][i], t[k][i], q[0]);
  row_sum(q, red, buf);
  const float r = 1.0f / sqrtf(fmaf(q[0], inv_c, eps));
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) t[k][i] *= r;
  return r;
}

template <int V, int NV>
__device__ __forceinline__ void load_row(float (&t)[NV][V], const Cols<V, NV>& cols, const void* p, int dt, size_t base,
                                         bool live) {
  Raw<V> raw[NV];
#pragma unroll
  for (int k = 0; k < NV; ++k)
    if (live && cols.in(k)) load_raw<V>(raw[k], p, dt, base + cols.at(k));
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    if (live && cols.in(k)) {
      unpack<V>(raw[k], dt, t[k]);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) t[k][i] = 0.f;
    }
  }
}

// Moments of a row for one norm: mean, sum of squares about it (rms: about 0), and of a gradient g the
// sums of g and of g (t - mean).
struct Moments {
  float mean, m2, g, gt;
};

// A thread's 8 NV values.
template <int NV>
__device__ __forceinline__ Moments moments_of(const float (&t)[NV][8], const float (*g)[8], int kind) {
  Moments m{0.f, 0.f, 0.f, 0.f};
  if (kind == kLayer) {
#pragma unroll
    for (int k = 0; k < NV; ++k) m.mean += ((t[k][0] + t[k][1]) + (t[k][2] + t[k][3])) + ((t[k][4] + t[k][5]) + (t[k][6] + t[k][7]));
    m.mean *= 1.0f / (8 * NV);
  }
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float d = t[k][i] - m.mean;
      m.m2 = fmaf(d, d, m.m2);
      if (g) {
        m.g += g[k][i];
        m.gt = fmaf(g[k][i], d, m.gt);
      }
    }
  return m;
}

// Two sets of n values each, their means d apart: both terms of the difference change sign with the order,
// so the two lanes that merge get the same bits.
template <bool GRAD>
__device__ __forceinline__ void merge_lanes(Moments& m, int lanes, float n) {
  const float mean = __shfl_xor_sync(0xffffffffu, m.mean, lanes), m2 = __shfl_xor_sync(0xffffffffu, m.m2, lanes);
  const float h = 0.5f * (mean - m.mean);
  if (GRAD) {
    const float g = __shfl_xor_sync(0xffffffffu, m.g, lanes), gt = __shfl_xor_sync(0xffffffffu, m.gt, lanes);
    m.gt = fmaf(g - m.g, h, m.gt + gt);  // t - common mean is t - own mean, less h or plus h
    m.g += g;
  }
  m.m2 = fmaf(2.f * n * h, h, m.m2 + m2);
  m.mean = 0.5f * (m.mean + mean);
}

constexpr int kRedMoments = 2 * 2 * (kThreads / 32);  // [2 buffers][warps][2 sets]

// The moments of K sets, n values a thread, over the row's threads, to all of them (GRAD0: the first set
// has a gradient). One barrier, as in row_sum, and so K is the same in all calls on one array.
template <int K, bool GRAD0>
__device__ __forceinline__ void row_moments(Moments (&m)[K], float n, float4* red, int& buf) {
  auto step = [&](int lanes) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (k == 0 && GRAD0)
        merge_lanes<true>(m[k], lanes, n);
      else
        merge_lanes<false>(m[k], lanes, n);
    }
    n *= 2.f;
  };
#pragma unroll
  for (int lanes = 1; lanes < 32; lanes *= 2) step(lanes);
  const int W = blockDim.x >> 5;
  if (W == 1) return;
  float4* slot = red + buf * (W * K);
  buf ^= 1;
  if ((threadIdx.x & 31) == 0) {
#pragma unroll
    for (int k = 0; k < K; ++k) slot[(threadIdx.x >> 5) * K + k] = make_float4(m[k].mean, m[k].m2, m[k].g, m[k].gt);
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < K; ++k) {  // lane i goes on with warp i % W's
    const float4 v = slot[(threadIdx.x & (W - 1)) * K + k];
    m[k] = Moments{v.x, v.y, v.z, v.w};
  }
  for (int lanes = 1; lanes < W; lanes *= 2) step(lanes);
}

__device__ __forceinline__ float rstd_of(const Moments& m, float inv_c, float eps) {
  const float v = fmaf(m.m2, inv_c, eps), r = rsqrtf(v);
  return v > 0.f && v < INFINITY ? r * fmaf(-0.5f * v * r, r, 1.5f) : r;  // a Newton step: rsqrtf is off by up to 2 steps
}

template <int V, int NV>
__global__ void __launch_bounds__(kThreads) residual_norm_kernel(const Params p) {
  __shared__ float red[kRedFloats];
  int buf = 0;
  const Cols<V, NV> cols(p);
  const int row = blockIdx.x * blockDim.y + threadIdx.y;
  const bool live = row < p.rows;
  const size_t r = live ? row : 0;
  const float inv_c = 1.0f / static_cast<float>(p.C);
  float y[NV][V], x[NV][V];
  load_row<V, NV>(y, cols, p.y, p.dty, r * p.ldy, live);
  load_row<V, NV>(x, cols, p.x, p.dtx, r * p.ldx, live);
  if (p.post != kNone) normalise<V, NV>(y, cols, p.post, inv_c, p.eps, red, buf);
  const size_t item = r / p.L;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    if (!cols.in(k)) continue;
    float g[V], w[V];
    param<V>(p.gate, item * p.ldgate + cols.at(k), 1.f, g);
    param<V>(p.post_w, cols.at(k), 1.f, w);
#pragma unroll
    for (int i = 0; i < V; ++i) x[k][i] = fmaf(p.alpha * g[i], y[k][i] * w[i], x[k][i]);
    if (live) store<V>(p.o0, p.dtx, r * p.ldo0 + cols.at(k), x[k]);
  }
  normalise<V, NV>(x, cols, p.pre, inv_c, p.eps, red, buf);
  if (!live) return;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    if (!cols.in(k)) continue;
    float a[V], b[V], w[V];
    param<V>(p.scale, item * p.ldscale + cols.at(k), 0.f, a);
    param<V>(p.shift, item * p.ldshift + cols.at(k), 0.f, b);
    param<V>(p.pre_w, cols.at(k), 1.f, w);
#pragma unroll
    for (int i = 0; i < V; ++i) x[k][i] = fmaf(x[k][i] * w[i], 1.0f + a[i], b[i]);
    store<V>(p.o1, p.dth, r * p.ldo1 + cols.at(k), x[k]);
  }
}

// g -> r (g - mean(g) - n mean(g n)), the gradient through normalise()
template <int V, int NV>
__device__ __forceinline__ void normalise_back(float (&g)[NV][V], const float (&n)[NV][V], const Cols<V, NV>& cols,
                                               int kind, float r, float inv_c, float* red, int& buf) {
  float s[2] = {0.f, 0.f};
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      s[0] += g[k][i];
      s[1] = fmaf(g[k][i], n[k][i], s[1]);
    }
  row_sum(s, red, buf);
  const float mg = kind == kLayer ? s[0] * inv_c : 0.f, mgn = s[1] * inv_c;
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) g[k][i] = r * (g[k][i] - mg - n[k][i] * mgn);
}

// One block a part: part_rows rows of one item, blockDim.y at a time.
template <int V, int NV>
__global__ void __launch_bounds__(kThreads, NV * V <= 8 ? 2 : 1) residual_norm_grad_kernel(const Params p) {
  __shared__ float red[kRedFloats];
  int buf = 0;
  const Cols<V, NV> cols(p);
  const int item = blockIdx.x / p.parts, part = blockIdx.x % p.parts;
  const int first = part * p.part_rows, last = min(p.L, first + p.part_rows);
  const float inv_c = 1.0f / static_cast<float>(p.C);
  float sum[kMaxSums][NV][V];
#pragma unroll
  for (int s = 0; s < kMaxSums; ++s)
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) sum[s][k][i] = 0.f;
  for (int l0 = first; l0 < last; l0 += blockDim.y) {
    const int l = l0 + threadIdx.y;
    const bool live = l < last;
    const size_t r = static_cast<size_t>(item) * p.L + (live ? l : first);
    float x[NV][V], y[NV][V], dh[NV][V], dx[NV][V];
    load_row<V, NV>(x, cols, p.x, p.dtx, r * p.ldx, live);
    load_row<V, NV>(dh, cols, p.dh, p.dth, r * p.lddh, live);
    load_row<V, NV>(y, cols, p.y, p.dty, r * p.ldy, live);
    load_row<V, NV>(dx, cols, p.dx, p.dtx, r * p.lddx, live && p.dx);
    const float rx = normalise<V, NV>(x, cols, p.pre, inv_c, p.eps, red, buf);
    const float ry = p.post != kNone ? normalise<V, NV>(y, cols, p.post, inv_c, p.eps, red, buf) : 1.f;
    float w[V], a[V];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if (!live || !cols.in(k)) continue;
      param<V>(p.scale, static_cast<size_t>(item) * p.ldscale + cols.at(k), 0.f, a);
      param<V>(p.pre_w, cols.at(k), 1.f, w);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float t = dh[k][i] * x[k][i];
        sum[0][k][i] += dh[k][i];
        sum[1][k][i] = fmaf(t, w[i], sum[1][k][i]);
        sum[2][k][i] = fmaf(t, 1.0f + a[i], sum[2][k][i]);
        dh[k][i] *= (1.0f + a[i]) * w[i];
      }
    }
    normalise_back<V, NV>(dh, x, cols, p.pre, rx, inv_c, red, buf);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if (!live || !cols.in(k)) continue;
      float g[V];
      param<V>(p.gate, static_cast<size_t>(item) * p.ldgate + cols.at(k), 1.f, g);
      param<V>(p.post_w, cols.at(k), 1.f, w);
#pragma unroll
      for (int i = 0; i < V; ++i) dx[k][i] += dh[k][i];
      store<V>(p.o0, p.dtx, r * p.ldo0 + cols.at(k), dx[k]);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float t = p.alpha * dx[k][i] * y[k][i];
        sum[3][k][i] = fmaf(t, w[i], sum[3][k][i]);
        sum[4][k][i] = fmaf(t, g[i], sum[4][k][i]);
        dx[k][i] *= p.alpha * g[i] * w[i];
      }
    }
    if (p.post != kNone) normalise_back<V, NV>(dx, y, cols, p.post, ry, inv_c, red, buf);
    if (live) {
#pragma unroll
      for (int k = 0; k < NV; ++k)
        if (cols.in(k)) store<V>(p.o1, p.dty, r * p.ldo1 + cols.at(k), dx[k]);
    }
  }
  if (!p.sums) return;
  const int where[kMaxSums] = {p.s_shift, p.s_scale, p.s_prew, p.s_gate, p.s_postw};
  float* out = p.part + (static_cast<size_t>(blockIdx.x) * blockDim.y + threadIdx.y) * p.sums * p.C;
#pragma unroll
  for (int s = 0; s < kMaxSums; ++s) {
    if (where[s] < 0) continue;
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (cols.in(k)) store<V>(out, ANIMA_F32, static_cast<size_t>(where[s]) * p.C + cols.at(k), sum[s][k]);
  }
}

// A ring of rows in shared memory ahead of the row that a block works on: bulk copies of whole rows, one
// barrier a place. HBM answers in 1.5 to 2 us under load, so 90 KB have to be on their way to each SM;
// registers held one row ahead (49 KB), and the backward of 16384 x 2048 took 128 us for 121 so.
constexpr int kMaxPlaces = 3;
struct Stream {
  const void* p;
  long long ld;  // bytes
  uint32_t bytes;  // of a row
};
template <int N>
struct Ring {
  Stream in[N];
  uint8_t* smem;
  uint64_t* full;  // [places]
  volatile int* abort_flag;
  uint32_t row_bytes;
  uint32_t armed;  // of the fetching thread: bit k place k was used, bit 8 + k the phase of its last row

  // One thread: row r to its place (what was there has been read).
  __device__ __forceinline__ void fetch(int k, size_t r) {
    if (armed >> k & 1u) armed ^= 256u << k;
    armed |= 1u << k;
    mbar_arrive_expect_tx(&full[k], row_bytes);
    uint8_t* d = smem + k * row_bytes;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (!in[i].bytes) continue;
      bulk_load_1d(d, static_cast<const uint8_t*>(in[i].p) + r * in[i].ld, in[i].bytes, &full[k]);
      d += in[i].bytes;
    }
  }
  // The fetching thread, before the block ends: after a wait that ran out, copies may be in flight.
  __device__ __forceinline__ void drain() const {
    if (!*abort_flag) return;
    for (int k = 0; k < kMaxPlaces; ++k) {
      if (!(armed >> k & 1u)) continue;
      const unsigned long long t0 = globaltimer();
      while (!mbar_test(smem_u32(&full[k]), armed >> (8 + k) & 1u)) {
        if (globaltimer() - t0 > kWaitTimeoutNs) {
          flag_error(kErrTimeoutDrain);
          break;
        }
      }
    }
  }
  // After a wait that ran out nothing is stored any more, but every thread still meets every barrier.
  __device__ __forceinline__ bool wait(int k, uint32_t phase) const {
    return mbar_wait(&full[k], phase, abort_flag, kErrTimeoutFull);
  }
};

template <int N>
__device__ __forceinline__ Ring<N> make_ring(const Stream (&in)[N], uint8_t* smem, uint64_t* full, int* abort_flag,
                                             int places) {
  Ring<N> r;
  r.row_bytes = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    r.in[i] = in[i];
    r.row_bytes += in[i].bytes;
  }
  r.smem = smem;
  r.full = full;
  r.abort_flag = abort_flag;
  r.armed = 0;
  if (threadIdx.x == 0) {
    for (int k = 0; k < places; ++k) mbar_init(&full[k], 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  __syncthreads();
  return r;
}

__device__ __forceinline__ uint32_t size_of(int dt) { return dt == ANIMA_F32 ? 4 : 2; }

// 8 elements of a row in the ring.
__device__ __forceinline__ void load8(const uint8_t* row, int dt, int c, float (&v)[8]) {
  Raw<8> r;
  load_raw<8>(r, row, dt, c);
  unpack<8>(r, dt, v);
}

// A block's rows: part_rows of one item.
struct Share {
  int first, last;
  size_t item, row0;
};
__device__ __forceinline__ Share share_of(const Params& p) {
  Share s;
  const int item = blockIdx.x / p.parts, part = blockIdx.x % p.parts;
  s.item = item;
  s.row0 = static_cast<size_t>(item) * p.L;
  s.first = part * p.part_rows;
  s.last = min(p.L, s.first + p.part_rows);
  return s;
}

// The parameters of a thread's columns, in registers for all of a block's rows (read for each row they
// came from L2, the ring leaves no L1: 121 us for 115; with one branch for eight conversions it is 102, 90%
// of the copy rate, and the forward of 4096 x 2048 takes 18.7 us, 82%). MODS: there is a
// modulation (gate, scale or shift), WEIGHTS: a norm weight; what is not there costs no registers.
template <int NV, bool MODS, bool WEIGHTS>
struct Columns {
  float scale[NV][8], gate[NV][8], pre[NV][8], post[NV][8];  // 1 + scale, alpha gate
  float alpha;
  __device__ __forceinline__ Columns(const Params& p, size_t item, int c0, int step) : alpha(p.alpha) {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = c0 + k * step;
      if (MODS) {
        param<8>(p.scale, item * p.ldscale + c, 0.f, scale[k]);
        param<8>(p.gate, item * p.ldgate + c, 1.f, gate[k]);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          scale[k][i] += 1.f;
          gate[k][i] *= alpha;
        }
      }
      if (WEIGHTS) {
        param<8>(p.pre_w, c, 1.f, pre[k]);
        param<8>(p.post_w, c, 1.f, post[k]);
      }
    }
  }
  // v (1 + scale), v pre_w, v alpha gate, v post_w
  __device__ __forceinline__ float by_scale(float v, int k, int i) const { return MODS ? v * scale[k][i] : v; }
  __device__ __forceinline__ float by_pre(float v, int k, int i) const { return WEIGHTS ? v * pre[k][i] : v; }
  __device__ __forceinline__ float by_gate(float v, int k, int i) const { return MODS ? v * gate[k][i] : v * alpha; }
  __device__ __forceinline__ float by_post(float v, int k, int i) const { return WEIGHTS ? v * post[k][i] : v; }
};

// The forward where every thread holds 8 NV columns (256, 512, 1024, 2048 and 4096 of them in all): one
// round of moments a norm.
template <int NV, bool MODS, bool WEIGHTS>
__global__ void __launch_bounds__(kThreads, NV == 1 ? 3 : 2) residual_norm_full_kernel(const Params p) {
  extern __shared__ __align__(16) uint8_t ring_smem[];
  __shared__ float4 red[kRedMoments];
  __shared__ uint64_t full[kMaxPlaces];
  __shared__ int abort_flag;
  int buf = 0;
  const int step = blockDim.x * 8, c0 = threadIdx.x * 8;
  const Share w = share_of(p);
  const float inv_c = 1.0f / static_cast<float>(p.C);
  const Stream in[2] = {{p.x, p.ldx * size_of(p.dtx), p.C * size_of(p.dtx)},
                        {p.y, p.ldy * size_of(p.dty), p.C * size_of(p.dty)}};
  const int places = p.places;
  auto ring = make_ring<2>(in, ring_smem, full, &abort_flag, places);
  if (threadIdx.x == 0)
    for (int k = 0; k < places; ++k)
      if (w.first + k < w.last) ring.fetch(k, w.row0 + w.first + k);
  const Columns<NV, MODS, WEIGHTS> cols(p, w.item, c0, step);
  float shift[NV][8];
  if (MODS) {
#pragma unroll
    for (int k = 0; k < NV; ++k) param<8>(p.shift, w.item * p.ldshift + c0 + k * step, 0.f, shift[k]);
  }
  int place = 0, before = -1;
  uint32_t phase = 0;
  for (int l = w.first; l < w.last; ++l) {
    const bool live = ring.wait(place, phase);
    const uint8_t* at = ring.smem + place * ring.row_bytes;
    const size_t r = w.row0 + l;
    float x[NV][8], y[NV][8];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      load8(at, p.dtx, c0 + k * step, x[k]);
      load8(at + in[0].bytes, p.dty, c0 + k * step, y[k]);
    }
    if (p.post != kNone) {
      Moments m[1] = {moments_of<NV>(y, nullptr, p.post)};
      row_moments<1, false>(m, 8 * NV, red, buf);
      const float rs = rstd_of(m[0], inv_c, p.eps);
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < 8; ++i) y[k][i] = (y[k][i] - m[0].mean) * rs;
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[k][i] += cols.by_gate(cols.by_post(y[k][i], k, i), k, i);
      if (live) store<8>(p.o0, p.dtx, r * p.ldo0 + c0 + k * step, x[k]);
    }
    Moments m[1] = {moments_of<NV>(x, nullptr, p.pre)};
    row_moments<1, false>(m, 8 * NV, red, buf);
    __syncwarp();
    // a barrier (one warp: an exchange) behind the last reads of the place before: its next row
    if (threadIdx.x == 0 && before >= 0 && l - 1 + places < w.last && !abort_flag) ring.fetch(before, r - 1 + places);
    before = place;
    if (++place == places) place = 0, phase ^= 1;
    const float rs = rstd_of(m[0], inv_c, p.eps);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float n = cols.by_pre((x[k][i] - m[0].mean) * rs, k, i);
        x[k][i] = MODS ? fmaf(n, cols.scale[k][i], shift[k][i]) : n;
      }
      if (live) store<8>(p.o1, p.dth, r * p.ldo1 + c0 + k * step, x[k]);
    }
  }
  if (threadIdx.x == 0) ring.drain();
}

// The backward there. A row's statistics and the sums of the pre-norm's gradient come from one round.
template <int NV, bool MODS, bool WEIGHTS>
__global__ void __launch_bounds__(kThreads, 2) residual_norm_grad_full_kernel(const Params p) {
  extern __shared__ __align__(16) uint8_t ring_smem[];
  __shared__ float4 red[kRedMoments];
  __shared__ float red2[kRedFloats];  // of row_sum
  __shared__ uint64_t full[kMaxPlaces];
  __shared__ int abort_flag;
  int buf = 0, buf2 = 0;
  const int step = blockDim.x * 8, c0 = threadIdx.x * 8;
  const Share w = share_of(p);
  const float inv_c = 1.0f / static_cast<float>(p.C);
  const Stream in[4] = {{p.x, p.ldx * size_of(p.dtx), p.C * size_of(p.dtx)},
                        {p.dh, p.lddh * size_of(p.dth), p.C * size_of(p.dth)},
                        {p.y, p.ldy * size_of(p.dty), p.C * size_of(p.dty)},
                        {p.dx, p.lddx * size_of(p.dtx), p.dx ? p.C * size_of(p.dtx) : 0u}};
  const int places = p.places;
  auto ring = make_ring<4>(in, ring_smem, full, &abort_flag, places);
  const uint32_t off_h = in[0].bytes, off_y = off_h + in[1].bytes, off_d = off_y + in[2].bytes;
  if (threadIdx.x == 0)
    for (int k = 0; k < places; ++k)
      if (w.first + k < w.last) ring.fetch(k, w.row0 + w.first + k);
  const Columns<NV, MODS, WEIGHTS> cols(p, w.item, c0, step);
  float s_shift[NV][8], s_scale[NV][8], s_gate[NV][8], s_prew[NV][8], s_postw[NV][8];
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int i = 0; i < 8; ++i) s_shift[k][i] = s_scale[k][i] = s_gate[k][i] = s_prew[k][i] = s_postw[k][i] = 0.f;
  int place = 0, before = -1;
  uint32_t phase = 0;
  for (int l = w.first; l < w.last; ++l) {
    const bool live = ring.wait(place, phase);
    const uint8_t* at = ring.smem + place * ring.row_bytes;
    const size_t r = w.row0 + l;
    float x[NV][8], h[NV][8], y[NV][8];
    Moments m[2];
    {
      float g[NV][8];  // the gradient of n
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        load8(at, p.dtx, c0 + k * step, x[k]);
        load8(at + off_h, p.dth, c0 + k * step, h[k]);
#pragma unroll
        for (int i = 0; i < 8; ++i) g[k][i] = cols.by_pre(cols.by_scale(h[k][i], k, i), k, i);
      }
      m[0] = moments_of<NV>(x, g, p.pre);
    }
    float rs_y = 1.f;
    m[1].mean = 0.f;
    if (p.post != kNone) {
#pragma unroll
      for (int k = 0; k < NV; ++k) load8(at + off_y, p.dty, c0 + k * step, y[k]);
      m[1] = moments_of<NV>(y, nullptr, p.post);
      row_moments<2, true>(m, 8 * NV, red, buf);
      rs_y = rstd_of(m[1], inv_c, p.eps);
    } else {
      Moments m1[1] = {m[0]};
      row_moments<1, true>(m1, 8 * NV, red, buf);
      m[0] = m1[0];
#pragma unroll
      for (int k = 0; k < NV; ++k) load8(at + off_y, p.dty, c0 + k * step, y[k]);
    }
    __syncwarp();
    // a barrier (one warp: an exchange) behind the last reads of the place before: its next row
    if (threadIdx.x == 0 && before >= 0 && l - 1 + places < w.last && !abort_flag) ring.fetch(before, r - 1 + places);
    before = place;
    if (++place == places) place = 0, phase ^= 1;
    const float rs = rstd_of(m[0], inv_c, p.eps);
    const float mg = p.pre == kLayer ? m[0].g * inv_c * rs : 0.f, mgn = m[0].gt * rs * rs * inv_c;
    float s2[2] = {0.f, 0.f};
    float d[NV][8];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if (p.dx) {
        load8(at + off_d, p.dtx, c0 + k * step, d[k]);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) d[k][i] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float n = (x[k][i] - m[0].mean) * rs, hp = cols.by_pre(h[k][i], k, i), hs = cols.by_scale(h[k][i], k, i);
        if (MODS) {
          s_shift[k][i] += h[k][i];
          s_scale[k][i] = fmaf(hp, n, s_scale[k][i]);
        }
        if (WEIGHTS) s_prew[k][i] = fmaf(hs, n, s_prew[k][i]);
        // dx' + rs (g - mean(g) - n mean(g n))
        d[k][i] += fmaf(rs, cols.by_pre(hs, k, i), -fmaf(n, mgn, mg));
      }
      if (live) store<8>(p.o0, p.dtx, r * p.ldo0 + c0 + k * step, d[k]);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float u = (y[k][i] - m[1].mean) * rs_y;
        if (MODS) s_gate[k][i] = fmaf(cols.alpha * cols.by_post(d[k][i], k, i), u, s_gate[k][i]);
        const float t = cols.by_gate(d[k][i], k, i);
        if (WEIGHTS) s_postw[k][i] = fmaf(t, u, s_postw[k][i]);
        d[k][i] = cols.by_post(t, k, i);
        if (p.post != kNone) {
          y[k][i] = u;
          s2[0] += d[k][i];
          s2[1] = fmaf(d[k][i], u, s2[1]);
        }
      }
      if (p.post == kNone && live) store<8>(p.o1, p.dty, r * p.ldo1 + c0 + k * step, d[k]);
    }
    if (p.post != kNone) {
      row_sum(s2, red2, buf2);
      const float m0 = p.post == kLayer ? s2[0] * inv_c : 0.f, m1 = s2[1] * inv_c;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
#pragma unroll
        for (int i = 0; i < 8; ++i) d[k][i] = rs_y * (d[k][i] - m0 - y[k][i] * m1);
        if (live) store<8>(p.o1, p.dty, r * p.ldo1 + c0 + k * step, d[k]);
      }
    }
  }
  if (threadIdx.x == 0) ring.drain();
  if (!p.sums) return;
  float* out = p.part + static_cast<size_t>(blockIdx.x) * p.sums * p.C + c0;
  auto put = [&](int where, const float(&v)[NV][8]) {
    if (where < 0) return;
#pragma unroll
    for (int k = 0; k < NV; ++k) store<8>(out, ANIMA_F32, static_cast<size_t>(where) * p.C + k * step, v[k]);
  };
  if (MODS) {
    put(p.s_shift, s_shift);
    put(p.s_scale, s_scale);
    put(p.s_gate, s_gate);
  }
  if (WEIGHTS) {
    put(p.s_prew, s_prew);
    put(p.s_postw, s_postw);
  }
}

struct SumParams {
  const float* part;  // [items][parts][sums][C]
  int items, parts, sums, C;
  float* out[kMaxSums];
  int per_item[kMaxSums];  // out [items][C], else [C] over all items
  unsigned end[kMaxSums];  // the block behind the sum's last
};

// out = the partial rows added in a fixed order. A block takes 32 columns of one output row (the sums' rows one
// after another: an item is no grid axis of its own, which would end at 65535); its warps each add every
// blockDim.y-th partial, then the first adds the warps' sums.
__global__ void __launch_bounds__(1024) partial_sum_kernel(const SumParams p) {
  __shared__ float red[32][32];
  int s = 0;
  while (blockIdx.x >= p.end[s]) ++s;
  const unsigned at = blockIdx.x - (s ? p.end[s - 1] : 0u), column_blocks = (p.C + 31) / 32;
  const unsigned item = at / column_blocks;
  const int c = (at - item * column_blocks) * 32 + threadIdx.x, warps = blockDim.y;
  const size_t n = static_cast<size_t>(p.parts) * (p.per_item[s] ? 1 : p.items);
  const size_t stride = static_cast<size_t>(p.sums) * p.C;
  const float* base = p.part + (static_cast<size_t>(item) * p.parts * p.sums + s) * p.C + c;
  float t = 0.f;
  if (c < p.C) {
#pragma unroll 4
    for (size_t i = threadIdx.y; i < n; i += warps) t += base[i * stride];
  }
  red[threadIdx.y][threadIdx.x] = t;
  __syncthreads();
  if (threadIdx.y || c >= p.C) return;
  t = 0.f;
  for (int i = 0; i < warps; ++i) t += red[i][threadIdx.x];
  p.out[s][static_cast<size_t>(item) * p.C + c] = t;
}

struct Shape {
  int V, NV, T, Y;  // columns a vector, vectors a thread, threads a row, rows a block
  bool full;        // every thread holds 8 NV columns, and the warps merge in pairs: the kernels with a ring
};

Shape shape_of(int C, bool vec) {
  Shape s;
  s.V = vec && C % 8 == 0 ? 8 : 1;
  const int n = C / s.V;
  s.NV = 1;
  while (static_cast<long long>(s.NV) * kThreads < n) s.NV *= 2;
  if (s.V == 1) s.NV = s.NV <= 8 ? 8 : 16;
  s.T = ((n + s.NV - 1) / s.NV + 31) / 32 * 32;
  s.full = s.V == 8 && (C == 256 || C == 512 || C == 1024 || C == 2048 || C == 4096);
  s.Y = s.full ? 1 : kThreads / s.T;
  return s;
}

// Rows of one item that a block takes, with as many blocks as `threads` of them an SM make, or one row each
// where there are not as many rows. Up to 2048 columns the SMs hold them all at once. At 4096 they do not: the
// forward's registers let two blocks of its three in (a wave and a half), and two places of four fp32 streams,
// 128 KB, one block of the backward's two.
void parts_of(const Shape& s, int items, int L, int sms, int threads, int& parts, int& part_rows) {
  const int blocks = threads / (s.T * s.Y) < 16 ? threads / (s.T * s.Y) : 16;
  const int want = blocks * sms / items > 1 ? blocks * sms / items : 1;  // (a block past a whole wave would double it)
  const int most = (L + s.Y - 1) / s.Y;
  parts = want < most ? want : most;
  part_rows = ((L + parts - 1) / parts + s.Y - 1) / s.Y * s.Y;
  parts = (L + part_rows - 1) / part_rows;
}
constexpr int kGradThreads = 512, kForwardThreads = 768;  // an SM, by the launch bounds up to 2048 columns

// Places of a ring: three, or two where three would leave an SM with fewer blocks than that.
int places_of(const Shape& s, int threads, int row_bytes) { return kMaxPlaces * row_bytes * (threads / s.T) <= 208 * 1024 ? kMaxPlaces : 2; }
int size_of_host(int dt) { return dt == ANIMA_F32 ? 4 : 2; }

int count_sums(const anima_residual_norm_args* a) {
  return (a->dshift != nullptr) + (a->dscale != nullptr) + (a->dpre_w != nullptr) + (a->dgate != nullptr) +
         (a->dpost_w != nullptr);
}

int check(const char* fn, const anima_residual_norm_args* a, bool grad) {
  ANIMA_REQUIRE(a->rows >= 0 && a->rows <= 1 << 30 && a->cols > 0 && a->cols <= kMaxCols, "%s: %d rows of %d columns (at most 2^30 of %d)", fn,
                a->rows, a->cols, kMaxCols);
  ANIMA_REQUIRE(a->rows_per_item > 0 && a->rows % a->rows_per_item == 0, "%s: %d rows are not items of %d rows", fn,
                a->rows, a->rows_per_item);
  for (const int dt : {a->x_dtype, a->y_dtype, a->h_dtype})
    ANIMA_REQUIRE(dt == ANIMA_F32 || dt == ANIMA_BF16 || dt == ANIMA_F16, "%s: dtype %d", fn, dt);
  ANIMA_REQUIRE(a->post >= kNone && a->post <= kLayer, "%s: post norm %d (0 none, 1 rms, 2 layer)", fn, a->post);
  ANIMA_REQUIRE(a->pre == kRms || a->pre == kLayer, "%s: pre norm %d (1 rms, 2 layer)", fn, a->pre);
  ANIMA_REQUIRE(a->eps >= 0.f, "%s: eps %g", fn, a->eps);
  ANIMA_REQUIRE(!a->post_w || a->post != kNone, "%s: post_w without a post norm", fn);
  if (a->rows == 0) return ANIMA_OK;
  ANIMA_REQUIRE(a->x_out && a->y, "%s: NULL data pointer", fn);
  ANIMA_REQUIRE(a->ldx_out >= a->cols && a->ldy >= a->cols, "%s: a row stride is below %d columns", fn, a->cols);
  for (const long long ld : {a->gate ? a->ld_gate : 0LL, a->scale ? a->ld_scale : 0LL, a->shift ? a->ld_shift : 0LL})
    ANIMA_REQUIRE(ld >= 0, "%s: negative stride of a modulation", fn);
  if (!grad) {
    ANIMA_REQUIRE(a->x && a->h && a->ldx >= a->cols && a->ldh >= a->cols, "%s: x or h is NULL or its stride too small",
                  fn);
    return ANIMA_OK;
  }
  ANIMA_REQUIRE(a->dh && a->dx && a->dy, "%s: dh, dx or dy is NULL", fn);
  ANIMA_REQUIRE(a->lddh >= a->cols && a->lddx >= a->cols && a->lddy >= a->cols &&
                    (!a->dx_out || a->lddx_out >= a->cols),
                "%s: a row stride is below %d columns", fn, a->cols);
  ANIMA_REQUIRE((!a->dgate || a->gate) && (!a->dscale || a->scale) && (!a->dshift || a->shift) &&
                    (!a->dpost_w || a->post_w) && (!a->dpre_w || a->pre_w),
                "%s: a gradient is asked for whose parameter is NULL", fn);
  return ANIMA_OK;
}

bool aligned(const void* p, int dt, long long ld) {
  return !p || (reinterpret_cast<uintptr_t>(p) % 16 == 0 && (ld * (dt == ANIMA_F32 ? 4 : 2)) % 16 == 0);
}

// Whether every tensor can be read and written in 16-byte vectors of a row.
bool vectors_ok(const anima_residual_norm_args* a, bool grad) {
  const int f = ANIMA_F32;
  bool ok = aligned(a->y, a->y_dtype, a->ldy) && aligned(a->x_out, a->x_dtype, a->ldx_out) &&
            aligned(a->gate, f, a->ld_gate) && aligned(a->scale, f, a->ld_scale) && aligned(a->shift, f, a->ld_shift) &&
            aligned(a->post_w, f, 0) && aligned(a->pre_w, f, 0);
  if (!grad) return ok && aligned(a->x, a->x_dtype, a->ldx) && aligned(a->h, a->h_dtype, a->ldh);
  return ok && aligned(a->dh, a->h_dtype, a->lddh) && aligned(a->dx_out, a->x_dtype, a->lddx_out) &&
         aligned(a->dx, a->x_dtype, a->lddx) && aligned(a->dy, a->y_dtype, a->lddy) && aligned(a->workspace, f, 0);
}

void fill(Params& p, const anima_residual_norm_args* a) {
  p.y = a->y;
  p.ldy = a->ldy;
  p.dtx = a->x_dtype;
  p.dty = a->y_dtype;
  p.dth = a->h_dtype;
  p.rows = a->rows;
  p.C = a->cols;
  p.L = a->rows_per_item;
  p.post = a->post;
  p.pre = a->pre;
  p.alpha = a->alpha;
  p.eps = a->eps;
  p.gate = a->gate;
  p.scale = a->scale;
  p.shift = a->shift;
  p.post_w = a->post_w;
  p.pre_w = a->pre_w;
  p.ldgate = a->ld_gate;
  p.ldscale = a->ld_scale;
  p.ldshift = a->ld_shift;
}

using Kernel = void (*)(const Params);

}  // namespace resnorm
}  // namespace anima

extern "C" int anima_residual_norm(anima_ctx* ctx, const anima_residual_norm_args* a) {
  using namespace anima::resnorm;
  ANIMA_REQUIRE(ctx && a, "anima_residual_norm: NULL argument");
  ANIMA_ON_DEVICE(ctx);
  int st = check("anima_residual_norm", a, false);
  if (st || a->rows == 0) return st;
  const Shape s = shape_of(a->cols, vectors_ok(a, false));
  Params p{};
  fill(p, a);
  p.x = a->x;
  p.ldx = a->ldx;
  p.o0 = a->x_out;
  p.ldo0 = a->ldx_out;
  p.o1 = a->h;
  p.ldo1 = a->ldh;
  Kernel fn = s.V == 8 ? (s.NV == 1 ? residual_norm_kernel<8, 1> : residual_norm_kernel<8, 2>)
                       : (s.NV == 8 ? residual_norm_kernel<1, 8> : residual_norm_kernel<1, 16>);
  long long grid = (static_cast<long long>(a->rows) + s.Y - 1) / s.Y;
  int smem = 0;
  if (s.full) {
    const Kernel fns[2][2][2] = {{{residual_norm_full_kernel<1, false, false>, residual_norm_full_kernel<1, false, true>},
                                  {residual_norm_full_kernel<1, true, false>, residual_norm_full_kernel<1, true, true>}},
                                 {{residual_norm_full_kernel<2, false, false>, residual_norm_full_kernel<2, false, true>},
                                  {residual_norm_full_kernel<2, true, false>, residual_norm_full_kernel<2, true, true>}}};
    fn = fns[s.NV - 1][a->gate || a->scale || a->shift][a->pre_w || a->post_w];
    const int items = a->rows / a->rows_per_item;
    parts_of(s, items, a->rows_per_item, ctx->num_sms, kForwardThreads, p.parts, p.part_rows);
    grid = static_cast<long long>(items) * p.parts;
    ANIMA_REQUIRE(grid < (1LL << 31), "anima_residual_norm: %d items are too many", items);
    const int row = a->cols * (size_of_host(a->x_dtype) + size_of_host(a->y_dtype));
    p.places = places_of(s, kForwardThreads, row);
    smem = p.places * row;
    st = set_max_dynamic_smem(reinterpret_cast<const void*>(fn), kMaxPlaces * kMaxCols * 8);
    if (st) return st;
  }
  ProfScope prof(ctx, "residual_norm", 0, static_cast<double>(a->rows) * a->cols * 12);
  fn<<<static_cast<unsigned>(grid), dim3(s.T, s.Y), smem, ctx->stream>>>(p);
  return check_launch("residual_norm_kernel");
}

extern "C" int anima_residual_norm_backward_workspace(anima_ctx* ctx, const anima_residual_norm_args* a, size_t* bytes) {
  using namespace anima::resnorm;
  ANIMA_REQUIRE(ctx && a && bytes, "anima_residual_norm_backward_workspace: NULL argument");
  *bytes = 0;
  int st = check("anima_residual_norm_backward_workspace", a, true);
  if (st || a->rows == 0) return st;
  // the larger of the two shapes, so that the answer does not depend on alignments
  for (const bool vec : {false, true}) {
    const Shape s = shape_of(a->cols, vec);
    int parts, part_rows;
    parts_of(s, a->rows / a->rows_per_item, a->rows_per_item, ctx->num_sms, kGradThreads, parts, part_rows);
    const size_t n = static_cast<size_t>(a->rows / a->rows_per_item) * parts * s.Y * count_sums(a) * a->cols * 4;
    if (n > *bytes) *bytes = n;
  }
  return ANIMA_OK;
}

extern "C" int anima_residual_norm_backward(anima_ctx* ctx, const anima_residual_norm_args* a) {
  using namespace anima::resnorm;
  ANIMA_REQUIRE(ctx && a, "anima_residual_norm_backward: NULL argument");
  ANIMA_ON_DEVICE(ctx);
  int st = check("anima_residual_norm_backward", a, true);
  if (st || a->rows == 0) return st;
  const int items = a->rows / a->rows_per_item;
  const Shape s = shape_of(a->cols, vectors_ok(a, true));
  Params p{};
  fill(p, a);
  p.x = a->x_out;
  p.ldx = a->ldx_out;
  p.dh = a->dh;
  p.lddh = a->lddh;
  p.dx = a->dx_out;
  p.lddx = a->lddx_out;
  p.o0 = a->dx;
  p.ldo0 = a->lddx;
  p.o1 = a->dy;
  p.ldo1 = a->lddy;
  parts_of(s, items, a->rows_per_item, ctx->num_sms, kGradThreads, p.parts, p.part_rows);
  p.sums = count_sums(a);
  const size_t need = static_cast<size_t>(items) * p.parts * s.Y * p.sums * a->cols * 4;
  ANIMA_REQUIRE(need == 0 || (a->workspace && a->workspace_bytes >= need),
                "anima_residual_norm_backward: a workspace of %zu bytes is needed, %zu are given", need,
                a->workspace ? a->workspace_bytes : 0);
  p.part = static_cast<float*>(a->workspace);
  SumParams sp{};
  int k = 0;
  auto slot = [&](float* out, bool per_item) {
    if (!out) return -1;
    sp.out[k] = out;
    sp.per_item[k] = per_item;
    return k++;
  };
  p.s_shift = slot(a->dshift, true);
  p.s_scale = slot(a->dscale, true);
  p.s_gate = slot(a->dgate, true);
  p.s_prew = slot(a->dpre_w, false);
  p.s_postw = slot(a->dpost_w, false);
  const bool mods = a->gate || a->scale || a->shift, weights = a->pre_w || a->post_w;
  Kernel fn = s.V == 8 ? (s.NV == 1 ? residual_norm_grad_kernel<8, 1> : residual_norm_grad_kernel<8, 2>)
                       : (s.NV == 8 ? residual_norm_grad_kernel<1, 8> : residual_norm_grad_kernel<1, 16>);
  int smem = 0;
  if (s.full) {
    const Kernel fns[2][2][2] = {{{residual_norm_grad_full_kernel<1, false, false>, residual_norm_grad_full_kernel<1, false, true>},
                                  {residual_norm_grad_full_kernel<1, true, false>, residual_norm_grad_full_kernel<1, true, true>}},
                                 {{residual_norm_grad_full_kernel<2, false, false>, residual_norm_grad_full_kernel<2, false, true>},
                                  {residual_norm_grad_full_kernel<2, true, false>, residual_norm_grad_full_kernel<2, true, true>}}};
    fn = fns[s.NV - 1][a->gate || a->scale || a->shift][a->pre_w || a->post_w];
    const int row = a->cols * (size_of_host(a->x_dtype) * (a->dx_out ? 2 : 1) + size_of_host(a->y_dtype) + size_of_host(a->h_dtype));
    p.places = places_of(s, kGradThreads, row);
    smem = p.places * row;
    st = set_max_dynamic_smem(reinterpret_cast<const void*>(fn), 2 * kMaxCols * 16);
    if (st) return st;
  }
  long long blocks = 0;  // of the sums
  for (int i = 0; i < k; ++i) {
    blocks += static_cast<long long>((a->cols + 31) / 32) * (sp.per_item[i] ? items : 1);
    sp.end[i] = static_cast<unsigned>(blocks);
  }
  ANIMA_REQUIRE(static_cast<long long>(items) * p.parts < (1LL << 31) && blocks < (1LL << 31),
                "anima_residual_norm_backward: %d items are too many", items);
  ProfScope prof(ctx, "residual_norm.grad", 0, static_cast<double>(a->rows) * a->cols * 20);
  fn<<<items * p.parts, dim3(s.T, s.Y), smem, ctx->stream>>>(p);
  st = check_launch("residual_norm_grad_kernel");
  if (st || p.sums == 0) return st;
  sp.part = p.part;
  sp.items = items;
  sp.parts = p.parts * s.Y;
  sp.sums = p.sums;
  sp.C = a->cols;
  // (32 warps for a sum over more partials than two blocks an SM leave: with 8 each would add dozens in turn)
  const bool many = static_cast<long long>(sp.parts) * items > 2LL * ctx->num_sms;
  partial_sum_kernel<<<static_cast<unsigned>(blocks), dim3(32, many ? 32 : 8), 0, ctx->stream>>>(sp);
  return check_launch("partial_sum_kernel");
}
