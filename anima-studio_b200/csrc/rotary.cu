// Rotary positions on q and k in one launch: both pair layouts, part of a head, angles in 64 bits
// from positions and inverse frequencies, and the inverse rotation (the gradient's). The table form
// that the DiT and the text models use is anima_rope.
//
// A pair (x0, x1) of one head's first R dims at position p and inverse frequency f becomes
//   y0 = m (x0 cos pf - x1 sin pf),  y1 = m (x1 cos pf + x0 sin pf);
// the inverse turns by -pf (its transpose, so the gradient of y is mapped to that of x). The angle is
// taken in turns, t = p f / (2 pi) in 64 bits, less its nearest whole number, and only then rounded to
// 32 bits: at p = 2^31 the fraction still has 2^-24 turns, where a 32-bit angle would be noise.
//
// Bound by HBM: each element is read and written once. A thread owns two 16-byte vectors that hold
// whole pairs (half layout: dims e.. and R/2 + e..; interleaved: 2 adjacent vectors) of one row, in four
// heads, and issues its eight loads first. Meanwhile the block's threads share the angles of its rows, one
// sine and cosine each. 8192 rows of 32 heads of 128 in fp16 take 24.1 us (a device copy 24.8): 34 with
// 16-bit values converted one by one, which the conversion unit does at a quarter of the rate, 38 to 51
// with fewer heads a thread; 16381 rows of 24 heads in fp32 take 66 us.

#include "internal.h"
#include "sm100.cuh"

namespace anima {
namespace rotary {

struct Side {
  const void* x;
  void* y;
  long long ldx, ldy;
};

struct Params {
  Side q, k;
  const double* inv_freq;  // [R / 2]
  const int* positions;    // [rows], or NULL: offset + row % rows_per_item
  long long offset;
  int rows, rows_per_item;
  int Hq, Hk, D, R;
  int interleaved, inverse, in_place_rest;  // in_place_rest: y is x on both sides, the rest of a head stays
  float mscale;
  int units;  // per (row, head): a rotated unit holds V pairs, a copied one 2 V elements
  int rot_units;
  int q_chunks, chunks;  // of kHeads heads: q's, all
};

template <typename T>
__device__ __forceinline__ float ld1(T v);
template <>
__device__ __forceinline__ float ld1<float>(float v) { return v; }
template <>
__device__ __forceinline__ float ld1<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float ld1<__half>(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T st1(float v);
template <>
__device__ __forceinline__ float st1<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 st1<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half st1<__half>(float v) { return __float2half_rn(v); }

template <typename T, int V>
struct Vec {  // V elements that are converted one by one
  T e[V];
  __device__ __forceinline__ void get(float* x) const {
#pragma unroll
    for (int j = 0; j < V; ++j) x[j] = ld1<T>(e[j]);
  }
  __device__ __forceinline__ void set(const float* x) {
#pragma unroll
    for (int j = 0; j < V; ++j) e[j] = st1<T>(x[j]);
  }
};
template <>
struct alignas(16) Vec<float, 4> {
  float e[4];
  __device__ __forceinline__ void get(float* x) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = e[j];
  }
  __device__ __forceinline__ void set(const float* x) {
#pragma unroll
    for (int j = 0; j < 4; ++j) e[j] = x[j];
  }
};
// 16-bit elements as they lie in four words, converted in pairs.
template <>
struct alignas(16) Vec<__half, 8> {
  uint32_t w[4];
  __device__ __forceinline__ void get(float* x) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
      x[2 * j] = f.x;
      x[2 * j + 1] = f.y;
    }
  }
  __device__ __forceinline__ void set(const float* x) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const __half2 h = __floats2half2_rn(x[2 * j], x[2 * j + 1]);
      w[j] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
};
template <>
struct alignas(16) Vec<__nv_bfloat16, 8> {
  uint32_t w[4];
  __device__ __forceinline__ void get(float* x) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[2 * j] = __uint_as_float(w[j] << 16);
      x[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
    }
  }
  __device__ __forceinline__ void set(const float* x) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * j], x[2 * j + 1]);
      w[j] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
};

// cos and sin of position * frequency, times m.
__device__ __forceinline__ void angle(double pos, double f, float m, bool inverse, float& c, float& s) {
  double t = pos * f * 0.15915494309189533577;  // 1 / (2 pi)
  t -= rint(t);
  sincospif(2.0f * static_cast<float>(t), &s, &c);
  c *= m;
  s *= inverse ? -m : m;
}

// y0 = x0 c - x1 s, y1 = x1 c + x0 s of N pairs, two at a time where there are two. The sums' order is
// written out, so that every form of the kernel rounds alike.
template <int N>
__device__ __forceinline__ void turn(const float* x0, const float* x1, const float* c, const float* s, float* y0, float* y1) {
  if constexpr (N % 2 == 0) {
#pragma unroll
    for (int j = 0; j < N; j += 2) {
      const f2 a = make_float2(x0[j], x0[j + 1]), b = make_float2(x1[j], x1[j + 1]), cj = make_float2(c[j], c[j + 1]),
               sj = make_float2(s[j], s[j + 1]), ms = make_float2(-s[j], -s[j + 1]);
      const f2 u = fma2(a, cj, mul2(b, ms)), v = fma2(b, cj, mul2(a, sj));
      y0[j] = u.x;
      y0[j + 1] = u.y;
      y1[j] = v.x;
      y1[j + 1] = v.y;
    }
  } else {
    y0[0] = fmaf(x0[0], c[0], __fmul_rn(x1[0], -s[0]));
    y1[0] = fmaf(x1[0], c[0], __fmul_rn(x0[0], s[0]));
  }
}

constexpr int kHeads = 4;  // heads of one thread, their loads in flight together
constexpr int kThreads = 256;
constexpr int kAngles = 2048;

// A thread's two vectors in up to kHeads heads, all of q or all of k.
template <typename T, int V>
struct Item {
  Vec<T, V> a[kHeads], b[kHeads];
  T* dst;
  int u, heads, e0, e1;
  bool live, two;  // two: V = 1, a copied unit at an odd end has one element

  __device__ __forceinline__ void load(const Params& p, int row, int chunk, int unit) {
    u = unit;
    const bool rot = u < p.rot_units;
    live = row < p.rows && (rot || !p.in_place_rest);
    if (!live) return;
    const bool is_q = chunk < p.q_chunks;
    const Side& sd = is_q ? p.q : p.k;
    const int h0 = (is_q ? chunk : chunk - p.q_chunks) * kHeads;
    heads = min(kHeads, (is_q ? p.Hq : p.Hk) - h0);
    e0 = !rot ? p.R + (u - p.rot_units) * 2 * V : p.interleaved ? u * 2 * V : u * V;
    e1 = e0 + (rot && !p.interleaved ? p.R / 2 : V);
    two = e1 < p.D;
    const long long col = static_cast<long long>(h0) * p.D;
    const T* src = static_cast<const T*>(sd.x) + row * sd.ldx + col;
    dst = static_cast<T*>(sd.y) + row * sd.ldy + col;
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
      if (i >= heads) continue;
      a[i] = *reinterpret_cast<const Vec<T, V>*>(src + i * p.D + e0);
      if (two) b[i] = *reinterpret_cast<const Vec<T, V>*>(src + i * p.D + e1);
    }
  }

  // cos, sin: the row's tables
  __device__ __forceinline__ void turn_and_store(const Params& p, const float* cos, const float* sin) {
    if (!live) return;
    const bool rot = u < p.rot_units;
    float c[V], s[V];
    if (rot) {
      // (V > 1: u V is a whole number of vectors, and so is a row's table)
      if constexpr (V >= 4) {
#pragma unroll
        for (int j = 0; j < V; j += 4) {
          const float4 cv = *reinterpret_cast<const float4*>(cos + u * V + j), sv = *reinterpret_cast<const float4*>(sin + u * V + j);
          c[j] = cv.x; c[j + 1] = cv.y; c[j + 2] = cv.z; c[j + 3] = cv.w;
          s[j] = sv.x; s[j + 1] = sv.y; s[j + 2] = sv.z; s[j + 3] = sv.w;
        }
      } else {
        c[0] = cos[u];
        s[0] = sin[u];
      }
    }
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
      if (i >= heads) continue;
      if (rot) {
        float x[2 * V], y[2 * V];
        a[i].get(x);
        b[i].get(x + V);
        if (p.interleaved) {
          float x0[V], x1[V], y0[V], y1[V];
#pragma unroll
          for (int j = 0; j < V; ++j) {
            x0[j] = x[2 * j];
            x1[j] = x[2 * j + 1];
          }
          turn<V>(x0, x1, c, s, y0, y1);
#pragma unroll
          for (int j = 0; j < V; ++j) {
            y[2 * j] = y0[j];
            y[2 * j + 1] = y1[j];
          }
        } else {
          turn<V>(x, x + V, c, s, y, y + V);
        }
        a[i].set(y);
        b[i].set(y + V);
      }
      *reinterpret_cast<Vec<T, V>*>(dst + i * p.D + e0) = a[i];
      if (two) *reinterpret_cast<Vec<T, V>*>(dst + i * p.D + e1) = b[i];
    }
  }
};

// V = 16 bytes of elements, or 1 where sizes or alignment do not allow vectors.
// A block's threads: (unit, chunk of heads, row), so that no index takes a division.
template <typename T, int V>
__global__ void __launch_bounds__(kThreads, 3) rotary_kernel(const Params p) {
  __shared__ __align__(16) float cos[kAngles], sin[kAngles];
  const int row = blockIdx.x * blockDim.z + threadIdx.z, half = p.R / 2, at = threadIdx.z * half;
  Item<T, V> it;
  it.load(p, row, threadIdx.y, threadIdx.x);
  if (row < p.rows) {
    const double pos = p.positions ? static_cast<double>(p.positions[row])
                                   : static_cast<double>(p.offset + row % p.rows_per_item);
    for (int j = threadIdx.y * blockDim.x + threadIdx.x; j < half; j += blockDim.x * blockDim.y)
      angle(pos, p.inv_freq[j], p.mscale, p.inverse != 0, cos[at + j], sin[at + j]);
  }
  __syncthreads();
  for (int chunk = threadIdx.y; chunk < p.chunks; chunk += blockDim.y)
    for (int u = threadIdx.x; u < p.units; u += blockDim.x) {
      if (u != static_cast<int>(threadIdx.x) || chunk != static_cast<int>(threadIdx.y)) it.load(p, row, chunk, u);
      it.turn_and_store(p, cos + at, sin + at);
    }
}

template <typename T>
int launch(anima_ctx* ctx, Params& p, bool vec_ok) {
  constexpr int V = 16 / static_cast<int>(sizeof(T));
  // whole vectors: the pairs of a unit fill both of its vectors, and so do the copied dims
  const bool vec = vec_ok && p.D % V == 0 && (p.interleaved ? p.R % (2 * V) == 0 : (p.R / 2) % V == 0) &&
                   (p.D - p.R) % (2 * V) == 0;
  const int v = vec ? V : 1;
  p.rot_units = p.R / (2 * v);
  p.units = p.rot_units + (p.D - p.R + 2 * v - 1) / (2 * v);
  p.q_chunks = (p.Hq + kHeads - 1) / kHeads;
  p.chunks = p.q_chunks + (p.Hk + kHeads - 1) / kHeads;
  // as many rows as the threads have items for, and the tables room
  const int x = p.units < kThreads ? p.units : kThreads;
  const int y = kThreads / x < p.chunks ? kThreads / x : p.chunks;
  int z = kThreads / (x * y);
  const int most = kAngles / (p.R / 2);
  if (z > most) z = most;
  if (z > 64) z = 64;
  const dim3 block(x, y, z);
  const int grid = (p.rows + z - 1) / z;
  if (vec)
    rotary_kernel<T, V><<<grid, block, 0, ctx->stream>>>(p);
  else
    rotary_kernel<T, 1><<<grid, block, 0, ctx->stream>>>(p);
  return check_launch("rotary_kernel");
}

}  // namespace rotary
}  // namespace anima

extern "C" int anima_rotary(anima_ctx* ctx, const anima_rotary_args* a) {
  ANIMA_REQUIRE(ctx && a, "anima_rotary: NULL argument");
  ANIMA_ON_DEVICE(ctx);
  ANIMA_REQUIRE(a->dtype == ANIMA_F32 || a->dtype == ANIMA_BF16 || a->dtype == ANIMA_F16, "anima_rotary: dtype %d",
                a->dtype);
  ANIMA_REQUIRE(a->rows >= 0 && a->rows <= 1 << 30 && a->Hq >= 0 && a->Hk >= 0 && a->Hq + a->Hk > 0 && a->Hq <= 1024 && a->Hk <= 1024,
                "anima_rotary: %d rows, %d and %d heads", a->rows, a->Hq, a->Hk);
  ANIMA_REQUIRE(a->D > 0 && a->D <= 65536 && a->R >= 2 && a->R % 2 == 0 && a->R <= a->D && a->R / 2 <= rotary::kAngles,
                "anima_rotary: %d rotated of %d dims (an even number, at most the head and %d)", a->R, a->D,
                2 * rotary::kAngles);
  if (a->rows == 0) return ANIMA_OK;
  ANIMA_REQUIRE(a->inv_freq, "anima_rotary: inv_freq is NULL");
  ANIMA_REQUIRE((a->Hq == 0 || (a->q && a->out_q)) && (a->Hk == 0 || (a->k && a->out_k)),
                "anima_rotary: NULL data pointer");
  const long long qc = static_cast<long long>(a->Hq) * a->D, kc = static_cast<long long>(a->Hk) * a->D;
  ANIMA_REQUIRE(a->Hq == 0 || (a->ldq >= qc && a->ldoq >= qc), "anima_rotary: q's row stride is below its %lld columns",
                qc);
  ANIMA_REQUIRE(a->Hk == 0 || (a->ldk >= kc && a->ldok >= kc), "anima_rotary: k's row stride is below its %lld columns",
                kc);
  ANIMA_REQUIRE((a->Hq == 0 || a->q != a->out_q || a->ldq == a->ldoq) &&
                    (a->Hk == 0 || a->k != a->out_k || a->ldk == a->ldok),
                "anima_rotary: in place, the row strides of input and output have to agree");
  ANIMA_REQUIRE(a->positions || a->rows_per_item > 0, "anima_rotary: rows_per_item %d without positions",
                a->rows_per_item);
  rotary::Params p{};
  p.q = {a->q, a->out_q, a->ldq, a->ldoq};
  p.k = {a->k, a->out_k, a->ldk, a->ldok};
  p.inv_freq = a->inv_freq;
  p.positions = a->positions;
  p.offset = a->offset;
  p.rows = a->rows;
  p.rows_per_item = a->rows_per_item > 0 ? a->rows_per_item : 1;
  p.Hq = a->Hq;
  p.Hk = a->Hk;
  p.D = a->D;
  p.R = a->R;
  p.interleaved = a->interleaved != 0;
  p.inverse = a->inverse != 0;
  p.in_place_rest = (a->Hq == 0 || a->q == a->out_q) && (a->Hk == 0 || a->k == a->out_k);
  p.mscale = a->mscale;
  const int esz = a->dtype == ANIMA_F32 ? 4 : 2, v = 16 / esz;
  auto al = [&](const void* x, long long ld) { return reinterpret_cast<uintptr_t>(x) % 16 == 0 && ld % v == 0; };
  const bool vec = (a->Hq == 0 || (al(a->q, a->ldq) && al(a->out_q, a->ldoq))) &&
                   (a->Hk == 0 || (al(a->k, a->ldk) && al(a->out_k, a->ldok)));
  ProfScope prof(ctx, "rotary", 0, 2.0 * esz * a->rows * static_cast<double>(qc + kc));
  if (a->dtype == ANIMA_F32) return rotary::launch<float>(ctx, p, vec);
  if (a->dtype == ANIMA_BF16) return rotary::launch<__nv_bfloat16>(ctx, p, vec);
  return rotary::launch<__half>(ctx, p, vec);
}
