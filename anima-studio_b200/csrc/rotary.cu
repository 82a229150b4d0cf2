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
// whole pairs (half layout: dims e.. and R/2 + e..; interleaved: 2 adjacent vectors) of one row, so
// its V cos/sin pairs are computed once and stay in registers over a chunk of heads; the loads of
// four heads are issued before the first is used.

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
struct alignas(sizeof(T) * V) Vec {
  T e[V];
};

// cos and sin of position * frequency, times m.
__device__ __forceinline__ void angle(double pos, double f, float m, bool inverse, float& c, float& s) {
  double t = pos * f * 0.15915494309189533577;  // 1 / (2 pi)
  t -= rint(t);
  sincospif(2.0f * static_cast<float>(t), &s, &c);
  c *= m;
  s *= inverse ? -m : m;
}

// Written out, so that every form of the kernel fuses the same product into the sum.
__device__ __forceinline__ float turn0(float x0, float x1, float c, float s) { return fmaf(x0, c, -__fmul_rn(x1, s)); }
__device__ __forceinline__ float turn1(float x0, float x1, float c, float s) { return fmaf(x1, c, __fmul_rn(x0, s)); }

constexpr int kHeads = 8;  // heads of one thread
constexpr int kBatch = 4;  // heads whose loads are in flight together
constexpr int kThreads = 128;

// V = 16 bytes of elements, or 1 where sizes or alignment do not allow vectors.
template <typename T, int V>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const Params p) {
  const long long id = static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x;
  const int row = static_cast<int>(id / p.units);
  if (row >= p.rows) return;
  const int u = static_cast<int>(id - static_cast<long long>(row) * p.units);
  const bool rot = u < p.rot_units;
  if (!rot && p.in_place_rest) return;
  // the two vectors of the unit within a head
  int e0, e1;
  if (!rot) {
    e0 = p.R + (u - p.rot_units) * 2 * V;
    e1 = e0 + V;
  } else if (p.interleaved) {
    e0 = u * 2 * V;
    e1 = e0 + V;
  } else {
    e0 = u * V;
    e1 = e0 + p.R / 2;
  }
  const bool two = e1 < p.D;  // V = 1: a copied unit at an odd end has one element
  float c[V], s[V];
  if (rot) {
    const double pos = p.positions ? static_cast<double>(p.positions[row])
                                   : static_cast<double>(p.offset + row % p.rows_per_item);
#pragma unroll
    for (int i = 0; i < V; ++i) angle(pos, p.inv_freq[u * V + i], p.mscale, p.inverse != 0, c[i], s[i]);
  }
  const int h0 = blockIdx.y * kHeads, h1 = min(h0 + kHeads, p.Hq + p.Hk);
  for (int hb = h0; hb < h1; hb += kBatch) {
    Vec<T, V> a[kBatch], b[kBatch];
    T* dst[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int h = hb + i;
      dst[i] = nullptr;
      if (h >= h1) continue;
      const bool is_q = h < p.Hq;
      const Side& sd = is_q ? p.q : p.k;
      const long long col = static_cast<long long>(is_q ? h : h - p.Hq) * p.D;
      const T* src = static_cast<const T*>(sd.x) + row * sd.ldx + col;
      dst[i] = static_cast<T*>(sd.y) + row * sd.ldy + col;
      a[i] = *reinterpret_cast<const Vec<T, V>*>(src + e0);
      if (two) b[i] = *reinterpret_cast<const Vec<T, V>*>(src + e1);
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (!dst[i]) continue;
      if (rot) {
        float x[2 * V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
          x[j] = ld1<T>(a[i].e[j]);
          x[V + j] = ld1<T>(b[i].e[j]);
        }
        float y[2 * V];
        if (p.interleaved) {
#pragma unroll
          for (int j = 0; j < V; ++j) {
            y[2 * j] = turn0(x[2 * j], x[2 * j + 1], c[j], s[j]);
            y[2 * j + 1] = turn1(x[2 * j], x[2 * j + 1], c[j], s[j]);
          }
        } else {
#pragma unroll
          for (int j = 0; j < V; ++j) {
            y[j] = turn0(x[j], x[V + j], c[j], s[j]);
            y[V + j] = turn1(x[j], x[V + j], c[j], s[j]);
          }
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {
          a[i].e[j] = st1<T>(y[j]);
          b[i].e[j] = st1<T>(y[V + j]);
        }
      }
      *reinterpret_cast<Vec<T, V>*>(dst[i] + e0) = a[i];
      if (two) *reinterpret_cast<Vec<T, V>*>(dst[i] + e1) = b[i];
    }
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
  const long long blocks = (static_cast<long long>(p.rows) * p.units + kThreads - 1) / kThreads;
  ANIMA_REQUIRE(blocks < (1LL << 31), "anima_rotary: %d rows are too many", p.rows);
  const dim3 grid(static_cast<unsigned>(blocks), (p.Hq + p.Hk + kHeads - 1) / kHeads);
  if (vec)
    rotary_kernel<T, V><<<grid, kThreads, 0, ctx->stream>>>(p);
  else
    rotary_kernel<T, 1><<<grid, kThreads, 0, ctx->stream>>>(p);
  return check_launch("rotary_kernel");
}

}  // namespace rotary
}  // namespace anima

extern "C" int anima_rotary(anima_ctx* ctx, const anima_rotary_args* a) {
  ANIMA_REQUIRE(ctx && a, "anima_rotary: NULL argument");
  ANIMA_ON_DEVICE(ctx);
  ANIMA_REQUIRE(a->dtype == ANIMA_F32 || a->dtype == ANIMA_BF16 || a->dtype == ANIMA_F16, "anima_rotary: dtype %d",
                a->dtype);
  ANIMA_REQUIRE(a->rows >= 0 && a->Hq >= 0 && a->Hk >= 0 && a->Hq + a->Hk > 0 && a->Hq <= 65536 && a->Hk <= 65536,
                "anima_rotary: %d rows, %d and %d heads", a->rows, a->Hq, a->Hk);
  ANIMA_REQUIRE(a->D > 0 && a->D <= 65536 && a->R >= 2 && a->R % 2 == 0 && a->R <= a->D,
                "anima_rotary: %d rotated of %d dims (an even number, at most the head)", a->R, a->D);
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
