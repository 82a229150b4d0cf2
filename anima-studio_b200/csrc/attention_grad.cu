// The backward pass of attention on tcgen05 (kind::f16), head_dim 64 and 128, bf16 and fp16: recomputes
// the probabilities from q, k and the forward's row statistic lse, and writes dq, dk, dv.
//
//   S = scale Q K^T, P = exp(S - lse), dP = dO V^T, delta = rowsum(dO O), dS = P (dP - delta)
//   dV = P^T dO, dK = scale dS^T Q, dQ = scale dS K
//
// Two kinds of work units, in one launch. A k/v unit holds 128 keys of one k/v head and walks the
// query blocks that see them (of every q head of the group, and of every batch item that shares the
// K/V), with dV and dK in tensor memory. A q unit holds 128 queries of one head and walks its key
// blocks, with dQ in tensor memory. S and dP are so computed twice, 7 products for the 5 that the
// gradients need; in return nothing is added up in memory between units, so there are no atomics and
// the same inputs give the same bits.
//
// 576 threads: warps 0-15 turn S and dP into P and dS (warp w: the 32 tensor-memory lanes of quadrant
// w % 4, column quarter w / 4), warp 16 loads tiles by TMA, warp 17 allocates tensor memory and issues
// the products. A k/v unit computes the transposed S^T = K Q^T and dP^T = V dO^T (lanes = keys), so that
// P^T and dS^T, rounded to 16 bits and written back over S^T and dP^T, are the A operand of
// dV += P^T dO and dK += dS^T Q straight from tensor memory, with the Q and dO tiles that are in
// shared memory anyway as their MN-major B operand. Issue order per block:
//   dV(i) S(i+1) [dS(i) written] dK(i) dP(i+1)
// so the exponentials of block i + 1 overlap dK(i) and dP(i+1), and the products dS(i) overlap dV(i)
// and S(i+1). A q unit has dP twice in tensor memory, and S is read into registers at once, so S(i+1)
// and dP(i+1) are computed while block i is: S(i+1) dP(i+1) | [dS(i) written] dQ(i).
// A k/v unit's lse and delta belong to columns, the same for all lanes. Loading them costs dearly there
// (beside products that read both operands from shared memory, 8 16-byte loads a warp took 5700 cycles
// for 190), so the tensor core adds them: S^T and dP^T get one more step of 16 inner indices, a constant
// column times each value's 16-bit parts, three of them: in bf16 value = hi + mid + low to 2^-24 of it; in
// fp16, whose range is short, lse / scale = 2^15 hi + 2^5 mid + low, up to 2^31 and to 2^-33 of it or 2^-25.
// Tensor memory, k/v unit: S^T [0,128) dP^T [128,256) dV [256,256+D) dK [256+D,256+2D);
// q unit: S [0,128), dP [128,256) and [384,512), dQ [256,256+D).
//
// Bound by the tensor core and the card's power: 4096 x 4096, 16 heads of 128 in bf16 takes 357 to 371 us (two
// cards), 926 to 962 TFLOP/s of the gradients' 10 Lq Lk D H and 1297 to 1347 of the 14 that are executed
// (cuBLAS: 1646 for milliseconds, 1405 for seconds); 8192 x 8192 causal with 8 k/v heads 707 to 730 us,
// 4096 x 4096 of 64 dims 273 to 282 us (there the exponentials bound it).
//
// Roundings. P and dS round to the operands' type before their products (fp32 sums). In fp16 both are
// moved into its range by powers of two that are undone in fp32: P <= 1 by 2^14; dS by a factor from
// the bound |dS| <= 2 max|dO_i| max|V_j| of the k/v head, so that gradients of any size keep their
// digits. bf16 has fp32's range and needs neither.
//
// delta taken from the rounded output is off by up to half a step of sum |dO O|, next to nothing beside dS's
// own rounding in a row of many keys, but not in one of few (a causal sequence's first rows, which have its
// largest gradients; short prompts). Where all keys of a query block lie in one key block - the first block
// of a causal sequence, all of them up to 128 keys - its q units therefore go first, in a launch of their
// own, take delta = sum_j P_ij dP_ij from the tile and leave it to the k/v units.
//
// Masks: a query row that sees no key has lse = -inf, P = 0 and no gradient. Keys past key_len get
// dK = dV = 0 whatever they hold: P and dS are selected, not multiplied, to 0, and a q unit clears
// their rows of K in shared memory (0 x NaN is not 0).

#include "internal.h"
#include "sm100.cuh"

namespace anima {
namespace agrad {

using attn::arrive_one_lane;
using attn::ATOM;
using attn::ex2;
using attn::pack2;
using attn::TILE;

constexpr int THREADS = 576;
constexpr int MATH_WARPS = 16;
constexpr int TILE_BYTES = 2 * ATOM;  // a tile's slot: 128 rows of 128 16-bit columns (64: half of it is used)
// shared memory: the unit's two tiles | ring of up to 3 first tiles | ring of 2 second tiles | row
// statistics of the ring's stages | barriers. A k/v unit: K, V | Q | dO; a q unit: Q, dO | K | V.
constexpr int OFF_X = 0;
constexpr int OFF_Y0 = OFF_X + 2 * TILE_BYTES;
constexpr int Y0_STAGES = 3;
constexpr int OFF_Y1 = OFF_Y0 + Y0_STAGES * TILE_BYTES;
constexpr int Y1_STAGES = 2;
// a k/v unit needs only two stages of Q: the third's place holds the statistics
constexpr int KV_Y0_STAGES = 2;
constexpr int STAT_TILE = TILE * 32;                             // 128 rows of 16 16-bit columns
constexpr int OFF_STAT = OFF_Y0 + KV_Y0_STAGES * TILE_BYTES;  // [2 stages][lse | delta][STAT_TILE]
constexpr int OFF_ONES = OFF_STAT + 2 * 2 * STAT_TILE;        // [lse | delta][STAT_TILE]
static_assert(OFF_ONES + 2 * STAT_TILE <= OFF_Y1, "the statistics fit the place of a tile");
constexpr int OFF_BAR = OFF_Y1 + Y1_STAGES * TILE_BYTES;
constexpr int SMEM_BYTES = OFF_BAR + 256 + 1024;
static_assert(SMEM_BYTES <= 232448, "fits a block's shared memory");
constexpr float kP16Shift = 14.0f;  // fp16: P is held as 2^14 P
// fp16: the units of the parts that lse / scale enters the product in. The first is the largest power of two
// that fp16 holds; what it leaves, at most 2^-11 of 2^31, is within fp16 in units of 2^5; what that leaves, at
// most 2^9, in units of 1. (One unit of 128 for all three ended at 2^23: with softmax scales around 1e-6, or
// q.k past 8e6, P became 0 or inf.)
__device__ constexpr float kLse16[3] = {32768.0f, 32.0f, 1.0f};

struct Params {
  int B, H, group, Lq, Lk, Lqp;  // Lqp: Lq rounded up to whole tiles
  int kv_batch;                  // 1 where the items share one K/V
  int Hk, kv_heads, walk_heads;  // k/v heads; of all K/V items; (item, q head) pairs that share one
  int q_col, k_col, v_col;
  int causal;
  const int* key_len;
  float scale, scale_log2;
  const float* nlse2;   // [B][H][Lqp] -lse log2(e) (fp16: + 14), -inf for rows without a key
  float* ndelta;        // [B][H][Lqp] -delta
  uint8_t* stat;        // [B][H][nqb][lse | delta][STAT_TILE] nlse2 / scale_log2 and ndelta in 16-bit parts
  const unsigned* top;  // fp16: [kv_batch][Hk][2] largest |dO_i|^2 and |V_j|^2, as bits
  void *dq, *dk, *dv;
  long long lddq, lddk, lddv, dq_bs, dk_bs, dv_bs;
  int grad_dtype;
  int kv_units, q_units, nkb, nqb, kv_splits, q_splits;
  int q_first;  // the first q unit of this launch
  int single;   // this launch has only q units of a single key block, which compute delta themselves
  float* kv_part;  // [split][unit][dv | dk][D / 4][128] float4, where kv_splits > 1
  float* q_part;   // [split][unit][D / 4][128] float4
};

// The keys of an item that count.
__device__ __forceinline__ int keys_of(const Params& p, int kvb) {
  return p.key_len ? max(0, min(p.Lk, p.key_len[kvb])) : p.Lk;
}

// fp16: floor(log2) of the bound 2 max|dO_i| max|V_j| of a k/v head's |dS| (and twice its |delta|).
__device__ __forceinline__ int ds_exponent(const unsigned* top, int kv_head) {
  const float bound = 2.f * sqrtf(__uint_as_float(top[2 * kv_head])) * sqrtf(__uint_as_float(top[2 * kv_head + 1]));
  if (!(bound > 0.f) || bound == INFINITY) return 0;
  return min(max(ilogbf(bound), -100), 100);
}
// The power of two that moves dS into fp16 (2^15 at most), and the one that delta / it fits fp16 with.
__device__ __forceinline__ float ds_scale(int e) { return ldexpf(1.f, 14 - e); }
__device__ __forceinline__ float delta_unit(int e) { return ldexpf(1.f, min(max(e - 14, -24), 15)); }

// Where column 0 of a statistics row lies: K-major without swizzle, 8 rows x 16 bytes in a row of 128.
__device__ __forceinline__ int stat_row(int r) { return (r >> 3) * 256 + (r & 7) * 16; }

// Blocks that a mask cuts and whole ones are two copies of the code: the selects cost a whole block a
// third of its issue slots.
struct Yes { static constexpr bool value = true; };
struct No { static constexpr bool value = false; };

// v as the sum of three 16-bit values, each times its unit, a power of two (-inf and NaN: the first alone),
// packed for the first three columns.
template <bool BF16>
__device__ __forceinline__ uint2 three_parts(float v, float u0 = 1.f, float u1 = 1.f, float u2 = 1.f) {
  const float unit[3] = {u0, u1, u2};
  float part[3];
  float rest = v;
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    const float t = rest / unit[i];
    part[i] = BF16 ? __bfloat162float(__float2bfloat16_rn(t)) : __half2float(__float2half_rn(t));
    rest = fabsf(part[i]) < INFINITY ? fmaf(-unit[i], part[i], rest) : 0.f;
  }
  return make_uint2(pack2<BF16>(part[0], part[1]), pack2<BF16>(part[2], 0.f));
}

// The statistics' tiles: rows of 8 in 256 bytes, the second 8 columns 128 bytes on, no swizzle.
constexpr uint32_t kStatHi = (256u >> 4) | (1u << 14);
__device__ __forceinline__ uint32_t stat_lo(uint32_t saddr) { return (saddr >> 4) | ((128u >> 4) << 16); }

struct Bars {
  uint64_t *x_full, *y0_full, *y1_full, *y0_empty, *y1_empty, *s_full, *s_free, *dp_full, *p_full, *ds_full, *acc_done, *drain;
};
// (ds_full is two barriers, used in turn: a q unit's dP(i + 1) is on its way before dS(i) is waited for, so
// the math warps can finish dS(i + 1) before the issuing warp has looked at dS(i), and on a single barrier
// it would then see the next phase of the same parity and wait for good. A k/v unit gives out dP(i + 1)
// after dS(i) only, and S(i + 1) after P(i), so one p_full and one s_full, dp_full and s_free cannot be
// passed by.)
constexpr int kBars = 1 + 3 + 2 + 3 + 2 + 1 + 1 + 2 + 1 + 2 + 1 + 1;

// What a block does: a k/v unit or a q unit, and its range of iterations.
struct Work {
  bool kv;
  int unit, split;
  int blk;         // key block of a k/v unit, query block of a q unit
  int b, h;        // k/v unit: K/V item and k/v head; q unit: item and q head
  int lo, n;       // first iteration and their number
  int per_head;    // k/v unit: iterations (query blocks) of one q head
};

__device__ __forceinline__ Work work_of(const Params& p) {
  Work w;
  int id = blockIdx.x;
  const int kv_ctas = p.kv_units * p.kv_splits;
  w.kv = id < kv_ctas;
  int total;
  if (w.kv) {
    w.unit = p.kv_splits == 1 ? id : id / p.kv_splits;
    w.split = id - w.unit * p.kv_splits;
    const int heads = p.kv_heads;
    // causal: early key blocks are seen by most queries, so they go first; else head by head
    const int bh = p.causal ? w.unit % heads : w.unit / p.nkb;
    w.blk = p.causal ? w.unit / heads : w.unit % p.nkb;
    w.b = bh / p.Hk;
    w.h = bh - w.b * p.Hk;
    const int q0 = p.causal ? w.blk : 0;
    w.per_head = w.blk * TILE < keys_of(p, w.b) ? max(0, p.nqb - q0) : 0;
    total = w.per_head * p.walk_heads;
    w.lo = 0;
    w.n = total;
    if (p.kv_splits > 1) {
      w.lo = static_cast<int>(static_cast<long long>(total) * w.split / p.kv_splits);
      w.n = static_cast<int>(static_cast<long long>(total) * (w.split + 1) / p.kv_splits) - w.lo;
    }
  } else {
    id -= kv_ctas;
    w.unit = p.q_splits == 1 ? id : id / p.q_splits;
    w.split = id - w.unit * p.q_splits;
    w.unit += p.q_first;
    const int heads = p.B * p.H;
    const int bh = p.causal ? w.unit % heads : w.unit / p.nqb;
    w.blk = p.causal ? p.nqb - 1 - w.unit / heads : w.unit % p.nqb;
    w.b = bh / p.H;
    w.h = bh - w.b * p.H;
    total = (keys_of(p, p.kv_batch > 1 ? w.b : 0) + TILE - 1) / TILE;
    if (p.causal) total = min(total, w.blk + 1);
    w.lo = 0;
    w.n = total;
    if (p.q_splits > 1) {
      w.lo = total * w.split / p.q_splits;
      w.n = total * (w.split + 1) / p.q_splits - w.lo;
    }
    w.per_head = 0;
  }
  return w;
}

// Iteration i of a k/v unit: the item, q head and query block.
__device__ __forceinline__ void kv_iteration(const Params& p, const Work& w, int i, int& b, int& h, int& qb) {
  const int it = w.lo + i;
  const int hh = it / w.per_head;  // (item, head of the group)
  qb = it - hh * w.per_head + (p.causal ? w.blk : 0);
  const int g = hh % p.group;
  b = p.kv_batch > 1 ? w.b : hh / p.group;
  h = w.h * p.group + g;
}

// 16-bit values of a column quarter lie at the quarter's own columns, so none of a row's four warps
// overwrites what another still reads: k-step k (16 of the 128 inner indices, 8 columns) of the A operand.
__device__ __forceinline__ uint32_t quarter_cols(int k) { return (k >> 1) * 32 + (k & 1) * 8; }

// N neighbouring columns of an fp32 gradient's row.
template <int N>
__device__ __forceinline__ void put(void* out, size_t at, const float (&v)[N]) {
  float4* d = reinterpret_cast<float4*>(static_cast<float*>(out) + at);
#pragma unroll
  for (int t = 0; t < N / 4; ++t) d[t] = make_float4(v[4 * t], v[4 * t + 1], v[4 * t + 2], v[4 * t + 3]);
}

// 2^x of a pair on the FMA and integer pipes: x = n + f, |f| <= 1/2, by adding 1.5 2^23 (whose sum has n
// in its low bits), 2^f by a polynomial of degree 4 (least largest relative error, 2.6e-6), times 2^n put
// together from n's bits (the reduction of Cody and Waite, Software Manual for the Elementary Functions, 1980).
// To share a softmax's exponentials between the special-function unit and the FMA pipe is a published idea
// for attention on this architecture, not this code's own. x below -127 gives 0, NaN stays NaN.
__device__ __forceinline__ f2 exp2_fma(f2 x) {
  asm("max.NaN.f32 %0, %0, 0fC2FE0000;" : "+f"(x.x));  // -127
  asm("max.NaN.f32 %0, %0, 0fC2FE0000;" : "+f"(x.y));
  const f2 m = add2(x, dup2(12582912.0f));
  const f2 f = sub2(x, add2(m, dup2(-12582912.0f)));
  f2 q = fma2(dup2(0.009570101f), f, dup2(0.05591786f));
  q = fma2(q, f, dup2(0.24024744f));
  q = fma2(q, f, dup2(0.6931218f));
  q = fma2(q, f, dup2(0.9999993f));
  const f2 e = make_float2(__int_as_float((__float_as_int(m.x) << 23) + 0x3F800000),
                           __int_as_float((__float_as_int(m.y) << 23) + 0x3F800000));
  return mul2(q, e);
}
// The special-function unit gives 16 powers a cycle and SM, 1024 cycles for a block: every kFmaEvery-th
// pair goes the other way.
constexpr int kFmaEvery = 4;
__device__ __forceinline__ f2 exp2_pair(f2 x, int t) {
  if ((t / 2) % kFmaEvery == kFmaEvery - 1) return exp2_fma(x);
  return make_float2(ex2(x.x), ex2(x.y));
}

// Values that are computed here and not later (the compiler would move them behind the next wait).
template <int N>
__device__ __forceinline__ void settle(float (&v)[N]) {
#pragma unroll
  for (int t = 0; t < N; t += 8)
    asm volatile("" : "+f"(v[t]), "+f"(v[t + 1]), "+f"(v[t + 2]), "+f"(v[t + 3]), "+f"(v[t + 4]), "+f"(v[t + 5]),
                 "+f"(v[t + 6]), "+f"(v[t + 7]));
}

template <bool BF16, int HD>
__global__ void __launch_bounds__(THREADS, 1)
    attention_grad_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                          const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_do,
                          const __grid_constant__ CUtensorMap tm_dq, const __grid_constant__ CUtensorMap tm_dk,
                          const __grid_constant__ CUtensorMap tm_dv, const Params p) {
  constexpr int ATOMS = HD / 64;
  constexpr int BYTES = ATOMS * ATOM;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + OFF_BAR);
  const Bars bar{bars,      bars + 1,  bars + 4,  bars + 6,  bars + 9,  bars + 11,
                 bars + 12, bars + 13, bars + 15, bars + 16, bars + 18, bars + 19};
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + kBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  // the same for all lanes, and known to be
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  constexpr int kProducerWarp = MATH_WARPS, kMmaWarp = MATH_WARPS + 1;
  const uint32_t lead = elect_lead();
  const Work w = work_of(p);
  const int y0_stages = w.kv ? KV_Y0_STAGES : Y0_STAGES;

  // The loading thread also sets up the barriers and starts the first loads, so that they are on their way
  // while the others get ready: that took 3900 cycles beside the 7000 that a q unit of four blocks works.
  const int kvb = p.kv_batch > 1 ? w.b : 0;
  const int hk = w.kv ? w.h : w.h / p.group;
  auto load = [&](int off, const CUtensorMap* tm, uint64_t* fb, int col, int row, int item) {
#pragma unroll
    for (int t = 0; t < ATOMS; ++t) tma_load_3d(smem + off + t * ATOM, tm, fb, col + 64 * t, row, item);
  };
  auto load_y0 = [&](int i, int place, int b, int h, int qb) {
    uint64_t* fb = &bar.y0_full[place];
    if (w.kv) {
      // the statistics come and go with Q: its place is freed last
      mbar_arrive_expect_tx(fb, BYTES + 2 * STAT_TILE);
      load(OFF_Y0 + place * TILE_BYTES, &tm_q, fb, p.q_col + h * HD, qb * TILE, b);
      bulk_load_1d(smem + OFF_STAT + place * 2 * STAT_TILE,
                   p.stat + ((static_cast<size_t>(b) * p.H + h) * p.nqb + qb) * (2 * STAT_TILE), 2 * STAT_TILE, fb);
    } else {
      mbar_arrive_expect_tx(fb, BYTES);
      load(OFF_Y0 + place * TILE_BYTES, &tm_k, fb, p.k_col + hk * HD, (w.lo + i) * TILE, kvb);
    }
  };
  auto load_y1 = [&](int i, int place, int b, int h, int qb) {
    uint64_t* fb = &bar.y1_full[place];
    mbar_arrive_expect_tx(fb, BYTES);
    if (w.kv) {
      load(OFF_Y1 + place * TILE_BYTES, &tm_do, fb, h * HD, qb * TILE, b);
    } else {
      load(OFF_Y1 + place * TILE_BYTES, &tm_v, fb, p.v_col + hk * HD, (w.lo + i) * TILE, kvb);
    }
  };
  if (warp == kProducerWarp && lane == 0) {
    for (int i = 0; i < kBars; ++i) {
      const bool math = i == 12 || (i >= 15 && i <= 17);  // s_free, p_full, ds_full
      mbar_init(bars + i, math ? MATH_WARPS : 1);
    }
    *abort_flag = 0;
    fence_mbar_init();
    fence_proxy_async_smem();
    if (w.n > 0) {
      int b = 0, h = 0, qb = 0;
      if (w.kv) kv_iteration(p, w, 0, b, h, qb);
      mbar_arrive_expect_tx(bar.x_full, 2 * BYTES);
      if (w.kv) {
        load(OFF_X, &tm_k, bar.x_full, p.k_col + hk * HD, w.blk * TILE, kvb);
        load_y0(0, 0, b, h, qb);
        load(OFF_X + TILE_BYTES, &tm_v, bar.x_full, p.v_col + hk * HD, w.blk * TILE, kvb);
      } else {
        load(OFF_X, &tm_q, bar.x_full, p.q_col + w.h * HD, w.blk * TILE, w.b);
        load_y0(0, 0, b, h, qb);
        load(OFF_X + TILE_BYTES, &tm_do, bar.x_full, w.h * HD, w.blk * TILE, w.b);
      }
      load_y1(0, 0, b, h, qb);
    }
  }
  if (w.kv && threadIdx.x < 2 * TILE) {  // the constant columns: 1 (or fp16's units) three times, then zeros
    const int which = threadIdx.x / TILE;
    uint8_t* row = smem + OFF_ONES + which * STAT_TILE + stat_row(threadIdx.x % TILE);
    uint32_t first = pack2<BF16>(1.f, 1.f), third = pack2<BF16>(1.f, 0.f);
    if (!BF16) {
      const float d = delta_unit(ds_exponent(p.top, w.b * (p.H / p.group) + w.h));
      first = which ? pack2<BF16>(d, d) : pack2<BF16>(kLse16[0], kLse16[1]);
      third = pack2<BF16>(which ? d : kLse16[2], 0.f);
    }
    *reinterpret_cast<uint4*>(row) = make_uint4(first, third, 0u, 0u);
    *reinterpret_cast<uint4*>(row + 128) = make_uint4(0u, 0u, 0u, 0u);
    fence_proxy_async_smem();
  }
  if (warp == kMmaWarp) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t t_s = tmem, t_dp = tmem + 128, t_acc = tmem + 256, t_acc2 = tmem + 256 + HD, t_dp1 = tmem + 384;

  if (warp == kProducerWarp) {
    if (lane == 0 && w.n > 0) {
      // what is in flight: for each full barrier (x, y0[3], y1[2]), armed and the parity of its last arm
      uint32_t armed = 2u | 2u << 2 | 2u << 8;
      auto arm = [&](int i, uint32_t ph) { armed = (armed & ~(3u << (2 * i))) | ((2u | ph) << (2 * i)); };
      int s0 = 1, s1 = 1;  // block 0 is on its way
      uint32_t ph0 = 0, ph1 = 0;
      for (int i = 1; i < w.n; ++i) {
        int b = 0, h = 0, qb = 0;
        if (w.kv) kv_iteration(p, w, i, b, h, qb);
        if (!mbar_wait(&bar.y0_empty[s0], ph0 ^ 1, abort_flag, kErrTimeoutEmpty)) break;
        load_y0(i, s0, b, h, qb);
        arm(1 + s0, ph0);
        if (!mbar_wait(&bar.y1_empty[s1], ph1 ^ 1, abort_flag, kErrTimeoutEmpty)) break;
        load_y1(i, s1, b, h, qb);
        arm(4 + s1, ph1);
        if (++s0 == y0_stages) s0 = 0, ph0 ^= 1;
        if (++s1 == Y1_STAGES) s1 = 0, ph1 ^= 1;
      }
      // every copy this thread started lands before the block exits: another warp's wait can run out after
      // the last of them was issued (on the way all are waited for anyway)
      for (int i = 0; i < 6; ++i) {
        const uint32_t a = (armed >> (2 * i)) & 3u;
        if (a & 2u) mbar_settle(bars + i, a & 1u);
      }
    }
  } else if (warp == kMmaWarp) {
    if (w.n > 0) {
      constexpr uint32_t id_s = idesc_f16(TILE, TILE, BF16, false);
      constexpr uint32_t id_acc = idesc_f16(TILE, HD, BF16, true);
      // low words of the unit's tiles and the rings' first places, read along the head's dims (K-major)
      // and along the rows (MN-major); a place further is TILE_BYTES on
      const uint32_t x0 = desc_lo(smem_u32(smem + OFF_X), 16), x1 = x0 + (TILE_BYTES >> 4);
      const uint32_t y0 = desc_lo(smem_u32(smem + OFF_Y0), 16), y1 = desc_lo(smem_u32(smem + OFF_Y1), 16);
      constexpr uint32_t kRows = (ATOM >> 4) - 1 << 16;  // from the K-major word to the MN-major one
      constexpr uint32_t kPlace = TILE_BYTES >> 4;
      // d = A B^T over the head's dims, both tiles K-major in shared memory
      auto dims_product = [&](uint32_t d, uint32_t a, uint32_t b) {
#pragma unroll
        for (int k = 0; k < HD / 16; ++k) {
          const uint32_t off = ((k >> 2) * ATOM + (k & 3) * 32) >> 4;
          umma_ss(d, a + off, b + off, id_s, k > 0 ? 1u : 0u, lead);
        }
      };
      // d += a column's statistic in every lane (which: 0 lse, 1 delta), from Q's place s
      const uint32_t ones = stat_lo(smem_u32(smem + OFF_ONES)), stats = stat_lo(smem_u32(smem + OFF_STAT));
      auto add_statistic = [&](uint32_t d, int which, int s) {
        if (w.kv)
          umma_ss(d, ones + which * (STAT_TILE >> 4), stats + (2 * s + which) * (STAT_TILE >> 4), id_s, 1u, lead, kStatHi);
      };
      // d (+)= A B, A 128 x 128 16-bit in tensor memory, B's rows the inner index
      auto rows_product = [&](uint32_t d, uint32_t a, uint32_t b, bool first) {
#pragma unroll
        for (int k = 0; k < TILE / 16; ++k)
          umma_ts(d, a + quarter_cols(k), b + kRows + k * (16 * 128 >> 4), id_acc, (!first || k > 0) ? 1u : 0u, lead);
      };
      auto full = [&](uint64_t* fb, uint32_t ph) { return warp_wait(fb, ph, lead, abort_flag, kErrTimeoutFull); };
      bool ok = full(bar.x_full, 0) && full(&bar.y0_full[0], 0);
      if (ok) {
        tc_fence_after();
        dims_product(t_s, x0, y0);
        add_statistic(t_s, 0, 0);
        umma_commit(bar.s_full, lead);
        ok = full(&bar.y1_full[0], 0);
      }
      if (ok) {
        dims_product(t_dp, x1, y1);
        add_statistic(t_dp, 1, 0);
        umma_commit(bar.dp_full, lead);
      }
      if (w.kv) {
        int s = 0;  // stage of block i (both rings have two)
        uint32_t ph = 0;
        for (int i = 0; ok && i < w.n; ++i) {
          const int s1 = s ^ 1;
          const uint32_t ph1 = s1 ? ph : ph ^ 1;
          const bool more = i + 1 < w.n;
          if (!(ok = full(bar.p_full, i & 1))) break;
          tc_fence_after();
          rows_product(t_acc, t_s, y1 + s * kPlace, i == 0);  // dV
          umma_commit(&bar.y1_empty[s], lead);
          if (more) {
            if (!(ok = full(&bar.y0_full[s1], ph1))) break;
            dims_product(t_s, x0, y0 + s1 * kPlace);
            add_statistic(t_s, 0, s1);
            umma_commit(bar.s_full, lead);
          }
          if (!(ok = full(&bar.ds_full[i & 1], (i >> 1) & 1))) break;
          tc_fence_after();
          rows_product(t_acc2, t_dp, y0 + s * kPlace, i == 0);  // dK
          umma_commit(&bar.y0_empty[s], lead);
          if (more) {
            if (!(ok = full(&bar.y1_full[s1], ph1))) break;
            dims_product(t_dp, x1, y1 + s1 * kPlace);
            add_statistic(t_dp, 1, s1);
            umma_commit(bar.dp_full, lead);
          }
          s = s1;
          ph = ph1;
        }
      } else {
        int r0 = 0, n0 = 1;  // ring places of K: block i, block i + 1
        uint32_t pn0 = 0;    // the phase of the latter
        if (ok) umma_commit(&bar.y1_empty[0], lead);
        for (int i = 0; ok && i < w.n; ++i) {
          if (i + 1 < w.n) {
            const int s1 = (i + 1) & 1;
            if (!(ok = full(bar.s_free, i & 1) && full(&bar.y0_full[n0], pn0))) break;
            tc_fence_after();
            dims_product(t_s, x0, y0 + n0 * kPlace);
            umma_commit(bar.s_full, lead);
            if (++n0 == Y0_STAGES) n0 = 0, pn0 ^= 1;
            if (!(ok = full(&bar.y1_full[s1], ((i + 1) >> 1) & 1))) break;
            dims_product(s1 ? t_dp1 : t_dp, x1, y1 + s1 * kPlace);
            umma_commit(&bar.dp_full[s1], lead);
            umma_commit(&bar.y1_empty[s1], lead);
          }
          if (!(ok = full(&bar.ds_full[i & 1], (i >> 1) & 1))) break;
          tc_fence_after();
          rows_product(t_acc, i & 1 ? t_dp1 : t_dp, y0 + r0 * kPlace, i == 0);  // dQ
          umma_commit(&bar.y0_empty[r0], lead);
          if (++r0 == Y0_STAGES) r0 = 0;
        }
      }
      // every product this warp issued completes before the block frees tensor memory, whether a wait of
      // this warp ran out or one of the math warps'
      uint64_t* done = ok ? bar.acc_done : bar.drain;
      umma_commit(done, lead);
      mbar_settle(done, 0);
    }
  } else {
    const int qt = warp >> 2, quad = warp & 3;
    const int row = quad * 32 + lane;
    const uint32_t lane_addr = static_cast<uint32_t>(quad * 32) << 16;
    const f2 sc2 = dup2(p.scale_log2);
    const int kv_len = keys_of(p, p.kv_batch > 1 ? w.b : 0);
    float cds = 1.f;  // fp16: dS is held as c dS
    if (!BF16)
      cds = ds_scale(ds_exponent(p.top, (p.kv_batch > 1 ? w.b : 0) * (p.H / p.group) + (w.kv ? w.h : w.h / p.group)));
    const f2 c2 = dup2(BF16 ? 1.f : cds * exp2f(-kP16Shift));  // P arrives as 2^14 P
    bool ok = true;
    float pr[32];  // this quarter row of P
    for (int i = 0; i < w.n; ++i) {
      if (w.kv) {
        int b, h, qb;
        kv_iteration(p, w, i, b, h, qb);
        // lanes are keys: a hidden key's whole row, and on the diagonal block queries before the key
        const bool diag = p.causal && qb == w.blk;
        const bool masked = diag || w.blk * TILE + TILE > kv_len;
        const int first = w.blk * TILE + row >= kv_len ? TILE : (diag ? row : 0);  // first query that sees it
        if (!(ok = warp_wait(bar.s_full, i & 1, lead, abort_flag, kErrTimeoutFull))) break;
        tc_fence_after();
        const uint32_t ts = t_s + lane_addr + 32 * qt, td = t_dp + lane_addr + 32 * qt;
        auto probabilities = [&](auto mask, const uint32_t(&r)[32]) {
          uint32_t pk[16];
#pragma unroll
          for (int t = 0; t < 32; t += 4) {
            const f2 a0 = mul2(make_float2(__uint_as_float(r[t]), __uint_as_float(r[t + 1])), sc2);
            const f2 a1 = mul2(make_float2(__uint_as_float(r[t + 2]), __uint_as_float(r[t + 3])), sc2);
            const f2 e0 = exp2_pair(a0, t), e1 = exp2_pair(a1, t + 2);
            float e[4] = {e0.x, e0.y, e1.x, e1.y};
            if constexpr (decltype(mask)::value) {
#pragma unroll
              for (int u = 0; u < 4; ++u)
                if (32 * qt + t + u < first) e[u] = 0.f;
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) pr[t + u] = e[u];
            pk[t / 2] = pack2<BF16>(e[0], e[1]);
            pk[t / 2 + 1] = pack2<BF16>(e[2], e[3]);
          }
          tmem_st16(ts, pk);
        };
        {
          uint32_t r[32];
          tmem_ld32(ts, r);
          tmem_ld_wait(r);
          if (masked) probabilities(Yes{}, r); else probabilities(No{}, r);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        arrive_one_lane(bar.p_full);
        if (!(ok = warp_wait(bar.dp_full, i & 1, lead, abort_flag, kErrTimeoutFull))) break;
        tc_fence_after();
        auto gradients = [&](auto mask, const uint32_t(&r)[32]) {
          uint32_t pk[16];
#pragma unroll
          for (int t = 0; t < 32; t += 4) {
            f2 g0 = make_float2(__uint_as_float(r[t]), __uint_as_float(r[t + 1]));
            f2 g1 = make_float2(__uint_as_float(r[t + 2]), __uint_as_float(r[t + 3]));
            f2 p0 = make_float2(pr[t], pr[t + 1]), p1 = make_float2(pr[t + 2], pr[t + 3]);
            if (!BF16) p0 = mul2(p0, c2), p1 = mul2(p1, c2);
            g0 = mul2(g0, p0);
            g1 = mul2(g1, p1);
            if constexpr (decltype(mask)::value) {  // 0 whatever dP is
              const int q = 32 * qt + t;
              if (q < first) g0.x = 0.f;
              if (q + 1 < first) g0.y = 0.f;
              if (q + 2 < first) g1.x = 0.f;
              if (q + 3 < first) g1.y = 0.f;
            }
            pk[t / 2] = pack2<BF16>(g0.x, g0.y);
            pk[t / 2 + 1] = pack2<BF16>(g1.x, g1.y);
          }
          tmem_st16(td, pk);
        };
        {
          uint32_t r[32];
          tmem_ld32(td, r);
          tmem_ld_wait(r);
          if (masked) gradients(Yes{}, r); else gradients(No{}, r);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        arrive_one_lane(&bar.ds_full[i & 1]);
      } else {
        const int kb = w.lo + i;
        const size_t at = (static_cast<size_t>(w.b) * p.H + w.h) * p.Lqp + static_cast<size_t>(w.blk) * TILE + row;
        const f2 nlse2 = dup2(p.nlse2[at]);
        f2 ndelta = dup2(p.ndelta[at]);
        // lanes are queries: the row's visible keys of this block end at `end`
        const int left = kv_len - kb * TILE;
        const bool masked = left < TILE || (p.causal && kb == w.blk);
        const int end = p.causal && kb == w.blk ? min(left, row + 1) : left;
        const uint32_t ts = t_s + lane_addr + 32 * qt, td = (i & 1 ? t_dp1 : t_dp) + lane_addr + 32 * qt;
        // (one iteration in a launch of single blocks, and every math warp meets its barrier once)
        auto meet = [&]() { asm volatile("bar.sync 1, %0;" ::"n"(MATH_WARPS * 32) : "memory"); };
        if (!(ok = warp_wait(bar.s_full, i & 1, lead, abort_flag, kErrTimeoutFull))) {
          if (p.single) meet();
          break;
        }
        tc_fence_after();
        auto probabilities = [&](const uint32_t(&r)[32]) {
#pragma unroll
          for (int t = 0; t < 32; t += 2) {
            const f2 a = fma2(make_float2(__uint_as_float(r[t]), __uint_as_float(r[t + 1])), sc2, nlse2);
            const f2 e = exp2_pair(a, t);
            pr[t] = e.x;
            pr[t + 1] = e.y;
          }
        };
        {
          uint32_t r[32];
          tmem_ld32(ts, r);
          tmem_ld_wait(r);
          tc_fence_before();
          __syncwarp();
          arrive_one_lane(bar.s_free);  // S(i + 1) may overwrite it
          probabilities(r);
          settle(pr);
        }
        if (!(ok = warp_wait(&bar.dp_full[i & 1], (i >> 1) & 1, lead, abort_flag, kErrTimeoutFull))) {
          if (p.single) meet();
          break;
        }
        tc_fence_after();
        auto gradients = [&](auto mask, const uint32_t(&r)[32]) {
          uint32_t pk[16];
#pragma unroll
          for (int t = 0; t < 32; t += 2) {
            f2 g = add2(make_float2(__uint_as_float(r[t]), __uint_as_float(r[t + 1])), ndelta);
            f2 pp = make_float2(pr[t], pr[t + 1]);
            if (!BF16) pp = mul2(pp, c2);
            g = mul2(g, pp);
            if constexpr (decltype(mask)::value) {  // 0 whatever S and dP are
              if (32 * qt + t >= end) g.x = 0.f;
              if (32 * qt + t + 1 >= end) g.y = 0.f;
            }
            pk[t / 2] = pack2<BF16>(g.x, g.y);
          }
          tmem_st16(td, pk);
        };
        {
          uint32_t r[32];
          tmem_ld32(td, r);
          tmem_ld_wait(r);
          if (p.single) {
            float d = 0.f;
#pragma unroll
            for (int t = 0; t < 32; ++t)
              if (32 * qt + t < end) d = fmaf(pr[t], __uint_as_float(r[t]), d);
            float* red = reinterpret_cast<float*>(smem + OFF_Y0 + 2 * TILE_BYTES);  // a place no load goes to
            red[qt * TILE + row] = d;
            meet();
            d = (red[row] + red[TILE + row]) + (red[2 * TILE + row] + red[3 * TILE + row]);
            if (!BF16) d *= exp2f(-kP16Shift);
            ndelta = dup2(-d);
            if (qt == 0) {
              p.ndelta[at] = -d;
              float v = -d;
              if (!BF16) v /= delta_unit(ds_exponent(p.top, (p.kv_batch > 1 ? w.b : 0) * (p.H / p.group) + w.h / p.group));
              const uint2 parts = three_parts<BF16>(v);
              *reinterpret_cast<uint4*>(p.stat + (((static_cast<size_t>(w.b) * p.H + w.h) * p.nqb + w.blk) * 2 + 1) * STAT_TILE +
                                        stat_row(row)) = make_uint4(parts.x, parts.y, 0u, 0u);
            }
          }
          if (masked) gradients(Yes{}, r); else gradients(No{}, r);
        }
        if (left < TILE && p.key_len) {
          // K's rows behind key_len may hold anything, and dS K multiplies them by 0
          const int s0 = i % Y0_STAGES;
          if (!(ok = warp_wait(&bar.y0_full[s0], (i / Y0_STAGES) & 1, lead, abort_flag, kErrTimeoutFull))) break;
          const int n = (TILE - left) * 8;  // 16-byte pieces of an atom's rows
          for (int t = threadIdx.x; t < n * ATOMS; t += MATH_WARPS * 32)
            *reinterpret_cast<uint4*>(smem + OFF_Y0 + s0 * TILE_BYTES + (t / n) * ATOM + left * 128 + (t % n) * 16) =
                make_uint4(0, 0, 0, 0);
          fence_proxy_async_smem();
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        arrive_one_lane(&bar.ds_full[i & 1]);
      }
    }
    if (ok && w.n > 0) ok = warp_wait(bar.acc_done, 0, lead, abort_flag, kErrTimeoutAcc);
    if (ok) {
      tc_fence_after();
      const bool split = (w.kv ? p.kv_splits : p.q_splits) > 1;
      const int r = w.blk * TILE + row;
      const int accs = w.kv ? 2 : 1;  // dV, dK
#pragma unroll 1
      for (int a = 0; a < accs; ++a) {
        constexpr int NC = HD / 4;  // columns of a quarter
        const int c0 = NC * qt;
        float v[NC];
        if (w.n > 0) {
          uint32_t u[NC];
          const uint32_t at = (a ? t_acc2 : t_acc) + lane_addr + c0;
          if constexpr (NC == 32) tmem_ld32(at, u); else tmem_ld16(at, u);
          tmem_ld_wait(u);
          float f = BF16 ? 1.f : exp2f(-kP16Shift);
          if (!w.kv || a) f = BF16 ? p.scale : p.scale / cds;
#pragma unroll
          for (int t = 0; t < NC; ++t) v[t] = __uint_as_float(u[t]) * f;
        } else {
#pragma unroll
          for (int t = 0; t < NC; ++t) v[t] = 0.f;
        }
        if (split) {
          const size_t slot = w.kv ? (static_cast<size_t>(w.split) * p.kv_units + w.unit) * 2 + a
                                   : static_cast<size_t>(w.split) * p.q_units + w.unit;
          float4* d = reinterpret_cast<float4*>(w.kv ? p.kv_part : p.q_part) + (slot * (HD / 4) + c0 / 4) * TILE + row;
#pragma unroll
          for (int t = 0; t < NC / 4; ++t) d[t * TILE] = make_float4(v[4 * t], v[4 * t + 1], v[4 * t + 2], v[4 * t + 3]);
        } else if (p.grad_dtype != ANIMA_F32) {
          // a warp's 32 x NC piece through shared memory (the unit's own tiles are done with) to a TMA store,
          // which leaves out the rows behind the last: stored from registers, 16 bytes of 32 rows at a time,
          // a tile took 3500 cycles
          uint8_t* piece = smem + OFF_X + (a * MATH_WARPS + warp) * (32 * NC * 2);
          uint4* d = reinterpret_cast<uint4*>(piece + lane * NC * 2);
#pragma unroll
          for (int t = 0; t < NC / 8; ++t)
            d[t] = make_uint4(pack2<BF16>(v[8 * t], v[8 * t + 1]), pack2<BF16>(v[8 * t + 2], v[8 * t + 3]),
                              pack2<BF16>(v[8 * t + 4], v[8 * t + 5]), pack2<BF16>(v[8 * t + 6], v[8 * t + 7]));
          fence_proxy_async_smem();
          __syncwarp();
          const int r0 = w.blk * TILE + quad * 32;
          if (lead && r0 < (w.kv ? p.Lk : p.Lq)) {
            tma_store_3d(w.kv ? (a ? &tm_dk : &tm_dv) : &tm_dq, piece, w.h * HD + c0, r0, w.b);
            bulk_commit();
          }
        } else if (w.kv) {
          if (r < p.Lk)
            put<NC>(a ? p.dk : p.dv,
                    (a ? w.b * p.dk_bs + r * p.lddk : w.b * p.dv_bs + r * p.lddv) + static_cast<size_t>(w.h) * HD + c0, v);
        } else if (r < p.Lq) {
          put<NC>(p.dq, w.b * p.dq_bs + r * p.lddq + static_cast<size_t>(w.h) * HD + c0, v);
        }
      }
      if (lead) bulk_wait_all();  // shared memory stays until the stores have read it, and they are done
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ------------------------------------------------------------------ before and after it

// delta and the scaled row statistic of every (item, head, query), padded to whole tiles with rows
// that no key sees, in fp32 for the q units and in 16-bit parts for the k/v units; D / 8 threads a row
// and head, 16 bytes each. Bound by reading out and dout once.
struct PrepParams {
  const void* out;
  const void* dout;
  const float* lse;
  long long ldo, o_bs, lddo, do_bs;
  int out_dtype, H, group, Lq, Lqp, kv_batch;
  float shift;  // 14 in fp16
  float inv_scale_log2;
  float *nlse2, *ndelta;
  uint8_t* stat;
  const unsigned* top;
};

constexpr int kPrepRows = 2;  // (row, head) pairs of a thread, their loads in flight together

template <bool BF16, int HD>
__global__ void __launch_bounds__(256) attention_grad_prep_kernel(const PrepParams p) {
  using resnorm::load_raw;
  using resnorm::unpack;
  constexpr int TPR = HD / 8, PAIRS = 256 / TPR;
  const int b = blockIdx.y, t = threadIdx.x % TPR;
  const unsigned pairs = static_cast<unsigned>(p.Lqp) * p.H;
  unsigned row[kPrepRows], h[kPrepRows];
  bool in[kPrepRows], real[kPrepRows];
  resnorm::Raw<8> o[kPrepRows], g[kPrepRows];
  float lse[kPrepRows];
#pragma unroll
  for (int u = 0; u < kPrepRows; ++u) {
    const unsigned id = (blockIdx.x * kPrepRows + u) * PAIRS + threadIdx.x / TPR;
    in[u] = id < pairs;
    row[u] = id / p.H;
    h[u] = id - row[u] * p.H;
    real[u] = in[u] && row[u] < static_cast<unsigned>(p.Lq);
    lse[u] = -INFINITY;
    if (real[u]) {
      const size_t col = static_cast<size_t>(h[u]) * HD + 8 * t;
      load_raw<8>(o[u], p.out, p.out_dtype, b * p.o_bs + row[u] * p.ldo + col);
      load_raw<8>(g[u], p.dout, BF16 ? ANIMA_BF16 : ANIMA_F16, b * p.do_bs + row[u] * p.lddo + col);
      lse[u] = p.lse[(static_cast<size_t>(b) * p.H + h[u]) * p.Lq + row[u]];
    }
  }
#pragma unroll
  for (int u = 0; u < kPrepRows; ++u) {
    float d = 0.f;
    if (real[u]) {
      float x[8], y[8];
      unpack<8>(o[u], p.out_dtype, x);
      unpack<8>(g[u], BF16 ? ANIMA_BF16 : ANIMA_F16, y);
#pragma unroll
      for (int j = 0; j < 8; ++j) d = fmaf(x[j], y[j], d);
    }
#pragma unroll
    for (int s = TPR / 2; s > 0; s >>= 1) d += __shfl_xor_sync(0xffffffffu, d, s);
    if (!in[u]) continue;
    const size_t bh = static_cast<size_t>(b) * p.H + h[u];
    const float nl = lse[u] == -INFINITY ? -INFINITY : fmaf(lse[u], -1.4426950408889634f, p.shift);
    // the row's lanes share its writes
    if (t == 0) p.nlse2[bh * p.Lqp + row[u]] = nl;
    if (t == 1) p.ndelta[bh * p.Lqp + row[u]] = -d;
    if (t >= 2 && t < 6) {
      const int which = (t - 2) >> 1, half = t & 1;
      uint8_t* tile = p.stat + ((bh * (p.Lqp / TILE) + row[u] / TILE) * 2 + which) * STAT_TILE + stat_row(row[u] % TILE) + half * 128;
      uint2 parts = make_uint2(0u, 0u);
      if (!half) {
        if (which) {
          float v = -d;
          if (!BF16) v /= delta_unit(ds_exponent(p.top, (p.kv_batch > 1 ? b : 0) * (p.H / p.group) + h[u] / p.group));
          parts = three_parts<BF16>(v);
        } else if (BF16) {
          parts = three_parts<BF16>(nl * p.inv_scale_log2);
        } else {
          parts = three_parts<BF16>(nl * p.inv_scale_log2, kLse16[0], kLse16[1], kLse16[2]);
        }
      }
      *reinterpret_cast<uint4*>(tile) = make_uint4(parts.x, parts.y, 0u, 0u);
    }
  }
}

// fp16: the largest |dO_i|^2 and |V_j|^2 of each k/v head, over all queries and the keys that count. Block
// row y: a k/v head's V, then a q head's dO; D / 8 threads a row, 16 bytes each, every thread four rows
// whose loads are in flight together.
struct TopParams {
  const __half *v, *dout;
  long long ldv, v_bs, lddo, do_bs;
  int H, group, Lq, Lk, kv_batch;
  int b0;  // the launch's first item
  const int* key_len;
  unsigned* top;
};
constexpr int kTopRows = 4;
template <int HD>
__global__ void __launch_bounds__(256) attention_grad_top_kernel(const TopParams p) {
  constexpr int TPR = HD / 8, ROWS = 256 / TPR;
  const int b = p.b0 + blockIdx.z, Hk = p.H / p.group;
  const bool is_v = blockIdx.y < Hk;
  const int h = is_v ? blockIdx.y : blockIdx.y - Hk;
  if (is_v && b >= p.kv_batch) return;
  const int kvb = p.kv_batch > 1 ? b : 0;
  const int len = is_v ? (p.key_len ? min(p.Lk, p.key_len[kvb]) : p.Lk) : p.Lq;
  const __half* base = (is_v ? p.v + b * p.v_bs : p.dout + b * p.do_bs) + h * HD + 8 * (threadIdx.x % TPR);
  const long long ld = is_v ? p.ldv : p.lddo;
  const int row0 = blockIdx.x * (ROWS * kTopRows) + threadIdx.x / TPR;
  uint4 w[kTopRows];
#pragma unroll
  for (int u = 0; u < kTopRows; ++u) {
    const int j = row0 + u * ROWS;
    w[u] = j < len ? *reinterpret_cast<const uint4*>(base + j * ld) : make_uint4(0u, 0u, 0u, 0u);
  }
  float best = 0.f;
#pragma unroll
  for (int u = 0; u < kTopRows; ++u) {
    const uint32_t q[4] = {w[u].x, w[u].y, w[u].z, w[u].w};
    float n = 0.f;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&q[c]));
      n = fmaf(x.x, x.x, fmaf(x.y, x.y, n));
    }
#pragma unroll
    for (int s = TPR / 2; s > 0; s >>= 1) n += __shfl_xor_sync(0xffffffffu, n, s);
    best = fmaxf(best, n);
  }
#pragma unroll
  for (int s = 16; s >= TPR; s >>= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, s));
  // (bits of values that are not negative are ordered as the values; a maximum hangs on no order)
  if (threadIdx.x % 32 == 0 && best > 0.f)
    atomicMax(p.top + 2 * (kvb * Hk + (is_v ? h : h / p.group)) + (is_v ? 1 : 0), __float_as_uint(best));
}

// The gradients of split units: the splits' partial sums added in order. A thread has four columns of
// one row; the rows of a warp are neighbours, as the partials lie.
template <int HD>
__global__ void __launch_bounds__(128) attention_grad_join_kernel(const Params p) {
  const int kv_tiles = p.kv_splits > 1 ? p.kv_units * 2 : 0;
  int tile = blockIdx.x;
  const bool kv = tile < kv_tiles;
  if (!kv) tile -= kv_tiles;
  const int unit = kv ? tile / 2 : tile, a = kv ? tile % 2 : 0;
  const int splits = kv ? p.kv_splits : p.q_splits, tiles = kv ? p.kv_units * 2 : p.q_units;
  const float4* part = reinterpret_cast<const float4*>(kv ? p.kv_part : p.q_part) +
                       (static_cast<size_t>(tile) * (HD / 4) + blockIdx.y) * TILE + threadIdx.x;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i = 0; i < splits; ++i) {
    const float4 v = part[static_cast<size_t>(i) * tiles * (HD / 4) * TILE];
    s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
  }
  int bh, blk, b, h;
  if (kv) {
    const int Hk = p.H / p.group, heads = p.kv_units / p.nkb;
    bh = p.causal ? unit % heads : unit / p.nkb;
    blk = p.causal ? unit / heads : unit % p.nkb;
    b = bh / Hk;
    h = bh - b * Hk;
  } else {
    const int heads = p.B * p.H;
    bh = p.causal ? unit % heads : unit / p.nqb;
    blk = p.causal ? p.nqb - 1 - unit / heads : unit % p.nqb;
    b = bh / p.H;
    h = bh - b * p.H;
  }
  const int r = blk * TILE + threadIdx.x;
  if (r >= (kv ? p.Lk : p.Lq)) return;
  void* out = kv ? (a ? p.dk : p.dv) : p.dq;
  const size_t at = (kv ? (a ? b * p.dk_bs + r * p.lddk : b * p.dv_bs + r * p.lddv) : b * p.dq_bs + r * p.lddq) +
                    static_cast<size_t>(h) * HD + blockIdx.y * 4;
  if (p.grad_dtype == ANIMA_F32) {
    *reinterpret_cast<float4*>(static_cast<float*>(out) + at) = s;
  } else {
    uint2 w;
    if (p.grad_dtype == ANIMA_BF16)
      w = make_uint2(pack2<true>(s.x, s.y), pack2<true>(s.z, s.w));
    else
      w = make_uint2(pack2<false>(s.x, s.y), pack2<false>(s.z, s.w));
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(out) + at) = w;
  }
}

// ------------------------------------------------------------------ host side

struct Plan {
  int group, kv_batch, Lqp, nkb, nqb, kv_units, q_units, kv_splits, q_splits;
  size_t lse_off, delta_off, stat_off, top_off, top_bytes, kv_off, q_off, bytes;
};

// Units are split along their walk only where there are too few of them to fill the SMs: each split
// writes and reads back an fp32 tile, and joining is a launch more, so a split keeps at least four
// blocks (about 5 us of work against the 2 to 3 us that joining costs).
int splits_of(long long blocks, long long all_units, int sms) {
  long long s = 1;
  if (all_units < sms) s = sms / all_units;
  if (s > blocks / 4) s = blocks / 4;
  if (s > 16) s = 16;
  return s < 1 ? 1 : static_cast<int>(s);
}

int plan_of(const anima_ctx* ctx, const anima_attention_args* a, Plan& pl) {
  pl.group = a->group > 1 ? a->group : 1;
  const bool bcast = a->batch > 1 && a->k_bstride == 0 && a->v_bstride == 0;
  pl.kv_batch = bcast ? 1 : a->batch;
  pl.nqb = (a->Lq + TILE - 1) / TILE;
  pl.nkb = (a->Lk + TILE - 1) / TILE;
  pl.Lqp = pl.nqb * TILE;
  const long long kv = static_cast<long long>(pl.kv_batch) * (a->heads / pl.group) * pl.nkb;
  const long long q = static_cast<long long>(a->batch) * a->heads * pl.nqb;
  ANIMA_REQUIRE(kv < (1LL << 26) && q < (1LL << 26) && a->Lq <= (1 << 30) && a->Lk <= (1 << 30),
                "anima_attention_backward: problem too large");
  const long long walk = static_cast<long long>(pl.nqb) * pl.group * (a->batch / pl.kv_batch);
  ANIMA_REQUIRE(walk < (1LL << 31), "anima_attention_backward: problem too large");
  pl.kv_units = static_cast<int>(kv);
  pl.q_units = static_cast<int>(q);
  pl.kv_splits = splits_of(walk, kv + q, ctx->num_sms);
  pl.q_splits = splits_of(pl.nkb, kv + q, ctx->num_sms);
  size_t at = 0;
  auto take = [&](size_t n) {
    const size_t o = at;
    at += (n + 255) / 256 * 256;
    return o;
  };
  const size_t stat = static_cast<size_t>(a->batch) * a->heads * pl.Lqp * 4;
  pl.lse_off = take(stat);
  pl.delta_off = take(stat);
  pl.stat_off = take(static_cast<size_t>(a->batch) * a->heads * pl.nqb * 2 * STAT_TILE);
  pl.top_bytes = a->dtype == ANIMA_F16 ? static_cast<size_t>(pl.kv_batch) * (a->heads / pl.group) * 8 : 0;
  pl.top_off = take(pl.top_bytes);
  const size_t tile = static_cast<size_t>(TILE) * a->head_dim * 4;
  pl.kv_off = take(pl.kv_splits > 1 ? tile * 2 * pl.kv_units * pl.kv_splits : 0);
  pl.q_off = take(pl.q_splits > 1 ? tile * pl.q_units * pl.q_splits : 0);
  pl.bytes = at;
  return ANIMA_OK;
}

int check(const char* fn, const anima_attention_grad_args* g) {
  const anima_attention_args* a = &g->fwd;
  ANIMA_REQUIRE(a->batch > 0 && a->heads > 0 && a->Lq > 0 && a->Lk > 0, "%s: empty problem", fn);
  ANIMA_REQUIRE(a->head_dim == 64 || a->head_dim == 128, "%s: head_dim %d (64 or 128)", fn, a->head_dim);
  ANIMA_REQUIRE(a->dtype == ANIMA_BF16 || a->dtype == ANIMA_F16, "%s: q/k/v dtype must be bf16 or f16", fn);
  ANIMA_REQUIRE(a->heads % (a->group > 1 ? a->group : 1) == 0, "%s: %d heads do not form groups of %d", fn, a->heads,
                a->group);
  const int st = check_scale(fn, a);
  if (st) return st;
  ANIMA_REQUIRE(a->batch == 1 || (a->k_bstride == 0 && a->v_bstride == 0) || (a->k_bstride > 0 && a->v_bstride > 0),
                "%s: k and v batch strides must both be zero (shared) or both positive", fn);
  return ANIMA_OK;
}

// Items are a grid axis of the passes before the gradients, which ends at 65535: as many launches as that takes.
constexpr int kAxis = 65535;

// Of the next n items (moved here: an item's number in the kernel cost it 0.5 of 18 us).
void advance(PrepParams& p, long long n) {
  auto move = [](const void* q, long long elements, int dt) {
    return static_cast<const void*>(static_cast<const uint8_t*>(q) + elements * (dt == ANIMA_F32 ? 4 : 2));
  };
  p.out = move(p.out, n * p.o_bs, p.out_dtype);
  p.dout = move(p.dout, n * p.do_bs, ANIMA_BF16);
  p.lse += n * p.H * p.Lq;
  p.nlse2 += n * p.H * p.Lqp;
  p.ndelta += n * p.H * p.Lqp;
  p.stat += n * p.H * (p.Lqp / TILE) * 2 * STAT_TILE;
  if (p.kv_batch > 1) p.top += n * (p.H / p.group) * 2;
}

template <bool BF16, int HD>
int launch(anima_ctx* ctx, const anima_attention_grad_args* g, const Plan& pl, const Params& p, PrepParams& pp,
           const CUtensorMap (&tm)[7]) {
  const anima_attention_args* a = &g->fwd;
  const long long pairs = static_cast<long long>(pl.Lqp) * a->heads;
  ANIMA_REQUIRE(pairs < (1LL << 31), "anima_attention_backward: problem too large");
  constexpr int kPairs = kPrepRows * 256 / (HD / 8);  // of a block
  ProfScope prof(ctx, "attn.grad", 10.0 * a->batch * a->heads * static_cast<double>(a->Lq) * a->Lk * HD, 0);
  if (!BF16) {
    ANIMA_CUDA(cudaMemsetAsync(const_cast<unsigned*>(pp.top), 0, pl.top_bytes, ctx->stream));
    const int Hk = a->heads / pl.group;
    ANIMA_REQUIRE(Hk + a->heads <= kAxis, "anima_attention_backward: too many heads");
    TopParams tp{};
    tp.v = static_cast<const __half*>(a->v) + a->v_off;
    tp.dout = static_cast<const __half*>(g->dout);
    tp.ldv = a->ldv;
    tp.v_bs = pl.kv_batch > 1 ? a->v_bstride : 0;
    tp.lddo = g->lddo;
    tp.do_bs = pp.do_bs;
    tp.H = a->heads;
    tp.group = pl.group;
    tp.Lq = a->Lq;
    tp.Lk = a->Lk;
    tp.kv_batch = pl.kv_batch;
    tp.key_len = a->key_len;
    tp.top = const_cast<unsigned*>(pp.top);
    constexpr int kRows = kTopRows * 256 / (HD / 8);  // of a block
    const int blocks = ((a->Lq > a->Lk ? a->Lq : a->Lk) + kRows - 1) / kRows;
    for (tp.b0 = 0; tp.b0 < a->batch; tp.b0 += kAxis)
      attention_grad_top_kernel<HD>
          <<<dim3(blocks, Hk + a->heads, a->batch - tp.b0 < kAxis ? a->batch - tp.b0 : kAxis), 256, 0, ctx->stream>>>(tp);
    const int st = check_launch("attention_grad_top_kernel");
    if (st) return st;
  }
  for (int left = a->batch; left > 0; left -= kAxis, advance(pp, kAxis))
    attention_grad_prep_kernel<BF16, HD>
        <<<dim3(static_cast<unsigned>((pairs + kPairs - 1) / kPairs), left < kAxis ? left : kAxis), 256, 0, ctx->stream>>>(pp);
  int st = check_launch("attention_grad_prep_kernel");
  if (st) return st;
  const auto fn = attention_grad_kernel<BF16, HD>;
  st = set_max_dynamic_smem(reinterpret_cast<const void*>(fn), SMEM_BYTES);
  if (st) return st;
  int q_units = pl.q_units;
  if (a->causal || a->Lk <= TILE) {
    // (in a causal problem the first query blocks are the last units)
    Params p1 = p;
    p1.kv_units = 0;
    p1.q_splits = 1;
    p1.single = 1;
    const int n = a->causal ? a->batch * a->heads : q_units;
    q_units -= n;
    p1.q_first = q_units;
    fn<<<n, THREADS, SMEM_BYTES, ctx->stream>>>(tm[0], tm[1], tm[2], tm[3], tm[4], tm[5], tm[6], p1);
    st = check_launch("attention_grad_kernel (single blocks)");
    if (st) return st;
  }
  const long long ctas = static_cast<long long>(pl.kv_units) * pl.kv_splits + static_cast<long long>(q_units) * pl.q_splits;
  ANIMA_REQUIRE(ctas < (1LL << 31), "anima_attention_backward: problem too large");
  fn<<<static_cast<unsigned>(ctas), THREADS, SMEM_BYTES, ctx->stream>>>(tm[0], tm[1], tm[2], tm[3], tm[4], tm[5], tm[6], p);
  st = check_launch("attention_grad_kernel");
  const int tiles = (pl.kv_splits > 1 ? pl.kv_units * 2 : 0) + (pl.q_splits > 1 ? q_units : 0);
  if (st || tiles == 0) return st;
  attention_grad_join_kernel<HD><<<dim3(tiles, HD / 4), TILE, 0, ctx->stream>>>(p);
  return check_launch("attention_grad_join_kernel");
}

}  // namespace agrad
}  // namespace anima

extern "C" int anima_attention_backward_workspace(anima_ctx* ctx, const anima_attention_grad_args* g, size_t* bytes) {
  ANIMA_REQUIRE(ctx && g && bytes, "anima_attention_backward_workspace: NULL argument");
  int st = agrad::check("anima_attention_backward_workspace", g);
  if (st) return st;
  agrad::Plan pl;
  st = agrad::plan_of(ctx, &g->fwd, pl);
  if (st) return st;
  *bytes = pl.bytes;
  return ANIMA_OK;
}

extern "C" int anima_attention_backward(anima_ctx* ctx, const anima_attention_grad_args* g) {
  using namespace anima::agrad;
  ANIMA_REQUIRE(ctx && g, "anima_attention_backward: NULL argument");
  ANIMA_ON_DEVICE(ctx);
  int st = check("anima_attention_backward", g);
  if (st) return st;
  const anima_attention_args* a = &g->fwd;
  ANIMA_REQUIRE(a->q && a->k && a->v && a->out && g->lse && g->dout && g->dq && g->dk && g->dv,
                "anima_attention_backward: NULL data pointer");
  ANIMA_REQUIRE(a->out_dtype == ANIMA_F32 || a->out_dtype == ANIMA_BF16 || a->out_dtype == ANIMA_F16,
                "anima_attention_backward: out_dtype %d", a->out_dtype);
  ANIMA_REQUIRE(g->grad_dtype == ANIMA_F32 || g->grad_dtype == a->dtype,
                "anima_attention_backward: grad_dtype %d (f32 or that of q)", g->grad_dtype);
  Plan pl;
  st = plan_of(ctx, a, pl);
  if (st) return st;
  const long long cq = static_cast<long long>(a->heads) * a->head_dim, ck = cq / pl.group;
  ANIMA_REQUIRE(a->q_off >= 0 && a->k_off >= 0 && a->v_off >= 0 && a->ldq >= a->q_off + cq && a->ldk >= a->k_off + ck &&
                    a->ldv >= a->v_off + ck && a->ldo >= cq && g->lddo >= cq && g->lddq >= cq && g->lddk >= ck &&
                    g->lddv >= ck,
                "anima_attention_backward: row stride too small");
  ANIMA_REQUIRE(a->q_off % 8 == 0 && a->k_off % 8 == 0 && a->v_off % 8 == 0, "anima_attention_backward: column offsets "
                "must be multiples of 8");
  const bool many = a->batch > 1;
  const struct {
    const void* p;
    long long ld, bs;
    bool batched;
  } all[8] = {{a->q, a->ldq, a->q_bstride, many},
              {a->k, a->ldk, a->k_bstride, pl.kv_batch > 1},
              {a->v, a->ldv, a->v_bstride, pl.kv_batch > 1},
              {a->out, a->ldo, a->o_bstride, many},
              {g->dout, g->lddo, g->do_bstride, many},
              {g->dq, g->lddq, g->dq_bstride, many},
              {g->dk, g->lddk, g->dk_bstride, pl.kv_batch > 1},
              {g->dv, g->lddv, g->dv_bstride, pl.kv_batch > 1}};
  for (const auto& t : all)
    ANIMA_REQUIRE(reinterpret_cast<uintptr_t>(t.p) % 16 == 0 && t.ld % 8 == 0 && (!t.batched || (t.bs % 8 == 0 && t.bs > 0)),
                  "anima_attention_backward: tensors must be 16-byte aligned, row and batch strides positive multiples "
                  "of 8 elements");
  ANIMA_REQUIRE(g->workspace && g->workspace_bytes >= pl.bytes && reinterpret_cast<uintptr_t>(g->workspace) % 256 == 0,
                "anima_attention_backward: a workspace of %zu bytes (256-byte aligned) is needed, %zu are given", pl.bytes,
                g->workspace ? g->workspace_bytes : 0);
  CUtensorMap tm[7] = {};
  const CUtensorMapDataType dt =
      a->dtype == ANIMA_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const uint32_t box[3] = {64, anima::attn::TILE, 1};
  const struct {
    const void* p;
    long long ld, bs;
    int L, batch;
  } maps[4] = {{a->q, a->ldq, a->q_bstride, a->Lq, a->batch},
               {a->k, a->ldk, a->k_bstride, a->Lk, pl.kv_batch},
               {a->v, a->ldv, a->v_bstride, a->Lk, pl.kv_batch},
               {g->dout, g->lddo, g->do_bstride, a->Lq, a->batch}};
  for (int i = 0; i < 4; ++i) {
    const auto& m = maps[i];
    const uint64_t dims[3] = {static_cast<uint64_t>(m.ld), static_cast<uint64_t>(m.L), static_cast<uint64_t>(m.batch)};
    const uint64_t str[2] = {static_cast<uint64_t>(m.ld) * 2, static_cast<uint64_t>(m.batch > 1 ? m.bs : m.ld * m.L) * 2};
    st = make_tmap(&tm[i], dt, 3, m.p, dims, str, box, CU_TENSOR_MAP_SWIZZLE_128B);
    if (st) return st;
  }
  if (g->grad_dtype != ANIMA_F32) {  // dq, dk, dv: a warp's piece of a tile
    const uint32_t piece[3] = {static_cast<uint32_t>(a->head_dim) / 4, 32, 1};
    const struct {
      const void* p;
      long long ld, bs, cols;
      int L, batch;
    } outs[3] = {{g->dq, g->lddq, g->dq_bstride, cq, a->Lq, a->batch},
                 {g->dk, g->lddk, g->dk_bstride, ck, a->Lk, pl.kv_batch},
                 {g->dv, g->lddv, g->dv_bstride, ck, a->Lk, pl.kv_batch}};
    for (int i = 0; i < 3; ++i) {
      const auto& m = outs[i];
      const uint64_t dims[3] = {static_cast<uint64_t>(m.cols), static_cast<uint64_t>(m.L), static_cast<uint64_t>(m.batch)};
      const uint64_t str[2] = {static_cast<uint64_t>(m.ld) * 2, static_cast<uint64_t>(m.batch > 1 ? m.bs : m.ld * m.L) * 2};
      st = make_tmap(&tm[4 + i], dt, 3, m.p, dims, str, piece, CU_TENSOR_MAP_SWIZZLE_NONE);
      if (st) return st;
    }
  }
  unsigned char* ws = static_cast<unsigned char*>(g->workspace);
  const float scale = a->scale > 0.f ? a->scale : 1.0f / sqrtf(static_cast<float>(a->head_dim));
  Params p{};
  p.B = a->batch;
  p.H = a->heads;
  p.group = pl.group;
  p.Lq = a->Lq;
  p.Lk = a->Lk;
  p.Lqp = pl.Lqp;
  p.kv_batch = pl.kv_batch;
  p.Hk = a->heads / pl.group;
  p.kv_heads = pl.kv_batch * p.Hk;
  p.walk_heads = pl.group * (a->batch / pl.kv_batch);
  p.q_col = a->q_off;
  p.k_col = a->k_off;
  p.v_col = a->v_off;
  p.causal = a->causal ? 1 : 0;
  p.key_len = a->key_len;
  p.scale = scale;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.nlse2 = reinterpret_cast<float*>(ws + pl.lse_off);
  p.ndelta = reinterpret_cast<float*>(ws + pl.delta_off);
  p.stat = ws + pl.stat_off;
  p.top = reinterpret_cast<unsigned*>(ws + pl.top_off);
  p.dq = g->dq;
  p.dk = g->dk;
  p.dv = g->dv;
  p.lddq = g->lddq;
  p.lddk = g->lddk;
  p.lddv = g->lddv;
  p.dq_bs = many ? g->dq_bstride : 0;
  p.dk_bs = pl.kv_batch > 1 ? g->dk_bstride : 0;
  p.dv_bs = pl.kv_batch > 1 ? g->dv_bstride : 0;
  p.grad_dtype = g->grad_dtype;
  p.kv_units = pl.kv_units;
  p.q_units = pl.q_units;
  p.nkb = pl.nkb;
  p.nqb = pl.nqb;
  p.kv_splits = pl.kv_splits;
  p.q_splits = pl.q_splits;
  p.kv_part = reinterpret_cast<float*>(ws + pl.kv_off);
  p.q_part = reinterpret_cast<float*>(ws + pl.q_off);
  PrepParams pp{};
  pp.out = a->out;
  pp.dout = g->dout;
  pp.lse = g->lse;
  pp.ldo = a->ldo;
  pp.o_bs = many ? a->o_bstride : 0;
  pp.lddo = g->lddo;
  pp.do_bs = many ? g->do_bstride : 0;
  pp.out_dtype = a->out_dtype;
  pp.H = a->heads;
  pp.group = pl.group;
  pp.Lq = a->Lq;
  pp.Lqp = pl.Lqp;
  pp.kv_batch = pl.kv_batch;
  pp.shift = a->dtype == ANIMA_F16 ? kP16Shift : 0.f;
  pp.nlse2 = reinterpret_cast<float*>(ws + pl.lse_off);
  pp.ndelta = reinterpret_cast<float*>(ws + pl.delta_off);
  pp.stat = ws + pl.stat_off;
  pp.inv_scale_log2 = 1.0f / p.scale_log2;
  pp.top = reinterpret_cast<unsigned*>(ws + pl.top_off);
  if (a->dtype == ANIMA_BF16)
    return a->head_dim == 128 ? launch<true, 128>(ctx, g, pl, p, pp, tm) : launch<true, 64>(ctx, g, pl, p, pp, tm);
  return a->head_dim == 128 ? launch<false, 128>(ctx, g, pl, p, pp, tm) : launch<false, 64>(ctx, g, pl, p, pp, tm);
}
