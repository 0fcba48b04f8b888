// Masked and paged attention on the tensor cores (bf16, fp16); the mathematics is in attention_view.cuh.
//
// One CTA per 256 query rows of one sequence and head (two tiles of 128 rows that share every K and V tile), one
// CTA per SM, 12 warps:
//   warps 0-7    two softmax warpgroups, one per query tile, one thread per row (its TMEM lane).  A row's scores sit
//                in one thread's registers, so the cap, the bias, the distance and the mask are applied once, and
//                the row's maximum needs no exchange.  A tile of 128 keys is taken in parts of 64, or 32 with a cap.
//   warp 8       TMA producer: K and V tiles of 128 keys into a ring (dense: one box; paged: a box per page, pages outside
//                the sequence read a coordinate outside the pool and fill with zeros).  Thread 0 has asked for Q before.
//   warps 9, 10  one MMA stream per query tile: S(j + 1) = Q K_{j+1}^T as soon as S(j) is in registers, then
//                O += P(j) V_j.
//   warp 11      per key: bias, distance and position of the tile, into the ring (only when there are any).  Without a cap
//                bias and distance ride in the QK product: an extra K=16 chunk holds 1, 1, 1 in columns 0 to 2 of every query row and bias /
//                scale, split into three 16-bit values that add up to its 24 bits, in those of the key row (adding it
//                in the softmax measured 20% slower).  fp16, whose largest value is 65,504: 2^15 and 2^6 in columns 3 and 4 for the
//                upper parts of larger ones.
// TMEM: S_t at 128 t, P_t at 256 + 64 t (16-bit, the A operand of PV), O_t at 384 + 64 t.
//
// Most tiles are seen whole by all rows of a warp and move no row's maximum by 2^kRescale: their probabilities are formed straight from
// the products, with the maximum as it is, and the tile's maximum is looked at afterwards; the first tile, tiles that the
// mask cuts and tiles after a miss take their maximum first.  With a cap this lets its polynomial (FMA pipe) run beside the
// exponentials: 213 -> 154 us (1024 rows, 8192 keys, 37 heads; parts of 64 keys instead of 32 leave the compiler too few
// registers to interleave them: 186); without a cap 127 -> 117.  Scores beyond half the cap, and keys of mass 0 in the places
// whose exponential the FMA pipe takes, send their part of a tile the other way: 8232 rows and keys of 16 heads take 582 us
// with scores within half the cap, 1420 beyond it; without a cap 404, with one such key in every 64 485 us.
//
// The two warps of an SM sub-partition compute their exponentials at the same time and leave the unit idle at the same time
// (3200 clocks per 256 x 128 scores, 2100 of them in exponentials); making them take turns measured 8% slower, starting one
// half a tile later 6%.  An eighth of the exponentials on the FMA pipe is 6% faster.
//
// Why this shape: a wait costs 50 to 100 clocks even when what it waits for is long there, a tile's arithmetic 510
// (two warps per SM sub-partition, bound by the exponential unit) per 64 keys.  64-key steps with a wait for each
// product spent as long in waits as in arithmetic (890 clocks a step, two CTAs of 128 rows); so the softmax waits
// twice per 128 keys.  Two query tiles per CTA because two CTAs of 128 rows load K and V twice, 24 bytes per SM clock
// and more, near what L2 gives.
//
// Work that is skipped: key tiles outside the union of the rows' intervals.  Masks are evaluated in the tiles that
// some row of a warp sees in part only.  A hidden key has probability 0; what its value holds still meets that 0 in
// the PV product, so a row that comes out with a value that is not finite is computed again, key by key, by its
// warp (exact_row): rows are right whatever the hidden values are, and finite inputs pay one test per row.  Those that do not
// pay much more: 1041 rows of 16 heads over 5000 keys 65 us, with NaN in the 100 values behind them 184 ms.
//
// The last, partly filled wave of blocks is split over the keys (up to 8 parts a block).  Every part writes O, maximum
// and sum to the workspace and counts itself; the part that comes last joins all of them in order, so the result
// does not depend on which one that is.  (Parts in a cluster, joined in distributed shared memory, need whole clusters of
// SMs at a time, 128 of 148 for clusters of 8, and one split for all blocks: a frame of 1041 rows over 33,969 keys took 405 us.)
//
// The running maximum is lazy: O is rescaled only when a row's maximum grows by more than 2^8 (fp16: 2^15.9); the new one is set 2^4
// above it (fp16: 2^4 below), so that the next tiles seldom exceed it again (4% for four clips of 2058 keys).  Probabilities
// are rounded to the value type for the PV product; sums, maxima and O are fp32.
#include <cudaTypedefs.h>

#include <atomic>
#include <cstring>

#include "attention_view.cuh"
#include "host_common.h"
#include "masked_host.h"

namespace vb200 {
namespace {

constexpr int kBM = 128, kQT = 2, kBN = 128;
constexpr int kStages = 4;
constexpr int kTileBytes = kBN * kHeadDim * 2;  // 16 KB: a Q, K or V tile
constexpr int kSoftmaxWarps = 8;
constexpr int kWarpProducer = 8, kWarpMma = 9, kWarpKeys = 11;
constexpr int kThreads = 12 * 32;
// P stays <= 2^kRescale, and a row's largest P above 2^(-kMargin - 1).  bf16 has fp32's exponents, so a margin above the maximum
// costs no bits.  fp16 loses what falls below its smallest step 2^-24, so its P reach up to the type's largest value (65,504), and
// the largest stays above 2^3: a key loses at most 2^-28 of the largest probability per rounding.  (Room to grow is time: 8232 rows and
// keys with a deviation of 4 take 414 us with -3, 427 with -4, 445 with -5, 498 with -7; 427 with +4 and 2^8 as in bf16.)
template <typename T>
constexpr float kRescale = std::is_same<T, __half>::value ? 15.9f : 8.f;
template <typename T>
constexpr float kMargin = std::is_same<T, __half>::value ? -4.f : 4.f;

constexpr int kOffQ = 0;
constexpr int kOffStage = kQT * kTileBytes;
// The bias chunk of a tile: 128 rows x 16 columns, no swizzle: [16 row groups][2 column halves][8 rows][16 bytes]
constexpr int kExtraBytes = 4096;
constexpr int kOffExtra = kOffStage + kStages * 2 * kTileBytes;   // the query rows' chunk, then one per stage
constexpr int kOffKeys = kOffExtra + (1 + kStages) * kExtraBytes;  // [stage][2][128] fp32: bias, position
constexpr int kOffBar = kOffKeys + kStages * 2 * kBN * 4;
constexpr int kBarQ = 0, kBarFull = 1, kBarEmpty = kBarFull + kStages, kBarS = kBarEmpty + kStages, kBarSFree = kBarS + kQT,
              kBarP = kBarSFree + kQT, kBarO = kBarP + kQT, kBarTail = kBarO + kQT, kNumBars = kBarTail + 1;
constexpr int kOffMisc = kOffBar + kNumBars * 8;  // TMEM base; per query tile: first and last key; whether this part is the last
constexpr int kSmemBytes = kOffMisc + 32 + 1024;
constexpr int kMaxSplit = 8;
constexpr size_t kPartBytes = static_cast<size_t>(kQT) * kBM * (kHeadDim + 2) * 4;  // O, then (maximum, sum), of a block's rows
constexpr uint32_t kTmemCols = 512, kTmemP = 256, kTmemO = 384;

// S = Q K^T: four K=16 steps of head_dim 64, the first overwrites, and with use_x the bias chunk (xa, xb).
__device__ __forceinline__ void issue_qk(uint32_t d, uint64_t a, uint64_t b, uint64_t xa, uint64_t xb, uint32_t use_x, uint32_t idesc,
                                         uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred e, pf, pt, px;\n\t.reg .b64 a1, a2, a3, b1, b2, b3;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "setp.ne.b32 pf, 0, 0;\n\t"
      "setp.eq.b32 pt, 0, 0;\n\t"
      "setp.ne.and.b32 px, %7, 0, e;\n\t"
      "add.s64 a1, %1, 2;\n\tadd.s64 b1, %2, 2;\n\t"
      "add.s64 a2, %1, 4;\n\tadd.s64 b2, %2, 4;\n\t"
      "add.s64 a3, %1, 6;\n\tadd.s64 b3, %2, 6;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, pf;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a1, b1, %3, pt;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a2, b2, %3, pt;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a3, b3, %3, pt;\n\t"
      "@px tcgen05.mma.cta_group::1.kind::f16 [%0], %5, %6, %3, pt;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%4];\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(bar), "l"(xa), "l"(xb), "r"(use_x)
      : "memory");
}

// O (+)= P V over a key tile: eight K=16 steps; P in TMEM (8 columns of packed pairs a step), V MN-major (2048 bytes a
// step).  Commits to both barriers.
__device__ __forceinline__ void issue_pv(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc_first, uint32_t bar,
                                         uint32_t bar2) {
  asm volatile(
      "{\n\t.reg .pred e, pf, pt;\n\t.reg .b64 b1, b2, b3, b4, b5, b6, b7;\n\t.reg .b32 a1, a2, a3, a4, a5, a6, a7;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "setp.ne.b32 pf, %4, 0;\n\t"
      "setp.eq.b32 pt, 0, 0;\n\t"
      "add.s32 a1, %1, 8;\n\tadd.s64 b1, %2, 128;\n\t"
      "add.s32 a2, %1, 16;\n\tadd.s64 b2, %2, 256;\n\t"
      "add.s32 a3, %1, 24;\n\tadd.s64 b3, %2, 384;\n\t"
      "add.s32 a4, %1, 32;\n\tadd.s64 b4, %2, 512;\n\t"
      "add.s32 a5, %1, 40;\n\tadd.s64 b5, %2, 640;\n\t"
      "add.s32 a6, %1, 48;\n\tadd.s64 b6, %2, 768;\n\t"
      "add.s32 a7, %1, 56;\n\tadd.s64 b7, %2, 896;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, pf;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a1], b1, %3, pt;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a2], b2, %3, pt;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a3], b3, %3, pt;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a4], b4, %3, pt;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a5], b5, %3, pt;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a6], b6, %3, pt;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a7], b7, %3, pt;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%5];\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%6];\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc_first), "r"(bar), "r"(bar2)
      : "memory");
}

__device__ __forceinline__ float u2f(uint32_t u) { return __uint_as_float(u); }
__device__ __forceinline__ uint32_t f2u(float f) { return __float_as_uint(f); }

// Blocks below n_full run whole; the rest in `split` parts each.
struct TileSplit {
  int blocks;        // row blocks (an upper bound where sequences are ragged)
  int n_full, split;
  uint8_t* parts;    // [blocks * H - n_full][split][kPartBytes]
  unsigned* counters;  // [blocks * H - n_full], zero at the launch
};

// Both 16-bit halves of x times f.
template <typename T>
__device__ __forceinline__ uint32_t scale2(uint32_t x, float f) {
  const T* h = reinterpret_cast<const T*>(&x);
  const float lo = to_f32<T>(h[0]) * f, hi = to_f32<T>(h[1]) * f;
  return std::is_same<T, __nv_bfloat16>::value ? pack_bf16x2(lo, hi) : pack_f16x2(lo, hi);
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  return sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value ? pack_bf16x2(lo, hi) : pack_f16x2(lo, hi);
}

// The polynomials of tanh for cap * log2(e) * tanh(r s) / r in r^2, each coefficient twice for the packed instructions.
// A polynomial whose coefficients leave the range of normal numbers (a cap far from the scale) has limit -1 and is not used.
struct CapPoly {
  uint64_t near_[4], far_[6];
  float near_limit, far_limit;  // 1/2 and 1
};

template <int N>
__device__ __forceinline__ float max_of(const uint32_t (&r)[N]) {
  float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int c = 0; c < N; c += 8) {
#pragma unroll
    for (int u = 0; u < 4; ++u) mx[u] = fmax3(mx[u], u2f(r[c + 2 * u]), u2f(r[c + 2 * u + 1]));
  }
  return fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
}

// r <- cap * log2(e) * tanh(r s).  On the FMA pipe while no score of the warp is beyond half the cap (five packed
// instructions a pair) or the cap (seven), else two uses of the exponential unit per score.
template <int N>
__device__ __forceinline__ void cap_scores(uint32_t (&r)[N], const AttnView& a, const CapPoly& k) {
  float far = 0.f;
#pragma unroll
  for (int c = 0; c < N; c += 2) far = fmax3(far, fabsf(u2f(r[c])), fabsf(u2f(r[c + 1])));
  far *= a.scale;
  if (__all_sync(0xffffffffu, far <= k.near_limit)) {
#pragma unroll
    for (int c = 0; c < N; c += 2) {
      const uint64_t y = pk2(u2f(r[c]), u2f(r[c + 1])), z = fmul2(y, y);
      uint64_t f = ffma2(k.near_[3], z, k.near_[2]);
      f = ffma2(f, z, k.near_[1]);
      f = ffma2(f, z, k.near_[0]);
      float x0, x1;
      upk2(fmul2(f, y), x0, x1);
      r[c] = f2u(x0);
      r[c + 1] = f2u(x1);
    }
  } else if (__all_sync(0xffffffffu, far <= k.far_limit)) {
#pragma unroll
    for (int c = 0; c < N; c += 2) {
      const uint64_t y = pk2(u2f(r[c]), u2f(r[c + 1])), z = fmul2(y, y);
      uint64_t f = ffma2(k.far_[5], z, k.far_[4]);
      f = ffma2(f, z, k.far_[3]);
      f = ffma2(f, z, k.far_[2]);
      f = ffma2(f, z, k.far_[1]);
      f = ffma2(f, z, k.far_[0]);
      float x0, x1;
      upk2(fmul2(f, y), x0, x1);
      r[c] = f2u(x0);
      r[c + 1] = f2u(x1);
    }
  } else {
#pragma unroll
    for (int c = 0; c < N; ++c) r[c] = f2u(a.cap * tanh_fast(u2f(r[c]) * a.scale));
  }
}

// The scores of N keys: products in r -> scores of which mul times is the log2 domain, hidden keys at -inf.  kCap: the cap and
// the tile's values per key are applied here.  apart: the distance too, key by key.
template <bool kCap, int N>
__device__ __forceinline__ float form_scores(uint32_t (&r)[N], const AttnView& a, const CapPoly& k, const float* keys, bool apart,
                                             float slope, float pos, int lo, int hi, bool partly) {
  float mul = a.scale;
  if constexpr (kCap) {
    cap_scores(r, a, k);
#pragma unroll
    for (int c = 0; c < N; c += 4) {
      const float4 y = *reinterpret_cast<const float4*>(keys + c);
      r[c] = f2u(u2f(r[c]) + y.x);
      r[c + 1] = f2u(u2f(r[c + 1]) + y.y);
      r[c + 2] = f2u(u2f(r[c + 2]) + y.z);
      r[c + 3] = f2u(u2f(r[c + 3]) + y.w);
    }
    mul = 1.f;
  }
  if (apart) {
#pragma unroll
    for (int c = 0; c < N; c += 4) {
      const float4 y = *reinterpret_cast<const float4*>(keys + kBN + c);
      r[c] = f2u(fmaf(-slope, fabsf(pos - y.x), u2f(r[c]) * mul));
      r[c + 1] = f2u(fmaf(-slope, fabsf(pos - y.y), u2f(r[c + 1]) * mul));
      r[c + 2] = f2u(fmaf(-slope, fabsf(pos - y.z), u2f(r[c + 2]) * mul));
      r[c + 3] = f2u(fmaf(-slope, fabsf(pos - y.w), u2f(r[c + 3]) * mul));
    }
    mul = 1.f;
  }
  if (partly) {
    lo = min(max(lo, 0), N);
    hi = min(max(hi, 0), N);
#pragma unroll
    for (int w = 0; w < N / 32; ++w) {
      // bits [lo, hi) of this word of 32 columns
      const int l0 = min(max(lo - 32 * w, 0), 32), h0 = min(max(hi - 32 * w, 0), 32);
      const uint32_t up = h0 >= 32 ? 0xffffffffu : (1u << h0) - 1u;
      const uint32_t dn = l0 >= 32 ? 0u : 0xffffffffu << l0;
      const uint32_t see = up & dn;
#pragma unroll
      for (int c = 0; c < 32; ++c)
        if (!((see >> c) & 1u)) r[32 * w + c] = f2u(-INFINITY);
    }
  }
  return mul;
}

// p[c] <- (2^(r[2c] mul + off), 2^(r[2c+1] mul + off)) in 16 bits; returns the sum of the unrounded values.
template <typename T, int N>
__device__ __forceinline__ float probabilities(const uint32_t (&r)[N], float mul, float off, uint32_t* p) {
  const uint64_t neg_m2 = pk2(off, off), mul2 = pk2(mul, mul);
  uint64_t ls0 = pk2(0.f, 0.f), ls1 = pk2(0.f, 0.f);
#pragma unroll
  for (int c = 0; c < N / 2; ++c) {
    float e0, e1, q0, q1;
    upk2(ffma2(pk2(u2f(r[2 * c]), u2f(r[2 * c + 1])), mul2, neg_m2), e0, e1);
    q0 = ex2_approx(e0);
    q1 = ex2_approx(e1);
    if (c & 1) ls1 = fadd2(ls1, pk2(q0, q1));
    else ls0 = fadd2(ls0, pk2(q0, q1));
    p[c] = pack2<T>(q0, q1);
  }
  float a0, a1, b0, b1;
  upk2(ls0, a0, a1);
  upk2(ls1, b0, b1);
  return (a0 + a1) + (b0 + b1);
}

constexpr float kLeast = -125.f;  // the lowest exponent that exp2_pair takes; its 7.5e-5 are 1/52 of what rounding to bf16 may take, 1/6 for fp16

__device__ __forceinline__ float fmin3_nan(float a, float b, float c) {  // NaN if one of them is
  float d;
  asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Probabilities of keys that every row of the warp sees, straight from the products and with the maximum that the row has so far,
// so that the exponential unit, the FMA pipe (cap, exponents, sums) and the ALU (maxima) work side by side instead of one
// after the other.  False for a row whose maximum grows by more than 2^most or, with a cap, whose scores leave the polynomial's
// range: then nothing of it holds, and r is as it was.  off: what is added to a score, less the maximum; most: by how much a
// score may exceed it.  kEvery: one pair in so many takes exp2_pair; a score below its range, or NaN there, is a miss too.
template <typename T, bool kCap, int kEvery, int N>
__device__ __forceinline__ bool probabilities_at_once(const uint32_t (&r)[N], const AttnView& a, const CapPoly& k, const float* keys,
                                                      float off, float most, uint32_t* p, float& sum) {
  const uint64_t off2 = pk2(off, off), mul2 = pk2(a.scale, a.scale);
  uint64_t ls[2] = {pk2(0.f, 0.f), pk2(0.f, 0.f)};
  float top[2] = {-INFINITY, -INFINITY}, far[2] = {0.f, 0.f}, low[2] = {0.f, 0.f};
#pragma unroll
  for (int c = 0; c < N; c += 4) {
    float4 key = make_float4(0.f, 0.f, 0.f, 0.f);
    if constexpr (kCap) key = *reinterpret_cast<const float4*>(keys + c);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const float x0 = u2f(r[c + 2 * u]), x1 = u2f(r[c + 2 * u + 1]);
      const uint64_t x = pk2(x0, x1);
      uint64_t e;
      if constexpr (kCap) {
        far[u] = fmax3(far[u], fabsf(x0), fabsf(x1));
        const uint64_t z = fmul2(x, x);
        uint64_t f = ffma2(k.near_[3], z, k.near_[2]);
        f = ffma2(f, z, k.near_[1]);
        f = ffma2(f, z, k.near_[0]);
        e = fadd2(ffma2(f, x, u ? pk2(key.z, key.w) : pk2(key.x, key.y)), off2);
      } else {
        e = ffma2(x, mul2, off2);
      }
      float e0, e1;
      upk2(e, e0, e1);
      top[u] = fmax3(top[u], e0, e1);
      float q0, q1;
      if (kEvery > 0 && (c / 2 + u) % kEvery == kEvery - 1) {
        low[u] = fmin3_nan(low[u], e0, e1);
        exp2_pair(e, q0, q1);
      } else {
        q0 = ex2_approx(e0);
        q1 = ex2_approx(e1);
      }
      ls[u] = fadd2(ls[u], pk2(q0, q1));
      p[c / 2 + u] = pack2<T>(q0, q1);
    }
  }
  float a0, a1, b0, b1;
  upk2(ls[0], a0, a1);
  upk2(ls[1], b0, b1);
  sum = (a0 + a1) + (b0 + b1);
  return fmaxf(top[0], top[1]) <= most && low[0] >= kLeast && low[1] >= kLeast && (!kCap || fmaxf(far[0], far[1]) * a.scale <= k.near_limit);
}

// What the chunk's 16-bit values hold of bias / scale; their products are exact in fp32.  fp16: up to kPlainBias in columns 0 to 2,
// beyond it 2^15 c3 + 2^6 c4 + what is left, where c3 and c4 take 11 bits each.
template <typename T>
constexpr float kMostBias = std::is_same<T, __nv_bfloat16>::value ? 1e30f : 1.9e9f;
constexpr float kPlainBias = 60000.f;

// kForm: 0 plain scores; 1 with a bias, in the product; 2 with a cap, bias and distance in the softmax; 3 with a distance and no
// cap, in the product like a bias.
//
// Distance.  Where positions are token indices and all keys of a tile lie on one side of all rows, slope |pos - key| is
// slope |pos - ref|, one number per row, plus slope |ref - key|, one per key, with ref the tile's key nearest to the rows:
// the second is a bias like any other, and the first goes where the maximum is subtracted.  The few tiles among the rows'
// own positions, tiles of explicit positions and negative slopes take the distance key by key in the softmax.  (All tiles key
// by key 251 us, so 180, without a distance 160: six streams of 42 to 542 new tokens over 1900 to 9600; a frame of 1041 tokens over
// 32,928 keys 414, 311, 277.)  With a distance the
// tiles are taken last to first: a causal row then meets its largest scores first, and its maximum hardly ever grows.
//
// A bias that does not fit in the product: one below the range (the type's lowest value, say) hides its key there, as -inf
// does, and a row that ends with no probability, or with a maximum so low that such a key might count, is computed again
// by exact_row; one above the range, or NaN, makes its scores infinite or NaN, and exact_row computes those rows too.
// In the rows that stay, a key that such a bias hides could count only if its q.k were half the range, and then the rounding of its
// fp32 sum, 64 * 2^-24 of that, is 14 nats or more.  That holds from scales of 2^-8 (fp16) and 2^-76 (bf16) on; calls with smaller
// ones go to the few-row kernel.
template <typename T, bool kPaged, int kForm>
__global__ void __launch_bounds__(kThreads, 1)
    masked_attention_tc_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
                               const __grid_constant__ CUtensorMap tmap_v, const __grid_constant__ AttnView a, const TileSplit w,
                               const __grid_constant__ CapPoly poly) {
  constexpr bool kBF16 = std::is_same<T, __nv_bfloat16>::value;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // blocks in descending order, so that under causal masks the longest start first
  int item = static_cast<int>(blockIdx.x), piece = 0, split = 1;
  if (item >= w.n_full) {
    split = w.split;
    const int x = item - w.n_full;
    item = w.n_full + x / split;
    piece = x % split;
  }
  const int vb = w.blocks - 1 - item / a.H, head = item % a.H, hk = head / a.group;
  AttnSeq s;
  int blk;
  if (!locate_block<kPaged>(a, vb, kQT * kBM, 1, s, blk)) return;
  const int row_first = blk * kQT * kBM;

  auto bar = [=](int i) -> uint32_t { return sbase + kOffBar + 8 * i; };
  int* key_lo = reinterpret_cast<int*>(smem + kOffMisc + 8);
  int* key_hi = key_lo + kQT;
  volatile int* last_part = key_hi + kQT;
  // keys of a tile that are in registers at a time
  constexpr int kPart = kForm == 2 ? 32 : 64, kParts = kBN / kPart;
  // one pair of exponentials in this many on the FMA pipe, which idles beside the exponential unit (8232 rows and keys with
  // masses: 431 us without, 419 one in 16, 405 one in 8, 418 one in 4).  None with a cap, whose polynomial fills the pipe, or with a
  // distance, whose scores often lie below the polynomial's range (307 -> 337 us for a frame).
  constexpr int kEvery = kForm <= 1 ? 8 : 0;
  constexpr bool in_product = kForm == 1 || kForm == 3;
  constexpr bool per_key = kForm != 0;  // without a bias and a distance form 2's ring holds zeros

  if (threadIdx.x == 0) {
    mbar_init(bar(kBarQ), 1);
    mbar_init(bar(kBarTail), 1);
    for (int i = 0; i < kStages; ++i) {
      mbar_init(bar(kBarFull + i), per_key ? 2 : 1);
      mbar_init(bar(kBarEmpty + i), kQT);
    }
    for (int t = 0; t < kQT; ++t) {
      mbar_init(bar(kBarS + t), 1);
      mbar_init(bar(kBarSFree + t), 4);
      mbar_init(bar(kBarP + t), 4);
      mbar_init(bar(kBarO + t), 1);
      key_lo[t] = 0x7fffffff;
      key_hi[t] = 0;
    }
    fence_barrier_init();
    // the query rows are on their way before the keys are known
    mbar_arrive_expect_tx(bar(kBarQ), kQT * kTileBytes);
    for (int t = 0; t < kQT; ++t)
      tma_load_4d(sbase + kOffQ + t * kTileBytes, &tmap_q, bar(kBarQ), 0, s.row0 + row_first + t * kBM, head, s.batch);
  }
  if (warp == kWarpMma) {
    tmem_alloc(sbase + kOffMisc, kTmemCols);
    tmem_relinquish();
  }
  if constexpr (in_product) {
    // the query rows' chunk: 1, 1, 1 in columns 0 to 2, fp16 also 2^15 and 2^6; the key rows' chunks: zero beyond
    const uint32_t one = kBF16 ? 0x3F80u : 0x3C00u, upper = kBF16 ? 0u : 0x7800u, middle = kBF16 ? 0u : 0x5400u;
    for (int x = threadIdx.x; x < (1 + kStages) * kExtraBytes / 16; x += kThreads) {
      const bool q = x < kExtraBytes / 16 && ((x >> 3) & 1) == 0;
      *reinterpret_cast<uint4*>(smem + kOffExtra + 16 * x) = make_uint4(q ? one | one << 16 : 0u, q ? one | upper << 16 : 0u, q ? middle : 0u, 0u);
    }
    fence_proxy_async_smem();  // generic writes become visible to the tensor core
  }
  if (warp == kWarpProducer && lane == 0) {
    prefetch_tmap(&tmap_q);
    prefetch_tmap(&tmap_k);
    prefetch_tmap(&tmap_v);
  }
  int2 be = make_int2(0, 0);  // keys of this thread's row
  const bool valid = warp < kSoftmaxWarps && row_first + static_cast<int>(threadIdx.x) < s.rows;
  if (valid) be = row_range<kPaged>(a, s, row_first + threadIdx.x);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem + kOffMisc);
  if (warp < kSoftmaxWarps) {
    const int lo = __reduce_min_sync(0xffffffffu, be.y > be.x ? be.x : 0x7fffffff);
    const int hi = __reduce_max_sync(0xffffffffu, be.y);
    if (lane == 0 && hi > 0) {
      atomicMin(&key_lo[warp >> 2], lo);
      atomicMax(&key_hi[warp >> 2], hi);
    }
  }
  __syncthreads();
  // key tiles [j0, j1) of each query tile, [p0, p1) of this CTA's part of their union
  int j0[kQT], j1[kQT], p0 = 0x7fffffff, p1 = 0;
#pragma unroll
  for (int t = 0; t < kQT; ++t) {
    const int hi = key_hi[t];
    j0[t] = hi > 0 ? key_lo[t] / kBN : 0;
    j1[t] = (hi + kBN - 1) / kBN;
    if (hi > 0) {
      p0 = min(p0, j0[t]);
      p1 = max(p1, j1[t]);
    }
  }
  if (p1 == 0) p0 = 0;
  {
    const int first = p0, n = p1 - p0;
    p0 = first + static_cast<int>(static_cast<long long>(n) * piece / split);
    p1 = first + static_cast<int>(static_cast<long long>(n) * (piece + 1) / split);
  }
#pragma unroll
  for (int t = 0; t < kQT; ++t) {
    j0[t] = min(max(j0[t], p0), p1);
    j1[t] = max(min(j1[t], p1), j0[t]);
  }
  if (j0[0] == j1[0] && j0[1] == j1[1]) p1 = p0;  // the part lies between the two query tiles' keys

  // Tiles are counted by u from 0 to n_tiles; first to last, or last to first with a distance.  Query tile t takes [ua, ub).
  const int n_tiles = p1 - p0;
  const bool down = kForm == 3 || (kForm == 2 && a.slope != nullptr);
  auto tile_of = [=](int u) -> int { return down ? p1 - 1 - u : p0 + u; };
  int ua[kQT], ub[kQT];
#pragma unroll
  for (int t = 0; t < kQT; ++t) {
    ua[t] = down ? p1 - j1[t] : j0[t] - p0;
    ub[t] = down ? p1 - j0[t] : j1[t] - p0;
    if (n_tiles == 0) ua[t] = ub[t] = 0;
  }
  const float slope = down ? __ldg(a.slope + head) * kLog2E : 0.f;
  const bool by_side = down && a.qpos == nullptr && a.kpos == nullptr && slope >= 0.f;
  const int pos_first = s.keys - s.rows + row_first;
  // 1: all keys of the tile at or before all rows; -1: at or behind; 0: neither, or not asked
  auto side_of = [=](int j) -> int {
    return !by_side ? 0 : j * kBN + kBN - 1 <= pos_first ? 1 : j * kBN >= pos_first + kQT * kBM - 1 ? -1 : 0;
  };

  // Paged: the tile whose last page the sequence fills in part.  The slots behind the last key hold anything, NaN perhaps, so
  // their values are overwritten with zeros before the PV product reads them: by warp 11, which takes the tiles in order, and
  // without values per key by the producer behind its last tile.  -1: none in this part.
  int tail = -1;
  if (kPaged && (s.keys & (kBN - 1)) != 0) {
    const int j = s.keys / kBN;
    if ((j >= j0[0] && j < j1[0]) || (j >= j0[1] && j < j1[1])) tail = down ? p1 - 1 - j : j - p0;
  }

  // Called by a warp that is in step with the ring: it knows that the fills of the tail's stage before the tail have landed, and
  // no later one starts before kBarTail.  (A parity says which of two fills has landed, no more: a warp that comes to it from the
  // start would take another tile for the tail.)  Whole rows, so the swizzle inside a row does not matter.
  auto clear_tail = [&]() -> bool {
    const int st = tail % kStages;
    const bool ok = __all_sync(0xffffffffu, mbar_wait(bar(kBarFull + st), (tail / kStages) & 1, a.err));
    uint4* v = reinterpret_cast<uint4*>(smem + kOffStage + (2 * st + 1) * kTileBytes);
    for (int x = (s.keys & (kBN - 1)) * 8 + lane; ok && x < kBN * 8; x += 32) v[x] = make_uint4(0u, 0u, 0u, 0u);
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0 && ok) mbar_arrive(bar(kBarTail));
    return ok;
  };

  // A wait that runs out makes its role go on without waiting (or leave), so that every thread reaches the end and
  // TMEM is freed.
  if (warp >= kSoftmaxWarps) {
    if (warp == kWarpProducer) {
      // ------------------------------- producer -------------------------------
      const int npg = kPaged ? kBN >> a.page_shift : 1;       // boxes per tile
      const int which = lane / npg, pg = lane - which * npg;  // K (0) or V (1), box of the tile
      auto page_at = [&](int j) -> int {
        const int slot = ((j * kBN) >> a.page_shift) + pg;
        return static_cast<long long>(slot) << a.page_shift < s.keys ? page_of(a, s, slot) : a.pages;
      };
      int id = 0;
      if (kPaged && which < 2 && n_tiles > 0) id = page_at(tile_of(0));
      if (n_tiles == 0) mbar_wait(bar(kBarQ), 0, a.err);  // the query rows land before the CTA leaves
      int n = 0;
      bool ok = true;
      for (; n < n_tiles; ++n) {
        const int st = n % kStages;
        if (n >= kStages) ok = __all_sync(0xffffffffu, mbar_wait(bar(kBarEmpty + st), (n / kStages - 1) & 1, a.err));
        if (!ok) break;
        // a tile between the two query tiles' keys is not loaded
        const bool used = (n >= ua[0] && n < ub[0]) || (n >= ua[1] && n < ub[1]);
        if (lane == 0) {
          if (used) mbar_arrive_expect_tx(bar(kBarFull + st), 2 * kTileBytes);
          else mbar_arrive(bar(kBarFull + st));
        }
        __syncwarp();
        const uint32_t dst = sbase + kOffStage + st * 2 * kTileBytes;
        if constexpr (kPaged) {
          if (which < 2) {
            if (used)
              tma_load_4d(dst + which * kTileBytes + pg * (kTileBytes / npg), which ? &tmap_v : &tmap_k, bar(kBarFull + st), 0, hk, 0, id);
            if (n + 1 < n_tiles) id = page_at(tile_of(n + 1));
          }
        } else if (lane < 2 && used) {
          tma_load_4d(dst + lane * kTileBytes, lane ? &tmap_v : &tmap_k, bar(kBarFull + st), 0, tile_of(n) * kBN, hk, s.batch);
        }
      }
      if (!ok) {  // the copies in flight land before the CTA leaves
        mbar_wait(bar(kBarQ), 0, a.err);
        for (int u = max(n - kStages, 0); u < n; ++u) mbar_wait(bar(kBarFull + u % kStages), (u / kStages) & 1, a.err);
      }
      // tiles first to last, so the tail, where there is one, is the last that was asked for
      if (kPaged && !per_key && ok && tail >= 0) clear_tail();
    } else if (warp < kWarpMma + kQT) {
      // ------------------------------- MMA issuer of query tile t -------------------------------
      const int t = warp - kWarpMma;
      const int ja = t == 0 ? ua[0] : ua[1], jb = t == 0 ? ub[0] : ub[1];
      constexpr uint32_t idesc_qk = idesc_f16(kBM, kBN, kBF16 ? 1 : 0, 0, 0);
      constexpr uint32_t idesc_pv = idesc_f16(kBM, kHeadDim, kBF16 ? 1 : 0, 0, 1);
      const uint64_t q_desc = smem_desc_sw128(sbase + kOffQ + t * kTileBytes, 16, 1024);
      const uint64_t k_desc = smem_desc_sw128(sbase + kOffStage, 16, 1024);
      const uint64_t v_desc = smem_desc_sw128(sbase + kOffStage + kTileBytes, 16384, 1024);
      auto stage_off = [=](int j) -> uint64_t { return static_cast<uint64_t>((j % kStages) * (2 * kTileBytes >> 4)); };
      auto wait_all = [&](int b, int parity) -> bool {
        return __all_sync(0xffffffffu, mbar_wait(bar(b), static_cast<uint32_t>(parity), a.err));
      };
      auto full = [&](int j) -> bool { return wait_all(kBarFull + j % kStages, (j / kStages) & 1); };
      const uint64_t qx_desc = smem_desc_noswz(sbase + kOffExtra, 128, 256);
      const uint64_t kx_desc = smem_desc_noswz(sbase + kOffExtra + kExtraBytes, 128, 256);
      auto qk = [&](int j) {
        issue_qk(tmem + t * 128, q_desc, k_desc + stage_off(j), qx_desc,
                 kx_desc + static_cast<uint64_t>((j % kStages) * (kExtraBytes >> 4)), in_product ? 1u : 0u, idesc_qk, bar(kBarS + t));
      };
      bool ok = true;
      // tiles that only the other query tile reads are released as they come
      for (int j = 0; j < ja && ok; ++j) {
        ok = full(j);
        if (ok && lane == 0) mbar_arrive(bar(kBarEmpty + j % kStages));
      }
      if (ok && ja < jb) {
        ok = wait_all(kBarQ, 0) && full(ja);
        tc_fence_after();
        if (ok) qk(ja);
      }
      for (int j = ja; j < jb && ok; ++j) {
        const int n = j - ja;
        if (j + 1 < jb) {
          ok = full(j + 1) && wait_all(kBarSFree + t, n & 1);
          if (!ok) break;
          tc_fence_after();
          qk(j + 1);
        }
        ok = wait_all(kBarP + t, n & 1) && (!kPaged || j != tail || wait_all(kBarTail, 0));
        if (!ok) break;
        tc_fence_after();
        issue_pv(tmem + kTmemO + t * kHeadDim, tmem + kTmemP + t * kHeadDim, v_desc + stage_off(j), idesc_pv, n > 0 ? 1u : 0u,
                 bar(kBarO + t), bar(kBarEmpty + j % kStages));
      }
      for (int j = jb; j < n_tiles && ok; ++j) {
        ok = full(j);
        if (ok && lane == 0) mbar_arrive(bar(kBarEmpty + j % kStages));
      }
    } else if (warp == kWarpKeys) {
      // ------------------------------- per-key bias and position -------------------------------
      const float inv = 1.f / a.scale;  // a.scale = scale * log2(e) without a cap
      bool ok = true;
      for (int n = 0; per_key && n < n_tiles && ok; ++n) {
        const int j = tile_of(n), st = n % kStages, side = side_of(j);
        float b[4], kp[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int key = j * kBN + u * 32 + lane;
          b[u] = kp[u] = 0.f;
          if (key < s.keys) {
            long long at = s.batch * a.bias_sb + key;
            bool there = true;
            if constexpr (kPaged) {
              const int id = page_of(a, s, key >> a.page_shift);
              there = id < a.pages;
              at = (static_cast<long long>(id) << a.page_shift) + (key & ((1 << a.page_shift) - 1));
            }
            if (a.bias != nullptr && there) b[u] = __ldg(a.bias + at);
            if (down) kp[u] = key_position<kPaged>(a, s, position_origin<kPaged>(a, s, row_first), key);
          }
        }
        if (n >= kStages) ok = __all_sync(0xffffffffu, mbar_wait(bar(kBarEmpty + st), (n / kStages - 1) & 1, a.err));
        if (!ok) break;
        float* dst = reinterpret_cast<float*>(smem + kOffKeys) + st * 2 * kBN;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int k = u * 32 + lane;
          const float away = side > 0 ? slope * static_cast<float>(k - (kBN - 1)) : side < 0 ? -slope * static_cast<float>(k) : 0.f;
          if (down) dst[kBN + k] = kp[u];
          if constexpr (in_product) {
            float x = fmaf(b[u], kLog2E, away) * inv, mid = 0.f, lo = 0.f, c3 = 0.f, c4 = 0.f;
            if (fabsf(x) <= kMostBias<T>) {
              if (!kBF16 && fabsf(x) > kPlainBias) {
                c3 = to_f32<T>(from_f32<T>(x * 0x1p-15f));
                x = fmaf(c3, -0x1p15f, x);
                c4 = to_f32<T>(from_f32<T>(x * 0x1p-6f));
                x = fmaf(c4, -0x1p6f, x);
              }
              const float hi = to_f32<T>(from_f32<T>(x));
              mid = to_f32<T>(from_f32<T>(x - hi));
              lo = x - hi - mid;
              x = hi;
            } else {
              x = x < 0.f ? -INFINITY : x > 0.f ? INFINITY : x;
            }
            uint8_t* chunk = smem + kOffExtra + (1 + st) * kExtraBytes + (k >> 3) * 256 + (k & 7) * 16;
            if constexpr (kBF16) *reinterpret_cast<uint2*>(chunk) = make_uint2(pack2<T>(x, mid), pack2<T>(lo, 0.f));
            else *reinterpret_cast<uint4*>(chunk) = make_uint4(pack2<T>(x, mid), pack2<T>(lo, c3), pack2<T>(c4, 0.f), 0u);
          } else {
            dst[k] = bias_log2(b[u]) + away;
          }
        }
        if constexpr (in_product) fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(kBarFull + st));
        if (kPaged && n == tail) ok = clear_tail();
      }
    }
  } else {
    // ------------------------------- softmax -------------------------------
    const int t = warp >> 2;
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t s_addr = tmem + lane_off + t * 128;
    const uint32_t p_addr = tmem + lane_off + kTmemP + t * kHeadDim;
    const uint32_t o_addr = tmem + lane_off + kTmemO + t * kHeadDim;
    const int i = row_first + t * kBM + row;  // token of the sequence
    const float pos = by_side ? static_cast<float>(t * kBM + row) : down && valid ? row_position<kPaged>(a, s, position_origin<kPaged>(a, s, row_first), i) : 0.f;
    // keys that every row of the warp sees
    const int all_lo = __reduce_max_sync(0xffffffffu, valid ? be.x : 0);
    const int all_hi = __reduce_min_sync(0xffffffffu, valid ? be.y : 0x7fffffff);
    const int ja = t == 0 ? ua[0] : ua[1], jb = t == 0 ? ub[0] : ub[1];
    float m_run = -INFINITY, l_run = 0.f;  // the running maximum is a whole number, so that a rescaling is exact
    int rest = 1, back = 0;  // tiles until the next try at once: not the first, whose maximum is unknown, and more after each miss
    bool ok = true;
    auto wait_for = [&](int b, int parity) {
      if (ok) ok = mbar_wait(bar(b), static_cast<uint32_t>(parity), a.err);
    };

#pragma unroll 1
    for (int u = ja; u < jb; ++u) {
      const int n = u - ja, st = u % kStages, j = tile_of(u);
      const int side = side_of(j);
      const bool apart = down && side == 0;
      {
        // the scores and, for the softmax, the tile's keys, looked at together
        const uint32_t ps = n & 1, pf = (u / kStages) & 1;
        const bool wait_keys = kForm == 2 || apart;
        const bool s_there = mbar_try_wait(bar(kBarS + t), ps), keys_there = !wait_keys || mbar_try_wait(bar(kBarFull + st), pf);
        if (!s_there) wait_for(kBarS + t, ps);
        if (!keys_there) wait_for(kBarFull + st, pf);
      }
      __syncwarp();
      tc_fence_after();
      const float* keys = reinterpret_cast<const float*>(smem + kOffKeys) + st * 2 * kBN;
      const int key0 = j * kBN;
      // what the row's own distance adds to every score of the tile
      const float rel = static_cast<float>(key0 - pos_first);
      const float add = side == 0 ? 0.f : -slope * (side > 0 ? pos - (rel + static_cast<float>(kBN - 1)) : rel - pos);
      uint32_t r[kPart];
      auto load = [&](int h) {
#pragma unroll
        for (int c = 0; c < kPart; c += 32)
          tmem_ld32x32b_x32_nowait(s_addr + h * kPart + c, *reinterpret_cast<uint32_t(*)[32]>(&r[c]));
        tmem_wait_ld();
#pragma unroll
        for (int c = 0; c < kPart; c += 32) reg_fence32(*reinterpret_cast<uint32_t(*)[32]>(&r[c]));
        if (h == kParts - 1) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(kBarSFree + t));
        }
      };
      auto o_at_rest = [&] {  // PV(n - 1) has read P, and O is at rest
        if (n == 0) return;
        wait_for(kBarO + t, (n - 1) & 1);
        __syncwarp();
        tc_fence_after();
      };
      auto store = [&](int h, const uint32_t (&p)[kPart / 2]) {
        if constexpr (kPart == 64) tmem_st32x32b_x32(p_addr + h * 32, *reinterpret_cast<const uint32_t(*)[32]>(&p[0]));
        else tmem_st32x32b_x16(p_addr + h * 16, *reinterpret_cast<const uint32_t(*)[16]>(&p[0]));
      };
      int h = 0;           // parts of the tile that are done
      bool loaded = false;  // part h is in r
      if (!apart && key0 >= all_lo && key0 + kBN <= all_hi && --rest < 0) {
#pragma unroll
        for (int g = 0; g < kParts; ++g) {
          if (g != h) continue;  // an earlier part missed
          load(g);
          uint32_t p[kPart / 2];
          float sum;
          const bool none = m_run == -INFINITY;
          if (__all_sync(0xffffffffu, probabilities_at_once<T, kForm == 2, kEvery>(r, a, poly, keys + g * kPart, none ? add : add - m_run,
                                                                           none ? -INFINITY : kRescale<T>, p, sum))) {
            l_run += sum;
            if (g == 0) o_at_rest();
            store(g, p);
            h = g + 1;
          } else {
            loaded = true;
            break;
          }
        }
        back = h == kParts ? 0 : min(2 * back + 1, 15);
        rest = h == kParts ? 0 : back >> 1;
      }
#pragma unroll 1
      for (; h < kParts; ++h) {
        if (!loaded) load(h);
        loaded = false;
        const int first = key0 + h * kPart;
        const float mul = form_scores<kForm == 2>(r, a, poly, keys + h * kPart, apart, slope, pos, be.x - first, be.y - first,
                                                  first < all_lo || first + kPart > all_hi);
        const float m_new = fmaf(max_of(r), mul, add);
        const bool grow = m_new > m_run + kRescale<T>;
        const bool need = __any_sync(0xffffffffu, grow);
        float f = 1.f;  // what O, and the probabilities of the parts before, are to be multiplied by
        if (need) {
          const float m_tgt = grow ? ceilf(m_new) + kMargin<T> : m_run;
          f = grow ? ex2_approx(m_run - m_tgt) : 1.f;
          l_run *= f;
          m_run = m_tgt;
        }
        uint32_t p[kPart / 2];
        l_run += probabilities<T>(r, mul, add - (m_run == -INFINITY ? 0.f : m_run), p);
        if (h == 0) o_at_rest();
        if (need) {
          if (n > 0) {
#pragma unroll 1
            for (int c = 0; c < kHeadDim; c += 16) {
              uint32_t o[16];
              tmem_ld32x32b_x16(o_addr + c, o);
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = f2u(u2f(o[e]) * f);
              tmem_st32x32b_x16(o_addr + c, o);
            }
          }
          // by a power of two: exactly, but for what fp16 holds in less than 11 bits, which rounds to its step once more
#pragma unroll 1
          for (int c = 0; c < h * (kPart / 2); c += 16) {
            uint32_t o[16];
            tmem_wait_st();
            tmem_ld32x32b_x16(p_addr + c, o);
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = scale2<T>(o[e], f);
            tmem_st32x32b_x16(p_addr + c, o);
          }
        }
        store(h, p);
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(kBarP + t));
    }
    uint32_t o[kHeadDim];
#pragma unroll
    for (int c = 0; c < kHeadDim; ++c) o[c] = 0u;
    if (jb > ja) {
      wait_for(kBarO + t, (jb - ja - 1) & 1);
      __syncwarp();
      tc_fence_after();
      tmem_ld32x32b_x32_nowait(o_addr, *reinterpret_cast<uint32_t(*)[32]>(&o[0]));
      tmem_ld32x32b_x32_nowait(o_addr + 32, *reinterpret_cast<uint32_t(*)[32]>(&o[32]));
      tmem_wait_ld();
      reg_fence32(*reinterpret_cast<uint32_t(*)[32]>(&o[0]));
      reg_fence32(*reinterpret_cast<uint32_t(*)[32]>(&o[32]));
    }
    const bool write = valid && ok;
    uint4* orow = reinterpret_cast<uint4*>(static_cast<uint8_t*>(a.out) + 2 * (s.batch * a.o_sb + head * a.o_sh + (s.row0 + i) * a.o_sn));
    float z = 0.f;  // NaN unless every value of the row is finite
    auto put8 = [&](int c, const float (&x)[8], float inv, bool none) {
      uint32_t v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        z = fmaf(x[2 * e], 0.f, fmaf(x[2 * e + 1], 0.f, z));
        v[e] = pack2<T>(x[2 * e] * inv, x[2 * e + 1] * inv);
      }
      orow[c] = none ? make_uint4(0u, 0u, 0u, 0u) : make_uint4(v[0], v[1], v[2], v[3]);  // no visible key: 0
    };
    bool again = false;
    // rows for exact_row: not finite, or only keys whose bias did not fit
    auto redo = [&](bool not_finite) {
      return not_finite || (in_product && (kForm == 1 || a.bias != nullptr || slope * (kBN - 1) > kMostBias<T> * a.scale) && be.y > be.x && (l_run == 0.f || m_run < -0.5f * kMostBias<T> * a.scale));
    };
    if (split > 1) {
      // columns of four, rows side by side: [16][256] float4, so that a warp's stores and loads are whole lines
      const size_t slot0 = static_cast<size_t>(item - w.n_full) * split;
      auto part_o = [&](int k) { return reinterpret_cast<float4*>(w.parts + (slot0 + k) * kPartBytes) + t * kBM + row; };
      auto part_ml = [&](int k) {
        return reinterpret_cast<float2*>(w.parts + (slot0 + k) * kPartBytes + static_cast<size_t>(kQT) * kBM * kHeadDim * 4) + t * kBM + row;
      };
      if (jb > ja) {
#pragma unroll
        for (int c = 0; c < kHeadDim / 4; ++c)
          part_o(piece)[c * kQT * kBM] = make_float4(u2f(o[4 * c]), u2f(o[4 * c + 1]), u2f(o[4 * c + 2]), u2f(o[4 * c + 3]));
      }
      *part_ml(piece) = make_float2(m_run, l_run);
      __threadfence();
      named_bar_sync(1, kSoftmaxWarps * 32);
      if (threadIdx.x == 0)
        *last_part = atomicAdd(w.counters + (item - w.n_full), 1u) == static_cast<unsigned>(split - 1);
      named_bar_sync(1, kSoftmaxWarps * 32);
      if (write && *last_part != 0) {
        __threadfence();
        float f[kMaxSplit];
        m_run = -INFINITY;
#pragma unroll
        for (int k = 0; k < kMaxSplit; ++k)
          if (k < split) m_run = fmaxf(m_run, __ldcg(part_ml(k)).x);
        const float mu = m_run == -INFINITY ? 0.f : m_run;
        l_run = 0.f;
#pragma unroll
        for (int k = 0; k < kMaxSplit; ++k) {
          f[k] = 0.f;
          if (k < split) {
            const float2 ml = __ldcg(part_ml(k));
            if (ml.y != 0.f) {  // a part without keys of this row has no O
              f[k] = ex2_approx(ml.x - mu);
              l_run = fmaf(ml.y, f[k], l_run);
            }
          }
        }
        const float inv = 1.f / l_run;
#pragma unroll 1
        for (int c = 0; c < kHeadDim / 8; ++c) {
          float4 y[kMaxSplit][2];
#pragma unroll
          for (int k = 0; k < kMaxSplit; ++k) {
            if (k < split && f[k] != 0.f) {
              y[k][0] = __ldcg(part_o(k) + 2 * c * kQT * kBM);
              y[k][1] = __ldcg(part_o(k) + (2 * c + 1) * kQT * kBM);
            } else {
              y[k][0] = y[k][1] = make_float4(0.f, 0.f, 0.f, 0.f);
            }
          }
          float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int k = 0; k < kMaxSplit; ++k) {
            x[0] = fmaf(y[k][0].x, f[k], x[0]);
            x[1] = fmaf(y[k][0].y, f[k], x[1]);
            x[2] = fmaf(y[k][0].z, f[k], x[2]);
            x[3] = fmaf(y[k][0].w, f[k], x[3]);
            x[4] = fmaf(y[k][1].x, f[k], x[4]);
            x[5] = fmaf(y[k][1].y, f[k], x[5]);
            x[6] = fmaf(y[k][1].z, f[k], x[6]);
            x[7] = fmaf(y[k][1].w, f[k], x[7]);
          }
          put8(c, x, inv, l_run == 0.f);
        }
        again = redo(l_run != 0.f && !(z * inv == 0.f));
      }
    } else if (write) {
      const float inv = 1.f / l_run;
#pragma unroll
      for (int c = 0; c < kHeadDim / 8; ++c) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = u2f(o[8 * c + e]);
        put8(c, x, inv, l_run == 0.f);
      }
      again = redo(l_run != 0.f && !(z * inv == 0.f));
    }
    __syncwarp();  // a row's first result is written before its second
    unsigned rows = __ballot_sync(0xffffffffu, again);
    while (rows) {
      const int e = __ffs(rows) - 1;
      rows &= rows - 1;
      exact_row<T, kPaged>(a, s, row_first + warp * 32 + e, head);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kWarpMma) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

template <typename T, bool kPaged, int kForm>
int launch_form(const AttnView& a, const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const TileSplit& w, long long grid,
                cudaStream_t st) {
  auto kernel = masked_attention_tc_kernel<T, kPaged, kForm>;
  // per device: the opt-in to the shared memory
  static std::atomic<bool> ready[64];
  int dev = 0;
  VB200_CHECK_CUDA(cudaGetDevice(&dev), "cudaGetDevice");
  if (dev < 0 || dev >= 64 || !ready[dev].load(std::memory_order_acquire)) {
    VB200_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes), "cudaFuncSetAttribute");
    if (dev >= 0 && dev < 64) ready[dev].store(true, std::memory_order_release);
  }
  CapPoly poly{};
  if (kForm == 2) {
    auto twice = [](double x) {
      const float f = static_cast<float>(x);
      uint32_t u;
      memcpy(&u, &f, 4);
      return static_cast<uint64_t>(u) << 32 | u;
    };
    const double s2 = static_cast<double>(a.scale) * a.scale;
    double f = static_cast<double>(a.cap) * a.scale;
    poly.near_limit = 0.5f;
    poly.far_limit = 1.f;
    for (int i = 0; i < 6; ++i, f *= s2) {
      const bool normal = f > 1e-34 && f < 1e34;
      if (i < 4) poly.near_[i] = twice(kTanhNear[i] * f);
      poly.far_[i] = twice(kTanhFar[i] * f);
      if (i < 4 && !normal) poly.near_limit = -1.f;
      if (!normal) poly.far_limit = -1.f;
    }
  }
  kernel<<<static_cast<unsigned>(grid), kThreads, kSmemBytes, st>>>(tq, tk, tv, a, w, poly);
  VB200_CHECK_LAUNCH("masked_attention_tc_kernel");
  return VB200_OK;
}

template <typename T, bool kPaged>
int launch(const AttnView& a, const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const TileSplit& w, long long grid,
           cudaStream_t st) {
  if (a.cap != 0.f) return launch_form<T, kPaged, 2>(a, tq, tk, tv, w, grid, st);
  if (a.slope != nullptr) return launch_form<T, kPaged, 3>(a, tq, tk, tv, w, grid, st);
  return a.bias != nullptr ? launch_form<T, kPaged, 1>(a, tq, tk, tv, w, grid, st) : launch_form<T, kPaged, 0>(a, tq, tk, tv, w, grid, st);
}

// One CTA per SM: the items (row blocks x heads) run whole while they fill waves of all SMs; those of the last wave in
// k parts each take ceil(rest * k / SMs) rounds of 1/k of an item plus a ramp of about three key tiles.  The cheapest k.
struct Plan {
  long long blocks, items, n_full;
  int split;
  size_t counter_bytes, bytes;
};

Plan plan_of(bool paged, long long rows, long long seqs, long long H, long long most_keys, int sms) {
  Plan p{};
  p.blocks = paged ? rows / (kQT * kBM) + seqs : (rows + kQT * kBM - 1) / (kQT * kBM) * seqs;
  p.items = p.n_full = p.blocks * H;
  p.split = 1;
  const double tiles = static_cast<double>((most_keys + kBN - 1) / kBN), ramp = 3.0 / tiles;
  const long long rest = sms > 0 ? p.items % sms : 0;
  if (rest == 0) return p;
  double best = 1.0 + ramp;
  for (int k = 2; k <= kMaxSplit && 2 * k <= tiles; ++k) {
    const double cost = static_cast<double>((rest * k + sms - 1) / sms) * (1.0 / k + ramp);
    if (cost < best - 1e-9) {
      best = cost;
      p.split = k;
    }
  }
  if (p.split > 1) {
    p.n_full = p.items - rest;
    p.counter_bytes = align_up(static_cast<size_t>(rest) * sizeof(unsigned), 256);
    p.bytes = p.counter_bytes + static_cast<size_t>(rest) * p.split * kPartBytes;
  }
  return p;
}

}  // namespace

size_t tile_attention_workspace(bool paged, long long rows, long long seqs, long long H, long long most_keys) {
  return plan_of(paged, rows, seqs, H, most_keys, sm_count_of_device()).bytes;
}

int tile_attention(int dtype, bool paged, const AttnView& a, long long most_keys, void* workspace, size_t workspace_bytes, cudaStream_t st) {
  Plan p = plan_of(paged, a.Nq, paged ? a.n_seq : a.B, a.H, most_keys, sm_count_of_device());
  // Whole blocks where there is no room for parts, and where rows have intervals and the blocks fill a wave: they see fewer keys
  // than the plan counts, and their parts are mostly start and end (four clips of 2058 keys: 143 -> 129 us; 4116 rows that see
  // all of 32,928 keys: 1135 -> 1150).
  if (p.split > 1 && (workspace == nullptr || workspace_bytes < p.bytes || (a.range != nullptr && p.n_full > 0))) {
    p.split = 1;
    p.n_full = p.items;
  }
  const long long grid = p.n_full + (p.items - p.n_full) * p.split;
  VB200_REQUIRE(grid < (1ll << 31), "attention: too many work items");
  TileSplit w{};
  w.blocks = static_cast<int>(p.blocks);
  w.n_full = static_cast<int>(p.n_full);
  w.split = p.split;
  if (p.split > 1) {
    VB200_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 255u) == 0, "attention: workspace must be 256-byte aligned");
    w.counters = static_cast<unsigned*>(workspace);
    w.parts = static_cast<uint8_t*>(workspace) + p.counter_bytes;
    VB200_CHECK_CUDA(cudaMemsetAsync(w.counters, 0, p.counter_bytes, st), "zeroing the counters");
  }
  CUtensorMap tq, tk, tv;
  int rc = rows_map(&tq, a.q, dtype, a.Nq, a.H, paged ? 1 : a.B, a.q_sn, a.q_sh, a.q_sb, kBM);
  if (rc != VB200_OK) return rc;
  if (paged) {
    if ((rc = pool_map(&tk, a.k, dtype, a, kBN)) != VB200_OK || (rc = pool_map(&tv, a.v, dtype, a, kBN)) != VB200_OK) return rc;
    return dtype == VB200_BF16 ? launch<__nv_bfloat16, true>(a, tq, tk, tv, w, grid, st) : launch<__half, true>(a, tq, tk, tv, w, grid, st);
  }
  if ((rc = rows_map(&tk, a.k, dtype, a.Nk, a.Hkv, a.B, a.k_sn, a.k_sh, a.k_sb, kBN)) != VB200_OK ||
      (rc = rows_map(&tv, a.v, dtype, a.Nk, a.Hkv, a.B, a.v_sn, a.v_sh, a.v_sb, kBN)) != VB200_OK)
    return rc;
  return dtype == VB200_BF16 ? launch<__nv_bfloat16, false>(a, tq, tk, tv, w, grid, st) : launch<__half, false>(a, tq, tk, tv, w, grid, st);
}

}  // namespace vb200
