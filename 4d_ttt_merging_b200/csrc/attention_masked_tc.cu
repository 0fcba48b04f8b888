// Masked and paged attention on the tensor cores (bf16, fp16); the mathematics is in attention_view.cuh.
//
// One CTA per 256 query rows of one sequence and head (two tiles of 128 rows), one CTA per SM, 12 warps:
//   warps 0-7   two softmax warpgroups, one per query tile, one thread per row (its TMEM lane).  A row's
//               scores of a key tile sit in one thread's registers, so the cap, the bias, the distance and the
//               mask are applied once, and the row's maximum needs no exchange.
//   warp 8      TMA producer: Q once; K and V tiles of 128 keys into a ring (dense: one box; paged: a box per page,
//               pages outside the sequence read a coordinate outside the pool and fill with zeros).
//   warp 9      TMEM and the MMA stream: S_t = Q_t K_j^T one tile ahead, O_t += P_t V_j, as the softmax releases them.
//   warp 10     per key: bias and position of the tile, into the ring (only when there are any).
// TMEM: S_t at 128 t, P_t at 256 + 64 t (16-bit, the A operand of PV), O_t at 384 + 64 t.
//
// Work that is skipped: key tiles outside the union of a query tile's intervals.  Masks are evaluated in the tiles
// that some row of a warp sees in part only.  A hidden key has probability 0; what its value holds still meets that
// 0 in the PV product, so a row that comes out with a value that is not finite is computed again, key by key, by its
// warp (exact_row): rows are right whatever the hidden values are, and finite inputs pay one test per row.
//
// When the blocks do not fill the GPU, the key tiles of each are split over a cluster of 2, 4 or 8 CTAs;
// (O, maximum, sum) of the parts meet in distributed shared memory and are joined in rank order (no workspace, no second
// launch, the same bits at every run).
//
// The running maximum is lazy: O_t is rescaled only when a row's maximum grows by more than 2^8.  Probabilities are
// rounded to the value type for the PV product; sums, maxima and O are fp32.
#include <cudaTypedefs.h>

#include <atomic>

#include "attention_mma.cuh"
#include "attention_view.cuh"
#include "host_common.h"
#include "masked_host.h"

namespace vb200 {
namespace {

constexpr int kBM = 128, kQT = 2, kBN = 128;
constexpr int kStages = 4;
constexpr int kTileBytes = kBM * kHeadDim * 2;
constexpr int kSoftmaxWarps = 8;
constexpr int kWarpProducer = 8, kWarpMma = 9, kWarpKeys = 10;
constexpr int kThreads = 12 * 32;
// Register split: the block launches with 168 a thread (64512 of the SM's 65536); the softmax warpgroups rise to
// 200, the third drops to 104.  The host refuses to launch a build with another count.
constexpr int kLaunchRegs = 168, kRegsHigh = 200, kRegsLow = 104;
static_assert(kSoftmaxWarps * 32 * kRegsHigh + 128 * kRegsLow == kThreads * kLaunchRegs, "register split");
constexpr float kRescale = 8.f;  // P stays <= 2^8
constexpr int kPolyPairs = 1;    // of every 8 exponent pairs, those on the FMA pipe

constexpr int kOffQ = 0;
constexpr int kOffStage = kQT * kTileBytes;
constexpr int kOffKeys = kOffStage + kStages * 2 * kTileBytes;  // [stage][2][128] fp32: bias, position
constexpr int kOffBar = kOffKeys + kStages * 2 * kBN * 4;
constexpr int kBarQ = 0, kBarFull = 1, kBarEmpty = kBarFull + kStages, kBarS = kBarEmpty + kStages, kBarP = kBarS + kQT,
              kBarO = kBarP + kQT, kBarSFree = kBarO + kQT, kNumBars = kBarSFree + kQT;
constexpr int kOffMisc = kOffBar + kNumBars * 8;  // tmem slot, abort flag, per tile: first and last key
constexpr int kSmemBytes = kOffMisc + 32 + 1024;
constexpr int kPartStride = kHeadDim + 4;  // floats; parts of a split overlay Q and the ring
constexpr int kOffPartMl = kQT * kBM * kPartStride * 4;
static_assert(kOffPartMl + kQT * kBM * 8 <= kOffKeys, "the parts fit");
constexpr uint32_t kTmemCols = 512, kTmemP = 256, kTmemO = 384;

// S_t = Q_t K^T: four K=16 steps of head_dim 64; the first overwrites.
__device__ __forceinline__ void issue_qk(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred e, pf, pt;\n\t.reg .b64 a1, a2, a3, b1, b2, b3;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "setp.ne.b32 pf, 0, 0;\n\t"
      "setp.eq.b32 pt, 0, 0;\n\t"
      "add.s64 a1, %1, 2;\n\tadd.s64 b1, %2, 2;\n\t"
      "add.s64 a2, %1, 4;\n\tadd.s64 b2, %2, 4;\n\t"
      "add.s64 a3, %1, 6;\n\tadd.s64 b3, %2, 6;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, pf;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a1, b1, %3, pt;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a2, b2, %3, pt;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a3, b3, %3, pt;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%4];\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(bar)
      : "memory");
}

__device__ __forceinline__ float u2f(uint32_t u) { return __uint_as_float(u); }
__device__ __forceinline__ uint32_t f2u(float f) { return __float_as_uint(f); }

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
__device__ __forceinline__ uint32_t peer_address(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ float4 peer_load4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ float2 peer_load2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr));
  return v;
}

// One output row by one warp, key by key, two channels per lane: for rows whose tile result is not finite.
template <typename T, bool kPaged>
__device__ __noinline__ void exact_row(const AttnView& a, AttnSeq s, int i, int head) {
  const int lane = threadIdx.x & 31, hk = head / a.group;
  const int2 be = row_range<kPaged>(a, s, i);
  const float slope = a.slope == nullptr ? 0.f : __ldg(a.slope + head) * kLog2E;
  const float pos = row_position<kPaged>(a, s, i);
  const T* q = static_cast<const T*>(a.q) + s.batch * a.q_sb + head * a.q_sh + static_cast<long long>(s.row0 + i) * a.q_sn + 2 * lane;
  const float q0 = to_f32<T>(q[0]) * a.scale, q1 = to_f32<T>(q[1]) * a.scale;
  float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
  for (int j = be.x; j < be.y; ++j) {
    long long ko, vo, bo;
    if constexpr (kPaged) {
      const int id = page_of(a, s, j >> a.page_shift), at = j & ((1 << a.page_shift) - 1);
      if (id >= a.pages) continue;
      ko = id * a.k_sb + at * a.k_sn;
      vo = id * a.v_sb + at * a.v_sn;
      bo = (static_cast<long long>(id) << a.page_shift) + at;
    } else {
      ko = s.batch * a.k_sb + j * a.k_sn;
      vo = s.batch * a.v_sb + j * a.v_sn;
      bo = s.batch * a.bias_sb + j;
    }
    const float b = a.bias == nullptr ? 0.f : bias_log2(__ldg(a.bias + bo));
    if (b == -INFINITY) continue;  // mass 0
    const T* k = static_cast<const T*>(a.k) + ko + hk * a.k_sh + 2 * lane;
    const T* v = static_cast<const T*>(a.v) + vo + hk * a.v_sh + 2 * lane;
    float x = q0 * to_f32<T>(k[0]) + q1 * to_f32<T>(k[1]);
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
    if (a.cap != 0.f) x = a.cap * tanh_fast(x);
    x += b;
    if (a.slope != nullptr)
      x = fmaf(-slope, fabsf(pos - (!kPaged && a.kpos != nullptr ? __ldg(a.kpos + s.batch * a.kpos_sb + j) : static_cast<float>(j))), x);
    const float mn = fmaxf(m, x), mu = mn == -INFINITY ? 0.f : mn;
    const float corr = ex2_approx(m - mu), p = ex2_approx(x - mu);
    m = mn;
    l = l * corr + p;
    o0 = o0 * corr + p * to_f32<T>(v[0]);
    o1 = o1 * corr + p * to_f32<T>(v[1]);
  }
  T* out = static_cast<T*>(a.out) + s.batch * a.o_sb + head * a.o_sh + static_cast<long long>(s.row0 + i) * a.o_sn + 2 * lane;
  out[0] = from_f32<T>(l == 0.f ? 0.f : o0 / l);
  out[1] = from_f32<T>(l == 0.f ? 0.f : o1 / l);
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  return sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value ? pack_bf16x2(lo, hi) : pack_f16x2(lo, hi);
}

template <typename T, bool kPaged>
__global__ void __launch_bounds__(kThreads, 1)
    masked_attention_tc_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
                               const __grid_constant__ CUtensorMap tmap_v, const __grid_constant__ AttnView a, int blocks, int split) {
  constexpr bool kBF16 = std::is_same<T, __nv_bfloat16>::value;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // blocks in descending order, so that under causal masks the longest start first
  const int item = static_cast<int>(blockIdx.x) / split, piece = static_cast<int>(blockIdx.x) - item * split;
  const int vb = blocks - 1 - item / a.H, head = item % a.H, hk = head / a.group;
  AttnSeq s;
  int blk;
  if (!locate_block<kPaged>(a, vb, kQT * kBM, 1, s, blk)) return;  // the whole cluster shares the item
  const int row_first = blk * kQT * kBM;

  auto bar = [=](int i) -> uint32_t { return sbase + kOffBar + 8 * i; };
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + kOffMisc + 4);
  int* key_lo = reinterpret_cast<int*>(smem + kOffMisc + 8);
  int* key_hi = key_lo + kQT;
  const bool per_key = a.bias != nullptr || a.slope != nullptr;

  if (threadIdx.x == 0) {
    mbar_init(bar(kBarQ), 1);
    for (int i = 0; i < kStages; ++i) {
      mbar_init(bar(kBarFull + i), per_key ? 2 : 1);
      mbar_init(bar(kBarEmpty + i), 1);
    }
    for (int t = 0; t < kQT; ++t) {
      mbar_init(bar(kBarS + t), 1);
      mbar_init(bar(kBarP + t), kBM);
      mbar_init(bar(kBarO + t), 1);
      mbar_init(bar(kBarSFree + t), kBM);
      key_lo[t] = 0x7fffffff;
      key_hi[t] = 0;
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == kWarpMma) {
    tmem_alloc(sbase + kOffMisc, kTmemCols);
    tmem_relinquish();
  }
  if (warp == kWarpProducer && lane == 0) {
    prefetch_tmap(&tmap_q);
    prefetch_tmap(&tmap_k);
    prefetch_tmap(&tmap_v);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem + kOffMisc);
  int2 be = make_int2(0, 0);
  if (warp < kSoftmaxWarps) {
    const int i = row_first + static_cast<int>(threadIdx.x);
    if (i < s.rows) be = row_range<kPaged>(a, s, i);
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

  // Each role's code is dominated by its own setmaxnreg, with no merge point in between.
  if (warp >= kSoftmaxWarps) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsLow));
    if (warp == kWarpProducer) {
      // ------------------------------- producer -------------------------------
      const int npg = kPaged ? kBN >> a.page_shift : 1;
      const int which = lane / npg, pg = lane - which * npg;  // K (0) or V (1), page of the tile
      auto page_at = [&](int j) -> int {
        const int slot = ((j * kBN) >> a.page_shift) + pg;
        return static_cast<long long>(slot) << a.page_shift < s.keys ? page_of(a, s, slot) : a.pages;
      };
      int id = 0;
      if (kPaged && which < 2 && p0 < p1) id = page_at(p0);
      if (lane == 0 && p0 < p1) {
        mbar_arrive_expect_tx(bar(kBarQ), kQT * kTileBytes);
        for (int t = 0; t < kQT; ++t)
          tma_load_4d(sbase + kOffQ + t * kTileBytes, &tmap_q, bar(kBarQ), 0, s.row0 + row_first + t * kBM, head, s.batch);
      }
      for (int j = p0; j < p1; ++j) {
        const int n = j - p0, st = n % kStages;
        bool ok = *abort_flag == 0;
        if (n >= kStages) ok = mbar_wait(bar(kBarEmpty + st), (n / kStages - 1) & 1, a.err) && ok;
        if (!__all_sync(0xffffffffu, ok)) {
          if (lane == 0) *abort_flag = 1;
          break;
        }
        // a tile between the two query tiles' keys is not loaded
        const bool used = (j >= j0[0] && j < j1[0]) || (j >= j0[1] && j < j1[1]);
        if (!used) {
          if (lane == 0) mbar_arrive(bar(kBarFull + st));
          if (kPaged && which < 2 && j + 1 < p1) id = page_at(j + 1);
          continue;
        }
        if (lane == 0) mbar_arrive_expect_tx(bar(kBarFull + st), 2 * kTileBytes);
        __syncwarp();
        const uint32_t dst = sbase + kOffStage + st * 2 * kTileBytes;
        if constexpr (kPaged) {
          if (which < 2) {
            tma_load_4d(dst + which * kTileBytes + pg * (kTileBytes / npg), which ? &tmap_v : &tmap_k, bar(kBarFull + st), 0, hk, 0, id);
            if (j + 1 < p1) id = page_at(j + 1);
          }
        } else if (lane < 2) {
          tma_load_4d(dst + lane * kTileBytes, lane ? &tmap_v : &tmap_k, bar(kBarFull + st), 0, j * kBN, hk, s.batch);
        }
      }
    } else if (warp == kWarpMma) {
      // ------------------------------- MMA issuer -------------------------------
      constexpr uint32_t idesc_qk = idesc_f16(kBM, kBN, kBF16 ? 1 : 0, 0, 0);
      constexpr uint32_t idesc_pv = idesc_f16(kBM, kHeadDim, kBF16 ? 1 : 0, 0, 1);
      const uint64_t q_desc = smem_desc_sw128(sbase + kOffQ, 16, 1024);
      const uint64_t k_desc = smem_desc_sw128(sbase + kOffStage, 16, 1024);
      const uint64_t v_desc = smem_desc_sw128(sbase + kOffStage + kTileBytes, 16384, 1024);
      auto stage_off = [=](int j) -> uint64_t { return static_cast<uint64_t>(((j - p0) % kStages) * (2 * kTileBytes >> 4)); };
      auto wait_all = [&](int b, int parity) -> bool {
        return __all_sync(0xffffffffu, mbar_wait(bar(b), static_cast<uint32_t>(parity), a.err));
      };
      auto qk = [&](int t, int j) {
        issue_qk(tmem + t * 128, q_desc + t * (kTileBytes >> 4), k_desc + stage_off(j), idesc_qk, bar(kBarS + t));
      };
      bool ok = true;
      if (p0 < p1) {
        ok = wait_all(kBarQ, 0) && wait_all(kBarFull, 0);
        if (ok) {
          tc_fence_after();
#pragma unroll
          for (int t = 0; t < kQT; ++t)
            if (j0[t] == p0 && j1[t] > p0) qk(t, p0);
        }
      }
      for (int j = p0; j < p1 && ok; ++j) {
        if (__any_sync(0xffffffffu, *abort_flag != 0)) {
          ok = false;
          break;
        }
        const int st = (j - p0) % kStages;
        if (j + 1 < p1) ok = wait_all(kBarFull + (j + 1 - p0) % kStages, ((j + 1 - p0) / kStages) & 1);
        const bool last1 = j >= j0[1] && j < j1[1];
        bool any = false;
#pragma unroll
        for (int t = 0; t < kQT; ++t) {
          if (ok && j + 1 >= j0[t] && j + 1 < j1[t]) {
            if (j >= j0[t]) ok = wait_all(kBarSFree + t, (j - j0[t]) & 1);
            if (ok) {
              tc_fence_after();
              qk(t, j + 1);
            }
          }
          if (ok && j >= j0[t] && j < j1[t]) {
            ok = wait_all(kBarP + t, (j - j0[t]) & 1);
            if (ok) {
              tc_fence_after();
              issue_pv_group(tmem + kTmemO + t * kHeadDim, tmem + kTmemP + t * kHeadDim, v_desc + stage_off(j), idesc_pv,
                             j > j0[t] ? 1u : 0u, bar(kBarO + t), bar(kBarEmpty + st), (t == kQT - 1 || !last1) ? 1u : 0u);
              any = true;
            }
          }
        }
        if (ok && !any && lane == 0) mbar_arrive(bar(kBarEmpty + st));  // a tile between the two query tiles' keys
      }
      if (!ok && lane == 0) *abort_flag = 1;
    } else if (warp == kWarpKeys && per_key) {
      // ------------------------------- per-key bias and position -------------------------------
      for (int j = p0; j < p1; ++j) {
        const int n = j - p0, st = n % kStages;
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
            if (a.bias != nullptr && there) b[u] = bias_log2(__ldg(a.bias + at));
            if (a.slope != nullptr)
              kp[u] = !kPaged && a.kpos != nullptr ? __ldg(a.kpos + s.batch * a.kpos_sb + key) : static_cast<float>(key);
          }
        }
        bool ok = *abort_flag == 0;
        if (n >= kStages) ok = mbar_wait(bar(kBarEmpty + st), (n / kStages - 1) & 1, a.err) && ok;
        if (!__all_sync(0xffffffffu, ok)) {
          if (lane == 0) *abort_flag = 1;
          break;
        }
        float* dst = reinterpret_cast<float*>(smem + kOffKeys) + st * 2 * kBN;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          dst[u * 32 + lane] = b[u];
          dst[kBN + u * 32 + lane] = kp[u];
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(kBarFull + st));
      }
    }
    if (split > 1) {
      __syncwarp();
      cluster_arrive();
      cluster_wait();
      cluster_arrive();
      cluster_wait();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsHigh));
    // ------------------------------- softmax -------------------------------
    const int t = warp >> 2;
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t s_addr = tmem + lane_off + t * 128;
    const uint32_t p_addr = tmem + lane_off + kTmemP + t * kHeadDim;
    const uint32_t o_addr = tmem + lane_off + kTmemO + t * kHeadDim;
    const int i = row_first + t * kBM + row;  // token of the sequence
    const bool valid = i < s.rows;
    const bool cap = a.cap != 0.f, has_bias = a.bias != nullptr, dist = a.slope != nullptr;
    const bool formed = cap || has_bias || dist;  // the scores are brought to the log2 domain before the maximum
    const float mul = formed ? 1.f : a.scale;
    const float slope = dist ? __ldg(a.slope + head) * kLog2E : 0.f;
    const float pos = dist && valid ? row_position<kPaged>(a, s, i) : 0.f;
    float m_run = -INFINITY, l_run = 0.f;
    bool ok = true;
    const int ja = t == 0 ? j0[0] : j0[1], jb = t == 0 ? j1[0] : j1[1];

    for (int j = ja; j < jb; ++j) {
      const int n = j - ja;
      ok = ok && !*abort_flag;
      if (ok) ok = mbar_wait(bar(kBarS + t), n & 1, a.err);
      if (ok && per_key) ok = mbar_wait(bar(kBarFull + (j - p0) % kStages), ((j - p0) / kStages) & 1, a.err);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      uint32_t r[kBN];
      tc_fence_after();
#pragma unroll
      for (int c = 0; c < kBN; c += 32) tmem_ld32x32b_x32_nowait(s_addr + c, *reinterpret_cast<uint32_t(*)[32]>(&r[c]));
      tmem_wait_ld();
#pragma unroll
      for (int c = 0; c < kBN; c += 32) reg_fence32(*reinterpret_cast<uint32_t(*)[32]>(&r[c]));
      tc_fence_before();
      mbar_arrive(bar(kBarSFree + t));
      if (formed) {
        const float* keys = reinterpret_cast<const float*>(smem + kOffKeys) + ((j - p0) % kStages) * 2 * kBN;
        if (cap) {
#pragma unroll
          for (int c = 0; c < kBN; ++c) r[c] = f2u(a.cap * tanh_fast(u2f(r[c]) * a.scale));
          if (has_bias) {
#pragma unroll
            for (int c = 0; c < kBN; c += 4) {
              const float4 b = *reinterpret_cast<const float4*>(keys + c);
              r[c] = f2u(u2f(r[c]) + b.x);
              r[c + 1] = f2u(u2f(r[c + 1]) + b.y);
              r[c + 2] = f2u(u2f(r[c + 2]) + b.z);
              r[c + 3] = f2u(u2f(r[c + 3]) + b.w);
            }
          }
        } else {
          // without a bias the ring holds zeros
          const uint64_t sc = pk2(a.scale, a.scale);
#pragma unroll
          for (int c = 0; c < kBN; c += 4) {
            const float4 b = *reinterpret_cast<const float4*>(keys + c);
            float x0, x1;
            upk2(ffma2(pk2(u2f(r[c]), u2f(r[c + 1])), sc, pk2(b.x, b.y)), x0, x1);
            r[c] = f2u(x0);
            r[c + 1] = f2u(x1);
            upk2(ffma2(pk2(u2f(r[c + 2]), u2f(r[c + 3])), sc, pk2(b.z, b.w)), x0, x1);
            r[c + 2] = f2u(x0);
            r[c + 3] = f2u(x1);
          }
        }
        if (dist) {
#pragma unroll
          for (int c = 0; c < kBN; c += 4) {
            const float4 p = *reinterpret_cast<const float4*>(keys + kBN + c);
            r[c] = f2u(fmaf(-slope, fabsf(pos - p.x), u2f(r[c])));
            r[c + 1] = f2u(fmaf(-slope, fabsf(pos - p.y), u2f(r[c + 1])));
            r[c + 2] = f2u(fmaf(-slope, fabsf(pos - p.z), u2f(r[c + 2])));
            r[c + 3] = f2u(fmaf(-slope, fabsf(pos - p.w), u2f(r[c + 3])));
          }
        }
      }
      {
        const int lo = min(max(be.x - j * kBN, 0), kBN), hi = min(max(be.y - j * kBN, 0), kBN);
        if (__any_sync(0xffffffffu, lo > 0 || hi < kBN)) {
#pragma unroll
          for (int w = 0; w < kBN / 32; ++w) {
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
      }
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int c = 0; c < kBN; c += 8) {
#pragma unroll
        for (int u = 0; u < 4; ++u) mx[u] = fmax3(mx[u], u2f(r[c + 2 * u]), u2f(r[c + 2 * u + 1]));
      }
      const float m_new = fmaxf(m_run, fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * mul);
      const bool grow = m_new > m_run + kRescale;
      const bool need = __any_sync(0xffffffffu, grow);
      const float m_tgt = grow ? m_new : m_run;
      const float alpha = grow ? ex2_approx(m_run - m_tgt) : 1.f;
      const float m_use = m_tgt == -INFINITY ? 0.f : m_tgt;
      const uint64_t neg_m2 = pk2(-m_use, -m_use), mul2 = pk2(mul, mul);
      uint64_t ls0 = pk2(0.f, 0.f), ls1 = pk2(0.f, 0.f);
#pragma unroll
      for (int c = 0; c < kBN / 2; ++c) {
        float e0, e1, q0, q1;
        upk2(ffma2(pk2(u2f(r[2 * c]), u2f(r[2 * c + 1])), mul2, neg_m2), e0, e1);
        if ((c & 7) < kPolyPairs) {
          exp2_poly2(e0, e1, q0, q1);
          // a hidden key's probability is exactly 0 (the polynomial's 2^-125 times a hidden 3e38 would show), and
          // a score that is NaN stays NaN
          upk2(ffma2(pk2(e0, e1), pk2(0.f, 0.f), pk2(q0, q1)), q0, q1);
          q0 = e0 < -125.f ? 0.f : q0;
          q1 = e1 < -125.f ? 0.f : q1;
        } else {
          q0 = ex2_approx(e0);
          q1 = ex2_approx(e1);
        }
        if (c & 1) ls1 = fadd2(ls1, pk2(q0, q1));
        else ls0 = fadd2(ls0, pk2(q0, q1));
        r[c] = pack2<T>(q0, q1);
      }
      float a0, a1, b0, b1;
      upk2(ls0, a0, a1);
      upk2(ls1, b0, b1);
      l_run = l_run * alpha + ((a0 + a1) + (b0 + b1));
      m_run = m_tgt;
      if (n > 0) {
        // PV_t(j-1) is complete before P_t is overwritten or O_t rescaled
        ok = __all_sync(0xffffffffu, mbar_wait(bar(kBarO + t), (n - 1) & 1, a.err));
        if (!ok) break;
        tc_fence_after();
        if (need) {
#pragma unroll 1
          for (int c = 0; c < kHeadDim; c += 16) {
            uint32_t o[16];
            tmem_ld32x32b_x16(o_addr + c, o);
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = f2u(u2f(o[e]) * alpha);
            tmem_st32x32b_x16(o_addr + c, o);
          }
        }
      }
      tmem_st32x32b_x32(p_addr, *reinterpret_cast<const uint32_t(*)[32]>(&r[0]));
      tmem_st32x32b_x32(p_addr + 32, *reinterpret_cast<const uint32_t(*)[32]>(&r[32]));
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(bar(kBarP + t));
    }
    if (ok && jb > ja) ok = __all_sync(0xffffffffu, mbar_wait(bar(kBarO + t), (jb - ja - 1) & 1, a.err));
    uint32_t o[kHeadDim];
#pragma unroll
    for (int c = 0; c < kHeadDim; ++c) o[c] = 0u;
    if (ok && jb > ja) {
      tc_fence_after();
      tmem_ld32x32b_x32_nowait(o_addr, *reinterpret_cast<uint32_t(*)[32]>(&o[0]));
      tmem_ld32x32b_x32_nowait(o_addr + 32, *reinterpret_cast<uint32_t(*)[32]>(&o[32]));
      tmem_wait_ld();
      reg_fence32(*reinterpret_cast<uint32_t(*)[32]>(&o[0]));
      reg_fence32(*reinterpret_cast<uint32_t(*)[32]>(&o[32]));
    }
    if (!ok) *abort_flag = 1;
    uint8_t* out_head = static_cast<uint8_t*>(a.out) + 2 * (s.batch * a.o_sb + head * a.o_sh);
    if (split == 1) {
      bool again = false;
      if (ok && valid) {
        const float inv = l_run == 0.f ? 0.f : 1.f / l_run;
        uint4* orow = reinterpret_cast<uint4*>(out_head + 2 * (s.row0 + i) * a.o_sn);
        float z = 0.f;
#pragma unroll
        for (int c = 0; c < kHeadDim / 8; ++c) {
          uint32_t w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x = u2f(o[8 * c + 2 * e]), y = u2f(o[8 * c + 2 * e + 1]);
            z = fmaf(x, 0.f, fmaf(y, 0.f, z));  // NaN unless every value is finite
            w[e] = pack2<T>(x * inv, y * inv);
          }
          orow[c] = l_run == 0.f ? make_uint4(0u, 0u, 0u, 0u) : make_uint4(w[0], w[1], w[2], w[3]);
        }
        again = l_run != 0.f && !(z * inv == 0.f);
      }
      __syncwarp();  // a row's first result is written before its second
      unsigned rows = __ballot_sync(0xffffffffu, again);
      while (rows) {
        const int b = __ffs(rows) - 1;
        rows &= rows - 1;
        exact_row<T, kPaged>(a, s, row_first + t * kBM + (warp & 3) * 32 + b, head);
      }
    } else {
      // The parts overlay Q and the ring: every load into them has been consumed, and every tensor-core read of
      // them is complete, once both query tiles are.
      named_bar_sync(1, kSoftmaxWarps * 32);
      float* mine = reinterpret_cast<float*>(smem) + (t * kBM + row) * kPartStride;
#pragma unroll
      for (int c = 0; c < kHeadDim; c += 4)
        *reinterpret_cast<float4*>(mine + c) = make_float4(u2f(o[c]), u2f(o[c + 1]), u2f(o[c + 2]), u2f(o[c + 3]));
      *reinterpret_cast<float2*>(smem + kOffPartMl + 8 * (t * kBM + row)) = make_float2(m_run, l_run);
      cluster_arrive();
      cluster_wait();
      const int per = kQT * kBM / split;  // rows joined by this CTA, 16 lanes per row
      for (int x = threadIdx.x; x < per * 16; x += kSoftmaxWarps * 32) {
        const int rr = piece * per + (x >> 4), c4 = (x & 15) * 4;
        const uint32_t ml = sbase + kOffPartMl + 8 * rr, ov = sbase + 4 * (rr * kPartStride + c4);
        float mx = -INFINITY;
        for (int w = 0; w < split; ++w) mx = fmaxf(mx, peer_load2(peer_address(ml, w)).x);
        const float mu = mx == -INFINITY ? 0.f : mx;
        float sum = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int w = 0; w < split; ++w) {
          const float2 v = peer_load2(peer_address(ml, w));
          const float4 y = peer_load4(peer_address(ov, w));
          const float f = ex2_approx(v.x - mu);
          if (v.y == 0.f) continue;  // a part without keys of this row: its O may hold 0 * NaN
          sum = fmaf(v.y, f, sum);
          acc.x = fmaf(y.x, f, acc.x);
          acc.y = fmaf(y.y, f, acc.y);
          acc.z = fmaf(y.z, f, acc.z);
          acc.w = fmaf(y.w, f, acc.w);
        }
        const int tok = row_first + rr;
        bool again = false;
        if (tok < s.rows) {
          const float inv = sum == 0.f ? 0.f : 1.f / sum;
          *reinterpret_cast<uint2*>(out_head + 2 * ((s.row0 + tok) * a.o_sn + c4)) =
              sum == 0.f ? make_uint2(0u, 0u) : make_uint2(pack2<T>(acc.x * inv, acc.y * inv), pack2<T>(acc.z * inv, acc.w * inv));
          const float z = fmaf(acc.x, 0.f, fmaf(acc.y, 0.f, fmaf(acc.z, 0.f, acc.w * 0.f)));
          again = sum != 0.f && !(z * inv == 0.f);
        }
        // per * 16 is a multiple of 256, so whole warps run this together
        __syncwarp();  // a row's first result is written before its second
        const unsigned bad = __ballot_sync(0xffffffffu, again);
        const int first_row = row_first + piece * per + ((x - lane) >> 4);
        if (bad & 0xffffu) exact_row<T, kPaged>(a, s, first_row, head);
        if (bad >> 16) exact_row<T, kPaged>(a, s, first_row + 1, head);
      }
      cluster_arrive();  // the peers read this CTA's part before it leaves
      cluster_wait();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kWarpMma) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

int rows_map(CUtensorMap* map, const void* base, int dtype, long long n, long long heads, long long batch, long long sn, long long sh,
             long long sb, int box) {
  // (channel, row, head, batch); dimensions of size one get a harmless stride
  if (n == 1) sn = kHeadDim;
  if (heads == 1) sh = sn * n;
  if (batch == 1) sb = sh * heads;
  const uint64_t dims[4] = {kHeadDim, static_cast<uint64_t>(n), static_cast<uint64_t>(heads), static_cast<uint64_t>(batch)};
  const uint64_t str[3] = {static_cast<uint64_t>(sn) * 2, static_cast<uint64_t>(sh) * 2, static_cast<uint64_t>(sb) * 2};
  const uint32_t b[4] = {kHeadDim, static_cast<uint32_t>(box), 1, 1};
  return encode_tiled_map(map, dtype == VB200_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, base, dims,
                          str, b, CU_TENSOR_MAP_SWIZZLE_128B);
}

int pool_map(CUtensorMap* map, const void* base, int dtype, const AttnView& a) {
  // (channel, head, slot, page): contiguous pools
  const int page = 1 << a.page_shift;
  const uint64_t dims[4] = {kHeadDim, static_cast<uint64_t>(a.Hkv), static_cast<uint64_t>(page), static_cast<uint64_t>(a.pages)};
  const uint64_t row = static_cast<uint64_t>(a.Hkv) * kHeadDim * 2;
  const uint64_t str[3] = {kHeadDim * 2, row, row * page};
  const uint32_t b[4] = {kHeadDim, 1, static_cast<uint32_t>(page), 1};
  return encode_tiled_map(map, dtype == VB200_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, base, dims,
                          str, b, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <typename T, bool kPaged>
int launch(const AttnView& a, const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, long long blocks, int split,
           cudaStream_t st) {
  auto kernel = masked_attention_tc_kernel<T, kPaged>;
  // per device: the opt-in to the shared memory, and the register count that the split inside the kernel needs
  static std::atomic<bool> ready[64];
  int dev = 0;
  VB200_CHECK_CUDA(cudaGetDevice(&dev), "cudaGetDevice");
  if (dev < 0 || dev >= 64 || !ready[dev].load(std::memory_order_acquire)) {
    cudaFuncAttributes fa{};
    VB200_CHECK_CUDA(cudaFuncGetAttributes(&fa, kernel), "cudaFuncGetAttributes");
    if (fa.numRegs != kLaunchRegs)
      return set_error(VB200_EUNSUPPORTED, "masked_attention_tc_kernel was built with %d registers per thread; its register split needs %d",
                       fa.numRegs, kLaunchRegs);
    VB200_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes), "cudaFuncSetAttribute");
    if (dev >= 0 && dev < 64) ready[dev].store(true, std::memory_order_release);
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks * a.H * split));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmemBytes;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = static_cast<unsigned>(split);
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = split > 1 ? 1 : 0;
  VB200_CHECK_CUDA(cudaLaunchKernelEx(&cfg, kernel, tq, tk, tv, a, static_cast<int>(blocks), split), "masked_attention_tc_kernel");
  VB200_CHECK_LAUNCH("masked_attention_tc_kernel");
  return VB200_OK;
}

}  // namespace

int tile_attention(int dtype, bool paged, const AttnView& a, long long most_keys, cudaStream_t st) {
  const long long blocks = paged ? static_cast<long long>(a.Nq) / (kQT * kBM) + a.n_seq
                                 : (static_cast<long long>(a.Nq) + kQT * kBM - 1) / (kQT * kBM) * a.B;
  // One CTA per SM: `blocks * H` items take ceil(items / SMs) rounds.  Splitting the keys s ways makes the rounds 1/s
  // as long plus a ramp of about three key tiles each; the cheapest s is taken.
  const int sms = sm_count_of_device();
  const long long items = blocks * a.H;
  const double tiles = static_cast<double>((most_keys + kBN - 1) / kBN);
  int split = 1;
  if (sms > 0) {
    double best = 0.0;
    for (int k = 1; k <= 8; k *= 2) {
      if (k > 1 && k > tiles) break;
      const double cost = static_cast<double>((items * k + sms - 1) / sms) * (1.0 / k + 3.0 / tiles);
      if (k == 1 || cost < best - 1e-9) {
        best = cost;
        split = k;
      }
    }
  }
  VB200_REQUIRE(items * split < (1ll << 31), "attention: too many work items");
  CUtensorMap tq, tk, tv;
  int rc = rows_map(&tq, a.q, dtype, a.Nq, a.H, paged ? 1 : a.B, a.q_sn, a.q_sh, a.q_sb, kBM);
  if (rc != VB200_OK) return rc;
  if (paged) {
    if ((rc = pool_map(&tk, a.k, dtype, a)) != VB200_OK || (rc = pool_map(&tv, a.v, dtype, a)) != VB200_OK) return rc;
    return dtype == VB200_BF16 ? launch<__nv_bfloat16, true>(a, tq, tk, tv, blocks, split, st)
                               : launch<__half, true>(a, tq, tk, tv, blocks, split, st);
  }
  if ((rc = rows_map(&tk, a.k, dtype, a.Nk, a.Hkv, a.B, a.k_sn, a.k_sh, a.k_sb, kBN)) != VB200_OK ||
      (rc = rows_map(&tv, a.v, dtype, a.Nk, a.Hkv, a.B, a.v_sn, a.v_sh, a.v_sb, kBN)) != VB200_OK)
    return rc;
  return dtype == VB200_BF16 ? launch<__nv_bfloat16, false>(a, tq, tk, tv, blocks, split, st)
                             : launch<__half, false>(a, tq, tk, tv, blocks, split, st);
}

}  // namespace vb200
