// Masked and paged attention for few query rows per key head (a token per stream, a handful of special tokens) and for
// fp32 inputs.  The mathematics is in attention_view.cuh.
//
// Both kernels give a CTA some (query row, head of the group) pairs of one sequence and one key head, so a key is read
// once for all heads that share it; its 8 warps take the keys in turn, each with its own running maximum, sum and
// accumulators, joined once at the end in a fixed order.  The keys are split over a cluster of up to 8 CTAs when the
// pairs alone do not fill the GPU; the parts meet in distributed shared memory, so there is no workspace and no second
// launch.
//
//   few_rows_kernel (bf16, fp16): 8 or 16 pairs, on the warp-level matrix instructions (m16n8k16) with the keys, and then
//     the channels, as their 16 rows and the pairs as their 8 columns.  Bound by reading K and V
//     (256 bytes a key): each warp has a ring of its own of 3 steps of 16 keys, filled by TMA two steps ahead (two tiles
//     of 2 KB a step, issued by one lane).  The channels of the QK product and of the output are permuted so that a lane's
//     operands are whole 16-byte vectors of the swizzled tiles, read without bank conflicts.  (The same ring filled by
//     16-byte asynchronous copies spent a third of its time issuing them and reached 4.6 TB/s, loads into registers spilled
//     and reached 3.7, the FMA pipe 2.2 with one row per key head and 0.7 with eight.)  A tcgen05 tile has 128 rows of
//     which these would use 1 to 16.
//   rows_attention_kernel (fp32): up to 4 pairs, on the FMA pipe: eight lanes hold one key, 8 channels each.
#include <cooperative_groups.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "attention_view.cuh"
#include "host_common.h"
#include "masked_host.h"

namespace cg = cooperative_groups;

namespace vb200 {
namespace {

constexpr int kRowWarps = 8;

// 8 channels of a row as four packed fp32 pairs
struct Key8 {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = __ldg(reinterpret_cast<const float4*>(p));
    b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  }
  __device__ __forceinline__ void zero() { a = b = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ void unpack(uint64_t (&x)[4]) const {
    x[0] = pk2(a.x, a.y);
    x[1] = pk2(a.z, a.w);
    x[2] = pk2(b.x, b.y);
    x[3] = pk2(b.z, b.w);
  }
};

// Joins `parts` results (O, running maximum, running sum) of one output value: part(k) gives their addresses.
template <typename F>
__device__ __forceinline__ void join(int parts, F part, int ch, float& mx, float& sum, float& o) {
  mx = -INFINITY;
  sum = o = 0.f;
  for (int k = 0; k < parts; ++k) mx = fmaxf(mx, part(k)[kHeadDim]);
  const float mu = mx == -INFINITY ? 0.f : mx;
  for (int k = 0; k < parts; ++k) {
    const float* p = part(k);
    if (p[kHeadDim + 1] == 0.f) continue;  // no visible key: its O may hold 0 * NaN
    const float f = ex2_approx(p[kHeadDim] - mu);
    sum = fmaf(p[kHeadDim + 1], f, sum);
    o = fmaf(p[ch], f, o);
  }
}

// resident CTAs: as many as the registers of R rows (their queries and sums) allow
template <int R, bool kPaged>
__global__ void __launch_bounds__(kRowWarps * 32, R <= 2 ? 3 : 2) rows_attention_kernel(const AttnView a, int split) {
  using T = float;
  constexpr int U = 2;  // loads in flight per lane: 4 x (K, V) vectors of 16 bytes
  constexpr int kStep = 4 * U;               // keys per warp and step; divides every page size
  __shared__ float part[kRowWarps][R][kHeadDim + 2];  // output row, running maximum, running sum
  __shared__ float fin[R][kHeadDim + 2];
  __shared__ int2 rng[R];
  __shared__ float pos[R], slp[R];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int sub = lane & 7, grp = lane >> 3;
  const int item = blockIdx.x / split, piece = blockIdx.x - item * split;
  const int vb = item / a.Hkv, hk = item - vb * a.Hkv;
  AttnSeq s;
  int blk;
  if (!locate_block<kPaged>(a, vb, R, a.group, s, blk)) return;  // the whole cluster shares the item
  const long long pair0 = static_cast<long long>(blk) * R;
  const int pairs = static_cast<int>(min(static_cast<long long>(R), static_cast<long long>(s.rows) * a.group - pair0));

  const int origin = position_origin<kPaged>(a, s, static_cast<int>(pair0 / a.group));
  if (threadIdx.x < R) {
    const int r = threadIdx.x;
    int2 be = make_int2(0, 0);
    float p = 0.f, sl = 0.f;
    if (r < pairs) {
      const int i = static_cast<int>((pair0 + r) / a.group), g = static_cast<int>((pair0 + r) % a.group);
      be = row_range<kPaged>(a, s, i);
      if (a.slope != nullptr) {
        p = row_position<kPaged>(a, s, origin, i);
        sl = __ldg(a.slope + hk * a.group + g) * kLog2E;
      }
    }
    rng[r] = be;
    pos[r] = p;
    slp[r] = sl;
  }
  uint64_t q2[R][4];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    Key8 x;
    x.zero();
    if (r < pairs) {
      const int i = static_cast<int>((pair0 + r) / a.group), g = static_cast<int>((pair0 + r) % a.group);
      x.load(static_cast<const T*>(a.q) + s.batch * a.q_sb + (hk * a.group + g) * a.q_sh +
             static_cast<long long>(s.row0 + i) * a.q_sn + sub * 8);
    }
    x.unpack(q2[r]);
#pragma unroll
    for (int i = 0; i < 4; ++i) q2[r][i] = fmul2(q2[r][i], pk2(a.scale, a.scale));
  }
  __syncthreads();
  // keys that some row sees [lo, hi), and those that every row sees [lo_all, hi_all)
  int lo = 0x7fffffff, hi = 0, lo_all = 0, hi_all = 0x7fffffff;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int2 be = rng[r];
    if (be.y > be.x) {
      lo = min(lo, be.x);
      hi = max(hi, be.y);
    }
    if (r < pairs) {
      lo_all = max(lo_all, be.x);
      hi_all = min(hi_all, be.y);
    }
  }
  if (hi == 0) lo = 0;
  lo &= ~15;
  const int steps = (hi - lo + kStep - 1) / kStep;
  const int c0 = static_cast<int>(static_cast<long long>(steps) * piece / split);
  const int c1 = static_cast<int>(static_cast<long long>(steps) * (piece + 1) / split);

  float m[R], l[R];
  uint64_t acc[R][4];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[r][i] = pk2(0.f, 0.f);
  }
  const T* kb = static_cast<const T*>(a.k) + s.batch * a.k_sb * (kPaged ? 0 : 1) + hk * a.k_sh + sub * 8;
  const T* vb_ = static_cast<const T*>(a.v) + s.batch * a.v_sb * (kPaged ? 0 : 1) + hk * a.v_sh + sub * 8;
  const float* bias = a.bias == nullptr ? nullptr : a.bias + (kPaged ? 0 : s.batch * a.bias_sb);
  const bool cap = a.cap != 0.f, dist = a.slope != nullptr;
  const int slot_mask = (1 << a.page_shift) - 1;

  for (int c = c0 + warp; c < c1; c += kRowWarps) {
    const int key0 = lo + c * kStep;
    const bool full = key0 >= lo_all && key0 + kStep <= hi_all;  // also: every key exists
    int at0 = key0;  // dense: key index; paged: slot inside the page
    long long koff = 0, voff = 0, boff = 0;
    bool there = true;
    if constexpr (kPaged) {
      const int id = page_of(a, s, key0 >> a.page_shift);
      there = id < a.pages;
      at0 = key0 & slot_mask;
      koff = id * a.k_sb;
      voff = id * a.v_sb;
      boff = static_cast<long long>(id) << a.page_shift;
    }
    Key8 kr[U], vr[U];
    float bs[U], kp[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int off = u * 4 + grp;
      if (there && (full || key0 + off < s.keys)) {
        kr[u].load(kb + koff + static_cast<long long>(at0 + off) * a.k_sn);
        vr[u].load(vb_ + voff + static_cast<long long>(at0 + off) * a.v_sn);
        bs[u] = bias == nullptr ? 0.f : bias_log2(__ldg(bias + boff + at0 + off));
        kp[u] = !dist ? 0.f : key_position<kPaged>(a, s, origin, key0 + off);
      } else {
        kr[u].zero();
        vr[u].zero();
        bs[u] = kp[u] = 0.f;
      }
    }
    float x[U][R];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      uint64_t k2[4];
      kr[u].unpack(k2);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        uint64_t d = fmul2(q2[r][0], k2[0]);
#pragma unroll
        for (int i = 1; i < 4; ++i) d = ffma2(q2[r][i], k2[i], d);
        float d0, d1;
        upk2(d, d0, d1);
        x[u][r] = d0 + d1;
      }
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1)
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int r = 0; r < R; ++r) x[u][r] += __shfl_xor_sync(0xffffffffu, x[u][r], o);
    if (cap) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int r = 0; r < R; ++r) x[u][r] = a.cap * tanhf(x[u][r]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int r = 0; r < R; ++r) x[u][r] += bs[u];
    if (dist) {
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int u = 0; u < U; ++u) x[u][r] = fmaf(-slp[r], fabsf(pos[r] - kp[u]), x[u][r]);
    }
    unsigned hide = 0;  // bit u * R + r: the row does not see the key (U * R <= 32)
    bool plain = full;  // a key of bias -inf (mass 0) is hidden too
#pragma unroll
    for (int u = 0; u < U; ++u) plain = plain && bs[u] != -INFINITY;
    if (!plain) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int2 be = rng[r];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int key = key0 + u * 4 + grp;
          if (!there || key < be.x || key >= be.y || bs[u] == -INFINITY) {
            hide |= 1u << (u * R + r);
            x[u][r] = -INFINITY;
          }
        }
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float mn = m[r];
#pragma unroll
      for (int u = 0; u < U; ++u) mn = fmaxf(mn, x[u][r]);
      const float mu = mn == -INFINITY ? 0.f : mn;
      const float corr = ex2_approx(m[r] - mu);
      m[r] = mn;
      float sum = 0.f;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        x[u][r] = ex2_approx(x[u][r] - mu);
        sum += x[u][r];
      }
      l[r] = fmaf(l[r], corr, sum);
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[r][i] = fmul2(acc[r][i], pk2(corr, corr));
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      uint64_t v2[4];
      vr[u].unpack(v2);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (plain || !((hide >> (u * R + r)) & 1u)) {  // a hidden value is not multiplied by 0: it may be NaN
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[r][i] = ffma2(pk2(x[u][r], x[u][r]), v2[i], acc[r][i]);
        }
      }
    }
  }

  // join the four lane groups of the warp, then the warps
#pragma unroll
  for (int r = 0; r < R; ++r) {
    float o[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) upk2(acc[r][i], o[2 * i], o[2 * i + 1]);
#pragma unroll
    for (int d = 8; d < 32; d <<= 1) {
      const float mo = __shfl_xor_sync(0xffffffffu, m[r], d), lo2 = __shfl_xor_sync(0xffffffffu, l[r], d);
      const float mn = fmaxf(m[r], mo), mu = mn == -INFINITY ? 0.f : mn;
      const float ca = ex2_approx(m[r] - mu), cb = ex2_approx(mo - mu);
      m[r] = mn;
      l[r] = l[r] * ca + lo2 * cb;
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = o[i] * ca + __shfl_xor_sync(0xffffffffu, o[i], d) * cb;
    }
    if (grp == 0) {
#pragma unroll
      for (int i = 0; i < 8; ++i) part[warp][r][sub * 8 + i] = o[i];
      if (sub == 0) {
        part[warp][r][kHeadDim] = m[r];
        part[warp][r][kHeadDim + 1] = l[r];
      }
    }
  }
  __syncthreads();
  auto store = [&](int idx, float o, float sum) {
    const int r = idx / kHeadDim, ch = idx - r * kHeadDim;
    if (r >= pairs) return;
    const int i = static_cast<int>((pair0 + r) / a.group), g = static_cast<int>((pair0 + r) % a.group);
    const float y = sum == 0.f ? 0.f : o / sum;  // no visible key: 0
    static_cast<T*>(a.out)[s.batch * a.o_sb + (hk * a.group + g) * a.o_sh + static_cast<long long>(s.row0 + i) * a.o_sn + ch] =
        from_f32<T>(y);
  };
  for (int idx = threadIdx.x; idx < R * kHeadDim; idx += kRowWarps * 32) {
    const int r = idx / kHeadDim, ch = idx - r * kHeadDim;
    float mx, sum, o;
    join(kRowWarps, [&](int w) -> const float* { return part[w][r]; }, ch, mx, sum, o);
    if (split == 1) {
      store(idx, o, sum);
    } else {
      fin[r][ch] = o;
      if (ch == 0) {
        fin[r][kHeadDim] = mx;
        fin[r][kHeadDim + 1] = sum;
      }
    }
  }
  if (split > 1) {
    cg::cluster_group cl = cg::this_cluster();
    cl.sync();
    const int per = (R * kHeadDim + split - 1) / split;
    for (int idx = piece * per + threadIdx.x; idx < min((piece + 1) * per, R * kHeadDim); idx += kRowWarps * 32) {
      const int r = idx / kHeadDim, ch = idx - r * kHeadDim;
      float mx, sum, o;
      join(split, [&](int w) -> const float* { return cl.map_shared_rank(&fin[0][0], w) + r * (kHeadDim + 2); }, ch, mx, sum, o);
      store(idx, o, sum);
    }
    cl.sync();  // the peers read this CTA's part before it leaves
  }
}

// ---------------------------------------------------------------- bf16, fp16

__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __nv_bfloat16*) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half*) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

constexpr int kRing = 3;  // steps of 16 keys in a warp's ring
constexpr float kRoom = 8.f;  // a row's maximum grows by up to 2^8 before O is rescaled
// A new maximum has P = 2^kUp.  fp16 loses what falls below its smallest step 2^-24, so its P go up to 2^(7 + 8), near the top of
// the type; bf16 has fp32's exponents.
template <typename T>
constexpr float kUp = std::is_same<T, __half>::value ? 7.f : 0.f;
constexpr int kSide = 16 * kHeadDim * 2;  // K or V of a step: 16 rows of 128 bytes, 128-byte swizzle
constexpr int kRowsRing = kRowWarps * kRing * 2 * kSide;
constexpr int kRowsSmem = kRowsRing + 1024;  // slack for the alignment of the swizzle

// The 8 x 8 matrix of 16-bit values that a warp holds (lane: row g, columns 2 t, 2 t + 1), transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// kN: columns of pairs, 8 kN pairs.
//
// Operand layouts, with g = lane / 4 and t = lane % 4: A holds rows g and g + 8 at k = 2t, 2t+1, 2t+8, 2t+9; B holds those k of
// column g; the result has columns 2t, 2t+1 of rows g and g + 8.
//   S^T = K Q^T, step s of 4: k = 2t, 2t+1, 2t+8, 2t+9 stand for channels 16 t + 4 s .. + 3, so A is words of the lane's own K
//     vectors (chunks 2 t and 2 t + 1 of rows g and 8 + g); a row is a key, a column a pair.
//   O^T += V^T P^T: k is the key, and S^T transposed 8 x 8 is P^T as B; row g (g + 8) of tile j of 4 stands for channel
//     8 g + 2 j (+ 1), so A is one word's channels of the lane's own V vectors (chunk g of rows 2t, 2t+1, 2t+8, 2t+9).
// (With the pairs as rows, 16 of which 1 to 8 were used, the matrix instructions, twice as many, bounded the kernel: 4.4 TB/s.)
template <typename T, bool kPaged, int kN>
__global__ void __launch_bounds__(kRowWarps * 32, 2) few_rows_kernel(const __grid_constant__ AttnView a, int split, const __grid_constant__ CUtensorMap tmap_k,
                                                                       const __grid_constant__ CUtensorMap tmap_v) {
  constexpr int kRows = 8 * kN;
  extern __shared__ uint8_t ring_raw[];
  // [warp][kRing][K, V] steps; afterwards the warps' parts
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(ring_raw) + 1023) & ~uintptr_t(1023));
  using Part = float[kRows][kHeadDim + 2];  // O row, running maximum, running sum
  static_assert(sizeof(Part) * kRowWarps <= kRowsRing, "the parts fit");
  __shared__ __align__(8) uint64_t full_bar[kRowWarps][kRing];
  Part* part = reinterpret_cast<Part*>(ring);
  __shared__ Part fin;
  __shared__ int bad[kRows];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int item = blockIdx.x / split, piece = blockIdx.x - item * split;
  const int vb = item / a.Hkv, hk = item - vb * a.Hkv;
  AttnSeq s;
  int blk;
  if (!locate_block<kPaged>(a, vb, kRows, a.group, s, blk)) return;  // the whole cluster shares the item
  const long long pair0 = static_cast<long long>(blk) * kRows;
  const int pairs = static_cast<int>(min(static_cast<long long>(kRows), static_cast<long long>(s.rows) * a.group - pair0));
  auto token_of = [&](int r) { return static_cast<int>((pair0 + r) / a.group); };
  auto head_of = [&](int r) { return hk * a.group + static_cast<int>((pair0 + r) % a.group); };
  const int origin = position_origin<kPaged>(a, s, token_of(0));
  if (threadIdx.x < kRows) bad[threadIdx.x] = 0;
  const uint32_t bars = smem_u32(&full_bar[warp][0]);
  if (lane == 0) {
    for (int k = 0; k < kRing; ++k) mbar_init(bars + 8 * k, 1);
    fence_barrier_init();
    prefetch_tmap(&tmap_k);
    prefetch_tmap(&tmap_v);
  }
  __syncwarp();

  // queries in operand order: row 8 n + g
  uint32_t q[kN][4][2];
#pragma unroll
  for (int n = 0; n < kN; ++n) {
    const int r = 8 * n + g;
    uint4 x = make_uint4(0u, 0u, 0u, 0u), y = x;
    if (r < pairs) {
      const T* p = static_cast<const T*>(a.q) + s.batch * a.q_sb + head_of(r) * a.q_sh +
                   static_cast<long long>(s.row0 + token_of(r)) * a.q_sn + 16 * t;
      x = __ldg(reinterpret_cast<const uint4*>(p));
      y = __ldg(reinterpret_cast<const uint4*>(p + 8));
    }
    q[n][0][0] = x.x, q[n][0][1] = x.y, q[n][1][0] = x.z, q[n][1][1] = x.w;
    q[n][2][0] = y.x, q[n][2][1] = y.y, q[n][3][0] = y.z, q[n][3][1] = y.w;
  }
  // the lane's columns of the products, rows 8 n + 2 t and + 1: intervals, positions
  int2 be[kN][2];
  float pos[kN][2], slp[kN][2];
  int lo = 0x7fffffff, hi = 0, lo_all = 0, hi_all = 0x7fffffff;
#pragma unroll
  for (int n = 0; n < kN; ++n) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = 8 * n + 2 * t + e;
      be[n][e] = make_int2(0, 0);
      pos[n][e] = slp[n][e] = 0.f;
      if (r < pairs) {
        const int2 x = row_range<kPaged>(a, s, token_of(r));
        be[n][e] = x;
        if (a.slope != nullptr) {
          pos[n][e] = row_position<kPaged>(a, s, origin, token_of(r));
          slp[n][e] = __ldg(a.slope + head_of(r)) * kLog2E;
        }
        if (x.y > x.x) {
          lo = min(lo, x.x);
          hi = max(hi, x.y);
        }
        lo_all = max(lo_all, x.x);
        hi_all = min(hi_all, x.y);
      }
    }
  }
  // keys that some row sees [lo, hi), and those that every row sees [lo_all, hi_all): the same in every warp
  lo = __reduce_min_sync(0xffffffffu, lo) & ~15;
  hi = __reduce_max_sync(0xffffffffu, hi);
  lo_all = __reduce_max_sync(0xffffffffu, lo_all);
  hi_all = __reduce_min_sync(0xffffffffu, hi_all);
  const int steps = hi > 0 ? (hi - lo + 15) / 16 : 0;
  const int c0 = static_cast<int>(static_cast<long long>(steps) * piece / split);
  const int c1 = static_cast<int>(static_cast<long long>(steps) * (piece + 1) / split);

  const float* bias = a.bias == nullptr ? nullptr : a.bias + (kPaged ? 0 : s.batch * a.bias_sb);
  const int slot_mask = (1 << a.page_shift) - 1;
  auto page_at = [&](int c) -> int { return kPaged && c < c1 ? page_of(a, s, (lo + 16 * c) >> a.page_shift) : a.pages; };
  // TMA of step c (16 keys of one page) into place `at` of the warp's ring; past the tensor, or a page that there is not,
  // reads zeros.  After a wait that ran out nothing more is asked for: what is in flight was asked for before that wait.
  const uint32_t mine = smem_u32(ring) + warp * kRing * 2 * kSide;
  bool ok = true;
  auto fetch = [&](int c, int page, int at) {
    if (ok && c < c1 && lane == 0) {
      const uint32_t dst = mine + at * 2 * kSide, bar = bars + 8 * at;
      const int key0 = lo + 16 * c;
      mbar_arrive_expect_tx(bar, 2 * kSide);
      if constexpr (kPaged) {
        tma_load_4d(dst, &tmap_k, bar, 0, hk, key0 & slot_mask, page);
        tma_load_4d(dst + kSide, &tmap_v, bar, 0, hk, key0 & slot_mask, page);
      } else {
        tma_load_4d(dst, &tmap_k, bar, 0, key0, hk, s.batch);
        tma_load_4d(dst + kSide, &tmap_v, bar, 0, key0, hk, s.batch);
      }
    }
  };
  // the bias of key `lane` of step c, in lanes 0 to 15
  auto bias_at = [&](int c, int page) -> float {
    const int key = lo + 16 * c + lane;
    if (bias == nullptr || lane >= 16 || c >= c1 || key >= s.keys || (kPaged && page >= a.pages)) return 0.f;
    return bias_log2(__ldg(bias + (kPaged ? (static_cast<long long>(page) << a.page_shift) + (key & slot_mask) : key)));
  };

  float m[kN][2], l[kN][2], o[kN][4][4];
#pragma unroll
  for (int n = 0; n < kN; ++n) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      m[n][e] = -INFINITY;
      l[n][e] = 0.f;
    }
#pragma unroll
    for (int x = 0; x < 16; ++x) o[n][x >> 2][x & 3] = 0.f;
  }

  // page numbers are looked up one step before their tiles are asked for, biases one step before they are used
  int here[kRing], cur = 0, phase = 0;
#pragma unroll
  for (int k = 0; k < kRing - 1; ++k) {
    here[k] = page_at(c0 + warp + k * kRowWarps);
    fetch(c0 + warp + k * kRowWarps, here[k], k);
  }
  here[kRing - 1] = page_at(c0 + warp + (kRing - 1) * kRowWarps);
  float bias_next = bias_at(c0 + warp, here[0]);
  for (int c = c0 + warp; c < c1; c += kRowWarps) {
    const int key0 = lo + 16 * c, left = s.keys - key0;  // keys from key0 on
    const bool there = !kPaged || here[0] < a.pages;
    // into the place that the step before this one has left
    fetch(c + (kRing - 1) * kRowWarps, here[kRing - 1], cur == 0 ? kRing - 1 : cur - 1);
    const float bias_here = bias_next;
    bias_next = bias_at(c + kRowWarps, here[1]);
#pragma unroll
    for (int k = 0; k + 1 < kRing; ++k) here[k] = here[k + 1];
    here[kRing - 1] = page_at(c + kRing * kRowWarps);
    if (ok) ok = mbar_wait(bars + 8 * cur, phase, a.err);
    const uint8_t* kt = ring + (warp * kRing + cur) * 2 * kSide;
    const uint8_t* vt = kt + kSide;
    if (++cur == kRing) {
      cur = 0;
      phase ^= 1;
    }
    struct { uint4 k[2][2], v[4]; float bias[2]; } x;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int kr = 8 * (u >> 1) + g, kc = 2 * t + (u & 1), vr = 8 * (u >> 1) + 2 * t + (u & 1);
      x.k[u >> 1][u & 1] = *reinterpret_cast<const uint4*>(kt + kr * 128 + ((kc ^ (kr & 7)) << 4));
      x.v[u] = *reinterpret_cast<const uint4*>(vt + vr * 128 + ((g ^ (vr & 7)) << 4));
      // slots behind the last key hold anything
      if (kPaged && vr >= left) x.v[u] = make_uint4(0u, 0u, 0u, 0u);
    }
    __syncwarp();  // the step is in registers: its place can be filled
    x.bias[0] = x.bias[1] = 0.f;
    if (bias != nullptr) {
      x.bias[0] = __shfl_sync(0xffffffffu, bias_here, g);
      x.bias[1] = __shfl_sync(0xffffffffu, bias_here, 8 + g);
    }
    const uint32_t* kw[2] = {reinterpret_cast<const uint32_t*>(&x.k[0][0]), reinterpret_cast<const uint32_t*>(&x.k[1][0])};
    const uint32_t* vw[4] = {reinterpret_cast<const uint32_t*>(&x.v[0]), reinterpret_cast<const uint32_t*>(&x.v[1]),
                             reinterpret_cast<const uint32_t*>(&x.v[2]), reinterpret_cast<const uint32_t*>(&x.v[3])};
    const bool full = there && key0 >= lo_all && key0 + 16 <= hi_all;
    float kp[2] = {0.f, 0.f};
    if (a.slope != nullptr) {
#pragma unroll
      for (int u = 0; u < 2; ++u) kp[u] = key_position<kPaged>(a, s, origin, min(key0 + 8 * u + g, s.keys - 1));  // beyond: hidden
    }
    uint32_t p[kN][2];
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      float sc[4] = {0.f, 0.f, 0.f, 0.f};  // keys g (0, 1) and 8 + g (2, 3), rows 8 n + 2 t and + 1
#pragma unroll
      for (int c4 = 0; c4 < 4; ++c4) {
        const uint32_t ka[4] = {kw[0][2 * c4], kw[1][2 * c4], kw[0][2 * c4 + 1], kw[1][2 * c4 + 1]};
        mma16816(sc, ka, q[n][c4][0], q[n][c4][1], static_cast<T*>(nullptr));
      }
      float mx[2] = {-INFINITY, -INFINITY};
      if (full && a.cap == 0.f && a.slope == nullptr) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          sc[e] = fmaf(sc[e], a.scale, x.bias[e >> 1]);
          mx[e & 1] = fmaxf(mx[e & 1], sc[e]);
        }
      } else
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int u = e >> 1, r = e & 1, key = key0 + 8 * u + g;
        float y = sc[e] * a.scale;
        if (a.cap != 0.f) y = a.cap * tanh_fast(y);
        y += x.bias[u];
        if (a.slope != nullptr) y = fmaf(-slp[n][r], fabsf(pos[n][r] - kp[u]), y);
        if (!full && (!there || key < be[n][r].x || key >= be[n][r].y)) y = -INFINITY;
        sc[e] = y;
        mx[r] = fmaxf(mx[r], y);
      }
      // Lazy running maximum: O is rescaled when some row's grows by more than 2^8.  The lanes' own maxima tell whether one
      // does; only then are they brought together.  m: the maximum less kUp.
      constexpr float most = kRoom + kUp<T>;
      if (__any_sync(0xffffffffu, mx[0] > m[n][0] + most || mx[1] > m[n][1] + most)) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], d));
          if (mx[r] > m[n][r] + most) {
            const float f = ex2_approx(m[n][r] - (mx[r] - kUp<T>));
            m[n][r] = mx[r] - kUp<T>;
            l[n][r] *= f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              o[n][j][r] *= f;
              o[n][j][2 + r] *= f;
            }
          }
        }
      }
      float pr[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float mu = m[n][e & 1];
        pr[e] = ex2_approx(sc[e] - (mu == -INFINITY ? 0.f : mu));
      }
      l[n][0] += pr[0] + pr[2];
      l[n][1] += pr[1] + pr[3];
      p[n][0] = transpose8(std::is_same<T, __nv_bfloat16>::value ? pack_bf16x2(pr[0], pr[1]) : pack_f16x2(pr[0], pr[1]));
      p[n][1] = transpose8(std::is_same<T, __nv_bfloat16>::value ? pack_bf16x2(pr[2], pr[3]) : pack_f16x2(pr[2], pr[3]));
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t va[4] = {__byte_perm(vw[0][j], vw[1][j], 0x5410), __byte_perm(vw[0][j], vw[1][j], 0x7632),
                              __byte_perm(vw[2][j], vw[3][j], 0x5410), __byte_perm(vw[2][j], vw[3][j], 0x7632)};
#pragma unroll
      for (int n = 0; n < kN; ++n) mma16816(o[n][j], va, p[n][0], p[n][1], static_cast<T*>(nullptr));
    }
  }

  __syncthreads();  // every tile has been read: the ring becomes the parts
#pragma unroll
  for (int n = 0; n < kN; ++n) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) l[n][r] += __shfl_xor_sync(0xffffffffu, l[n][r], d);
      float* row = part[warp][8 * n + 2 * t + r];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        row[8 * g + 2 * j] = o[n][j][r];
        row[8 * g + 2 * j + 1] = o[n][j][2 + r];
      }
      if (g == 0) {
        row[kHeadDim] = m[n][r];
        row[kHeadDim + 1] = l[n][r];
      }
    }
  }
  __syncthreads();
  auto store = [&](int idx, float y, float sum) {
    const int r = idx / kHeadDim, ch = idx - r * kHeadDim;
    if (r >= pairs) return;
    const float z = sum == 0.f ? 0.f : y / sum;  // no visible key: 0
    if (!(z * 0.f == 0.f)) bad[r] = 1;
    static_cast<T*>(a.out)[s.batch * a.o_sb + head_of(r) * a.o_sh + static_cast<long long>(s.row0 + token_of(r)) * a.o_sn + ch] =
        from_f32<T>(z);
  };
  for (int idx = threadIdx.x; idx < kRows * kHeadDim; idx += kRowWarps * 32) {
    const int r = idx / kHeadDim, ch = idx - r * kHeadDim;
    float mm, sum, y;
    join(kRowWarps, [&](int w) -> const float* { return part[w][r]; }, ch, mm, sum, y);
    if (split == 1) {
      store(idx, y, sum);
    } else {
      fin[r][ch] = y;
      if (ch == 0) {
        fin[r][kHeadDim] = mm;
        fin[r][kHeadDim + 1] = sum;
      }
    }
  }
  if (split > 1) {
    cg::cluster_group cl = cg::this_cluster();
    cl.sync();
    const int per = kRows * kHeadDim / split;  // whole rows: split is at most 8
    for (int idx = piece * per + threadIdx.x; idx < (piece + 1) * per; idx += kRowWarps * 32) {
      const int r = idx / kHeadDim, ch = idx - r * kHeadDim;
      float mm, sum, y;
      join(split, [&](int w) -> const float* { return cl.map_shared_rank(&fin[0][0], w) + r * (kHeadDim + 2); }, ch, mm, sum, y);
      store(idx, y, sum);
    }
    cl.sync();  // the peers read this CTA's part before it leaves
  }
  __syncthreads();
  for (int r = warp; r < kRows; r += kRowWarps)
    if (bad[r]) exact_row<T, kPaged>(a, s, token_of(r), head_of(r));
}

template <typename... P, typename... A>
int launch_cluster(void (*kernel)(P...), long long items, int split, int smem, const char* what, cudaStream_t st, const A&... args) {
  VB200_REQUIRE(items * split < (1ll << 31), "attention: too many work items");
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(items * split));
  cfg.blockDim = dim3(kRowWarps * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = static_cast<unsigned>(split);
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = split > 1 ? 1 : 0;
  VB200_CHECK_CUDA(cudaLaunchKernelEx(&cfg, kernel, args...), what);
  VB200_CHECK_LAUNCH(what);
  return VB200_OK;
}

template <bool kPaged>
int launch_f32(const AttnView& a, int R, long long items, int split, cudaStream_t st) {
  auto kernel = R == 1 ? rows_attention_kernel<1, kPaged> : R == 2 ? rows_attention_kernel<2, kPaged> : rows_attention_kernel<4, kPaged>;
  return launch_cluster(kernel, items, split, 0, "rows_attention_kernel", st, a, split);
}

template <typename T, bool kPaged, int kN>
int launch_16(const AttnView& a, const CUtensorMap& tk, const CUtensorMap& tv, long long items, int split, cudaStream_t st) {
  auto kernel = few_rows_kernel<T, kPaged, kN>;
  static std::atomic<bool> ready[64];  // per device: the opt-in to the shared memory
  int dev = 0;
  VB200_CHECK_CUDA(cudaGetDevice(&dev), "cudaGetDevice");
  if (dev < 0 || dev >= 64 || !ready[dev].load(std::memory_order_acquire)) {
    VB200_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRowsSmem), "cudaFuncSetAttribute");
    if (dev >= 0 && dev < 64) ready[dev].store(true, std::memory_order_release);
  }
  return launch_cluster(kernel, items, split, kRowsSmem, "few_rows_kernel", st, a, split, tk, tv);
}

template <typename T>
int launch_16(const AttnView& a, bool paged, bool wide, long long items, int split, cudaStream_t st) {
  const int dtype = std::is_same<T, __nv_bfloat16>::value ? VB200_BF16 : VB200_F16;
  CUtensorMap tk, tv;
  int rc;
  if (paged) {
    if ((rc = pool_map(&tk, a.k, dtype, a, 16)) != VB200_OK || (rc = pool_map(&tv, a.v, dtype, a, 16)) != VB200_OK) return rc;
    return wide ? launch_16<T, true, 2>(a, tk, tv, items, split, st) : launch_16<T, true, 1>(a, tk, tv, items, split, st);
  }
  if ((rc = rows_map(&tk, a.k, dtype, a.Nk, a.Hkv, a.B, a.k_sn, a.k_sh, a.k_sb, 16)) != VB200_OK ||
      (rc = rows_map(&tv, a.v, dtype, a.Nk, a.Hkv, a.B, a.v_sn, a.v_sh, a.v_sb, 16)) != VB200_OK)
    return rc;
  return wide ? launch_16<T, false, 2>(a, tk, tv, items, split, st) : launch_16<T, false, 1>(a, tk, tv, items, split, st);
}

}  // namespace

int rows_attention(int dtype, bool paged, const AttnView& a, long long most_keys, cudaStream_t st) {
  // Pairs per CTA.  16 bits: 8, or 16 where a sequence has more on average.  fp32: as many as a sequence has on average, at
  // most 4 (17 rows of 16 heads over 1041 keys of 4 key heads: 15.9 us, with up to 8 pairs 28.7; 1041 rows over 1041 keys of
  // 16: 368 and 394).  Longer sequences take several blocks, shorter ones leave rows idle; both are right.
  const long long seqs = paged ? a.n_seq : a.B;
  const long long total = static_cast<long long>(a.Nq) * a.group;  // of all sequences (paged), or of one
  const long long mean = paged ? (total + seqs - 1) / seqs : total;
  const int R = dtype != VB200_F32 ? (mean <= 8 ? 8 : 16) : mean <= 1 ? 1 : mean <= 2 ? 2 : 4;
  const long long blocks = paged ? total / R + a.n_seq : (total + R - 1) / R * a.B;
  const long long items = blocks * a.Hkv;
  // Split the keys while the GPU is not filled and a piece keeps at least 256 keys.  fp32: up to two CTAs per SM.  16 bits: while
  // the doubled split leaves room, three CTAs on two SMs; beyond that clusters no longer all fit at once (64 items of 2000 keys:
  // 17.5 us in 4 parts, 13.3 in 2; 128 of 4000: 38 and 31).  Once more, for even ends of ragged sequences, while there are not
  // four CTAs per SM and a piece keeps 1024 keys (32 sequences of 500 to 9000: 175 -> 157 us; with twice as many parts 122 ->
  // 140).  Up to 8 parts, the portable size of a cluster (16 gained 5% for one sequence of 32,928 keys).
  int split = 1;
  const long long sms = sm_count_of_device();
  const long long busy = (paged ? std::max((total + R - 1) / R, seqs) : blocks) * a.Hkv;
  const long long fill = dtype == VB200_F32 ? 2 * sms : 3 * sms / 4 + 1;
  while (split < 8 && ((busy * split < fill && most_keys / (2 * split) >= 256) || (busy * split < 4 * sms && most_keys / (2 * split) >= 1024)))
    split *= 2;
  if (dtype == VB200_F32) return paged ? launch_f32<true>(a, R, items, split, st) : launch_f32<false>(a, R, items, split, st);
  return dtype == VB200_BF16 ? launch_16<__nv_bfloat16>(a, paged, R > 8, items, split, st) : launch_16<__half>(a, paged, R > 8, items, split, st);
}

}  // namespace vb200
