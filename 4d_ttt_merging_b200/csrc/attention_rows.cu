// Masked and paged attention for few query rows per key head (a token per stream, a handful of special
// tokens) and for fp32 inputs, on the FMA pipe.  The mathematics is in attention_view.cuh.
//
// One CTA takes R (query row, head of the group) pairs of one sequence and one key head, so a key is
// read once for all heads that share it.  Eight lanes hold one key (8 channels each); the 4 keys of a
// load and the U loads of a step are independent, each lane group keeps its own running maximum and sum
// (no exchange per step), and groups, warps and the CTAs of a cluster are joined once at the end in a
// fixed order.  The keys are split over a cluster of up to 8 CTAs when the pairs alone do not fill the
// GPU; the parts meet in distributed shared memory, so there is no workspace and no second launch.
//
// Bound: reading K and V (256 bytes a key in 16 bits) at 23 bytes per SM clock; 1 row costs about 10
// warp instructions per key of the 44 that fit in that time, 8 rows about 45.
#include <cooperative_groups.h>

#include "attention_view.cuh"
#include "host_common.h"
#include "masked_host.h"

namespace cg = cooperative_groups;

namespace vb200 {
namespace {

constexpr int kRowWarps = 8;

template <typename T>
struct Key8;  // 8 channels of a row as four packed fp32 pairs
template <>
struct Key8<float> {
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
template <typename T>
struct Key8 {
  uint4 a;
  __device__ __forceinline__ void load(const T* p) { a = __ldg(reinterpret_cast<const uint4*>(p)); }
  __device__ __forceinline__ void zero() { a = make_uint4(0u, 0u, 0u, 0u); }
  __device__ __forceinline__ void unpack(uint64_t (&x)[4]) const {
    const T* e = reinterpret_cast<const T*>(&a);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = pk2(to_f32<T>(e[2 * i]), to_f32<T>(e[2 * i + 1]));
  }
};

template <typename T, int R, bool kPaged>
__global__ void __launch_bounds__(kRowWarps * 32, R <= 4 ? 2 : 1) rows_attention_kernel(const AttnView a, int split) {
  constexpr int U = sizeof(T) == 4 ? 2 : 4;  // loads in flight per lane: 4 x (K, V) vectors of 16 bytes
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

  if (threadIdx.x < R) {
    const int r = threadIdx.x;
    int2 be = make_int2(0, 0);
    float p = 0.f, sl = 0.f;
    if (r < pairs) {
      const int i = static_cast<int>((pair0 + r) / a.group), g = static_cast<int>((pair0 + r) % a.group);
      be = row_range<kPaged>(a, s, i);
      if (a.slope != nullptr) {
        p = row_position<kPaged>(a, s, i);
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
    Key8<T> x;
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
    Key8<T> kr[U], vr[U];
    float bs[U], kp[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int off = u * 4 + grp;
      if (there && (full || key0 + off < s.keys)) {
        kr[u].load(kb + koff + static_cast<long long>(at0 + off) * a.k_sn);
        vr[u].load(vb_ + voff + static_cast<long long>(at0 + off) * a.v_sn);
        bs[u] = bias == nullptr ? 0.f : bias_log2(__ldg(bias + boff + at0 + off));
        kp[u] = !dist ? 0.f : (!kPaged && a.kpos != nullptr ? __ldg(a.kpos + s.batch * a.kpos_sb + key0 + off)
                                                            : static_cast<float>(key0 + off));
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
        for (int r = 0; r < R; ++r) x[u][r] = a.cap * (sizeof(T) == 4 ? tanhf(x[u][r]) : tanh_fast(x[u][r]));
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
    float mx = -INFINITY, sum = 0.f, o = 0.f;
#pragma unroll
    for (int w = 0; w < kRowWarps; ++w) mx = fmaxf(mx, part[w][r][kHeadDim]);
    const float mu = mx == -INFINITY ? 0.f : mx;
#pragma unroll
    for (int w = 0; w < kRowWarps; ++w) {
      const float f = ex2_approx(part[w][r][kHeadDim] - mu);
      sum = fmaf(part[w][r][kHeadDim + 1], f, sum);
      o = fmaf(part[w][r][ch], f, o);
    }
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
      float mx = -INFINITY, sum = 0.f, o = 0.f;
      for (int w = 0; w < split; ++w) mx = fmaxf(mx, cl.map_shared_rank(&fin[0][0], w)[r * (kHeadDim + 2) + kHeadDim]);
      const float mu = mx == -INFINITY ? 0.f : mx;
      for (int w = 0; w < split; ++w) {
        const float* f = cl.map_shared_rank(&fin[0][0], w) + r * (kHeadDim + 2);
        const float e = ex2_approx(f[kHeadDim] - mu);
        sum = fmaf(f[kHeadDim + 1], e, sum);
        o = fmaf(f[ch], e, o);
      }
      store(idx, o, sum);
    }
    cl.sync();  // the peers read this CTA's part before it leaves
  }
}

template <typename T, int R, bool kPaged>
int launch_one(const AttnView& a, long long items, int split, cudaStream_t st) {
  VB200_REQUIRE(items * split < (1ll << 31), "attention: too many work items");
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(items * split));
  cfg.blockDim = dim3(kRowWarps * 32);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = static_cast<unsigned>(split);
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = split > 1 ? 1 : 0;
  VB200_CHECK_CUDA(cudaLaunchKernelEx(&cfg, rows_attention_kernel<T, R, kPaged>, a, split), "rows_attention_kernel");
  VB200_CHECK_LAUNCH("rows_attention_kernel");
  return VB200_OK;
}

template <typename T, bool kPaged>
int launch_rows(const AttnView& a, int R, long long items, int split, cudaStream_t st) {
  switch (R) {
    case 1: return launch_one<T, 1, kPaged>(a, items, split, st);
    case 2: return launch_one<T, 2, kPaged>(a, items, split, st);
    case 4: return launch_one<T, 4, kPaged>(a, items, split, st);
    default: return launch_one<T, 8, kPaged>(a, items, split, st);
  }
}

}  // namespace

int rows_attention(int dtype, bool paged, const AttnView& a, long long most_keys, cudaStream_t st) {
  // Pairs per CTA: as many as a sequence has on average, at most 8 (registers).  Longer ones take
  // several blocks, shorter ones leave pairs idle; both are right.
  const long long seqs = paged ? a.n_seq : a.B;
  const long long mean = (static_cast<long long>(a.Nq) * (paged ? 1 : seqs) * a.group + seqs - 1) / seqs;
  const int R = mean <= 1 ? 1 : mean <= 2 ? 2 : mean <= 4 ? 4 : 8;
  const long long blocks = paged ? static_cast<long long>(a.Nq) * a.group / R + a.n_seq
                                 : (static_cast<long long>(a.Nq) * a.group + R - 1) / R * a.B;
  const long long items = blocks * a.Hkv;
  // Split the keys while two CTAs per SM are not filled and a piece keeps at least 256 keys.
  int split = 1;
  const long long fill = 2ll * sm_count_of_device();
  const long long busy = paged ? (static_cast<long long>(a.Nq) * a.group + R - 1) / R * a.Hkv : items;
  while (split < 8 && busy * split < fill && most_keys / (2 * split) >= 256) split *= 2;
  if (dtype == VB200_F32)
    return paged ? launch_rows<float, true>(a, R, items, split, st) : launch_rows<float, false>(a, R, items, split, st);
  if (dtype == VB200_BF16)
    return paged ? launch_rows<__nv_bfloat16, true>(a, R, items, split, st)
                 : launch_rows<__nv_bfloat16, false>(a, R, items, split, st);
  return paged ? launch_rows<__half, true>(a, R, items, split, st) : launch_rows<__half, false>(a, R, items, split, st);
}

}  // namespace vb200
