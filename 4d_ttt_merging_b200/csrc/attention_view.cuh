// What the masked and the paged attention share: the launch arguments, the map from a block of
// query rows to its sequence, the interval of keys that a row sees, and the addresses of keys in a
// dense tensor or in the pages of a cache.
//
//   x_ij = cap tanh(scale q_i.k_j / cap) + bias_j - slope_h |pos_i - pos_j|
//   o_i  = sum_j e^{x_ij} v_j / sum_j e^{x_ij}  over the keys j in [begin_i, end_i); 0 when empty
//
// Everything below works in the log2 domain: scale, cap, bias and slope carry a factor log2(e).
#pragma once

#include "common.cuh"

namespace vb200 {

constexpr float kLog2E = 1.4426950408889634f;
constexpr float kLowest = -3.4028234663852886e38f;
constexpr int kHeadDim = 64;

struct AttnView {
  const void *q, *k, *v;
  void* out;
  // element strides: {batch, head, token}; paged k / v: {page, head, slot}, q / out: {unused, head, row}
  long long q_sb, q_sh, q_sn, k_sb, k_sh, k_sn, v_sb, v_sh, v_sn, o_sb, o_sh, o_sn;
  int B, H, Hkv, group;        // group = H / Hkv query heads share one key head
  int Nq, Nk;                  // dense: rows and keys; paged: Nq = rows of q in all sequences
  const float* bias;           // per key (natural log), dense [B or 1][Nk], paged [pages][page]; may be null
  long long bias_sb;
  const int* range;            // [B or 1][Nq][2] or null (paged: [Nq][2] or null)
  long long range_sb;
  const float* slope;          // [H] or null
  const float *qpos, *kpos;    // dense, with slope: positions, or null for the token index
  long long qpos_sb, kpos_sb;
  float scale;                 // scale * log2(e) without a cap; scale / cap with one
  float cap;                   // cap * log2(e), 0 without a cap
  // paged
  const int *table, *length, *sequence, *offsets;
  long long table_stride;
  int n_seq, slots, pages, page_shift, max_pages, causal;
  unsigned* err;
};

// The sequence that a block of query rows belongs to.
struct AttnSeq {
  int rows;        // query rows of the sequence
  int row0;        // its first row in q and out
  int keys;        // keys it holds
  int batch;       // dense batch entry
  const int* pages;  // paged: its table row
};

// Blocks of `per` units (rows, or row x head pairs: `mult` units per row) over ragged sequences,
// without a host that knows their lengths: sequence i's blocks start at index offsets[i] * mult / per
// + i.  The starts of two neighbours differ by at least ceil(rows * mult / per), so blocks never
// overlap; indices between a sequence's last block and the next start are empty.  Returns false for
// an empty index.  Called by the whole block (it has a barrier): the threads look at the starts side by side, one load deep,
// where a search would make log2(sequences) dependent ones (0.6 us each).  Offsets that do not ascend or leave [0, Nq], and slots out of range, set the error
// word and leave the sequence out.
template <bool kPaged>
__device__ __forceinline__ bool locate_block(const AttnView& a, int index, int per, int mult, AttnSeq& s, int& block) {
  if constexpr (!kPaged) {
    const int per_batch = (a.Nq * mult + per - 1) / per;  // host: Nq * mult < 2^31
    s.batch = index / per_batch;
    block = index - s.batch * per_batch;
    s.rows = a.Nq;
    s.row0 = 0;
    s.keys = a.Nk;
    s.pages = nullptr;
    return s.batch < a.B;
  } else {
    auto start = [&](int i) -> long long {
      const int o = min(max(__ldg(a.offsets + i), 0), a.Nq);
      return static_cast<long long>(o) * mult / per + i;
    };
    int upto = 0;  // sequences that start at or before the index
    for (int base = 0; base < a.n_seq; base += blockDim.x) {
      const int i = base + static_cast<int>(threadIdx.x);
      const int here = __syncthreads_count(i < a.n_seq && start(i) <= index);
      upto += here;
      if (here < static_cast<int>(blockDim.x)) break;  // the same in every thread
    }
    const int lo = max(upto - 1, 0);
    const int o0 = __ldg(a.offsets + lo), o1 = __ldg(a.offsets + lo + 1);
    const int slot = a.sequence == nullptr ? lo : __ldg(a.sequence + lo);
    if (o0 < 0 || o1 < o0 || o1 > a.Nq || slot < 0 || slot >= a.slots) {
      if (threadIdx.x == 0) atomicOr(a.err, kErrBadArgument);
      return false;
    }
    const long long b = index - start(lo);
    s.rows = o1 - o0;
    if (b < 0 || b * per >= static_cast<long long>(s.rows) * mult) return false;
    block = static_cast<int>(b);
    s.row0 = o0;
    s.batch = 0;
    // a length beyond the table's room (a damaged handle) reads no further than the table
    s.keys = min(max(__ldg(a.length + slot), 0), static_cast<int>(min(static_cast<long long>(a.max_pages) << a.page_shift, 0x7fffffffll)));
    s.pages = a.table + slot * a.table_stride;
    return true;
  }
}

// [begin, end) of row i of the sequence, inside [0, keys); empty as [0, 0).
template <bool kPaged>
__device__ __forceinline__ int2 row_range(const AttnView& a, const AttnSeq& s, int i) {
  int b = 0, e = s.keys;
  if (a.range != nullptr) {
    const int* r = a.range + (kPaged ? 0 : s.batch * a.range_sb) + 2ll * (s.row0 + i);
    b = max(__ldg(r), 0);
    e = min(__ldg(r + 1), s.keys);
  } else if (kPaged && a.causal) {
    e = min(e, s.keys - s.rows + i + 1);
  }
  return e > b ? make_int2(b, e) : make_int2(0, 0);
}

// Positions in fp32.  Token indices are counted from that of a row of the block (its first, say): fp32 holds every whole number up
// to 2^24 only, and in a longer sequence the distances between neighbours would be lost; counted so, a distance d is off by
// 2^-24 d at most.  Positions that are given stand as they are.
template <bool kPaged>
__device__ __forceinline__ int position_origin(const AttnView& a, const AttnSeq& s, int row) {
  return !kPaged && (a.qpos != nullptr || a.kpos != nullptr) ? 0 : s.keys - s.rows + row;
}
template <bool kPaged>
__device__ __forceinline__ float row_position(const AttnView& a, const AttnSeq& s, int origin, int i) {
  if (!kPaged && a.qpos != nullptr) return __ldg(a.qpos + s.batch * a.qpos_sb + i);
  return static_cast<float>(s.keys - s.rows + i - origin);
}
template <bool kPaged>
__device__ __forceinline__ float key_position(const AttnView& a, const AttnSeq& s, int origin, int j) {
  if (!kPaged && a.kpos != nullptr) return __ldg(a.kpos + s.batch * a.kpos_sb + j);
  return static_cast<float>(j - origin);
}

// Page of a key tile's slot, or `pages` (outside the pool) with the error word set when the table
// holds no page there.
__device__ __forceinline__ int page_of(const AttnView& a, const AttnSeq& s, int slot) {
  const int id = __ldg(s.pages + slot);
  if (id < 0 || id >= a.pages) {
    atomicOr(a.err, kErrBadArgument);
    return a.pages;
  }
  return id;
}

// Log2-domain bias of a key.  A finite bias stays finite: the type's lowest value times log2(e) would overflow, and a row
// whose every key has it would come out empty instead of uniform.
__device__ __forceinline__ float bias_log2(float b) {
  const float x = b * kLog2E;
  return fabsf(b) == INFINITY ? b : x > -kLowest ? -kLowest : x < kLowest ? kLowest : x;
}

// tanh(y) / y as a polynomial in y^2, fitted here for minimum maximum relative error (least squares reweighted to equal
// ripples): degree 3 for |y| <= 1/2 (5e-7), degree 5 for |y| <= 1 (6e-7); 7e-7 evaluated in fp32.
constexpr double kTanhNear[4] = {0.999999463558197, -0.33326318860054016, 0.13190296292304993, -0.04440222308039665};
constexpr double kTanhFar[6] = {0.9999994039535522,    -0.3332904279232025,  0.13281433284282684,
                                -0.051605671644210815, 0.016743112355470657, -0.0030670592095702887};

// tanh for scores held in fp32 and probabilities rounded to 16 bits, to 7e-7 relative: times any cap, 7e-7 of the score.  The
// polynomial up to 1/2, beyond it 1 - 2 / (e^{2y} + 1), which is good to 2e-7 absolute (ex2.approx and rcp.approx to 2^-22
// relative, the subtraction rounds at 2^-24): a score far below its cap would lose all its bits there.  e^{2y} = inf gives 1, 0 gives -1.
__device__ __forceinline__ float tanh_fast(float y) {
  constexpr float c0 = static_cast<float>(kTanhNear[0]), c1 = static_cast<float>(kTanhNear[1]), c2 = static_cast<float>(kTanhNear[2]),
                  c3 = static_cast<float>(kTanhNear[3]);
  const float z = y * y, e = ex2_approx(y * (2.f * kLog2E));
  const float f = fmaf(fmaf(fmaf(c3, z, c2), z, c1), z, c0);
  return fabsf(y) <= 0.5f ? f * y : 1.f - __fdividef(2.f, e + 1.f);
}

// One output row by one warp, key by key, two channels per lane: for rows that a tensor-core kernel finds not finite.  There a
// hidden key's probability 0 meets its value, whatever that is, in the product; here hidden keys are not read.
template <typename T, bool kPaged>
__device__ __noinline__ void exact_row(const AttnView& a, AttnSeq s, int i, int head) {
  const int lane = threadIdx.x & 31, hk = head / a.group;
  const int2 be = row_range<kPaged>(a, s, i);
  const float slope = a.slope == nullptr ? 0.f : __ldg(a.slope + head) * kLog2E;
  const int origin = position_origin<kPaged>(a, s, i);
  const float pos = row_position<kPaged>(a, s, origin, i);
  const T* q = static_cast<const T*>(a.q) + s.batch * a.q_sb + head * a.q_sh + static_cast<long long>(s.row0 + i) * a.q_sn + 2 * lane;
  const float q0 = to_f32<T>(q[0]) * a.scale, q1 = to_f32<T>(q[1]) * a.scale;
  float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
  for (int j0 = be.x; j0 < be.y; j0 += 32) {
    // each lane looks at one key: where it lies, its bias; keys of mass 0 are left out
    long long ko = 0, vo = 0;
    float b = -INFINITY, kp = 0.f;
    if (j0 + lane < be.y) {
      const int j = j0 + lane;
      b = 0.f;
      if constexpr (kPaged) {
        const int id = page_of(a, s, j >> a.page_shift), at = j & ((1 << a.page_shift) - 1);
        ko = id * a.k_sb + at * a.k_sn;
        vo = id * a.v_sb + at * a.v_sn;
        if (id >= a.pages) b = -INFINITY;
        else if (a.bias != nullptr) b = bias_log2(__ldg(a.bias + (static_cast<long long>(id) << a.page_shift) + at));
      } else {
        ko = s.batch * a.k_sb + j * a.k_sn;
        vo = s.batch * a.v_sb + j * a.v_sn;
        if (a.bias != nullptr) b = bias_log2(__ldg(a.bias + s.batch * a.bias_sb + j));
      }
      if (a.slope != nullptr) kp = key_position<kPaged>(a, s, origin, j);
    }
    for (unsigned some = __ballot_sync(0xffffffffu, b != -INFINITY); some != 0; some &= some - 1) {
      const int from = __ffs(some) - 1;
      const T* k = static_cast<const T*>(a.k) + __shfl_sync(0xffffffffu, ko, from) + hk * a.k_sh + 2 * lane;
      const T* v = static_cast<const T*>(a.v) + __shfl_sync(0xffffffffu, vo, from) + hk * a.v_sh + 2 * lane;
      float x = q0 * to_f32<T>(k[0]) + q1 * to_f32<T>(k[1]);
#pragma unroll
      for (int d = 16; d >= 1; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
      if (a.cap != 0.f) x = a.cap * tanh_fast(x);
      x += __shfl_sync(0xffffffffu, b, from);
      const float at = __shfl_sync(0xffffffffu, kp, from);
      if (a.slope != nullptr) x = fmaf(-slope, fabsf(pos - at), x);
      const float mn = fmaxf(m, x), mu = mn == -INFINITY ? 0.f : mn;
      const float corr = ex2_approx(m - mu), p = ex2_approx(x - mu);
      m = mn;
      l = l * corr + p;
      o0 = o0 * corr + p * to_f32<T>(v[0]);
      o1 = o1 * corr + p * to_f32<T>(v[1]);
    }
  }
  T* out = static_cast<T*>(a.out) + s.batch * a.o_sb + head * a.o_sh + static_cast<long long>(s.row0 + i) * a.o_sn + 2 * lane;
  out[0] = from_f32<T>(l == 0.f ? 0.f : o0 / l);
  out[1] = from_f32<T>(l == 0.f ? 0.f : o1 / l);
}

}  // namespace vb200
