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
// an empty index.  Offsets that do not ascend or leave [0, Nq], and slots out of range, set the error
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
    int lo = 0, hi = a.n_seq;  // the last i with start(i) <= index
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (start(mid) <= index) lo = mid;
      else hi = mid;
    }
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

template <bool kPaged>
__device__ __forceinline__ float row_position(const AttnView& a, const AttnSeq& s, int i) {
  if (!kPaged && a.qpos != nullptr) return __ldg(a.qpos + s.batch * a.qpos_sb + i);
  return static_cast<float>(s.keys - s.rows + i);
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

// tanh for scores held in fp32 and probabilities rounded to 16 bits: 1 - 2 / (e^{2y} + 1).  Absolute
// error about 2e-7 (ex2.approx and rcp.approx are good to 2^-22 relative, the subtraction rounds at
// 2^-24), which times a cap of 100 moves a probability by 2e-5 relative, 1/100 of its rounding to
// bf16; e^{2y} = inf gives 1, 0 gives -1.
__device__ __forceinline__ float tanh_fast(float y) {
  const float e = ex2_approx(y * (2.f * kLog2E));
  return 1.f - __fdividef(2.f, e + 1.f);
}

}  // namespace vb200
