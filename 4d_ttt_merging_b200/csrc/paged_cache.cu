// Page operations of a streamed key / value cache: append, fork, free, compact.
//
// State (all on the device): pools k, v [pages][page][kv heads][64] and log_mass [pages][page]; per slot a
// table row of page numbers (-1: none) and a length; per page a reference count (0: free).
//
//   append   sequence i's chunk goes behind its tokens.  New pages are the free ones, lowest number first,
//            in the order of the call's sequences.  A partly filled last page that another slot shares
//            is first copied (its filled rows only).  All or nothing: when the pool or a table row is too short,
//            nothing changes and the error word gets kErrCacheFull
//            (kErrBadArgument for offsets that do not ascend).
//   fork     every source row is read before any target row is written; a target releases what it held; of
//            several pairs with one target the last counts.
//   free     the slots' pages lose a reference each, the slots become empty.
//   compact  with L pages in use, the j-th used page >= L moves into the j-th free page < L.  Sources and
//            destinations are disjoint, so the copies need no order.
//
// The bookkeeping is a few thousand integers: one CTA (one cluster for fork) with block-wide scans, bound by the
// latency of its dependent loads.  The copies are bound by HBM: each moved byte is read and written
// once, a warp per token row (append) or 16 KB pieces of a page (compact), at least 64 bytes in flight per lane.
// Integer atomics only, so results do not depend on timing.
#include <cooperative_groups.h>

#include "common.cuh"
#include "host_common.h"

namespace cg = cooperative_groups;

namespace vb200 {
namespace {

static __device__ unsigned g_cache_err;

constexpr int kBook = 1024;  // threads of the bookkeeping CTAs
constexpr int kForkCtas = 8;
constexpr int kFewSlots = 128;

struct CacheView {
  uint8_t *k, *v;
  float* mass;
  int *table, *length, *refs;
  int pages, page, slots, max_pages;
  int row_vecs;  // 16-byte vectors of one token's K (or V) row
};

// Exclusive prefix sum over the block; `total` gets the sum.  red holds 33 ints.
__device__ __forceinline__ int block_scan(int x, int* red, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int inc = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += y;
  }
  __syncthreads();  // red may still be read by the previous scan
  if (lane == 31) red[warp] = inc;
  __syncthreads();
  if (warp == 0) {
    int w = red[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += y;
    }
    red[lane] = w;
  }
  __syncthreads();
  total = red[31];
  return inc - x + (warp > 0 ? red[warp - 1] : 0);
}

// ---------------------------------------------------------------- append

struct AppendWork {
  int* status;  // [0] 1: the appends take place
  int* old_len;   // [n] length before the call, -1: the sequence is left out
  int* copy_src;  // [n] shared last page to copy, or -1
  int* first;     // [n] first table slot that gets a new page
  int* start;     // [n] index of its first new page among the call's
  int* claim;     // [slots]
  int* free_list;  // [pages]
};

__global__ void __launch_bounds__(kBook, 1)
    append_plan_kernel(const CacheView c, const int* __restrict__ sequence, const int* __restrict__ offsets, int n, int tokens,
                       AppendWork w) {
  __shared__ int red[33];
  __shared__ int fail;
  __shared__ int slots[kFewSlots];
  const int tid = threadIdx.x;
  if (tid == 0) fail = 0;
  // The first of a slot's mentions counts.  Few sequences compare their slots in shared memory; many claim them in the
  // workspace, two more round trips to memory.
  if (n <= kFewSlots) {
    if (tid < n) slots[tid] = sequence[tid];
    __syncthreads();
  } else {
    for (int i = tid; i < n; i += kBook) {
      const int slot = sequence[i];
      if (slot >= 0 && slot < c.slots) w.claim[slot] = 0x7fffffff;
    }
    __syncthreads();
    for (int i = tid; i < n; i += kBook) {
      const int slot = sequence[i];
      if (slot >= 0 && slot < c.slots) atomicMin(&w.claim[slot], i);
    }
    __syncthreads();
  }
  auto first_mention = [&](int i, int slot) {
    if (n > kFewSlots) return w.claim[slot] == i;
    // as many steps for every lane: lanes that left the loop one by one would make the loads below one by one (36 -> 9 us for
    // 64 sequences)
    bool before = false;
#pragma unroll 8
    for (int k = 0; k < n; ++k) before |= k < i && slots[k] == slot;
    return !before;
  };
  long long needs = 0;
  for (int base = 0; base < n; base += kBook) {
    const int i = base + tid;
    int need = 0, old = -1, first = 0, src = -1;
    if (i < n) {
      const int slot = sequence[i], o0 = offsets[i], o1 = offsets[i + 1];
      if (o0 < 0 || o1 < o0 || o1 > tokens) {  // with ascending offsets the sums below fit in 32 bits
        atomicOr(&fail, 2);
      } else if (slot < 0 || slot >= c.slots || !first_mention(i, slot)) {
        atomicOr(&g_cache_err, kErrBadArgument);  // a slot out of range or named before: left out
      } else {
        const int count = o1 - o0;
        old = max(c.length[slot], 0);
        const int have = (old + c.page - 1) / c.page;
        const long long want = (static_cast<long long>(old) + count + c.page - 1) / c.page;
        if (want > c.max_pages) {
          atomicOr(&fail, 1);
        } else {
          if (count > 0 && old % c.page != 0) {
            const int last = c.table[static_cast<long long>(slot) * c.max_pages + have - 1];
            if (last < 0 || last >= c.pages) {
              atomicOr(&fail, 2);
            } else if (c.refs[last] > 1) {
              src = last;
            }
          }
          first = have - (src >= 0 ? 1 : 0);
          need = static_cast<int>(want) - first;
        }
      }
    }
    int total;
    const int before = block_scan(need, red, total);
    if (i < n) {
      w.old_len[i] = old;
      w.copy_src[i] = src;
      w.first[i] = first;
      w.start[i] = static_cast<int>(min(needs + before, 0x7fffffffll));
    }
    needs += total;  // at most 1024 * max_pages a round; more than the pool fails below
    if (needs > c.pages) break;
  }
  __syncthreads();
  if (needs > c.pages || fail) {
    if (tid == 0) {
      w.status[0] = 0;
      atomicOr(&g_cache_err, (fail & 2) ? kErrBadArgument : kErrCacheFull);
    }
    return;
  }
  // the lowest free pages, four per thread and round
  int found = 0;
  for (int base = 0; base < c.pages && found < needs; base += 4 * kBook) {
    const int p = base + 4 * tid;
    int f = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (p + k < c.pages && c.refs[p + k] == 0) f |= 1 << k;
    int total;
    int at = found + block_scan(__popc(f), red, total);
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if ((f >> k) & 1) w.free_list[at++] = p + k;
    found += total;
  }
  __syncthreads();
  if (found < needs) {
    if (tid == 0) {
      w.status[0] = 0;
      atomicOr(&g_cache_err, kErrCacheFull);
    }
    return;
  }
  if (tid == 0) w.status[0] = 1;
  const int lane = tid & 31;
  for (int i = tid >> 5; i < n; i += kBook / 32) {
    const int old = w.old_len[i];
    if (old < 0) continue;
    const int slot = sequence[i], len = old + offsets[i + 1] - offsets[i];
    const int first = w.first[i], need = (len + c.page - 1) / c.page - first;
    for (int j = lane; j < need; j += 32) {
      const int p = w.free_list[w.start[i] + j];
      c.table[static_cast<long long>(slot) * c.max_pages + first + j] = p;
      c.refs[p] = 1;
    }
    if (lane == 0) {
      if (w.copy_src[i] >= 0) atomicSub(&c.refs[w.copy_src[i]], 1);
      c.length[slot] = len;
    }
  }
}

// One warp per row: the call's tokens, then the filled rows of shared last pages.
__global__ void __launch_bounds__(256)
    append_write_kernel(const CacheView c, const int* __restrict__ sequence, const int* __restrict__ offsets, int n, int tokens,
                        const uint8_t* __restrict__ k, const uint8_t* __restrict__ v, long long k_st, long long k_sh, long long v_st,
                        long long v_sh, int head_vecs, const float* __restrict__ mass, AppendWork w) {
  const int lane = threadIdx.x & 31;
  const long long row = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  cudaGridDependencySynchronize();  // launched while the plan still runs
  if (w.status[0] == 0) return;
  const uint8_t *ks, *vs;
  const float* ms = nullptr;
  long long dst;  // row of the pools
  long long ksh = k_sh, vsh = v_sh;
  if (row < tokens) {
    const int t = static_cast<int>(row);
    int lo = 0, hi = n;  // the last i with offsets[i] <= t
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (__ldg(offsets + mid) <= t) lo = mid;
      else hi = mid;
    }
    const int o0 = __ldg(offsets + lo);
    const int old = w.old_len[lo];
    if (old < 0 || t < o0 || t >= __ldg(offsets + lo + 1)) return;  // before the first, behind the last, or left out
    const int at = old + t - o0;
    const int slot = __ldg(sequence + lo);
    const int p = c.table[static_cast<long long>(slot) * c.max_pages + at / c.page];
    dst = static_cast<long long>(p) * c.page + at % c.page;
    ks = k + t * k_st;
    vs = v + t * v_st;
    if (mass != nullptr) ms = mass + t;
  } else {
    const long long x = row - tokens;
    const int i = static_cast<int>(x / c.page), r = static_cast<int>(x - static_cast<long long>(i) * c.page);
    if (i >= n) return;
    const int src = w.copy_src[i], old = w.old_len[i];
    if (src < 0 || r >= old % c.page) return;
    const int p = c.table[static_cast<long long>(__ldg(sequence + i)) * c.max_pages + old / c.page];
    dst = static_cast<long long>(p) * c.page + r;
    const long long from = static_cast<long long>(src) * c.page + r;
    ks = c.k + from * c.row_vecs * 16;
    vs = c.v + from * c.row_vecs * 16;
    ksh = vsh = static_cast<long long>(head_vecs) * 16;
    if (c.mass != nullptr) ms = c.mass + from;
  }
  uint4* kd = reinterpret_cast<uint4*>(c.k) + dst * c.row_vecs;
  uint4* vd = reinterpret_cast<uint4*>(c.v) + dst * c.row_vecs;
  constexpr int U = 4;
  for (int b = lane; b < c.row_vecs; b += 32 * U) {
    uint4 x[U], y[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = b + 32 * u;
      if (i < c.row_vecs) {
        const int h = i / head_vecs, e = i - h * head_vecs;
        x[u] = *reinterpret_cast<const uint4*>(ks + h * ksh + e * 16);
        y[u] = *reinterpret_cast<const uint4*>(vs + h * vsh + e * 16);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = b + 32 * u;
      if (i < c.row_vecs) {
        kd[i] = x[u];
        vd[i] = y[u];
      }
    }
  }
  // a cache with masses whose call brings none: mass 1
  if (lane == 0 && c.mass != nullptr) c.mass[dst] = ms != nullptr ? *ms : 0.f;
}

// ---------------------------------------------------------------- free

__global__ void __launch_bounds__(256) free_kernel(const CacheView c, const int* __restrict__ sequence) {
  const int slot = sequence[blockIdx.x];
  if (slot < 0 || slot >= c.slots) {
    if (threadIdx.x == 0) atomicOr(&g_cache_err, kErrBadArgument);
    return;
  }
  int* row = c.table + static_cast<long long>(slot) * c.max_pages;
  for (int j = threadIdx.x; j < c.max_pages; j += 256) {
    if (row[j] < 0) continue;
    const int p = atomicExch(&row[j], -1);  // a slot named twice gives its pages back once
    if (p >= 0 && p < c.pages) atomicSub(&c.refs[p], 1);
  }
  if (threadIdx.x == 0) c.length[slot] = 0;
}

// ---------------------------------------------------------------- fork

// claim [slots], snap [n][max_pages], len [n]
__global__ void __launch_bounds__(kBook, 1)
    fork_kernel(const CacheView c, const int* __restrict__ source, const int* __restrict__ target, int n, int* claim, int* snap, int* len) {
  cg::cluster_group cl = cg::this_cluster();
  const int tid = blockIdx.x * kBook + threadIdx.x, all = kForkCtas * kBook;
  auto valid = [&](int i) {
    const int s = source[i], t = target[i];
    return s >= 0 && s < c.slots && t >= 0 && t < c.slots;
  };
  for (int i = tid; i < n; i += all) {
    if (valid(i)) claim[target[i]] = -1;
    else atomicOr(&g_cache_err, kErrBadArgument);
  }
  cl.sync();
  // 32 table entries of a pair per warp and step, the same ones in both passes (a row per warp: 12.1 us for 64 pairs of 134
  // pages, now 10.3)
  const int warp = tid >> 5, lane = tid & 31, warps = all / 32, chunks = (c.max_pages + 31) / 32;
  const long long units = static_cast<long long>(n) * chunks;
  for (long long u = warp; u < units; u += warps) {
    const int i = static_cast<int>(u / chunks), j = static_cast<int>(u - static_cast<long long>(i) * chunks) * 32 + lane;
    if (!valid(i)) continue;
    const int s = source[i];
    if (j < c.max_pages) snap[static_cast<long long>(i) * c.max_pages + j] = c.table[static_cast<long long>(s) * c.max_pages + j];
    if (j == 0) {
      len[i] = c.length[s];
      atomicMax(&claim[target[i]], i);
    }
  }
  cl.sync();
  for (long long u = warp; u < units; u += warps) {
    const int i = static_cast<int>(u / chunks), j = static_cast<int>(u - static_cast<long long>(i) * chunks) * 32 + lane;
    if (!valid(i) || source[i] == target[i] || __ldcg(&claim[target[i]]) != i) continue;
    int* row = c.table + static_cast<long long>(target[i]) * c.max_pages;
    if (j < c.max_pages) {
      const int p = snap[static_cast<long long>(i) * c.max_pages + j], old = row[j];  // snap: written by this lane
      if (p >= 0 && p < c.pages) atomicAdd(&c.refs[p], 1);
      if (old >= 0 && old < c.pages) atomicSub(&c.refs[old], 1);
      row[j] = p;
    }
    if (j == 0) c.length[target[i]] = len[i];
  }
}

// ---------------------------------------------------------------- compact

struct CompactWork {
  int* moves;  // [0] number of moves
  int* from;   // [pages]
  int* to;     // [pages]
  int* map;    // [pages], for pages that move
};

__global__ void __launch_bounds__(kBook, 1) compact_plan_kernel(const CacheView c, int* used, CompactWork w) {
  __shared__ int red[33];
  const int tid = threadIdx.x;
  int live = 0;
  for (int p = tid; p < c.pages; p += kBook) live += c.refs[p] > 0;
  int L;
  block_scan(live, red, L);
  int movers = 0, holes = 0;
  for (int base = 0; base < c.pages; base += 4 * kBook) {
    const int p = base + 4 * tid;
    int mv = 0, ho = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (p + k >= c.pages) continue;
      const bool on = c.refs[p + k] > 0;
      if (p + k >= L) w.map[p + k] = p + k;
      if (on && p + k >= L) mv |= 1 << k;
      if (!on && p + k < L) ho |= 1 << k;
    }
    int total;
    // both counts in one scan: at most 4096 of each in a round
    const int at = block_scan(__popc(mv) | (__popc(ho) << 16), red, total);
    int m = movers + (at & 0xffff), h = holes + (at >> 16);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if ((mv >> k) & 1) w.from[m++] = p + k;
      if ((ho >> k) & 1) w.to[h++] = p + k;
    }
    movers += total & 0xffff;
    holes += total >> 16;
  }
  __syncthreads();  // as many movers as holes
  for (int i = tid; i < movers; i += kBook) {
    const int a = w.from[i], b = w.to[i];
    w.map[a] = b;
    c.refs[b] = c.refs[a];
    c.refs[a] = 0;
  }
  if (tid == 0) {
    w.moves[0] = movers;
    used[0] = L;
  }
}

// 16 KB pieces of the moving pages, and the tables' new page numbers.
__global__ void __launch_bounds__(256) compact_move_kernel(const CacheView c, const int* __restrict__ used, CompactWork w) {
  cudaGridDependencySynchronize();  // launched while the plan still runs
  const int moves = w.moves[0], L = used[0];
  if (moves == 0) return;
  constexpr int U = 4;
  const long long vecs = static_cast<long long>(c.page) * c.row_vecs;  // of one page of K (or V)
  const int pieces = static_cast<int>((vecs + 256 * U - 1) / (256 * U));
  const long long total = static_cast<long long>(moves) * 2 * pieces;
  for (long long x = blockIdx.x; x < total; x += gridDim.x) {
    const long long m = x / (2 * pieces);
    const int rest = static_cast<int>(x - m * 2 * pieces), piece = rest >> 1;
    uint4* pool = reinterpret_cast<uint4*>(rest & 1 ? c.v : c.k);
    const int from = w.from[m], to = w.to[m];
    const uint4* src = pool + from * vecs;
    uint4* dst = pool + to * vecs;
    const long long b = static_cast<long long>(piece) * 256 * U + threadIdx.x;
    uint4 r[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (b + 256 * u < vecs) r[u] = src[b + 256 * u];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (b + 256 * u < vecs) dst[b + 256 * u] = r[u];
    if (rest == 0 && c.mass != nullptr && threadIdx.x < c.page)
      c.mass[static_cast<long long>(to) * c.page + threadIdx.x] = c.mass[static_cast<long long>(from) * c.page + threadIdx.x];
  }
  const long long entries = static_cast<long long>(c.slots) * c.max_pages;
  for (long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; i < entries; i += static_cast<long long>(gridDim.x) * 256) {
    const int p = c.table[i];
    if (p >= L && p < c.pages) c.table[i] = w.map[p];
  }
}

// ---------------------------------------------------------------- host

// Launches a kernel that may start before the one in front of it on the stream has ended (it waits itself).
template <typename... P, typename... A>
cudaError_t launch_behind(void (*kernel)(P...), unsigned grid, cudaStream_t st, const A&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

int element_size(int dtype) { return dtype == VB200_F32 ? 4 : 2; }

int view_of(const vb200_paged_cache* cache, int dtype, CacheView& c) {
  VB200_REQUIRE(cache != nullptr, "cache: null handle");
  VB200_REQUIRE(dtype == VB200_BF16 || dtype == VB200_F16 || dtype == VB200_F32, "cache: unsupported dtype code %d", dtype);
  VB200_REQUIRE(cache->k && cache->v && cache->table && cache->length && cache->references, "cache: null pointer in the handle");
  VB200_REQUIRE(cache->page_size == 16 || cache->page_size == 32 || cache->page_size == 64 || cache->page_size == 128,
                "cache: pages of 16, 32, 64 or 128 tokens (got %lld)", (long long)cache->page_size);
  VB200_REQUIRE(cache->pages >= 1 && cache->pages < (1ll << 30) && cache->slots >= 1 && cache->slots < (1ll << 30) &&
                    cache->max_pages >= 1 && cache->max_pages * cache->page_size < (1ll << 31) && cache->kv_heads >= 1 &&
                    cache->kv_heads <= 1024,
                "cache: sizes out of range");
  VB200_REQUIRE(((reinterpret_cast<uintptr_t>(cache->k) | reinterpret_cast<uintptr_t>(cache->v)) & 15u) == 0,
                "cache: pools must be 16-byte aligned");
  c.k = static_cast<uint8_t*>(cache->k);
  c.v = static_cast<uint8_t*>(cache->v);
  c.mass = cache->log_mass;
  c.table = cache->table;
  c.length = cache->length;
  c.refs = cache->references;
  c.pages = static_cast<int>(cache->pages);
  c.page = static_cast<int>(cache->page_size);
  c.slots = static_cast<int>(cache->slots);
  c.max_pages = static_cast<int>(cache->max_pages);
  c.row_vecs = static_cast<int>(cache->kv_heads) * 64 * element_size(dtype) / 16;
  return VB200_OK;
}

}  // namespace

unsigned cache_error_word(int clear) {
  unsigned v = 0;
  cudaMemcpyFromSymbol(&v, g_cache_err, sizeof(v));
  if (clear) {
    const unsigned z = 0;
    cudaMemcpyToSymbol(g_cache_err, &z, sizeof(z));
  }
  return v;
}

}  // namespace vb200

using namespace vb200;

extern "C" size_t vb200_cache_append_workspace_size(int64_t n, int64_t slots, int64_t pages) {
  if (n < 0 || slots < 0 || pages < 0) return 0;
  return align_up(static_cast<size_t>(4 + 4 * n + slots + pages) * 4, 256);
}

extern "C" int vb200_cache_append(const vb200_paged_cache* cache, int dtype, const int32_t* sequence, const int32_t* offsets, int64_t n,
                                  const void* k, const void* v, const float* log_mass, int64_t tokens, const int64_t* k_strides,
                                  const int64_t* v_strides, void* workspace, size_t workspace_bytes, void* stream) {
  CacheView c;
  int rc = view_of(cache, dtype, c);
  if (rc != VB200_OK) return rc;
  VB200_REQUIRE(n >= 0 && n < (1ll << 24) && tokens >= 0 && tokens < (1ll << 31), "cache_append: sizes out of range");
  if (n == 0) return VB200_OK;
  VB200_REQUIRE(sequence && offsets && workspace && (tokens == 0 || (k && v && k_strides && v_strides)), "cache_append: null pointer argument");
  VB200_REQUIRE(log_mass == nullptr || c.mass != nullptr, "cache_append: the cache holds no log-masses");
  VB200_REQUIRE(workspace_bytes >= vb200_cache_append_workspace_size(n, cache->slots, cache->pages), "cache_append: workspace too small");
  const int es = element_size(dtype);
  if (tokens > 0) {
    VB200_REQUIRE(((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15u) == 0 && (tokens == 1 || ((k_strides[0] | v_strides[0]) * es) % 16 == 0) &&
                      (cache->kv_heads == 1 || ((k_strides[1] | v_strides[1]) * es) % 16 == 0),
                  "cache_append: rows must be 16-byte aligned");
  }
  if ((rc = check_sm100()) != VB200_OK) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  AppendWork w;
  int* p = static_cast<int*>(workspace);
  w.status = p;
  w.old_len = p + 4;
  w.copy_src = w.old_len + n;
  w.first = w.copy_src + n;
  w.start = w.first + n;
  w.claim = w.start + n;
  w.free_list = w.claim + c.slots;
  append_plan_kernel<<<1, kBook, 0, st>>>(c, sequence, offsets, static_cast<int>(n), static_cast<int>(tokens), w);
  VB200_CHECK_LAUNCH("append_plan_kernel");
  const long long rows = tokens + n * c.page;
  VB200_REQUIRE((rows + 7) / 8 < (1ll << 31), "cache_append: too many rows");
  const int64_t zero[2] = {0, 0};
  const int64_t *ks = tokens > 0 ? k_strides : zero, *vs = tokens > 0 ? v_strides : zero;
  VB200_CHECK_CUDA(launch_behind(append_write_kernel, static_cast<unsigned>((rows + 7) / 8), st, c, sequence, offsets, static_cast<int>(n),
                                 static_cast<int>(tokens), static_cast<const uint8_t*>(k), static_cast<const uint8_t*>(v),
                                 static_cast<long long>(ks[0] * es), static_cast<long long>(ks[1] * es), static_cast<long long>(vs[0] * es),
                                 static_cast<long long>(vs[1] * es), 64 * es / 16, log_mass, w),
                   "append_write_kernel");
  VB200_CHECK_LAUNCH("append_write_kernel");
  return VB200_OK;
}

extern "C" int vb200_cache_free(const vb200_paged_cache* cache, int dtype, const int32_t* sequence, int64_t n, void* stream) {
  CacheView c;
  int rc = view_of(cache, dtype, c);
  if (rc != VB200_OK) return rc;
  VB200_REQUIRE(n >= 0 && n < (1ll << 24), "cache_free: sizes out of range");
  if (n == 0) return VB200_OK;
  VB200_REQUIRE(sequence != nullptr, "cache_free: null pointer argument");
  if ((rc = check_sm100()) != VB200_OK) return rc;
  free_kernel<<<static_cast<unsigned>(n), 256, 0, static_cast<cudaStream_t>(stream)>>>(c, sequence);
  VB200_CHECK_LAUNCH("free_kernel");
  return VB200_OK;
}

extern "C" size_t vb200_cache_fork_workspace_size(int64_t n, int64_t slots, int64_t max_pages) {
  if (n < 0 || slots < 0 || max_pages < 0) return 0;
  return align_up(static_cast<size_t>(slots + n * (max_pages + 1)) * 4, 256);
}

extern "C" int vb200_cache_fork(const vb200_paged_cache* cache, int dtype, const int32_t* source, const int32_t* target, int64_t n,
                                void* workspace, size_t workspace_bytes, void* stream) {
  CacheView c;
  int rc = view_of(cache, dtype, c);
  if (rc != VB200_OK) return rc;
  VB200_REQUIRE(n >= 0 && n < (1ll << 24), "cache_fork: sizes out of range");
  if (n == 0) return VB200_OK;
  VB200_REQUIRE(source && target && workspace, "cache_fork: null pointer argument");
  VB200_REQUIRE(workspace_bytes >= vb200_cache_fork_workspace_size(n, cache->slots, cache->max_pages), "cache_fork: workspace too small");
  if ((rc = check_sm100()) != VB200_OK) return rc;
  int* claim = static_cast<int*>(workspace);
  int* snap = claim + c.slots;
  int* len = snap + n * c.max_pages;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(kForkCtas);
  cfg.blockDim = dim3(kBook);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = kForkCtas;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  VB200_CHECK_CUDA(cudaLaunchKernelEx(&cfg, fork_kernel, c, source, target, static_cast<int>(n), claim, snap, len), "fork_kernel");
  VB200_CHECK_LAUNCH("fork_kernel");
  return VB200_OK;
}

extern "C" size_t vb200_cache_compact_workspace_size(int64_t pages) {
  return pages < 0 ? 0 : align_up(static_cast<size_t>(4 + 3 * pages) * 4, 256);
}

extern "C" int vb200_cache_compact(const vb200_paged_cache* cache, int dtype, int32_t* used, void* workspace, size_t workspace_bytes,
                                   void* stream) {
  CacheView c;
  int rc = view_of(cache, dtype, c);
  if (rc != VB200_OK) return rc;
  VB200_REQUIRE(used && workspace, "cache_compact: null pointer argument");
  VB200_REQUIRE(workspace_bytes >= vb200_cache_compact_workspace_size(cache->pages), "cache_compact: workspace too small");
  if ((rc = check_sm100()) != VB200_OK) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  CompactWork w;
  int* p = static_cast<int*>(workspace);
  w.moves = p;
  w.from = p + 4;
  w.to = w.from + c.pages;
  w.map = w.to + c.pages;
  compact_plan_kernel<<<1, kBook, 0, st>>>(c, used, w);
  VB200_CHECK_LAUNCH("compact_plan_kernel");
  // eight CTAs of 256 threads fill an SM; no more than there can be pieces
  const long long most = static_cast<long long>(c.pages) * 2 * ((static_cast<long long>(c.page) * c.row_vecs + 1023) / 1024);
  const unsigned grid = static_cast<unsigned>(most < 148 * 8 ? most : 148 * 8);
  VB200_CHECK_CUDA(launch_behind(compact_move_kernel, grid, st, c, static_cast<const int*>(used), w), "compact_move_kernel");
  VB200_CHECK_LAUNCH("compact_move_kernel");
  return VB200_OK;
}
