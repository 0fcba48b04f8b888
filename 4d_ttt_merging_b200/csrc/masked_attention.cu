// Entry points of the masked and the paged attention: argument checks and the choice of kernel.
#include <cudaTypedefs.h>

#include <atomic>
#include <cmath>
#include <initializer_list>
#include <mutex>

#include "attention_view.cuh"
#include "host_common.h"
#include "masked_host.h"

namespace vb200 {
namespace {

static __device__ unsigned g_masked_err;

// What does not change about a device: that it is an sm_100 one, its SMs, the address of its error word.
struct DeviceFacts {
  int sms;
  unsigned* err;
};

int device_facts(DeviceFacts& f) {
  static DeviceFacts known[64];
  static std::atomic<bool> ready[64];
  int dev = 0;
  VB200_CHECK_CUDA(cudaGetDevice(&dev), "cudaGetDevice");
  if (dev >= 0 && dev < 64 && ready[dev].load(std::memory_order_acquire)) {
    f = known[dev];
    return VB200_OK;
  }
  const int rc = check_sm100();
  if (rc != VB200_OK) return rc;
  VB200_CHECK_CUDA(cudaDeviceGetAttribute(&f.sms, cudaDevAttrMultiProcessorCount, dev), "cudaDeviceGetAttribute");
  VB200_CHECK_CUDA(cudaGetSymbolAddress(reinterpret_cast<void**>(&f.err), g_masked_err), "cudaGetSymbolAddress(g_masked_err)");
  if (dev >= 0 && dev < 64) {
    static std::mutex write;
    std::lock_guard<std::mutex> lock(write);
    known[dev] = f;
    ready[dev].store(true, std::memory_order_release);
  }
  return VB200_OK;
}

int fill_mods(const vb200_score_mods* m, AttnView& a) {
  VB200_REQUIRE(std::isfinite(m->scale) && m->scale > 0.f, "attention: scale must be positive and finite");
  VB200_REQUIRE(m->softcap >= 0.f && std::isfinite(m->softcap), "attention: softcap must be 0 (none) or positive and finite");
  a.range = m->key_range;
  a.range_sb = m->key_range_sb;
  a.slope = m->slope;
  if (m->softcap > 0.f) {
    a.scale = m->scale / m->softcap;
    a.cap = m->softcap * kLog2E;
    VB200_REQUIRE(std::isfinite(a.scale) && std::isfinite(a.cap), "attention: softcap out of range");
  } else {
    a.scale = m->scale * kLog2E;
    a.cap = 0.f;
    VB200_REQUIRE(std::isfinite(a.scale), "attention: scale out of range");
  }
  return VB200_OK;
}

// 16-byte rows: base address and the strides of dimensions longer than one
bool aligned(const void* p, const int64_t* s, std::initializer_list<int64_t> sizes, int es) {
  bool ok = (reinterpret_cast<uintptr_t>(p) & 15u) == 0;
  int i = 0;
  for (int64_t n : sizes) {
    ok = ok && (n <= 1 || (s[i] * es) % 16 == 0);
    ++i;
  }
  return ok;
}

// fp32; at most 16 (row, head) pairs per key head, since a tile of the other kernel has 128 rows of one head, so below that
// its tiles are nearly empty and the heads of a group read their keys one by one; or at most 32 blocks of 16 pairs in
// all, where either kernel leaves SMs idle and the lighter one ends sooner (17 rows, 16 heads, 1041 keys: 12 against 18 us,
// 16,464 keys: 29 against 35; 33 rows and 4116 keys, beyond the rule: 27 against 20).
//
// The rule sees the mean of a paged call's rows (the host does not know the chunks), so a call that mixes long chunks with single
// tokens takes one kernel for all: 32 streams of 500 to 9000 keys, 16 heads, take 121 us with a token each; with one chunk
// of 300 rows among them 213 (by itself 27), with one of 1041 rows 190 (45).  Such calls are better made apart.
bool few_rows(int dtype, int64_t rows, int64_t group, int64_t heads_and_sequences) {
  return dtype == VB200_F32 || rows * group <= 16 || (rows * group + 15) / 16 * heads_and_sequences <= 32;
}

// The tile kernel adds bias and distance inside the QK product, where what it can hold of them shrinks with the scale
// (attention_masked_tc.cu); below these scales the few-row kernel, which adds them in fp32, takes the call whatever its rows.
bool bias_beyond_product(int dtype, const vb200_score_mods* m, bool bias) {
  return m->softcap == 0.f && (bias || m->slope != nullptr) && m->scale < (dtype == VB200_F16 ? 0x1p-8f : 0x1p-76f);
}

}  // namespace

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

int pool_map(CUtensorMap* map, const void* base, int dtype, const AttnView& a, int box) {
  // (channel, head, slot, page): contiguous pools
  const int page = 1 << a.page_shift;
  const uint64_t dims[4] = {kHeadDim, static_cast<uint64_t>(a.Hkv), static_cast<uint64_t>(page), static_cast<uint64_t>(a.pages)};
  const uint64_t row = static_cast<uint64_t>(a.Hkv) * kHeadDim * 2;
  const uint64_t str[3] = {kHeadDim * 2, row, row * page};
  const uint32_t b[4] = {kHeadDim, 1, static_cast<uint32_t>(page < box ? page : box), 1};
  return encode_tiled_map(map, dtype == VB200_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, base, dims,
                          str, b, CU_TENSOR_MAP_SWIZZLE_128B);
}

int sm_count_of_device() {
  DeviceFacts f;
  return device_facts(f) == VB200_OK ? f.sms : 0;
}

unsigned masked_error_word(int clear) {
  unsigned v = 0;
  cudaMemcpyFromSymbol(&v, g_masked_err, sizeof(v));
  if (clear) {
    const unsigned z = 0;
    cudaMemcpyToSymbol(g_masked_err, &z, sizeof(z));
  }
  return v;
}

}  // namespace vb200

using namespace vb200;

extern "C" size_t vb200_masked_attention_workspace_size(int dtype, int64_t B, int64_t H, int64_t Hkv, int64_t Nq, int64_t Nk) {
  if (B < 1 || H < 1 || Hkv < 1 || Nq < 1 || Nk < 1 || few_rows(dtype, Nq, H / Hkv, Hkv * B)) return 0;
  return tile_attention_workspace(false, Nq, B, H, Nk);
}

extern "C" size_t vb200_paged_attention_workspace_size(int dtype, int64_t rows, int64_t H, const vb200_paged_cache* cache, int64_t n) {
  if (cache == nullptr || rows < 1 || H < 1 || n < 1 || cache->kv_heads < 1 || cache->max_pages < 1 || cache->page_size < 1 ||
      few_rows(dtype, (rows + n - 1) / n, H / cache->kv_heads, cache->kv_heads * n))
    return 0;
  return tile_attention_workspace(true, rows, n, H, cache->max_pages * cache->page_size);
}

extern "C" int vb200_masked_attention(int dtype, const void* q, const void* k, const void* v, void* out, int64_t B, int64_t H,
                                      int64_t Hkv, int64_t Nq, int64_t Nk, int64_t D, const int64_t* qs, const int64_t* ks,
                                      const int64_t* vs, const int64_t* os, const vb200_score_mods* mods, void* workspace,
                                      size_t workspace_bytes, void* stream) {
  VB200_REQUIRE(dtype == VB200_BF16 || dtype == VB200_F16 || dtype == VB200_F32, "masked_attention: unsupported dtype code %d", dtype);
  VB200_REQUIRE(D == kHeadDim, "masked_attention supports head_dim=64 only (got %lld)", (long long)D);
  VB200_REQUIRE(B >= 1 && H >= 1 && Hkv >= 1 && H % Hkv == 0 && Nq >= 0 && Nk >= 1,
                "masked_attention: invalid sizes B=%lld H=%lld Hkv=%lld Nq=%lld Nk=%lld", (long long)B, (long long)H, (long long)Hkv,
                (long long)Nq, (long long)Nk);
  VB200_REQUIRE(Nk < (1ll << 31) - 128 && B * H < 65536 && Nq * (H / Hkv) < (1ll << 31) - 256,
                "masked_attention: sizes exceed the kernels' index range");
  VB200_REQUIRE(mods != nullptr, "masked_attention: null mods");
  if (Nq == 0) return VB200_OK;
  VB200_REQUIRE(q && k && v && out && qs && ks && vs && os, "masked_attention: null pointer argument");
  const int es = dtype == VB200_F32 ? 4 : 2;
  VB200_REQUIRE(aligned(q, qs, {B, H, Nq}, es) && aligned(k, ks, {B, Hkv, Nk}, es) && aligned(v, vs, {B, Hkv, Nk}, es) &&
                    aligned(out, os, {B, H, Nq}, es),
                "masked_attention: rows must be 16-byte aligned");
  AttnView a{};
  int rc = fill_mods(mods, a);
  if (rc != VB200_OK) return rc;
  DeviceFacts facts;
  if ((rc = device_facts(facts)) != VB200_OK) return rc;
  a.err = facts.err;
  a.q = q, a.k = k, a.v = v, a.out = out;
  a.q_sb = qs[0], a.q_sh = qs[1], a.q_sn = qs[2];
  a.k_sb = ks[0], a.k_sh = ks[1], a.k_sn = ks[2];
  a.v_sb = vs[0], a.v_sh = vs[1], a.v_sn = vs[2];
  a.o_sb = os[0], a.o_sh = os[1], a.o_sn = os[2];
  a.B = static_cast<int>(B), a.H = static_cast<int>(H), a.Hkv = static_cast<int>(Hkv), a.group = static_cast<int>(H / Hkv);
  a.Nq = static_cast<int>(Nq), a.Nk = static_cast<int>(Nk);
  a.bias = mods->key_bias, a.bias_sb = mods->key_bias_sb;
  a.qpos = mods->q_position, a.qpos_sb = mods->q_position_sb;
  a.kpos = mods->k_position, a.kpos_sb = mods->k_position_sb;
  if (few_rows(dtype, Nq, a.group, Hkv * B) || bias_beyond_product(dtype, mods, a.bias != nullptr))
    return rows_attention(dtype, false, a, Nk, static_cast<cudaStream_t>(stream));
  return tile_attention(dtype, false, a, Nk, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}

extern "C" int vb200_paged_attention(int dtype, const void* q, void* out, int64_t rows, int64_t H, int64_t D, const int64_t* qs,
                                     const int64_t* os, const vb200_paged_cache* cache, const int32_t* sequence, const int32_t* offsets,
                                     int64_t n, int causal, const vb200_score_mods* mods, void* workspace, size_t workspace_bytes,
                                     void* stream) {
  VB200_REQUIRE(dtype == VB200_BF16 || dtype == VB200_F16 || dtype == VB200_F32, "paged_attention: unsupported dtype code %d", dtype);
  VB200_REQUIRE(D == kHeadDim, "paged_attention supports head_dim=64 only (got %lld)", (long long)D);
  VB200_REQUIRE(cache != nullptr && mods != nullptr, "paged_attention: null handle or mods");
  VB200_REQUIRE(cache->page_size == 16 || cache->page_size == 32 || cache->page_size == 64 || cache->page_size == 128,
                "paged_attention: pages of 16, 32, 64 or 128 tokens (got %lld)", (long long)cache->page_size);
  VB200_REQUIRE(H >= 1 && H < 65536 && cache->kv_heads >= 1 && H % cache->kv_heads == 0, "paged_attention: H=%lld is no multiple of %lld key heads",
                (long long)H, (long long)cache->kv_heads);
  VB200_REQUIRE(n >= 0 && n < (1ll << 24) && rows >= 0 && rows * (H / cache->kv_heads) < (1ll << 31) - 256 && cache->pages >= 1 &&
                    cache->pages < (1ll << 30) && cache->slots >= 1 && cache->slots < (1ll << 30) && cache->max_pages >= 1 &&
                    cache->max_pages * cache->page_size < (1ll << 31) - 128,
                "paged_attention: sizes exceed the kernels' index range");
  if (n == 0 || rows == 0) return VB200_OK;
  VB200_REQUIRE(q && out && qs && os && offsets && cache->k && cache->v && cache->table && cache->length, "paged_attention: null pointer argument");
  VB200_REQUIRE(sequence != nullptr || n <= cache->slots, "paged_attention: more sequences than slots");
  const int es = dtype == VB200_F32 ? 4 : 2;
  VB200_REQUIRE(aligned(q, qs, {H, rows}, es) && aligned(out, os, {H, rows}, es) && aligned(cache->k, nullptr, {}, es) &&
                    aligned(cache->v, nullptr, {}, es),
                "paged_attention: rows must be 16-byte aligned");
  AttnView a{};
  int rc = fill_mods(mods, a);
  if (rc != VB200_OK) return rc;
  DeviceFacts facts;
  if ((rc = device_facts(facts)) != VB200_OK) return rc;
  a.err = facts.err;
  a.q = q, a.k = cache->k, a.v = cache->v, a.out = out;
  a.q_sh = qs[0], a.q_sn = qs[1], a.o_sh = os[0], a.o_sn = os[1];
  a.Hkv = static_cast<int>(cache->kv_heads);
  a.k_sh = a.v_sh = kHeadDim;
  a.k_sn = a.v_sn = static_cast<long long>(a.Hkv) * kHeadDim;
  a.k_sb = a.v_sb = a.k_sn * cache->page_size;
  a.B = 1, a.H = static_cast<int>(H), a.group = static_cast<int>(H / cache->kv_heads);
  a.Nq = static_cast<int>(rows), a.Nk = 0;
  a.bias = cache->log_mass;
  a.table = cache->table, a.length = cache->length, a.sequence = sequence, a.offsets = offsets;
  a.table_stride = cache->max_pages;
  a.n_seq = static_cast<int>(n), a.slots = static_cast<int>(cache->slots), a.pages = static_cast<int>(cache->pages);
  a.page_shift = cache->page_size == 16 ? 4 : cache->page_size == 32 ? 5 : cache->page_size == 64 ? 6 : 7;
  a.max_pages = static_cast<int>(cache->max_pages), a.causal = causal;
  // What the splits over the keys are planned for: the host does not know the lengths, so a short stream in a table with room for
  // many keys is split like a long one.  Room for 65,536: 8 chunks of 300 rows over 1100 keys 43 -> 90 us, 1041 rows over 2701
  // 45 -> 64; decode, and a frame over 32,928 keys, as with a table that is just wide enough.
  const int64_t most = cache->max_pages * cache->page_size;
  if (few_rows(dtype, (rows + n - 1) / n, a.group, cache->kv_heads * n) || bias_beyond_product(dtype, mods, a.bias != nullptr))
    return rows_attention(dtype, true, a, most, static_cast<cudaStream_t>(stream));
  return tile_attention(dtype, true, a, most, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}
