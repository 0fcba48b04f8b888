// Host side shared by the masked and the paged attention: the two launchers behind their entry points.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <cstddef>

namespace vb200 {

struct AttnView;

int sm_count_of_device();  // SMs of the current device, 0 when unknown

// TMA maps of 16-bit rows of 64 channels, 128-byte swizzle.  rows_map: (channel, row, head, batch) with strides in elements,
// `box` rows of one head at a time; pool_map: (channel, head, slot, page) of a contiguous pool, boxes of one head and at
// most `box` slots of a page.
int rows_map(CUtensorMap* map, const void* base, int dtype, long long n, long long heads, long long batch, long long sn, long long sh,
             long long sb, int box);
int pool_map(CUtensorMap* map, const void* base, int dtype, const AttnView& a, int box);

// The kernels for few rows (bf16, fp16: warp-level matrix instructions) and for fp32 (FMA pipe); they take any number of rows.
// most_keys bounds the keys of a sequence.
int rows_attention(int dtype, bool paged, const AttnView& a, long long most_keys, cudaStream_t st);

// The tensor-core kernel: bf16 and fp16.  Without the workspace its last wave runs unsplit.
int tile_attention(int dtype, bool paged, const AttnView& a, long long most_keys, void* workspace, size_t workspace_bytes, cudaStream_t st);
size_t tile_attention_workspace(bool paged, long long rows, long long seqs, long long H, long long most_keys);

}  // namespace vb200
