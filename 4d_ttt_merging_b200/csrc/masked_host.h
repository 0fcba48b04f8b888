// Host side shared by the masked and the paged attention: the two launchers behind their entry points.
#pragma once

#include <cuda_runtime.h>

#include <cstddef>

namespace vb200 {

struct AttnView;

int sm_count_of_device();  // SMs of the current device, 0 when unknown

// The FMA-pipe kernel: any type, any number of rows; most_keys bounds the keys of a sequence.
int rows_attention(int dtype, bool paged, const AttnView& a, long long most_keys, cudaStream_t st);

// The tensor-core kernel: bf16 and fp16.  Without the workspace its last wave runs unsplit.
int tile_attention(int dtype, bool paged, const AttnView& a, long long most_keys, void* workspace, size_t workspace_bytes, cudaStream_t st);
size_t tile_attention_workspace(bool paged, long long rows, long long seqs, long long H, long long most_keys);

}  // namespace vb200
