// Host side shared by the masked and the paged attention: the two launchers behind their entry points.
#pragma once

#include <cuda_runtime.h>

namespace vb200 {

struct AttnView;

int sm_count_of_device();  // SMs of the current device, 0 when unknown

// The FMA-pipe kernel: any type, any number of rows; most_keys bounds the keys of a sequence.
int rows_attention(int dtype, bool paged, const AttnView& a, long long most_keys, cudaStream_t st);

// The tensor-core kernel: bf16 and fp16.
int tile_attention(int dtype, bool paged, const AttnView& a, long long most_keys, cudaStream_t st);

}  // namespace vb200
