// The few-row form of the head's cross entropy (xent_small.cu).
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "../../include/mamba3_b200.h"

namespace m3b {

// A lane holds the sums of four weight rows and every hidden row (32 at 8 rows), which is what bounds the form.
// 21251 x 1408 forward and backward, captured, 8 rows here and 9 in the tensor-core form: 112 - 124 and 134 - 140 us in bf16,
// 104 - 127 and 121 - 127 in fp16, 111 - 144 and 652 in fp32 (the planes of the weight, twice).
constexpr int kSmallXentRows = 8;

size_t small_xent_saved(const m3b_linear_xent_args* a);
// Workspace bytes, and with `run` the launches, of either direction.
int small_xent_fwd(const m3b_linear_xent_args* a, void* workspace, size_t* need, bool run, cudaStream_t st);
int small_xent_bwd(const m3b_linear_xent_args* a, void* workspace, size_t* need, bool run, cudaStream_t st);

}  // namespace m3b
