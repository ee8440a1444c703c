// The few-row form of the head's cross entropy (xent_small.cu).
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "../../include/mamba3_b200.h"

namespace m3b {

constexpr int kSmallXentRows = 8;

size_t small_xent_saved(const m3b_linear_xent_args* a);
// Workspace bytes, and with `run` the launches, of either direction.
int small_xent_fwd(const m3b_linear_xent_args* a, void* workspace, size_t* need, bool run, cudaStream_t st);
int small_xent_bwd(const m3b_linear_xent_args* a, void* workspace, size_t* need, bool run, cudaStream_t st);

}  // namespace m3b
