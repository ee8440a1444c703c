// The few-row form of the gated feed-forward block (ffn_small.cu).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace m3b {

constexpr int kSmallRows = 8;

struct SmallFfn {
  int M, D, F;
  int64_t x_stride, res_stride, ld_act;
  const void *x, *w_gate, *w_up, *w_down, *b_gate, *b_up, *b_down, *residual;
  void *act, *out;  // act in the activations' type, rows ld_act apart
  float scale;
  int vec;  // every row starts on 16 bytes and holds whole 16-byte vectors
};
int launch_small_ffn(const SmallFfn& p, int dtype, cudaStream_t st);

}  // namespace m3b
