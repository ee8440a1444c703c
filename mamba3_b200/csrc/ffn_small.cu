// Gated feed-forward block for a few rows (decoding): the two products as matrix-vector kernels.
//
//   act[m, f] = silu(x_m . Wg_f + bg_f) (x_m . Wu_f + bu_f)       glu_rows_kernel
//   out[m, d] = residual[m, d] + s (act_m . Wd_d + bd_d)          down_rows_kernel
//
// Bound by the weights' bytes (6 d_model d_ff of them in 16 bits), below that by latency: a warp owns
// whole weight rows, so sums stay in registers and shuffles, and its loads of them are in flight
// together.  The second kernel is a programmatic dependent of the first: it starts early and has its
// first eight loads of every row in registers before it waits for act.  fp32 multiply-adds on CUDA
// cores: with up to kSmallRows rows they stay below the time of the bytes (8 rows of 2048 x 5504:
// 270 M multiply-adds, 8 us, beside 67 MB, 10 us); more rows go to the tensor cores.
#include "ffn_small.h"

#include "common.cuh"
#include "launch.h"

namespace m3b {

namespace {

constexpr int kWarps = 4;

// 16 bytes of a row as floats.
template <typename T>
constexpr int kVec = 16 / (int)sizeof(T);
template <typename T>
__device__ __forceinline__ void widen(const uint4& w, float (&v)[kVec<T>]) {
  if constexpr (sizeof(T) == 4) {
    v[0] = __uint_as_float(w.x), v[1] = __uint_as_float(w.y), v[2] = __uint_as_float(w.z), v[3] = __uint_as_float(w.w);
  } else {
    const T* x = reinterpret_cast<const T*>(&w);
#pragma unroll
    for (int e = 0; e < kVec<T>; ++e) v[e] = io<T>::ld(x + e);
  }
}
template <typename T>
__device__ __forceinline__ uint4 load16(const T* p) {
  return __ldg(reinterpret_cast<const uint4*>(p));
}
template <int N>
__device__ __forceinline__ void warp_sums(float (&a)[N]) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) a[i] += __shfl_xor_sync(0xffffffffu, a[i], o);
}

// Two columns f of act per warp: four weight rows beside the rows of x.
template <typename T, int M>
__global__ void __launch_bounds__(32 * kWarps) glu_rows_kernel(SmallFfn p) {
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int f0 = (blockIdx.x * kWarps + (threadIdx.x >> 5)) * 2;
  if (f0 >= p.F) return;
  const int f1 = f0 + 1 < p.F ? f0 + 1 : f0;
  const T* x = static_cast<const T*>(p.x);
  const T* w[4] = {static_cast<const T*>(p.w_gate) + (int64_t)f0 * p.D, static_cast<const T*>(p.w_up) + (int64_t)f0 * p.D,
                   static_cast<const T*>(p.w_gate) + (int64_t)f1 * p.D, static_cast<const T*>(p.w_up) + (int64_t)f1 * p.D};
  float a[4 * M];
#pragma unroll
  for (int i = 0; i < 4 * M; ++i) a[i] = 0.f;
  constexpr int V = kVec<T>;
  if (p.vec) {
#pragma unroll 2
    for (int c = lane * V; c < p.D; c += 32 * V) {
      uint4 raw[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) raw[j] = load16(w[j] + c);
      float wv[4][V];
#pragma unroll
      for (int j = 0; j < 4; ++j) widen<T>(raw[j], wv[j]);
#pragma unroll
      for (int m = 0; m < M; ++m) {
        float xv[V];
        widen<T>(load16(x + (m < p.M ? m : 0) * p.x_stride + c), xv);
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int e = 0; e < V; ++e) a[4 * m + j] = fmaf(xv[e], wv[j][e], a[4 * m + j]);
      }
    }
  } else {
    for (int c = lane; c < p.D; c += 32)
#pragma unroll
      for (int m = 0; m < M; ++m) {
        const float xv = io<T>::ld(x + (m < p.M ? m : 0) * p.x_stride + c);
#pragma unroll
        for (int j = 0; j < 4; ++j) a[4 * m + j] = fmaf(xv, io<T>::ld(w[j] + c), a[4 * m + j]);
      }
  }
  warp_sums(a);
  T* act = static_cast<T*>(p.act);
#pragma unroll
  for (int m = 0; m < M; ++m)
#pragma unroll
    for (int j = 0; j < 2; ++j)
      if (lane == 2 * m + j && m < p.M && f0 + j < p.F) {
        float g = a[4 * m + 2 * j], u = a[4 * m + 2 * j + 1];
        if (p.b_gate) {
          g += io<T>::ld(static_cast<const T*>(p.b_gate) + f0 + j);
          u += io<T>::ld(static_cast<const T*>(p.b_up) + f0 + j);
        }
        io<T>::st(act + m * p.ld_act + f0 + j, g * sigmoid_fast(g) * u);
      }
}

// One output column d per warp.
template <typename T, int M>
__global__ void __launch_bounds__(32 * kWarps) down_rows_kernel(SmallFfn p) {
  constexpr int V = kVec<T>, kAhead = 8;  // 16-byte loads a lane: 2048 values of 16 bits, 1024 of 32
  const int lane = threadIdx.x & 31, d = blockIdx.x * kWarps + (threadIdx.x >> 5);
  const bool live = d < p.D;
  const T* w = static_cast<const T*>(p.w_down) + (int64_t)(live ? d : 0) * p.F;
  uint4 raw[kAhead];
  if (p.vec) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int c = (k * 32 + lane) * V;
      raw[k] = c < p.F ? load16(w + c) : make_uint4(0u, 0u, 0u, 0u);
    }
  }
  pdl_wait_primary();  // act is written by the kernel before
  if (!live) return;
  const T* act = static_cast<const T*>(p.act);
  float a[M];
#pragma unroll
  for (int m = 0; m < M; ++m) a[m] = 0.f;
  auto add = [&](int c, const uint4& r) {
    float wv[V];
    widen<T>(r, wv);
#pragma unroll
    for (int m = 0; m < M; ++m) {
      float xv[V];
      widen<T>(*reinterpret_cast<const uint4*>(act + (m < p.M ? m : 0) * p.ld_act + c), xv);
#pragma unroll
      for (int e = 0; e < V; ++e) a[m] = fmaf(xv[e], wv[e], a[m]);
    }
  };
  if (p.vec) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int c = (k * 32 + lane) * V;
      if (c < p.F) add(c, raw[k]);
    }
#pragma unroll 4
    for (int c = (kAhead * 32 + lane) * V; c < p.F; c += 32 * V) add(c, load16(w + c));
  } else {
    for (int c = lane; c < p.F; c += 32) {
      const float wv = io<T>::ld(w + c);
#pragma unroll
      for (int m = 0; m < M; ++m) a[m] = fmaf(io<T>::ld(act + (m < p.M ? m : 0) * p.ld_act + c), wv, a[m]);
    }
  }
  warp_sums(a);
#pragma unroll
  for (int m = 0; m < M; ++m)
    if (lane == m && m < p.M) {
      float y = a[m];
      if (p.b_down) y += io<T>::ld(static_cast<const T*>(p.b_down) + d);
      y *= p.scale;
      if (p.residual) y += io<T>::ld(static_cast<const T*>(p.residual) + m * p.res_stride + d);
      io<T>::st(static_cast<T*>(p.out) + (int64_t)m * p.D + d, y);
    }
}

template <typename T, int M>
int launch(const SmallFfn& p, cudaStream_t st) {
  glu_rows_kernel<T, M><<<(p.F + 2 * kWarps - 1) / (2 * kWarps), 32 * kWarps, 0, st>>>(p);
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3((p.D + kWarps - 1) / kWarps);
  cfg.blockDim = dim3(32 * kWarps);
  cfg.stream = st;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, down_rows_kernel<T, M>, p);
  if (e != cudaSuccess) return fail(M3B_ERR_CUDA, "gated_ffn: %s", cudaGetErrorString(e));
  return check_launch("gated_ffn");
}

template <typename T>
int pick(const SmallFfn& p, cudaStream_t st) {
  if (p.M <= 1) return launch<T, 1>(p, st);
  if (p.M <= 2) return launch<T, 2>(p, st);
  if (p.M <= 4) return launch<T, 4>(p, st);
  return launch<T, 8>(p, st);
}

}  // namespace

int launch_small_ffn(const SmallFfn& p, int dtype, cudaStream_t st) {
  if (dtype == M3B_BF16) return pick<__nv_bfloat16>(p, st);
  if (dtype == M3B_F16) return pick<__half>(p, st);
  return pick<float>(p, st);
}

}  // namespace m3b
