// Cross entropy of the language-model head for a few rows (at most kSmallXentRows): matrix-vector kernels.
//
//   z = h W^T, the maximum and sum of each block's columns       logits_rows_kernel
//   lse, the losses and their sum                                loss_rows_kernel
//   dz = w (exp(z - lse) - onehot);  dW = dz^T h;  dh's shares   grads_rows_kernel
//   dh                                                           dhidden_rows_kernel
//
// Bound by the weight's bytes: read once forward, once backward, and written once as dW.  With so few
// rows the logits are small beside it (4 bytes a row and column, against the weight's row), so they are kept
// and never made twice.  fp32 multiply-adds on CUDA cores from the operands as they are: 8 rows of 1408 x
// 21251 are 240 M of them a product, 7 us, beside 120 MB, 18 us, in fp32, where the tensor cores' six plane
// products of padded rows and the planes themselves cost far more.  Every sum has a fixed order.
// Measured, forward and backward: those 8 fp32 rows 143 us (the tensor-core form 583), of them 45 the logits
// and 51 the gradients (4.7 TB/s); 8 rows of 2048 x 50257 bf16 244 us, 81 and 147 (2.8 TB/s: eight products
// of every 16-bit weight and their conversions, 128 registers a thread); 1 row of 768 x 32000 bf16 is bound
// by the host's calls (140 us; on the device 9, 7, 30).
#include "xent_small.h"

#include <float.h>

#include "carve.h"
#include "common.cuh"
#include "launch.h"

namespace m3b {

namespace {

constexpr int kWarps = 4;        // of the logits' and gradients' blocks
constexpr int kRowsWarp = 4;     // weight rows of a warp: their loads are in flight together
constexpr int kRun = 128;        // weight rows whose dz are made at once
constexpr int kSliceStep = 32;   // weight rows of a block: a multiple of this
constexpr int kAhead = 8;        // of them, rows loaded ahead
constexpr int kGroups = 16;      // dh: groups of shares summed side by side
constexpr float kToLog2 = 1.4426950408889634f;

struct SmallXent {
  int T, D, V, reduction;
  int64_t h_stride, ignore;
  const void *h, *w;
  const int64_t* target;
  float* loss;
  const float* dloss;
  void *dh, *dw;
  int* err;
  // saved, kept rows in order
  float* hs;     // [kept][D]
  float* z;      // [kept][V]
  float2* stat;  // [kept] maximum, and log of the sum of exp(z - maximum)
  int* row;      // [kept]
  int* tgt;      // [kept]; -2 out of range
  int* pos;      // [T]: place among the kept, -1 ignored
  int* count;
  // workspace
  float2* part;  // [block][M] maximum and sum
  int parts;
  float* share;  // [slice][M][D] of dh
  int slices, slice_rows;
  int vec;       // rows start on, and are, whole vectors
};

// Rows of a kernel's form: 1, 2, 4 or 8.
int form_of(int64_t T) { return T <= 1 ? 1 : T <= 2 ? 2 : T <= 4 ? 4 : 8; }

template <typename T>
constexpr int kVec = 16 / (int)sizeof(T);
template <typename T, int N>  // N values of a row as floats
__device__ __forceinline__ void load_row(const T* p, float (&v)[N]) {
  static_assert(N * sizeof(T) == 16 || N * sizeof(T) == 8, "vector loads");
  if constexpr (sizeof(T) == 4) {
    const float4 r = __ldg(reinterpret_cast<const float4*>(p));
    v[0] = r.x, v[1] = r.y, v[2] = r.z, v[3] = r.w;
  } else if constexpr (N == 8) {
    const uint4 r = __ldg(reinterpret_cast<const uint4*>(p));
    const T* x = reinterpret_cast<const T*>(&r);
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = io<T>::ld(x + e);
  } else {
    const uint2 r = __ldg(reinterpret_cast<const uint2*>(p));
    const T* x = reinterpret_cast<const T*>(&r);
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = io<T>::ld(x + e);
  }
}
template <typename T>
__device__ __forceinline__ void store_row4(T* p, const float (&v)[4]) {
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
    alignas(8) T x[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) io<T>::st(x + e, v[e]);
    *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(x);
  }
}

// Bit t: row t is kept.  For whole warps.
__device__ __forceinline__ unsigned kept_rows(const SmallXent& p, int lane) {
  const int64_t t = lane < p.T ? p.target[lane] : p.ignore;
  return __ballot_sync(0xffffffffu, t != p.ignore);
}
__device__ __forceinline__ int nth_row(unsigned kept, int m) {
  for (; m > 0; --m) kept &= kept - 1;
  return __ffs(kept) - 1;
}

// (maximum, sum of exp(z - maximum)) of two sets of columns; the least maximum is -FLT_MAX, so that
// a set of -infinities has a sum of 0.
__device__ __forceinline__ float2 join(float2 a, float2 b) {
  const float top = fmaxf(a.x, b.x);
  return make_float2(top, a.y * exp2f((a.x - top) * kToLog2) + b.y * exp2f((b.x - top) * kToLog2));
}

template <typename T, int M>
__global__ void __launch_bounds__(32 * kWarps, 4) logits_rows_kernel(SmallXent p) {
  __shared__ float2 stat[kWarps][M];
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const unsigned kept = kept_rows(p, lane);
  const int n = __popc(kept);
  if (n == 0) return;
  const T* x[M];
#pragma unroll
  for (int m = 0; m < M; ++m)
    x[m] = static_cast<const T*>(p.h) + (int64_t)nth_row(kept, m < n ? m : 0) * p.h_stride;
  // the kept rows for the backward pass
  const int64_t at = (int64_t)blockIdx.x * (32 * kWarps) + threadIdx.x, all = (int64_t)gridDim.x * (32 * kWarps);
#pragma unroll
  for (int m = 0; m < M; ++m)
    if (m < n)
      for (int64_t c = at; c < p.D; c += all) p.hs[(int64_t)m * p.D + c] = io<T>::ld(x[m] + c);

  const int64_t v0 = ((int64_t)blockIdx.x * kWarps + warp) * kRowsWarp;
  const T* w[kRowsWarp];
#pragma unroll
  for (int j = 0; j < kRowsWarp; ++j)
    w[j] = static_cast<const T*>(p.w) + (v0 + j < p.V ? v0 + j : p.V - 1) * p.D;
  float a[kRowsWarp * M];
#pragma unroll
  for (int i = 0; i < kRowsWarp * M; ++i) a[i] = 0.f;
  constexpr int N = kVec<T>;
  if (p.vec) {
#pragma unroll 2
    for (int c = lane * N; c < p.D; c += 32 * N) {
      float wv[kRowsWarp][N];
#pragma unroll
      for (int j = 0; j < kRowsWarp; ++j) load_row(w[j] + c, wv[j]);
#pragma unroll
      for (int m = 0; m < M; ++m) {
        float xv[N];
        load_row(x[m] + c, xv);
#pragma unroll
        for (int j = 0; j < kRowsWarp; ++j)
#pragma unroll
          for (int e = 0; e < N; ++e) a[kRowsWarp * m + j] = fmaf(xv[e], wv[j][e], a[kRowsWarp * m + j]);
      }
    }
  } else {
    for (int c = lane; c < p.D; c += 32)
#pragma unroll
      for (int m = 0; m < M; ++m) {
        const float xv = io<T>::ld(x[m] + c);
#pragma unroll
        for (int j = 0; j < kRowsWarp; ++j) a[kRowsWarp * m + j] = fmaf(xv, io<T>::ld(w[j] + c), a[kRowsWarp * m + j]);
      }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < kRowsWarp * M; ++i) a[i] += __shfl_xor_sync(0xffffffffu, a[i], o);
  // lane kRowsWarp m + j has row m's logit of column v0 + j
  const int m = lane / kRowsWarp, j = lane % kRowsWarp;
  float mine = 0.f;
#pragma unroll
  for (int i = 0; i < kRowsWarp * M; ++i) mine = lane == i ? a[i] : mine;
  const bool live = m < n && m < M && v0 + j < p.V;
  if (live) p.z[(int64_t)m * p.V + v0 + j] = mine;
  float top = live ? fmaxf(mine, -FLT_MAX) : -FLT_MAX;
#pragma unroll
  for (int o = 1; o < kRowsWarp; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  float sum = live ? exp2f((mine - top) * kToLog2) : 0.f;
#pragma unroll
  for (int o = 1; o < kRowsWarp; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (j == 0 && m < M) stat[warp][m] = make_float2(top, sum);
  __syncthreads();
  if (threadIdx.x < M) {
    float2 s = stat[0][threadIdx.x];
#pragma unroll
    for (int k = 1; k < kWarps; ++k) s = join(s, stat[k][threadIdx.x]);
    p.part[(int64_t)blockIdx.x * M + threadIdx.x] = s;
  }
}

// One block: warp w takes every (32 / M)-th run of 32 parts of row w % M.
template <int M>
__global__ void __launch_bounds__(1024) loss_rows_kernel(SmallXent p) {
  __shared__ float2 stat[32];
  __shared__ float row_loss[M];
  pdl_wait_primary();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const unsigned kept = kept_rows(p, lane);
  const int n = __popc(kept);
  constexpr int kSets = 32 / M;
  float2 s = make_float2(-FLT_MAX, 0.f);
  if (warp % M < n) {
#pragma unroll 4
    for (int64_t b = (warp / M) * 32 + lane; b < p.parts; b += 32 * kSets) s = join(s, __ldcg(p.part + b * M + warp % M));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    s = join(s, make_float2(__shfl_xor_sync(0xffffffffu, s.x, o), __shfl_xor_sync(0xffffffffu, s.y, o)));
  if (lane == 0) stat[warp] = s;
  __syncthreads();
  const int m = threadIdx.x;
  if (m < n) {
    s = stat[m];
    for (int k = 1; k < kSets; ++k) s = join(s, stat[k * M + m]);
    const int r = nth_row(kept, m);
    const int64_t t = p.target[r];
    const bool ok = t >= 0 && t < p.V;
    if (!ok) record_error(p.err, M3B_ERR_INVALID_ARG);
    const float nan = __int_as_float(0x7fffffff), ln = logf(s.y);
    const float l = ok ? (s.x - __ldcg(p.z + (int64_t)m * p.V + t)) + ln : nan;
    p.stat[m] = make_float2(s.x, ok ? ln : nan);
    p.row[m] = r;
    p.tgt[m] = ok ? (int)t : -2;
    row_loss[m] = l;
    if (p.reduction == 0) p.loss[r] = l;
  }
  if (m < p.T) {
    const bool k = kept >> m & 1;
    p.pos[m] = k ? __popc(kept & ((1u << m) - 1)) : -1;
    if (!k && p.reduction == 0) p.loss[m] = 0.f;
  }
  if (m == 0) *p.count = n;
  __syncthreads();
  if (m == 0 && p.reduction != 0) {
    double x = 0.0;
    for (int k = 0; k < n; ++k) x += (double)row_loss[k];
    *p.loss = (float)(p.reduction == 1 ? x / (double)n : x);
  }
}

// A thread owns four columns of d_model: its part of the kept rows and of dh stay in registers while the
// block walks its slice of the vocabulary, kRun rows' dz at a time in shared memory.
template <typename T, int M>
__global__ void __launch_bounds__(32 * kWarps, 4) grads_rows_kernel(SmallXent p) {
  __shared__ alignas(16) float dz[kRun][M];
  pdl_launch_dependents();
  const int tid = threadIdx.x, n = *p.count;
  const int64_t c0 = ((int64_t)blockIdx.x * (32 * kWarps) + tid) * 4;
  const bool in = c0 < p.D;
  float2 h[M][2], acc[M][2];  // pairs: packed fp32 arithmetic halves the multiply-adds' instructions
  auto kept_at = [&](int m, int e) { return m < n && c0 + e < p.D ? p.hs[(int64_t)m * p.D + c0 + e] : 0.f; };
#pragma unroll
  for (int m = 0; m < M; ++m)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      h[m][e] = make_float2(kept_at(m, 2 * e), kept_at(m, 2 * e + 1));
      acc[m][e] = make_float2(0.f, 0.f);
    }
  const T* w = static_cast<const T*>(p.w);
  T* dw = static_cast<T*>(p.dw);
  const int64_t begin = (int64_t)blockIdx.y * p.slice_rows;
  const int64_t end = begin + p.slice_rows < p.V ? begin + p.slice_rows : p.V;
  for (int64_t r0 = begin; r0 < end; r0 += kRun) {
    const int rows = end - r0 < kRun ? (int)(end - r0) : kRun;
    __syncthreads();
    for (int i = tid; i < M * kRun; i += 32 * kWarps) {
      const int m = i / kRun, r = i % kRun;
      float x = 0.f;
      if (m < n && r < rows) {
        const float weight = p.reduction == 0 ? p.dloss[p.row[m]] : p.reduction == 1 ? *p.dloss / (float)n : *p.dloss;
        const float2 st = p.stat[m];  // apart: the maximum would cost their sum its last bits
        x = exp2f(((p.z[(int64_t)m * p.V + r0 + r] - st.x) - st.y) * kToLog2);
        x = weight * (p.tgt[m] == r0 + r ? x - 1.f : x);
      }
      dz[r][m] = x;
    }
    __syncthreads();
    if (!in) continue;
    for (int k = 0; k < rows; k += kAhead) {
      float wv[kAhead][4];
      if (p.dh) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          const T* src = w + (r0 + (k + i < rows ? k + i : rows - 1)) * p.D + c0;
          if (p.vec) {
            load_row(src, wv[i]);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) wv[i][e] = c0 + e < p.D ? io<T>::ld(src + e) : 0.f;
          }
        }
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        if (k + i >= rows) break;
        float z[M];
#pragma unroll
        for (int m = 0; m < M; ++m) z[m] = dz[k + i][m];
        if (p.dh) {
#pragma unroll
          for (int m = 0; m < M; ++m)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              acc[m][e] = fma2(make_float2(z[m], z[m]), make_float2(wv[i][2 * e], wv[i][2 * e + 1]), acc[m][e]);
        }
        if (p.dw) {
          float2 q[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
          for (int m = 0; m < M; ++m)
#pragma unroll
            for (int e = 0; e < 2; ++e) q[e] = fma2(make_float2(z[m], z[m]), h[m][e], q[e]);
          const float g[4] = {q[0].x, q[0].y, q[1].x, q[1].y};
          T* dst = dw + (r0 + k + i) * p.D + c0;
          if (p.vec) {
            store_row4(dst, g);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (c0 + e < p.D) io<T>::st(dst + e, g[e]);
          }
        }
      }
    }
  }
  if (!p.dh || !in) return;
#pragma unroll
  for (int m = 0; m < M; ++m)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (m < n && c0 + e < p.D)
        p.share[((int64_t)blockIdx.y * M + m) * p.D + c0 + e] = e & 1 ? acc[m][e / 2].y : acc[m][e / 2].x;
}

// 32 columns of one row per block: the slices' shares, kGroups sums side by side.
template <typename T>
__global__ void __launch_bounds__(32 * kGroups) dhidden_rows_kernel(SmallXent p, int M) {
  __shared__ float sum[kGroups][32];
  pdl_wait_primary();
  const int lane = threadIdx.x & 31, g = threadIdx.x >> 5, t = blockIdx.y, m = p.pos[t];
  const int64_t c = (int64_t)blockIdx.x * 32 + lane;
  float x = 0.f;
  if (m >= 0 && c < p.D) {
#pragma unroll 8
    for (int s = g; s < p.slices; s += kGroups) x += __ldcg(p.share + ((int64_t)s * M + m) * p.D + c);
  }
  sum[g][lane] = x;
  __syncthreads();
  if (g != 0 || c >= p.D) return;
#pragma unroll
  for (int k = 1; k < kGroups; ++k) x += sum[k][lane];
  io<T>::st(static_cast<T*>(p.dh) + (int64_t)t * p.D + c, x);
}

size_t carve_saved(const m3b_linear_xent_args* a, SmallXent* p) {
  Carve c(a->saved);
  p->T = (int)a->rows, p->D = a->d_model, p->V = a->vocab, p->reduction = a->reduction;
  p->hs = static_cast<float*>(c.take((size_t)a->rows * a->d_model * 4));
  p->z = static_cast<float*>(c.take((size_t)a->rows * a->vocab * 4));
  p->stat = static_cast<float2*>(c.take(kSmallXentRows * 8));
  p->row = static_cast<int*>(c.take(kSmallXentRows * 4));
  p->tgt = static_cast<int*>(c.take(kSmallXentRows * 4));
  p->pos = static_cast<int*>(c.take(kSmallXentRows * 4));
  p->count = static_cast<int*>(c.take(4));
  return c.at;
}

template <typename T, int M>
int run_fwd(const SmallXent& p, cudaStream_t st) {
  logits_rows_kernel<T, M><<<(unsigned)p.parts, 32 * kWarps, 0, st>>>(p);
  const int rc = check_launch("linear_xent");
  return rc != M3B_OK ? rc : launch_dependent(loss_rows_kernel<M>, dim3(1), 1024, st, p);
}
template <typename T, int M>
int run_bwd(const SmallXent& p, cudaStream_t st) {
  const unsigned blocks = (unsigned)((p.D + 128 * kWarps - 1) / (128 * kWarps));
  grads_rows_kernel<T, M><<<dim3(blocks, (unsigned)p.slices), 32 * kWarps, 0, st>>>(p);
  const int rc = check_launch("linear_xent_bwd");
  if (rc != M3B_OK || !p.dh) return rc;
  return launch_dependent(dhidden_rows_kernel<T>, dim3((unsigned)((p.D + 31) / 32), (unsigned)p.T), 32 * kGroups, st, p, M);
}
template <typename T>
int pick(const SmallXent& p, bool bwd, cudaStream_t st) {
  switch (form_of(p.T)) {
    case 1: return bwd ? run_bwd<T, 1>(p, st) : run_fwd<T, 1>(p, st);
    case 2: return bwd ? run_bwd<T, 2>(p, st) : run_fwd<T, 2>(p, st);
    case 4: return bwd ? run_bwd<T, 4>(p, st) : run_fwd<T, 4>(p, st);
    default: return bwd ? run_bwd<T, 8>(p, st) : run_fwd<T, 8>(p, st);
  }
}
int pick(const SmallXent& p, int dtype, bool bwd, cudaStream_t st) {
  if (dtype == M3B_BF16) return pick<__nv_bfloat16>(p, bwd, st);
  if (dtype == M3B_F16) return pick<__half>(p, bwd, st);
  return pick<float>(p, bwd, st);
}

}  // namespace

size_t small_xent_saved(const m3b_linear_xent_args* a) {
  SmallXent p{};
  m3b_linear_xent_args b = *a;
  b.saved = nullptr;
  return carve_saved(&b, &p);
}

int small_xent_fwd(const m3b_linear_xent_args* a, void* workspace, size_t* need, bool run, cudaStream_t st) {
  SmallXent p{};
  carve_saved(a, &p);
  const int rows = kWarps * kRowsWarp, n = a->dtype == M3B_F32 ? 4 : 8;
  p.parts = (int)((p.V + (int64_t)rows - 1) / rows);
  *need = (size_t)p.parts * form_of(p.T) * sizeof(float2);
  if (!run) return M3B_OK;
  p.part = static_cast<float2*>(workspace);
  p.h_stride = a->hidden_stride, p.ignore = a->ignore_index;
  p.h = a->hidden, p.w = a->weight, p.target = a->target, p.loss = a->loss, p.err = a->err;
  p.vec = p.D % n == 0 && p.h_stride % n == 0 && aligned16(p.h) && aligned16(p.w);
  return pick(p, a->dtype, false, st);
}

int small_xent_bwd(const m3b_linear_xent_args* a, void* workspace, size_t* need, bool run, cudaStream_t st) {
  SmallXent p{};
  carve_saved(a, &p);
  // four blocks a SM: all resident
  const int64_t blocks = (p.D + 128 * kWarps - 1) / (128 * kWarps), want = (int64_t)num_sms() * 4 / blocks;
  const int64_t rows = (p.V + (want > 1 ? want : 1) - 1) / (want > 1 ? want : 1);
  p.slice_rows = (int)((rows + kSliceStep - 1) / kSliceStep * kSliceStep);
  p.slices = (int)((p.V + (int64_t)p.slice_rows - 1) / p.slice_rows);
  *need = a->dhidden ? (size_t)p.slices * form_of(p.T) * p.D * 4 : 4;
  if (!run) return M3B_OK;
  p.share = static_cast<float*>(workspace);
  p.w = a->weight, p.dloss = a->dloss, p.dh = a->dhidden, p.dw = a->dweight;
  p.vec = p.D % 4 == 0 && aligned16(p.w) && aligned16(p.dw);
  if (!p.dh && !p.dw) return M3B_OK;
  return pick(p, a->dtype, true, st);
}

}  // namespace m3b
