// Global gradient norm over many tensors and clipping (m3b_grad_clip).
//
//   norm = sqrt(sum_i sum |g_i|^2) or max |g|;  out_i = g_i min(1, max_norm / (norm + 1e-6))
//
// Two passes over the gradients, both bound by HBM: every tensor is cut into chunks of kChunk
// values, one block per chunk.  The first pass leaves one fp64 partial per chunk; every block of the
// second adds the partials in the same fixed order, so no atomics and no host round trip.  The
// tensors' descriptions travel in the kernel's parameters, kPerLaunch at a time, so the call copies
// nothing to the device and can be captured into a CUDA graph.
#include "common.cuh"
#include "launch.h"

namespace m3b {

namespace {

constexpr int kThreads = 256;
constexpr int kChunk = 8192;       // values per block: 32 a thread
constexpr int kPerLaunch = 96;     // tensors per launch: their table fits the 4 KB of kernel parameters

struct Table {
  const void* g[kPerLaunch];
  void* o[kPerLaunch];
  int64_t n[kPerLaunch];
  int32_t chunk0[kPerLaunch + 1];  // first chunk of each tensor within this launch
  uint8_t gdt[kPerLaunch], odt[kPerLaunch];
  int count;
};

struct ClipParams {
  double* part;      // one per chunk of all tensors
  int64_t base;      // chunks of the launches before this one
  int64_t chunks;    // of all tensors
  int norm_inf;
  float max_norm;
  float* norm;
};

__device__ __forceinline__ int tensor_of(const Table& t, int chunk) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.chunk0[mid] <= chunk) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ bool all16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// A NaN stays: fmax would drop it.
__device__ __forceinline__ double join(double a, double b, bool inf) { return inf ? (a > b || a != a ? a : b) : a + b; }

__device__ __forceinline__ double block_join(double x, bool inf) {
  __shared__ double sm[kThreads / 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x = join(x, __shfl_xor_sync(0xffffffffu, x, o), inf);
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = x;
  __syncthreads();
  x = sm[0];
#pragma unroll
  for (int k = 1; k < kThreads / 32; ++k) x = join(x, sm[k], inf);
  return x;
}

__global__ void __launch_bounds__(kThreads) norm_kernel(const __grid_constant__ Table t, const __grid_constant__ ClipParams p) {
  const int i = tensor_of(t, blockIdx.x);
  const int64_t at = (int64_t)(blockIdx.x - t.chunk0[i]) * kChunk;
  const int n = (int)(t.n[i] - at < kChunk ? t.n[i] - at : kChunk);
  const int dt = t.gdt[i];
  const bool vec = all16(t.g[i]);
  float s = 0.f;
  auto add = [&](float v) { s = p.norm_inf ? (fabsf(v) > s || v != v ? fabsf(v) : s) : fmaf(v, v, s); };
  for (int c = threadIdx.x * 8; c < n; c += kThreads * 8) {
    if (vec && c + 8 <= n) {
      float v[8];
      ldf8(t.g[i], at + c, dt, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) add(v[e]);
    } else {
      for (int e = c; e < c + 8 && e < n; ++e) add(ldf(t.g[i], at + e, dt));
    }
  }
  double own = (double)s;
  if (!p.norm_inf && !(s > 1e-28f && s < 1e34f)) {
    // squares that leave fp32's range: this thread's values once more in fp64 (a run of zeros, or
    // gradients below 1e-15 or above 1e16; a NaN stays one)
    own = 0.0;
    for (int c = threadIdx.x * 8; c < n; c += kThreads * 8)
      for (int e = c; e < c + 8 && e < n; ++e) {
        const double v = (double)ldf(t.g[i], at + e, dt);
        own = fma(v, v, own);
      }
  }
  const double x = block_join(own, p.norm_inf != 0);
  if (threadIdx.x == 0) p.part[p.base + blockIdx.x] = x;
}

__device__ __forceinline__ double total(const ClipParams& p) {
  double x = 0.0;
  for (int64_t k = threadIdx.x; k < p.chunks; k += kThreads) x = join(x, p.part[k], p.norm_inf != 0);
  x = block_join(x, p.norm_inf != 0);
  return p.norm_inf ? x : sqrt(x);
}

__global__ void __launch_bounds__(kThreads) total_kernel(const __grid_constant__ ClipParams p) {
  const double x = total(p);
  if (threadIdx.x == 0) *p.norm = (float)x;
}

__global__ void __launch_bounds__(kThreads) clip_kernel(const __grid_constant__ Table t, const __grid_constant__ ClipParams p) {
  const double norm = total(p);
  if (blockIdx.x == 0 && p.base == 0 && threadIdx.x == 0) *p.norm = (float)norm;
  double c = (double)p.max_norm / (norm + 1e-6);
  if (c > 1.0) c = 1.0;  // a NaN norm stays
  const float scale = (float)c;
  const int i = tensor_of(t, blockIdx.x);
  if (scale == 1.f && t.o[i] == t.g[i]) return;
  const int64_t at = (int64_t)(blockIdx.x - t.chunk0[i]) * kChunk;
  const int n = (int)(t.n[i] - at < kChunk ? t.n[i] - at : kChunk);
  const int gdt = t.gdt[i], odt = t.odt[i];
  const bool vec = all16(t.g[i]) && all16(t.o[i]);
  for (int k = threadIdx.x * 8; k < n; k += kThreads * 8) {
    if (vec && k + 8 <= n) {
      float v[8];
      ldf8(t.g[i], at + k, gdt, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] *= scale;
      if (odt == M3B_BF16) store8<__nv_bfloat16>(static_cast<__nv_bfloat16*>(t.o[i]) + at + k, v);
      else if (odt == M3B_F16) store8<__half>(static_cast<__half*>(t.o[i]) + at + k, v);
      else store8<float>(static_cast<float*>(t.o[i]) + at + k, v);
    } else {
      for (int e = k; e < k + 8 && e < n; ++e) stf(t.o[i], at + e, odt, ldf(t.g[i], at + e, gdt) * scale);
    }
  }
}

bool dtype_ok(int d) { return d == M3B_F32 || d == M3B_BF16 || d == M3B_F16; }

int64_t chunks_of(const m3b_grad_clip_args* a) {
  int64_t c = 0;
  for (int64_t i = 0; i < a->n; ++i) c += a->numel[i] > 0 ? (a->numel[i] + kChunk - 1) / kChunk : 0;
  return c;
}

}  // namespace

}  // namespace m3b

extern "C" size_t m3b_grad_clip_workspace(const m3b_grad_clip_args* a) {
  if (!a || a->n < 0 || (a->n && !a->numel)) return 0;
  return (size_t)(m3b::chunks_of(a) + 1) * 8;
}

extern "C" int m3b_grad_clip(const m3b_grad_clip_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace m3b;
  clear_error();
  if (!a || a->n < 0 || !a->norm || (a->n && (!a->grads || !a->numel || !a->grad_dtype)) ||
      (a->n && a->outs && !a->out_dtype))
    return fail(M3B_ERR_INVALID_ARG, "grad_clip: null pointer");
  if (a->norm_type != 0 && a->norm_type != 2) return fail(M3B_ERR_INVALID_ARG, "grad_clip: norm_type 2 or 0 (infinity)");
  for (int64_t i = 0; i < a->n; ++i) {
    if (a->numel[i] < 0 || !dtype_ok(a->grad_dtype[i]) || (a->outs && !dtype_ok(a->out_dtype[i])))
      return fail(M3B_ERR_INVALID_ARG, "grad_clip: tensor %lld: size or dtype", (long long)i);
    if (a->numel[i] && (!a->grads[i] || (a->outs && !a->outs[i])))
      return fail(M3B_ERR_INVALID_ARG, "grad_clip: tensor %lld: null pointer", (long long)i);
    if (a->numel[i] && a->outs && a->outs[i] == a->grads[i] && a->out_dtype[i] != a->grad_dtype[i])
      return fail(M3B_ERR_INVALID_ARG, "grad_clip: tensor %lld: in place needs one dtype", (long long)i);
  }
  const int64_t chunks = chunks_of(a);
  if (chunks > (int64_t(1) << 30)) return fail(M3B_ERR_UNSUPPORTED, "grad_clip: too many values");
  if (!workspace || workspace_bytes < (size_t)(chunks + 1) * 8)
    return fail(M3B_ERR_WORKSPACE, "grad_clip: workspace of %zu bytes", workspace_bytes);
  if (reinterpret_cast<uintptr_t>(workspace) & 7) return fail(M3B_ERR_ALIGNMENT, "grad_clip: workspace");
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  ClipParams p{static_cast<double*>(workspace), 0, chunks, a->norm_type == 0, a->max_norm, a->norm};
  for (int pass = 0; pass < (a->outs ? 2 : 1); ++pass) {
    p.base = 0;
    for (int64_t i = 0; i < a->n;) {
      Table t{};
      int c = 0;
      for (; i < a->n && t.count < kPerLaunch; ++i) {
        if (a->numel[i] == 0) continue;
        t.g[t.count] = a->grads[i];
        t.o[t.count] = a->outs ? a->outs[i] : nullptr;
        t.n[t.count] = a->numel[i];
        t.gdt[t.count] = (uint8_t)a->grad_dtype[i];
        t.odt[t.count] = a->outs ? (uint8_t)a->out_dtype[i] : 0;
        t.chunk0[t.count++] = c;
        c += (int)((a->numel[i] + kChunk - 1) / kChunk);
      }
      if (c == 0) continue;
      if (pass == 0) norm_kernel<<<c, kThreads, 0, st>>>(t, p);
      else clip_kernel<<<c, kThreads, 0, st>>>(t, p);
      p.base += c;
    }
    if (pass == 0 && (!a->outs || chunks == 0)) total_kernel<<<1, kThreads, 0, st>>>(p);
  }
  return check_launch("grad_clip");
}
