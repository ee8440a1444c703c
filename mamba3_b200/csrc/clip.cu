// Global gradient norm over many tensors and clipping (m3b_grad_clip).
//
//   norm = sqrt(sum_i sum |g_i|^2) or max |g|;  out_i = g_i min(1, max_norm / (norm + 1e-6))
//
// Two passes over the gradients, both bound by HBM.  Every tensor is cut into chunks;
// the blocks of a grid that fills the GPU a few times walk all tensors' chunks.  The first pass leaves one
// fp64 partial per block; every block of the second adds them in the same fixed order (a few
// thousand values out of L2), so there are no atomics and no host round trip.  The second pass walks
// the chunks backwards: what the first one read last is still in L2.  The tensors' descriptions travel
// in the kernel's parameters (up to kMany tensors a launch; a small table for short lists, whose launch
// is quicker), so the call copies nothing to the device and can be captured into a CUDA graph.
// 238 M bf16 gradients into fp32: 76 us (476 MB, 6.3 TB/s) and 282 us (1.43 GB, 5.1 TB/s: reads and writes mixed
// in the ratio 1 : 2); 600 M fp32 gradients into others, 1120 us (7.2 GB with the second read, 6.4 TB/s).
#include "common.cuh"
#include "launch.h"

namespace m3b {

namespace {

constexpr int kThreads = 256;
// Bytes of a chunk in either pass: 64 or 128 a thread, in 16-byte loads that are in flight together;
// the few form (32 a thread) is for lists that would leave SMs without a chunk.
constexpr int kNormBytes = 16384, kClipBytes = 32768, kFewBytes = 8192;
constexpr int kNormBlocks = 32, kClipBlocks = 16;  // blocks per SM of a grid (8 and 4 resident: the rest even out the SMs)
constexpr int kFew = 64, kMany = 1000;  // tensors per launch: 32 bytes each, of at most 32764 bytes of parameters

template <int N>
struct Table {
  const void* g[N];
  void* o[N];
  int64_t n[N];
  int32_t chunk0[N];  // first chunk of each tensor within this launch
  uint8_t gdt[N], odt[N];
  int count, chunks, chunk;
};

struct ClipParams {
  double* part;      // one per block of all the first pass's launches
  int base, parts;   // blocks of the launches before this one; of all launches
  int norm_inf;
  float max_norm;
  float* norm;
};

template <int N>
__device__ __forceinline__ int tensor_of(const Table<N>& t, int chunk) {
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

// Eight values as they lie in memory.
template <typename T>
struct Raw {
  uint4 w[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int k = 0; k < (int)(sizeof(T) / 2); ++k) w[k] = __ldg(reinterpret_cast<const uint4*>(p) + k);
  }
  __device__ __forceinline__ void values(float (&v)[8]) const {
    const T* x = reinterpret_cast<const T*>(w);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = io<T>::ld(x + e);
  }
};

// f(offset, values, count) for this thread's runs of eight among the n values of a chunk; a whole
// aligned chunk has its loads in flight at once.
template <int BYTES, typename T, typename F>
__device__ __forceinline__ void runs(const T* g, int n, bool vec, F&& f) {
  constexpr int kRuns = BYTES / (int)sizeof(T) / kThreads / 8;
  if (vec && n == kRuns * kThreads * 8) {
    Raw<T> raw[kRuns];
#pragma unroll
    for (int k = 0; k < kRuns; ++k) raw[k].load(g + (k * kThreads + (int)threadIdx.x) * 8);
#pragma unroll
    for (int k = 0; k < kRuns; ++k) {
      float v[8];
      raw[k].values(v);
      f((k * kThreads + (int)threadIdx.x) * 8, v, 8);
    }
    return;
  }
  for (int c = (int)threadIdx.x * 8; c < n; c += kThreads * 8) {
    float v[8];
    if (vec && c + 8 <= n) {
      load8<T>(g + c, v);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = c + e < n ? io<T>::ld(g + c + e) : 0.f;
    }
    f(c, v, n - c < 8 ? n - c : 8);
  }
}

__device__ __forceinline__ int chunk_len(int bytes, int dt) { return dt == M3B_F32 ? bytes / 4 : bytes / 2; }

template <int N>
__global__ void __launch_bounds__(kThreads, 8)
    norm_kernel(const __grid_constant__ Table<N> t, const __grid_constant__ ClipParams p) {
  double all = 0.0;
  for (int chunk = blockIdx.x; chunk < t.chunks; chunk += gridDim.x) {
    const int i = tensor_of(t, chunk);
    const int dt = t.gdt[i], len = chunk_len(t.chunk, dt);
    const int64_t at = (int64_t)(chunk - t.chunk0[i]) * len;
    const int n = (int)(t.n[i] - at < len ? t.n[i] - at : len);
    const bool vec = all16(t.g[i]);
    float s = 0.f;
    auto add8 = [&](int, const float(&v)[8], int) {  // values past a short run are zeros
#pragma unroll
      for (int e = 0; e < 8; ++e)
        s = p.norm_inf ? (fabsf(v[e]) > s || v[e] != v[e] ? fabsf(v[e]) : s) : fmaf(v[e], v[e], s);
    };
    if (dt == M3B_BF16) runs<kNormBytes>(static_cast<const __nv_bfloat16*>(t.g[i]) + at, n, vec, add8);
    else if (dt == M3B_F16) runs<kNormBytes>(static_cast<const __half*>(t.g[i]) + at, n, vec, add8);
    else runs<kNormBytes>(static_cast<const float*>(t.g[i]) + at, n, vec, add8);
    double own = (double)s;
    if (!p.norm_inf && !(s > 1e-28f && s < 1e34f)) {
      // squares that leave fp32's range: the values once more in fp64 (a run of zeros, or gradients
      // below 1e-15 or above 1e16; a NaN stays one)
      own = 0.0;
      for (int c = threadIdx.x * 8; c < n; c += kThreads * 8)
        for (int e = c; e < c + 8 && e < n; ++e) {
          const double v = (double)ldf(t.g[i], at + e, dt);
          own = fma(v, v, own);
        }
    }
    all = join(all, own, p.norm_inf != 0);
  }
  const double x = block_join(all, p.norm_inf != 0);
  if (threadIdx.x == 0) p.part[p.base + blockIdx.x] = x;
}

__device__ __forceinline__ double total(const ClipParams& p) {
  double x = 0.0;
  for (int k = threadIdx.x; k < p.parts; k += kThreads) x = join(x, p.part[k], p.norm_inf != 0);
  x = block_join(x, p.norm_inf != 0);
  return p.norm_inf ? x : sqrt(x);
}

__global__ void __launch_bounds__(kThreads) total_kernel(const __grid_constant__ ClipParams p) {
  const double x = total(p);
  if (threadIdx.x == 0) *p.norm = (float)x;
}

template <typename G, typename O>
__device__ __forceinline__ void scale_runs(const G* g, O* o, int n, bool vec, float scale) {
  runs<kClipBytes>(g, n, vec, [&](int c, float(&v)[8], int len) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] *= scale;
    if (vec && len == 8) {
      store8<O>(o + c, v);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < len) io<O>::st(o + c + e, v[e]);
    }
  });
}
template <typename G>
__device__ __forceinline__ void scale_chunk(const void* src, void* o, int64_t at, int n, bool vec, int odt, float scale) {
  const G* g = static_cast<const G*>(src) + at;
  if (odt == M3B_BF16) scale_runs(g, static_cast<__nv_bfloat16*>(o) + at, n, vec, scale);
  else if (odt == M3B_F16) scale_runs(g, static_cast<__half*>(o) + at, n, vec, scale);
  else scale_runs(g, static_cast<float*>(o) + at, n, vec, scale);
}

template <int N>
__global__ void __launch_bounds__(kThreads, 4)
    clip_kernel(const __grid_constant__ Table<N> t, const __grid_constant__ ClipParams p) {
  pdl_wait_primary();
  const double norm = total(p);
  if (blockIdx.x == 0 && p.base == 0 && threadIdx.x == 0) *p.norm = (float)norm;
  double c = (double)p.max_norm / (norm + 1e-6);
  if (c > 1.0) c = 1.0;  // a NaN norm stays
  const float scale = (float)c;
  for (int chunk = t.chunks - 1 - (int)blockIdx.x; chunk >= 0; chunk -= gridDim.x) {
    const int i = tensor_of(t, chunk);
    if (scale == 1.f && t.o[i] == t.g[i]) continue;
    const int gdt = t.gdt[i], odt = t.odt[i], len = chunk_len(t.chunk, gdt);
    const int64_t at = (int64_t)(chunk - t.chunk0[i]) * len;
    const int n = (int)(t.n[i] - at < len ? t.n[i] - at : len);
    const bool vec = all16(t.g[i]) && all16(t.o[i]);
    if (gdt == M3B_BF16) scale_chunk<__nv_bfloat16>(t.g[i], t.o[i], at, n, vec, odt, scale);
    else if (gdt == M3B_F16) scale_chunk<__half>(t.g[i], t.o[i], at, n, vec, odt, scale);
    else scale_chunk<float>(t.g[i], t.o[i], at, n, vec, odt, scale);
  }
}

int64_t chunks_in(const m3b_grad_clip_args* a, int64_t i, int bytes) {
  const int64_t len = a->grad_dtype[i] == M3B_F32 ? bytes / 4 : bytes / 2;
  return (a->numel[i] + len - 1) / len;
}

// One launch of either pass over the tensors from `i` on that fit the table; returns its blocks.
template <int N>
int launch_pass(const m3b_grad_clip_args* a, int64_t* i, int pass, int chunk, const ClipParams& p, cudaStream_t st, int* rc) {
  Table<N> t;
  t.count = t.chunks = 0;
  t.chunk = chunk;
  for (; *i < a->n && t.count < N; ++*i) {
    const int64_t k = *i;
    if (a->numel[k] == 0) continue;
    t.g[t.count] = a->grads[k];
    t.o[t.count] = a->outs ? a->outs[k] : nullptr;
    t.n[t.count] = a->numel[k];
    t.gdt[t.count] = (uint8_t)a->grad_dtype[k];
    t.odt[t.count] = a->outs ? (uint8_t)a->out_dtype[k] : 0;
    t.chunk0[t.count++] = t.chunks;
    t.chunks += (int)chunks_in(a, k, chunk);
  }
  if (t.count == 0) return 0;
  const int most = num_sms() * (pass == 0 ? kNormBlocks : kClipBlocks), blocks = t.chunks < most ? t.chunks : most;
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cfg.attrs = at;
  cfg.numAttrs = pass == 1 ? 1 : 0;  // the second pass's launch overlaps the end of the first's
  const cudaError_t e = pass == 0 ? cudaLaunchKernelEx(&cfg, norm_kernel<N>, t, p) : cudaLaunchKernelEx(&cfg, clip_kernel<N>, t, p);
  if (e != cudaSuccess) *rc = fail(M3B_ERR_CUDA, "grad_clip: %s", cudaGetErrorString(e));
  return blocks;
}

bool dtype_ok(int d) { return d == M3B_F32 || d == M3B_BF16 || d == M3B_F16; }

// Partials of the first pass: at most one per block of each launch.
int64_t parts_of(const m3b_grad_clip_args* a) {
  const int64_t launches = a->n <= kFew ? 1 : (a->n + kMany - 1) / kMany;
  return launches * num_sms() * kNormBlocks;
}

}  // namespace

}  // namespace m3b

extern "C" size_t m3b_grad_clip_workspace(const m3b_grad_clip_args* a) {
  return !a || a->n < 0 ? 0 : (size_t)m3b::parts_of(a) * 8;
}

extern "C" int m3b_grad_clip(const m3b_grad_clip_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace m3b;
  clear_error();
  if (!a || a->n < 0 || !a->norm || (a->n && (!a->grads || !a->numel || !a->grad_dtype)) ||
      (a->n && a->outs && !a->out_dtype))
    return fail(M3B_ERR_INVALID_ARG, "grad_clip: null pointer");
  if (a->norm_type != 0 && a->norm_type != 2) return fail(M3B_ERR_INVALID_ARG, "grad_clip: norm_type 2 or 0 (infinity)");
  int64_t chunks = 0;
  for (int64_t i = 0; i < a->n; ++i) {
    if (a->numel[i] < 0 || !dtype_ok(a->grad_dtype[i]) || (a->outs && !dtype_ok(a->out_dtype[i])))
      return fail(M3B_ERR_INVALID_ARG, "grad_clip: tensor %lld: size or dtype", (long long)i);
    if (a->numel[i] && (!a->grads[i] || (a->outs && !a->outs[i])))
      return fail(M3B_ERR_INVALID_ARG, "grad_clip: tensor %lld: null pointer", (long long)i);
    if (a->numel[i] && a->outs && a->outs[i] == a->grads[i] && a->out_dtype[i] != a->grad_dtype[i])
      return fail(M3B_ERR_INVALID_ARG, "grad_clip: tensor %lld: in place needs one dtype", (long long)i);
    chunks += chunks_in(a, i, kClipBytes);
    if (chunks > (int64_t(1) << 28)) return fail(M3B_ERR_UNSUPPORTED, "grad_clip: too many values");
  }
  if (!workspace || workspace_bytes < (size_t)parts_of(a) * 8)
    return fail(M3B_ERR_WORKSPACE, "grad_clip: workspace of %zu bytes", workspace_bytes);
  if (reinterpret_cast<uintptr_t>(workspace) & 7) return fail(M3B_ERR_ALIGNMENT, "grad_clip: workspace");
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  ClipParams p{static_cast<double*>(workspace), 0, 0, a->norm_type == 0, a->max_norm, a->norm};
  const bool few = chunks < num_sms() * 2;
  int rc = M3B_OK;
  for (int pass = 0; pass < (a->outs && chunks ? 2 : 1); ++pass) {
    const int chunk = few ? kFewBytes : pass == 0 ? kNormBytes : kClipBytes;
    p.base = 0;
    for (int64_t i = 0; i < a->n && rc == M3B_OK;)
      p.base += a->n <= kFew ? launch_pass<kFew>(a, &i, pass, chunk, p, st, &rc)
                            : launch_pass<kMany>(a, &i, pass, chunk, p, st, &rc);
    if (rc != M3B_OK) return rc;
    if (pass == 0) p.parts = p.base;
  }
  if (!a->outs || chunks == 0) total_kernel<<<1, kThreads, 0, st>>>(p);
  return check_launch("grad_clip");
}
