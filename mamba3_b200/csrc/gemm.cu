// Host side of the matrix-product kernel (gemm.cuh): tensor maps, launches, and the packing of
// operands that the TMA cannot read in place.
#include "gemm.cuh"

#include <mutex>

namespace m3b {

namespace {

// One thread per eight destination columns, one row of blocks per matrix: fp32 values become three bf16
// planes, 16-bit values are copied; columns past `cols` are zero (rows hold whole eights).  Bound by HBM:
// 21251 x 1408 fp32, 120 MB in and 180 out, 60 us (two columns a thread with 64-bit divisions: 84).
template <bool F32>
__global__ void pack_kernel(const __grid_constant__ PackList l) {
  pdl_wait_primary();
  pdl_launch_dependents();
  const auto& m = l.m[blockIdx.y];
  const int64_t eights = m.ld / 8, n = m.rows * eights;
  const bool small = n <= 0xffffffffll;  // a 32-bit division is several times shorter
  const bool vec = (reinterpret_cast<uintptr_t>(m.src) & 15) == 0 && m.src_ld % (F32 ? 4 : 8) == 0;
  uint16_t* dst = static_cast<uint16_t*>(m.dst);
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t r = small ? (uint32_t)i / (uint32_t)eights : i / eights, c = 8 * (i - r * eights);
    uint16_t* to = dst + r * m.ld + c;
    if constexpr (F32) {
      const float* src = static_cast<const float*>(m.src) + r * m.src_ld + c;
      float v[8];
      if (vec && c + 8 <= m.cols) {
        const float4 a = __ldg(reinterpret_cast<const float4*>(src)), b = __ldg(reinterpret_cast<const float4*>(src) + 1);
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = c + e < m.cols ? src[e] : 0.f;
      }
      uint32_t w[3][4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        uint16_t x[3], y[3];
        split_planes(v[2 * e], x);
        split_planes(v[2 * e + 1], y);
#pragma unroll
        for (int k = 0; k < 3; ++k) w[k][e] = x[k] | (uint32_t)y[k] << 16;
      }
#pragma unroll
      for (int k = 0; k < 3; ++k)
        *reinterpret_cast<uint4*>(to + k * m.plane) = make_uint4(w[k][0], w[k][1], w[k][2], w[k][3]);
    } else {
      const uint16_t* src = static_cast<const uint16_t*>(m.src) + r * m.src_ld + c;
      uint4 w;
      if (vec && c + 8 <= m.cols) {
        w = __ldg(reinterpret_cast<const uint4*>(src));
      } else {
        uint32_t x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = c + e < m.cols ? src[e] : 0;
        w = make_uint4(x[0] | x[1] << 16, x[2] | x[3] << 16, x[4] | x[5] << 16, x[6] | x[7] << 16);
      }
      *reinterpret_cast<uint4*>(to) = w;
    }
  }
}

using KernelFn = void (*)(const GemmParams);

// Single CTAs are for forward passes of at most 128 rows, kEpi*Sums for 16-bit operands; other forms are null.
template <int EPI>
KernelFn pick(bool pair, bool planes) {
  if constexpr (EPI == kEpiLseSums || EPI == kEpiDlogitSums || EPI == kEpiDgluSums) {
    if (planes) return nullptr;
    if (pair) return (KernelFn)gemm_kernel<EPI, true, false>;
    if constexpr (EPI == kEpiLseSums) return (KernelFn)gemm_kernel<EPI, false, false>;
    return nullptr;
  } else {
    if (pair) return planes ? (KernelFn)gemm_kernel<EPI, true, true> : (KernelFn)gemm_kernel<EPI, true, false>;
    if constexpr (EPI == kEpiFinal || EPI == kEpiGlu || EPI == kEpiLse)
      return planes ? (KernelFn)gemm_kernel<EPI, false, true> : (KernelFn)gemm_kernel<EPI, false, false>;
    return nullptr;
  }
}

KernelFn kernel_of(int epi, bool pair, bool planes) {
  switch (epi) {
    case kEpiStore: return pick<kEpiStore>(pair, planes);
    case kEpiFinal: return pick<kEpiFinal>(pair, planes);
    case kEpiAcc: return pick<kEpiAcc>(pair, planes);
    case kEpiGlu: return pick<kEpiGlu>(pair, planes);
    case kEpiDglu: return pick<kEpiDglu>(pair, planes);
    case kEpiLse: return pick<kEpiLse>(pair, planes);
    case kEpiLseSums: return pick<kEpiLseSums>(pair, planes);
    case kEpiDlogitSums: return pick<kEpiDlogitSums>(pair, planes);
    case kEpiDgluSums: return pick<kEpiDgluSums>(pair, planes);
    default: return pick<kEpiDlogit>(pair, planes);
  }
}

cudaLaunchConfig_t config(unsigned grid, bool pair, cudaStream_t st, cudaLaunchAttribute* at) {
  cudaLaunchConfig_t cfg{};
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = pair ? 2 : 1;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kGmThreads);
  cfg.dynamicSmemBytes = kGmSmem;
  cfg.stream = st;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  return cfg;
}

// Per device: opt the kernels into their shared memory and count the CTA pairs that can be resident.
int device_setup(int* pairs) {
  static std::mutex mu;
  static int done[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64)
    return fail(M3B_ERR_CUDA, "gemm: no current device");
  std::lock_guard<std::mutex> lk(mu);
  if (done[dev]) {
    *pairs = done[dev];
    return M3B_OK;
  }
  for (int epi = 0; epi < kEpiCount; ++epi)
    for (int k = 0; k < 4; ++k) {
      const KernelFn fn = kernel_of(epi, (k & 1) != 0, k >= 2);
      if (!fn) continue;
      const cudaError_t e = cudaFuncSetAttribute((const void*)fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kGmSmem);
      if (e != cudaSuccess) return fail(M3B_ERR_CUDA, "gemm: cudaFuncSetAttribute: %s", cudaGetErrorString(e));
    }
  cudaLaunchAttribute at[2];
  cudaLaunchConfig_t cfg = config(2 * (unsigned)(num_sms() / 2), true, nullptr, at);
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, (const void*)kernel_of(kEpiStore, true, false), &cfg) != cudaSuccess || n <= 0) {
    cudaGetLastError();
    return fail(M3B_ERR_UNSUPPORTED, "gemm: no CTA pair can be resident on this device");
  }
  done[dev] = n;
  *pairs = n;
  return M3B_OK;
}

}  // namespace

namespace {
int encode(CUtensorMap* m, const GemmOperand& o, int box_cols, int box_rows, CUtensorMapSwizzle swizzle, bool f16) {
  const EncodeTiledFn enc = encode_tiled();
  if (!enc) return fail(M3B_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
  const cuuint64_t dims[3] = {(cuuint64_t)o.cols, (cuuint64_t)o.rows, (cuuint64_t)o.planes};
  const cuuint64_t strides[2] = {(cuuint64_t)o.ld * 2, (cuuint64_t)(o.planes > 1 ? o.plane : o.rows * o.ld) * 2};
  const cuuint32_t box[3] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows, 1};
  const cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = CUDA_SUCCESS;
  for (int attempt = 0; attempt < 2; ++attempt) {
    r = enc(m, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(o.p),
            dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_ERROR_INVALID_CONTEXT) break;
    // a host thread that has made no runtime call yet (autograd's): bind the device's context to it
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaSetDevice(dev) != cudaSuccess) break;
  }
  if (r == CUDA_SUCCESS) return M3B_OK;
  return fail(M3B_ERR_CUDA, "cuTensorMapEncodeTiled refused %p: %lld x %lld, rows %lld apart, %d planes (%d)", o.p,
              (long long)o.rows, (long long)o.cols, (long long)o.ld, o.planes, (int)r);
}
}  // namespace

int gemm_map(CUtensorMap* m, const GemmOperand& o, bool mn_major, int box_rows, bool f16) {
  return encode(m, o, kGmBK, mn_major ? kGmBK : box_rows, CU_TENSOR_MAP_SWIZZLE_128B, f16);
}

int gemm_out_map(CUtensorMap* m, const GemmOperand& o, bool f16) {
  return encode(m, o, 32, 32, CU_TENSOR_MAP_SWIZZLE_64B, f16);
}

int gemm_columns(int64_t M, int64_t N, bool planes) {
  return planes || ((M + 255) / 256) * ((N + 127) / 128) <= num_sms() / 2 ? 128 : 256;
}

size_t plan_gemm(GemmParams& p, int epi, bool pair) {
  const int tile_m = gemm_tile_m(pair), tile_n = epi == kEpiGlu ? p.bn / 2 : p.bn;
  const double workers = pair ? num_sms() / 2 : num_sms();
  auto length = [&](const GemmSub& s) { return (double)(s.nk[0] + s.nk[1]) * p.npass; };
  double longest = 0.0, work = 0.0;
  for (int i = 0; i < p.nsub; ++i) {
    GemmSub& s = p.sub[i];
    s.mt = (s.M + tile_m - 1) / tile_m;
    s.nt = (s.N + tile_n - 1) / tile_n;
    s.split = 1;
    work += length(s) * s.mt * s.nt;
    longest = length(s) > longest ? length(s) : longest;
  }
  auto part_bytes = [&](const GemmSub& s, int split) { return (double)split * s.mt * tile_m * s.nt * p.bn * 4.0; };
  if (epi == kEpiStore || epi == kEpiFinal || epi == kEpiAcc) {
    // How finely to split K: the length no job may pass, from none to many small ones, by an estimate in
    // K blocks (0.36 us each).  Equal jobs finish in whole rounds; drawn ones leave half the longest
    // idle.  A split costs the parts' way out and in (3 TB/s measured: 1.1 MB a block) and a launch.
    // 16384 x 768 x 2112: 50 us whole, 94 us in two; 4096 tokens x 768 into 768 x 32000 (30 tiles of 500
    // blocks beside 375 of 39): 240 us whole, 160 us in four.
    double best = 0.0, limit = longest;
    for (double most = longest; most >= 4.0; most *= 0.8) {
      double jobs = 0.0, sum = 0.0, top = 0.0, extra = 0.0, one = 0.0;
      for (int i = 0; i < p.nsub; ++i) {
        const GemmSub& s = p.sub[i];
        const int split = (int)((length(s) + most - 1.0) / most);
        const double len = (length(s) + split - 1.0) / split + 4.0, n = (double)s.mt * s.nt * split;
        jobs += n;
        sum += n * len;
        top = len > top ? len : top;
        one = len;
        if (split > 1) extra += part_bytes(s, split + 1) / 1.1e6;
      }
      if (extra > 0.0) extra += 8.0;
      double t = sum / workers + top / 2.0 > top ? sum / workers + top / 2.0 : top;
      if (p.nsub == 1) t = (double)(int64_t)((jobs + workers - 1.0) / workers) * one;
      if (best == 0.0 || t + extra < best * 0.98) {
        best = t + extra;
        limit = most;
      }
    }
    for (int i = 0; i < p.nsub; ++i) p.sub[i].split = (int)((length(p.sub[i]) + limit - 1.0) / limit);
  }
  size_t bytes = 0;
  for (int i = 0; i < p.nsub; ++i) {
    if (p.sub[i].split < 1) p.sub[i].split = 1;
    if (p.sub[i].split > 1) bytes += (size_t)part_bytes(p.sub[i], p.sub[i].split);
  }
  for (int i = 1; i < p.nsub; ++i)  // longest jobs first
    for (int k = i; k > 0 && length(p.sub[k]) / p.sub[k].split > length(p.sub[k - 1]) / p.sub[k - 1].split; --k) {
      const GemmSub t = p.sub[k];
      p.sub[k] = p.sub[k - 1];
      p.sub[k - 1] = t;
    }
  return bytes;
}

int launch_gemm(GemmParams& p, int epi, bool pair, void* parts, cudaStream_t st) {
  int pairs = 0;
  const int rc = device_setup(&pairs);
  if (rc != M3B_OK) return rc;
  const int tile_m = gemm_tile_m(pair);
  int64_t jobs = 0, pieces = 0;
  float* at = static_cast<float*>(parts);
  for (int i = 0; i < p.nsub; ++i) {
    GemmSub& s = p.sub[i];
    jobs += (int64_t)s.mt * s.nt * s.split;
    if (s.split > 1) {
      s.part = at;
      at += (size_t)s.split * s.mt * tile_m * s.nt * p.bn;
      pieces += (int64_t)((s.M + 31) / 32) * ((s.N + 31) / 32);
    }
  }
  if (jobs == 0) return M3B_OK;
  if (jobs > (int64_t(1) << 30)) return fail(M3B_ERR_UNSUPPORTED, "gemm: too many tiles");
  const KernelFn fn = kernel_of(epi, pair, p.npass > 1);
  if (!fn) return fail(M3B_ERR_UNSUPPORTED, "gemm: no single-CTA kernel of this form");
  if (p.wait_ns == 0) p.wait_ns = kWaitLimitNs;
  const int64_t most = pair ? pairs : num_sms();
  const unsigned workers = (unsigned)(jobs < most ? jobs : most);
  cudaLaunchAttribute attr[2];
  const cudaLaunchConfig_t cfg = config(pair ? 2 * workers : workers, pair, st, attr);
  const cudaError_t e = cudaLaunchKernelEx(&cfg, fn, p);
  if (e != cudaSuccess) return fail(M3B_ERR_CUDA, "gemm_kernel: %s", cudaGetErrorString(e));
  if (pieces) {
    int split = 1, warps = 1;  // warps to a piece
    for (int i = 0; i < p.nsub; ++i) split = p.sub[i].split > split ? p.sub[i].split : split;
    while (warps < 8 && warps * 2 < split) warps *= 2;
    const unsigned grid = (unsigned)((pieces + 8 / warps - 1) / (8 / warps));
    const int rj = launch_dependent(epi == kEpiFinal ? gemm_join_kernel<kEpiFinal> : gemm_join_kernel<kEpiAcc>,
                                    dim3(grid), 256, st, p, tile_m, warps);
    if (rj != M3B_OK) return rj;
  }
  return check_launch("gemm_kernel");
}

int launch_pack(const PackList& l, int dtype, cudaStream_t st) {
  int64_t n = 0;
  for (int i = 0; i < l.n; ++i) n = l.m[i].rows * (l.m[i].ld / 8) > n ? l.m[i].rows * (l.m[i].ld / 8) : n;
  if (n == 0) return M3B_OK;
  const int64_t blocks = (n + 255) / 256, most = (int64_t)num_sms() * 16;
  const dim3 grid((unsigned)(blocks < most ? blocks : most), l.n);
  return launch_dependent(dtype == M3B_F32 ? pack_kernel<true> : pack_kernel<false>, grid, 256, st, l);
}

}  // namespace m3b
